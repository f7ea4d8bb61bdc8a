"""Layer norm over the last axis, with a weight and bias per column or per head and column.

    y = (x - mean) * rstd * weight + bias

`weight` and `bias` [C] are the usual norm of a model's width; [H,C] norm each head's output of a recurrence by itself, on
`[B,T,H,C]` tensors as the operators of this package return them.  The kernels are in csrc/layer_norm.hip; what is said in
`linear.py` on streams, graphs, transforms and devices holds here too.
"""
from __future__ import annotations

from typing import Optional

import torch as th

from . import handwritten as hw
from .handwritten import DTYPES, require

MAX_COLUMNS = 16384


def _check(x, weight, bias):
    C = x.shape[-1] if x.ndim else 0
    fits = lambda p: p is None or ((p.shape == (C,) or p.shape == x.shape[-2:]) and p.dtype in (x.dtype, th.float32) and p.device == x.device)  # noqa: E731
    if 1 <= C <= MAX_COLUMNS and x.dtype in DTYPES and x.device.type in _DEVICES and fits(weight) and fits(bias) \
            and (weight is None or bias is None or weight.shape == bias.shape):
        return
    what = 'layer_norm'
    require(x.ndim >= 1 and x.dtype in DTYPES, f'{what}: x is bfloat16, float16 or float32 with at least one dimension (got {x.dtype} {list(x.shape)})')
    require(1 <= C <= MAX_COLUMNS, f'{what}: rows of 1 to {MAX_COLUMNS} columns (got {C})')
    for name, p in (('weight', weight), ('bias', bias)):
        if p is not None:
            require(p.shape == (C,) or p.shape == x.shape[-2:], f'{what}: {name} is [C] = [{C}] or [H, C] of x {list(x.shape)} (got {list(p.shape)})')
            require(p.dtype in (x.dtype, th.float32), f'{what}: {name} is float32 or of the type of x (got {p.dtype})')
            require(p.device == x.device, f'{what}: all tensors must live on the same device ({p.device} and {x.device})')
    require(weight is None or bias is None or weight.shape == bias.shape, f'{what}: weight and bias have the same shape')
    require(False, f'{what} runs on the GPU only (got a {x.device} tensor); `.naive` is plain PyTorch')


_DEVICES = ('cuda', 'meta')


def layer_norm(x: th.Tensor, weight: Optional[th.Tensor] = None, bias: Optional[th.Tensor] = None, eps: float = 1e-5) -> th.Tensor:
    """Layer norm of each row `x[..., :]`.

    x       [..., C], bfloat16, float16 or float32, C from 1 to 16384, any strides (a layout whose leading dimensions do not
            fold into one, or whose columns are not next to each other, is copied first)
    weight, bias  [C], or [H,C] with x [..., H, C]; float32 or the type of x; None: one, zero

    Sums are fp32 (mean first, then squares of the differences).  Differentiable once, backwards, in x, weight and
    bias (a forward-mode tangent is refused); gradients are deterministic.
    """
    _check(x, weight, bias)
    weight, bias = (p if p is None or p.is_contiguous() else p.contiguous() for p in (weight, bias))
    return hw.op('layer_norm')(x, weight, bias, float(eps))


def _naive(x, weight=None, bias=None, eps=1e-5, dtype=th.float32):
    """The same operator in plain PyTorch (any device, differentiable), computed in `dtype`."""
    z = x.to(dtype)
    z = z - z.mean(-1, keepdim=True)
    z = z / ((z * z).mean(-1, keepdim=True) + eps).sqrt()
    z = z if weight is None else z * weight.to(dtype)
    z = z if bias is None else z + bias.to(dtype)
    return z.to(x.dtype)


layer_norm.naive = _naive
layer_norm.naive_fp64 = lambda *args, **kwargs: _naive(*args, **kwargs, dtype=th.double)
