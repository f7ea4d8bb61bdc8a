"""Layer norm over the last axis, with a weight and bias per column or per head and column.

    y = (x - mean) * rstd * weight + bias

`weight` and `bias` [C] are the usual norm of a model's width; [H,C] norm each head's output of a recurrence by itself, on
`[B,T,H,C]` tensors as the operators of this package return them.  The kernels are in csrc/layer_norm.hip; what is said in
`linear.py` on streams, graphs and devices holds here too.
"""
from __future__ import annotations

from typing import Optional

import torch as th

from . import handwritten as hw
from .handwritten import DTYPES, require

SOURCE = 'layer_norm.hip'
MAX_COLUMNS = 16384
THREADS = 256 * 2 * 256         # in flight: two workgroups of 256 per compute unit (measured from one half to sixteen: 5.0 TB/s at two, 3.9 at eight)

_ARGS = '3q2q2q11qd'


def _shape_rule(C: int, dtype: th.dtype):
    """(WIDE, threads, 16-byte pieces per lane, lanes per row): a row stays in the registers of up to 64 lanes with four
    pieces each; wider rows take a workgroup of 256, then 1024 threads."""
    pieces = -(-C * (4 if dtype == th.float32 else 2) // 16)
    for k in (1, 2, 4):
        if pieces <= 64 * k:
            lanes = 1
            while lanes * k < pieces:
                lanes *= 2
            return 0, 256, k, lanes
    k = 4 if dtype == th.float32 else 2
    return (1, 256, k, 256) if pieces <= 256 * k else (1, 1024, k, 1024)


def _defines(C, dtype, backward):
    wide, threads, k, lanes = _shape_rule(C, dtype)
    return (('IN', DTYPES[dtype]), ('K', k), ('TH', threads), ('GL', lanes), ('WIDE', wide), ('BACKWARD', int(backward)))


def builds():
    """Every code object of this module: (source, kernel, defines)."""
    out = set()
    for dt in DTYPES:
        for C in (1 << i for i in range(MAX_COLUMNS.bit_length())):
            out |= {(SOURCE, 'ln_fw', _defines(C, dt, False)), (SOURCE, 'ln_bw', _defines(C, dt, True))}
    return sorted(out)


def _rows(x: th.Tensor, per_head: bool):
    """`x` as (tensor, outer stride, head stride): the dimensions in front of the heads as one, copied only if they cannot be."""
    lead = x.shape[:-2] if per_head else x.shape[:-1]
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    for _ in range(2):
        dims = [(n, s) for n, s in zip(lead, x.stride()) if n != 1]
        if all(dims[i][1] == dims[i + 1][0] * dims[i + 1][1] for i in range(len(dims) - 1)):
            break
        x = x.contiguous()
    return x, dims[-1][1] if dims else 0, x.stride(-2) if per_head else 0


def _wide(x, C, *strides):
    size = x.element_size()
    return C * size % 16 == 0 and x.data_ptr() % 16 == 0 and all(s * size % 16 == 0 for s in strides)


def _launch(name, x, dy, out, weight, bias, dw, db, heads, teams, eps, lanes, strides):
    C = x.shape[-1]
    defines = _defines(C, x.dtype, name == 'ln_bw')
    threads, wide = defines[2][1], defines[4][1]
    vec = _wide(x, C, *strides[:2]) and (dy is None or _wide(dy, C, *strides[2:]))
    grid = teams if wide else -(-teams * lanes // threads)
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    code = lambda t: 2 if t is None else DTYPES[t.dtype]  # noqa: E731
    hw.launch(hw.kernel(x.device, SOURCE, name, defines), x.device, grid, threads, _ARGS, x.data_ptr(), ptr(dy), out.data_ptr(), ptr(weight), ptr(bias),
              ptr(dw), ptr(db), x.numel() // C, heads, C, *strides, code(weight), code(bias), int(vec), teams, eps)


def _teams(x, heads):
    """(teams, lanes per team): as many rows side by side as keep the chip busy, a multiple of `heads` (a team keeps its head)."""
    C = x.shape[-1]
    lanes = _shape_rule(C, x.dtype)[3]
    outers = x.numel() // C // heads
    return min(outers, max(1, THREADS // (lanes * heads))) * heads, lanes


def _per_head(x, weight, bias):
    p = weight if weight is not None else bias
    return p is not None and p.ndim == 2


def _forward(x, weight, bias, eps):
    y = th.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y
    per_head = _per_head(x, weight, bias)
    heads = x.shape[-2] if per_head else 1
    x, so, sh = _rows(x, per_head)
    teams, lanes = _teams(x, heads)
    _launch('ln_fw', x, None, y, weight, bias, None, None, heads, teams, eps, lanes, (so, sh, 0, 0))
    return y


def _backward(x, weight, bias, dy, eps, need_w, need_b):
    dx = th.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = th.empty(weight.shape, dtype=weight.dtype, device=x.device) if need_w else None
    db = th.empty(bias.shape, dtype=bias.dtype, device=x.device) if need_b else None
    C = x.shape[-1]
    if x.numel() == 0:
        for t in (dw, db):
            if t is not None:
                t.zero_()
        return dx, dw, db
    per_head = _per_head(x, weight, bias)
    heads = x.shape[-2] if per_head else 1
    x, so, sh = _rows(x, per_head)
    dy, yo, yh = _rows(dy, per_head)
    teams, lanes = _teams(x, heads)
    pw = th.empty((teams, C), dtype=th.float32, device=x.device) if need_w else None
    pb = th.empty((teams, C), dtype=th.float32, device=x.device) if need_b else None
    _launch('ln_bw', x, dy, dx, weight, None, pw, pb, heads, teams, eps, lanes, (so, sh, yo, yh))
    hw.slice_sums([(p, d) for p, d in ((pw, dw), (pb, db)) if p is not None], teams // heads)
    return dx, dw, db


_lib = th.library.Library('flex_rnn', 'FRAGMENT')
_lib.define('layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor')
_lib.define('layer_norm_backward(Tensor x, Tensor? weight, Tensor? bias, Tensor dy, float eps, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)')


def _backward_op(x, weight, bias, dy, eps, need_w, need_b):
    return tuple(x.new_empty(0) if t is None else t for t in _backward(x, weight, bias, dy, eps, need_w, need_b))


_lib.impl('layer_norm', _forward, 'CUDA')
_lib.impl('layer_norm_backward', _backward_op, 'CUDA')


@th.library.register_fake('flex_rnn::layer_norm', lib=_lib)
def _(x, weight, bias, eps):
    return x.new_empty(x.shape)


@th.library.register_fake('flex_rnn::layer_norm_backward', lib=_lib)
def _(x, weight, bias, dy, eps, need_w, need_b):
    return x.new_empty(x.shape), weight.new_empty(weight.shape) if need_w else x.new_empty(0), bias.new_empty(bias.shape) if need_b else x.new_empty(0)


_fw_op = th.ops.flex_rnn.layer_norm.default
_bw_op = th.ops.flex_rnn.layer_norm_backward.default


class _LayerNorm(th.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.eps = eps
        return _fw_op(x, weight, bias, eps)

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = hw.once(_bw_op, x, weight, bias, dy, ctx.eps, need[1], need[2])
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None


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

    Sums are fp32 (mean first, then squares of the differences).  Differentiable once in x, weight and bias; gradients are
    deterministic.
    """
    _check(x, weight, bias)
    weight, bias = (p if p is None or p.is_contiguous() else p.contiguous() for p in (weight, bias))
    if th.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _fw_op(x, weight, bias, float(eps))


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
