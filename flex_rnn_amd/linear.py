"""Linear attention with a decay for each head, as block products on the matrix cores.

    S_t = exp(g_t) S_(t-1) + v_t k_t^T,    y_t = scale * S_t q_t

The recurrence of `ops.retention` and `ops.mamba2` (and of `ops.gla` with one gate per head), whose decay is a number per
token and head: a block of tokens is then a handful of matrix products, where `jit` walks the sequence a token at a time.
Recurrences whose decay differs along the state's columns, or that read the state to update it (delta rules), are `jit`'s.

    y, state = linear_attention(q, k, v, g, state)              # a prompt, or training (differentiable)
    y = linear_attention_step(q, k, v, g, state)                # one token; `state` is updated in place

The kernels are in csrc/linear_attention.hip, their launches and gradients in csrc/frnn_ops.cpp.  Like the compiled operators
they run on the GPU only, on the current stream of the tensors' device, without synchronising, and can be captured into a HIP
graph after a first call with the same types, sizes and layouts (a captured backward pass: while no graph of the same leaves
from the default stream is alive; it says so).  `torch.func.vmap` runs them once per element; a step under vmap and
`torch.func.grad` are errors.  `linear_attention.naive` and `linear_attention.naive_fp64` are the per-token loop
in plain PyTorch.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch as th

from . import handwritten as hw
from .handwritten import DTYPES, require

MAX_HEAD = 256                  # largest M and N
MAX_TOKENS = 2 ** 31 - 65       # longest sequence (positions are 32 bits, rounded up to blocks)
MAX_ROW = 2 ** 24 - 1           # a token's elements over all heads (offsets within a block of 32 tokens are 31 bits)


def _check(q, k, v, g, state, lead, what, types=True):
    """Argument checks shared by the prompt and the single-token form; `lead`: the dimensions in front of the heads."""
    n, sq, sv, dt = len(lead), q.shape, v.shape, q.dtype
    if len(sq) == len(sv) == n + 2 and sq == k.shape and sq[:n] == sv[:n] and sq[n] >= 1 and sv[n] >= 1 and sv[n] % sq[n] == 0 \
            and 1 <= sq[-1] <= MAX_HEAD and 1 <= sv[-1] <= MAX_HEAD and (n == 1 or sq[1] <= MAX_TOKENS and sv[2] * sv[3] <= MAX_ROW and sq[2] * sq[3] <= MAX_ROW) \
            and dt in DTYPES and k.dtype == dt and v.dtype == dt and g.dtype in (dt, th.float32) and g.shape in (sv[n:n + 1], sv[:n + 1]) \
            and (state is None or (state.shape == (sq[0], sv[n], sv[-1], sq[-1]) and state.dtype in (dt, th.float32))):
        return
    names = '[' + ', '.join(lead) + ', '
    require(q.ndim == n + 2 and k.ndim == n + 2 and v.ndim == n + 2, f'{what}: q and k are {names}Hk, N] and v is {names}H, M]')
    require(q.shape == k.shape, f'{what}: q {list(q.shape)} and k {list(k.shape)} differ')
    require(q.shape[:n] == v.shape[:n], f'{what}: q {list(q.shape)} and v {list(v.shape)} differ in {names[1:-2]}')
    B, Hk, N = q.shape[0], q.shape[-2], q.shape[-1]
    H, M = v.shape[-2], v.shape[-1]
    require(Hk >= 1 and H >= 1 and H % Hk == 0, f'{what}: {H} heads of v do not divide into {Hk} heads of q and k')
    require(1 <= N <= MAX_HEAD and 1 <= M <= MAX_HEAD, f'{what}: head sizes from 1 to {MAX_HEAD} (q and k have {N}, v has {M})')
    require(n == 1 or q.shape[1] <= MAX_TOKENS, f'{what}: sequences of up to {MAX_TOKENS} tokens')
    require(n == 1 or H * M <= MAX_ROW and Hk * N <= MAX_ROW, f'{what}: a token has up to {MAX_ROW} elements over all heads (v has {H * M}, q and k {Hk * N})')
    require(not types or dt in DTYPES and dt == k.dtype == v.dtype, f'{what}: q, k and v are of one type, bfloat16, float16 or float32 (got {dt}, {k.dtype}, {v.dtype})')
    require(not types or g.dtype in (dt, th.float32), f'{what}: g is float32 or of the type of q (got {g.dtype})')
    require(tuple(g.shape) in ((H,), (*v.shape[:n], H)), f'{what}: g is [H] or {names}H] with H = {H} (got {list(g.shape)})')
    require(state is None or tuple(state.shape) == (B, H, M, N), f'{what}: the state is [B, H, M, N] = {[B, H, M, N]} (got {list(state.shape) if state is not None else None})')
    require(state is None or not types or state.dtype in (dt, th.float32), f'{what}: the state is float32 or of the type of q (got {state.dtype if state is not None else None})')


def _check_device(what, first, *others):
    dev = first.device
    if dev.type not in ('cuda', 'meta'):
        require(False, f'{what} runs on the GPU only (got a {dev} tensor); `.naive` is the plain PyTorch loop')
    for t in others:
        if t is not None and t.device != dev:
            require(False, f'{what}: all tensors must live on the same device ({t.device} and {dev})')


def linear_attention(q: th.Tensor, k: th.Tensor, v: th.Tensor, g: th.Tensor, state: Optional[th.Tensor] = None, *,
                     lengths: Optional[th.Tensor] = None, scale: float = 1.0) -> Tuple[th.Tensor, th.Tensor]:
    """`S_t = exp(g_t) S_(t-1) + v_t k_t^T`, `y_t = scale * S_t q_t` over whole sequences; returns `(y, final state)`.

    q, k    [B,T,Hk,N]; Hk divides H (heads h * Hk // H share a query and key)
    v       [B,T,H,M], of the same type (bfloat16, float16, float32); M and N from 1 to 256, T from 0
    g       the decay's logarithm, [B,T,H] or [H], float32 or the type of q; -inf forgets everything before the token
            (and its gradient is zero, as wherever exp(g) is)
    state   [B,H,M,N], float32 or the type of q; None: zero, and the final state is float32
    lengths [B], int64 or int32: sequence b ends after `lengths[b]` tokens (clamped to 0..T); what is behind is not
            looked at, its `y` and gradients are zero, and the final state is the one after the last real token

    Any strides.  Sums and the state are fp32.  Differentiable once, backwards, in q, k, v, g and state (a forward-mode tangent is
    refused); gradients are deterministic (which of them are asked for may change the last bit of the others).  An infinity or
    NaN in q, k, v or a result's gradient leaves NaN in what it is a factor of, and nothing else (but in the gradient of g: up to
    255 tokens in front of it, too).
    """
    _check(q, k, v, g, state, ('B', 'T'), 'linear_attention')
    _check_device('linear_attention', q, k, v, g, state, lengths)
    if lengths is not None:
        require(tuple(lengths.shape) == (q.shape[0],) and lengths.dtype in (th.int64, th.int32),
                f'linear_attention: lengths is int64 or int32 [B] = [{q.shape[0]}] (got {lengths.dtype} {list(lengths.shape)})')
        lengths = lengths.to(th.int64).contiguous()
    return hw.op('linear_attention')(q, k, v, g, state, lengths, float(scale))


def linear_attention_step(q: th.Tensor, k: th.Tensor, v: th.Tensor, g: th.Tensor, state: th.Tensor, *, scale: float = 1.0) -> th.Tensor:
    """One token of `linear_attention` for decoding: `state` [B,H,M,N] is updated in place, y [B,H,M] is returned.

    q, k [B,Hk,N], v [B,H,M], g [B,H] or [H]; types as there.  Any strides, except that no two elements of the state may
    share memory, nor may one with another argument.  Not differentiable (inputs that want gradients or have a
    tangent are refused): with T = 1, `linear_attention` is.
    """
    _check(q, k, v, g, state, ('B',), 'linear_attention_step')
    _check_device('linear_attention_step', q, k, v, g, state)
    if th.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or state.requires_grad):
        require(False, 'linear_attention_step updates the state in place and cannot be differentiated: use linear_attention, or th.no_grad()')
    if not state.is_contiguous():
        require(not _overlaps(state), 'linear_attention_step: elements of the state share memory')
    return hw.op('linear_attention_step')(q, k, v, g, state, float(scale))


def _overlaps(t: th.Tensor) -> bool:
    """Whether two indices of `t` may name the same element (the dimensions do not nest)."""
    end = 0
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= end:
            return True
        end += stride * (size - 1)
    return False


def _naive(q, k, v, g, state=None, *, lengths=None, scale=1.0, dtype=th.float32):
    """The same operator as a loop over tokens in plain PyTorch (any device and type, differentiable), computed in `dtype`."""
    _check(q, k, v, g, state, ('B', 'T'), 'linear_attention', types=False)
    B, T, Hk, N = q.shape
    H, M = v.shape[2:]
    s_dtype = th.float32 if state is None else state.dtype
    S = th.zeros(B, H, M, N, dtype=dtype, device=q.device) if state is None else state.to(dtype)
    ys = []
    for t in range(T):
        qt, kt = (x[:, t].to(dtype).repeat_interleave(H // Hk, 1)[..., None, :] for x in (q, k))
        gt = g.to(dtype).expand(B, H) if g.ndim == 1 else g[:, t].to(dtype)
        new = gt.exp()[..., None, None] * S + v[:, t].to(dtype)[..., None] * kt
        yt = (new * qt).sum(-1) * scale
        if lengths is not None:
            real = (t < lengths)[:, None, None]
            new, yt = th.where(real[..., None], new, S), th.where(real, yt, 0.0)
        S = new
        ys.append(yt)
    y = th.stack(ys, 1) if ys else v.new_empty(B, 0, H, M, dtype=dtype)
    return y.to(v.dtype), S.to(s_dtype)


def _naive_fp64(*args, **kwargs):
    return _naive(*args, **kwargs, dtype=th.double)


linear_attention.naive = _naive
linear_attention.naive_fp64 = _naive_fp64

hw.load_if_built()
