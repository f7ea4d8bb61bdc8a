"""Linear attention with a decay for each head, as block products on the matrix cores.

    S_t = exp(g_t) S_(t-1) + v_t k_t^T,    y_t = scale * S_t q_t

The recurrence of `ops.retention` and `ops.mamba2` (and of `ops.gla` with one gate per head), whose decay is a number per
token and head: a block of tokens is then a handful of matrix products, where `jit` walks the sequence a token at a time.
Recurrences whose decay differs along the state's columns, or that read the state to update it (delta rules), are `jit`'s.

    y, state = linear_attention(q, k, v, g, state)              # a prompt, or training (differentiable)
    y = linear_attention_step(q, k, v, g, state)                # one token; `state` is updated in place

The kernels are in csrc/linear_attention.hip.  Like the compiled operators they run on the GPU only, on the current stream of
the tensors' device, without synchronising, and can be captured into a HIP graph after a first call with the same types
and head sizes; `linear_attention.naive` and `linear_attention.naive_fp64` are the per-token loop in plain PyTorch.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch as th

from . import handwritten as hw
from .handwritten import DTYPES, require

SOURCE = 'linear_attention.hip'
MAX_HEAD = 256                  # largest M and N
MAX_TOKENS = 2 ** 31 - 65       # longest sequence (positions are 32 bits, rounded up to blocks)
WIDTHS = (64, 128, 256)         # what M and N are padded to
BLOCK = 32                      # tokens per block
WORKGROUPS = 512                # two per compute unit: below this a sequence is split into segments
MAX_SEGMENTS = 16
BORDER = 8                      # blocks between the borders at which the gradient of g starts anew

# argument blocks (see the structs in the source): Tensor 6 fields, Gate 5, States 6
_JOB = struct.Struct('<6q6q6q6q6q6q7q5q8q2d')
_BLOCK = struct.Struct('<5qq6q')
_GATE = '3q5qqq5q'
_STEP = '6q6q6q5q6qq8qd'


def _width(n: int) -> int:
    return next(w for w in WIDTHS if n <= w)


def _block_defines(dtype, width, out=1, dots=0, fast=1, wide=0):
    w = _width(width)
    nbuf = 2 if dtype == th.bfloat16 and w <= 128 else 1
    occ = 2
    return (('KERNEL_BLOCK', 1), ('IN', DTYPES[dtype]), ('W', w), ('OUT', out), ('DOTS', dots), ('FAST', fast), ('WIDE', wide), ('NBUF', nbuf), ('OCC', occ))


_GATE_DEFINES = (('KERNEL_GATE', 1), ('IN', 0))


def _step_defines(dtype):
    return (('KERNEL_STEP', 1), ('IN', DTYPES[dtype]))


def builds():
    """Every code object of this module: (source, kernel, defines)."""
    out = [(SOURCE, 'la_gate', _GATE_DEFINES)]
    for dt in DTYPES:
        out.append((SOURCE, 'la_step', _step_defines(dt)))
        for w in WIDTHS:
            out += [(SOURCE, 'la_block', _block_defines(dt, w, *x)) for x in
                    [(o, d, fast, 0) for o, d in ((1, 0), (1, 1), (0, 0)) for fast in (0, 1)] + [(1, d, 1, 1) for d in (0, 1) if dt != th.float32]]
    return out


# ------------------------------------------------------------------ argument blocks
def _tensor(t: th.Tensor, time: bool):
    """Fields of struct Tensor for [batch, (time,) heads, width]."""
    at, size = t.data_ptr(), t.element_size()
    if time:
        sb, st, sh, sn = t.stride()
    else:
        (sb, sh, sn), st = t.stride(), 0
    wide = sn == 1 and t.shape[-1] % 8 == 0 and (at | sb * size | st * size | sh * size) % 16 == 0
    return at, sb, st, sh, sn, int(wide)


def _near(t: th.Tensor) -> th.Tensor:
    """`t` [B,T,heads,n], copied if a block of its tokens spans more than the 31 bits that offsets within a block have."""
    return t if (BLOCK * t.stride(1) + MAX_HEAD * t.stride(3)) * t.element_size() < 2 ** 31 else t.contiguous()


def _gate(g: th.Tensor):
    code = DTYPES[g.dtype]
    if g.ndim == 1:
        return g.data_ptr(), 0, 0, g.stride(0), code
    if g.ndim == 2:
        return g.data_ptr(), g.stride(0), 0, g.stride(1), code
    return g.data_ptr(), g.stride(0), g.stride(1), g.stride(2), code


def _states(s: Optional[th.Tensor]):
    """[B,H,M,N] with rows N, columns M (as the walks that produce y and dv hold it)."""
    return (0, 0, 0, 0, 0, 2) if s is None else (s.data_ptr(), s.stride(0), s.stride(1), s.stride(3), s.stride(2), DTYPES[s.dtype])


def _states_t(s: Optional[th.Tensor]):
    """[B,H,M,N] with rows M, columns N (dq and dk)."""
    return (0, 0, 0, 0, 0, 2) if s is None else (s.data_ptr(), *s.stride(), DTYPES[s.dtype])


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _segments(groups: int, blocks: int) -> Tuple[int, int]:
    """(segments, blocks per segment) of a walk over `blocks` blocks by `groups` workgroups side by side."""
    n = min(-(-WORKGROUPS // max(groups, 1)), blocks // 16, MAX_SEGMENTS)
    if n <= 1:
        return 1, blocks
    per = -(-blocks // n)
    return -(-blocks // per), per


# ------------------------------------------------------------------ launches
_NO_TENSOR = (0, 0, 0, 0, 0, 1)
_NO_JOB = bytes(_JOB.size)
_OUT_TYPE = 6 * 6 + 6           # its field


class _Role:
    """One operand of a walk: its tensor, argument fields and heads."""

    def __init__(self, t: th.Tensor):
        self.fields, self.heads = _tensor(t, True), t.shape[2]


def _job(q, k, v, x, width, C, init, fin, out, strides, out_type, back=0, pairs=0, in_scale=1.0, out_scale=1.0, dots=0, marks=0, inner=0):
    """The fields of struct Job that are known before segments are; `local` and `totals` follow in `_walk`."""
    return [(*q.fields, *k.fields, *v.fields, *(_NO_TENSOR if x is None else x.fields), *init, *fin, out, *strides, out_type, dots, marks, inner),
            (q.heads, k.heads, v.heads, 1 if x is None else x.heads, width, C, back, pairs, in_scale, out_scale),
            C % 4 == 0 and all(r is None or r.fields[5] for r in (q, k, v, x))]


_block_kernels = {}


def _block_kernel(dev, *key):
    k = _block_kernels.get((dev.index, key))
    if k is None:
        k = _block_kernels[dev.index, key] = hw.kernel(dev, SOURCE, 'la_block', _block_defines(*key))
    return k


def _walk(dev, dtype, jobs, gate, lengths, B, T, H, dots=0):
    """Runs up to two walks of one width side by side, each in segments where the batch alone does not fill the chip."""
    width = _width(jobs[0][1][4])
    tiles = max(-(-j[1][5] // 64) for j in jobs)
    blocks = -(-T // BLOCK)
    nseg, per = _segments(len(jobs) * B * H * tiles, blocks)
    fast = int(all(j[2] for j in jobs))
    wide = int(fast and jobs[0][0][_OUT_TYPE] == 2 and dtype != th.float32)
    size = B * H * (nseg - 1)
    local = totals = None
    if nseg > 1:
        local = th.empty((len(jobs), size * tiles * 64 * width), dtype=th.float32, device=dev)
        totals = th.empty((len(jobs), size), dtype=th.float64, device=dev)
    blob = b''.join([_JOB.pack(*head, 0 if local is None else local[i].data_ptr(), 0 if totals is None else totals[i].data_ptr(), *tail)
                     for i, (head, tail, _) in enumerate(jobs)] + [_NO_JOB] * (2 - len(jobs))
                    + [_BLOCK.pack(*gate, _ptr(lengths), B, T, H, nseg, per, tiles)])
    for out in ((0, 1) if nseg > 1 else (1,)):
        k = _block_kernel(dev, dtype, width, out, dots if out else 0, fast, wide if out else 0)
        groups = B * H * (nseg if out else nseg - 1)
        hw.launch_bytes(k, dev, -(-groups // 8) * 8 * tiles, len(jobs), 256, blob)


def _forward(q, k, v, g, state, lengths, scale):
    B, T, Hk, N = k.shape
    H, M = v.shape[2], v.shape[3]
    dev = q.device
    q, k, v = _near(q), _near(k), _near(v)
    y = th.empty((B, T, H, M), dtype=v.dtype, device=dev)
    out = th.empty((B, H, M, N), dtype=th.float32, device=dev) if state is None else th.empty_like(state)
    job = _job(_Role(q), _Role(k), _Role(v), None, N, M, _states(state), _states(out), y.data_ptr(), (T * H * M, H * M, M, 0, 1), DTYPES[v.dtype], out_scale=scale)
    _walk(dev, q.dtype, [job], _gate(g), lengths, B, T, H)
    return y, out


def _backward(q, k, v, g, state, lengths, dy, dstate, scale, need_g, need_state):
    B, T, Hk, N = k.shape
    H, M = v.shape[2], v.shape[3]
    dev, dt = q.device, q.dtype
    q, k, v, dy = _near(q), _near(k), _near(v), _near(dy)
    gate = _gate(g)
    dq, dk, dv = (th.empty(x.shape, dtype=dt, device=dev) for x in (q, k, v))
    ds = th.empty_like(state) if need_state else None
    # heads that share a query and key each have their own share of its gradient
    share = H // Hk
    pq, pk, type_ = (dq, dk, DTYPES[dt]) if share == 1 else (*th.empty((2, share, B, T, Hk, N), dtype=th.float32, device=dev), 2)
    strides = (T * Hk * N, Hk * N, N, B * T * Hk * N, share)
    rq, rk, rv, ry = (_Role(t) for t in (q, k, v, dy))
    none, extra = _states(None), [{}, {}]
    tiles, blocks = -(-N // 64), -(-T // BLOCK)
    if need_g:
        borders = -(-blocks // BORDER) + 2
        dots = th.empty((2, tiles, B * H, T), dtype=th.float32, device=dev)
        marks = th.empty(B * H * borders * -(-N // 16) * 16 * _width(M), dtype=th.float32, device=dev)
        inner = th.empty((B * H * borders, tiles * 4), dtype=th.float64, device=dev)
        extra = [dict(dots=d.data_ptr(), marks=marks.data_ptr(), inner=inner.data_ptr()) for d in dots]
    of_q = _job(ry, rv, rk, rq, M, N, _states_t(state), none, pq.data_ptr(), strides, type_, pairs=1, out_scale=scale, **extra[0])
    of_k = _job(rv, ry, rq, rk, M, N, _states_t(dstate), _states_t(ds), pk.data_ptr(), strides, type_, back=1, in_scale=scale, **extra[1])
    of_v = _job(rk, rq, ry, None, N, M, _states(dstate), none, dv.data_ptr(), (T * H * M, H * M, M, 0, 1), DTYPES[dt], back=1, in_scale=scale)
    # dq's walk multiplies with what dk's wrote down, so it comes later.  dv's goes along with dk's, at the price of dk's three
    # parts of the state, where one kernel serves both and the chip has room for them side by side (B2 T500 H8 64x48 fp32:
    # 21 us less); by itself it takes two thirds of the time.
    together = _width(M) == _width(N) and (share == 1 or dt == th.float32) and 2 * B * H * max(tiles, -(-M // 64)) <= WORKGROUPS
    for jobs, dots_ in (([of_k, of_v] if together else [of_k], 1), ([of_q], 1)) if need_g else (([of_q, of_k], 0),):
        _walk(dev, dt, jobs, gate, lengths, B, T, H, dots=dots_)
    if not (need_g and together):
        _walk(dev, dt, [of_v], gate, lengths, B, T, H)
    if share > 1:
        hw.slice_sums([(pq, dq), (pk, dk)], share)
    dg = None
    if need_g:
        per_head = g.ndim == 1
        dg = th.empty(g.shape, dtype=g.dtype, device=dev)
        out = th.empty((B, T, H), dtype=th.float32, device=dev) if per_head else dg
        hw.launch(hw.kernel(dev, SOURCE, 'la_gate', _GATE_DEFINES), dev, B * H * -(-blocks // 32), 1024, _GATE,
                  dots[0].data_ptr(), dots[1].data_ptr(), inner.data_ptr(), *gate, out.data_ptr(), _ptr(lengths), B, T, H, tiles, DTYPES[out.dtype])
        if per_head:
            hw.slice_sums([(out, dg)], B * T)
    return dq, dk, dv, dg, ds


def _step(q, k, v, g, state, scale):
    B, Hk, N = k.shape
    H, M = v.shape[1], v.shape[2]
    dev = q.device
    y = th.empty((B, H, M), dtype=v.dtype, device=dev)
    size = state.element_size()
    ve = 16 // size
    wide = state.stride(3) == 1 and N % ve == 0 and state.data_ptr() % 16 == 0 and all(state.stride(i) * size % 16 == 0 for i in range(3))
    lanes = 1
    while lanes < 64 and lanes * (ve if wide else 1) < N:
        lanes *= 2
    rows = min(M, 256 // lanes * 4)
    hw.launch(hw.kernel(dev, SOURCE, 'la_step', _step_defines(q.dtype)), dev, B * H * -(-M // rows), 256, _STEP,
              *_tensor(q, False), *_tensor(k, False), *_tensor(v, False), *_gate(g), *_states_t(state), y.data_ptr(),
              B, H, Hk, M, N, int(wide), lanes, rows, scale)
    return y


# ------------------------------------------------------------------ operators
_lib = th.library.Library('flex_rnn', 'FRAGMENT')
_lib.define('linear_attention(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? state, Tensor? lengths, float scale) -> (Tensor, Tensor)')
_lib.define('linear_attention_backward(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? state, Tensor? lengths, Tensor dy, Tensor? dstate, '
            'float scale, bool need_g, bool need_state) -> (Tensor, Tensor, Tensor, Tensor, Tensor)')
_lib.define('linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor g, Tensor(a!) state, float scale) -> Tensor')


def _backward_op(q, k, v, g, state, lengths, dy, dstate, scale, need_g, need_state):
    out = _backward(q, k, v, g, state, lengths, dy, dstate, scale, need_g, need_state)
    return tuple(q.new_empty(0) if x is None else x for x in out)       # (an operator returns tensors)


_lib.impl('linear_attention', _forward, 'CUDA')
_lib.impl('linear_attention_backward', _backward_op, 'CUDA')
_lib.impl('linear_attention_step', _step, 'CUDA')


@th.library.register_fake('flex_rnn::linear_attention', lib=_lib)
def _(q, k, v, g, state, lengths, scale):
    B, T, H, M = v.shape
    return (v.new_empty((B, T, H, M)), v.new_empty((B, H, M, k.shape[3]), dtype=th.float32) if state is None else th.empty_like(state))


@th.library.register_fake('flex_rnn::linear_attention_backward', lib=_lib)
def _(q, k, v, g, state, lengths, dy, dstate, scale, need_g, need_state):
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), g.new_empty(g.shape) if need_g else q.new_empty(0),
            th.empty_like(state) if need_state else q.new_empty(0))


@th.library.register_fake('flex_rnn::linear_attention_step', lib=_lib)
def _(q, k, v, g, state, scale):
    return v.new_empty(v.shape)


_fw_op = th.ops.flex_rnn.linear_attention.default
_bw_op = th.ops.flex_rnn.linear_attention_backward.default
_step_op = th.ops.flex_rnn.linear_attention_step.default


class _LinearAttention(th.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, state, lengths, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, g, state, lengths)
        ctx.scale = scale
        return _fw_op(q, k, v, g, state, lengths, scale)

    @staticmethod
    def backward(ctx, dy, dstate):
        q, k, v, g, state, lengths = ctx.saved_tensors
        if dy is None and dstate is None:
            return (None,) * 7
        if dy is None:
            dy = th.zeros_like(v)
        need = ctx.needs_input_grad
        dq, dk, dv, dg, ds = hw.once(_bw_op, q, k, v, g, state, lengths, dy, dstate, ctx.scale, need[3], need[4])
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dg if need[3] else None, ds if need[4] else None, None, None


def _check(q, k, v, g, state, lead, what, types=True):
    """Argument checks shared by the prompt and the single-token form; `lead`: the dimensions in front of the heads."""
    n, sq, sv, dt = len(lead), q.shape, v.shape, q.dtype
    if len(sq) == len(sv) == n + 2 and sq == k.shape and sq[:n] == sv[:n] and sq[n] >= 1 and sv[n] >= 1 and sv[n] % sq[n] == 0 \
            and 1 <= sq[-1] <= MAX_HEAD and 1 <= sv[-1] <= MAX_HEAD and (n == 1 or sq[1] <= MAX_TOKENS) \
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
    state   [B,H,M,N], float32 or the type of q; None: zero, and the final state is float32
    lengths [B], int64 or int32: sequence b ends after `lengths[b]` tokens (clamped to 0..T); what is behind is not
            looked at, its `y` and gradients are zero, and the final state is the one after the last real token

    Any strides.  Sums and the state are fp32.  Differentiable once in q, k, v, g and state; gradients are deterministic.
    """
    _check(q, k, v, g, state, ('B', 'T'), 'linear_attention')
    _check_device('linear_attention', q, k, v, g, state, lengths)
    if lengths is not None:
        require(tuple(lengths.shape) == (q.shape[0],) and lengths.dtype in (th.int64, th.int32),
                f'linear_attention: lengths is int64 or int32 [B] = [{q.shape[0]}] (got {lengths.dtype} {list(lengths.shape)})')
        lengths = lengths.to(th.int64).contiguous()
    if th.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or (state is not None and state.requires_grad)):
        return _LinearAttention.apply(q, k, v, g, state, lengths, float(scale))
    return _fw_op(q, k, v, g, state, lengths, float(scale))


def linear_attention_step(q: th.Tensor, k: th.Tensor, v: th.Tensor, g: th.Tensor, state: th.Tensor, *, scale: float = 1.0) -> th.Tensor:
    """One token of `linear_attention` for decoding: `state` [B,H,M,N] is updated in place, y [B,H,M] is returned.

    q, k [B,Hk,N], v [B,H,M], g [B,H] or [H]; types as there.  Any strides, except that no two elements of the state may
    share memory.  Not differentiable: with T = 1, `linear_attention` is.
    """
    _check(q, k, v, g, state, ('B',), 'linear_attention_step')
    _check_device('linear_attention_step', q, k, v, g, state)
    if th.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or state.requires_grad):
        require(False, 'linear_attention_step updates the state in place and cannot be differentiated: use linear_attention, or th.no_grad()')
    if not state.is_contiguous():
        require(not _overlaps(state), 'linear_attention_step: elements of the state share memory')
    return _step_op(q, k, v, g, state, float(scale))


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
