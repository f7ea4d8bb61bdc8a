"""Cases and 64-bit references shared by the tests of linear attention and layer norm.

Bounds.  Let u be half a step of the inputs' type (bf16 2^-8, fp16 2^-11, fp32 2^-24) and |.|-run the same operator on
absolute values (with |dy|, |dstate| in gradients): the sum of the absolute values of everything that a result sums.
  - one rounding of the decayed products or of the state as a factor: u times the |.|-run (the two parts of a result, the
    block's own and the state's, are disjoint); fp16 and fp32 round these to 15 and 23 bits, which is less
  - the result's own rounding: u times the result, at most the |.|-run
  - sums in fp32, n terms: n 2^-24 times the |.|-run; n = M + N + tokens covers every chain of sums (products over M or N,
    blocks of tokens, the state over the sequence), as each addition rounds by at most 2^-24 of a partial sum
so 2u + (M + N + tokens) 2^-24 times the |.|-run bounds the error of an element of y, the states and dq, dk, dv.  States
and their gradients in fp32 keep three parts of 8 bits (2^-24) whatever the inputs' type: u = 2^-24 there.
"""
import math

import torch as th

import flex_rnn_amd as F

HALF_STEP = {dt: th.finfo(dt).eps / 2 for dt in (th.bfloat16, th.float16, th.float32)}


def make(dtype, B, T, H, Hk, M, N, g='token', g_dtype=th.float32, state=th.float32, lengths=None, resets=0.0, seed=0):
    """Inputs on the CPU: (q, k, v, g, state), lengths."""
    gen = th.Generator().manual_seed(seed)
    randn = lambda *s: th.randn(*s, generator=gen)  # noqa: E731
    q, k, v = randn(B, T, Hk, N), randn(B, T, Hk, N) / math.sqrt(N), randn(B, T, H, M)
    gate = -0.3 * th.rand(H, generator=gen) if g == 'head' else -th.nn.functional.softplus(randn(B, T, H) - 1)
    if resets:
        gate = th.where(th.rand(gate.shape, generator=gen) < resets, -math.inf, gate)
    s = None if state is None else randn(B, H, M, N).to(state)
    lens = None if lengths is None else th.tensor(lengths, dtype=th.int64)
    return [q.to(dtype), k.to(dtype), v.to(dtype), gate.to(g_dtype), s], lens


def cotangents(inputs, seed=1):
    q, k, v, g, s = inputs
    gen = th.Generator().manual_seed(seed)
    dy = th.randn(v.shape, generator=gen).to(v.dtype)
    ds = th.randn(v.shape[0], v.shape[2], v.shape[3], q.shape[3], generator=gen).to(th.float32 if s is None else s.dtype)
    return dy, ds


def run64(inputs, lengths, scale, dy=None, ds=None):
    """(y, state) and, with cotangents, the gradients of the inputs, from the per-token loop in 64 bits."""
    xs = [None if x is None else x.detach().double() for x in inputs]
    if dy is None:
        return F.linear_attention.naive_fp64(*xs, lengths=lengths, scale=scale)
    # (a step whose decay is zero passes no gradient to its logarithm: the loop's exp(-inf) * state says so by itself)
    xs = [None if x is None else x.requires_grad_() for x in xs]
    y, s = F.linear_attention.naive_fp64(*xs, lengths=lengths, scale=scale)
    leaves = [x for x in xs if x is not None]
    # (through linear functions of y and the state, so that an output without a graph, T = 0, needs no case of its own)
    loss = (y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()
    if not loss.requires_grad:
        return y.detach(), s.detach(), [th.zeros_like(x) for x in leaves]
    grads = th.autograd.grad(loss, leaves, allow_unused=True)
    return y.detach(), s.detach(), [th.zeros_like(x) if d is None else d for d, x in zip(grads, leaves)]


def absolute(inputs):
    q, k, v, g, s = inputs
    return [q.abs(), k.abs(), v.abs(), g, None if s is None else s.abs()]


def assert_within(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, f'{what}: shape {list(got.shape)}, expected {list(want.shape)}'
    assert bool(th.isfinite(got).all()), f'{what}: not finite'
    over = (got - want).abs() - bound
    if over.numel():
        worst = int(over.argmax())
        assert bool((over <= 0).all()), \
            f'{what}: element {worst} is {float(got.flatten()[worst])}, expected {float(want.flatten()[worst])} within {float(bound.flatten()[worst])}'


def bound_of_dg(inputs, lengths, absolute_grads, absolute_state, ds, size):
    """Bound of the gradient of g [B,T,H], `size` relative to what is summed for a token: q.dq and k.dk of the tokens from its block's
    start to the next border (blocks of 32; borders in front of every 8th, in front of the last and behind it), and the product of
    state and gradient there, all of absolute values - the products behind the border are no part of it.  In the |.|-run that
    product is the gradient of g at the border's own token; behind the last token it is the final state times its gradient."""
    q, k, v, g, s = inputs
    B, T, H = v.shape[:3]
    share = H // q.shape[2]
    dots = sum((x.double().abs() * absolute_grads[i]).sum(-1).repeat_interleave(share, 2) for i, x in ((0, q), (1, k)))       # [B,T,Hk]: over all its heads
    upto = th.cat([th.zeros(B, 1, H, dtype=th.float64), dots.cumsum(1)], 1)
    end = (absolute_state * ds.double().abs()).sum((-1, -2))
    out = th.zeros(B, T, H, dtype=th.float64)
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        blocks = (n + 31) // 32
        for c in range(blocks):
            at = next(x for x in range(c + 1, blocks + 1) if x % 8 == 0 or x + 1 >= blocks)
            stop = min(32 * at, n)
            border = end[b] if stop == n else absolute_grads[3][b, stop]
            out[b, 32 * c:min(32 * c + 32, n)] = upto[b, stop] - upto[b, 32 * c] + border
    return out * size
