"""Linear attention and layer norm on the GPU against the per-token loop (and plain norm) in 64 bits.  The bounds are
derived in `linear_cases.py` and beside the norm's tests; nothing is tuned to what the kernels give."""
import math

import pytest
import torch as th

import flex_rnn_amd as F
from flex_rnn_amd import examples

import linear_cases as lc
import warm

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = th.bfloat16, th.float16, th.float32


def _gpu(xs):
    return [None if x is None else x.cuda() for x in xs]


def _bounds(inputs, lens, scale, tokens, dy=None, ds=None):
    """Bounds of y, state and gradients (see linear_cases)."""
    q, k, v, g, s = inputs
    u = lc.HALF_STEP[q.dtype]
    sums = (q.shape[3] + v.shape[3] + tokens) * 2.0 ** -24
    s_dtype = FP32 if s is None else s.dtype
    a = lc.run64(lc.absolute(inputs), lens, abs(scale), None if dy is None else dy.abs(), None if ds is None else ds.abs())
    of_state = 2 * lc.HALF_STEP[s_dtype] + 2.0 ** -24 + sums
    out = [a[0] * (2 * u + sums), a[1] * of_state]
    if dy is None:
        return out
    names = ['q', 'k', 'v', 'g'] + (['state'] if s is not None else [])
    grads = dict(zip(names, a[2]))
    # shared heads: shares are summed in fp32 numbers, already rounded to u each
    for n in 'qkv':
        out.append(grads[n] * (2 * u + sums))
    # g: what is summed from token to token (q.dq and k.dk of every head, at most one span of blocks), and the marks
    B, T, H = v.shape[:3]
    share = H // q.shape[2]
    per_token = sum((x.double().abs() * grads[n]).sum(-1).repeat_interleave(share, 2) for n, x in (('q', q), ('k', k)))
    span = 32 * 8          # a block's tokens, the blocks between borders
    pad = -T % span
    folded = th.nn.functional.pad(per_token, (0, 0, 0, pad)).reshape(B, -1, span, H).sum(2, keepdim=True).expand(-1, -1, span, -1).reshape(B, -1, H)[:, :T]
    # (the product at a span's border: at most what follows sums to, plus the final state's with its gradient)
    end = (a[1].double() * ds.double().abs()).sum((-1, -2))[:, None]
    dg = (folded + per_token.flip(1).cumsum(1).flip(1) + end) * (sums + 2.0 ** -22)
    if g.ndim == 1:
        dg = dg.sum((0, 1))
        out.append(dg + grads['g'] * 2.0 ** -20)
    else:
        out.append(dg)
    out[-1] = out[-1] + grads['g'].abs() * lc.HALF_STEP[g.dtype]
    if s is not None:
        out.append(grads['state'] * of_state)
    return out


FORWARD = [
    # dtype, B, T, H, Hk, M, N, options
    (BF16, 2, 64, 2, 2, 64, 64, {}),
    (BF16, 1, 1, 3, 1, 128, 128, {}),
    (BF16, 1, 0, 2, 2, 16, 16, {}),
    (BF16, 0, 8, 2, 2, 16, 16, {}),
    (BF16, 2, 31, 2, 1, 17, 5, dict(g_dtype=BF16, state=BF16)),
    (BF16, 1, 33, 4, 2, 1, 1, dict(state=None)),
    (BF16, 2, 200, 2, 2, 256, 256, dict(g='head')),
    (BF16, 1, 130, 2, 2, 80, 103, dict(resets=0.1)),
    (BF16, 1, 1100, 1, 1, 128, 128, {}),
    (BF16, 3, 70, 6, 3, 72, 40, dict(lengths=(70, 0, 33))),
    (FP16, 2, 65, 4, 4, 64, 128, dict(g_dtype=FP16, state=FP16)),
    (FP16, 1, 100, 2, 1, 256, 56, dict(resets=0.05)),
    (FP16, 1, 600, 2, 2, 30, 64, {}),
    (FP32, 2, 64, 2, 2, 16, 16, {}),
    (FP32, 1, 97, 3, 1, 48, 200, dict(lengths=(1,))),
    (FP32, 1, 1030, 1, 1, 128, 64, dict(resets=0.02)),
    (FP32, 1, 40, 2, 2, 256, 256, {}),
    (FP16, 1, 8230, 1, 1, 16, 16, dict(resets=0.01)),          # as many segments as there are
]


@pytest.mark.parametrize('case', FORWARD, ids=str)
def test_forward(case):
    *shape, opts = case
    print(f'case linear attention {case}', flush=True)
    inputs, lens = lc.make(*shape, **opts)
    want = lc.run64(inputs, lens, 0.7)
    bounds = _bounds(inputs, lens, 0.7, shape[2])
    got = F.linear_attention(*_gpu(inputs), lengths=None if lens is None else lens.cuda(), scale=0.7)
    assert got[0].dtype == shape[0] and got[1].dtype == (FP32 if inputs[4] is None else inputs[4].dtype)
    for name, x, w, b in zip(('y', 'state'), got, want, bounds):
        lc.assert_within(x, w, b, name)


GRADIENT = [
    (BF16, 2, 64, 2, 2, 64, 64, {}),
    (BF16, 1, 1, 2, 2, 128, 128, {}),
    (BF16, 1, 0, 2, 2, 16, 16, {}),
    (BF16, 2, 31, 4, 1, 17, 5, dict(g_dtype=BF16, state=BF16)),
    (BF16, 1, 70, 2, 2, 256, 64, dict(g='head')),
    (BF16, 1, 90, 2, 1, 64, 256, dict(resets=0.1)),
    (BF16, 1, 1100, 1, 1, 64, 64, {}),
    (BF16, 3, 70, 6, 3, 72, 40, dict(lengths=(70, 0, 33), state=None)),
    (FP16, 2, 65, 4, 4, 64, 128, dict(g_dtype=FP16, state=FP16)),
    (FP16, 1, 300, 2, 1, 30, 56, dict(g='head', g_dtype=FP16)),
    (FP32, 2, 64, 2, 2, 16, 16, {}),
    (FP32, 1, 97, 3, 1, 48, 100, dict(lengths=(64,))),
    (FP32, 1, 1030, 2, 2, 16, 32, dict(resets=0.02)),
    (FP32, 1, 33, 1, 1, 256, 256, {}),
    (BF16, 2, 300, 4, 2, 16, 64, {}),                          # shares of many elements
]


def _gradients(inputs, lens, scale, dy, ds):
    leaves = [x.detach().requires_grad_() for x in inputs if x is not None]
    y, s = F.linear_attention(*leaves, lengths=lens, scale=scale)
    return [y, s, *th.autograd.grad((y, s), leaves, (dy, ds))]


@pytest.mark.parametrize('case', GRADIENT, ids=str)
def test_gradients(case):
    *shape, opts = case
    print(f'case linear attention gradients {case}', flush=True)
    inputs, lens = lc.make(*shape, **opts)
    dy, ds = lc.cotangents(inputs)
    y, s, grads = lc.run64(inputs, lens, 0.7, dy, ds)
    bounds = _bounds(inputs, lens, 0.7, shape[2], dy, ds)
    got = _gradients(_gpu(inputs), None if lens is None else lens.cuda(), 0.7, dy.cuda(), ds.cuda())
    names = ['y', 'state', 'dq', 'dk', 'dv', 'dg', 'dstate']
    for name, x, w, b in zip(names, got, [y, s, *grads], bounds):
        lc.assert_within(x, w, b, name)
    for x, leaf in zip(got[2:], [i for i in inputs if i is not None]):
        assert x.dtype == leaf.dtype


def test_gradient_against_differences():
    print('case linear attention differences', flush=True)
    inputs, _ = lc.make(FP32, 1, 50, 4, 2, 24, 16)
    dy, ds = lc.cotangents(inputs)
    xs = _gpu(inputs)
    grads = _gradients(xs, None, 1.0, dy.cuda(), ds.cuda())[2:]

    def loss(args):
        y, s = F.linear_attention(*args)
        return float((y.double() * dy.cuda().double()).sum() + (s.double() * ds.cuda().double()).sum())

    # the third-order term of a central difference with step h is below h^2 times the loss' size; its rounding is fp32's
    # 2^-22 of the loss' absolute sum over h: 1 % of the slope holds for both at h = 2^-6 with slopes of this size
    h = 2.0 ** -6
    for i, g in enumerate(grads):
        gen = th.Generator().manual_seed(i)
        d = th.randn(xs[i].shape, generator=gen).cuda()
        d = d / d.norm()
        up, down = [list(xs) for _ in range(2)]
        up[i], down[i] = xs[i] + h * d, xs[i] - h * d
        slope = (loss(up) - loss(down)) / (2 * h)
        assert abs(slope - float((g * d).sum())) < 1e-2 * max(1.0, float(g.norm())), i


def test_what_is_behind_the_last_token_is_not_looked_at():
    print('case padding', flush=True)
    B, T, H = 6, 70, 2
    lengths = (0, 1, 33, 64, 70, 500)
    inputs, lens = lc.make(BF16, B, T, H, H, 64, 64, lengths=lengths)
    dy, ds = lc.cotangents(inputs)
    clean = _gradients(_gpu(inputs), lens.cuda(), 1.0, dy.cuda(), ds.cuda())
    behind = th.arange(T)[None] >= lens[:, None]
    for bad in (math.nan, math.inf, -math.inf):
        spoiled = [x.clone() for x in inputs[:4]]
        for x in spoiled:
            x[behind] = bad
        d = dy.clone()
        d[behind] = bad
        got = _gradients(_gpu(spoiled) + [inputs[4].cuda()], lens.to(th.int32).cuda(), 1.0, d.cuda(), ds.cuda())
        for name, a, b in zip(('y', 'state', 'dq', 'dk', 'dv', 'dg', 'dstate'), got, clean):
            assert th.equal(a, b), (bad, name)
    for x in (clean[0], *clean[2:6]):
        assert bool((x.cpu()[behind] == 0).all())
    assert th.equal(clean[1][0].cpu(), inputs[4][0]) and th.equal(clean[6][0].cpu(), ds[0])
    # negative lengths are empty sequences
    y, s = F.linear_attention(*_gpu(inputs), lengths=th.full((B,), -3).cuda())
    assert bool((y == 0).all()) and th.equal(s.cpu(), inputs[4])


@pytest.mark.parametrize('value', [-math.inf, th.finfo(FP32).min, 0.0])
def test_decays_at_their_ends(value):
    """Every token forgets what came before (y_t = scale v_t k_t.q_t, no gradient for g), or nothing is forgotten."""
    print(f'case gates {value}', flush=True)
    inputs, _ = lc.make(FP32, 1, 70, 2, 2, 32, 16)
    inputs[3] = th.full_like(inputs[3], value)
    dy, ds = lc.cotangents(inputs)
    y, s, grads = lc.run64(inputs, None, 1.0, dy, ds)
    bounds = _bounds(inputs, None, 1.0, 70, dy, ds)
    got = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())
    if value != 0.0:
        grads[3] = th.zeros_like(grads[3])
    for x, w, b in zip(got, [y, s, *grads], bounds):
        lc.assert_within(x, w, b, f'gate {value}')


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize('T', [1, 33, 300])
def test_gradient_of_decays_that_leave_little(dtype, T):
    """With g near -20, g's gradient is e^-20 of the products that it is made of, and zero for the first token after an empty
    state.  Every term that is summed has that factor, so the result keeps fp32's precision relative to itself: 2^-24 for each
    of at most M + N + 64 terms in a chain of sums, M = N = 32, in the 2-norm (below 2e-5)."""
    print(f'case fast decays {dtype} {T}', flush=True)
    for state in (FP32, None):
        inputs, _ = lc.make(dtype, 2, T, 2, 1, 32, 32, state=state)
        inputs[3] = inputs[3] - 20
        dy, ds = lc.cotangents(inputs)
        want = lc.run64(inputs, None, 1.0, dy, ds)[2][3]
        got = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())[5].cpu().double()
        assert float((got - want).norm()) <= 128 * 2.0 ** -24 * 2 * float(want.norm()), state
        if state is None:
            assert bool((got[:, 0] == 0).all())


def test_strides_and_broadcast_inputs():
    print('case strides', flush=True)
    B, T, H, M, N = 2, 75, 2, 64, 64
    inputs, _ = lc.make(BF16, B, T, H, H, M, N)
    dy, ds = lc.cotangents(inputs)
    want = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())
    q, k, v, g, s = _gpu(inputs)
    time_inner = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)          # noqa: E731  [B,H,T,n] in memory
    columns_apart = lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)       # noqa: E731  columns H apart
    packed = th.cat([q, k, v], -1)                                                 # one projection's output, cut up
    odd = th.empty(B * T * H * N + 1, dtype=BF16, device='cuda')[1:].view(B, T, H, N).copy_(q)     # 2-byte aligned
    variants = {
        'time inner': [time_inner(q), time_inner(k), time_inner(v), g.transpose(1, 2).contiguous().transpose(1, 2), s],
        'columns apart': [columns_apart(q), columns_apart(k), columns_apart(v), g, s.mT.contiguous().mT],
        'packed': [packed[..., :N], packed[..., N:2 * N], packed[..., 2 * N:], g, s],
        'odd address': [odd, k, v, g, s],
        'time far apart': [x.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3) for x in (q, k, v)] + [g, s],
    }
    for name, xs in variants.items():
        got = _gradients(xs, None, 1.0, time_inner(dy.cuda()), ds.cuda().mT.contiguous().mT)
        for a, b in zip(got, want):
            assert th.equal(a, b), name
    # one query for all tokens and heads, one value for the batch, a scalar's gradient for every element of y
    y, s1 = F.linear_attention(q[:1, :1, :1].expand(B, T, H, N), k, v[:1].expand(B, T, H, M), g, s)
    y2, s2 = F.linear_attention(q[:1, :1, :1].expand(B, T, H, N).contiguous(), k, v[:1].expand(B, T, H, M).contiguous(), g, s)
    assert th.equal(y, y2) and th.equal(s1, s2)
    base = q[:1, :1, :1].clone().requires_grad_()
    y, _ = F.linear_attention(base.expand(B, T, H, N), k, v, g, s)
    grad, = th.autograd.grad(y.sum(), base)
    full = base.detach().expand(B, T, H, N).contiguous().requires_grad_()
    y, _ = F.linear_attention(full, k, v, g, s)
    whole, = th.autograd.grad(y, full, th.ones_like(y))
    # (torch sums bfloat16 in fp32 and rounds once: half a step of the sum and of each addend's share)
    assert bool(((grad.double() - whole.double().sum((0, 1, 2), keepdim=True)).abs() <= 2 ** -8 * whole.double().abs().sum((0, 1, 2), keepdim=True)).all())
    assert th.empty_like(s.mT).stride() == F.linear_attention(q, k, v, g, s.mT)[1].stride()


def test_offsets_beyond_32_bits():
    """Batches, tokens, rows and states that lie gigabytes apart, as in a pool, against the same numbers side by side."""
    print('case far apart', flush=True)
    B, T, H, M, N = 2, 33, 2, 64, 64
    inputs, _ = lc.make(BF16, B, T, H, H, M, N, state=BF16)
    dy, ds = [t.cuda() for t in lc.cotangents(inputs)]
    xs = _gpu(inputs)
    want = _gradients(xs, None, 1.0, dy, ds)
    pool = th.empty(2 ** 31 + 2 ** 27, dtype=BF16, device='cuda')
    far_batch = pool.as_strided((B, T, H, N), (2 ** 31, H * N, N, 1))
    far_token = pool.as_strided((B, T, H, N), (H * N, 2 ** 26, N, 1), 2 ** 20)
    far_state = pool.as_strided((B, H, M, N), (2 ** 31, M * N, N, 1), 2 ** 19)
    for at in (far_batch, far_token):
        at.copy_(xs[1])
        far_state.copy_(xs[4])
        got = _gradients([xs[0], at, xs[2], xs[3], far_state], None, 1.0, dy, ds)
        assert all(th.equal(a, b) for a, b in zip(got, want))
    state = xs[4].clone()
    y = F.linear_attention_step(xs[0][:, 0], xs[1][:, 0], xs[2][:, 0], xs[3][:, 0], state)
    assert th.equal(y, F.linear_attention_step(xs[0][:, 0], xs[1][:, 0], xs[2][:, 0], xs[3][:, 0], far_state)) and th.equal(state, far_state)
    rows = pool.as_strided((3, 100), (2 ** 30, 1), 2 ** 18)
    rows.copy_(th.randn(3, 100, device='cuda'))
    assert th.equal(F.layer_norm(rows), F.layer_norm(rows.contiguous()))


def test_threads_on_streams_of_their_own():
    print('case threads', flush=True)
    import threading
    inputs, _ = lc.make(FP16, 1, 450, 2, 1, 24, 40)
    dy, ds = [t.cuda() for t in lc.cotangents(inputs)]
    xs = _gpu(inputs)
    th.cuda.synchronize()
    results = [None] * 4

    def run(i):
        stream = th.cuda.Stream()
        with th.cuda.stream(stream):
            out = [_gradients(xs, None, 1.0, dy, ds) + [F.layer_norm(xs[2])] for _ in range(5)]
        stream.synchronize()
        results[i] = out

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    want = _gradients(xs, None, 1.0, dy, ds) + [F.layer_norm(xs[2])]
    for r in results:
        assert all(th.equal(a, b) for out in r for a, b in zip(out, want))


def test_partial_gradients():
    print('case partial gradients', flush=True)
    inputs, _ = lc.make(BF16, 1, 40, 2, 2, 64, 64)
    dy, ds = lc.cotangents(inputs)
    want = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())
    q, k, v, g, s = _gpu(inputs)
    v.requires_grad_()
    # (which gradients are asked for decides which walks share a launch, and so how many parts dv's state is rounded to: every
    # result is within 2u + sums of the |.|-run, so two of them are within twice that)
    exact = lc.run64(inputs, None, 1.0, dy, ds)[2][2]
    bound = _bounds(inputs, None, 1.0, 40, dy, ds)[4]
    y, sT = F.linear_attention(q, k, v, g, s)
    lc.assert_within(th.autograd.grad((y, sT), v, (dy.cuda(), ds.cuda()))[0], exact, bound, 'dv alone')
    lc.assert_within(want[4], exact, bound, 'dv')
    # only one of the results is used
    y, sT = F.linear_attention(q, k, v, g, s)
    only_y, = th.autograd.grad(y, v, dy.cuda())
    y, sT = F.linear_attention(q, k, v, g, s)
    only_s, = th.autograd.grad(sT, v, ds.cuda())
    for name, got, cot in (('y', only_y, (dy, 0 * ds)), ('state', only_s, (0 * dy, ds))):
        lc.assert_within(got, lc.run64(inputs, None, 1.0, *cot)[2][2], _bounds(inputs, None, 1.0, 40, *cot)[4], f'dv of the {name} alone')
    for f in (lambda: F.linear_attention(q, k, v, g, s)[0], lambda: F.layer_norm(v)):
        d, = th.autograd.grad(f(), v, dy.cuda(), create_graph=True)
        with pytest.raises(RuntimeError, match='differentiated once'):
            d.sum().backward()


def test_twice_gives_the_same_bits():
    print('case same bits', flush=True)
    for shape in ((BF16, 2, 300, 4, 2, 64, 128), (BF16, 1, 700, 2, 1, 128, 128)):
        inputs, _ = lc.make(*shape)
        dy, ds = lc.cotangents(inputs)
        a, b = (_gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda()) for _ in range(2))
        assert all(th.equal(x, y) for x, y in zip(a, b))


STEP = [
    (BF16, 2, 4, 2, 128, 128, {}),
    (BF16, 1, 2, 2, 64, 64, dict(state=BF16)),
    (BF16, 3, 3, 1, 17, 5, dict(state=BF16, g_dtype=BF16)),
    (BF16, 0, 2, 2, 16, 16, {}),
    (FP16, 2, 2, 2, 30, 256, dict(state=FP16)),
    (FP16, 1, 2, 1, 256, 72, dict(g='head')),
    (FP32, 2, 2, 2, 1, 1, {}),
    (FP32, 1, 5, 5, 200, 100, dict(resets=0.3)),
]


@pytest.mark.parametrize('case', STEP, ids=str)
def test_step(case):
    dtype, B, H, Hk, M, N, opts = case
    print(f'case step {case}', flush=True)
    inputs, _ = lc.make(dtype, B, 1, H, Hk, M, N, **opts)
    want = lc.run64(inputs, None, 0.7)
    a = lc.run64(lc.absolute(inputs), None, 0.7)
    sums = (N + 4) * 2.0 ** -24
    q, k, v, g, s = _gpu(inputs)
    token = [q[:, 0], k[:, 0], v[:, 0], g if g.ndim == 1 else g[:, 0]]
    # the state in several layouts: as it is, transposed in memory, a slice of a pool, with odd strides
    pool = th.full((B + 2, H, M, N), 7.0, dtype=s.dtype, device='cuda')
    wide = th.full((B, H, M, N + 3), 7.0, dtype=s.dtype, device='cuda')
    for name, state in (('plain', s.clone()), ('transposed', s.clone().mT.contiguous().mT), ('pool', pool[1:1 + B]), ('odd', wide[..., 1:1 + N])):
        state.copy_(s)
        y = F.linear_attention_step(*token, state, scale=0.7)
        lc.assert_within(y, want[0][:, 0], a[0][:, 0] * (lc.HALF_STEP[dtype] + sums), f'y {name}')
        lc.assert_within(state, want[1], a[1] * (lc.HALF_STEP[s.dtype] + sums), f'state {name}')
    assert bool((pool[0] == 7).all()) and bool((pool[1 + B:] == 7).all()) and bool((wide[..., 0] == 7).all()) and bool((wide[..., 1 + N:] == 7).all())


def _serve(q, k, v, g, state, lengths, weight, bias, prompt, attend, step, normed):
    """A padded batch's prompt, then a token at a time for all sequences, with the norm of each head."""
    y, state = attend(q[:, :prompt], k[:, :prompt], v[:, :prompt], g[:, :prompt], state, lengths=lengths, scale=0.5)
    outs = [normed(y, weight, bias)]
    for t in range(prompt, q.shape[1]):
        y, state = step(q[:, t], k[:, t], v[:, t], g[:, t], state)
        outs.append(normed(y, weight, bias)[:, None])
    return th.cat(outs, 1), state


def test_prompt_steps_and_norm_together():
    print('case serving', flush=True)
    B, P, T, H, M, N = 3, 50, 56, 2, 64, 64
    inputs, lens = lc.make(FP32, B, T, H, 1, M, N, lengths=(50, 7, 0))
    gen = th.Generator().manual_seed(3)
    weight, bias = th.randn(H, M, generator=gen), th.randn(H, M, generator=gen)

    def plain_step(q, k, v, g, s):
        y, s = F.linear_attention.naive_fp64(q[:, None], k[:, None], v[:, None], g[:, None], s, scale=0.5)
        return y[:, 0], s

    xs = [x.double() for x in inputs]
    want = _serve(*xs, lens, weight.double(), bias.double(), P, F.linear_attention.naive_fp64, plain_step, F.layer_norm.naive_fp64)

    def step(q, k, v, g, s):
        return F.linear_attention_step(q, k, v, g, s, scale=0.5), s

    with th.no_grad():
        got = _serve(*_gpu(inputs), lens.cuda(), weight.cuda(), bias.cuda(), P, F.linear_attention, step, F.layer_norm)
    a = lc.run64(lc.absolute(inputs), lens, 0.5)
    sums = (M + N + T) * 2.0 ** -24
    lc.assert_within(got[1], want[1], (a[1].max() + want[1].abs()) * 4 * sums, 'state')
    # A norm divides by a row's deviation: an error e of a row's elements is at most 2 e rstd |w| behind it, e below `sums`
    # times what the row sums (padding rows are zero: the norm gives the bias)
    raw, _ = _serve(*xs, lens, weight.double(), bias.double(), P, F.linear_attention.naive_fp64, plain_step, lambda y, w, b: y)
    rstd = 1 / (raw.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    size = F.linear_attention.naive_fp64(*lc.absolute(xs), scale=0.5)[0].amax(-1, keepdim=True)
    bound = (2 * size * rstd * weight.abs() * 4 + want[0].abs()) * sums * 2
    lc.assert_within(got[0], want[0], bound, 'y')


def test_training_through_both():
    """The gradient of norm(linear attention) against the 64-bit chain, in the 2-norm: each operator's result is within a few
    2^-24 times the length of its sums; 200 terms and a norm's division by deviations near 1 leave 1e-4 ample room."""
    print('case training chain', flush=True)
    inputs, _ = lc.make(FP32, 2, 60, 4, 2, 32, 32)
    gen = th.Generator().manual_seed(5)
    weight, bias, dy = (th.randn(*s, generator=gen) for s in ((4, 32), (4, 32), (2, 60, 4, 32)))

    def grads(xs, w, b, d, attend, norm):
        leaves = [x.detach().requires_grad_() for x in (*xs, w, b)]
        y, _ = attend(*leaves[:5])
        return th.autograd.grad((norm(y, leaves[5], leaves[6]) * d).sum(), leaves)

    want = grads([x.double() for x in inputs], weight.double(), bias.double(), dy.double(), F.linear_attention.naive_fp64, F.layer_norm.naive_fp64)
    got = grads(_gpu(inputs), weight.cuda(), bias.cuda(), dy.cuda(), F.linear_attention, F.layer_norm)
    for name, a, b in zip(('q', 'k', 'v', 'g', 'state', 'weight', 'bias'), got, want):
        assert float((a.cpu().double() - b).norm() / b.norm()) < 1e-4, name


def test_other_streams_and_graphs():
    print('case streams and graphs', flush=True)
    shape = (BF16, 2, 150, 4, 2, 64, 64)
    sets = [_gpu(lc.make(*shape, seed=i)[0]) for i in range(3)]
    dys = [[t.cuda() for t in lc.cotangents(lc.make(*shape, seed=i)[0], seed=10 + i)] for i in range(3)]
    weight, bias = th.randn(4, 64, device='cuda'), th.randn(4, 64, device='cuda')

    def work(xs, d):
        y, s = F.linear_attention(*xs)
        z = F.layer_norm(y, weight, bias)
        state = s.clone()
        token = F.linear_attention_step(xs[0][:, 0], xs[1][:, 0], xs[2][:, 0], xs[3][:, 0], state)
        grads = th.ops.flex_rnn.linear_attention_backward(*xs, None, d[0], d[1], 1.0, True, True)
        back = th.ops.flex_rnn.layer_norm_backward(y, weight, bias, d[0], 1e-5, True, True)
        return [y, s, z, state, token, *grads, *back]

    want = [work(xs, d) for xs, d in zip(sets, dys)]
    th.cuda.synchronize()
    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(side):
        got = work(sets[1], dys[1])
    th.cuda.current_stream().wait_stream(side)
    assert all(th.equal(a, b) for a, b in zip(got, want[1]))
    # one graph, replayed on other inputs, with eager work in between
    xs, d = [x.clone() for x in sets[0]], [t.clone() for t in dys[0]]
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        out = work(xs, d)
    for i in (1, 2, 0, 1):
        for a, b in zip(xs + d, sets[i] + dys[i]):
            a.copy_(b)
        graph.replay()
        eager = work(sets[(i + 1) % 3], dys[(i + 1) % 3])
        th.cuda.synchronize()
        assert all(th.equal(a, b) for a, b in zip(out, want[i])), i
        assert all(th.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3])), i
    # two graphs of one shape do not share their workspaces
    other, xs2 = th.cuda.CUDAGraph(), [x.clone() for x in sets[2]]
    with th.cuda.graph(other):
        out2 = work(xs2, [t.clone() for t in dys[2]])
    with th.cuda.stream(side):
        other.replay()
    graph.replay()
    th.cuda.synchronize()
    assert all(th.equal(a, b) for a, b in zip(out, want[1])) and all(th.equal(a, b) for a, b in zip(out2[:3], want[2][:3]))


def test_captured_training_step():
    print('case captured training', flush=True)
    inputs, _ = lc.make(BF16, 1, 100, 2, 2, 64, 64)
    dy, ds = [t.cuda() for t in lc.cotangents(inputs)]
    xs = _gpu(inputs)
    want = _gradients(xs, None, 1.0, dy, ds)
    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(side):
        leaves = [x.clone().requires_grad_() for x in xs]
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph, stream=side):
            y, s = F.linear_attention(*leaves)
            grads = th.autograd.grad((y, s), leaves, (dy, ds))
    for _ in range(3):
        for x in grads:
            x.zero_()
        graph.replay()
        th.cuda.synchronize()
        assert all(th.equal(a, b) for a, b in zip([y, s, *grads], want))


def test_captured_gradients_for_an_earlier_graph_are_refused():
    """A leaf whose eager graph is alive belongs to that graph's stream; a captured backward pass may not wait for it."""
    print('case capture beside an eager graph', flush=True)
    inputs, _ = lc.make(BF16, 1, 40, 2, 2, 64, 64)
    dy, ds = [t.cuda() for t in lc.cotangents(inputs)]
    leaves = [x.requires_grad_() for x in _gpu(inputs)]
    for f in (lambda: F.linear_attention(*leaves)[0], lambda: F.layer_norm(leaves[2])):
        want = th.autograd.grad(f(), leaves[2], dy)[0]
        alive = f()
        th.cuda.synchronize()
        with pytest.raises(RuntimeError, match='a stream outside the capture'):
            with th.cuda.graph(th.cuda.CUDAGraph()):
                th.autograd.grad(f(), leaves[2], dy)
        th.cuda.synchronize()
        del alive
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph):
            got = th.autograd.grad(f(), leaves[2], dy)[0]
        for _ in range(3):
            got.zero_()
            graph.replay()
            th.cuda.synchronize()
            assert th.equal(got, want)


def test_compiles_without_a_break():
    print('case torch.compile', flush=True)
    inputs, _ = lc.make(BF16, 1, 40, 2, 2, 64, 64)
    xs = _gpu(inputs)
    w = th.randn(2, 64, device='cuda')

    def f(q, k, v, g, s, w):
        y, s = F.linear_attention(q, k, v, g, s, scale=0.5)
        return F.layer_norm(y, w, w), s

    leaves = [x.detach().requires_grad_() for x in (*xs, w)]
    want = f(*leaves)
    dwant = th.autograd.grad(want, leaves, [th.ones_like(x) for x in want])
    got = th.compile(f, backend='aot_eager', fullgraph=True)(*leaves)
    dgot = th.autograd.grad(got, leaves, [th.ones_like(x) for x in got])
    assert all(th.equal(a, b) for a, b in zip((*got, *dgot), (*want, *dwant)))


# ------------------------------------------------------------------ layer norm
# Bounds: K = (C + 16) 2^-24 covers a chain of C fp32 additions and the few operations around it.  The mean is off by at most
# K mean|x|, so a normalised element by K (rstd (|x| + mean|x|) + |xhat|) =: K A; y = xhat w + b adds its own rounding u.
# dx = rstd (d - mean(d) - xhat mean(d xhat)) has three terms, with xhat's error twice in the last: 4 K rstd (|d| + mean|d| +
# A mean(|d| A)) covers them.  dw sums rows of dy xhat: (K + rows 2^-24) sum |dy| A.
NORM = [
    (BF16, (64, 32, 128), 'heads', FP32), (BF16, (5, 3, 17), 'heads', BF16), (BF16, (7, 1), 'columns', BF16), (BF16, (3, 5, 4096), 'columns', FP32),
    (BF16, (300, 600), 'columns', BF16), (BF16, (2, 16384), 'columns', FP32), (BF16, (1, 2, 1000), 'none', FP32), (BF16, (0, 4, 64), 'heads', FP32),
    (FP16, (33, 4, 64), 'heads', FP16), (FP16, (9, 1111), 'columns', FP32), (FP16, (40, 5000), 'bias', FP16),
    (FP32, (70, 2, 24), 'heads', FP32), (FP32, (5, 4095), 'columns', FP32), (FP32, (3, 9000), 'weight', FP32), (FP32, (64,), 'columns', FP32),
    (BF16, (700, 5), 'columns', FP32), (BF16, (20, 8), 'columns', BF16), (FP16, (6, 3, 9), 'heads', FP32), (FP16, (5, 8191), 'columns', FP16), (FP32, (9, 3), 'columns', FP32),
    (BF16, (40, 64, 1024), 'heads', FP32), (FP32, (700, 5), 'columns', FP32), (FP32, (3, 6001), 'columns', FP32), (FP32, (2, 16383), 'bias', FP32), (BF16, (300, 16381), 'columns', BF16),
]


@pytest.mark.parametrize('case', NORM, ids=str)
def test_layer_norm(case):
    dtype, shape, which, w_dtype = case
    print(f'case norm {case}', flush=True)
    gen = th.Generator().manual_seed(0)
    randn = lambda *s: th.randn(*s, generator=gen)  # noqa: E731
    x = (randn(*shape) * 2 + 3).to(dtype)
    p_shape = shape[-2:] if which == 'heads' else shape[-1:]
    w = None if which in ('none', 'bias') else (1 + randn(*p_shape)).to(w_dtype)
    b = None if which in ('none', 'weight') else randn(*p_shape).to(w_dtype)
    dy = randn(*shape).to(dtype)
    leaves = [t.double().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    y = F.layer_norm.naive_fp64(*args)
    grads = th.autograd.grad(y, leaves, dy.double())
    C = shape[-1]
    rows = max(1, x.numel() // C)
    K, u, uw = (C + 16) * 2.0 ** -24, lc.HALF_STEP[dtype], lc.HALF_STEP[w_dtype]
    xd = x.double()
    rstd = 1 / (xd.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    A = rstd * (xd.abs() + xd.abs().mean(-1, keepdim=True)) + ((xd - xd.mean(-1, keepdim=True)) * rstd).abs()
    wd = 1.0 if w is None else w.double().abs()
    d = dy.double().abs() * wd
    bounds = [4 * K * rstd * (d + d.mean(-1, keepdim=True) + A * (d * A).mean(-1, keepdim=True)) + u * grads[0].abs()]
    lead = tuple(range(x.ndim - len(p_shape)))
    over = (lambda t: t.sum(lead)) if lead else (lambda t: t)
    if w is not None:
        bounds.append((K + rows * 2.0 ** -24) * over(dy.double().abs() * A) + uw * grads[1].abs())
    if b is not None:
        bounds.append((rows + 16) * 2.0 ** -24 * over(dy.double().abs()) + uw * grads[-1].abs())
    leaves = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    got = F.layer_norm(*args)
    assert got.dtype == dtype
    lc.assert_within(got, y, 2 * K * (A * wd + (0.0 if b is None else b.double().abs())) + u * y.detach().abs(), 'y')
    for name, a, want, bound in zip(('dx', 'dw', 'db'), th.autograd.grad(got, leaves, dy.cuda()), grads, bounds):
        lc.assert_within(a, want, bound, name)
    with th.no_grad():
        assert th.equal(F.layer_norm(*args), got)


def test_layer_norm_strides():
    print('case norm strides', flush=True)
    x, w = th.randn(6, 5, 4, 64, device='cuda').bfloat16(), th.randn(4, 64, device='cuda')
    dy = th.randn_like(x)
    base = th.ops.flex_rnn.layer_norm_backward(x, w, w, dy, 1e-5, True, True)
    wide = th.zeros(6, 5, 4, 72, device='cuda').bfloat16()
    apart = [lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: t.mT.contiguous().mT, lambda t: wide.clone()[..., 1:65].copy_(t),
             lambda t: wide.clone()[..., :64].copy_(t), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)]
    for f in apart:
        assert th.equal(F.layer_norm(f(x), w, w), F.layer_norm(x, w, w))
        for a, b in zip(th.ops.flex_rnn.layer_norm_backward(f(x), w, w, f(dy), 1e-5, True, True), base):
            assert th.equal(a, b)
    assert th.equal(F.layer_norm(x, w.mT.contiguous().mT, w), F.layer_norm(x, w, w))
    y = F.layer_norm(x.requires_grad_(), w)
    a, = th.autograd.grad(y.sum(), x, retain_graph=True)          # (a gradient of y that is one number, expanded)
    b, = th.autograd.grad(y, x, th.ones_like(y))
    assert th.equal(a, b)


def test_layer_norm_rows_that_do_not_vary_or_are_not_finite():
    print('case norm rows', flush=True)
    x = th.randn(8, 64, device='cuda')
    x[1], x[2, 5], x[3, 7], x[4] = 3.0, math.nan, math.inf, 0.0
    y = F.layer_norm(x)
    assert bool((y[1] == 0).all()) and bool((y[4] == 0).all()) and bool(th.isnan(y[2]).all()) and bool(th.isnan(y[3]).all())
    for i in (0, 5, 6, 7):
        assert bool(th.isfinite(y[i]).all())
    # a large common offset: the mean goes first, so what is left keeps its bits (x has 24 bits: 4096 + z holds 11 fewer)
    z = th.randn(4, 256, device='cuda').double()
    off = (4096 + z).float()
    want = F.layer_norm.naive_fp64(off.double())
    assert float((F.layer_norm(off).double() - want).abs().max()) < 256 * 2 ** -24 * 4096 * 2


@pytest.mark.parametrize('op', examples.CHUNKED_OPS)
def test_examples_command(op):
    print(f'case example --chunked --head-norm {op}', flush=True)
    a = warm.EXAMPLE_ARGS
    examples.main(['--op', op, '--chunked', '--head-norm', '--check-flex', '--batchsz', str(a['B']), '--seqlen', str(a['T']),
                   '--modeldim', str(a['D']), '--headsz', str(a['C'])])


# ------------------------------------------------------------------ linear attention: precision and borders
# What a result's own rounding (u = half a step of its type) does not explain: the decayed products and the state as a factor
# keep 2^-15 of themselves (two bfloat16 parts: what truncation to 8 bits leaves is at most 2^-7, its rounding 2^-8 of that),
# and with float16 a product leaves out that of the two lower parts (at most 2^-7 each, 2^-14); the exponentials and the three
# parts of what enters the state 2^-20 in all; sums as in linear_cases.
REST = {BF16: 2.0 ** -15, FP16: 2.0 ** -13}


@pytest.mark.parametrize('case', [
    (BF16, 1, 300, 2, 2, 128, 128, dict(g='head')),
    (BF16, 1, 300, 2, 2, 128, 128, {}),
    (BF16, 2, 200, 4, 1, 64, 64, dict(g='head')),
    (BF16, 1, 130, 1, 1, 256, 256, dict(g='head')),
    (BF16, 1, 200, 2, 1, 33, 100, dict(g='head')),
    (FP16, 1, 300, 2, 2, 64, 128, dict(g='head')),
], ids=str)
def test_nothing_but_the_result_is_rounded_to_the_inputs_type(case):
    *shape, opts = case
    print(f'case rounding {case}', flush=True)
    dtype = shape[0]
    inputs, _ = lc.make(*shape, **opts)
    dy, ds = lc.cotangents(inputs)
    y, _, grads = lc.run64(inputs, None, 0.7, dy, ds)
    ay, _, agrads = lc.run64(lc.absolute(inputs), None, 0.7, dy.abs(), ds.abs())
    u, rest = lc.HALF_STEP[dtype], REST[dtype] + 2.0 ** -20 + (shape[2] + shape[5] + shape[6]) * 2.0 ** -24
    got = _gradients(_gpu(inputs), None, 0.7, dy.cuda(), ds.cuda())
    q, k, v, g, s = _gpu(inputs)
    v.requires_grad_()
    dv, = th.autograd.grad(F.linear_attention(q, k, v, g, s, scale=0.7), v, (dy.cuda(), ds.cuda()))
    for name, x, w, a in (('y', got[0], y, ay), ('dq', got[2], grads[0], agrads[0]), ('dk', got[3], grads[1], agrads[1]),
                          ('dv', got[4], grads[2], agrads[2]), ('dv alone', dv, grads[2], agrads[2])):
        lc.assert_within(x, w, u * w.abs() + (1 + u) * rest * a, name)


@pytest.mark.parametrize('shape', [(BF16, 2, 70, 4, 2, 64, 64), (BF16, 1, 100, 2, 2, 128, 128), (BF16, 1, 70, 2, 2, 256, 200), (FP16, 1, 70, 2, 1, 72, 33),
                                   (FP32, 1, 70, 2, 2, 40, 64), (FP32, 1, 40, 2, 2, 128, 128)], ids=str)
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
def test_a_number_that_is_not_finite_reaches_no_earlier_token(shape, bad):
    """One element of one token, in the middle of a block: where the definition does not read it, every bit is as without it, and
    where it does the result is not finite.  (g's gradient sums over tokens on both sides of it, and is left out.)"""
    print(f'case not finite {shape} {bad}', flush=True)
    T, H, Hk = shape[2], shape[3], shape[4]
    inputs, _ = lc.make(*shape)
    dy, ds = lc.cotangents(inputs)
    clean = [x.cpu() for x in _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())]
    names = ('y', 'state', 'dq', 'dk', 'dv')
    at, group = min(45, T - 2), H // Hk
    share = slice(0, group)                       # the heads of v that read the first head of q and k
    for which in ('q', 'k', 'v', 'dy'):
        xs, d = [x.clone() for x in inputs], dy.clone()
        (d if which == 'dy' else xs['qkv'.index(which)])[0, at, 0, 3] = bad
        got = dict(zip(names, [x.cpu() for x in _gradients(_gpu(xs), None, 1.0, d.cuda(), ds.cuda())]))
        # what reads the element (batch 0): all of these are sums with it as a factor of one term or more
        reach = {n: th.zeros_like(x, dtype=th.bool) for n, x in zip(names, clean)}
        after, before, heads = slice(at, T), slice(0, at + 1), share if which in 'qk' else slice(0, 1)
        if which == 'q':
            reach['y'][0, at, heads] = True
            reach['dk'][0, before, 0, 3] = True
            reach['dv'][0, before, heads] = True
        elif which == 'k':
            reach['y'][0, after, heads] = True
            reach['state'][0, heads, :, 3] = True
            reach['dq'][0, after, 0, 3] = True
            reach['dv'][0, at, heads] = True
        elif which == 'v':
            reach['y'][0, after, 0, 3] = True
            reach['state'][0, 0, 3] = True
            reach['dq'][0, after, 0] = True
            reach['dk'][0, at, 0] = True
        else:
            reach['dq'][0, at, 0] = True
            reach['dk'][0, before, 0] = True
            reach['dv'][0, before, 0, 3] = True
        for n, x in zip(names, clean):
            keep = ~reach[n]
            assert th.equal(got[n][keep], x[keep]), (which, n)
            assert not bool(th.isfinite(got[n][reach[n]]).any()), (which, n)


def test_how_far_a_number_that_is_not_finite_reaches_in_the_gradient_of_the_decays():
    """g's gradient is summed between borders, 256 tokens at most: in front of a spoiled v (or k) that far, behind a spoiled dy
    (or q) not at all; other heads not at all."""
    print('case not finite, gradient of g', flush=True)
    inputs, _ = lc.make(BF16, 1, 600, 2, 2, 64, 64)
    dy, ds = lc.cotangents(inputs)
    clean = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())[5]
    for which, keep in (('k', slice(0, 500 - 255)), ('v', slice(0, 500 - 255)), ('q', slice(501, 600)), ('dy', slice(501, 600))):
        xs, d = [x.clone() for x in inputs], dy.clone()
        (d if which == 'dy' else xs['qkv'.index(which)])[0, 500, 0, 3] = math.nan
        got = _gradients(_gpu(xs), None, 1.0, d.cuda(), ds.cuda())[5]
        assert th.equal(got[:, keep, 0], clean[:, keep, 0]) and th.equal(got[:, :, 1], clean[:, :, 1]), which


@pytest.mark.parametrize('dtype,T,g', [(BF16, 300, 'token'), (FP16, 70, 'token'), (FP32, 600, 'token'), (BF16, 90, 'head')], ids=str)
@pytest.mark.parametrize('value', [-math.inf, -3e38, -104.0])
def test_gradient_of_a_decay_that_is_zero_is_zero(dtype, T, g, value):
    """exp(-104) rounds to zero in 32 bits (its least number is exp(-103.3)): such a token carries nothing over, whatever the
    sums around it round to."""
    print(f'case zero decays {dtype} {T} {g} {value}', flush=True)
    inputs, _ = lc.make(dtype, 2, T, 2, 1, 64, 32, g=g)
    gen = th.Generator().manual_seed(2)
    hit = th.rand(inputs[3].shape, generator=gen) < 0.1 if g == 'token' else th.tensor([True, False])
    inputs[3] = th.where(hit, value, inputs[3])
    dy, ds = lc.cotangents(inputs)
    got = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())[5].cpu()
    assert bool((got[hit] == 0).all()) and bool((got[~hit] != 0).any())


# every build of the walk that serves g's gradient, over enough blocks for borders and segments
GRADIENT_BUILDS = [
    (BF16, 1, 450, 2, 2, 64, 64, {}),
    (BF16, 1, 450, 2, 1, 64, 64, {}),
    (BF16, 1, 450, 2, 1, 60, 64, {}),
    (BF16, 1, 610, 2, 2, 128, 128, {}),
    (BF16, 1, 450, 4, 2, 128, 96, dict(lengths=(413,))),
    (BF16, 2, 450, 2, 2, 100, 128, dict(lengths=(450, 390))),
    (BF16, 1, 400, 1, 1, 256, 256, {}),
    (BF16, 1, 400, 2, 1, 192, 64, {}),
    (BF16, 1, 400, 1, 1, 203, 130, {}),
    (FP16, 1, 450, 2, 2, 64, 64, {}),
    (FP16, 1, 450, 2, 1, 64, 128, {}),
    (FP16, 1, 450, 2, 1, 61, 64, {}),
    (FP16, 1, 610, 2, 2, 128, 128, {}),
    (FP16, 1, 450, 4, 2, 96, 64, {}),
    (FP16, 1, 450, 2, 1, 100, 70, dict(resets=0.02)),
    (FP16, 1, 400, 1, 1, 256, 64, {}),
    (FP16, 1, 400, 2, 1, 192, 192, {}),
    (FP16, 1, 400, 1, 1, 201, 64, {}),
    (FP32, 1, 450, 2, 1, 64, 64, {}),
    (FP32, 1, 450, 2, 1, 63, 64, {}),
    (FP32, 1, 450, 2, 2, 128, 128, {}),
    (FP32, 1, 450, 2, 1, 128, 96, dict(resets=0.02)),
    (FP32, 1, 450, 2, 2, 101, 100, {}),
    (FP32, 1, 400, 1, 1, 256, 256, {}),
    (FP32, 1, 400, 1, 1, 131, 256, {}),
]


def _assert_gradients_within(inputs, lens, scale, dy, ds, got):
    """Every result of a training step against the 64-bit loop, as close as what stands at `REST` and in `bound_of_dg` says."""
    q, k, v, g, s = inputs
    u = lc.HALF_STEP[q.dtype]
    exact = 2.0 ** -20 + (v.shape[1] + v.shape[3] + q.shape[3]) * 2.0 ** -24
    rest = exact + REST.get(q.dtype, 0.0)
    y, sT, grads = lc.run64(inputs, lens, scale, dy, ds)
    ay, aT, agrads = lc.run64(lc.absolute(inputs), lens, abs(scale), dy.abs(), ds.abs())
    of_state = lc.HALF_STEP[s.dtype]
    for name, x, w, a in (('y', got[0], y, ay), ('dq', got[2], grads[0], agrads[0]), ('dk', got[3], grads[1], agrads[1]), ('dv', got[4], grads[2], agrads[2])):
        lc.assert_within(x, w, u * w.abs() + (1 + u) * rest * a, name)
    for name, x, w, a in (('state', got[1], sT, aT), ('dstate', got[6], grads[4], agrads[4])):
        lc.assert_within(x, w, of_state * w.abs() + (1 + of_state) * exact * a, name)
    lc.assert_within(got[5], grads[3], lc.HALF_STEP[g.dtype] * grads[3].abs() + lc.bound_of_dg(inputs, lens, agrads, aT, ds, exact), 'dg')


@pytest.mark.parametrize('case', GRADIENT_BUILDS, ids=str)
def test_gradients_of_every_build(case):
    *shape, opts = case
    print(f'case gradient build {case}', flush=True)
    inputs, lens = lc.make(*shape, **opts)
    dy, ds = lc.cotangents(inputs)
    got = _gradients(_gpu(inputs), None if lens is None else lens.cuda(), 0.7, dy.cuda(), ds.cuda())
    _assert_gradients_within(inputs, lens, 0.7, dy, ds, got)


@pytest.mark.parametrize('dtype', [BF16, FP32], ids=str)
def test_gradient_of_fast_decays_in_front_of_slow_ones(dtype):
    from test_linear import fast_then_slow
    print(f'case fast then slow {dtype}', flush=True)
    inputs, dy, ds = fast_then_slow(dtype)
    got = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())
    _assert_gradients_within(inputs, None, 1.0, dy, ds, got)
    # early tokens relative to themselves: a token's products are O(1) numbers of which e^-9 is left, so fp32's 2^-24 of each
    # of up to 256 + 64 terms is at most 320 2^-24 e^9 of the result
    want = lc.run64(inputs, None, 1.0, dy, ds)[2][3][:, :256]
    assert float((got[5].cpu().double()[:, :256] - want).norm()) <= 320 * 2.0 ** -24 * math.exp(9) * float(want.norm())


@pytest.mark.parametrize('dtype,M,N', [(BF16, 128, 128), (BF16, 256, 64), (FP16, 128, 256), (FP32, 256, 128)], ids=str)
def test_layouts_of_wide_heads(dtype, M, N):
    """Columns far apart, rows at odd addresses and cut out of wider ones give the bits of the plain layout, at every width."""
    print(f'case layouts {dtype} {M} {N}', flush=True)
    B, T, H = 1, 400, 2
    inputs, _ = lc.make(dtype, B, T, H, H, M, N)
    dy, ds = [t.cuda() for t in lc.cotangents(inputs)]
    xs = _gpu(inputs)
    want = _gradients(xs, None, 1.0, dy, ds)
    columns_apart = lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)       # noqa: E731
    cut = lambda x: th.cat([x[..., :1], x, x[..., :2]], -1)[..., 1:-2]             # noqa: E731
    for name, f in (('apart', columns_apart), ('cut', cut)):
        got = _gradients([f(x) for x in xs[:3]] + xs[3:], None, 1.0, f(dy), ds)
        for what, a, b in zip(('y', 'state', 'dq', 'dk', 'dv', 'dg', 'dstate'), got, want):
            assert th.equal(a, b), (name, what)


def test_transforms_of_torch_func():
    """vmap runs the operators once per element; a step under vmap and func.grad are errors, nothing comes out wrong."""
    print('case torch.func', flush=True)
    made = [_gpu(lc.make(FP32, 2, 40, 2, 1, 16, 24, seed=i)[0]) for i in range(3)]
    q, k, v, g, s = (th.stack(x) for x in zip(*made))
    y, state = th.func.vmap(F.linear_attention)(q, k, v, g, s)
    norm = th.func.vmap(F.layer_norm)(v)
    for i, xs in enumerate(made):
        want = F.linear_attention(*xs)
        assert th.equal(y[i], want[0]) and th.equal(state[i], want[1]) and th.equal(norm[i], F.layer_norm(xs[2]))
    for dims, at in ((0, s), (None, s[0])):
        with pytest.raises(RuntimeError, match='(?i)batching rule'):
            th.func.vmap(F.linear_attention_step, in_dims=(0, 0, 0, 0, dims))(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], at)
    for f in (lambda x: F.layer_norm(x).sum(), lambda x: F.linear_attention(*made[0][:2], x, *made[0][3:])[0].sum()):
        with pytest.raises(RuntimeError, match='functorch'):
            th.func.grad(f)(v[0])


def test_a_step_compiles_without_a_break():
    print('case torch.compile of a step', flush=True)
    inputs, _ = lc.make(BF16, 2, 1, 4, 2, 64, 64)
    q, k, v, g = (x[:, 0] for x in _gpu(inputs[:4]))
    s1 = inputs[4].cuda()
    s2 = s1.clone()

    def f(q, k, v, g, s):
        return F.layer_norm(F.linear_attention_step(q, k, v, g, s, scale=0.5))

    compiled = th.compile(f, backend='aot_eager', fullgraph=True)
    with th.no_grad():
        for _ in range(3):
            assert th.equal(compiled(q, k, v, g, s2), f(q, k, v, g, s1)) and th.equal(s1, s2)


def test_products_of_float32_have_no_bias():
    """y = q k v and the final state v k of single numbers, 65536 of them: each is off by a few 2^-24 of itself, to either side.  What
    two products drop and their sums round has an rms below 2^-23 (65536 independent ones average to 2^-31), so a mean of 2^-27
    is one that no luck explains; with the middle parts of factors cut off instead of rounded it is 2^-24.5 a product."""
    print('case bias', flush=True)
    inputs, _ = lc.make(FP32, 256, 1, 256, 256, 1, 1, state=None)
    q, k, v, g, _ = inputs
    y, s = F.linear_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda())
    want = v.double() * k.double()
    for name, got, w in (('state', s.cpu()[:, :, 0, 0], want[:, 0, :, 0]), ('y', y.cpu()[:, 0, :, 0], (want * q.double())[:, 0, :, 0])):
        off = (got.double() - w) / w
        assert float(off.abs().max()) < 2.0 ** -20 and abs(float(off.mean())) < 2.0 ** -27, (name, float(off.abs().max()), float(off.mean()))


def test_gradient_of_a_decay_that_all_tokens_share():
    """One number per head, the sum over all tokens of terms of either sign.  It is no further off (in the mean square over seeds)
    than if every token's q.dq and k.dk were exact and rounded to 32 bits once (0.41 2^-24 of them in the mean square), and each
    counted for the tokens in front of it in a span of 64, from 0 to 64 times (37 in the mean square): 16 2^-24 times the root of
    the number of tokens times the products."""
    print('case shared decay', flush=True)
    off = []
    for seed in range(6):
        inputs, _ = lc.make(FP32, 3, 1200, 1, 1, 32, 32, g='head', seed=seed)
        dy, ds = lc.cotangents(inputs, seed=10 + seed)
        q, k = inputs[:2]
        _, _, grads = lc.run64(inputs, None, 1.0, dy, ds)
        n = 3 * 1200
        each = ((q.double() * grads[0]).sum(-1) ** 2 + (k.double() * grads[1]).sum(-1) ** 2).mean().sqrt()
        got = _gradients(_gpu(inputs), None, 1.0, dy.cuda(), ds.cuda())[5]
        off.append(float((got.cpu().double() - grads[3]).abs() / (math.sqrt(256 * n) * 2.0 ** -24 * each)))
    assert sum(x * x for x in off) / len(off) < 1.0, off


@pytest.mark.parametrize('H,blocks', [(5, 2), (9, 4)])
def test_borders_further_apart_for_shared_decays_of_long_sequences(H, blocks):
    """Where states at every block would not fit: a shared decay's gradient against the sum of the gradients of the same decays per
    token.  Each q.dq and k.dk, rounded to 32 bits (0.41 2^-24 in the mean square), counts up to 256 times there (148 in the
    mean square) and 128 times here (74): 91 2^-24 times the root of the number of tokens times the products; four times that."""
    from flex_rnn_amd import handwritten
    print(f'case borders apart {H}', flush=True)
    T, M, N = 2 ** 18, 256, 256
    assert handwritten.blocks_between_borders(1, T, H, M, N, True) == blocks
    gen = th.Generator(device='cuda').manual_seed(0)
    randn = lambda *s: th.randn(*s, generator=gen, device='cuda')  # noqa: E731
    q, k, v, dy = randn(1, T, H, N).to(BF16), (randn(1, T, H, N) / 16).to(BF16), randn(1, T, H, M).to(BF16), randn(1, T, H, M).to(BF16)
    g = -0.02 - 0.3 * th.rand(H, generator=gen, device='cuda')
    back = th.ops.flex_rnn.linear_attention_backward
    dq, dk, _, shared, _ = back(q, k, v, g, None, None, dy, None, 1.0, True, False)
    each = ((q.float() * dq.float()).sum(-1).square() + (k.float() * dk.float()).sum(-1).square()).mean(1).sqrt()[0]
    apart = back(q, k, v, g.expand(1, T, H).contiguous(), None, None, dy, None, 1.0, True, False)[3].double().sum((0, 1))
    assert bool(((shared.double() - apart).abs() <= 4 * 91 * 2.0 ** -24 * math.sqrt(T) * each.double()).all())
