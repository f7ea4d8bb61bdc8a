"""Linear attention and layer norm without a GPU: refusals, the plain loop that the GPU tests compare with (against
`jit.naive` of the recurrences that it covers, and against differences), metadata, host-side planning."""
import os

import pytest
import torch as th

import flex_rnn_amd as F
from flex_rnn_amd import examples, handwritten, linear, ops, runtime

import linear_cases as lc


@pytest.fixture(scope='module', autouse=True)
def operators(runtime_lib):
    """The operators' library; built once if a run finds it missing."""
    if not os.path.isfile(handwritten.OPS_PATH):
        handwritten.build_library()
    return handwritten.load()


def _meta(*shape, dtype=th.bfloat16):
    return th.empty(shape, dtype=dtype, device='meta')


def test_public_names():
    import flex_rnn
    for name in ('linear_attention', 'linear_attention_step', 'layer_norm'):
        assert getattr(flex_rnn, name) is getattr(F, name)


BAD = [
    (dict(q=(2, 8, 4)), r'q and k are \[B, T, Hk, N\]'),
    (dict(k=(2, 8, 2, 16)), 'q .* and k .* differ'),
    (dict(v=(2, 9, 4, 16)), r'q .* and v .* differ in B, T'),
    (dict(v=(2, 8, 6, 16)), '6 heads of v do not divide into 4 heads'),
    (dict(v=(2, 8, 4, 257)), 'head sizes from 1 to 256'),
    (dict(q=(2, 8, 4, 0), k=(2, 8, 4, 0)), 'head sizes from 1 to 256'),
    (dict(v_dtype=th.float32), 'q, k and v are of one type'),
    (dict(dtype=th.float64, v_dtype=th.float64), 'q, k and v are of one type'),
    (dict(g=(2, 8, 3)), r'g is \[H\] or \[B, T, H\] with H = 4'),
    (dict(g=(2,)), r'g is \[H\]'),
    (dict(g_dtype=th.float16), 'g is float32 or of the type of q'),
    (dict(state=(2, 4, 16, 17)), r'the state is \[B, H, M, N\]'),
    (dict(state_dtype=th.float16), 'the state is float32 or of the type of q'),
    (dict(lengths=(3,)), r'lengths is int64 or int32 \[B\] = \[2\]'),
    (dict(lengths_dtype=th.float32), 'lengths is int64 or int32'),
    (dict(v=(2, 8, 2 ** 20, 16), g=(2 ** 20,), state=(2, 2 ** 20, 16, 16)), 'a token has up to 16777215 elements over all heads'),
]


@pytest.mark.parametrize('change,message', BAD)
def test_linear_attention_refuses(change, message):
    c = dict(q=(2, 8, 4, 16), k=(2, 8, 4, 16), v=(2, 8, 4, 16), g=(2, 8, 4), state=(2, 4, 16, 16), lengths=(2,), dtype=th.bfloat16,
             g_dtype=th.float32, state_dtype=th.float32, lengths_dtype=th.int64)
    c.update(change)
    c.setdefault('v_dtype', c['dtype'])
    args = [_meta(*c['q'], dtype=c['dtype']), _meta(*c['k'], dtype=c['dtype']), _meta(*c['v'], dtype=c['v_dtype']), _meta(*c['g'], dtype=c['g_dtype']),
            _meta(*c['state'], dtype=c['state_dtype'])]
    with pytest.raises(AssertionError, match=message):
        F.linear_attention(*args, lengths=_meta(*c['lengths'], dtype=c['lengths_dtype']))


def test_gpu_only_and_one_device():
    q = th.zeros(1, 4, 2, 8)
    with pytest.raises(AssertionError, match='runs on the GPU only'):
        F.linear_attention(q, q, q, th.zeros(2))
    with pytest.raises(AssertionError, match='runs on the GPU only'):
        F.layer_norm(q)
    with pytest.raises(AssertionError, match='runs on the GPU only'):
        F.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], th.zeros(2), th.zeros(1, 2, 8, 8))
    m = _meta(1, 4, 2, 8, dtype=th.float32)
    with pytest.raises(AssertionError, match='the same device'):
        F.linear_attention(m, m, m, th.zeros(2))
    with pytest.raises(AssertionError, match='the same device'):
        F.layer_norm(m, th.zeros(8))


def test_step_refuses():
    m, s = _meta(2, 4, 16), _meta(2, 4, 16, 16, dtype=th.float32)
    g = _meta(2, 4, dtype=th.float32)
    assert F.linear_attention_step(m, m, m, g, s).shape == (2, 4, 16)
    with pytest.raises(AssertionError, match='elements of the state share memory'):
        F.linear_attention_step(m, m, m, g, s[:1].expand(2, 4, 16, 16))
    with pytest.raises(AssertionError, match='cannot be differentiated'):
        F.linear_attention_step(m, m, m, g, s.clone().requires_grad_())
    with th.no_grad():
        F.linear_attention_step(m, m, m, g, s.clone().requires_grad_())
    with pytest.raises(AssertionError, match=r'g is \[H\] or \[B, H\]'):
        F.linear_attention_step(m, m, m, _meta(2, 3, dtype=th.float32), s)


def test_step_counts_as_a_change_of_its_state():
    """A state that autograd keeps for a backward pass and a step then overwrites is found out."""
    q, s = _meta(1, 4, 2, 16).requires_grad_(), _meta(1, 2, 16, 16, dtype=th.float32)
    g = _meta(2, dtype=th.float32)
    y, _ = F.linear_attention(q, q, q, g, s)
    with th.no_grad():
        F.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g, s)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward(th.empty_like(y))
    with th.inference_mode():
        m = _meta(1, 2, 16)
        F.linear_attention_step(m, m, m, g, _meta(1, 2, 16, 16, dtype=th.float32))


def test_overlap_rule():
    x = th.zeros(4, 6, 8, 10)
    assert not linear._overlaps(x) and not linear._overlaps(x.mT) and not linear._overlaps(x[:, ::2, 1:5]) and not linear._overlaps(x.permute(2, 0, 3, 1))
    assert linear._overlaps(x[:1].expand(4, 6, 8, 10)) and linear._overlaps(th.zeros(64).as_strided((1, 1, 8, 8), (64, 64, 4, 1)))


@pytest.mark.parametrize('kwargs,message', [
    (dict(x=(3, 16), weight=(15,)), r'weight is \[C\] = \[16\]'),
    (dict(x=(3, 16), weight=(2, 16)), r'weight is \[C\]'),
    (dict(x=(3, 2, 16), weight=(2, 16), bias=(16,)), 'the same shape'),
    (dict(x=(3, 16), weight=(16,), weight_dtype=th.float16), 'float32 or of the type of x'),
    (dict(x=(3, 16385)), 'rows of 1 to 16384 columns'),
    (dict(x=(3, 0)), 'rows of 1 to 16384 columns'),
    (dict(x=()), 'at least one dimension'),
    (dict(x=(3, 16), x_dtype=th.float64), 'x is bfloat16, float16 or float32'),
])
def test_layer_norm_refuses(kwargs, message):
    make = lambda n, dt: None if n not in kwargs else _meta(*kwargs[n], dtype=dt)  # noqa: E731
    with pytest.raises(AssertionError, match=message):
        F.layer_norm(make('x', kwargs.get('x_dtype', th.bfloat16)), make('weight', kwargs.get('weight_dtype', th.bfloat16)), make('bias', th.bfloat16))


def test_metadata_and_autograd_on_meta():
    q, v = _meta(2, 8, 2, 16).requires_grad_(), _meta(2, 8, 4, 32).requires_grad_()
    g, s = _meta(4, dtype=th.float32).requires_grad_(), _meta(2, 4, 32, 16).requires_grad_()
    y, sT = F.linear_attention(q, q, v, g, s)
    assert y.shape == v.shape and y.dtype == v.dtype and sT.shape == s.shape and sT.dtype == s.dtype
    grads = th.autograd.grad((y, sT), (q, v, g, s), (y, sT))
    assert [x.shape for x in grads] == [x.shape for x in (q, v, g, s)] and [x.dtype for x in grads] == [x.dtype for x in (q, v, g, s)]
    assert F.linear_attention(q, q, v, g)[1].dtype == th.float32
    w = _meta(4, 32, dtype=th.float32).requires_grad_()
    z = F.layer_norm(v, w, w)
    dv, dw = th.autograd.grad(z, (v, w), z)
    assert z.shape == v.shape and dv.shape == v.shape and dw.shape == w.shape and dw.dtype == th.float32


def test_plain_loop_is_the_recurrence_of_retention_and_mamba2():
    B, T, H, C = 2, 5, 3, 4
    gen = th.Generator().manual_seed(0)
    randn = lambda *s: th.randn(*s, generator=gen, dtype=th.float64)  # noqa: E731
    inputs, layer, steps = examples.build('mamba2', B, T, H * C, C, 'cpu')
    steps['step'].apply = steps['step'].naive_fp64
    want = layer(*inputs)
    x, dt, A, b, c, s = inputs
    got = F.linear_attention.naive_fp64(c, b, dt.unsqueeze(-1) * x, dt * A, s)
    for u, v in zip(got, want):
        assert th.allclose(u.double(), v.double(), rtol=1e-5, atol=1e-5)        # (both are rounded to float32 once)
    q, k, v, w = randn(B, T, H, C), randn(B, T, H, C), randn(B, T, H, C), th.rand(B, T, H, generator=gen, dtype=th.float64)
    s = randn(B, H, C, C)
    ret = F.jit(ops.retention)
    want = ret.naive_fp64(w[..., None, None], q.unsqueeze(-2), k.unsqueeze(-2), v.unsqueeze(-1), s)
    got = F.linear_attention.naive_fp64(q, k, v, w.log(), s)
    for u, x in zip(got, want):
        assert th.allclose(u, x, rtol=1e-12, atol=1e-12)


def test_plain_loop_lengths_and_gradients():
    inputs, lens = lc.make(th.float32, 3, 6, 4, 2, 5, 3, lengths=(0, 4, 9), resets=0.2)
    xs = [x.double() for x in inputs]
    y, s = F.linear_attention.naive(*xs, lengths=lens, scale=0.5, dtype=th.float64)
    assert bool((y[0] == 0).all()) and th.equal(s[0], xs[4][0]) and bool((y[1, 4:] == 0).all())
    cut = [xs[0][1:2, :4], xs[1][1:2, :4], xs[2][1:2, :4], xs[3][1:2, :4], xs[4][1:2]]
    y1, s1 = F.linear_attention.naive(*cut, scale=0.5, dtype=th.float64)
    assert th.equal(y[1, :4], y1[0]) and th.equal(s[1], s1[0])
    # gradients of the loop against differences
    xs[3] = xs[3].clamp(min=-3)
    f = lambda *a: F.linear_attention.naive(*a, lengths=lens, scale=0.5, dtype=th.float64)  # noqa: E731
    assert th.autograd.gradcheck(f, [x.requires_grad_() for x in xs], eps=1e-6, atol=1e-6)
    x, w, b = th.randn(3, 2, 5, dtype=th.float64), th.randn(2, 5, dtype=th.float64), th.randn(2, 5, dtype=th.float64)
    assert th.autograd.gradcheck(lambda *a: F.layer_norm.naive(*a, dtype=th.float64), [t.requires_grad_() for t in (x, w, b)], eps=1e-6, atol=1e-6)


def test_segments_cover_the_blocks():
    for groups in (1, 2, 7, 64, 511, 512, 5000):
        for blocks in (0, 1, 15, 16, 17, 35, 1024, 4097):
            nseg, per = handwritten.segments(groups, blocks)
            assert nseg >= 1 and nseg * per >= blocks and nseg <= 64
            assert nseg == 1 or (nseg - 1) * per < blocks          # no segment without a block
            assert groups < 512 or nseg == 1


def test_teams_keep_their_head_and_hold_a_row():
    for rows, heads, C in ((8192 * 32, 32, 128), (5, 5, 64), (37, 1, 1000), (192, 64, 4096), (70000, 1, 8), (600, 300, 512), (3, 1, 16384), (1, 1, 1)):
        for size in (2, 4):
            s = handwritten.norm_shape(rows, heads, C, size)
            assert s['teams'] % heads == 0 and heads <= s['teams'] <= rows
            assert s['lanes'] * s['pieces'] * 16 >= C * size and (s['wide'] or s['lanes'] <= 64) and s['lanes'] <= s['threads']


def test_every_kernel_that_an_operator_asks_for_is_prebuilt(monkeypatch):
    built = handwritten.builds()
    assert len(set(built)) == len(built)
    for dt in range(3):
        for C in (1, 5, 64, 100, 513, 600, 1000, 2047, 2049, 4096, 5000, 8192, 9000, 16384):
            s = handwritten.norm_shape(7, 1, C, 4 if dt == 2 else 2)
            for kind in (5, 6):
                fields = (dt, s['pieces'], s['lanes'].bit_length() - 1, s['wide'])
                key = kind
                for f in fields:
                    key = key << 6 | f
                assert handwritten.decode(key) in built and dict(handwritten.decode(key)[2])['GL'] == s['lanes']
    assert handwritten.decode(2)[1] == 'la_gate' and handwritten.decode(4)[1] == 'slice_sum' and handwritten.decode(3 << 6 | 1)[1] == 'la_step'
    key = 1
    for f in (0, 1, 1, 1, 1, 0):
        key = key << 6 | f
    assert handwritten.decode(key) in built and dict(handwritten.decode(key)[2]) == dict(KERNEL_BLOCK=1, IN=0, W=128, OUT=1, DOTS=1, FAST=1, WIDE=0, NBUF=2, OCC=2)
    with pytest.raises(KeyError):
        handwritten.decode(9)
    seen = []
    monkeypatch.setattr(handwritten, 'build', lambda *c, force=False: seen.append(c))
    assert handwritten.build_all() == len(seen) == len(built)


def test_a_kernel_that_cannot_be_loaded_is_an_error_not_a_crash():
    """The loader runs on a C++ frame: whatever goes wrong comes back as a message."""
    import ctypes
    text = ctypes.create_string_buffer(256)
    assert handwritten._load(0, 9, ctypes.addressof(text), 256) == 0 and b'KeyError' in text.value
    assert handwritten._load(0, 4, ctypes.addressof(text), 16) == 0 and len(text.value) == 15          # (no GPU here: cut to the room there is)


def test_missing_library_says_how_to_build_it(monkeypatch):
    monkeypatch.setattr(handwritten, '_lib', None)
    monkeypatch.setattr(handwritten, 'OPS_PATH', '/nowhere/libfrnn_ops.so')
    with pytest.raises(runtime.RuntimeError_, match='have not been built'):
        handwritten.op('layer_norm')


def _tangent_calls():
    m, s, g, c = _meta(1, 4, 2, 8, dtype=th.float32), _meta(1, 2, 8, 8, dtype=th.float32), _meta(2, dtype=th.float32), _meta(8, dtype=th.float32)
    t = m[:, 0]
    o = th.ops.flex_rnn
    return {
        'linear_attention': (lambda q, k, v, g, s: F.linear_attention(q, k, v, g, s), [m, m, m, g, s]),
        'linear_attention_step': (lambda q, k, v, g, s: F.linear_attention_step(q, k, v, g, s), [t, t, t, g, s]),
        'layer_norm': (lambda x, w, b: F.layer_norm(x, w, b), [m, c, c]),
        'linear_attention backward': (lambda q, k, v, g, s, d, e: o.linear_attention_backward(q, k, v, g, s, None, d, e, 1.0, True, True), [m, m, m, g, s, m, s]),
        'layer_norm backward': (lambda x, w, b, d: o.layer_norm_backward(x, w, b, d, 1e-5, True, True), [m, c, c, m]),
    }


@pytest.mark.parametrize('name', list(_tangent_calls()))
def test_forward_mode_derivatives_are_refused(name):
    """A tangent of any argument would be lost without a word: it is an error, with and without a graph being recorded."""
    import torch.autograd.forward_ad as fw
    f, args = _tangent_calls()[name]
    for i in range(len(args)):
        for record in (True, False):
            with fw.dual_level(), th.set_grad_enabled(record):
                xs = [a.clone() for a in args]
                xs[i] = fw.make_dual(xs[i], th.ones_like(xs[i]))
                with pytest.raises(RuntimeError, match='forward-mode'):
                    f(*xs)
    with fw.dual_level():
        f(*[a.clone() for a in args])
        xs = [fw.make_dual(a.clone(), th.ones_like(a)) for a in args]
        with fw._set_fwd_grad_enabled(False):
            f(*xs)
    xs = tuple(a.clone() for a in args)
    with pytest.raises(RuntimeError, match='forward-mode'):
        th.func.jvp(f, xs, tuple(th.ones_like(x) for x in xs))


def test_a_step_of_inputs_that_want_gradients_is_refused_below_the_public_function_too():
    t, s, g = _meta(1, 2, 8, dtype=th.float32), _meta(1, 2, 8, 8, dtype=th.float32), _meta(2, dtype=th.float32)
    call = th.ops.flex_rnn.linear_attention_step
    with pytest.raises(RuntimeError, match='cannot be differentiated'):
        call(t.clone().requires_grad_(), t, t, g, s, 1.0)
    with th.no_grad():
        call(t.clone().requires_grad_(), t, t, g, s, 1.0)
    call(t, t, t, g, s, 1.0)


def test_a_library_that_cannot_be_loaded_leaves_the_package_usable(monkeypatch, tmp_path):
    """A truncated file, or one linked against another PyTorch: the import goes on, the first call says what to do."""
    bad = tmp_path / 'libfrnn_ops.so'
    bad.write_bytes(b'\x7fELF not a library')
    monkeypatch.setattr(handwritten, '_lib', None)
    monkeypatch.setattr(handwritten, 'OPS_PATH', str(bad))
    handwritten.load_if_built()
    assert handwritten._lib is None
    with pytest.raises(runtime.RuntimeError_, match=r'cannot be loaded.*build\(\)'):
        F.layer_norm(_meta(2, 8))


def test_a_library_from_other_sources_is_not_taken():
    """The host code shares argument blocks with the kernels: its file's name stands for both, and for PyTorch."""
    name = handwritten.library_name
    sources = handwritten.sources()
    csrc = os.path.join(os.path.dirname(handwritten.__file__), 'csrc')
    used = {s for s, _, _ in handwritten.builds()} | {'frnn_ops.cpp'}
    for f in used:
        with open(os.path.join(csrc, f)) as h:
            assert sources[f] == h.read()
    assert 'frnn_rt.h' in sources and 'handwritten.py' in sources
    assert handwritten.OPS_PATH == os.path.join(os.path.dirname(handwritten.__file__), name(sources, th.__version__))
    assert name(sources, 'another PyTorch') != name(sources, th.__version__)
    for f in sources:
        assert name({**sources, f: sources[f] + ' '}, th.__version__) != name(sources, th.__version__)


def fast_then_slow(dtype):
    """Decays that leave e^-9 a token and then hardly any, with cotangents 2^26 times as large behind: what early tokens carry
    over is nothing against what late ones sum to."""
    inputs, _ = lc.make(dtype, 1, 700, 2, 1, 32, 32)
    dy, ds = lc.cotangents(inputs)
    early = th.arange(700) < 400
    inputs[3] = th.where(early[None, :, None], -9 + 0.1 * inputs[3], 0.02 * inputs[3])
    dy = (dy.float() * th.where(early, 1.0, 2.0 ** 26)[None, :, None, None]).to(dtype)
    return inputs, dy, ds


def test_the_bound_of_the_gradient_of_g_refuses_sums_over_a_whole_sequence():
    """What the borders are for: products rounded to 32 bits, summed from the sequence's end, miss the bound that the GPU's result
    has to keep; summed from the next border they keep it."""
    inputs, dy, ds = fast_then_slow(th.float32)
    y, s, grads = lc.run64(inputs, None, 1.0, dy, ds)
    ay, a_s, agrads = lc.run64(lc.absolute(inputs), None, 1.0, dy.abs(), ds.abs())
    bound = lc.bound_of_dg(inputs, None, agrads, a_s, ds, 2.0 ** -20 + (32 + 32 + 700) * 2.0 ** -24)
    q, k = (x.double().repeat_interleave(2, 2) for x in inputs[:2])
    v, gate = inputs[2].double(), inputs[3].double()
    # each head's own dq and dk, by giving it a query and key of its own
    own = [q, k, v, gate, inputs[4].double()]
    _, _, each = lc.run64(own, None, 1.0, dy, ds)
    rounded = [(x * d).sum(-1).float().double() for x, d in ((q, each[0]), (k, each[1]))]
    exact = [(x * d).sum(-1) for x, d in ((q, each[0]), (k, each[1]))]
    whole = (rounded[0] - rounded[1]).flip(1).cumsum(1).flip(1) + (s * ds.double()).sum((-1, -2))[:, None]
    assert bool(((whole - grads[3]).abs() > 10 * bound)[:, :256].any())
    fine = (exact[0] - exact[1]).flip(1).cumsum(1).flip(1) + (s * ds.double()).sum((-1, -2))[:, None]
    assert float((fine - grads[3]).abs().max()) < 1e-6 * float(grads[3].abs().max())        # (the formula itself, in 64 bits)
    spans = th.empty_like(whole)
    for t0, t1 in ((0, 256), (256, 512), (512, 672), (672, 700)):
        d = rounded[0][:, t0:t1] - rounded[1][:, t0:t1]
        border = grads[3][:, t1:t1 + 1] if t1 < 700 else (s * ds.double()).sum((-1, -2))[:, None]
        spans[:, t0:t1] = d.flip(1).cumsum(1).flip(1) + border
    assert bool(((spans - grads[3]).abs() <= bound).all())


def test_gpu_gradient_cases_reach_every_build_that_serves_the_gradient_of_g():
    """Each is a code object of its own: the widths of what is staged, the operands' layout, and shared heads choose it."""
    import test_gpu_linear as t
    names = {th.bfloat16: 0, th.float16: 1, th.float32: 2}
    reached = set()
    for case in t.GRADIENT_BUILDS:
        dtype, B, T, H, Hk, M, N, opts = case
        fast = int(M % 8 == 0 and N % 8 == 0)
        if T > 12 * 32:
            reached.add((names[dtype], next(w for w in (64, 128, 256) if M <= w), fast, int(bool(fast and H > Hk and dtype != th.float32))))
    built = {(d['IN'], d['W'], d['FAST'], d['WIDE']) for d in (dict(b[2]) for b in handwritten.builds()) if d.get('DOTS')}
    assert reached == built


def test_borders_of_shared_decays_fit_in_memory():
    """Between borders lie 8 blocks for decays per token; one for a shared decay, more where what is written down at them would
    take over 8 GiB."""
    every = handwritten.blocks_between_borders
    assert every(8, 1024, 32, 128, 128, False) == 8 and every(1, 2 ** 24, 64, 256, 256, False) == 8
    assert every(8, 1024, 32, 128, 128, True) == 1 and every(1, 0, 1, 1, 1, True) == 1
    last = 1
    for T in (2 ** 15, 2 ** 17, 2 ** 18, 2 ** 19, 2 ** 21, 2 ** 31 - 65):
        n = every(1, T, 32, 128, 128, True)
        size = 32 * -(-T // (32 * n)) * 128 * 128 * 4
        assert last <= n <= 8 and (size <= 2 ** 33 or n == 8) and (n == 1 or 2 * size > 2 ** 33)
        last = n
    assert last == 8
