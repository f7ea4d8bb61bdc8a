"""Cases, inputs and plain forms of the operators beside the compiled recurrences: linear attention with a decay for
each head (prompts, training, single tokens) and layer norm (forward, training).

A case's `op` is one of
  prompt      y, state = linear_attention(q, k, v, g, state, lengths=, scale=)
  train       the same with gradients of q, k, v, g and the initial state, for given gradients of y and the final state
  step        y = linear_attention_step(q, k, v, g, state, scale=), which updates the state in place
  norm        y = layer_norm(x, weight, bias, eps)
  norm_train  the same with gradients of x, weight and bias, for a given gradient of y

Shapes: q, k [B,T,Hk,N] (Hk divides H: heads share queries and keys), v [B,T,H,M], g the logarithm of the decay
[B,T,H] or [H], state [B,H,M,N], lengths [B] (tokens from there on are padding: y is zero and the state stands still);
x [...,C] or [...,Hw,C], weight and bias [C] or [Hw,C].

    S_t = exp(g_t) S_(t-1) + v_t k_t^T,   y_t = scale * S_t q_t
"""
import math

import torch as th

own = False

DTYPES = {'bf16': th.bfloat16, 'fp16': th.float16, 'fp32': th.float32}
SIZES = {'bf16': 2, 'fp16': 2, 'fp32': 4}
EPS = 1e-5
CHUNK = 64          # tokens per block of the plain form
NO_DECAY = -200.0   # exp of less is zero in 32 bits


def _linear(name, op, dtype, B, T, H, Hk, M, N, g='token', g_dtype='fp32', state='fp32', ragged=False, resets=0.0):
    c = dict(op=op, dtype=dtype, B=B, T=T, H=H, Hk=Hk, M=M, N=N, g=g, g_dtype=g_dtype, state=state, ragged=ragged,
             resets=resets)
    return c if name is None else dict(c, name=name)


def _norm(name, op, dtype, rows, Hw, C, w_dtype):
    c = dict(op=op, dtype=dtype, rows=rows, Hw=Hw, C=C, w_dtype=w_dtype)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # the smallest recurrence of the test-suite: a launch's latency
        _linear('prompt T64 H2 16x16 fp32', 'prompt', 'fp32', 1, 64, 2, 2, 16, 16, g_dtype='fp32'),
        # a batch of prompts, one pair of query and key for all heads (the mamba2 workload's shape)
        _linear('prompt B8 T1024 H64 64x128 bf16', 'prompt', 'bf16', 8, 1024, 64, 1, 64, 128),
        # one long document, a fixed decay for each head (retention)
        _linear('prompt T32768 H32 128x128 bf16', 'prompt', 'bf16', 1, 32768, 32, 32, 128, 128, g='head', state='none'),
        # a padded batch of packed documents (the decay of a document's first token is zero), odd head sizes
        _linear('prompt ragged B5 T777 80x56 fp16', 'prompt', 'fp16', 5, 777, 6, 3, 80, 56, g_dtype='fp16', state='fp16', ragged=True,
                resets=0.01),
        # a training step's mixer at the benchmark's size
        _linear('train B8 T1024 H32 128x128 bf16', 'train', 'bf16', 8, 1024, 32, 32, 128, 128),
        # training in 32 bits, packed documents, shared keys, a length that ends inside a block
        _linear('train B2 T500 H8 64x48 fp32', 'train', 'fp32', 2, 500, 8, 2, 64, 48, ragged=True, resets=0.02),
        # one token of one user
        _linear('step B1 H32 128x128 bf16', 'step', 'bf16', 1, 1, 32, 32, 128, 128),
        # one token of each of many users: the states are what counts
        _linear('step B128 H32 128x128 bf16', 'step', 'bf16', 128, 1, 32, 32, 128, 128),
        # the norm of each head's output: for one token, and for a batch of prompts
        _norm('norm 1x32x128 bf16', 'norm', 'bf16', 1, 32, 128, 'fp32'),
        _norm('norm 8192x32x128 bf16', 'norm', 'bf16', 8192, 32, 128, 'fp32'),
        # the same in training; a norm over the model's width in training
        _norm('norm_train 8192x32x128 bf16', 'norm_train', 'bf16', 8192, 32, 128, 'fp32'),
        _norm('norm_train 8192x4096 fp16', 'norm_train', 'fp16', 8192, 0, 4096, 'fp16'),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['prompt', 'prompt', 'train', 'train', 'step', 'norm', 'norm_train'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if op in ('norm', 'norm_train'):
        Hw = rng.choice([0, 0, rng.randint(2, 64)])
        C = _log_uniform(rng, 8, 512) if Hw else _log_uniform(rng, 8, 8192)
        if rng.random() < 0.5:
            C = max(8, C // 8 * 8)
        rows = _log_uniform(rng, 1, max(1, min(65536, (1 << 24) // (C * max(Hw, 1)))))
        return _norm(None, op, dtype, rows, Hw, C, rng.choice([dtype, 'fp32']))
    size = lambda: rng.choice([16, 32, 64, 96, 128, 192, 256, rng.randint(8, 256), rng.randint(8, 256) // 8 * 8])  # noqa: E731
    M, N = size(), size()
    Hk = _log_uniform(rng, 1, 16)
    H = Hk * rng.choice([1, 1, 1, 2, 4, 8])
    if op == 'step':
        B, T = _log_uniform(rng, 1, max(1, min(256, (1 << 25) // (H * M * N)))), 1
    else:
        most = (1 << 24) // (H * (M + N))
        B = _log_uniform(rng, 1, 8)
        T = _log_uniform(rng, 1, max(1, min(16384, most // B)))
    c = _linear(None, op, dtype, B, T, H, Hk, M, N, g=rng.choice(['token', 'token', 'head']), g_dtype=rng.choice([dtype, 'fp32']),
                state=rng.choice([dtype, 'fp32', 'fp32'] + (['none'] if op != 'step' else [])))
    if op != 'step':
        c['ragged'] = rng.random() < 0.3
        c['resets'] = rng.choice([0.0, 0.0, 0.02]) if c['g'] == 'token' else 0.0
    return c


def work(c):
    z = SIZES[c['dtype']]
    if c['op'] in ('norm', 'norm_train'):
        heads = max(c['Hw'], 1)
        n, w = c['rows'] * heads * c['C'], heads * c['C'] * SIZES[c['w_dtype']]
        if c['op'] == 'norm':
            return {'bytes': 2 * n * z + 2 * w, 'flops': 8 * n}
        return {'bytes': 4 * n * z + 4 * w, 'flops': 20 * n}
    B, T, H, Hk, M, N = (c[x] for x in ('B', 'T', 'H', 'Hk', 'M', 'N'))
    qk, v = B * T * Hk * N * z, B * T * H * M * z
    g = (H if c['g'] == 'head' else B * T * H) * SIZES[c['g_dtype']]
    s = B * H * M * N * SIZES['fp32' if c['state'] == 'none' else c['state']]
    s_in = 0 if c['state'] == 'none' else s
    tokens = B * T * H
    if c['op'] in ('prompt', 'step'):
        return {'bytes': 2 * qk + 2 * v + g + s + s_in, 'flops': 4 * tokens * M * N}
    # q, k, v, dy and the states are read, y, dq, dk, dv, dg and the states written
    return {'bytes': 4 * qk + 4 * v + 2 * g + 2 * (s + s_in), 'flops': (4 + 8) * tokens * M * N}


def prepare(c, seed):
    gen = th.Generator(device='cuda').manual_seed(seed)

    def randn(*shape):
        return th.randn(*shape, generator=gen, device='cuda')

    dt = DTYPES[c['dtype']]
    if c['op'] in ('norm', 'norm_train'):
        last = (c['Hw'], c['C']) if c['Hw'] else (c['C'],)
        w_dt = DTYPES[c['w_dtype']]
        s = {'c': c, 'x': (randn(c['rows'], *last) * 1.5 + 0.5).to(dt), 'weight': (1 + 0.3 * randn(*last)).to(w_dt),
             'bias': (0.2 * randn(*last)).to(w_dt)}
        if c['op'] == 'norm_train':
            s['dy'] = randn(c['rows'], *last).to(dt)
        return s
    B, T, H, Hk, M, N = (c[x] for x in ('B', 'T', 'H', 'Hk', 'M', 'N'))
    k = randn(B, T, Hk, N)
    k = k / (k * k).sum(-1, keepdim=True).sqrt()
    s = {'c': c, 'q': randn(B, T, Hk, N).to(dt), 'k': k.to(dt), 'v': randn(B, T, H, M).to(dt), 'scale': N ** -0.5,
         'lengths': None, 'state': None}
    if c['g'] == 'head':       # the fixed decays of retention
        g = th.log(1 - th.exp2(-2 - 6 * th.arange(H, device='cuda') / H - 0.1 * th.rand(H, generator=gen, device='cuda')))
    else:                      # gates as a model makes them: mostly slow, some that forget at once
        g = -0.5 * th.log1p(th.exp(1.5 * randn(B, T, H) - 1))
        if c['resets']:
            g = th.where(th.rand(B, T, H, generator=gen, device='cuda') < c['resets'], -math.inf, g)
    s['g'] = g.to(DTYPES[c['g_dtype']])
    if c['state'] != 'none':
        s['state'] = (0.5 * randn(B, H, M, N)).to(DTYPES[c['state']])
    if c['ragged']:
        lens = th.randint(0, T + 1, (B,), generator=gen, device='cuda')
        lens[seed % B] = T
        s['lengths'] = lens
    if c['op'] == 'step':
        for x in ('q', 'k', 'v', 'g'):
            s[x] = s[x] if x == 'g' and c['g'] == 'head' else s[x][:, 0].contiguous()
    if c['op'] == 'train':
        s['dy'] = randn(B, T, H, M).to(dt)
        s['dstate'] = (0.5 * randn(B, H, M, N)).to(th.float32 if s['state'] is None else s['state'].dtype)
    return s


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    import flex_rnn_amd as F
    op = s['c']['op']
    if op == 'prompt':
        return F.linear_attention(s['q'], s['k'], s['v'], s['g'], s['state'], lengths=s['lengths'], scale=s['scale'])
    if op == 'step':
        y = F.linear_attention_step(s['q'], s['k'], s['v'], s['g'], s['state'], scale=s['scale'])
        return y, s['state']
    if op == 'norm':
        return F.layer_norm(s['x'], s['weight'], s['bias'], EPS)
    if op == 'norm_train':
        xs = [s[n].detach().requires_grad_() for n in ('x', 'weight', 'bias')]
        y = F.layer_norm(*xs, EPS)
        return (y.detach(), *th.autograd.grad(y, xs, s['dy']))
    xs = [s[n].detach().requires_grad_() for n in ('q', 'k', 'v', 'g', 'state') if s[n] is not None]
    y, sT = F.linear_attention(*xs, lengths=s['lengths'], scale=s['scale'])
    return (y.detach(), sT.detach(), *th.autograd.grad((y, sT), xs, (s['dy'], s['dstate'])))


# ------------------------------------------------------------------ plain forms
def _blocks(x, T):
    """[B,T,H,...] -> [B,H,blocks,CHUNK,...], zeros behind the last token."""
    pad = -T % CHUNK
    x = th.cat([x, x.new_zeros(x.shape[0], pad, *x.shape[2:])], 1) if pad else x
    x = x.reshape(x.shape[0], -1, CHUNK, *x.shape[2:])
    return x.movedim(3, 1)


def _tokens(x, T):
    """The inverse of `_blocks`."""
    x = x.movedim(1, 3)
    return x.reshape(x.shape[0], -1, *x.shape[3:])[:, :T]


def _decays(diff, keep):
    """exp of differences of summed logarithms (64 bits) where `keep`, zero elsewhere."""
    return th.exp(diff.masked_fill(~keep, -math.inf)).float()


def _plain_linear(s):
    c = s['c']
    B, T, H, Hk, M, N = (c[x] for x in ('B', 'T', 'H', 'Hk', 'M', 'N'))
    train, scale = c['op'] == 'train', s['scale']
    q, k, v = s['q'].float(), s['k'].float(), s['v'].float()
    g = s['g'].double().clamp(min=NO_DECAY)
    g = g.expand(B, T, H) if c['g'] == 'head' else g
    dy = s['dy'].float() * scale if train else None
    real = None
    if s['lengths'] is not None:
        real = th.arange(T, device=v.device)[None, :, None, None] < s['lengths'][:, None, None, None]
        q, k, v = (th.where(real, x, 0.0) for x in (q, k, v))
        g = th.where(real[..., 0], g, 0.0)
        dy = th.where(real, dy, 0.0) if train else None
    q, k = (x.repeat_interleave(H // Hk, 2) for x in (q, k))
    q, k, v, G = _blocks(q, T), _blocks(k, T), _blocks(v, T), _blocks(g, T).cumsum(-1)
    nb = G.shape[2]
    low = th.ones(CHUNK, CHUNK, dtype=th.bool, device=v.device).tril()
    E = _decays(G[..., :, None] - G[..., None, :], low)
    from_start, to_end = th.exp(G).float()[..., None], th.exp(G[..., -1:] - G).float()[..., None]
    P = (q @ k.mT) * E
    # states in front of each block and behind the last: a product with the decays between blocks
    total = G[..., -1].cumsum(-1)
    before = th.cat([th.zeros_like(total[..., :1]), total], -1)                    # [B,H,nb+1]
    order = th.arange(nb + 1, device=v.device)
    between = _decays(before[..., :, None] - total[..., None, :], order[:, None] > order[None, :nb])
    KV = v.mT @ (k * to_end)
    S = (between @ KV.flatten(-2)).unflatten(-1, (M, N))
    if s['state'] is not None:
        S = S + th.exp(before).float()[..., None, None] * s['state'].float()[:, :, None]
    y = (P @ v + from_start * (q @ S[:, :, :-1].mT)) * scale
    y = _tokens(y, T).to(s['v'].dtype)
    s_dt = th.float32 if s['state'] is None else s['state'].dtype
    sT = S[:, :, -1].to(s_dt)
    if not train:
        return y, sT
    dy = _blocks(dy, T)
    W = dy @ v.mT
    R = W * E
    S = S[:, :, :-1]
    # gradients of the states behind each block, and of the initial one
    back = _decays(total[..., None, :] - total[..., :, None] - (G[..., -1])[..., None, :], order[:nb, None] < order[None, :nb])
    first = _decays((before[..., :-1])[..., None, :], th.ones(1, nb, dtype=th.bool, device=v.device))
    QD = (dy * from_start).mT @ q
    dsT = s['dstate'].float()[:, :, None]
    D = (back @ QD.flatten(-2)).unflatten(-1, (M, N)) + th.exp(total[..., -1:] - total).float()[..., None, None] * dsT
    ds0 = (first @ QD.flatten(-2)).unflatten(-1, (M, N)) + th.exp(total[..., -1:]).float()[..., None, None] * dsT
    dq_state, dk_state = from_start * (dy @ S), to_end * (v @ D)
    dq, dk = R @ k + dq_state, R.mT @ q + dk_state
    dv = P.mT @ dy + to_end * (k @ D.mT)
    PW = (P * W).double()
    a = PW.sum(-1) - PW.sum(-2) + (q * dq_state).double().sum(-1)
    b = (k * dk_state).double().sum(-1)
    dg = a.flip(-1).cumsum(-1).flip(-1) + b.cumsum(-1) - b + (th.exp(G[..., -1]) * (D * S).double().sum((-1, -2)))[..., None]
    dq, dk = (_tokens(x, T).unflatten(2, (Hk, H // Hk)).sum(3) for x in (dq, dk))
    dg = _tokens(dg, T)
    if real is not None:
        dg = th.where(real[..., 0], dg, 0.0)
    dg = dg.sum((0, 1)) if c['g'] == 'head' else dg
    out = (y, sT, dq.to(s['q'].dtype), dk.to(s['k'].dtype), _tokens(dv, T).to(s['v'].dtype), dg.to(s['g'].dtype))
    return out if s['state'] is None else (*out, ds0[:, :, 0].to(s_dt))


def _plain_step(s):
    c = s['c']
    q, k = (s[x].float().repeat_interleave(c['H'] // c['Hk'], 1) for x in ('q', 'k'))
    new = th.exp(s['g'].float())[..., None, None] * s['state'].float() + s['v'].float()[..., :, None] * k[..., None, :]
    y = s['scale'] * (new * q[..., None, :]).sum(-1)
    s['state'].copy_(new)
    return y.to(s['v'].dtype), s['state']


def _plain_norm(s):
    x, w = s['x'].float(), s['weight'].float()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / (((x - mean) ** 2).mean(-1, keepdim=True) + EPS).sqrt()
    xhat = (x - mean) * rstd
    y = (xhat * w + s['bias'].float()).to(s['x'].dtype)
    if s['c']['op'] == 'norm':
        return y
    dy = s['dy'].float()
    d = dy * w
    dx = rstd * (d - d.mean(-1, keepdim=True) - xhat * (d * xhat).mean(-1, keepdim=True))
    return y, dx.to(s['x'].dtype), (dy * xhat).sum(0).to(s['weight'].dtype), dy.sum(0).to(s['bias'].dtype)


def run(state):
    if own:
        return _own(state)
    op = state['c']['op']
    if op in ('norm', 'norm_train'):
        return _plain_norm(state)
    return _plain_step(state) if op == 'step' else _plain_linear(state)


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op in ('norm', 'norm_train'):
        x, w, b = (s[n].double() for n in ('x', 'weight', 'bias'))
        C = case['C']
        centred = x - x.sum(-1, keepdim=True) / C
        std = th.sqrt((centred * centred).sum(-1, keepdim=True) / C + EPS)
        y = centred / std * w + b
        if op == 'norm':
            return y
        dy = s['dy'].double()
        dn = dy * w                                            # the gradient of the normalised row
        dstd = -(dn * centred).sum(-1, keepdim=True) / std ** 2
        dc = dn / std + dstd * centred / (C * std)             # of the centred row
        return y, dc - dc.sum(-1, keepdim=True) / C, (dy * centred / std).sum(0), dy.sum(0)
    B, H, Hk, M, N = (case[x] for x in ('B', 'H', 'Hk', 'M', 'N'))
    T = case['T']
    d = {n: None if s[n] is None else s[n].double() for n in ('q', 'k', 'v', 'g', 'state')}
    if op == 'step':
        q, k, v = d['q'], d['k'], d['v']
        q, k = q.repeat_interleave(H // Hk, 1), k.repeat_interleave(H // Hk, 1)
        S = th.exp(d['g'])[..., None, None] * d['state'] + v[..., None] * k[..., None, :]
        return (S @ q[..., None])[..., 0] * s['scale'], S
    decay = th.exp(d['g']).expand(B, T, H)
    q, k = d['q'].repeat_interleave(H // Hk, 2), d['k'].repeat_interleave(H // Hk, 2)
    v = d['v']
    valid = th.arange(T, device=v.device)[None] < (th.full((B,), T, device=v.device) if s['lengths'] is None else s['lengths'])[:, None]
    decay = th.where(valid[..., None], decay, 1.0)
    q, k, v = (x * valid[..., None, None] for x in (q, k, v))
    S = th.zeros(B, H, M, N, dtype=th.float64, device=v.device) if d['state'] is None else d['state'].clone()
    y, dq = th.empty_like(v), th.empty_like(q)
    dy = s['dy'].double() * valid[..., None, None] * s['scale'] if op == 'train' else None
    for t in range(T):
        S.mul_(decay[:, t, :, None, None]).add_(v[:, t, :, :, None] * k[:, t, :, None, :])
        y[:, t] = (S @ q[:, t, :, :, None])[..., 0]
        if op == 'train':
            dq[:, t] = (dy[:, t, :, None, :] @ S)[..., 0, :]
    y = y * s['scale']
    if op == 'prompt':
        return y, S
    D = s['dstate'].double().clone()
    end = (D * S).sum((-1, -2))
    dk, dv = th.empty_like(k), th.empty_like(v)
    for t in range(T - 1, -1, -1):
        D.add_(dy[:, t, :, :, None] * q[:, t, :, None, :])
        dk[:, t] = (v[:, t, :, None, :] @ D)[..., 0, :]
        dv[:, t] = (D @ k[:, t, :, :, None])[..., 0]
        D.mul_(decay[:, t, :, None, None])
    # a step's logarithm scales what it carries over: all that comes after it less what enters after it
    through = (q * dq).sum(-1) - (k * dk).sum(-1)
    dg = through.flip(1).cumsum(1).flip(1) + end[:, None]
    dg = th.where(valid[..., None] & (decay > 0), dg, 0.0)
    dq, dk = (x.reshape(B, T, Hk, H // Hk, N).sum(3) * valid[..., None, None] for x in (dq, dk))
    dg = dg.sum((0, 1)) if case['g'] == 'head' else dg
    out = (y, S, dq, dk, dv * valid[..., None, None], dg)
    return out if s['state'] is None else (*out, D)
