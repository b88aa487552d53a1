"""What the speed of the token-mixing operators is measured on: one pass through one operator, as a user's program calls it.

Four paths:

* ``attention`` -- leaky attention, linear attention whose state leaks with a decay for each head: for every sample and
  head S[t] = (1 - decay / 4096) S[t-1] + key[t] (outer) value[t], out[t] = scale * query[t] S[t]; forward, or a training
  step with the gradients of everything that is learned;
* ``step``      -- the same for one token a sample, on a state that is kept between calls;
* ``norm``      -- group norm over the last axis with an activation behind it;
* ``dropout``   -- dropout whose mask comes from a counter (Philox-4x32 with ten rounds, sixteen bits a decision) and is
  never stored, with a decision of its own for each element or one for all time steps of a neuron.

``run`` computes them with elementary torch operations in float32, or, where ``own`` is set, through this package's entry
points.
"""
import math

import torch

own = False

DEVICE = 'cuda'
CHUNK = 128            # tokens that the plain form of the attention takes at once


def listed():
    return [
        # one small batch of short samples at inference: what a launch costs
        dict(name='attention_small', path='attention', train=False, dtype='float32', samples=4, tokens=200, heads=2,
             keys=64, values=64, spikes=True, learn=False, state=False, ragged=False),
        # queries, keys and values that are spikes of a dense layer's neurons, 256 of them; decays trained
        dict(name='attention_spikes_train', path='attention', train=True, dtype='float32', samples=32, tokens=1500,
             heads=4, keys=64, values=64, spikes=True, learn=True, state=False, ragged=False),
        # a wider layer over shorter samples in bfloat16, decays fixed
        dict(name='attention_half_train', path='attention', train=True, dtype='bfloat16', samples=64, tokens=1000,
             heads=8, keys=64, values=64, spikes=False, learn=False, state=False, ragged=False),
        # samples of different lengths that go on from an earlier part of themselves; heads of odd sizes
        dict(name='attention_ragged_train', path='attention', train=True, dtype='bfloat16', samples=16, tokens=1450,
             heads=8, keys=48, values=80, spikes=False, learn=True, state=True, ragged=True),
        # one long prompt before generation, which needs its last state
        dict(name='attention_prompt', path='attention', train=False, dtype='bfloat16', samples=1, tokens=32768, heads=8,
             keys=128, values=128, spikes=False, learn=False, state=True, ragged=False),
        # generation for one user: latency
        dict(name='step_one', path='step', dtype='float32', samples=1, heads=8, keys=64, values=64),
        # generation for many at once: the states are all there is to move
        dict(name='step_many', path='step', dtype='bfloat16', samples=256, heads=16, keys=128, values=128),
        # the norm of each head's result in a small batch at inference
        dict(name='norm_small', path='norm', train=False, dtype='float32', samples=800, pixels=1, channels=128, groups=2,
             activation='silu'),
        # the same in training, behind the attention over 32 samples of 1500 tokens
        dict(name='norm_tokens_train', path='norm', train=True, dtype='bfloat16', samples=48000, pixels=1, channels=256,
             groups=4, activation='silu'),
        # an image tensor with the channels last: groups that reach over a whole image
        dict(name='norm_image_train', path='norm', train=True, dtype='float32', samples=32, pixels=1024, channels=512,
             groups=32, activation='silu'),
        # dropout behind that norm
        dict(name='dropout_tokens_train', path='dropout', train=True, dtype='bfloat16', shape='48000x256', p=0.1,
             neurons=False),
        # whole neurons silenced in the largest time-innermost tensor of the neuron benchmarks
        dict(name='dropout_neurons_train', path='dropout', train=True, dtype='float32', shape='64x1024x2000', p=0.2,
             neurons=True),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head_size(rng):
    """16 to 128: any number, or a multiple of four or sixteen as most are."""
    grain = rng.choice((1, 4, 16, 16))
    return grain * _log_uniform(rng, 16 / grain, 128 / grain)


def draw(rng):
    path = rng.choice(('attention', 'attention', 'attention', 'step', 'norm', 'norm', 'dropout'))
    dtype = rng.choice(('float32', 'bfloat16'))
    if path == 'attention':
        train = rng.random() < 0.6
        heads, keys, values = _log_uniform(rng, 1, 16), _head_size(rng), _head_size(rng)
        # elements of the value tensor and, with them, of the others
        numel = _log_uniform(rng, 20000, 30000000)
        tokens = min(_log_uniform(rng, 1, 16384), max(1, numel // (heads * max(keys, values))))
        samples = max(1, min(256, numel // (heads * max(keys, values) * tokens)))
        return dict(path=path, train=train, dtype=dtype, samples=samples, tokens=tokens, heads=heads, keys=keys,
                    values=values, spikes=rng.random() < 0.3, learn=train and rng.random() < 0.5,
                    state=rng.random() < 0.4, ragged=rng.random() < 0.4)
    if path == 'step':
        samples, heads = _log_uniform(rng, 1, 256), _log_uniform(rng, 1, 16)
        return dict(path=path, dtype=dtype, samples=samples, heads=heads, keys=_head_size(rng),
                    values=_head_size(rng))
    if path == 'norm':
        image, train = rng.random() < 0.5, rng.random() < 0.6
        groups = rng.choice((1, 2, 4, 8, 16, 32))
        channels = groups * _log_uniform(rng, 4, 128 if groups < 8 else 24)
        pixels = rng.randint(7, 64) ** 2 if image else 1
        samples = max(1, min(64 if image else 65536, _log_uniform(rng, 20000, 17000000) // (channels * pixels)))
        return dict(path=path, train=train, dtype=dtype, samples=samples, pixels=pixels, channels=channels,
                    groups=groups, activation=rng.choice(('none', 'relu', 'silu', 'silu', 'gelu')))
    neurons = rng.random() < 0.4
    numel = _log_uniform(rng, 20000, 120000000 if neurons else 17000000)
    last = _log_uniform(rng, 50, 2000)
    return dict(path=path, train=rng.random() < 0.6, dtype=dtype, shape='%dx%d' % (max(1, numel // last), last),
                p=round(rng.uniform(0.05, 0.6), 3), neurons=neurons)


# ------------------------------------------------------------------------------------------------ state
def _decays(heads):
    """12-bit decays from 1024 (a memory of four steps) to 2 (one of two thousand), as many as there are heads."""
    at = torch.linspace(10, 1, heads, dtype=torch.float64) if heads > 1 else torch.tensor([5.0], dtype=torch.float64)
    return torch.round(2 ** at).float().to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    path, dtype = case['path'], getattr(torch, case['dtype'])
    st = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    def spikes(*shape):
        return (torch.rand(shape, generator=gen, device=DEVICE) < 0.1).float()

    if path == 'attention':
        n, t, h, k, v = (case[x] for x in ('samples', 'tokens', 'heads', 'keys', 'values'))
        make = spikes if case['spikes'] else normal
        st.update(query=make(n, t, h, k).to(dtype), key=make(n, t, h, k).to(dtype), value=make(n, t, h, v).to(dtype),
                  decay=_decays(h), scale=k ** -0.5, state=normal(n, h, k, v) * 4 if case['state'] else None,
                  lengths=None)
        if case['ragged']:
            lengths = torch.randint(0, t + 1, (n,), generator=gen, device=DEVICE)
            st['lengths'] = torch.where(torch.arange(n, device=DEVICE) == 0, torch.full_like(lengths, t), lengths).int()
        if case['train']:
            wrt = ['query', 'key', 'value'] + ['decay'] * case['learn'] + ['state'] * case['state']
            st['wrt'] = [st[x].requires_grad_() for x in wrt]
            st['upstream'] = [normal(n, t, h, v).to(dtype)] + ([normal(n, h, k, v)] if case['state'] else [])
    elif path == 'step':
        n, h, k, v = (case[x] for x in ('samples', 'heads', 'keys', 'values'))
        st.update(query=normal(n, h, k).to(dtype), key=normal(n, h, k).to(dtype), value=normal(n, h, v).to(dtype),
                  decay=_decays(h), scale=k ** -0.5, state=normal(n, h, k, v) * 4)
    elif path == 'norm':
        shape = (case['samples'], case['pixels'], case['channels'])
        st.update(x=(normal(*shape) * 2 + 0.5).to(dtype), weight=1 + 0.1 * normal(case['channels']),
                  bias=0.1 * normal(case['channels']))
        if case['train']:
            st['wrt'] = [st[x].requires_grad_() for x in ('x', 'weight', 'bias')]
            st['upstream'] = [normal(*shape).to(dtype)]
    else:
        shape = tuple(int(d) for d in case['shape'].split('x'))
        st.update(x=normal(*shape).to(dtype), seed=(seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), offset=seed % 1000)
        if case['train']:
            st['wrt'] = [st['x'].requires_grad_()]
            st['upstream'] = [normal(*shape).to(dtype)]
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_attention(st):
    """Chunks of CHUNK tokens: the products inside a chunk, and the state at its start, which is a weighted sum of what
    the chunks before it add."""
    q, k, v = (st[x].float().permute(0, 2, 1, 3) for x in ('query', 'key', 'value'))
    n, h, t, dk = q.shape
    dv = v.shape[-1]
    a = 1 - st['decay'] / 4096
    length = torch.full((n,), t, device=q.device) if st['lengths'] is None else st['lengths'].long()
    there = (torch.arange(t, device=q.device) < length[:, None])[:, None, :, None]
    k, v = torch.where(there, k, 0), torch.where(there, v, 0)
    chunks = -(-t // CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, chunks * CHUNK - t)).reshape(n, h, chunks, CHUNK, -1)
               for x in (q, k, v))

    def power(exponent):                          # a ** exponent for each head, 0 where the exponent is negative
        shape = (h,) + (1,) * exponent.dim()
        return torch.where(exponent >= 0, a.reshape(shape) ** exponent.clamp(min=0), 0)

    i = torch.arange(CHUNK, device=q.device)
    c = torch.arange(chunks, device=q.device)
    scores = torch.matmul(q, k.transpose(-1, -2)) * power(i[:, None] - i)[:, None]
    added = torch.matmul((k * power(CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2), v)
    start = torch.matmul(power(CHUNK * (c[:, None] - 1 - c)), added.reshape(n, h, chunks, dk * dv))
    start = start.reshape(n, h, chunks, dk, dv)
    if st['state'] is not None:
        start = start + power(CHUNK * c)[:, :, None, None] * st['state'][:, :, None]
    out = torch.matmul(scores, v) + power(i + 1)[:, None, :, None] * torch.matmul(q, start)
    out = out.reshape(n, h, chunks * CHUNK, dv)[:, :, :t] * st['scale']
    out = torch.where(there, out, 0).permute(0, 2, 1, 3).to(st['query'].dtype).contiguous()
    if st['state'] is None:
        return [out]
    left = length[:, None, None] - 1 - torch.arange(chunks * CHUNK, device=q.device)        # steps after a token
    weight = torch.where(left >= 0, a[:, None] ** left.clamp(min=0), 0).reshape(n, h, chunks, CHUNK, 1)
    last = torch.matmul((k * weight).reshape(n, h, -1, dk).transpose(-1, -2), v.reshape(n, h, -1, dv))
    return [out, last + (a ** length[:, None])[:, :, None, None] * st['state']]


def _plain_step(st):
    a = (1 - st['decay'] / 4096)[:, None, None]
    state = st['state'].mul_(a).add_(st['key'].float()[..., None] * st['value'].float()[:, :, None, :])
    out = torch.matmul(st['query'].float()[:, :, None, :], state)[:, :, 0] * st['scale']
    return [out.to(st['query'].dtype), state]


def _plain_norm(st):
    case, x = st['case'], st['x']
    n, s, c = x.shape
    y = x.float().reshape(n, s, case['groups'], -1)
    y = y - y.mean((1, 3), keepdim=True)
    y = y * torch.rsqrt((y * y).mean((1, 3), keepdim=True) + 1e-5)
    y = y.reshape(n, s, c) * st['weight'] + st['bias']
    if case['activation'] == 'relu':
        y = torch.where(y > 0, y, 0)
    elif case['activation'] == 'silu':
        y = y / (1 + torch.exp(-y))
    elif case['activation'] == 'gelu':
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return [y.to(x.dtype)]


def _times(a, b):
    """(high, low) 32 bits of the product of a 32-bit tensor and a 32-bit number, held in 64-bit tensors."""
    high = ((a >> 16) * b + (((a & 0xffff) * b) >> 16)) >> 16
    return high, (a * b) & 0xffffffff


def _plain_keep(count, seed, offset, limit):
    """keep[i], i < count: whether the sixteen bits of decision i are at or above ``limit``."""
    block = torch.arange((count + 7) // 8, device=DEVICE)
    w = [block & 0xffffffff, block >> 32, torch.full_like(block, offset & 0xffffffff), torch.full_like(block, offset >> 32)]
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(10):
        h0, l0 = _times(w[0], 0xD2511F53)
        h1, l1 = _times(w[2], 0xCD9E8D57)
        w = [h1 ^ w[1] ^ k0, l1, h0 ^ w[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    words = torch.stack(w, 1)
    return torch.stack((words & 0xffff, words >> 16), 2).reshape(-1)[:count] >= limit


def _limit(p):
    return round(p * 65536)


def _plain_dropout(st, x):
    case = st['case']
    limit = _limit(case['p'])
    if case['neurons']:
        keep = _plain_keep(x.numel() // x.shape[-1], st['seed'], st['offset'], limit).reshape(x.shape[:-1] + (1,))
    else:
        keep = _plain_keep(x.numel(), st['seed'], st['offset'], limit).reshape(x.shape)
    return torch.where(keep, x.float() * (65536 / (65536 - limit)), 0).to(x.dtype)


# ------------------------------------------------------------------------------------------------ one pass
def _own(st):
    import lava_dl_amd.slayer as slayer
    case = st['case']
    if case['path'] == 'attention':
        out = slayer.synapse.leaky_attention(st['query'], st['key'], st['value'], st['decay'], state=st['state'],
                                             lengths=st['lengths'], scale=st['scale'],
                                             return_state=st['state'] is not None)
        return list(out) if st['state'] is not None else [out]
    if case['path'] == 'step':
        return [slayer.synapse.leaky_attention_step(st['query'], st['key'], st['value'], st['decay'], st['state'],
                                                    scale=st['scale']), st['state']]
    if case['path'] == 'norm':
        return [slayer.neuron.norm.group_norm(st['x'], case['groups'], st['weight'], st['bias'],
                                              activation=case['activation'])]
    return [slayer.neuron.counter_dropout(st['x'], case['p'], st['seed'], st['offset'], per_neuron=case['neurons'])]


def _forward(st):
    if own:
        return _own(st)
    path = st['case']['path']
    return {'attention': _plain_attention, 'step': _plain_step, 'norm': _plain_norm}[path](st) if path != 'dropout' \
        else [_plain_dropout(st, st['x'])]


def run(state):
    case = state['case']
    if not case.get('train'):
        with torch.no_grad():
            return _forward(state)
    if case['path'] == 'dropout' and not own:                # the gradient passes where the value did
        with torch.no_grad():
            return [_plain_dropout(state, state['x']), _plain_dropout(state, state['upstream'][0])]
    out = _forward(state)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, state['wrt'], state['upstream']))


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attention(st):
    """The recurrence step by step, forwards for the results, the queries' and the decays' gradients, backwards for the
    others.  A step that lies behind a sample's end leaves its state as it is."""
    case = st['case']
    q, k, v = (st[x].detach().double() for x in ('query', 'key', 'value'))
    n, t, h, dk = q.shape
    dv = v.shape[-1]
    scale, a = st['scale'], (1 - st['decay'].detach().double() / 4096)
    lengths = [t] * n if st['lengths'] is None else st['lengths'].tolist()
    on = torch.tensor([[step < length for length in lengths] for step in range(t)], device=DEVICE, dtype=torch.float64)
    k, v = k * on.t()[:, :, None, None], v * on.t()[:, :, None, None]
    # what a step multiplies the state with: a, or 1 behind the end
    leak = (a * on[:, :, None] + (1 - on[:, :, None])).reshape(t, n * h, 1, 1)
    on = on.repeat_interleave(h, 1).reshape(t, n * h, 1, 1)
    q, k, v = (x.permute(1, 0, 2, 3).reshape(t, n * h, -1) for x in (q, k, v))

    def back(x, d):
        return x.reshape(t, n, h, d).permute(1, 0, 2, 3)

    first = torch.zeros(n, h, dk, dv, device=DEVICE, dtype=torch.float64)
    if st['state'] is not None:
        first = st['state'].detach().double()
    S = first.reshape(n * h, dk, dv).clone()
    out = torch.empty(t, n * h, dv, device=DEVICE, dtype=torch.float64)
    train = case['train']
    if train:
        dy = (st['upstream'][0].double() * scale).permute(1, 0, 2, 3).reshape(t, n * h, dv) * on[:, :, :, 0]
        dq, dk_, dv_ = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        W, slope = torch.zeros_like(S), torch.zeros(n * h, device=DEVICE, dtype=torch.float64)      # W = dS / da
    for s in range(t):
        if train and case['learn']:
            W = leak[s] * W + on[s] * S
        S = torch.baddbmm(S * leak[s], k[s][:, :, None], v[s][:, None, :])
        out[s] = torch.bmm(q[s][:, None, :], S)[:, 0] * on[s][:, :, 0]
        if train:
            dq[s] = torch.bmm(S, dy[s][:, :, None])[:, :, 0]
            if case['learn']:
                slope += (torch.bmm(q[s][:, None, :], W)[:, 0] * dy[s]).sum(1)
    got = [back(out, dv) * scale] + ([S.reshape(n, h, dk, dv)] if st['state'] is not None else [])
    if not train:
        return got
    D = torch.zeros_like(S)
    if st['state'] is not None:
        D = st['upstream'][1].double().reshape(n * h, dk, dv).clone()
        slope += (D * W).sum((1, 2))
    for s in range(t - 1, -1, -1):
        D = torch.baddbmm(D, q[s][:, :, None], dy[s][:, None, :])
        dk_[s] = torch.bmm(D, v[s][:, :, None])[:, :, 0] * on[s][:, :, 0]
        dv_[s] = torch.bmm(k[s][:, None, :], D)[:, 0] * on[s][:, :, 0]
        D = D * leak[s]
    got += [back(dq, dk), back(dk_, dk), back(dv_, dv)]
    if case['learn']:
        got.append(-slope.reshape(n, h).sum(0) / 4096)
    if st['state'] is not None:
        got.append(D.reshape(n, h, dk, dv))
    return got


def _exact_norm(st):
    """The formulas of the norm, the activation and their gradients."""
    case, x = st['case'], st['x'].detach().double()
    n, s, c = x.shape
    g = case['groups']
    w, b = st['weight'].detach().double(), st['bias'].detach().double()
    x = x.reshape(n, s, g, c // g)
    mean = x.mean((1, 3), keepdim=True)
    scale = ((x - mean).square().mean((1, 3), keepdim=True) + 1e-5) ** -0.5
    hat = (x - mean) * scale
    z = hat.reshape(n, s, c) * w + b
    if case['activation'] == 'relu':
        y, slope = z.clamp(min=0), (z > 0).double()
    elif case['activation'] == 'silu':
        gate = torch.sigmoid(z)
        y, slope = z * gate, gate * (1 + z * (1 - gate))
    elif case['activation'] == 'gelu':
        below = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        y, slope = z * below, below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)
    if not case['train']:
        return [y]
    dz = st['upstream'][0].double() * slope
    dhat = (dz * w).reshape(n, s, g, c // g)
    dx = scale * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    return [y, dx.reshape(n, s, c), (dz * hat.reshape(n, s, c)).sum((0, 1)), dz.sum((0, 1))]


def _exact_dropout(st):
    """The counter in numpy's unsigned 64-bit numbers on the host."""
    import numpy as np
    case, x = st['case'], st['x'].detach()
    count = x.numel() // (x.shape[-1] if case['neurons'] else 1)
    word = np.uint64(0xffffffff)
    block = np.arange((count + 7) // 8, dtype=np.uint64)
    w0, w1 = block & word, block >> np.uint64(32)
    w2, w3 = np.full_like(block, st['offset'] & 0xffffffff), np.full_like(block, st['offset'] >> 32)
    k0, k1 = st['seed'] & 0xffffffff, st['seed'] >> 32
    for r in range(10):
        m0, m1 = w0 * np.uint64(0xD2511F53), w2 * np.uint64(0xCD9E8D57)
        w0, w2 = ((m1 >> np.uint64(32)) ^ w1 ^ np.uint64((k0 + r * 0x9E3779B9) % (1 << 32)),
                  (m0 >> np.uint64(32)) ^ w3 ^ np.uint64((k1 + r * 0xBB67AE85) % (1 << 32)))
        w1, w3 = m1 & word, m0 & word
    halves = np.stack([w0, w1, w2, w3], 1).astype('<u4').reshape(-1).view('<u2')[:count]
    limit = _limit(case['p'])
    keep = torch.from_numpy(halves >= limit).to(DEVICE).reshape(x.shape[:-1] + (1,) if case['neurons'] else x.shape)
    return [torch.where(keep, y.double() * 65536 / (65536 - limit), 0)
            for y in [x] + (st['upstream'] if case['train'] else [])]


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case['path'] == 'attention':
            return _exact_attention(st)
        if case['path'] == 'step':
            state = st['state'].double() * (1 - st['decay'].double() / 4096)[:, None, None]
            state = state + st['key'].double()[..., None] * st['value'].double()[:, :, None, :]
            return [(st['query'].double()[..., None] * state).sum(2) * st['scale'], state]
        return _exact_norm(st) if case['path'] == 'norm' else _exact_dropout(st)


# ------------------------------------------------------------------------------------------------ figures
def work(case):
    """Inputs once, outputs once; the products of the recurrence as it stands: two a token forward, five more backward
    (the state and its adjoint again, and the gradients of query, key and value)."""
    size = 2 if case['dtype'] == 'bfloat16' else 4
    if case['path'] == 'attention':
        n, t, h, k, v = (case[x] for x in ('samples', 'tokens', 'heads', 'keys', 'values'))
        state = (8 if case['state'] else 0) * n * h * k * v
        forward = n * t * h * (2 * k + 2 * v) * size + state
        product = 2 * n * t * h * k * v
        if not case['train']:
            return {'bytes': forward, 'flops': 2 * product}
        return {'bytes': 2 * forward, 'flops': 7 * product}
    if case['path'] == 'step':
        n, h, k, v = (case[x] for x in ('samples', 'heads', 'keys', 'values'))
        return {'bytes': n * h * (8 * k * v + (2 * k + 2 * v) * size), 'flops': 5 * n * h * k * v}
    if case['path'] == 'norm':
        numel = case['samples'] * case['pixels'] * case['channels']
        return {'bytes': numel * size * (4 if case['train'] else 2), 'flops': numel * (40 if case['train'] else 14)}
    numel = math.prod(int(d) for d in case['shape'].split('x'))
    return {'bytes': numel * size * (4 if case['train'] else 2), 'flops': numel * (2 if case['train'] else 1)}
