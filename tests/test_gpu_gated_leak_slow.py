"""Slow leaks over long samples: how far a state is off does not grow with the tokens.

Tolerance.  With U = 2^-24, as factors of what they belong to: a leak is (5 + 1.5 |z|) U off, what a token adds (10 + 3 |z|) U.  A wave joins
up to 16 tokens in float32, from nothing, and each rounds the factor it keeps, the product and the sum: 48 U of what these tokens add, and of what they
lose 2 U a token, 32 U, the word between tiles 2 U more.  What a span loses as a whole is at most twice what its tokens lose one by one, where it
keeps a half, so 68 U; below a half the product itself is as good.  From wave to wave and tile to tile states are float64.  So a state
is off by what it had before, kept; by (5 + 1.5 |z| + 96) U of what leaks; by (10 + 3 |z| + 96) U of what is added.  Walking from the state
in front of a wave rounds it once and then three times a token, 52 U of the magnitudes; behind a state that was kept in float32 and at most
eight waves of the backward pass once more, 80 U.  Backwards alike."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24
T = 32768 + 77
DRIVES = [None, 'gain', 'variance']


def make(dtype):
    """Half of the channels with an input that stays the same, half with a white one."""
    gen = torch.Generator().manual_seed(31)
    gate = torch.tensor([-5.3, -5.0, -7.0, -3.0, -6.0, -8.0, -9.5, -2.0])
    decay = torch.tensor([16.0, 16, 16, 1, 64, 512, 4096, 37])
    z = gate.repeat(2).expand(T, 16).clone()
    z[:, 7] += torch.randn(T, generator=gen)
    x, g = torch.ones(T, 16), torch.full((T, 16), 0.5)
    x[:, 8:], g[:, 8:] = torch.randn(T, 8, generator=gen), torch.randn(T, 8, generator=gen)
    return dict(x=x.to(dtype), z=z.to(dtype), g=g.to(dtype), decay=decay.repeat(2), state=torch.ones(16), gs=torch.ones(16))


def exact(d, drive):
    """{name: (value, bound)} of one sample, float64."""
    x, z, g = (d[k].double().numpy() for k in 'xzg')
    open_ = 1 / (1 + np.exp(-z))
    leak = d['decay'].double().numpy() / 4096 * open_
    f, slope = np.ones_like(leak), np.zeros_like(leak)
    if drive == 'gain':
        f, slope = leak, np.ones_like(leak)
    elif drive == 'variance':
        f = np.sqrt(leak * (2 - leak))
        slope = (1 - leak) / f
    add = f * x
    off_leak, off_add = (5 + 1.5 * abs(z)) * U, (10 + 3 * abs(z)) * U
    h, m, e = np.empty((3, T + 1, 16))
    h[0], m[0], e[0] = d['state'].numpy(), abs(d['state'].numpy()), 0
    keep, more, kinds = 1 - leak, (off_add + 96 * U) * abs(add), (off_leak + 96 * U) * leak
    for t in range(T):
        h[t + 1] = keep[t] * h[t] + add[t]
        e[t + 1] = keep[t] * e[t] + kinds[t] * m[t] + more[t]
        m[t + 1] = keep[t] * m[t] + abs(add[t])
    D, md, ed = np.empty((3, T, 16))
    G, mg, eg = d['gs'].double().numpy(), abs(d['gs'].double().numpy()), np.zeros(16)
    for t in range(T - 1, -1, -1):
        D[t], md[t], ed[t] = g[t] + G, abs(g[t]) + mg, eg
        eg = keep[t] * eg + kinds[t] * md[t] + 96 * U * abs(g[t])
        G, mg = keep[t] * D[t], keep[t] * md[t]
    ed += 52 * U * md
    before, size = h[:-1], abs(slope * x) + m[:-1]
    off = ed * size + md * (e[:-1] + 80 * U * m[:-1] + 2 * off_add * size)
    dleak, gate = D * (slope * x - before), leak * (1 - open_)
    return {'out': (h[1:], e[1:] + 52 * U * m[1:]), 'last': (h[T], e[T] + U * m[T]), 'dx': (f * D, f * (ed + off_add * md)),
            'dz': (dleak * gate, off * gate + 2 * md * size * leak * off_add), 'dstate': (G, eg + U * mg)}


@pytest.mark.parametrize('drive', DRIVES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_long_samples(dtype, drive):
    """One sample, cut up among workgroups, and two hundred, each walked by one."""
    import lava_dl_amd.slayer as slayer
    d = make(dtype)
    want = exact(d, drive)
    for n in (1, 200):
        x, z, state = (d[k].to(DEV).expand(n, *d[k].shape).requires_grad_() for k in ('x', 'z', 'state'))
        leaves = [x, z, state]
        out, last = slayer.neuron.gated_leak(x, z, d['decay'].to(DEV), state, drive=drive, return_state=True)
        grads = torch.autograd.grad([out, last], leaves, [d['g'].to(DEV).expand(n, T, 16), d['gs'].to(DEV).expand(n, 16)])
        for k, v in zip(('out', 'last', 'dx', 'dz', 'dstate'), (out, last, *grads)):
            ref, bound = want[k]
            step = 2.0 ** -8 if v.dtype == torch.bfloat16 else U
            for i in {0, n - 1}:
                err = abs(v[i].detach().cpu().double().numpy() - ref)
                over = float((err - (bound + step * (abs(ref) + bound) + 2.0 ** -126)).max())
                assert over <= 0, (k, n, over)


def test_a_token_rounds_once():
    """One token's state is the exact one but for its leak's error and one rounding, half a unit in its last place."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(32)
    n, c, z, decay = 64, 501, -3.0, 512.0
    state, x = torch.randn(n, c, generator=gen), torch.randn(n, c, generator=gen) * 2.0 ** -10
    leak = decay / 4096 / (1 + np.exp(-z))
    want = state.double() * (1 - leak) + x.double()
    half = torch.ldexp(torch.ones(n, c, dtype=torch.float64), torch.frexp(want).exponent - 25)
    got = state.to(DEV)
    slayer.neuron.gated_leak_step(x.to(DEV), torch.full((n, c), z, device=DEV), torch.tensor([decay], device=DEV), got, None)
    err = (got.cpu().double() - want).abs()
    over = float((err - half * (1 + 2.0 ** -20) - (5 + 1.5 * abs(z)) * U * leak * state.double().abs()).max())
    assert over <= 0, over
