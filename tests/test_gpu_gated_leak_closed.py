"""Gates that are as good as closed, float32: leaks far below 1 to float32's digits.

Tolerance, relative.  U = 2^-24.  A leak is a sigmoid that is 6 U off times a decay over 4096, U: 7 U.  What one token adds to a state of zeros is the
leak times the input, 8 U; the gate's gradient g x leak (1 - open) four roundings more with that of 1 - open, 12 U; the input's, leak g, 8 U; the decay's,
g x open / 4096, 10 U."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24


def test_closed_gates():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(41)
    z = torch.linspace(-60, 0, 4801)
    x, g = torch.randn(2, 4801, generator=gen)
    decay = 4096 * torch.rand(4801, generator=gen)
    open_ = torch.special.expit(z.double())
    leak = decay.double() / 4096 * open_
    want = {'out': (leak * x, 8), 'dx': (leak * g, 8), 'dz': (g.double() * x * leak * (1 - open_), 12), 'ddecay': (g.double() * x * open_ / 4096, 10)}
    leaves = [v.to(DEV).requires_grad_() for v in (x.reshape(1, 1, -1), z.reshape(1, 1, -1), decay)]
    out = slayer.neuron.gated_leak(*leaves, drive='gain')
    got = dict(zip(('out', 'dx', 'dz', 'ddecay'), (out, *torch.autograd.grad(out, leaves, g.to(DEV).reshape(1, 1, -1)))))
    got['step'] = slayer.neuron.gated_leak_step(*(v.to(DEV)[None] for v in (x, z)), decay.to(DEV), torch.zeros(1, 4801, device=DEV))
    want['step'] = want['out']
    for k, (ref, bound) in want.items():
        off = ((got[k].detach().flatten().cpu().double() - ref).abs() / ref.abs() / U)[ref != 0]
        assert float(off.max()) <= bound, (k, float(off.max()))
