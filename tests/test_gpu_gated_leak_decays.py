"""The gated leak's gradient with respect to the decays where many terms meet in one: long walks, many samples, one decay for all.

Tolerance.  U = 2^-24.  A term is what the derivative with respect to a leak is, times how far its gate is open.  A lane adds up to 16 of them in
float32, tiles are added in float64; eight waves, and channels where they share a decay, are added in float32, at most 8 + 6 additions; rows in float64,
64 shares of them in 6 additions: 16 + 14 + 6 roundings and three conversions, under 40 U of the terms' magnitudes, however many there are."""
import pytest
import torch

from tests.test_gpu_gated_leak import DRIVES, exact, make, run

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24


@pytest.mark.parametrize('drive', DRIVES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,c,one', [(300, 600, 1, False), (70, 300, 130, False), (300, 600, 1, True), (200, 130, 67, True), (1030, 20, 3, False),
                                       (3, 2300, 5, True)])
def test_every_sample_counts(n, t, c, one, dtype, drive):
    """All samples and channels against float64: a workgroup that walks several tiles of a chain, and one for each tile."""
    gen = torch.Generator().manual_seed(n + t)
    d = make(gen, n, t, c, dtype)
    if one:
        d['decay'] = torch.tensor([300.0])
    want, bound = exact(dict(d, decay=d['decay'].expand(c)), drive)['ddecay']
    if one:
        want, bound = want.sum()[None], bound.sum()[None]
    got = run(d, drive)['ddecay'].cpu().double()
    over = float(((got - want).abs() - bound - U * want.abs()).max())
    assert over <= 0, (over, got, want, bound)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,c,one', [(200, 131077, 1, False), (200, 131077, 1, True), (1, 1048576 + 77, 1, False), (131077, 24, 1, False),
                                       (131077, 24, 2, True)])
def test_terms_that_are_alike(n, t, c, one, dtype):
    """Open gates and decays of 4096, a leak of 1: each token's state is its input and each derivative its own, to the bit.  The terms are -x g
    and no two of them round differently."""
    import lava_dl_amd.slayer as slayer
    x, g = (torch.tensor(v, dtype=dtype) for v in (1.2345679, 0.7654321))
    decay = torch.full((1 if one else c,), 4096.0, device=DEV, requires_grad=True)
    out, last = slayer.neuron.gated_leak(x.to(DEV).expand(n, t, c), torch.full((), 100.0, dtype=dtype, device=DEV).expand(n, t, c), decay,
                                         x.float().to(DEV).expand(n, c), drive=None, return_state=True)
    assert torch.equal(last, x.float().to(DEV).expand(n, c))
    got, = torch.autograd.grad(out, decay, g.to(DEV).expand(n, t, c))
    want = float(-x.double() * g.double() / 4096) * n * t * (c if one else 1)
    over = float((got.cpu().double() - want).abs().max()) / (U * abs(want))
    assert over <= 41, over                                             # the term's own rounding besides
