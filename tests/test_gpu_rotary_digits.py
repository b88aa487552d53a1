"""The sines and cosines of rotary positions to float32's digits, of small values too.

Tolerance, relative.  U = 2^-24.  Functions of the angle in float32 that are right to two units in the last place, 4 U, and take in what the
angle's rounding leaves, U, have 5 U and 2^-45 for terms of second order, with 2^-50 for the reference's own angle in float64; functions in
float64 that are rounded once have U."""
import pytest
import torch

from tests.test_gpu_rotary import angles

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24


@pytest.mark.parametrize('inverse', [False, True])
def test_sines_and_cosines(inverse):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(51)
    frequency = torch.cat([slayer.synapse.rotary_frequencies(64), torch.tensor([3.1415, 1.5708, 0.7854, 2.3562], dtype=torch.float64)])
    position = torch.cat([torch.arange(300), torch.randint(0, 1 << 40, (100,), generator=gen)])
    angle = angles(position, frequency)
    f = len(frequency)
    x = torch.zeros(1, 400, 1, 2 * f)
    x[..., :f] = 1                                                        # (1, 0) becomes (cosine, sine)
    x = x.to(DEV).requires_grad_()
    y, _ = slayer.synapse.rotary(x, None, frequency.to(DEV), position[None].to(DEV))
    if inverse:
        y, = torch.autograd.grad(y, x, x.detach())
    got = y.detach()[0, :, 0].cpu().double()
    want = torch.cat([angle.cos(), -angle.sin() if inverse else angle.sin()], -1)
    over = (got - want).abs() - (5 * U * want.abs() + 2.0 ** -45 + 2.0 ** -50)
    assert float(over.max()) <= 0, (float(over.max() / U), float(((got - want) / want / U)[want != 0].abs().max()))


def test_rounded_once():
    """Sine and cosine times the magnitude are float64 and rounded to float32 once, U; the series stop within U / 16 of the sum, the reference's own angle is
    within 2^-50."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(52)
    frequency = slayer.synapse.rotary_frequencies(64, 500000.0)
    position = torch.randint(-(1 << 30), 1 << 30, (500,), generator=gen)
    angle = angles(position, frequency)
    magnitude = 1.1
    x = torch.zeros(1, 500, 1, 64)
    x[..., :32] = 1
    y, _ = slayer.synapse.rotary(x.to(DEV), None, frequency.to(DEV), position[None].to(DEV), magnitude=magnitude)
    got = y[0, :, 0].cpu().double()
    want = float(torch.tensor(magnitude)) * torch.cat([angle.cos(), angle.sin()], -1)
    over = (got - want).abs() - ((1 + 1 / 16) * U * want.abs() + 2.0 ** -49)
    assert float(over.max()) <= 0, float(((got - want) / want / U).abs().max())
