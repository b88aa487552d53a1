"""The activation behind the norm by itself: zeros have a mean of 0, so z is the bias, exactly, and with one sample the bias' gradient is
the upstream gradient times the activation's slope.

Tolerance.  u = 2^-24.  SiLU in float32: exp within a unit in the last place (2 u), the sum, the division and the product round once
each: 6 u with what is of second order.  Its slope s (1 + z (1 - s)) has s within 4 u, so 1 - s within 4 u s + u, and three more
roundings.  In bfloat16 the result is rounded to 2^-8 of itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, DEV = 2.0 ** -24, 'cuda:0'


@pytest.mark.parametrize('between', [(), (2,)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_silu(between, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(1)
    z = torch.cat((torch.linspace(-60, 60, 1500), torch.randn(500, generator=gen) * 3))
    g = torch.randn(2000, generator=gen).to(dtype)
    x = torch.zeros(1, *between, 2000, device=DEV, dtype=dtype)
    bias = z.to(DEV).requires_grad_()
    y = slayer.neuron.norm.group_norm(x, 4, None, bias, activation='silu')
    up = torch.zeros_like(y)
    up[(0,) * (y.dim() - 1)] = g.to(DEV)
    grad, = torch.autograd.grad(y, bias, up)
    z, g = z.double(), g.double()
    s = torch.sigmoid(z)
    assert torch.equal(y, y[(slice(None),) + (slice(0, 1),) * len(between)].expand_as(y))
    off = (y.detach().cpu().double().reshape(-1, 2000)[0] - z * s).abs()
    if dtype == torch.bfloat16:
        assert bool((off <= (2.0 ** -8 * 1.01 + (4 + 1.5 * z.abs()) * U) * (z * s).abs()).all())
        return
    assert bool((off <= 6 * U * (z * s).abs()).all()), float((off / (z * s).abs()).max() / U)
    slope = s * (1 + z * (1 - s))
    tol = 6 * U * slope.abs() + s * (z.abs() * (4 * s + 1) * U + 3 * U * (1 + z.abs() * (1 - s)))
    off = (grad.cpu().double() / g - slope).abs() - 2 * U * slope.abs()                    # ... times the upstream gradient
    assert bool((off <= tol).all()), float((off / tol).max())
