"""Rotary positions against the same turns in float64, of angles from rational arithmetic.

Tolerance.  With U = 2^-24: the part of a turn that is left is rounded to float32, U of at most half a turn, which is pi U of an angle; the
sine and cosine of it are within two units in the last place, 4 U at most, the magnitude's product is U more: (pi + 5) U < 9 U of the
magnitude.  A result is two products and a sum: 9 U + 2 U of magnitude (|x| + |y|), 12 U with the terms of second order.  bfloat16 results:
half a step of theirs besides."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24
getcontext().prec = 60
TURN = 2 * Decimal('3.14159265358979323846264338327950288419716939937510582097494459')


def angles(position, frequency):
    """position * frequency less whole turns, float64 [..., F], of a tensor of integers."""
    f = [Decimal(v) for v in frequency.tolist()]
    left = [[float((Decimal(p) * v) % TURN) for v in f] for p in position.flatten().tolist()]
    return torch.tensor(left, dtype=torch.float64).reshape(*position.shape, len(f))


def turned(x, angle, layout, magnitude, sign=1):
    """(value, magnitudes) of x [..., H, D] turned by angle [..., F], both float64."""
    x, f = x.double(), angle.shape[-1]
    c, s = (magnitude * angle.cos())[..., None, :], (sign * magnitude * angle.sin())[..., None, :]
    a, b = (x[..., :f], x[..., f:2 * f]) if layout == 'halves' else (x[..., 0:2 * f:2], x[..., 1:2 * f:2])
    p, q, size = c * a - s * b, c * b + s * a, magnitude * (a.abs() + b.abs())
    y, m = ((torch.cat([p, q], -1), torch.cat([size, size], -1)) if layout == 'halves'
            else (torch.stack([p, q], -1).flatten(-2), torch.stack([size, size], -1).flatten(-2)))
    return torch.cat([y, x[..., 2 * f:]], -1), torch.cat([m, torch.zeros_like(x[..., 2 * f:])], -1)


def hold(got, x, angle, layout, magnitude, sign=1):
    want, size = turned(x, angle, layout, magnitude, sign)
    assert got.shape == want.shape and got.is_contiguous() and got.dtype == x.dtype
    err = (got.detach().cpu().double() - want).abs()
    bound = 12 * U * size + (2.0 ** -8 * (want.abs() + 12 * U * size) if got.dtype == torch.bfloat16 else 0)
    f = angle.shape[-1]
    assert not (err > bound + 2.0 ** -126).any(), float((err - bound).max())
    assert torch.equal(got[..., 2 * f:].cpu(), x[..., 2 * f:])                       # copied, to the bit


SHAPES = [(1, 1, 1, 1, 1, 0), (1, 2, 1, 1, 2, 1), (2, 3, 2, 1, 5, 2), (2, 7, 1, 3, 16, 8), (1, 70, 3, 3, 24, 5), (3, 33, 4, 2, 31, 15),
          (2, 65, 2, 2, 64, 32), (1, 130, 8, 8, 80, 24), (2, 9, 5, 5, 128, 63), (1, 5, 2, 2, 4096, 2048), (1, 40, 16, 16, 17, 8),
          (2, 20, 1, 1, 300, 7), (1, 300, 0, 1, 12, 6), (1, 3, 40, 7, 9, 4), (4, 600, 1, 1, 10, 5)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('layout', ['halves', 'pairs'])
@pytest.mark.parametrize('n,t,hq,hk,d,f', SHAPES)
def test_results_and_gradients(n, t, hq, hk, d, f, layout, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(d * 100 + t)
    q, k, gq, gk = (torch.randn(n, t, h, d, generator=gen).to(dtype) for h in (hq, hk, hq, hk))
    frequency = slayer.synapse.rotary_frequencies(2 * f)
    kinds = {'none': None, 'first': torch.randint(-500, 1000000, (n,), generator=gen),
             'each': torch.randint(0, 3000, (n, t), generator=gen).int()}
    for kind, position in kinds.items():
        at = torch.arange(t).expand(n, t) if position is None else position
        at = at[:, None] + torch.arange(t) if at.dim() == 1 else at
        angle = angles(at, frequency)
        a, b = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
        y, z = slayer.synapse.rotary(a, b, frequency.to(DEV), None if position is None else position.to(DEV), layout, 1.25)
        hold(y, q, angle, layout, 1.25)
        hold(z, k, angle, layout, 1.25)
        dq, dk = torch.autograd.grad([y, z], [a, b], [gq.to(DEV), gk.to(DEV)])
        hold(dq, gq, angle, layout, 1.25, -1)
        hold(dk, gk, angle, layout, 1.25, -1)


def test_far_positions():
    """Where a float64 product has no digits of the turn left."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(3)
    frequency = torch.cat([slayer.synapse.rotary_frequencies(16), torch.tensor([3.0, 1e-7, 2.5e-9], dtype=torch.float64)])
    position = torch.tensor([[0, 1, -1, 2 ** 31 - 1, 2 ** 31, -2 ** 40, 10 ** 15 + 1, 2 ** 53]])
    x = torch.randn(1, 8, 2, 22, generator=gen)
    y, none = slayer.synapse.rotary(x.to(DEV), None, frequency.to(DEV), position.to(DEV))
    assert none is None
    hold(y, x, angles(position, frequency), 'halves', 1.0)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strides_and_single_tokens(dtype):
    """Parts of one projection, turned axes, broadcast heads, odd addresses; a token a sample is that token of the sample."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(4)
    frequency = slayer.synapse.rotary_frequencies(14, 500.0)
    w = torch.randn(3, 21, 3, 4, 19, generator=gen).to(dtype)
    at = torch.randint(0, 90000, (3,), generator=gen)
    angle = angles(at[:, None] + torch.arange(21), frequency)
    projection, f, p = w.to(DEV), frequency.to(DEV), at.to(DEV)
    q, k, _ = projection.unbind(2)
    y, z = slayer.synapse.rotary(q, k, f, p)
    hold(y, w[:, :, 0], angle, 'halves', 1.0)
    hold(z, w[:, :, 1], angle, 'halves', 1.0)
    flat = torch.zeros(w[:, :, 0].numel() + 1, dtype=dtype, device=DEV)
    flat[1:] = q.flatten()
    for same in (q.transpose(1, 3).contiguous().transpose(1, 3), q.transpose(0, 2).contiguous().transpose(0, 2), flat[1:].view(q.shape)):
        assert torch.equal(slayer.synapse.rotary(same, None, f, p)[0], y)
    shared = k[:, :, :1].expand(-1, -1, 4, -1)
    assert torch.equal(slayer.synapse.rotary(q, shared, f, p)[1], z[:, :, :1].expand(-1, -1, 4, -1))
    for t in (0, 20):
        one = slayer.synapse.rotary(q[:, t], k[:, t], f, p + t)
        assert torch.equal(one[0], y[:, t]) and torch.equal(one[1], z[:, t])
    start = slayer.synapse.rotary(q[:, 0], k[:, 0], f)
    assert torch.equal(start[0], q[:, 0]) and torch.equal(start[1], k[:, 0])


def test_distance_alone_counts():
    """The product of a query and a key depends on how far apart they are, not on where."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(5)
    q, k = torch.randn(1, 1, 1, 64, generator=gen).to(DEV), torch.randn(1, 1, 1, 64, generator=gen).to(DEV)
    f = slayer.synapse.rotary_frequencies(64, device=DEV)
    size = float((q.abs() * k.abs()).sum())
    ref = None
    for at in (0, 17, 123456, 10 ** 9):
        a = slayer.synapse.rotary(q, None, f, torch.tensor([at + 40], device=DEV))[0]
        b = slayer.synapse.rotary(k, None, f, torch.tensor([at], device=DEV))[0]
        dot = float((a.double() * b.double()).sum())
        ref = dot if ref is None else ref
        assert abs(dot - ref) <= 2 * 2 * 24 * U * 2 * size


def test_second_derivatives():
    """A turn is linear: the gradient's gradient is the turn again."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(6)
    q = torch.randn(2, 5, 2, 8, generator=gen).to(DEV).requires_grad_()
    g = torch.randn(2, 5, 2, 8, generator=gen).to(DEV).requires_grad_()
    f = slayer.synapse.rotary_frequencies(8, device=DEV)
    y, _ = slayer.synapse.rotary(q, None, f)
    dq, = torch.autograd.grad(y, q, g, create_graph=True)
    v = torch.randn(2, 5, 2, 8, generator=gen).to(DEV)
    dg, = torch.autograd.grad(dq, g, v)
    assert torch.equal(dg, slayer.synapse.rotary(v, None, f)[0])


def test_one_of_the_gradients():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(7)
    q, k = torch.randn(2, 5, 2, 8, generator=gen).to(DEV), torch.randn(2, 5, 3, 8, generator=gen).to(DEV)
    f = slayer.synapse.rotary_frequencies(8, device=DEV)
    for i in range(2):
        a, b = q.clone().requires_grad_(i == 0), k.clone().requires_grad_(i == 1)
        out = slayer.synapse.rotary(a, b, f)
        g = torch.randn(out[i].shape, generator=gen).to(DEV)
        got, = torch.autograd.grad(out[i], (a, b)[i], g)
        hold(got, g.cpu(), angles(torch.arange(5).expand(2, 5), f.cpu()), 'halves', 1.0, -1)


def test_nothing_to_turn():
    import lava_dl_amd.slayer as slayer
    f = slayer.synapse.rotary_frequencies(8, device=DEV)
    for shape in ((0, 3, 2, 8), (3, 0, 2, 8), (3, 2, 0, 8), (0, 2, 8)):
        q = torch.zeros(shape, device=DEV, requires_grad=True)
        y, z = slayer.synapse.rotary(q, q, f)
        assert y.shape == z.shape == q.shape
        assert torch.autograd.grad([y, z], q, [y, z])[0].shape == q.shape


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_values_that_are_not_finite_stay_in_their_pair(bad):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(8)
    f = slayer.synapse.rotary_frequencies(12, device=DEV)
    for layout, pair in (('halves', (3, 9)), ('pairs', (6, 7))):
        x = torch.randn(1, 4, 2, 15, generator=gen).to(DEV)
        clean = slayer.synapse.rotary(x, None, f, layout=layout)[0]
        x[0, 2, 1, pair[0]] = bad
        got = slayer.synapse.rotary(x, None, f, layout=layout)[0]
        hit = torch.zeros_like(x, dtype=torch.bool)
        hit[0, 2, 1, list(pair)] = True
        assert torch.equal(torch.where(hit, 0, got), torch.where(hit, 0, clean)) and not torch.isfinite(got[hit]).any()


def test_gradients_are_differences():
    """A turn is linear, so a difference of results is the turn of the difference, and its product with any g is that of the gradient for g with the
    difference: within 12 * 2^-24 of the magnitudes on either side, and 2^-24 of the results that are subtracted."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(9)
    f = slayer.synapse.rotary_frequencies(24, device=DEV)
    for layout in ('halves', 'pairs'):
        x, v, g = (torch.randn(2, 30, 3, 29, generator=gen).to(DEV) for _ in range(3))
        leaf = x.clone().requires_grad_()
        y = slayer.synapse.rotary(leaf, None, f, layout=layout)[0]
        grad, = torch.autograd.grad(y, leaf, g)
        moved = slayer.synapse.rotary(x + v, None, f, layout=layout)[0]
        difference = ((moved.double() - y.detach().double()) * g).sum()
        step = (x + v).double() - x.double()
        size = ((x.abs() + (x + v).abs()).double().sum(-1) * g.abs().double().amax(-1)).sum() * 2
        assert float((difference - (grad.double() * step).sum()).abs()) <= 2 * 13 * U * float(size)
