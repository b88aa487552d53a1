"""Group norm over images whose pixels are not alike: a first pixel, a border or a single value far from the others.

Tolerance.  u = 2^-24.  With shapes cut as they are here a value's square passes at most 160 additions on its way into the variance (8
pixels of a thread, 128 threads, 16 sums of a join, a tree of 8) and so does its value on the way into the mean; all terms of the
variance are at least 0.  With two roundings a term the scale is within 160 u of itself (half of 320), the mean within 320 u of the mean of
magnitudes, and y = (x - mean) * scale within 160 u |y| + 320 u mean|x| scale + 8 u |y|; bfloat16 adds its rounding, 2^-8 |y|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, DEV = 2.0 ** -24, 'cuda:0'


def image(kind, n, pixels, c, gen):
    x = torch.randn(n, pixels, c, generator=gen)
    if kind == 'first pixel of 300':
        x[:, 0] = 300
    elif kind == 'first pixel of 1000':
        x[:, 0] = 1000
    elif kind == 'zero corner':
        x += 500
        x[:, :3] = 0
    elif kind == 'last pixel of -1000':
        x[:, -1] = -1000
    elif kind == 'one channel':
        x[:, 0, 3] = 3000
    return x


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,pixels,c,groups', [(1, 65536, 16, 1), (2, 4096, 64, 4), (3, 1021, 30, 5), (1, 2, 8, 2), (40, 777, 512, 32)])
@pytest.mark.parametrize('kind', ['first pixel of 300', 'first pixel of 1000', 'zero corner', 'last pixel of -1000', 'one channel'])
def test_no_pixel_costs_the_variance_digits(kind, n, pixels, c, groups, dtype):
    import lava_dl_amd.slayer as slayer
    x = image(kind, n, pixels, c, torch.Generator().manual_seed(pixels)).to(dtype)
    y = slayer.neuron.norm.group_norm(x.to(DEV), groups).cpu().double()
    g = x.double().reshape(n, pixels, groups, c // groups)
    mean = g.mean((1, 3), keepdim=True)
    scale = ((g - mean).square().mean((1, 3), keepdim=True) + 1e-5) ** -0.5
    ref = (g - mean) * scale
    tol = 168 * U * ref.abs() + 320 * U * g.abs().mean((1, 3), keepdim=True) * scale + (2.0 ** -8 * 1.01 * ref.abs() if dtype == torch.bfloat16 else 0)
    off = (y.reshape(g.shape) - ref).abs()                                    # (an image of zeros: both are 0)
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize('value', [2.5, 1000.1, -3e-5, 1e30])
@pytest.mark.parametrize('shape,groups', [((3, 16), 4), ((2, 9, 16), 4), ((1, 70000, 8), 2), ((5, 3001, 96), 3)])
def test_constant_groups_are_exactly_zero(shape, groups, value):
    import lava_dl_amd.slayer as slayer
    x = torch.full(shape, value, device=DEV)
    if len(shape) == 3:
        assert not slayer.neuron.norm.group_norm(x, groups).any()
    else:                                                                     # a row's mean is its sum by its width, rounded: 2 u |x|
        assert float(slayer.neuron.norm.group_norm(x, groups).abs().max()) <= 2 * U * abs(value) * 1e-5 ** -0.5
