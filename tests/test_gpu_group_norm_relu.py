"""Group norm with a ReLU behind it, nothing left out: y is continuous, so it is compared everywhere; where z lies so near to 0 that
rounding decides on which side, the upstream gradient is 0 and either slope is right.  Sizes, formulas and tolerances are those of the
norm's other tests."""
import pytest
import torch

from .test_gpu_group_norm import DEV, SIZES, close, formulas

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,between,c,groups', SIZES)
def test_relu(n, between, c, groups, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(n * 7 + c)
    x = (torch.randn(n, *between, c, generator=gen) * 2 + 3).to(dtype)
    g = torch.randn(n, *between, c, generator=gen).to(dtype)
    w, b = 1 + 0.3 * torch.randn(c, generator=gen), 0.3 * torch.randn(c, generator=gen)
    args = (x.double().reshape(n, -1, c), groups, w.double(), b.double(), 1e-3, 'relu')
    _, tol, z = formulas(*args, g.double().reshape(n, -1, c))
    near = (z.abs() <= 2 * tol[0]).reshape(g.shape)
    assert int(near.sum()) <= 8                                              # a few; the rest is what is tested
    g = g.masked_fill(near, 0)
    ref, tol, _ = formulas(*args, g.double().reshape(n, -1, c))
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = slayer.neuron.norm.group_norm(leaves[0], groups, leaves[1], leaves[2], eps=1e-3, activation='relu')
    got = [y, *torch.autograd.grad(y, leaves, g.to(DEV))]
    for a, r, t, name in zip(got, ref, tol, ('y', 'dx', 'dw', 'db')):
        close(a.reshape(r.shape), r, t, dtype == torch.bfloat16 and name in ('y', 'dx'), name)
