"""Leaky attention on whole numbers that float32 holds exactly: with a decay of 0 and a scale of 1 every product and every partial sum is
a whole number below 2^24, so float32 arithmetic in any order has no error and a result has one right value: the exact number, rounded
once to the type of the tensors.  Scores (or, in the gradients' passes, the products of values and gradients) reach beyond 2^17 and need
more than the sixteen bits that two bfloat16 numbers hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def exact(q, k, v, g):
    """(out, gradients of q, k, v) for a = 1, from the masked products."""
    mask = torch.tril(torch.ones(q.shape[1], q.shape[1], dtype=q.dtype))
    q, k, v, g = (x.transpose(1, 2) for x in (q, k, v, g))
    scores, products = (q @ k.transpose(-1, -2)) * mask, (g @ v.transpose(-1, -2)) * mask
    return [x.transpose(1, 2) for x in (scores @ v, products @ k, products.transpose(-1, -2) @ q, scores.transpose(-1, -2) @ g)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,h,k,v', [(2, 130, 2, 64, 64), (40, 100, 2, 64, 64), (40, 70, 2, 96, 48), (40, 70, 2, 48, 96), (1, 128, 1, 128, 128)])
@pytest.mark.parametrize('large', ['queries and keys', 'values and gradients'])
def test_whole_numbers_are_exact(n, t, h, k, v, large, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(t + k)
    wide = (k if large.startswith('q') else v)
    top = int((2 ** 24 / (0.45 * t * wide)) ** 0.5)               # a sum of t scores of (3/4 top)^2 wide, three quarters of them: below 2^24

    def numbers(size, big):
        if big:
            return torch.randint(top // 2, top + 1, (n, t, h, size), generator=gen).double()
        return torch.randint(-1, 2, (n, t, h, size), generator=gen).double() * (torch.rand(n, t, h, size, generator=gen) < 0.75)
    q, key = (numbers(k, large.startswith('q')) for _ in range(2))
    value, g = (numbers(v, large.startswith('v')) for _ in range(2))
    want = exact(q, key, value, g)
    assert max(float(x.max()) for x in exact(q.abs(), key.abs(), value.abs(), g.abs())) < 2 ** 24
    leaves = [x.to(DEV, dtype).requires_grad_() for x in (q, key, value)]
    assert all(torch.equal(x.detach().cpu().double(), y) for x, y in zip(leaves, (q, key, value)))
    out = slayer.synapse.leaky_attention(*leaves, torch.zeros(h, device=DEV))
    got = [out, *torch.autograd.grad(out, leaves, g.to(DEV, dtype))]
    for name, x, y in zip(('out', 'query', 'key', 'value'), got, want):
        x, y = x.detach().cpu(), y.to(dtype)
        assert torch.equal(x, y), f'{name}: {int((x != y).sum())} of {x.numel()} differ'


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('t', [64, 200, 1300])
def test_results_are_the_same_with_and_without_the_last_state(t, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(t)
    q, k, v = (torch.randn(2, t, 3, 48, generator=gen).to(DEV, dtype) for _ in range(3))
    decay = torch.tensor([3.0, 77.0, 900.0], device=DEV)
    both = slayer.synapse.leaky_attention(q, k, v, decay, return_state=True)[0]
    assert torch.equal(both, slayer.synapse.leaky_attention(q, k, v, decay))
