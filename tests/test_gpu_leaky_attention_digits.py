"""Leaky attention on whole numbers that float32 holds exactly: with a decay of 0 and a scale of 1 every product and every partial sum is
a whole number below 2^24, so float32 arithmetic in any order has no error and a result has one right value: the exact number, rounded
once to the type of the tensors.  Scores (or, in the gradients' passes, the products of values and gradients) reach beyond 2^17 and need
more than the sixteen bits that two bfloat16 numbers hold."""
import pytest
import torch

from .test_gpu_leaky_attention import SIZES, close, decays, factor, inputs, recurrence

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


@pytest.mark.parametrize('n,t,h,k,v,lengths', SIZES)
def test_decays_of_bfloat16_tensors_have_float32_gradients(n, t, h, k, v, lengths):
    """Scores, states and their derivatives enter products in three parts, within 2^-24: the bound is that of float32 tensors and
    2^-24 for each of the three products."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(t * 1000 + k + v)
    q, key, value, first = inputs(gen, n, t, h, k, v, torch.bfloat16, True)
    g, g_last = torch.randn(n, t, h, v, generator=gen).bfloat16(), torch.randn(n, h, k, v, generator=gen)
    ends = [t] * n if lengths is None else lengths

    def oracle(fix):
        a = (1 - decays(h).double() / 4096).requires_grad_()
        out = recurrence(*(fix(x.double()) for x in (q, key, value)), a, fix(first.double()), ends, 0.3)
        return torch.autograd.grad(out, a, [fix(g.double()), fix(g_last.double())])[0]
    decay = decays(h).to(DEV).requires_grad_()
    out = slayer.synapse.leaky_attention(*(x.to(DEV) for x in (q, key, value)), decay, state=first.to(DEV), scale=0.3, return_state=True,
                                         lengths=None if lengths is None else torch.tensor(lengths, device=DEV))
    got, = torch.autograd.grad(out, decay, [g.to(DEV), g_last.to(DEV)])
    close(got, oracle(lambda x: x) / -4096, oracle(torch.abs) / 4096, factor(k, v, t) + 3 * 2.0 ** -24, 'decay')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('large', ['scores', 'state'])
def test_the_gradient_of_the_decays_is_exact_for_whole_numbers(large, dtype):
    """The derivative of out[i] with respect to a is, at a = 1, sum over j < i of (i - j) (q[i] . k[j]) v[j] + (i + 1) q[i] S: whole
    numbers again, which need up to eighteen or twenty bits on their way into products.  Sums over samples are float64, 1 / 4096 is a power of two."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(3)
    n, t, h, k, v = 3, 9 if large == 'scores' else 5, 2, 16, 16

    def few(*shape):
        return torch.randint(-1, 2, shape, generator=gen).double() * (torch.rand(shape, generator=gen) < (0.4 if large == 'scores' else 0.25))
    q, key = few(n, t, h, k), few(n, t, h, k)
    if large == 'scores':
        value, g = (torch.randint(50, 101, (n, t, h, v), generator=gen).double() for _ in range(2))
        first = torch.zeros(n, h, k, v).double()
    else:
        value, g = few(n, t, h, v), few(n, t, h, v)
        first = torch.randint(1 << 16, 1 << 18, (n, h, k, v), generator=gen).double()

    def places(fix):                                                          # [n, h, t]: what each token adds to the slope
        Q, K, V, G, S = (fix(x) for x in (q.transpose(1, 2), key.transpose(1, 2), value.transpose(1, 2), g.transpose(1, 2), first))
        i = torch.arange(t, dtype=torch.float64)
        back = (i[:, None] - i).clamp(min=0)
        return ((((Q @ K.transpose(-1, -2)) * back) @ V + (i[:, None] + 1) * (Q @ S)) * G).sum(-1)
    assert float(places(torch.abs).max()) < 2 ** 24
    want = (places(lambda x: x).sum((0, 2)) / -4096).float()
    decay = torch.zeros(h, device=DEV, requires_grad=True)
    out = slayer.synapse.leaky_attention(*(x.to(DEV, dtype) for x in (q, key, value)), decay, state=first.float().to(DEV))
    got, = torch.autograd.grad(out, decay, g.to(DEV, dtype))
    assert torch.equal(got.cpu(), want), (got.tolist(), want.tolist())
