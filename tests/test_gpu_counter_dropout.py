"""Dropout from a counter on the GPU against the generator in numpy: every bit.  (The published known answers of the generator pin the
numpy form itself: tests/test_token_mixing_arguments.py.)"""
import pytest
import torch

from .util_philox import keep

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def reference(x, p, seed, offset, per_neuron):
    limit = round(p * 65536)
    scale = torch.tensor(65536 / (65536 - limit) if limit < 65536 else 0.0, dtype=torch.float32)
    count = x.numel() // x.shape[-1] if per_neuron else x.numel()
    mask = torch.from_numpy(keep(count, seed, offset, limit))
    mask = mask.reshape(x.shape[:-1] + (1,) if per_neuron else x.shape)
    return torch.where(mask, x.float() * scale, 0).to(x.dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(1,), (7,), (8,), (3, 5), (17, 64), (2, 3, 301), (5, 1), (4, 2048), (1000, 3), (2, 4, 5, 6, 50)])
@pytest.mark.parametrize('per_neuron', [False, True])
def test_every_decision(shape, per_neuron, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(len(shape))
    x = torch.randn(shape, generator=gen).to(dtype)
    for p, seed, offset in ((0.3, 1, 0), (0.999, (1 << 64) - 1, (1 << 64) - 1), (1e-4, 12345678901234567, 1 << 40)):
        y = slayer.neuron.counter_dropout(x.to(DEV), p, seed, offset, per_neuron=per_neuron)
        assert y.dtype == dtype and torch.equal(y.cpu(), reference(x, p, seed, offset, per_neuron))


@pytest.mark.parametrize('per_neuron', [False, True])
def test_gradient_passes_where_the_value_did(per_neuron):
    import lava_dl_amd.slayer as slayer
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(30, 77, device=DEV).to(dtype).requires_grad_()
        g = torch.randn(30, 77, device=DEV).to(dtype)
        y = slayer.neuron.counter_dropout(x, 0.4, 9, 3, per_neuron=per_neuron)
        grad, = torch.autograd.grad(y, x, g)
        assert torch.equal(grad.cpu(), reference(g.cpu(), 0.4, 9, 3, per_neuron))
        assert torch.equal(y.detach().cpu(), reference(x.detach().cpu(), 0.4, 9, 3, per_neuron))
    x = torch.randn(6, 8, device=DEV, requires_grad=True)                     # linear: a difference of any step is the gradient
    f = lambda t: slayer.neuron.counter_dropout(t, 0.5, 2, 2)                 # noqa: E731
    g = torch.ones_like(x).requires_grad_()
    first, = torch.autograd.grad(f(x), x, g, create_graph=True)
    assert torch.equal(first, f(torch.ones_like(x)))
    assert torch.equal(torch.autograd.grad(first.sum(), g)[0], f(torch.ones_like(x)))


def test_extremes_and_values_that_are_not_finite():
    import lava_dl_amd.slayer as slayer
    x = torch.randn(50, 40, device=DEV)
    assert torch.equal(slayer.neuron.counter_dropout(x, 0.0, 1), x)
    assert not slayer.neuron.counter_dropout(x, 1.0, 1).any()
    for per_neuron in (False, True):
        dropped = reference(torch.ones(50, 40), 0.5, 1, 0, per_neuron) == 0
        for bad in (float('nan'), float('inf')):
            y = slayer.neuron.counter_dropout(x.cpu().masked_fill(dropped, bad).to(DEV), 0.5, 1, per_neuron=per_neuron)
            assert torch.equal(y.cpu(), reference(x.cpu(), 0.5, 1, 0, per_neuron))


def test_layouts_and_streams():
    import lava_dl_amd.slayer as slayer
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(12, 33, 20, device=DEV).to(dtype)
        for per_neuron in (False, True):
            ref = slayer.neuron.counter_dropout(x, 0.2, 4, 5, per_neuron=per_neuron)
            odd = torch.empty(x.numel() + 1, device=DEV, dtype=dtype)[1:].view(x.shape)
            odd.copy_(x)
            turned = x.transpose(0, 2).contiguous().transpose(0, 2)
            for y in (odd, turned):
                assert torch.equal(slayer.neuron.counter_dropout(y, 0.2, 4, 5, per_neuron=per_neuron), ref)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = slayer.neuron.counter_dropout(x, 0.2, 4, 5, per_neuron=per_neuron)
            side.synchronize()
            assert torch.equal(other, ref)


def test_share_of_what_is_dropped():
    """2^20 decisions of probability p: within six standard deviations."""
    import lava_dl_amd.slayer as slayer
    x = torch.ones(1 << 20, device=DEV)
    for p in (0.1, 0.5, 0.9):
        share = float((slayer.neuron.counter_dropout(x, p, 77, 1) == 0).double().mean())
        assert abs(share - p) < 6 * (p * (1 - p) / (1 << 20)) ** 0.5 + 2.0 ** -17
    a, b = (slayer.neuron.counter_dropout(x, 0.5, 77, o) == 0 for o in (1, 2))
    assert abs(float((a == b).double().mean()) - 0.5) < 6 * 0.5 / (1 << 10)   # two offsets agree by chance


def test_more_elements_than_32_bits_count():
    import lava_dl_amd.slayer as slayer
    import numpy as np
    n = (1 << 32) + 64
    x = torch.ones(n, device=DEV, dtype=torch.bfloat16)
    y = slayer.neuron.counter_dropout(x, 0.5, 3, 4)
    first = (1 << 32) // 8                                                    # the block of the generator there
    want = keep(64, 3, 4, 32768, first=first)
    assert np.array_equal((y[-64:] != 0).cpu().numpy(), want)
    z = slayer.neuron.counter_dropout(x.view(-1, 1), 0.5, 3, 4, per_neuron=True)
    assert np.array_equal((z[-64:, 0] != 0).cpu().numpy(), want)


def test_module():
    import lava_dl_amd.slayer as slayer
    x = torch.randn(5, 6, 30, device=DEV)
    drop = slayer.neuron.CounterDropout(0.3, seed=8, per_neuron=True)
    first, second = drop(x), drop(x)
    assert torch.equal(first, slayer.neuron.counter_dropout(x, 0.3, 8, 0, per_neuron=True))
    assert torch.equal(second, slayer.neuron.counter_dropout(x, 0.3, 8, 1, per_neuron=True)) and drop.offset == 2
    drop.offset = 0
    assert torch.equal(drop(x), first)
    assert drop.eval()(x) is x
    empty = torch.empty(3, 0, device=DEV)
    for per_neuron in (False, True):
        assert slayer.neuron.counter_dropout(empty, 0.5, 1, per_neuron=per_neuron).shape == (3, 0)


def test_refusals():
    import lava_dl_amd.slayer as slayer
    x = torch.zeros(4, device=DEV)
    for p, seed, offset in ((-0.1, 0, 0), (1.1, 0, 0), (float('nan'), 0, 0), (0.5, -1, 0), (0.5, 0, 1 << 64)):
        with pytest.raises(ValueError):
            slayer.neuron.counter_dropout(x, p, seed, offset)
    for y in (x.half(), x.cpu(), x.int()):
        with pytest.raises(RuntimeError):
            slayer.neuron.counter_dropout(y, 0.5, 1)
    with pytest.raises(RuntimeError):
        slayer.neuron.counter_dropout(x[0], 0.5, 1, per_neuron=True)
    with pytest.raises(ValueError):
        slayer.neuron.CounterDropout(2.0)
