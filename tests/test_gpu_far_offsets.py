"""Gated leak, rotary positions and the norms around a block on tensors whose elements lie beyond 2^31 and 2^32 bytes: the last samples
and rows are, to the bit, those of a call on them alone (of the same form: sizes are chosen so that a workgroup walks its chain in both)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _memory():
    if torch.cuda.is_available() and torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of free device memory')
    yield
    torch.cuda.empty_cache()


def big(gen, *shape):
    x = torch.empty(shape, dtype=BF16, device=DEV)
    return x.normal_(generator=gen)


def test_gated_leak():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, z = big(gen, 4200, 200, 2600), big(gen, 4200, 200, 2600)             # 2.18e9 elements
    decay = torch.full((2600,), 700.0, device=DEV, requires_grad=True)
    out, last = slayer.neuron.gated_leak(x.requires_grad_(), z, decay, return_state=True)
    dx, = torch.autograd.grad(out, x, x.detach(), retain_graph=False)
    tail = [t.detach()[-12:].clone() for t in (x, z)]                       # 12 samples of 21 strips: as many chains as make a walk
    want, end = slayer.neuron.gated_leak(tail[0].requires_grad_(), tail[1], decay, return_state=True)
    dw, = torch.autograd.grad(want, tail[0], tail[0].detach())
    assert torch.equal(out[-12:], want) and torch.equal(last[-12:], end) and torch.equal(dx[-12:], dw)


def test_gated_leak_far_strides():
    """Samples more than 2^32 elements apart."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator(device=DEV).manual_seed(2)
    buffer = torch.empty((1 << 32) + 70000, dtype=BF16, device=DEV)
    x = buffer.as_strided((2, 300, 100), ((1 << 32) + 7, 130, 1))
    x.copy_(torch.randn(2, 300, 100, device=DEV, generator=gen))
    decay = torch.full((1,), 700.0, device=DEV)
    assert torch.equal(slayer.neuron.gated_leak(x, x, decay), slayer.neuron.gated_leak(x.contiguous(), x.contiguous(), decay))
    q = x.view(2, 300, 5, 20)
    f = slayer.synapse.rotary_frequencies(20, device=DEV)
    assert torch.equal(slayer.synapse.rotary(q, None, f)[0], slayer.synapse.rotary(q.contiguous(), None, f)[0])


def test_rotary():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator(device=DEV).manual_seed(3)
    q = big(gen, 3, 700000, 8, 130)                                         # 2.18e9 elements
    f = slayer.synapse.rotary_frequencies(128, device=DEV)
    out, _ = slayer.synapse.rotary(q, None, f)
    tail, _ = slayer.synapse.rotary(q[-1:, -5:], None, f, torch.tensor([699995], device=DEV))
    assert torch.equal(out[-1:, -5:], tail)


def test_residual_norm():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator(device=DEV).manual_seed(4)
    x = big(gen, 531000, 4100)                                              # 2.18e9 elements
    w = torch.randn(4100, device=DEV)
    y, total = slayer.neuron.norm.residual_norm(x.requires_grad_(), None, w, w, x.detach(), 0.5, 'silu')
    dx, = torch.autograd.grad([y, total], x, [x.detach(), x.detach()])
    tail = x.detach()[-3:].clone().requires_grad_()
    a, b = slayer.neuron.norm.residual_norm(tail, None, w, w, tail.detach(), 0.5, 'silu')
    da, = torch.autograd.grad([a, b], tail, [tail.detach(), tail.detach()])
    assert torch.equal(y[-3:], a) and torch.equal(total[-3:], b) and torch.equal(dx[-3:], da)
