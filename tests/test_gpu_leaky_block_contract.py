"""What the token-mixing layer promises beside its formulas."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def test_bfloat16_is_that_of_the_projections():
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(1)
    block = slayer.block.LeakyAttention(64, 4, 16, decay=[4095.0, 2051.0, 511.0, 3.3]).to(DEV)
    by_hand = copy.deepcopy(block)
    by_hand.project.bfloat16(), by_hand.back.bfloat16()
    block = block.to(torch.bfloat16)
    x = torch.randn(3, 70, 64, device=DEV).bfloat16()
    y, state = block(x, return_state=True)
    ref, last = by_hand(x, return_state=True)
    assert y.dtype == torch.bfloat16 and state.dtype == torch.float32
    assert torch.equal(y, ref) and torch.equal(state, last)
    assert torch.equal(block.step(x[:, 0], state), by_hand.step(x[:, 0], last)) and torch.equal(state, last)


@pytest.mark.parametrize('step', [False, True])
def test_trained_decays_stay_in_their_range(step):
    """A decay below 0 would be a state that grows without end, one above 4096 a state whose sign alternates."""
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(2)
    block = slayer.block.LeakyAttention(16, 3, 16, decay=[0.0, 30.0, 4096.0], train_decay=True).to(DEV)
    x = torch.randn(2, 50, 16, device=DEV)
    with torch.no_grad():
        ref, last = block(x, return_state=True)
        state = block.initial_state(2)
        first = block.step(x[:, 0], state)
        block.decay.add_(torch.tensor([-400.0, 0.0, 900.0], device=DEV))      # what an optimizer may do
    if step:
        moved = block.initial_state(2)
        assert torch.equal(block.step(x[:, 0], moved), first) and torch.equal(moved, state)
    else:
        y, end = block(x, return_state=True)
        assert torch.equal(y, ref) and torch.equal(end, last)
        again = block(x)                                                      # two calls, then the gradients of both
        grads = torch.autograd.grad(y.sum() + again.sum(), block.decay)[0]
        assert torch.isfinite(grads).all()
    assert block.decay.tolist() == [0.0, 30.0, 4096.0]


@pytest.mark.parametrize('n,t', [(0, 5), (2, 0), (0, 0)])
def test_no_samples_or_no_tokens(n, t):
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(3)
    block = slayer.block.LeakyAttention(24, 3, 8, dropout=0.5, train_decay=True).to(DEV)
    x = torch.zeros(n, t, 24, device=DEV, requires_grad=True)
    state = torch.randn(n, 3, 8, 8, device=DEV)
    y, last = block(x, state=state, return_state=True)
    assert y.shape == x.shape and torch.equal(last, state)
    y.sum().backward()
    assert x.grad.shape == x.shape and not any(p.grad.any() for p in block.parameters())
    if n == 0:
        assert block.step(x.detach().new_zeros(0, 24), state).shape == (0, 24)


def test_the_last_state_is_made_where_it_is_asked_for(monkeypatch):
    import lava_dl_amd.slayer as slayer
    import lava_dl_amd.slayer.block.attention as module
    torch.manual_seed(4)
    block = slayer.block.LeakyAttention(24, 3, 8).to(DEV)
    x, asked, call = torch.randn(2, 70, 24, device=DEV), [], module.leaky_attention

    def watched(*args, **names):
        result = call(*args, **names)
        asked.append(isinstance(result, tuple))
        return result
    monkeypatch.setattr(module, 'leaky_attention', watched)
    y = block(x)
    other, state = block(x, return_state=True)
    assert asked == [False, True] and torch.equal(y, other) and state.shape == (2, 3, 8, 8)


@pytest.mark.parametrize('reentrant', [False, True])
def test_recomputed_activations(reentrant):
    """Activation checkpointing gives the gradients of the result that it belongs to."""
    import lava_dl_amd.slayer as slayer
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(5)
    block = slayer.block.LeakyAttention(24, 3, 8, dropout=0.5, seed=11).to(DEV)
    x = torch.randn(2, 70, 24, device=DEV, requires_grad=True)
    y = block(x, offset=4)
    want = torch.autograd.grad(y.square().sum(), [x, *block.parameters()])
    again = checkpoint(lambda t: block(t, offset=4), x, use_reentrant=reentrant)
    assert torch.equal(again, y)
    again.square().sum().backward()
    assert all(torch.equal(a, b.grad) for a, b in zip(want, [x, *block.parameters()]))
    with pytest.raises(RuntimeError, match='offset'):
        checkpoint(block, x, use_reentrant=reentrant).sum().backward()


@pytest.mark.parametrize('reentrant', [False, True])
def test_layers_have_masks_of_their_own_and_checkpointing_repeats_them(reentrant):
    import lava_dl_amd.slayer as slayer
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(6)
    layers = [slayer.block.LeakyAttention(24, 3, 8, dropout=0.5).to(DEV) for _ in range(2)]
    wrt = [p for layer in layers for p in layer.parameters()]
    x = torch.randn(2, 70, 24, device=DEV, requires_grad=True)
    ones = torch.ones(140, 24, device=DEV)
    assert not torch.equal(layers[0].dropout(ones), layers[1].dropout(ones))

    def run(call):
        torch.manual_seed(7)
        y = x
        for layer in layers:
            y = call(layer, y)
        return y, torch.autograd.grad(y.square().sum(), [x, *wrt]) if call is not again else y.square().sum().backward()

    def again(layer, y):
        return checkpoint(layer, y, use_reentrant=reentrant)
    y, want = run(lambda layer, y: layer(y))
    other, _ = run(again)
    assert torch.equal(y, other) and all(torch.equal(a, b.grad) for a, b in zip(want, [x, *wrt]))
