"""The token-mixing operators and autograd: what a graph has saved, forward-mode differentiation, recomputation."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def tokens(gen, n=2, t=5, h=2, k=16, v=8):
    return [torch.randn(n, t, h, d, generator=gen).to(DEV) for d in (k, k, v)]


def test_a_saved_state_that_is_stepped_is_noticed():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(1)
    q, k, v = tokens(gen)
    decay, state = torch.tensor([50.0], device=DEV), torch.randn(2, 2, 16, 8, generator=gen).to(DEV)
    query = q.clone().requires_grad_()
    out = slayer.synapse.leaky_attention(query, k, v, decay, state=state)
    want, = torch.autograd.grad(out.sum(), query, retain_graph=True)
    copy = state.clone()
    slayer.synapse.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, copy)           # another tensor: nothing happens
    assert torch.equal(torch.autograd.grad(out.sum(), query, retain_graph=True)[0], want)
    with torch.no_grad():
        slayer.synapse.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state[:])    # a view of the saved one
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()


def test_a_state_of_inference_mode_is_stepped():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(2)
    q, k, v = tokens(gen)
    decay = torch.tensor([50.0], device=DEV)
    plain = torch.zeros(2, 2, 16, 8, device=DEV)
    ref = slayer.synapse.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, plain)
    with torch.inference_mode():
        state = torch.zeros(2, 2, 16, 8, device=DEV)
        assert torch.equal(slayer.synapse.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state), ref) and torch.equal(state, plain)
        again = torch.zeros_like(plain)
    plain.zero_()
    with torch.inference_mode():                                                           # an ordinary tensor in inference mode
        slayer.synapse.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, plain)
    assert torch.equal(plain, state) and not again.any()


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_tangents_are_refused(grad):
    """There is no rule for them: an error, not a result without its tangent."""
    import lava_dl_amd.slayer as slayer
    from torch.autograd import forward_ad
    gen = torch.Generator().manual_seed(3)
    q, k, v = tokens(gen)
    decay, state = torch.tensor([50.0, 7.0], device=DEV), torch.zeros(2, 2, 16, 8, device=DEV)
    w = torch.randn(8, generator=gen).to(DEV)
    calls = [(lambda *x: slayer.synapse.leaky_attention(*x[:4], state=x[4]), [q, k, v, decay, state]),
             (lambda *x: slayer.synapse.leaky_attention_step(*x), [q[:, 0], k[:, 0], v[:, 0], decay, state.clone()]),
             (lambda *x: slayer.neuron.norm.group_norm(x[0], 2, x[1], x[2], activation='silu'), [v.flatten(0, 2), w, w.clone()]),
             (lambda *x: slayer.neuron.norm.group_norm(x[0], 2, x[1], x[2], activation='silu'), [v.flatten(1, 2), w, w.clone()]),
             (lambda x: slayer.neuron.counter_dropout(x, 0.5, 1), [v])]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for call, inputs in calls:
            ref = call(*(x.clone() for x in inputs))                                       # no tangent: as ever
            for i in range(len(inputs)):
                x = [y.clone() for y in inputs]
                x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call(*x)
            assert torch.equal(call(*(x.clone() for x in inputs)), ref)


def test_neuron_dynamics_refuse_forward_mode_tangents():
    import lava_dl_amd.slayer as slayer
    from torch.autograd import forward_ad
    x, decay, state = torch.randn(2, 3, 20, device=DEV), torch.tensor([400.0], device=DEV), torch.tensor([0.0], device=DEV)
    li = slayer.neuron.dynamics.leaky_integrator.dynamics
    with forward_ad.dual_level():
        li(x, decay, state, 64)
        with pytest.raises((RuntimeError, NotImplementedError)):
            li(forward_ad.make_dual(x, torch.ones_like(x)), decay, state, 64)


@pytest.mark.parametrize('shape,groups', [((300, 64), 4), ((3, 500, 64), 4), ((2, 9000), 1)])
def test_a_norm_keeps_its_statistics_and_no_workspace(shape, groups):
    import lava_dl_amd.slayer as slayer
    x, w, b = (torch.randn(s, device=DEV, requires_grad=True) for s in (shape, shape[-1:], shape[-1:]))
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append((t.data_ptr(), t.untyped_storage().nbytes())) or t, lambda t: t):
        slayer.neuron.norm.group_norm(x, groups, w, b)
    given = {t.data_ptr() for t in (x, w, b)}
    assert [size for at, size in kept if at not in given] == [2 * shape[0] * groups * 4]


@pytest.mark.parametrize('wrt,kept_states', [(('q', 'k', 'v'), True), (('q',), True), (('k', 'v'), False), (('q', 'k', 'v', 'decay'), False)])
def test_attention_keeps_the_states_of_its_segments_for_the_query_alone(wrt, kept_states):
    """... whose pass takes them; with the decays' gradient it makes them again, beside their derivatives."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(4)
    q, k, v = tokens(gen, t=1500)
    x = dict(q=q, k=k, v=v, decay=torch.tensor([50.0, 3.0], device=DEV))
    leaves = [x[name].requires_grad_() for name in wrt]
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.data_ptr()) or t, lambda t: t):
        out = slayer.synapse.leaky_attention(*x.values())
    assert (len(set(kept) - {t.data_ptr() for t in x.values()}) == 1) == kept_states
    for once in range(2):                                                    # the graph may be run twice
        grads = torch.autograd.grad(out.square().sum(), leaves, retain_graph=True)
        assert once == 0 or all(torch.equal(a, b) for a, b in zip(grads, first))
        first = grads
