"""Gated leak, rotary positions and the norms around a block: graphs that are captured and replayed, streams, autograd's corners."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def calls(gen, dtype=torch.float32):
    """(name, function of its tensors, those tensors): sizes with several tiles and workgroups."""
    import lava_dl_amd.slayer as slayer
    rand = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    f = slayer.synapse.rotary_frequencies(16, device=DEV)
    at = torch.randint(0, 10 ** 6, (3,), generator=gen).to(DEV)
    x = lambda *s: rand(*s).to(dtype)
    return [('leak', lambda x, z, d, s: slayer.neuron.gated_leak(x, z, d, s, return_state=True),
             [x(3, 700, 130), x(3, 700, 130), rand(130).abs() * 500, rand(3, 130)]),
            ('rotary', lambda q, k: slayer.synapse.rotary(q, k, f, at), [x(3, 50, 4, 20), x(3, 50, 2, 20)]),
            ('norm', lambda a, r, g, w, i, s: slayer.neuron.norm.residual_norm(a, r, w, i, g, s, 'silu'),
             [x(70, 300), x(70, 300), x(70, 300), rand(300), rand(300), rand(300)])]


def forward_backward(call, inputs, upstream):
    out = call(*inputs)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, inputs, upstream))


@pytest.mark.parametrize('which', [0, 1, 2])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_captured_training_steps(which, dtype):
    """Two graphs of the same operator, captured one after the other and replayed in turn with eager work between, each with its own inputs."""
    gen = torch.Generator().manual_seed(1)
    name, call, inputs = calls(gen, dtype)[which]
    sets = []
    for _ in range(2):
        leaves = [x.detach().clone().requires_grad_() for x in inputs]
        with torch.no_grad():
            upstream = [torch.randn(o.shape, generator=gen).to(DEV).to(o.dtype) for o in call(*inputs)]
        sets.append((leaves, upstream))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for leaves, upstream in sets:
            forward_backward(call, leaves, upstream)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for leaves, upstream in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = forward_backward(call, leaves, upstream)
        graphs.append((graph, out))
    for turn in range(4):
        fresh = [[torch.randn(x.shape, generator=gen).to(DEV).to(x.dtype).abs() + 0.1 for x in leaves] for leaves, _ in sets]
        with torch.no_grad():
            for (leaves, _), new in zip(sets, fresh):
                for x, y in zip(leaves, new):
                    x.copy_(y)
        for graph, _ in graphs:
            graph.replay()
        if turn % 2:
            torch.cuda.synchronize()
        for (graph, out), (leaves, upstream), new in zip(graphs, sets, fresh):
            want = forward_backward(call, [y.requires_grad_() for y in new], upstream)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), (name, turn)


@pytest.mark.parametrize('which', [0, 1, 2])
def test_the_same_bits_on_any_stream_and_two_at_once(which):
    gen = torch.Generator().manual_seed(2)
    name, call, inputs = calls(gen)[which]
    leaves = [x.requires_grad_() for x in inputs]
    upstream = [torch.randn_like(o) for o in call(*leaves)]
    want = forward_backward(call, leaves, upstream)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(forward_backward(call, leaves, upstream))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_a_graph_of_autograd_is_run_twice():
    gen = torch.Generator().manual_seed(3)
    for name, call, inputs in calls(gen):
        leaves = [x.requires_grad_() for x in inputs]
        out = call(*leaves)
        g = [torch.randn_like(o) for o in out]
        once = torch.autograd.grad(out, leaves, g, retain_graph=True)
        again = torch.autograd.grad(out, leaves, g)
        assert all(torch.equal(a, b) for a, b in zip(once, again)), name


@pytest.mark.parametrize('which', [0, 2])
def test_second_derivatives_are_refused(which):
    gen = torch.Generator().manual_seed(4)
    name, call, inputs = calls(gen)[which]
    leaves = [x.requires_grad_() for x in inputs]
    out = call(*leaves)
    upstream = torch.ones_like(out[0]).requires_grad_()                         # what makes torch ask for the gradient's gradient
    grad, = torch.autograd.grad(out[0], leaves[0], upstream, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        grad.sum().backward()


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_tangents_are_refused(grad):
    import lava_dl_amd.slayer as slayer
    from torch.autograd import forward_ad
    gen = torch.Generator().manual_seed(5)
    every = calls(gen)
    x, z, d, s = every[0][2]
    every.append(('step', lambda x, z, d, s: slayer.neuron.gated_leak_step(x, z, d, s), [x[:, 0].clone(), z[:, 0].clone(), d, s]))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for name, call, inputs in every:
            call(*(x.clone() for x in inputs))
            for i in range(len(inputs)):
                x = [y.clone() for y in inputs]
                x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call(*x)


def test_a_saved_state_that_is_stepped_is_noticed():
    """The gated leak saves the states it needs and not the one it is given: a step on that one changes no gradient.  Gates that are
    overwritten are noticed."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(6)
    x, z = torch.randn(2, 9, 5, generator=gen).to(DEV).requires_grad_(), torch.randn(2, 9, 5, generator=gen).to(DEV)
    decay, state = torch.full((5,), 300.0, device=DEV), torch.randn(2, 5, generator=gen).to(DEV)
    out = slayer.neuron.gated_leak(x, z, decay, state)
    want, = torch.autograd.grad(out.sum(), x, retain_graph=True)
    with torch.no_grad():
        slayer.neuron.gated_leak_step(x[:, 0], z[:, 0], decay, state)
    assert torch.equal(torch.autograd.grad(out.sum(), x, retain_graph=True)[0], want)
    z.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()


def test_a_step_tells_autograd_that_the_state_was_written():
    import lava_dl_amd.slayer as slayer
    state = torch.ones(2, 5, device=DEV)
    w = torch.ones(2, 5, device=DEV, requires_grad=True)
    product = w * state
    with torch.no_grad():
        slayer.neuron.gated_leak_step(state * 2, state, torch.full((5,), 300.0, device=DEV), state[:])
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        product.sum().backward()
    with torch.inference_mode():
        fresh = torch.ones(2, 5, device=DEV)
        slayer.neuron.gated_leak_step(fresh * 2, fresh, torch.full((5,), 300.0, device=DEV), fresh)


def test_checkpointing_makes_the_same_gradients():
    from torch.utils.checkpoint import checkpoint
    gen = torch.Generator().manual_seed(7)
    for name, call, inputs in calls(gen):
        leaves = [x.requires_grad_() for x in inputs]
        g = [torch.randn_like(o) for o in call(*leaves)]
        want = torch.autograd.grad(call(*leaves), leaves, g)
        got = torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, g)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), name


def test_refusals():
    import lava_dl_amd.slayer as slayer
    x, d, s = torch.zeros(2, 3, 4, device=DEV), torch.ones(4, device=DEV), torch.zeros(2, 4, device=DEV)
    leak, step, rotary, norm = (slayer.neuron.gated_leak, slayer.neuron.gated_leak_step, slayer.synapse.rotary, slayer.neuron.norm.residual_norm)
    q, f = torch.zeros(2, 3, 2, 8, device=DEV), torch.ones(4, device=DEV, dtype=torch.float64)
    for match, call in [
            ('expected input and gate', lambda: leak(x, x[:, :2], d)), ('expected input and gate', lambda: leak(x[0], x[0], d)),
            ('different types', lambda: leak(x, x.to(torch.bfloat16), d)), ('float32 or bfloat16', lambda: leak(x.half(), x.half(), d)),
            ('decay', lambda: leak(x, x, d[:3])), ('decay', lambda: leak(x, x, d.double())), ('decay', lambda: leak(x, x, 5.0)),
            ('state', lambda: leak(x, x, d, s[:1])), ('state', lambda: leak(x, x, d, s.to(torch.bfloat16))),
            ('lengths', lambda: leak(x, x, d, lengths=torch.ones(2, device=DEV))), ('lengths', lambda: leak(x, x, d, lengths=[3, 3])),
            ('different devices', lambda: leak(x, x, d.cpu())), ('different devices', lambda: leak(x, x, d, s.cpu())),
            ('different devices', lambda: leak(x, x, d, lengths=torch.tensor([3, 3]))), ('no CPU', lambda: leak(x, x.cpu(), d)),
            ('expected input and gate', lambda: step(x, x, d, s)), ('state', lambda: step(x[:, 0], x[:, 0], d, s[:, :3])),
            ('contiguous', lambda: step(x[:, 0], x[:, 0], d, torch.zeros(4, 2, device=DEV).t())),
            ('no gradient', lambda: step(x[:, 0].requires_grad_(), x[:, 0], d, s)),
            ('expected query and key', lambda: rotary(q, q[:, :2], f)), ('expected query and key', lambda: rotary(q, q[..., :7], f)),
            ('expected query and key', lambda: rotary(q[0, 0], None, f)), ('expected query and key', lambda: rotary(torch.zeros(1, 1, 1, 5000, device=DEV), None, f)),
            ('frequency', lambda: rotary(q, q, f.float())), ('frequency', lambda: rotary(q, q, torch.ones(5, device=DEV, dtype=torch.float64))),
            ('position', lambda: rotary(q, q, f, torch.zeros(3, device=DEV, dtype=torch.int64))), ('position', lambda: rotary(q, q, f, torch.zeros(2, device=DEV))),
            ('position', lambda: rotary(q[:, 0], None, f, torch.zeros(2, 3, device=DEV, dtype=torch.int64))), ('position', lambda: rotary(q, q, f, 3)),
            ('different devices', lambda: rotary(q, q, f.cpu())), ('different devices', lambda: rotary(q, q, f, torch.zeros(2, dtype=torch.int64))),
            ('gate', lambda: norm(x, None, gate=x[:, :2])), ('residual', lambda: norm(x, x[:, :2])), ('residual', lambda: norm(x, x.to(torch.bfloat16))),
            ('weight', lambda: norm(x, None, d[:3])), ('inner', lambda: norm(x, None, inner=d.long())), ('scale', lambda: norm(x, None, scale=d[:3])),
            ('different devices', lambda: norm(x, None, d.cpu())), ('different devices', lambda: norm(x, x.cpu())),
            ('up to 8192', lambda: norm(torch.zeros(1, 8193, device=DEV), None)), ('up to 8192', lambda: norm(torch.zeros((), device=DEV), None))]:
        with pytest.raises(RuntimeError, match=match):
            call()
    for match, call in [('drive', lambda: leak(x, x, d, drive='other')), ('layout', lambda: rotary(q, q, f, layout='other')),
                        ('activation', lambda: norm(x, None, activation='gelu')), ('eps', lambda: norm(x, None, eps=-1.0))]:
        with pytest.raises(ValueError, match=match):
            call()
