"""Leaky attention on the GPU against the recurrence in float64, one token after the other.

Tolerances.  A result is a sum of terms; M is the same recurrence on magnitudes (for a gradient: its derivative), the sum of the
terms' magnitudes.  With u = 2^-24, a float32 evaluation in any order is off by less than the number of roundings a term goes
through times u M: 2 K in two products over the keys (K: the larger of keys and values, the gradients' products run over either),
128 in two sums over a chunk of 64 tokens, 4 for each chunk the state passes and 16 for weights.  bfloat16 tensors go through the
same sums as exact values; scores, states and leaked keys enter products as two numbers within 2^-16 of them (three products: 3 *
2^-16 M), and the result is rounded to 2^-8 of itself (eight significant bits)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEV = 'cuda:0'


def recurrence(q, k, v, a, state, lengths, scale):
    """(out, last state) in the type of the inputs; a: [H]."""
    n, t, h, dk = q.shape
    dv = v.shape[-1]
    S = torch.zeros(n, h, dk, dv, dtype=q.dtype) if state is None else state
    out = []
    for s in range(t):
        on = torch.tensor([s < length for length in lengths]).reshape(n, 1, 1, 1)
        S = torch.where(on, S * a[:, None, None] + k[:, s, :, :, None] * v[:, s, :, None, :], S)
        out.append(torch.where(on[..., 0], scale * torch.einsum('nhk,nhkv->nhv', q[:, s], S), 0))
    out = torch.stack(out, 1) if out else q.new_zeros(n, 0, h, dv)
    return out, S


def factor(k, v, t):
    return (2 * max(k, v) + 128 + 4 * (t // 64 + 1) + 16) * U


def close(got, ref, magnitude, rel, what):
    got, ref = got.detach().cpu().double(), ref.detach()
    assert got.shape == ref.shape, what
    half = 2.0 ** -8 if what.endswith('bfloat16') else 0.0
    tol = (rel + (3 * 2.0 ** -16 if half else 0.0)) * magnitude + half * ref.abs() * 1.01 + 1e-37
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - ref).abs() / tol).max())} of the bound'


def inputs(gen, n, t, h, k, v, dtype, state):
    q, key = (torch.randn(n, t, h, k, generator=gen).to(dtype) for _ in range(2))
    value = torch.randn(n, t, h, v, generator=gen).to(dtype)
    return q, key, value, torch.randn(n, h, k, v, generator=gen) if state else None


def decays(h):
    return torch.tensor([4096.0, 3.0, 1024.0, 100.5, 0.0][:h])


SIZES = [  # n, t, h, k, v, lengths
    (2, 1, 2, 16, 16, None), (1, 64, 3, 64, 64, None), (3, 65, 2, 20, 12, [65, 0, 1]), (2, 130, 1, 33, 7, [130, 64]),
    (2, 300, 5, 64, 64, [1, 300]), (1, 200, 2, 128, 128, None), (4, 63, 2, 1, 1, [63, 62, 0, 5]), (1, 129, 2, 48, 80, None),
    (2, 100, 2, 96, 40, [100, 37]), (1, 1300, 1, 32, 64, None), (2, 70, 2, 100, 128, None), (3, 520, 1, 8, 100, [520, 256, 255]),
    # heads enough for the joint pass of value's and key's gradients, in one piece and in segments
    (40, 70, 2, 64, 64, None), (23, 100, 3, 24, 40, list(range(0, 92, 4))), (9, 600, 2, 32, 64, [600, 0, 1, 64, 128, 300, 599, 512, 513]),
    (70, 65, 1, 56, 16, None), (35, 100, 2, 80, 48, None), (35, 130, 2, 16, 96, list(range(96, 131))), (70, 66, 1, 88, 8, None),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,h,k,v,lengths', SIZES)
@pytest.mark.parametrize('state', [False, True])
def test_results_and_gradients_follow_the_recurrence(n, t, h, k, v, lengths, state, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(t * 1000 + k + v)
    q, key, value, first = inputs(gen, n, t, h, k, v, dtype, state)
    decay, scale = decays(h), 0.3
    g, g_last = torch.randn(n, t, h, v, generator=gen).to(dtype), torch.randn(n, h, k, v, generator=gen)
    ends = [t] * n if lengths is None else lengths

    def oracle(magnitudes):
        fix = (lambda x: x.double().abs()) if magnitudes else (lambda x: x.double())
        leaves = [fix(x).requires_grad_() for x in (q, key, value)]
        a = (1 - decay.double() / 4096).requires_grad_()
        S = None if first is None else fix(first).requires_grad_()
        out, last = recurrence(*leaves, a, S, ends, scale)
        wrt = leaves + [a] + ([] if S is None else [S])
        return [out, last] + list(torch.autograd.grad([out, last], wrt, [fix(g), fix(g_last)], allow_unused=True))

    ref, mag = oracle(False), oracle(True)
    leaves = [x.to(DEV).requires_grad_() for x in (q, key, value, decay)] + ([first.to(DEV).requires_grad_()] if state else [])
    out, last = slayer.synapse.leaky_attention(*leaves[:4], state=leaves[4] if state else None, scale=scale, return_state=True,
                                               lengths=None if lengths is None else torch.tensor(lengths, device=DEV))
    assert out.dtype == dtype and out.is_contiguous() and last.dtype == torch.float32
    got = [out, last] + list(torch.autograd.grad([out, last], leaves, [g.to(DEV), g_last.to(DEV)]))
    ref[5], mag[5] = ref[5] / -4096, mag[5] / 4096                      # with respect to the decay
    rel, half = factor(k, v, t), 'bfloat16' if dtype == torch.bfloat16 else ''
    names = ['out ' + half, 'last', 'query ' + half, 'key ' + half, 'value ' + half, 'decay', 'state']
    for i, (x, name) in enumerate(zip(got, names)):
        # the float32 results of bfloat16 tensors: keys in three parts, 2^-24; the decay's gradient has its factors in two
        extra = 3 * 2.0 ** -16 if half and name == 'decay' else 2.0 ** -24
        close(x, ref[i], mag[i], rel + extra, name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gradients_against_differences(dtype):
    """The loss sum(out * g) + sum(last * g_last) is linear in the queries, the values and the first state, quadratic at most in
    nothing else but the decay: central differences of the float64 recurrence are exact but for it, where the step of 2^-6 decays
    leaves 1e-9 of the magnitude."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(5)
    n, t, h, k, v = 2, 90, 3, 24, 16
    q, key, value, first = inputs(gen, n, t, h, k, v, dtype, True)
    decay = torch.tensor([700.0, 30.0, 2000.0])
    g, g_last = torch.randn(n, t, h, v, generator=gen).to(dtype), torch.randn(n, h, k, v, generator=gen)
    leaves = [x.to(DEV).requires_grad_() for x in (q, key, value, decay, first)]
    out, last = slayer.synapse.leaky_attention(*leaves[:4], state=leaves[4], return_state=True)
    grads = torch.autograd.grad([out, last], leaves, [g.to(DEV), g_last.to(DEV)])
    base = [x.double() for x in (q, key, value, decay, first)]

    def loss(x, magnitude=False):
        a, gg, gl = 1 - x[3] / 4096, g.double(), g_last.double()
        if magnitude:
            x, gg, gl = [y.abs() for y in x], gg.abs(), gl.abs()
        o, last = recurrence(x[0], x[1], x[2], a, x[4], [t] * n, 1.0)
        return float((o * gg).sum() + (last * gl).sum())

    for i, grad in enumerate(grads):
        direction = torch.randn(base[i].shape, generator=gen).double()
        step = 2.0 ** -6
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + step * direction, base[i] - step * direction
        numeric = (loss(up) - loss(down)) / (2 * step)
        exact = float((grad.detach().cpu().double() * direction).sum())
        big = [x.abs() for x in base]
        big[3] = base[3]
        wide = list(big)
        wide[i] = big[i] + direction.abs() if i != 3 else base[3]
        size = abs(loss(wide, True)) if i != 3 else 90 * abs(loss(big, True)) / 2096          # |d a^n| <= n a^n / a
        rel = factor(k, v, t) + (2.0 ** -8 + 3 * 2.0 ** -16 if dtype == torch.bfloat16 else 0) + 1e-8
        assert abs(numeric - exact) <= rel * size, (i, numeric, exact, rel * size)


def test_layouts_of_the_inputs_do_not_matter():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        n, t, h, k, v = 2, 150, 4, 32, 48
        q, key, value = (x.to(DEV) for x in inputs(gen, n, t, h, k, v, dtype, False)[:3])
        decay = torch.tensor([50.0, 5.0, 500.0, 1.0], device=DEV)
        ref = slayer.synapse.leaky_attention(q, key, value, decay)
        heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, key, value)]
        packed = torch.cat((q, key, value), -1)
        views = list(packed.split((k, k, v), -1))
        odd = torch.empty(n, t, h, 2 * k + v + 1, device=DEV, dtype=dtype)
        odd[..., 1:] = packed                                               # rows that are not a multiple of 16 bytes
        unaligned = list(odd[..., 1:].split((k, k, v), -1))
        strided = [torch.stack((x, x), -1)[..., 0] for x in (q, key, value)]   # neighbours are not neighbours
        time_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, key, value)]
        for what in (heads_first, views, strided, time_first):
            assert torch.equal(slayer.synapse.leaky_attention(*what, decay), ref)
        one = slayer.synapse.leaky_attention(*unaligned, decay)              # another cut of the values: the order of nothing changes
        assert torch.equal(one, ref)
        shared = slayer.synapse.leaky_attention(q, key[:, :, :1].expand_as(key), value, decay)
        full = slayer.synapse.leaky_attention(q, key[:, :, :1].repeat(1, 1, h, 1), value, decay)
        assert torch.equal(shared, full)


def test_gradient_of_what_heads_share_is_the_sum():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(7)
    n, t, h, k, v = 2, 80, 3, 16, 16
    q, key, value = (x.to(DEV) for x in inputs(gen, n, t, h, k, v, torch.float32, False)[:3])
    g = torch.randn(n, t, h, v, generator=gen).to(DEV)
    decay = torch.tensor([300.0], device=DEV, requires_grad=True)            # one for all heads
    each = torch.full((h,), 300.0, device=DEV, requires_grad=True)
    one = key[:, :, :1].clone().requires_grad_()
    all_keys = key[:, :, :1].repeat(1, 1, h, 1).requires_grad_()
    a, b = torch.autograd.grad(slayer.synapse.leaky_attention(q, one.expand(n, t, h, k), value, decay), [one, decay], g)
    c, d = torch.autograd.grad(slayer.synapse.leaky_attention(q, all_keys, value, each), [all_keys, each], g)
    assert torch.allclose(a, c.sum(2, keepdim=True), rtol=4 * U, atol=8 * U * float(c.abs().max()))
    assert torch.allclose(b, d.sum(0, keepdim=True), rtol=1e-5, atol=4 * U * float(d.abs().sum()))


def test_one_decay_for_all_heads_is_that_decay_in_each():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(8)
    q, k, v = (x.to(DEV) for x in inputs(gen, 2, 100, 3, 16, 16, torch.float32, False)[:3])
    one = slayer.synapse.leaky_attention(q, k, v, torch.tensor([64.0], device=DEV))
    assert torch.equal(one, slayer.synapse.leaky_attention(q, k, v, torch.full((3,), 64.0, device=DEV)))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_sample_in_parts_and_token_by_token(dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(9)
    n, t, h, k, v = 2, 200, 3, 40, 24
    q, key, value = inputs(gen, n, t, h, k, v, dtype, False)[:3]
    decay = torch.tensor([40.0, 900.0, 4.0])
    ref, S = recurrence(*(x.double() for x in (q, key, value)), 1 - decay.double() / 4096, None, [t] * n, 0.5)
    mag, M = recurrence(*(x.double().abs() for x in (q, key, value)), 1 - decay.double() / 4096, None, [t] * n, 0.5)
    d = [x.to(DEV) for x in (q, key, value)]
    name, rel = str(dtype), factor(k, v, t) + 2.0 ** -24
    first, state = slayer.synapse.leaky_attention(*(x[:, :77] for x in d), decay.to(DEV), scale=0.5, return_state=True)
    rest, state = slayer.synapse.leaky_attention(*(x[:, 77:190] for x in d), decay.to(DEV), state=state, scale=0.5, return_state=True)
    close(torch.cat((first, rest), 1), ref[:, :190], mag[:, :190], rel, 'parts ' + name)
    for s in range(190, t):
        out = slayer.synapse.leaky_attention_step(*(x[:, s] for x in d), decay.to(DEV), state, scale=0.5)
        close(out, ref[:, s], mag[:, s], rel, f'step {s} ' + name)
    close(state, S, M, rel, 'state')


@pytest.mark.parametrize('n,h,k,v', [(1, 1, 1, 1), (2, 3, 64, 64), (3, 2, 128, 128), (2, 2, 33, 7), (1, 2, 5, 70), (4, 1, 100, 36)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_single_token(n, h, k, v, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(k * v)
    q, key = (torch.randn(n, h, k, generator=gen).to(dtype) for _ in range(2))
    value, state = torch.randn(n, h, v, generator=gen).to(dtype), torch.randn(n, h, k, v, generator=gen)
    decay = torch.tensor([123.0])
    a = 1 - 123 / 4096
    S = state.double() * a + key.double()[..., None] * value.double()[:, :, None]
    M = state.double().abs() * a + key.double().abs()[..., None] * value.double().abs()[:, :, None]
    on = state.to(DEV)
    out = slayer.synapse.leaky_attention_step(q.to(DEV), key.to(DEV), value.to(DEV), decay.to(DEV), on, scale=2.0)
    close(on, S, M, 4 * U, 'state')
    close(out, 2 * (q.double()[..., None] * S).sum(2), 2 * (q.double().abs()[..., None] * M).sum(2), (k + 8) * U, 'out ' + str(dtype))
    wide = torch.zeros(n, h, k + 3, device=DEV, dtype=dtype)                # a view of a larger tensor
    wide[..., 2:-1] = q.to(DEV)
    again = state.to(DEV)
    assert torch.equal(out, slayer.synapse.leaky_attention_step(wide[..., 2:-1], key.to(DEV), value.to(DEV), decay.to(DEV), again, scale=2.0))
    assert torch.equal(on, again)


def test_tokens_behind_the_end_are_not_read():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(10)
    for dtype in (torch.float32, torch.bfloat16):
        n, t, h, k, v = 4, 200, 2, 32, 32
        q, key, value, state = inputs(gen, n, t, h, k, v, dtype, True)
        lengths, decay = torch.tensor([0, 1, 128, 200], dtype=torch.int32), torch.tensor([20.0, 4096.0], device=DEV)
        g = torch.randn(n, t, h, v, generator=gen).to(dtype)
        behind = torch.arange(t)[None] >= lengths[:, None]
        results = []
        for fill in (0.0, float('nan'), float('inf')):
            x = [y.masked_fill(behind[..., None, None], fill).to(DEV).requires_grad_() for y in (q, key, value)]
            s = state.to(DEV).requires_grad_()
            out, last = slayer.synapse.leaky_attention(*x, decay, state=s, lengths=lengths.to(DEV), return_state=True)
            grads = torch.autograd.grad([out, last], x + [s], [g.masked_fill(behind[..., None, None], fill).to(DEV), torch.ones_like(last)])
            results.append([out, last, *grads])
        for a, b, c in zip(*results):
            assert torch.isfinite(a).all() and torch.equal(a, b) and torch.equal(a, c)
        out, last, gq, gk, gv, gs = results[0]
        for x in (out, gq, gk, gv):
            assert not x[behind.to(DEV)].any()
        assert torch.equal(last[0], state[0].to(DEV)) and torch.equal(gs[0], torch.ones_like(gs[0]))
        assert torch.equal(slayer.synapse.leaky_attention(*(y.to(DEV) for y in (q, key, value)), decay,
                                                          lengths=torch.tensor([900, 200, 201, 1 << 40], device=DEV)),
                           slayer.synapse.leaky_attention(*(y.to(DEV) for y in (q, key, value)), decay))      # at most T


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('t,s', [(200, 0), (200, 5), (200, 70), (200, 199), (64, 31), (130, 33), (1100, 700)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_values_that_are_not_finite_reach_no_earlier_token(t, s, bad, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(11)
    decay = torch.tensor([100.0, 4096.0], device=DEV)
    clean = [x.to(DEV) for x in inputs(gen, 2, t, 2, 20, 20, dtype, False)[:3]]
    ref = slayer.synapse.leaky_attention(*clean, decay)
    for which in range(3):
        x = list(clean)
        x[which] = x[which].clone()
        x[which][1, s, 0, 3] = bad
        y = slayer.synapse.leaky_attention(*x, decay)
        assert torch.equal(y[0], ref[0]) and torch.equal(y[1, :, 1], ref[1, :, 1]) and torch.equal(y[1, :s, 0], ref[1, :s, 0])
        if which == 0:
            assert not torch.isfinite(y[1, s, 0]).any() and torch.equal(y[1, s + 1:, 0], ref[1, s + 1:, 0])
        elif which == 1:
            assert not torch.isfinite(y[1, s:, 0]).any()
        else:
            assert not torch.isfinite(y[1, s:, 0, 3]).any()
            rest = [0, 1, 2] + list(range(4, 20))
            assert torch.equal(y[1, :, 0, rest], ref[1, :, 0, rest])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,s', [(2, 200, 70), (40, 200, 70), (40, 64, 31), (20, 1100, 700)])
def test_gradients_that_are_not_finite_reach_no_later_token(n, t, s, dtype):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(15)
    decay = torch.tensor([100.0, 4096.0], device=DEV)
    x = [y.to(DEV).requires_grad_() for y in inputs(gen, n, t, 2, 24, 24, dtype, False)[:3]]
    g = torch.randn(n, t, 2, 24, generator=gen).to(DEV).to(dtype)
    out = slayer.synapse.leaky_attention(*x, decay)
    ref = torch.autograd.grad(out, x, g, retain_graph=True)
    for bad in (float('nan'), float('inf')):
        h = g.clone()
        h[1, s, 0, 3] = bad
        got = torch.autograd.grad(out, x, h, retain_graph=True)
        for a, b in zip(got, ref):
            assert torch.equal(a[0], b[0]) and torch.equal(a[2:], b[2:]) and torch.equal(a[1, :, 1], b[1, :, 1])
            assert torch.equal(a[1, s + 1:, 0], b[1, s + 1:, 0])
        assert torch.equal(got[0][1, :s, 0], ref[0][1, :s, 0]) and not torch.isfinite(got[0][1, s, 0]).any()
        assert not torch.isfinite(got[1][1, :s + 1, 0]).any() and not torch.isfinite(got[2][1, :s + 1, 0, 3]).any()
        y = [v.detach().clone() for v in x]                                   # ... and a key that is not finite no earlier one's value
        y[1][1, s, 0, 5] = bad
        y = [v.requires_grad_() for v in y]
        dv = torch.autograd.grad(slayer.synapse.leaky_attention(*y, decay), y, g)[2]
        assert torch.equal(dv[1, :s, 0], ref[2][1, :s, 0]) and torch.equal(dv[1, s + 1:, 0], ref[2][1, s + 1:, 0])


def test_nothing_to_do():
    import lava_dl_amd.slayer as slayer
    decay = torch.tensor([5.0], device=DEV, requires_grad=True)
    state = torch.randn(2, 3, 8, 4, device=DEV, requires_grad=True)
    q, v = torch.empty(2, 0, 3, 8, device=DEV, requires_grad=True), torch.empty(2, 0, 3, 4, device=DEV, requires_grad=True)
    out, last = slayer.synapse.leaky_attention(q, q, v, decay, state=state, return_state=True)
    assert out.shape == (2, 0, 3, 4) and torch.equal(last, state)
    g = torch.autograd.grad(last, [state, decay, q, v], torch.ones_like(last))
    assert torch.equal(g[0], torch.ones_like(state)) and float(g[1]) == 0 and g[2].shape == q.shape
    none = torch.empty(0, 5, 3, 8, device=DEV)
    assert slayer.synapse.leaky_attention(none, none, none, decay.detach()).shape == none.shape
    assert slayer.synapse.leaky_attention_step(none[:, 0], none[:, 0], none[:, 0], decay.detach(),
                                               torch.empty(0, 3, 8, 8, device=DEV)).shape == (0, 3, 8)


def test_the_same_call_gives_the_same_bits_on_any_stream():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(12)
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, s = (x.to(DEV).requires_grad_() for x in inputs(gen, 2, 900, 2, 64, 64, dtype, True))
        decay = torch.tensor([9.0, 300.0], device=DEV, requires_grad=True)
        g = torch.randn(2, 900, 2, 64, generator=gen).to(DEV).to(dtype)

        def step():
            out, last = slayer.synapse.leaky_attention(q, k, v, decay, state=s, return_state=True)
            return [out, last, *torch.autograd.grad([out, last], [q, k, v, decay, s], [g, torch.ones_like(last)])]
        ref = step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = step()
        side.synchronize()
        for a, b in zip(ref, other):
            assert torch.equal(a, b)


def test_a_captured_graph_replays_the_call():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(13)
    q, k, v, state = (x.to(DEV) for x in inputs(gen, 2, 600, 2, 32, 32, torch.bfloat16, True))
    decay = torch.tensor([9.0, 300.0], device=DEV)
    one = [x[:, 0].contiguous() for x in (q, k, v)]

    def step(s):
        out, last = slayer.synapse.leaky_attention(q, k, v, decay, state=s, return_state=True)
        return out, slayer.synapse.leaky_attention_step(*one, decay, last), last
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(state)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen))
        state.copy_(torch.randn(state.shape, generator=gen))
        graph.replay()
        for a, b in zip(outs, step(state)):
            assert torch.equal(a, b), i
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(14)
    decay = torch.tensor([77.0, 5.0], device=DEV)
    big = torch.empty((1 << 31) + (1 << 20), dtype=torch.bfloat16, device=DEV)
    n, t, h, k = 2, 40, 2, 32
    ref = torch.randn(n, t, h, k, generator=gen).to(DEV).bfloat16()
    far = big.as_strided((n, t, h, k), ((1 << 31), h * k, k, 1))              # samples far apart
    far.copy_(ref)
    want = slayer.synapse.leaky_attention(ref, ref, ref, decay)
    assert torch.equal(slayer.synapse.leaky_attention(far, far, far, decay), want)
    apart = big.as_strided((n, t, h, k), (h * k, 1 << 25, k, 1))              # tokens far apart
    apart.copy_(ref)
    assert torch.equal(slayer.synapse.leaky_attention(apart, ref, apart, decay), want)
    one = big.as_strided((n, h, k), ((1 << 31), k, 1))
    one.copy_(ref[:, 0])
    a, b = torch.zeros(n, h, k, k, device=DEV), torch.zeros(n, h, k, k, device=DEV)
    assert torch.equal(slayer.synapse.leaky_attention_step(one, one, one, decay, a),
                       slayer.synapse.leaky_attention_step(*(ref[:, 0],) * 3, decay, b)) and torch.equal(a, b)


def test_refusals():
    import lava_dl_amd.slayer as slayer
    f = slayer.synapse.leaky_attention
    q, v, d = torch.zeros(2, 4, 3, 8, device=DEV), torch.zeros(2, 4, 3, 5, device=DEV), torch.zeros(3, device=DEV)
    bad = [dict(query=q.half(), key=q.half(), value=v.half()), dict(key=q.bfloat16()), dict(key=q[:, :3]), dict(value=v[:, :, :2]),
           dict(query=q[0], key=q[0], value=v[0]), dict(decay=d[:2]), dict(decay=d.double()), dict(decay=d.cpu()),
           dict(state=torch.zeros(2, 3, 8, 4, device=DEV)), dict(state=torch.zeros(2, 3, 8, 5, device=DEV).bfloat16()),
           dict(lengths=torch.zeros(3, device=DEV, dtype=torch.int32)), dict(lengths=torch.zeros(2, device=DEV)),
           dict(lengths=torch.zeros(2, dtype=torch.int32)), dict(query=q.cpu(), key=q.cpu(), value=v.cpu())]
    for change in bad:
        with pytest.raises(RuntimeError):
            f(**{**dict(query=q, key=q, value=v, decay=d), **change})
    wide = torch.zeros(1, 2, 1, 129, device=DEV)
    with pytest.raises(RuntimeError, match='128'):
        f(wide, wide, wide, d[:1])
    with pytest.raises(RuntimeError, match='128'):
        f(wide[..., :4], wide[..., :4], wide, d[:1])
    step, s = slayer.synapse.leaky_attention_step, torch.zeros(2, 3, 8, 5, device=DEV)
    with pytest.raises(RuntimeError, match='contiguous'):
        step(q[:, 0], q[:, 0], v[:, 0], d, torch.zeros(3, 2, 8, 5, device=DEV).transpose(0, 1))
    with pytest.raises(RuntimeError, match='no gradient'):
        step(q[:, 0].clone().requires_grad_(), q[:, 0], v[:, 0], d, s)
    with pytest.raises(RuntimeError):
        step(q[:, 0], q[:, 0], v[:, 0], d, s[:1])
