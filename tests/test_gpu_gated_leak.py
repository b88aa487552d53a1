"""The gated leak against the recurrence in float64, token by token.

Tolerance.  With U = 2^-24: a leak is decay times a sigmoid that is (3 + 1.5 |z|) U off, so (5 + 1.5 |z|) U with its own rounding; what a token
keeps, 1 - leak, is U + leak (5 + 1.5 |z|) U off; what it adds is (10 + 3 |z|) U off (the square root's argument has the leak twice, at most).
A state is then off by what it had before, kept; by the errors of those two factors; and by four roundings of it (a product of spans and
its sum, twice: inside a wave and between waves, tiles and windows).  ``bound`` runs that recurrence next to the state; results are held to
it, bfloat16 results to half a step of theirs besides.  Gradients likewise: the derivative with respect to the state runs backwards with the
same factors, and products of two things that are off are off by either, times the other's magnitude."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24
DRIVES = [None, 'gain', 'variance']


def make(gen, n, t, c, dtype=torch.float32, far=2.0, state=True):
    x, z, g = (torch.randn(n, t, c, generator=gen).to(dtype) for _ in range(3))
    decay = torch.round(2 ** torch.linspace(12, 3, c, dtype=torch.float64)).float()
    s, gs = torch.randn(n, c, generator=gen), torch.randn(n, c, generator=gen)
    return dict(x=x, z=(far * z.float() - 1).to(dtype), decay=decay, state=s if state else None, lengths=None, g=g, gs=gs)


def exact(d, drive):
    """Results and gradients in float64 with the bound of each: {name: (value, bound)}."""
    x, z = d['x'].double(), d['z'].double()
    n, t, c = x.shape
    open_ = torch.sigmoid(z)
    dec = d['decay'].double()
    leak = dec / 4096 * open_
    if drive is None:
        f, slope = torch.ones_like(leak), torch.zeros_like(leak)
    elif drive == 'gain':
        f, slope = leak, torch.ones_like(leak)
    else:
        f = (leak * (2 - leak)).sqrt()
        slope = torch.where(leak > 0, (1 - leak) / f.clamp_min(1e-300), 0)
    lengths = [t] * n if d['lengths'] is None else d['lengths']
    on = torch.tensor([[s < l for l in lengths] for s in range(t)], dtype=torch.bool).reshape(t, n).t()[:, :, None]
    zero = torch.zeros((), dtype=torch.float64)
    x, z = torch.where(on, x, zero), torch.where(on, z, zero)
    leak, f, slope = torch.where(on, leak, zero), torch.where(on, f, zero), torch.where(on, slope, zero)
    keep, add = 1 - leak, f * x
    off_keep = U + leak * (5 + 1.5 * z.abs()) * U
    off_add = (10 + 3 * z.abs()) * U
    h = torch.zeros(n, c, dtype=torch.float64) if d['state'] is None else d['state'].double()
    m, e = h.abs(), torch.zeros_like(h)
    H, E, M, before = [], [], [], []
    for s in range(t):
        before.append((h, m, e))
        e = keep[:, s] * e + off_keep[:, s] * m + off_add[:, s] * add[:, s].abs()
        m = keep[:, s] * m + add[:, s].abs()
        e = e + 4 * U * m
        h = keep[:, s] * h + add[:, s]
        H.append(h), E.append(e)
    if t:
        got = {'out': (torch.where(on, torch.stack(H, 1), zero), torch.where(on, torch.stack(E, 1), zero))}
    else:
        got = {'out': (x, x)}
    got['last'] = (h, e)
    g = torch.where(on, d['g'].double(), zero)
    D = d['gs'].double()
    md, ed = D.abs(), torch.zeros_like(D)
    dx, bx, dz, bz = (torch.zeros(n, t, c, dtype=torch.float64) for _ in range(4))
    dd, bd = torch.zeros(c, dtype=torch.float64), torch.zeros(c, dtype=torch.float64)
    for s in range(t - 1, -1, -1):
        ed = ed + 4 * U * (md + g[:, s].abs())
        D, md = D + g[:, s], md + g[:, s].abs()
        hb, mb, eb = before[s]
        dx[:, s], bx[:, s] = f[:, s] * D, f[:, s] * (ed + off_add[:, s] * md)
        inside, size = slope[:, s] * x[:, s] - hb, (slope[:, s] * x[:, s]).abs() + mb
        dleak, off = D * inside, ed * size + md * (eb + 2 * off_add[:, s] * size)
        gate = leak[:, s] * (1 - open_[:, s])
        dz[:, s] = dleak * gate
        bz[:, s] = off * gate + md * size * leak[:, s] * (10 + 3 * z[:, s].abs()) * U
        o = torch.where(on[:, s], open_[:, s], zero) / 4096
        dd += (dleak * o).sum(0)
        bd += ((off + 40 * U * md * size) * o).sum(0)                      # 40: the sums over tokens, waves, tiles and samples
        ed = keep[:, s] * ed + off_keep[:, s] * md + 4 * U * md
        D, md = keep[:, s] * D, keep[:, s] * md
    got.update(dx=(dx, bx), dz=(dz, bz), ddecay=(dd, bd), dstate=(D, ed))
    return got


def run(d, drive, views=lambda x: x, grads=True):
    import lava_dl_amd.slayer as slayer
    x, z, g = (views(d[k].to(DEV)) for k in ('x', 'z', 'g'))
    decay = d['decay'].to(DEV)
    state = None if d['state'] is None else d['state'].to(DEV)
    lengths = None if d['lengths'] is None else torch.tensor(d['lengths'], device=DEV, dtype=torch.int32)
    if not grads:
        out, last = slayer.neuron.gated_leak(x, z, decay, state, lengths, drive, True)
        return {'out': out, 'last': last}
    leaves = [v.detach().requires_grad_() for v in (x, z, decay)] + ([] if state is None else [state.requires_grad_()])
    out, last = slayer.neuron.gated_leak(*leaves[:3], state if state is None else leaves[3], lengths, drive, True)
    grads = torch.autograd.grad([out, last], leaves, [g, d['gs'].to(DEV)])
    return dict(zip(('out', 'last', 'dx', 'dz', 'ddecay', 'dstate'), (out.detach(), last.detach(), *grads)))


def hold(got, want, dtype):
    for k, v in got.items():
        ref, bound = want[k]
        assert v.shape == ref.shape, k
        step = 2.0 ** -8 if v.dtype == torch.bfloat16 else U
        err = (v.detach().cpu().double() - ref).abs()
        assert not torch.isnan(err).any(), k
        # the smallest normal number: what is below it may be lost
        over = err - (bound + step * (ref.abs() + bound) + 2.0 ** -126)
        assert float(over.max() if over.numel() else -1) <= 0, (k, float(err.max()), float(over.max()))


@pytest.mark.parametrize('drive', DRIVES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,c', [
    (1, 1, 1), (2, 1, 3), (3, 2, 64), (1, 15, 65), (2, 16, 2), (2, 17, 127), (1, 63, 128), (2, 64, 129), (1, 65, 130), (2, 127, 5),
    (1, 128, 66), (2, 129, 200), (1, 255, 257), (3, 256, 1), (2, 257, 63), (1, 300, 191), (2, 640, 96), (1, 1100, 129)])
def test_results_and_gradients(n, t, c, dtype, drive):
    gen = torch.Generator().manual_seed(n * 1000003 + t * 101 + c)
    d = make(gen, n, t, c, dtype)
    hold(run(d, drive), exact(d, drive), dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,c', [(6, 40, 33), (7, 129, 70), (9, 500, 131), (2, 700, 64)])
def test_lengths(n, t, c, dtype):
    """Samples without tokens, of one, that end at and around borders of waves and tiles; what lies behind is never read."""
    gen = torch.Generator().manual_seed(t)
    d = make(gen, n, t, c, dtype)
    ends = [0, 1, t, t - 1, 16, 17, 64, 128, 129]
    d['lengths'] = [min(ends[i % len(ends)], t) for i in range(n)]
    want = exact(d, 'variance')
    for i, length in enumerate(d['lengths']):
        for k in 'xzg':
            d[k][i, length:] = float('nan')
    got = run(d, 'variance')
    hold(got, want, dtype)
    for i, length in enumerate(d['lengths']):
        for k in ('out', 'dx', 'dz'):
            assert not got[k][i, length:].any()
    assert torch.equal(got['last'][0].cpu(), d['state'][0]) and torch.equal(got['dstate'][0].cpu(), d['gs'][0])


@pytest.mark.parametrize('lengths', [[-3, 1 << 40, 5], [0, 0, 0]])
def test_lengths_outside_are_the_nearest_inside(lengths):
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(5)
    d = make(gen, 3, 20, 9)
    inside = [min(max(l, 0), 20) for l in lengths]
    out = [slayer.neuron.gated_leak(d['x'].to(DEV), d['z'].to(DEV), d['decay'].to(DEV), lengths=torch.tensor(l, device=DEV)) for l in (lengths, inside)]
    assert torch.equal(*out)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,t,c', [(1, 9000, 64), (1, 20000, 3), (40, 1500, 130), (2048, 300, 4), (700, 400, 70)])
def test_long_samples_and_many(n, t, c, dtype):
    """Windows of tiles and what lies between windows; chains so many that a workgroup walks one; both directions.  Channels apart, so
    that a slice of them in float64 is the whole answer for it."""
    gen = torch.Generator().manual_seed(t)
    d = make(gen, n, t, c, dtype, state=True)
    got = run(d, 'gain')
    rows, cols = slice(0, 2), slice(0, 5)
    part = dict(d, **{k: d[k][rows, ..., cols] for k in ('x', 'z', 'g', 'state', 'gs')}, decay=d['decay'][cols])
    want = exact(part, 'gain')
    del want['ddecay']
    hold({k: got[k][rows, ..., cols] for k in want}, want, dtype)
    again = run(d, 'gain')
    for k in got:
        assert torch.equal(got[k], again[k]), k                                 # the same bits, whoever came first


def test_strides():
    """Views of one projection, broadcast samples, reversed axes, an address that is a multiple of one element only."""
    gen = torch.Generator().manual_seed(11)
    for dtype in (torch.float32, torch.bfloat16):
        d = make(gen, 2, 150, 67, dtype)
        want = exact(d, 'gain')
        wide = torch.zeros(2, 150, 3, 67, dtype=dtype, device=DEV)

        def view(x):
            wide_ = wide.clone()
            wide_[:, :, 1] = x
            return wide_[:, :, 1]

        def shifted(x):
            flat = torch.zeros(x.numel() + 1, dtype=dtype, device=DEV)
            flat[1:] = x.flatten()
            return flat[1:].view(x.shape)
        for views in (view, shifted, lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)):
            hold(run(d, 'gain', views), want, dtype)
        one = dict(d, **{k: d[k][:1].expand(2, -1, -1) for k in 'xzg'})
        hold(run(one, 'gain', lambda x: x[:1].expand(2, -1, -1)), exact(one, 'gain'), dtype)


def test_one_decay_for_all_channels_is_that_decay_in_each():
    gen = torch.Generator().manual_seed(12)
    for dtype, c, t in ((torch.float32, 130, 40), (torch.bfloat16, 131, 700), (torch.float32, 1, 300)):
        d = make(gen, 3, t, c, dtype)
        d['decay'] = torch.tensor([37.5]).expand(c).contiguous()
        each = run(d, 'variance')
        one = run(dict(d, decay=torch.tensor([37.5])), 'variance')
        for k in ('out', 'last', 'dx', 'dz', 'dstate'):
            assert torch.equal(each[k], one[k])
        assert one['ddecay'].shape == (1,)
        want, bound = exact(d, 'variance')['ddecay']
        assert abs(float(one['ddecay']) - float(want.sum())) <= float(bound.sum()) + U * abs(float(want.sum()))


def test_parts_and_tokens_make_the_whole():
    """A sample in parts, then token by token, is the sample."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(13)
    for dtype in (torch.float32, torch.bfloat16):
        for c in (1, 64, 133):
            d = make(gen, 3, 200, c, dtype)
            for drive in DRIVES:
                want = exact(d, drive)
                x, z, decay = (d[k].to(DEV) for k in ('x', 'z', 'decay'))
                state = d['state'].to(DEV)
                y, state = slayer.neuron.gated_leak(x[:, :150], z[:, :150], decay, state, drive=drive, return_state=True)
                parts = [y]
                for t in range(150, 200):
                    parts.append(slayer.neuron.gated_leak_step(x[:, t], z[:, t], decay, state, drive)[:, None])
                hold({'out': torch.cat(parts, 1), 'last': state}, want, dtype)


def test_gradients_are_differences():
    """The derivative along a random direction, from results a step apart in either direction; float64 is not offered, so the step is 2^-8 of
    unit directions and the tolerance its square, 2^-16, times the third derivative's size, next to the rounding 2^-24 / 2^-8 of the
    differences: 2^-13 of the sums of magnitudes holds both with room for third derivatives of up to four times the first."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(14)
    d = make(gen, 2, 40, 8, far=1.0)
    g, gs = d['g'].to(DEV), d['gs'].to(DEV)
    for drive in DRIVES:
        for name, unit in (('x', 1.0), ('z', 1.0), ('decay', 64.0), ('state', 1.0)):
            v = torch.randn(d[name].shape, generator=gen) * unit
            if name == 'decay':
                v = v * (d['decay'] < 2000) * d['decay'] / 2000

            def value(sign):
                e = dict(d, **{name: d[name] + sign * 2.0 ** -8 * v})
                out, last = slayer.neuron.gated_leak(*(e[k].to(DEV) for k in ('x', 'z', 'decay', 'state')), drive=drive, return_state=True)
                return (out.double() * g).sum() + (last.double() * gs).sum()
            slope = float(value(1) - value(-1)) / 2 ** -7
            got = run(d, drive)['d' + name]
            terms = got.double().cpu() * v.double()
            assert abs(slope - float(terms.sum())) <= 2.0 ** -13 * (float(terms.abs().sum()) + float((run(d, drive)['out'].double() * g).abs().sum())), (drive, name)


def test_gates_at_the_ends():
    """Gates far out and infinite: open ones replace the state by what they drive, closed ones keep it."""
    import lava_dl_amd.slayer as slayer
    for dtype in (torch.float32, torch.bfloat16):
        z = torch.tensor([float('-inf'), -200, -90, 90, 200, float('inf')], dtype=dtype, device=DEV).reshape(1, 6, 1).expand(2, 6, 70)
        x = torch.full((2, 6, 70), 3.0, dtype=dtype, device=DEV)
        decay, state = torch.tensor([4096.0], device=DEV), torch.full((2, 70), 7.0, device=DEV)
        want = {None: [10, 13, 16, 3, 3, 3], 'gain': [7, 7, 7, 3, 3, 3], 'variance': [7, 7, 7, 3, 3, 3]}
        for drive in DRIVES:
            out = slayer.neuron.gated_leak(x, z, decay, state, drive=drive)
            assert out[0, :, 0].tolist() == want[drive] and torch.equal(out, out[:1, :, :1].expand_as(out))
            leaves = [v.detach().clone().requires_grad_() for v in (x, z, decay, state)]
            grads = torch.autograd.grad(slayer.neuron.gated_leak(*leaves, drive=drive).sum(), leaves)
            assert all(torch.isfinite(v).all() for v in grads)
    nothing = torch.zeros(1, device=DEV)
    leaves = [v.detach().float().clone().requires_grad_() for v in (x, z.clamp(-9, 9), nothing, state)]
    for drive in DRIVES:                                                       # a decay of 0: no leak, whatever the gate
        grads = torch.autograd.grad(slayer.neuron.gated_leak(*leaves, drive=drive).sum(), leaves)
        assert all(torch.isfinite(v).all() for v in grads) and not grads[1].any()


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('t,at', [(40, 21), (500, 300), (5000, 4500)])
def test_values_that_are_not_finite_go_forwards(bad, t, at):
    """In one channel, from their token on; gradients of the input before it, and of all other channels, are as without."""
    gen = torch.Generator().manual_seed(t)
    for dtype in (torch.float32, torch.bfloat16):
        d = make(gen, 2, t, 67, dtype)
        clean = run(d, 'gain')
        d['x'][1, at, 65] = bad
        got = run(d, 'gain')
        hit = torch.zeros(2, t, 67, dtype=torch.bool, device=DEV)
        hit[1, at:, 65] = True
        assert torch.equal(torch.where(hit, 0, got['out']), torch.where(hit, 0, clean['out'])) and not torch.isfinite(got['out'][1, at, 65])
        assert torch.equal(got['dx'], clean['dx'])
        assert torch.equal(torch.where(hit, 0, got['dz']), torch.where(hit, 0, clean['dz']))
        assert torch.equal(got['ddecay'][:65], clean['ddecay'][:65]) and torch.equal(got['ddecay'][66:], clean['ddecay'][66:])


def test_no_samples_no_tokens():
    import lava_dl_amd.slayer as slayer
    for n, t in ((0, 5), (3, 0), (0, 0)):
        x, z = (torch.zeros(n, t, 7, device=DEV, requires_grad=True) for _ in range(2))
        decay = torch.full((7,), 5.0, device=DEV, requires_grad=True)
        state = torch.randn(n, 7, device=DEV, requires_grad=True)
        out, last = slayer.neuron.gated_leak(x, z, decay, state, return_state=True)
        assert out.shape == (n, t, 7) and torch.equal(last, state)
        grads = torch.autograd.grad([out, last], [x, z, decay, state], [torch.ones_like(out), torch.ones_like(last)])
        assert not grads[2].any() and torch.equal(grads[3], torch.ones_like(state))
    assert slayer.neuron.gated_leak_step(torch.zeros(0, 4, device=DEV), torch.zeros(0, 4, device=DEV), torch.ones(1, device=DEV),
                                         torch.zeros(0, 4, device=DEV)).shape == (0, 4)


def test_only_what_is_wanted():
    """Each gradient alone, of the results alone and of the state alone, is that of the whole pass."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(17)
    d = make(gen, 2, 150, 66)
    g, gs = d['g'].to(DEV), d['gs'].to(DEV)
    base = [d[k].to(DEV) for k in ('x', 'z', 'decay', 'state')]
    for upstream in ((g, gs), (g, None), (None, gs)):
        def grads(which):
            leaves = [v.clone().requires_grad_(i in which) for i, v in enumerate(base)]
            outs = slayer.neuron.gated_leak(*leaves, drive='variance', return_state=True)
            used = [(o, u) for o, u in zip(outs, upstream) if u is not None]
            return torch.autograd.grad([o for o, _ in used], [leaves[i] for i in which], [u for _, u in used])
        whole = grads([0, 1, 2, 3])
        for i in range(4):
            assert torch.equal(grads([i])[0], whole[i])
