"""The norms around a block with its gate, scale and residual stream against the same formulas in float64.

Tolerance.  With U = 2^-24: a sum of C squares in a thread's own order and a tree has at most 8 + 11 roundings of terms of one sign, so a
reciprocal rms is (19 / 2 + 3) U < 13 U off (division, root, mean).  u is 14 U off, the gate (10 U: 6 of its sigmoid, products), the branch with its
weight and scale 14 + 10 + 4 = 28 U of its magnitude, total 30 U of |residual| + |branch| =: m.  hat and y then 13 + 30 U of m / rms, and what the
rms takes from total's errors, 30 U of the largest m / rms: 80 U of (m + mean m) / rms covers both.  A gradient has three products more and a
mean over the row of products that are 80 U off: 200 U of the sums of magnitudes, written out in ``sizes``.  Sums over R rows: a thread's
rows one after the other, then a tree and 1024 parts in 64 shares: 200 U + (R / 256 + 40) U of the sum of magnitudes.  bfloat16
results: half a step of theirs besides."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24


def make(gen, shape, dtype, stream, inner=True, outer=True, scale=True, gate=True, residual=True):
    c = shape[-1]
    d = dict(input=torch.randn(shape, generator=gen).to(dtype), inner=None, outer=None, scale=None, gate=None, residual=None)
    if inner:
        d['inner'] = 1 + 0.3 * torch.randn(c, generator=gen)
    if outer:
        d['outer'] = 1 + 0.3 * torch.randn(c, generator=gen)
    if scale:
        d['scale'] = 0.5 + 0.3 * torch.randn(c, generator=gen)
    if gate:
        d['gate'] = (2 * torch.randn(shape, generator=gen)).to(dtype)
    if residual:
        d['residual'] = (2 * torch.randn(shape, generator=gen)).to(stream)
    d['gy'] = torch.randn(shape, generator=gen).to(dtype)
    d['gt'] = torch.randn(shape, generator=gen).to(stream if residual else dtype)
    return d


def exact(d, activation, eps=1e-5, factor=1.0, use=('gy', 'gt')):
    """{name: (value, size)}: the formulas, and what the tolerance is taken of."""
    get = lambda k: None if d[k] is None else d[k].double().reshape(-1, d[k].shape[-1]) if d[k].dim() > 1 else d[k].double()
    x, r, z = get('input'), get('residual'), get('gate')
    one = torch.ones(x.shape[-1], dtype=torch.float64)
    wi, wo, s = (one if d[k] is None else get(k) for k in ('inner', 'outer', 'scale'))
    s = s * factor
    mean = lambda v: v.mean(-1, keepdim=True)
    r1 = (mean(x * x) + eps) ** -0.5 if d['inner'] is not None else torch.ones(len(x), 1, dtype=torch.float64)
    u = x * r1
    if z is None:
        a, da = torch.ones_like(x), torch.zeros_like(x)
    elif activation in (None, 'none'):
        a, da = z, torch.ones_like(z)
    else:
        p = torch.sigmoid(z)
        a, da = (p, p * (1 - p)) if activation == 'sigmoid' else (z * p, p * (1 + z * (1 - p)))
    b = a * wi * u
    total = s * b + (0 if r is None else r)
    m = (s * b).abs() + (0 if r is None else r.abs())
    got = {'total': (total, m)}
    gy = get('gy') if 'gy' in use and d['outer'] is not None else torch.zeros_like(x)
    gt = get('gt') if 'gt' in use else torch.zeros_like(x)
    dt, mdt = gt, gt.abs()
    hat = mh = torch.zeros_like(x)
    if d['outer'] is not None:
        r2 = (mean(total * total) + eps) ** -0.5
        hat, mh = total * r2, (m + mean(m)) * r2
        got['y'] = (hat * wo, mh * wo.abs())
        dh, mdh = gy * wo, (gy * wo).abs()
        dt = dt + r2 * (dh - hat * mean(dh * hat))
        mdt = mdt + r2 * (mdh + mh * mean(mdh * mh))
    db, mdb = dt * s, mdt * s.abs()
    mz = a.abs() + (0 if z is None else p.abs() if activation == 'sigmoid' else (z.abs() if activation == 'silu' else 0))
    d_, md = db * a * wi, mdb * mz * wi.abs()
    dx, mdx = d_, md
    if d['inner'] is not None:
        dx = r1 * (d_ - u * mean(d_ * u))
        mdx = r1 * (md + u.abs() * mean(md * u.abs()))
    slope = da.abs() + (0 if z is None else 1 + z.abs() if activation == 'silu' else 1)
    got.update(input=(dx, mdx), residual=(dt, mdt), gate=(db * u * wi * da, mdb * (u * wi).abs() * slope))
    for k, v, size in (('scale', dt * b * factor, mdt * mz * (wi * u).abs() * abs(factor)), ('inner', db * a * u, mdb * mz * u.abs()),
                       ('outer', gy * hat, gy.abs() * mh)):
        got[k] = (v.sum(0), size.sum(0))
    return got


def run(d, activation, views=lambda x: x, use=('gy', 'gt'), wrt=('input', 'residual', 'gate', 'outer', 'inner', 'scale'), factor=None):
    import lava_dl_amd.slayer as slayer
    t = {k: None if v is None else views(v.to(DEV)) if v.dim() > 1 else v.to(DEV) for k, v in d.items()}
    leaves = {k: t[k].requires_grad_() for k in wrt if t[k] is not None}
    out = slayer.neuron.norm.residual_norm(t['input'], t['residual'], t['outer'], t['inner'], t['gate'], t['scale'] if factor is None else factor,
                                           activation)
    y, total = out if t['outer'] is not None else (None, out)
    outs = [(o, t[g]) for o, g in ((y, 'gy'), (total, 'gt')) if o is not None and g in use]
    grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs])
    got = dict(zip(leaves, grads), total=total.detach())
    if y is not None:
        got['y'] = y.detach()
    return got


def hold(got, want, rows):
    for k, v in got.items():
        ref, size = want[k]
        if v.dim() > 1:
            v = v.reshape(-1, v.shape[-1])
        assert v.shape == ref.shape, k
        units = {'total': 30, 'y': 80}.get(k, 200 if v.dim() > 1 else 240 + rows / 256)
        step = 2.0 ** -8 if v.dtype == torch.bfloat16 else U
        err = (v.cpu().double() - ref).abs()
        over = err - (units * U * size + step * (ref.abs() + units * U * size) + 2.0 ** -126)
        assert not torch.isnan(err).any() and float(over.max() if over.numel() else -1) <= 0, (k, float(err.max()), float(over.max()))


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize('dtype,stream', TYPES)
@pytest.mark.parametrize('rows,c', [(1, 1), (3, 2), (5, 3), (2, 4), (7, 7), (9, 8), (65, 9), (33, 31), (40, 32), (17, 33), (300, 64), (10, 65), (21, 127),
                                    (12, 128), (700, 129), (5, 256), (6, 257), (11, 500), (13, 512), (9, 513), (3, 1000), (30, 1024), (7, 1025),
                                    (5, 2048), (300, 2047), (4, 2050), (9, 4096), (2, 4097), (600, 4101), (3, 8192), (5, 8191)])
def test_results_and_gradients(rows, c, dtype, stream):
    gen = torch.Generator().manual_seed(rows * 10007 + c)
    d = make(gen, (rows, c), dtype, stream)
    hold(run(d, 'silu'), exact(d, 'silu'), rows)


@pytest.mark.parametrize('dtype,stream', TYPES)
@pytest.mark.parametrize('c', [5, 48, 130, 600])
@pytest.mark.parametrize('gate', [None, 'none', 'sigmoid', 'silu'])
def test_with_and_without(gate, c, dtype, stream):
    """Every choice of what there is."""
    for i, (inner, outer, scale, residual) in enumerate(itertools.product((True, False), repeat=4)):
        gen = torch.Generator().manual_seed(c + i)
        d = make(gen, (2, 11, c), dtype, stream, inner, outer, scale, gate is not None, residual)
        activation = 'sigmoid' if gate is None else gate
        want = exact(d, activation)
        hold(run(d, activation), want, 22)
        if outer:
            for use in (('gy',), ('gt',)):
                hold({k: v for k, v in run(d, activation, use=use).items()}, exact(d, activation, use=use), 22)


def test_many_rows():
    gen = torch.Generator().manual_seed(1)
    for dtype, stream in TYPES:
        for rows, c in ((20000, 24), (5000, 200), (3000, 1030)):
            d = make(gen, (rows, c), dtype, stream)
            got = run(d, 'sigmoid')
            hold(got, exact(d, 'sigmoid'), rows)
            again = run(d, 'sigmoid')
            assert all(torch.equal(got[k], again[k]) for k in got)


def test_each_gradient_alone_is_that_of_the_whole():
    gen = torch.Generator().manual_seed(2)
    for c in (100, 700):
        d = make(gen, (9, c), torch.float32, torch.float32)
        whole = run(d, 'silu')
        for k in ('input', 'residual', 'gate', 'outer', 'inner', 'scale'):
            assert torch.equal(run(d, 'silu', wrt=(k,))[k], whole[k])


def test_strides_and_addresses():
    """Parts of a projection, axes in another order, broadcast rows, odd addresses."""
    gen = torch.Generator().manual_seed(3)
    for (dtype, stream), c in itertools.product(TYPES, (13, 72, 520)):
        d = make(gen, (3, 5, c), dtype, stream)
        want = exact(d, 'silu')

        def part(x):
            wide = torch.zeros(3, 5, 2, c, dtype=x.dtype, device=DEV)
            wide[:, :, 1] = x
            return wide[:, :, 1].detach()

        def shifted(x):
            flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)
            flat[1:] = x.flatten()
            return flat[1:].view(x.shape).detach()
        for views in (part, shifted, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), lambda x: x.transpose(0, 2).contiguous().transpose(0, 2)):
            hold(run(d, 'silu', views), want, 15)


def test_a_number_for_the_scale():
    gen = torch.Generator().manual_seed(4)
    for factor in (0.25, -2.0, 0.0):
        d = make(gen, (6, 90), torch.float32, torch.float32, scale=False)
        hold(run(d, 'silu', factor=factor), exact(d, 'silu', factor=factor), 6)


def test_weights_of_another_type_and_shapes():
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(40, generator=gen).to(DEV)                                  # one row, one axis
    w = torch.randn(40, generator=gen).to(DEV).to(torch.bfloat16).requires_grad_()
    y, total = slayer.neuron.norm.residual_norm(x, None, w)
    assert torch.equal(total, x) and y.shape == (40,)
    assert torch.equal(y.detach(), slayer.neuron.norm.residual_norm(x, None, w.detach().float(), return_sum=False))
    dw, = torch.autograd.grad(y.sum(), w)
    assert dw.dtype == torch.bfloat16
    for shape in ((0, 7), (2, 0, 7), (1, 1, 1, 7)):
        a, b = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(7, device=DEV, requires_grad=True)
        y, total = slayer.neuron.norm.residual_norm(a, a, b, b, a, b)
        grads = torch.autograd.grad([y, total], [a, b], [y, total])
        assert y.shape == total.shape == grads[0].shape == torch.Size(shape) and not grads[1].any()


def test_values_that_are_not_finite_stay_in_their_row():
    gen = torch.Generator().manual_seed(6)
    for c in (40, 300, 2000):
        d = make(gen, (5, c), torch.float32, torch.float32)
        clean = run(d, 'silu')
        for k in ('input', 'residual', 'gate'):
            e = dict(d, **{k: d[k].clone()})
            e[k][3, c // 2] = float('nan')
            got = run(e, 'silu')
            for out in ('y', 'total', 'input', 'residual', 'gate'):
                assert torch.equal(got[out][[0, 1, 2, 4]], clean[out][[0, 1, 2, 4]])
            assert torch.isnan(got['y'][3]).all()


def test_gates_at_the_ends():
    import lava_dl_amd.slayer as slayer
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.full((6, 33), 2.0, dtype=dtype, device=DEV)
        z = torch.tensor([float('-inf'), -200, -90, 90, 200, float('inf')], dtype=dtype, device=DEV)[:, None].expand(6, 33)
        assert slayer.neuron.norm.residual_norm(x, None, gate=z)[:, 0].tolist() == [0, 0, 0, 2, 2, 2]


def test_a_zero_row_and_module():
    import lava_dl_amd.slayer as slayer
    m = slayer.neuron.norm.ResidualNorm(16, scale=0.1).to(DEV)
    x = torch.zeros(3, 16, device=DEV, requires_grad=True)
    y, total = m(x, x, x)
    grads = torch.autograd.grad([y, total], [x, m.weight, m.inner, m.scale], [torch.ones_like(y), torch.ones_like(y)])
    assert not y.any() and not total.any() and all(torch.isfinite(g).all() for g in grads)
    only = slayer.neuron.norm.ResidualNorm(16, inner=False, outer=False)
    assert list(only.parameters()) == [] and 'scale=False' in repr(only)
    half = x.detach().to(torch.bfloat16)
    y, total = m(half, x.detach(), half)
    assert y.dtype == torch.bfloat16 and total.dtype == torch.float32


def test_gradients_are_differences():
    """The derivative along a random direction from results h = 2^-6 to either side.  The difference is off by h^2 / 6 of third derivatives, which are
    some ten times the magnitudes at most where rows are of unit size (2^-12 * 10 / 6 < 2^-10), and by the results' rounding, 80 * 2^-24 / h = 2^-12:
    2^-9 of the sum of the terms' magnitudes."""
    import lava_dl_amd.slayer as slayer
    gen = torch.Generator().manual_seed(8)
    for c in (30, 300):
        d = make(gen, (4, c), torch.float32, torch.float32)
        d['residual'] = d['residual'] / 2
        got = run(d, 'silu')
        g, gt = d['gy'].double(), d['gt'].double()
        for k in ('input', 'residual', 'gate', 'outer', 'inner', 'scale'):
            v = torch.randn(d[k].shape, generator=gen)

            def value(sign):
                e = {n: None if t is None else t.to(DEV) for n, t in dict(d, **{k: d[k] + sign * 2.0 ** -6 * v}).items()}
                y, total = slayer.neuron.norm.residual_norm(e['input'], e['residual'], e['outer'], e['inner'], e['gate'], e['scale'], 'silu')
                return y.cpu().double() * g, total.cpu().double() * gt
            (a, b), (p, q) = value(1), value(-1)
            slope = float((a - p).sum() + (b - q).sum()) * 2 ** 5
            terms = got[k].cpu().double() * v.double()
            size = float(terms.abs().sum() + a.abs().sum() + b.abs().sum())
            assert abs(slope - float(terms.sum())) <= 2.0 ** -9 * size, (k, slope, float(terms.sum()))
