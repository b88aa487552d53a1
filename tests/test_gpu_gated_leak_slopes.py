"""The gated leak's gradients against differences of its own results, along directions in which they cannot hide.

The direction has the signs of the gradient, so that no part of the slope takes from another.  Tolerance: results are off by what the float64
recurrence says next to them, so the loss is, by the sum over the results, and the difference quotient by twice that over two steps; the
gradient by the same recurrence's bounds along the direction; and a difference is not a derivative, by as much as float64's difference is off
float64's gradient.  The slope is more than a hundred times all of that, which the test makes sure of: a gradient of zeros, or one of the other
sign, fails."""
import pytest
import torch

from tests.test_gpu_gated_leak import DRIVES, U, exact, make, run

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
NAMES = ['x', 'z', 'decay', 'state']


def cases(drive):
    """(name, inputs a step up and down, step times direction, slope in float64, tolerance)"""
    gen = torch.Generator().manual_seed(61)
    d = make(gen, 2, 40, 8, far=1.0)
    d.update({k: d[k].abs() for k in ('x', 'g', 'state', 'gs')})             # one sign, so that what the decays change adds up
    want = exact(d, drive)
    g, gs = d['g'].double(), d['gs'].double()

    def loss(e):
        got = exact(e, drive)
        (out, eo), (last, el) = got['out'], got['last']
        return float((out * g).sum() + (last * gs).sum()), float(((eo + U * out.abs()) * g.abs()).sum() + ((el + U * last.abs()) * gs.abs()).sum())
    for name in NAMES:
        grad, off = want['d' + name]
        size = torch.minimum(d['decay'], 4096 - d['decay']).double() if name == 'decay' else 1.0
        v = (2.0 ** -4 * size * grad.sign()).float()
        up, down = (dict(d, **{name: d[name] + s * v}) for s in (1, -1))
        v = (up[name].double() - down[name].double()) / 2                    # as float32 has it
        slope = float((grad * v).sum())
        (a, ea), (b, eb) = loss(up), loss(down)
        tolerance = (ea + eb) / 2 + abs((a - b) / 2 - slope) + float((off * v.abs()).sum()) + U * abs(slope)
        yield d, name, up, down, v, slope, tolerance


@pytest.mark.parametrize('drive', DRIVES)
def test_slopes(drive):
    import lava_dl_amd.slayer as slayer
    for d, name, up, down, v, slope, tolerance in cases(drive):
        assert abs(slope) > 100 * tolerance, (name, slope, tolerance)

        def loss(e):
            out, last = slayer.neuron.gated_leak(*(e[k].to(DEV) for k in NAMES[:3]), state=e['state'].to(DEV), drive=drive, return_state=True)
            return float((out.double() * d['g'].to(DEV)).sum() + (last.double() * d['gs'].to(DEV)).sum())
        rise = (loss(up) - loss(down)) / 2
        along = float((run(d, drive)['d' + name].double().cpu() * v).sum())
        assert abs(rise - along) <= tolerance, (name, rise, along, tolerance)
        assert abs(along - slope) <= tolerance, (name, along, slope)
