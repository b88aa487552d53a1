"""Gated leak, rotary positions and the norms around a block without a GPU: what the C entry points and the Python layer refuse before any launch,
and the angles."""
import ctypes
import math

import pytest
import torch

ONE = ctypes.c_void_p(16)          # non-null; never dereferenced on these paths
EINVAL, ENULL, ERANGE = -1, -2, -3


def leak(**change):
    from lava_dl_amd.slayer import _native as N
    args = dict(samples=2, tokens=100, channels=30, num_decays=30, decay=16, lengths=None, lengths_bytes=0, dtype=0, drive=1)
    args.update(change)
    return N.GatedLeak(**args)


@pytest.mark.parametrize('change,code', [
    (dict(samples=-1), EINVAL), (dict(tokens=-1), EINVAL), (dict(channels=0), EINVAL), (dict(dtype=2), EINVAL), (dict(drive=3), EINVAL),
    (dict(drive=-1), EINVAL), (dict(num_decays=2), EINVAL), (dict(lengths=16, lengths_bytes=2), EINVAL), (dict(decay=None), ENULL),
    (dict(tokens=(1 << 30) + 1), ERANGE), (dict(samples=1 << 24), ERANGE), (dict(channels=1 << 25, num_decays=1), ERANGE),
    (dict(samples=1 << 20, tokens=1 << 20), ERANGE)])
def test_gated_leak_refuses(change, code):
    from lava_dl_amd.slayer import _native as N
    L, a = N.lib(), ctypes.byref(leak(**change))
    assert L.slayer_gated_leak_workspace(a, 0) == L.slayer_gated_leak_workspace(a, 1) == L.slayer_gated_leak_starts(a) == code
    assert L.slayer_gated_leak_fwd(*[ONE] * 6, a, ONE, 1 << 40, None) == code
    assert L.slayer_gated_leak_bwd(*[ONE] * 9, a, ONE, 1 << 40, None) == code
    assert L.slayer_gated_leak_step(*[ONE] * 4, a, None) == code


def test_gated_leak_refuses_missing_tensors_and_workspace():
    from lava_dl_amd.slayer import _native as N
    L = N.lib()
    a = ctypes.byref(leak(tokens=1000))
    need, back = L.slayer_gated_leak_workspace(a, 0), L.slayer_gated_leak_workspace(a, 1)
    assert need > 0 and back > need and L.slayer_gated_leak_starts(a) == 2 * 16 * 30
    for i in (0, 3, 4):
        p = [ONE] * 6
        p[i] = None
        assert L.slayer_gated_leak_fwd(*p, a, ONE, need, None) == ENULL
    assert L.slayer_gated_leak_fwd(*[ONE] * 6, a, None, need, None) == ENULL
    assert L.slayer_gated_leak_fwd(*[ONE] * 6, a, ONE, need - 1, None) == EINVAL
    assert L.slayer_gated_leak_fwd(*[ONE] * 6, a, ctypes.c_void_p(20), need, None) == EINVAL        # words of 8 bytes
    for i in (0, 1, 4, 6, 7, 8):
        p = [ONE] * 9
        p[i] = None
        assert L.slayer_gated_leak_bwd(*p, a, ONE, back, None) == ENULL
    assert L.slayer_gated_leak_bwd(*[ONE] * 9, a, ONE, back - 1, None) == EINVAL
    assert L.slayer_gated_leak_step(ONE, None, ONE, ONE, a, None) == ENULL
    none = ctypes.byref(leak(samples=0))
    assert L.slayer_gated_leak_fwd(*[None] * 6, none, None, 0, None) == 0
    assert L.slayer_gated_leak_step(*[None] * 4, none, None) == 0
    assert L.slayer_gated_leak_fwd(*[ONE] * 6, None, ONE, 0, None) == ENULL
    assert L.slayer_gated_leak_workspace(ctypes.byref(leak(tokens=100)), 0) == 0                    # one tile: nothing to hand on


def test_rotary_refuses():
    from lava_dl_amd.slayer import _native as N
    L = N.lib()

    def call(p=(ONE,) * 4, **change):
        args = dict(samples=2, tokens=3, query_heads=2, key_heads=2, features=16, turned=16, frequency=16, dtype=0, magnitude=1.0)
        args.update(change)
        return L.slayer_rotary(*p, ctypes.byref(N.Rotary(**args)), 0, None)
    assert call(samples=-1) == EINVAL and call(tokens=-1) == EINVAL and call(query_heads=-1) == EINVAL and call(features=0) == EINVAL
    assert call(turned=17) == EINVAL and call(turned=18) == EINVAL and call(turned=-2) == EINVAL and call(dtype=2) == EINVAL
    assert call(position=16, position_bytes=2) == EINVAL and call(layout=2) == EINVAL
    assert call(features=4098) == ERANGE and call(query_heads=1 << 17) == ERANGE and call(tokens=1 << 31) == ERANGE
    assert call(samples=1 << 20, tokens=1 << 20) == ERANGE
    assert call(frequency=None) == ENULL
    for i in range(4):
        p = [ONE] * 4
        p[i] = None
        assert call(p) == ENULL
    assert call([None] * 4, samples=0) == 0 and call([None] * 4, query_heads=0, key_heads=0) == 0
    assert L.slayer_rotary(*[ONE] * 4, None, 0, None) == ENULL


def test_residual_norm_refuses():
    from lava_dl_amd.slayer import _native as N
    L = N.lib()

    def norm(**change):
        args = dict(rows=4, channels=12, inner=16, outer=16, scale=16, dtype=0, residual_dtype=0, activation=2, eps=1e-5, factor=1.0)
        args.update(change)
        return ctypes.byref(N.ResidualNorm(**args))
    need = L.slayer_residual_norm_workspace(norm())
    assert need > 0
    for change, code in ((dict(rows=-1), EINVAL), (dict(channels=0), EINVAL), (dict(dtype=2), EINVAL), (dict(residual_dtype=1), EINVAL),
                         (dict(activation=4), EINVAL), (dict(channels=8193), ERANGE), (dict(rows=1 << 40), ERANGE)):
        assert L.slayer_residual_norm_workspace(norm(**change)) == code
        assert L.slayer_residual_norm_fwd(*[ONE] * 6, norm(**change), None) == code
        assert L.slayer_residual_norm_bwd(*[ONE] * 12, norm(**change), ONE, 1 << 40, None) == code
    assert L.slayer_residual_norm_fwd(None, *[ONE] * 5, norm(), None) == ENULL                       # a weight and nowhere to put its result
    assert L.slayer_residual_norm_fwd(None, None, *[ONE] * 4, norm(outer=None), None) == ENULL       # nothing wanted
    assert L.slayer_residual_norm_fwd(*[ONE] * 3, None, ONE, ONE, norm(), None) == ENULL
    assert L.slayer_residual_norm_fwd(*[ONE] * 5, None, norm(), None) == ENULL                       # an activation without a gate
    assert L.slayer_residual_norm_fwd(*[ONE] * 6, norm(activation=0), None) == ENULL                 # a gate without an activation
    assert L.slayer_residual_norm_bwd(*[ONE] * 12, norm(), ONE, need - 1, None) == EINVAL
    assert L.slayer_residual_norm_bwd(*[ONE] * 12, norm(), None, need, None) == ENULL
    assert L.slayer_residual_norm_bwd(*[ONE] * 12, norm(scale=None), ONE, need, None) == ENULL       # a gradient of what there is not
    assert L.slayer_residual_norm_fwd(*[None] * 6, norm(rows=0), None) == 0
    assert L.slayer_residual_norm_fwd(*[ONE] * 6, None, None) == ENULL


def test_python_layer_refuses_cpu_tensors():
    import lava_dl_amd.slayer as slayer
    x = torch.zeros(1, 2, 4)
    for call in (lambda: slayer.neuron.gated_leak(x, x, torch.zeros(4)),
                 lambda: slayer.neuron.gated_leak_step(x[0], x[0], torch.zeros(4), x[0]),
                 lambda: slayer.synapse.rotary(x[None], None, torch.ones(2, dtype=torch.float64)),
                 lambda: slayer.neuron.norm.residual_norm(x, None)):
        with pytest.raises(RuntimeError, match='no CPU implementation'):
            call()


def test_angles():
    """Plain ones are powers of the base; scaled ones keep what they say they keep."""
    from lava_dl_amd.slayer.synapse import rotary_frequencies
    plain = rotary_frequencies(8, 10000.0)
    assert plain.dtype == torch.float64 and torch.allclose(plain, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15, atol=0)
    assert torch.equal(rotary_frequencies(8, scaling='linear', factor=4.0), plain / 4)
    based = rotary_frequencies(8, scaling='base', factor=4.0)
    assert based[0] == 1 and abs(float(based[-1]) - 0.001 / 4) < 1e-18 and (based <= plain).all()
    parts = rotary_frequencies(64, scaling='parts', factor=8.0, context=2048)
    whole = rotary_frequencies(64)
    turns = 2048 * whole / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], whole[turns >= 32]) and torch.allclose(parts[turns <= 1], whole[turns <= 1] / 8, rtol=1e-15, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (parts[between] < whole[between]).all() and (parts[between] > whole[between] / 8).all()
    assert rotary_frequencies(0).shape == (0,) and rotary_frequencies(2, scaling='base', factor=3.0).tolist() == [1.0]
    for bad in (dict(turned=7), dict(turned=8, scaling='other'), dict(turned=8, factor=0.0), dict(turned=8, base=-1.0),
                dict(turned=8, scaling='parts', factor=2.0), dict(turned=8, scaling='parts', factor=2.0, context=10, slow=5, fast=2)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)
