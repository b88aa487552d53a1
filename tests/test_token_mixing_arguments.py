"""The token-mixing operators without a GPU: arguments that the C entry points and the Python layer refuse before any launch, and the
generator of the dropout against its published answers."""
import ctypes

import numpy as np
import pytest
import torch

from .util_philox import philox

ONE = ctypes.c_void_p(16)          # non-null; never dereferenced on these paths
EINVAL, ENULL, ERANGE = -1, -2, -3


def test_published_answers_of_the_generator():
    """Known answers distributed with the generator's paper: counter, key, words."""
    for counter, key, words in (
            ([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
            ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
            ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])):
        assert philox(np.array([counter]), key)[0].tolist() == words


def attention(**change):
    from lava_dl_amd.slayer import _native as N
    args = dict(samples=2, tokens=100, heads=3, keys=16, values=16, num_decays=3, decay=16, lengths=None, lengths_bytes=0, dtype=0, scale=1.0)
    args.update(change)
    a = N.Attention(**args)
    for stride in (a.query_stride, a.key_stride, a.value_stride, a.grad_stride):
        stride[:] = (4800, 48, 16)
    return a


@pytest.mark.parametrize('change,code', [
    (dict(samples=-1), EINVAL), (dict(tokens=-1), EINVAL), (dict(heads=0), EINVAL), (dict(keys=0), EINVAL), (dict(values=0), EINVAL),
    (dict(dtype=2), EINVAL), (dict(num_decays=2), EINVAL), (dict(lengths=16, lengths_bytes=2), EINVAL), (dict(decay=None), ENULL),
    (dict(keys=129), ERANGE), (dict(values=129), ERANGE), (dict(tokens=(1 << 30) + 1), ERANGE), (dict(samples=1 << 25), ERANGE)])
def test_attention_refuses(change, code):
    from lava_dl_amd.slayer import _native as N
    L, a = N.lib(), ctypes.byref(attention(**change))
    assert L.slayer_leaky_attention_workspace(a, 0) == code
    assert L.slayer_leaky_attention_fwd(ONE, None, ONE, ONE, ONE, None, a, ONE, 1 << 30, None) == code
    assert L.slayer_leaky_attention_bwd(*[ONE] * 12, a, ONE, 1 << 30, None) == code
    assert L.slayer_leaky_attention_step(ONE, ONE, ONE, ONE, ONE, a, None) == code


def test_attention_refuses_missing_tensors_and_workspace():
    from lava_dl_amd.slayer import _native as N
    L = N.lib()
    a = ctypes.byref(attention(tokens=10000))
    need = L.slayer_leaky_attention_workspace(a, 0)
    assert need > 0 and L.slayer_leaky_attention_workspace(a, 1) > need
    assert L.slayer_leaky_attention_fwd(None, None, ONE, ONE, ONE, None, a, ONE, need, None) == ENULL
    assert L.slayer_leaky_attention_fwd(ONE, None, ONE, None, ONE, None, a, ONE, need, None) == ENULL
    assert L.slayer_leaky_attention_fwd(ONE, None, ONE, ONE, ONE, None, a, None, need, None) == ENULL
    assert L.slayer_leaky_attention_fwd(ONE, None, ONE, ONE, ONE, None, a, ONE, need - 1, None) == EINVAL
    assert L.slayer_leaky_attention_bwd(*[ONE] * 5, None, *[ONE] * 6, a, ONE, 1 << 40, None) == ENULL             # no gradient of out
    assert L.slayer_leaky_attention_bwd(ONE, ONE, None, ONE, ONE, *[ONE] * 7, a, ONE, 1 << 40, None) == ENULL     # state's without value's
    assert L.slayer_leaky_attention_bwd(None, ONE, ONE, ONE, ONE, *[ONE] * 7, a, ONE, 1 << 40, None) == ENULL     # decay's without query's
    assert L.slayer_leaky_attention_bwd(*[ONE] * 12, a, ONE, 0, None) == EINVAL
    assert L.slayer_leaky_attention_step(ONE, None, ONE, ONE, ONE, a, None) == ENULL
    none = ctypes.byref(attention(samples=0))
    assert L.slayer_leaky_attention_fwd(None, None, None, None, None, None, none, None, 0, None) == 0
    assert L.slayer_leaky_attention_step(None, None, None, None, None, none, None) == 0
    assert L.slayer_leaky_attention_fwd(ONE, None, ONE, ONE, ONE, None, None, ONE, 0, None) == ENULL


def test_group_norm_and_dropout_refuse():
    from lava_dl_amd.slayer import _native as N
    L = N.lib()

    def norm(dtype=0, samples=4, pixels=1, channels=12, groups=3, eps=1e-5, act=0, out=ONE, stats=ONE, floats=1 << 30):
        return L.slayer_group_norm_fwd(out, stats, stats, ONE, None, None, dtype, samples, pixels, channels, groups, eps, act, ONE, floats, None)
    assert norm(dtype=3) == EINVAL and norm(channels=13) == EINVAL and norm(groups=0) == EINVAL and norm(act=4) == EINVAL
    assert norm(samples=-1) == EINVAL and norm(out=None) == ENULL and norm(pixels=5, stats=None) == ENULL
    assert norm(pixels=5, floats=1) == EINVAL and norm(channels=3 << 24) == ERANGE and norm(samples=0, out=None) == 0
    assert L.slayer_group_norm_workspace(0, 4, 1, 12, 5, 0) == EINVAL and L.slayer_group_norm_workspace(0, 4, 1, 12, 3, 0) == 0
    assert L.slayer_group_norm_workspace(0, 4, 9, 12, 3, 1) > 0

    def drop(out=ONE, dtype=0, n=16, steps=0, limit=5):
        return L.slayer_dropout(out, ONE, dtype, n, steps, limit, 1.0, 1, 2, None)
    assert drop(out=None) == ENULL and drop(dtype=9) == EINVAL and drop(n=-1) == EINVAL and drop(steps=5) == EINVAL
    assert drop(limit=65537) == EINVAL and drop(limit=-1) == EINVAL and drop(n=1 << 41) == ERANGE and drop(out=None, n=0) == 0


def test_python_layer_refuses_cpu_tensors():
    import lava_dl_amd.slayer as slayer
    q, s = torch.zeros(1, 2, 3, 4), torch.zeros(1, 3, 4, 4)
    for call in (lambda: slayer.synapse.leaky_attention(q, q, q, torch.zeros(3)),
                 lambda: slayer.synapse.leaky_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(3), s),
                 lambda: slayer.neuron.norm.group_norm(q, 2),
                 lambda: slayer.neuron.counter_dropout(q, 0.5, 1)):
        with pytest.raises(RuntimeError, match='no CPU implementation'):
            call()
    with pytest.raises(ValueError):
        slayer.neuron.counter_dropout(q, 1.5, 1)
    assert slayer.neuron.CounterDropout(0.0)(q) is q and slayer.neuron.CounterDropout(0.5).eval()(q) is q
