"""Rotary positions: queries and keys turned by angles that grow with their position, so that their product depends on the distance
of two tokens.  With them the state of a leaky attention is a bank of resonators: it leaks and it turns.  The body is slayer_rotary of
libslayer_hip.so."""
import math

import torch

from .. import _native as N

LAYOUTS = {'halves': 0, 'pairs': 1}


def rotary_frequencies(turned, base=10000.0, scaling=None, factor=1.0, context=None, slow=1.0, fast=32.0, device=None):
    """The angles, in radians a token, that the ``turned // 2`` pairs of a head are turned by: base ** (-2 i / turned).

    Parameters
    ----------
    turned : int
        features that are turned, an even number.
    base : float
    scaling : None, 'linear', 'base' or 'parts'
        for contexts ``factor`` times as long as those that were trained.  'linear': all angles are divided by it.  'base': the base
        grows so that the slowest pair's angle is divided by it and the fastest one's stays.  'parts': pairs that turn fewer than
        ``slow`` times within ``context`` tokens are divided by it, those that turn more than ``fast`` times stay, those in
        between are mixed in proportion (a magnitude of 0.1 ln(factor) + 1 goes with it).
    factor : float
    context : int
        tokens of the trained context, for 'parts'.
    device : torch.device or None

    Returns
    -------
    torch.Tensor, float64 [turned // 2].
    """
    if turned < 0 or turned % 2:
        raise ValueError(f'turned has to be an even number of features, got {turned}')
    if scaling not in (None, 'linear', 'base', 'parts'):
        raise ValueError(f"unknown scaling {scaling!r}: one of [None, 'linear', 'base', 'parts']")
    if not factor > 0 or not base > 0:
        raise ValueError(f'base and factor have to be positive, got {base} and {factor}')
    exponent = torch.arange(0, turned, 2, dtype=torch.float64) / max(turned, 1)
    if scaling == 'base':
        if turned <= 2:                                    # one pair, which is the fastest
            return (base ** -exponent).to(device)
        base = base * factor ** (turned / (turned - 2))
    frequency = base ** -exponent
    if scaling == 'linear':
        frequency = frequency / factor
    if scaling == 'parts':
        if context is None or not 0 <= slow < fast:
            raise ValueError("scaling 'parts' needs the trained context, and slow below fast")
        stays = ((context * frequency / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        frequency = frequency * (stays + (1 - stays) / factor)
    return frequency.to(device)


def rotary(query, key, frequency, position=None, layout='halves', magnitude=1.0):
    """Turns pairs of the features of each head by position * frequency: (x, y) becomes magnitude * (c x - s y, c y + s x) with
    cosine c and sine s of that angle.  What lies behind the turned features is copied.

    Parameters
    ----------
    query, key : torch.Tensor
        float32 or bfloat16 GPU tensors [N, T, H, D] of one type, or [N, H, D] for one token of each sample; key may have another
        number of heads, or be None.  D at most 4096.  Any strides, as for ``leaky_attention``.
    frequency : torch.Tensor
        float64, F angles in radians a token, 2 F at most D (``rotary_frequencies``).
    position : torch.Tensor or None
        int32 or int64: N positions of the samples' first tokens, or [N, T] of every token; None: 0.
    layout : 'halves' or 'pairs'
        the pairs are features (i, i + F) or (2 i, 2 i + 1).
    magnitude : float

    Returns
    -------
    A pair of tensors, contiguous, of the shapes and type of query and key (None for a key that is None).  Angles are made in float64
    and do not lose digits far out (positions up to 2**53); products are float32.  Gradients are those of query and key (frequencies have none).
    """
    if layout not in LAYOUTS:
        raise ValueError(f'unknown layout {layout!r}: one of {list(LAYOUTS)}')
    device, _ = N.require_elements(query) if key is None else N.require_elements(query, key)
    shape, other = query.shape, None if key is None else key.shape
    if len(shape) not in (3, 4) or not 1 <= shape[-1] <= 4096 or \
            (other is not None and (len(other) != len(shape) or other[:-2] != shape[:-2] or other[-1] != shape[-1])):
        raise RuntimeError(f'expected query and key [N, T, H, D] or [N, H, D] with D up to 4096, got {tuple(shape)}'
                           + ('' if other is None else f' and {tuple(other)}'))
    if not torch.is_tensor(frequency) or frequency.dtype is not torch.float64 or frequency.dim() != 1 or \
            2 * frequency.shape[0] > shape[-1]:
        raise RuntimeError(f'frequency: expected up to {shape[-1] // 2} float64 values')
    if frequency.device != device:
        raise RuntimeError(f'tensors on different devices: {device} and {frequency.device}')
    if position is not None:
        if not torch.is_tensor(position) or position.dtype not in (torch.int64, torch.int32) or \
                not (position.shape == shape[:1] or len(shape) == 4 and position.shape == shape[:2]):
            raise RuntimeError(f'position: expected int32 or int64 values {[shape[0]]}' + (f' or {list(shape[:2])}' if len(shape) == 4 else ''))
        if position.device != device:
            raise RuntimeError(f'tensors on different devices: {device} and {position.device}')
        position = position.contiguous()
    return _turn(query, key, frequency.contiguous(), position, LAYOUTS[layout], float(magnitude), 0)


def _turn(query, key, *args):
    if N.wants_grad(query, key):
        return _Rotary.apply(query, key, *args)
    return _run(query, key, *args)


def _rows(x):
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _place(x):
    """``x`` as the kernel reads it, its address, its heads, the strides of its samples, tokens and heads, and room for the result."""
    if x is None:
        return None, None, 0, 0, 0, 0, None, None
    x = _rows(x)
    out = N.empty_as(x)
    if x.dim() == 4:
        sample, token, head, _ = x.stride()
    else:
        (sample, head, _), token = x.stride(), 0
    return x, x.data_ptr(), x.shape[-2], sample, token, head, out, out.data_ptr()


def _run(query, key, frequency, position, layout, magnitude, inverse):
    given = query if query is not None else key
    shape = given.shape
    query, a, query_heads, qn, qt, qh, out_query, to_query = _place(query)      # (the copies have to live until the launch)
    key, b, key_heads, kn, kt, kh, out_key, to_key = _place(key)
    width = each = 0
    if position is not None:
        width, each = position.element_size(), position.dim() == 2
    call = N.Rotary(shape[0], shape[1] if len(shape) == 4 else 1, query_heads, key_heads, shape[-1], 2 * frequency.shape[0],
                    frequency.data_ptr(), N.ptr(position), width, each, layout, N.ELEMENT_TYPES[given.dtype], magnitude, qn, qt, qh,
                    kn, kt, kh)
    with N.device_guard(given.device):
        N.check(N.lib().slayer_rotary(to_query, to_key, a, b, call, inverse, N.stream_handle()))
    return out_query, out_key


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, frequency, position, layout, magnitude, inverse):
        ctx.save_for_backward(frequency, position)
        ctx.args = (layout, magnitude, 1 - inverse)
        ctx.set_materialize_grads(False)
        return _run(query, key, frequency, position, layout, magnitude, inverse)

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        frequency, position = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            grad_query = None
        if not ctx.needs_input_grad[1]:
            grad_key = None
        if grad_query is None and grad_key is None:
            return (None,) * 7
        return (*_turn(grad_query, grad_key, frequency, position, *ctx.args), None, None, None, None, None)
