"""Leaky attention: linear attention whose state leaks, with a decay for each head.

The state of a head is a matrix that leaks like the current of a CUBA neuron and is driven by outer products of keys and
values instead of weighted spikes.  The bodies are slayer_leaky_attention_fwd / bwd / step of libslayer_hip.so.
"""
import torch

from .. import _native as N

_LARGEST = 128         # keys and values of a head


def leaky_attention(query, key, value, decay, state=None, lengths=None, scale=1.0, return_state=False):
    """S[t] = (1 - decay / 4096) S[t-1] + key[t] (outer) value[t], out[t] = scale * query[t] S[t], for each sample and head.

    Parameters
    ----------
    query, key : torch.Tensor
        float32 or bfloat16 GPU tensors [N, T, H, K], K at most 128.
    value : torch.Tensor
        [N, T, H, V] of the same type, V at most 128.  Any strides: what has neighbouring elements along the last axis is
        read where it lies, what has not (the time-innermost tensors of the neurons, turned) is copied first.
    decay : torch.Tensor
        float32, one value or one for each head: 12-bit decays as the neurons have them, 0 keeps everything, 4096 nothing.
        Need not be whole; may be trained.
    state : torch.Tensor or None
        float32 [N, H, K, V], the state in front of the first token; None: zeros.
    lengths : torch.Tensor or None
        int32 or int64 GPU tensor of N token counts; None: T for every sample.  Tokens behind a sample's end are not read,
        their outputs and gradients are 0, and its last state is the one at its end.
    scale : float
    return_state : bool
        also return the last state, float32 [N, H, K, V], for the next part of a sample or ``leaky_attention_step``.

    Returns
    -------
    torch.Tensor [N, T, H, V], contiguous, of the type of the inputs; with ``return_state`` a pair of it and the state.

    The states and all sums are float32; gradients are those of query, key, value, decay (the derivative with respect to
    the decay itself) and state.  A value that is not finite leaves values that are not finite (an infinity may leave a NaN) in
    the results that it reaches, and in no others.
    """
    device, dtype = N.require_elements(query, key, value)
    if query.dim() != 4 or key.shape != query.shape or value.dim() != 4 or value.shape[:3] != query.shape[:3]:
        raise RuntimeError(f'expected query and key [N, T, H, K] and value [N, T, H, V], got {tuple(query.shape)}, '
                           f'{tuple(key.shape)} and {tuple(value.shape)}')
    n, t, h, k = query.shape
    _check_sizes(h, k, value.shape[3])
    _check_decay(decay, h, device)
    if state is not None:
        _check_state(state, (n, h, k, value.shape[3]), device)
    if lengths is not None:
        if not torch.is_tensor(lengths) or lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != (n,):
            raise RuntimeError(f'lengths: expected {n} int32 or int64 values')
        if lengths.device != device:
            raise RuntimeError(f'tensors on different devices: {device} and {lengths.device}')
        lengths = lengths.contiguous()
    inputs = (query, key, value, decay, state)
    if N.wants_grad(*(x for x in inputs if x is not None)):
        out, last = _LeakyAttention.apply(*inputs, lengths, float(scale), return_state)
    else:
        out, last = _forward(*inputs, lengths, float(scale), return_state)[:2]
    return (out, last) if return_state else out


def leaky_attention_step(query, key, value, decay, state, scale=1.0):
    """``leaky_attention`` for one token of each sample, in generation: ``state`` is updated in place.

    Parameters
    ----------
    query, key : torch.Tensor
        float32 or bfloat16 GPU tensors [N, H, K].
    value : torch.Tensor
        [N, H, V] of the same type.
    decay : torch.Tensor
        as for ``leaky_attention``.
    state : torch.Tensor
        float32 [N, H, K, V], contiguous.
    scale : float

    Returns
    -------
    torch.Tensor [N, H, V] of the type of the inputs.  There is no gradient: the state it would need is overwritten.  (A graph
    that has saved the state, as ``leaky_attention`` does with the one it starts from, says so when it is run backward.)
    """
    device, dtype = N.require_elements(query, key, value)
    shape, wide = query.shape, value.shape
    if len(shape) != 3 or key.shape != shape or len(wide) != 3 or wide[:2] != shape[:2]:
        raise RuntimeError(f'expected query and key [N, H, K] and value [N, H, V], got {tuple(query.shape)}, '
                           f'{tuple(key.shape)} and {tuple(value.shape)}')
    n, h, k = shape
    v = wide[2]
    _check_sizes(h, k, v)
    _check_decay(decay, h, device)
    _check_state(state, (n, h, k, v), device)
    if not state.is_contiguous():
        raise RuntimeError('the state is updated in place and has to be contiguous')
    if N.wants_grad(query, key, value, decay, state):
        raise RuntimeError('leaky_attention_step has no gradient: call it under torch.no_grad(), or leaky_attention')
    query, key, value, decay = _rows(query), _rows(key), _rows(value), decay.contiguous()
    out = torch.empty(wide, dtype=query.dtype, device=device)
    (qn, qh, _), (kn, kh, _), (vn, vh, _) = query.stride(), key.stride(), value.stride()
    args = N.Attention(n, 1, h, k, v, decay.numel(), decay.data_ptr(), None, 0, dtype, scale, (qn, 0, qh), (kn, 0, kh), (vn, 0, vh))
    with N.device_guard(device):
        N.check(N.lib().slayer_leaky_attention_step(out.data_ptr(), state.data_ptr(), query.data_ptr(), key.data_ptr(), value.data_ptr(),
                                                    args, N.stream_handle()))
    N.written(state)
    return out


def _check_sizes(heads, keys, values):
    if heads < 1 or not 1 <= keys <= _LARGEST or not 1 <= values <= _LARGEST:
        raise RuntimeError(f'expected at least one head with 1 to {_LARGEST} keys and values, got {heads} heads with {keys} '
                           f'and {values}')


def _check_decay(decay, heads, device):
    if not torch.is_tensor(decay) or decay.dtype is not torch.float32 or decay.dim() != 1 or decay.shape[0] not in (1, heads):
        raise RuntimeError(f'decay: expected one float32 value or {heads}')
    if decay.device != device:
        raise RuntimeError(f'tensors on different devices: {device} and {decay.device}')


def _check_state(state, shape, device):
    if not torch.is_tensor(state) or state.dtype is not torch.float32 or state.shape != shape:
        raise RuntimeError(f'state: expected a float32 tensor {list(shape)}')
    if state.device != device:
        raise RuntimeError(f'tensors on different devices: {device} and {state.device}')


def _rows(x):
    """``x`` as the kernels read it: neighbouring elements along the last axis."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _call(query, key, value, decay, lengths, scale):
    """The structure of the C calls."""
    n, t, h, k = query.shape
    return N.Attention(n, t, h, k, value.shape[3], decay.numel(), decay.data_ptr(), N.ptr(lengths),
                       0 if lengths is None else lengths.element_size(), N.ELEMENT_TYPES[query.dtype], scale, query.stride()[:3],
                       key.stride()[:3], value.stride()[:3])


def _workspace(args, backward, device):
    floats = N.lib().slayer_leaky_attention_workspace(args, backward)
    if floats < 0:
        N.check(int(floats))
    return torch.empty(floats, dtype=torch.float32, device=device) if floats else None, floats


def _forward(query, key, value, decay, state, lengths, scale, return_state):
    query, key, value, decay = _rows(query), _rows(key), _rows(value), decay.contiguous()
    state = None if state is None else state.contiguous()
    n, t, h, k = query.shape
    v = value.shape[3]
    out = torch.empty((n, t, h, v), dtype=query.dtype, device=query.device)
    last = torch.empty((n, h, k, v), dtype=torch.float32, device=query.device) if return_state else None
    args = _call(query, key, value, decay, lengths, scale)
    with N.device_guard(query.device):
        workspace, floats = _workspace(args, 0, query.device)
        N.check(N.lib().slayer_leaky_attention_fwd(N.ptr(out), N.ptr(last), N.ptr(query), N.ptr(key), N.ptr(value), N.ptr(state),
                                                   args, N.ptr(workspace), floats, N.stream_handle()))
    return out, last, query, key, value, decay, state, workspace


class _LeakyAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, decay, state, lengths, scale, return_state):
        out, last, *saved, starts = _forward(query, key, value, decay, state, lengths, scale, return_state)
        if not ctx.needs_input_grad[0] or ctx.needs_input_grad[3]:           # who else has no use for the states of the segments
            starts = None
        ctx.save_for_backward(*saved, starts, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_last):
        query, key, value, decay, state, starts, lengths = ctx.saved_tensors
        if grad_out is None:
            if grad_last is None:
                return (None,) * 8
            grad_out = value.new_zeros(query.shape[:3] + value.shape[3:])
        grad_out = _rows(grad_out)
        grad_last = None if grad_last is None else grad_last.contiguous()
        need = ctx.needs_input_grad
        new = [torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None
               for x, wanted in zip((query, key, value, decay, state), (need[0] or need[3], need[1], need[2] or need[4], *need[3:5]))]
        args = _call(query, key, value, decay, lengths, ctx.scale)
        args.grad_stride[:] = grad_out.stride()[:3]
        with N.device_guard(query.device):
            workspace, floats = _workspace(args, 1, query.device)
            N.check(N.lib().slayer_leaky_attention_bwd(*(N.ptr(x) for x in new), N.ptr(grad_out), N.ptr(grad_last), N.ptr(query),
                                                       N.ptr(key), N.ptr(value), N.ptr(state), N.ptr(starts),
                                                       args, N.ptr(workspace), floats, N.stream_handle()))
        return (*(x if wanted else None for x, wanted in zip(new, need)), None, None, None)
