"""Gated leak: the leaky integrator whose leak a token's gate opens, for tensors with the channels last.

A gated linear recurrence of the neurons' own kind: the decay is the 12-bit one of the leaky integrator, and the gate says for each token
how much of it acts.  The bodies are slayer_gated_leak_fwd / bwd / step of libslayer_hip.so."""
import torch

from .. import _native as N

DRIVES = {None: 0, 'none': 0, 'gain': 1, 'variance': 2}


def gated_leak(input, gate, decay, state=None, lengths=None, drive='gain', return_state=False):
    """leak[t] = decay / 4096 * sigmoid(gate[t]), h[t] = (1 - leak[t]) h[t-1] + drive(leak[t]) * input[t], for each sample and channel.

    Parameters
    ----------
    input, gate : torch.Tensor
        float32 or bfloat16 GPU tensors [N, T, C] of one type, N * ceil(C / 64) below 2**23 (C / 128 for bfloat16).  Any strides: what
        has neighbouring elements along the last axis is read where it lies (two views of one projection, say), what has not is copied first.
    decay : torch.Tensor
        float32, one value or one for each channel: the 12-bit decay of an open gate, 0 to 4096 (a state that an open gate
        replaces).  Need not be whole; may be trained.  1 - decay / 4096 is the least that a token keeps of the state.
    state : torch.Tensor or None
        float32 [N, C], the state in front of the first token; None: zeros.
    lengths : torch.Tensor or None
        int32 or int64 GPU tensor of N token counts; None: T for every sample.  Tokens behind a sample's end are not read,
        their outputs and gradients are 0, and its last state is the one at its end.
    drive : None, 'none', 'gain' or 'variance'
        what the input is multiplied with: 1; the leak, so that a constant input is what the state goes to; or
        sqrt(leak (2 - leak)), so that the state of a white input has the input's variance (its derivative where the leak is 0
        counts as 0).
    return_state : bool
        also return the last state, float32 [N, C], for the next part of a sample or ``gated_leak_step``.

    Returns
    -------
    torch.Tensor [N, T, C], contiguous, of the type of the inputs; with ``return_state`` a pair of it and the state.

    The states and all sums are float32; gradients are those of input, gate, decay (the derivative with respect to the decay itself)
    and state.  A value that is not finite leaves values that are not finite (an infinity may leave a NaN) in the results that it
    reaches, and in no others.
    """
    code = _drive(drive)
    device, dtype = N.require_elements(input, gate)
    if input.dim() != 3 or gate.shape != input.shape or input.shape[2] < 1:
        raise RuntimeError(f'expected input and gate [N, T, C], got {tuple(input.shape)} and {tuple(gate.shape)}')
    n, t, c = input.shape
    _check_decay(decay, c, device)
    if state is not None:
        _check_state(state, (n, c), device)
    if lengths is not None:
        if not torch.is_tensor(lengths) or lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != (n,):
            raise RuntimeError(f'lengths: expected {n} int32 or int64 values')
        if lengths.device != device:
            raise RuntimeError(f'tensors on different devices: {device} and {lengths.device}')
        lengths = lengths.contiguous()
    inputs = (input, gate, decay, state)
    if N.wants_grad(*inputs):
        out, last = _GatedLeak.apply(*inputs, lengths, code, return_state)
    else:
        out, last = _forward(*inputs, lengths, code, return_state, False)[:2]
    return (out, last) if return_state else out


def gated_leak_step(input, gate, decay, state, drive='gain'):
    """``gated_leak`` for one token of each sample, in generation: ``state`` is updated in place.

    Parameters
    ----------
    input, gate : torch.Tensor
        float32 or bfloat16 GPU tensors [N, C] of one type, N and C as for ``gated_leak``.
    decay, drive : as for ``gated_leak``.
    state : torch.Tensor
        float32 [N, C], contiguous.  It is rounded at every call: a leak below 2**-25 leaves it as it is.

    Returns
    -------
    torch.Tensor [N, C] of the type of the inputs: the state, rounded.  There is no gradient: the state it would need is overwritten.
    """
    code = _drive(drive)
    device, dtype = N.require_elements(input, gate)
    shape = input.shape
    if len(shape) != 2 or gate.shape != shape or shape[1] < 1:
        raise RuntimeError(f'expected input and gate [N, C], got {tuple(input.shape)} and {tuple(gate.shape)}')
    n, c = shape
    _check_decay(decay, c, device)
    _check_state(state, shape, device)
    if not state.is_contiguous():
        raise RuntimeError('the state is updated in place and has to be contiguous')
    if N.wants_grad(input, gate, decay, state):
        raise RuntimeError('gated_leak_step has no gradient: call it under torch.no_grad(), or gated_leak')
    input, gate, decay = _rows(input), _rows(gate), decay.contiguous()
    out = N.empty_as(input)
    args = N.GatedLeak(n, 1, c, decay.shape[0], decay.data_ptr(), None, 0, dtype, code, input.stride(0), 0, gate.stride(0))
    with N.device_guard(device):
        N.check(N.lib().slayer_gated_leak_step(out.data_ptr(), state.data_ptr(), input.data_ptr(), gate.data_ptr(), args,
                                               N.stream_handle()))
    N.written(state)
    return out


def _drive(drive):
    if drive not in DRIVES:
        raise ValueError(f'unknown drive {drive!r}: one of {list(DRIVES)}')
    return DRIVES[drive]


def _check_decay(decay, channels, device):
    if not torch.is_tensor(decay) or decay.dtype is not torch.float32 or decay.dim() != 1 or decay.shape[0] not in (1, channels):
        raise RuntimeError(f'decay: expected one float32 value or {channels}')
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


def _call(input, gate, decay, lengths, drive):
    """The structure of the C calls."""
    n, t, c = input.shape
    a, b = input.stride(), gate.stride()
    return N.GatedLeak(n, t, c, decay.shape[0], decay.data_ptr(), N.ptr(lengths), 0 if lengths is None else lengths.element_size(),
                       N.ELEMENT_TYPES[input.dtype], drive, a[0], a[1], b[0], b[1])


def _floats(count, device):
    if count < 0:
        N.check(int(count))
    return torch.empty(count, dtype=torch.float32, device=device) if count else None


def _forward(input, gate, decay, state, lengths, drive, return_state, keep):
    input, gate, decay = _rows(input), _rows(gate), decay.contiguous()
    state = None if state is None else state.contiguous()
    n, _, c = input.shape
    device = input.device
    out = N.empty_as(input)
    last = torch.empty((n, c), dtype=torch.float32, device=device) if return_state else None
    args = _call(input, gate, decay, lengths, drive)
    lib = N.lib()
    with N.device_guard(device):
        starts = _floats(lib.slayer_gated_leak_starts(args), device) if keep else None
        floats = lib.slayer_gated_leak_workspace(args, 0)
        workspace = _floats(floats, device)
        N.check(lib.slayer_gated_leak_fwd(out.data_ptr(), N.ptr(last), N.ptr(starts), input.data_ptr(), gate.data_ptr(), N.ptr(state), args,
                                          N.ptr(workspace), floats, N.stream_handle()))
    return out, last, input, gate, decay, starts


class _GatedLeak(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, gate, decay, state, lengths, drive, return_state):
        out, last, *saved = _forward(input, gate, decay, state, lengths, drive, return_state, True)
        ctx.save_for_backward(*saved, lengths)
        ctx.drive = drive
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @N.once_differentiable
    def backward(ctx, grad_out, grad_last):
        if grad_out is None and grad_last is None:
            return (None,) * 7
        input, gate, decay, starts, lengths = ctx.saved_tensors
        grad_out = torch.zeros_like(input) if grad_out is None else _rows(grad_out)
        grad_last = None if grad_last is None else grad_last.contiguous()
        need = ctx.needs_input_grad
        grad_input, grad_gate = N.empty_as(input), N.empty_as(gate)
        grad_decay = torch.empty_like(decay) if need[2] else None
        grad_state = torch.empty((input.shape[0], input.shape[2]), dtype=torch.float32, device=input.device) if need[3] else None
        args = _call(input, gate, decay, lengths, ctx.drive)
        args.grad_sample, args.grad_token, _ = grad_out.stride()
        lib = N.lib()
        with N.device_guard(input.device):
            floats = lib.slayer_gated_leak_workspace(args, 1)
            workspace = _floats(floats, input.device)
            N.check(lib.slayer_gated_leak_bwd(grad_input.data_ptr(), grad_gate.data_ptr(), N.ptr(grad_decay), N.ptr(grad_state),
                                              grad_out.data_ptr(), N.ptr(grad_last), input.data_ptr(), gate.data_ptr(),
                                              N.ptr(starts), args, N.ptr(workspace), floats, N.stream_handle()))
        return grad_input if need[0] else None, grad_gate if need[1] else None, grad_decay, grad_state, None, None, None
