"""Neuron dropout (counterpart of neuron/dropout.py:10-35 in the reference), and dropout whose mask comes from a counter
and is never stored (slayer_dropout of libslayer_hip.so)."""
import torch
import torch.nn.functional as F

from .. import _native as N


class Dropout(torch.nn.Dropout3d):
    """Drops whole neurons: a dropped neuron stays silent for every time step of the sample (the surviving
    ones are scaled by 1 / (1 - p), as torch's dropout does)."""

    def forward(self, input):
        shape = input.shape
        per_neuron = input.reshape((shape[0], -1, 1, 1, shape[-1]))       # one channel per neuron, time last
        return F.dropout3d(per_neuron, self.p, self.training, self.inplace).reshape(shape)


def counter_dropout(input, p, seed, offset=0, per_neuron=False):
    """Sets elements of ``input`` to zero with probability ``p`` and scales the others by the inverse of the share that
    stays.  Which ones is a function of ``seed``, ``offset`` and an element's place alone: the same call gives the same
    mask again, on any layout and for either type, and the backward pass works it out anew instead of keeping it.

    Parameters
    ----------
    input : torch.Tensor
        float32 or bfloat16 GPU tensor of any shape.
    p : float
        probability in [0, 1], rounded to a multiple of 1/65536: a decision takes sixteen bits of the generator
        (Philox-4x32 with ten rounds).  The scale is the inverse of what the rounded probability leaves.
    seed, offset : int
        0 <= seed, offset < 2**64.  Different offsets give masks that have nothing to do with each other: count it up
        from call to call.  A captured graph replays the numbers it was captured with.
    per_neuron : bool
        one decision for all elements along the last axis (the time steps of a neuron).

    Returns
    -------
    torch.Tensor, contiguous, of the shape and type of ``input``.
    """
    if not 0 <= p <= 1:
        raise ValueError(f'dropout probability has to be between 0 and 1, got {p}')
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError(f'seed and offset have to be between 0 and 2**64 - 1, got {seed} and {offset}')
    if per_neuron and torch.is_tensor(input) and input.dim() == 0:
        raise RuntimeError('per_neuron needs an axis of time steps, got a tensor without axes')
    if N.wants_grad(input):
        return _CounterDropout.apply(input, float(p), int(seed), int(offset), bool(per_neuron))
    return _dropout(input, float(p), int(seed), int(offset), bool(per_neuron))


def _dropout(input, p, seed, offset, per_neuron):
    device, dtype = N.require_elements(input)
    input = input.contiguous()
    out = torch.empty_like(input)
    limit = round(p * 65536)
    scale = 65536 / (65536 - limit) if limit < 65536 else 0.0
    with N.device_guard(device):
        N.check(N.lib().slayer_dropout(N.ptr(out), N.ptr(input), dtype, input.numel(), input.shape[-1] if per_neuron else 0,
                                       limit, scale, seed, offset, N.stream_handle()))
    return out


class _CounterDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, p, seed, offset, per_neuron):
        ctx.args = (p, seed, offset, per_neuron)
        return _dropout(input, *ctx.args)

    @staticmethod
    def backward(ctx, grad_output):
        p, seed, offset, per_neuron = ctx.args
        return counter_dropout(grad_output, p, seed, offset, per_neuron), None, None, None, None


class CounterDropout(torch.nn.Module):
    """:func:`counter_dropout` while training, the identity otherwise.

    ``seed`` None: every call draws a seed of its own from torch's host generator, so layers (and processes that are seeded
    differently) have masks of their own, ``torch.manual_seed`` repeats them, and activation checkpointing, which restores the
    generator, repeats that of the call it makes again.

    An integer ``seed``: ``offset`` counts the calls made while training; set it (and ``seed``) to repeat them.  It is part of the
    ``state_dict``, so that a run that is taken up again goes on with it.  Layers of equal shape and seed have equal masks.  A call inside a backward pass is one that was made before, as activation checkpointing makes
    it: counting on would give it another mask than the result it belongs to, so it is refused.  Give ``forward`` the offset of
    the call then."""

    def __init__(self, p=0.5, seed=None, per_neuron=False):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError(f'dropout probability has to be between 0 and 1, got {p}')
        self.p, self.seed, self.per_neuron, self.offset = p, seed, per_neuron, 0

    def forward(self, input, offset=None):
        """``offset``: as for :func:`counter_dropout`; None: counted up (0 where every call has a seed of its own)."""
        if not self.training or self.p == 0:
            return input
        if self.seed is None:
            seed = int(torch.empty((), dtype=torch.int64, device='cpu').random_())
            return counter_dropout(input, self.p, seed, offset or 0, self.per_neuron)
        if offset is None:
            if torch._C._current_graph_task_id() != -1:
                raise RuntimeError('CounterDropout: a call inside a backward pass (activation checkpointing?) would count on and '
                                   'take another mask than the call it repeats: pass that call\'s offset, or leave the seed to '
                                   'torch\'s generator (seed=None)')
            offset = self.offset
            self.offset += 1
        return counter_dropout(input, self.p, self.seed, offset, self.per_neuron)

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        if self.seed is not None:                           # its 64 bits in a signed number
            destination[prefix + 'offset'] = torch.tensor(self.offset - (self.offset >> 63 << 64), device='cpu')

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        key = prefix + 'offset'
        if key in state_dict:                               # (one from a module without a seed has none)
            self.offset = int(state_dict[key]) % (1 << 64)
            if key in unexpected_keys:
                unexpected_keys.remove(key)

    def extra_repr(self):
        return f'p={self.p}, seed={self.seed}, per_neuron={self.per_neuron}'
