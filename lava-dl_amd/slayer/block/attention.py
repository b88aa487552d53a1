"""A token-mixing layer of the operators that belong together: leaky attention, group norm of each head's result with an
activation, dropout from a counter, between two dense projections."""
import torch

from ..neuron.base import P_SCALE
from ..neuron.dropout import CounterDropout
from ..neuron.norm import GroupNorm
from ..synapse.attention import leaky_attention, leaky_attention_step


class LeakyAttention(torch.nn.Module):
    """Tokens [N, T, C] to tokens [N, T, C]: query, key and value of each head from one projection, leaky attention with
    a decay for each head, the heads' results normalised, activated and thinned out, and a projection back.

    Parameters
    ----------
    features : int
        C.
    heads, head_features : int
        heads and the keys and values of each (at most 128).
    decay : sequence of float or None
        12-bit decays of the heads, 0 to 4096; None: from 512 (a memory of eight tokens) to 4 (of a thousand), each the
        same factor from the next.
    train_decay : bool
        the decays are trained parameters; those that training has moved out of 0 to 4096 are set to the nearer end where they
        are used next, as the neurons' are.
    dropout : float
        probability; per element.
    activation : as for ``slayer.neuron.norm.group_norm``.
    seed : int or None
        of the dropout, as for ``slayer.neuron.CounterDropout``.

    The projections take the type of the tokens (``.to(torch.bfloat16)`` makes them bfloat16); decays, the norm's
    weights and the state are float32 all the same (a bfloat16 decay of 4095 would be one of 4096, which remembers nothing).
    """

    def __init__(self, features, heads, head_features=64, decay=None, train_decay=False, dropout=0.0, activation='silu', seed=None):
        super().__init__()
        if decay is None:
            decay = [512 / 128 ** (i / max(heads - 1, 1)) for i in range(heads)]
        if len(decay) != heads:
            raise ValueError(f'expected {heads} decays, got {len(decay)}')
        if not all(0 <= d <= P_SCALE for d in decay):
            raise ValueError(f'decays have to be between 0 and {P_SCALE}, got {list(decay)}')
        self.heads, self.head_features = heads, head_features
        self.scale = head_features ** -0.5
        self.project = torch.nn.Linear(features, 3 * heads * head_features, bias=False)
        self.norm = GroupNorm(heads, heads * head_features, activation=activation)
        self.dropout = CounterDropout(dropout, seed)
        self.back = torch.nn.Linear(heads * head_features, features, bias=False)
        decay = torch.tensor(decay, dtype=torch.float32)
        if train_decay:
            self.decay = torch.nn.Parameter(decay)
        else:
            self.register_buffer('decay', decay)

    def _apply(self, fn, recurse=True):
        """As torch's, but what is float32 stays float32 where ``fn`` changes types."""
        def keep(t):
            changed = fn(t)
            return changed if changed.dtype == t.dtype else t.to(changed.device)

        if recurse:
            for child in self.children():
                child._apply(keep if child is self.norm else fn)
        return super()._apply(keep, recurse=False)

    def _decay(self):
        if isinstance(self.decay, torch.nn.Parameter):
            self.decay.data.clamp_(0, P_SCALE)
        return self.decay

    def _heads(self, x):
        """query, key and value, views of one tensor [..., heads, head_features]."""
        return self.project(x).unflatten(-1, (3, self.heads, self.head_features)).unbind(-3)

    def _finish(self, y, offset=None):
        rows = y.reshape(y.shape[:-2].numel(), self.heads * self.head_features)
        return self.back(self.dropout(self.norm(rows), offset).view(*y.shape[:-2], rows.shape[1]))

    def forward(self, x, state=None, lengths=None, return_state=False, offset=None):
        """``x``: [N, T, C]; ``state``, ``lengths`` and ``return_state`` as for ``slayer.synapse.leaky_attention``, ``offset`` as
        for ``slayer.neuron.CounterDropout``."""
        mixed = leaky_attention(*self._heads(x), self._decay(), state, lengths, self.scale, return_state)
        return (self._finish(mixed[0], offset), mixed[1]) if return_state else self._finish(mixed, offset)

    def initial_state(self, samples):
        """The state in front of a first token: zeros, float32."""
        return torch.zeros(samples, self.heads, self.head_features, self.head_features, device=self.decay.device)

    @torch.no_grad()
    def step(self, x, state):
        """One token of each sample in generation: ``x`` [N, C] to [N, C], ``state`` is updated in place."""
        return self._finish(leaky_attention_step(*self._heads(x), self._decay(), state, self.scale))
