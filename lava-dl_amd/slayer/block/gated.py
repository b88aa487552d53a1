"""A token-mixing layer of gated leaky integrators between two dense projections."""
import torch

from ..neuron.base import P_SCALE
from ..neuron.gated import gated_leak, gated_leak_step
from ..utils.types import KeepsTypes


class GatedLeak(KeepsTypes):
    """Tokens [N, T, C] to tokens [N, T, C]: input and gate of each channel from one projection, the gated leak along the tokens, and a
    projection back.

    Parameters
    ----------
    features : int
        C.
    channels : int or None
        of the gated leak; None: as many as there are features.
    decay : sequence of float or None
        12-bit decays of the channels' open gates, 0 to 4096; None: from 4096 (an open gate replaces the state) to 16 (it keeps 255 of
        256), each the same factor from the next.
    train_decay : bool
        the decays are trained parameters; those that training has moved out of 0 to 4096 are set to the nearer end where they
        are used next, as the neurons' are.
    drive : as for ``slayer.neuron.gated_leak``.

    The projections take the type of the tokens (``.to(torch.bfloat16)`` makes them bfloat16); decays and the state are float32
    all the same.
    """

    def __init__(self, features, channels=None, decay=None, train_decay=False, drive='gain'):
        super().__init__()
        channels = features if channels is None else channels
        if decay is None:
            decay = [P_SCALE / 256 ** (i / max(channels - 1, 1)) for i in range(channels)]
        if len(decay) != channels:
            raise ValueError(f'expected {channels} decays, got {len(decay)}')
        if not all(0 <= d <= P_SCALE for d in decay):
            raise ValueError(f'decays have to be between 0 and {P_SCALE}, got {list(decay)}')
        self.channels, self.drive = channels, drive
        self.project = torch.nn.Linear(features, 2 * channels)
        self.back = torch.nn.Linear(channels, features, bias=False)
        decay = torch.tensor(decay, dtype=torch.float32)
        if train_decay:
            self.decay = torch.nn.Parameter(decay)
        else:
            self.register_buffer('decay', decay)

    def _decay(self):
        if isinstance(self.decay, torch.nn.Parameter):
            self.decay.data.clamp_(0, P_SCALE)
        return self.decay

    def _parts(self, x):
        """input and gate, views of one tensor [..., 2, channels]."""
        return self.project(x).unflatten(-1, (2, self.channels)).unbind(-2)

    def forward(self, x, state=None, lengths=None, return_state=False):
        """``x``: [N, T, C]; ``state``, ``lengths`` and ``return_state`` as for ``slayer.neuron.gated_leak``."""
        mixed = gated_leak(*self._parts(x), self._decay(), state, lengths, self.drive, return_state)
        return (self.back(mixed[0]), mixed[1]) if return_state else self.back(mixed)

    def initial_state(self, samples):
        """The state in front of a first token: zeros, float32."""
        return torch.zeros(samples, self.channels, device=self.decay.device)

    @torch.no_grad()
    def step(self, x, state):
        """One token of each sample in generation: ``x`` [N, C] to [N, C], ``state`` is updated in place."""
        return self.back(gated_leak_step(*self._parts(x), self._decay(), state, self.drive))
