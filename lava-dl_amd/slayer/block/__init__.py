"""The part of a block's forward pass that follows the synapse: neuron, one-step delay, axonal delay; and layers that
mix tokens."""
from .attention import LeakyAttention
from .base import step_delay, neuron_delay
from .gated import GatedLeak

__all__ = ['GatedLeak', 'LeakyAttention', 'step_delay', 'neuron_delay']
