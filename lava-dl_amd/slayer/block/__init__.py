"""The part of a block's forward pass that follows the synapse: neuron, one-step delay, axonal delay; and a layer that
mixes tokens."""
from .attention import LeakyAttention
from .base import step_delay, neuron_delay

__all__ = ['LeakyAttention', 'step_delay', 'neuron_delay']
