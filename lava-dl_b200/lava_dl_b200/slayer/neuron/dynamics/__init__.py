"""Neuron dynamics primitives (mirror of ``lava.lib.dl.slayer.neuron.dynamics``)."""

from . import leaky_integrator, adaptive_threshold, resonator, adaptive_phase_th, adaptive_resonator
from . import linear_attention

__all__ = ['leaky_integrator', 'adaptive_threshold', 'resonator', 'adaptive_phase_th', 'adaptive_resonator',
           'linear_attention']
