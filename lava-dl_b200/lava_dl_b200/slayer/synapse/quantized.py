"""Dense synapse in 8-bit integers (no counterpart in lava-dl, whose synapses multiply weights on the
8-bit grid as floats): the inference form of ``Dense``."""

import torch

from ... import _ops


class QuantDense(torch.nn.Module):
    """Fully connected synapse with 8-bit weights and 8-bit activations, inference only.

    Every time step of every sample is rounded to 8 bits with its own power of two as the step (the
    smallest whose 127-fold reaches the largest magnitude); the sums are whole numbers.  Spikes, and
    graded spikes on a binary grid of at most 7 bits, are held exactly: with weights that lie on the
    grid of ``weight_scale`` the output is that of the float synapse.

    Parameters
    ----------
    weight : int8 tensor
        ``[out_neurons, in_neurons]``; at most 131072 inputs.
    weight_scale : float tensor
        what a weight of 1 stands for, 1 element or one per output neuron.
    in_shape : tuple or None
        ``(channels, height, width)`` of an ``NCHWT`` input; ``None`` is ``(in_neurons, 1, 1)``.
    """

    def __init__(self, weight, weight_scale, in_shape=None):
        super().__init__()
        if weight.dim() != 2 or weight.dtype != torch.int8:
            raise TypeError(f'expected an int8 weight of 2 dimensions, got {weight.dtype} of {weight.dim()}')
        out_neurons, in_neurons = weight.shape
        if not 1 <= in_neurons <= 131072:
            raise ValueError(f'1 to 131072 input neurons are supported, found {in_neurons}')
        if weight_scale.numel() not in (1, out_neurons):
            raise ValueError(f'weight_scale must have 1 or {out_neurons} elements, found {weight_scale.numel()}')
        self.in_neurons, self.out_neurons = in_neurons, out_neurons
        self.in_shape = (in_neurons, 1, 1) if in_shape is None else tuple(in_shape)
        if len(self.in_shape) != 3 or self.in_shape[0] * self.in_shape[1] * self.in_shape[2] != in_neurons:
            raise ValueError(f'in_shape {self.in_shape} does not hold {in_neurons} input neurons')
        self.complex = False
        # rows padded to whole 16-byte words once, here
        self.register_buffer('weight_q', torch.nn.functional.pad(weight.detach(), (0, -in_neurons % 16)).contiguous())
        scale = weight_scale.detach().to(device=weight.device, dtype=torch.float32).reshape(-1)
        self.register_buffer('weight_scale', scale.expand(out_neurons).contiguous())

    @classmethod
    def from_dense(cls, dense, step=None, mask=None):
        """From a ``synapse.Dense``, its pre-hook applied.

        Parameters
        ----------
        dense : synapse.Dense
        step : float or None
            grid of the weights (``2 / w_scale`` of the neuron whose ``quantize_8bit`` is the pre-hook):
            kept exactly.  ``None`` rounds every output neuron's weights to 1/127 of their largest.
        mask : tensor or None
            multiplied onto the weights before the pre-hook.
        """
        with torch.no_grad():
            if dense.weight_norm_enabled:
                weight = torch._weight_norm(dense.weight_v, dense.weight_g, 0)
            else:
                weight = dense.weight.detach()
            if mask is not None:
                weight = weight * mask
            if dense.pre_hook_fx is not None:
                weight = dense.pre_hook_fx(weight)
            in_shape = tuple(weight.shape[1:4])
            weight = weight.reshape(weight.shape[0], -1).float()
            if step is None:
                scale = weight.abs().amax(1) / 127
                scale = torch.where(scale > 0, scale, torch.ones_like(scale))
            else:
                scale = torch.full((weight.shape[0],), float(step), device=weight.device)
            grid = torch.round(weight / scale[:, None])
            if not bool(((grid >= -128) & (grid <= 127)).all()):
                raise ValueError(f'weights beyond 8 bits of step {step}')
            return cls(grid.to(torch.int8), scale, in_shape)

    @property
    def shape(self):
        return torch.Size((self.out_neurons,) + self.in_shape + (1,))

    def forward(self, input):
        """``NCT`` or ``NCHWT`` input -> ``NCT`` (``NC11T``)."""
        if torch.is_grad_enabled() and input.requires_grad:
            raise RuntimeError('QuantDense is an inference synapse: its rounding has no gradient')
        if input.dim() == 3:
            return self._product(input)
        if input.dim() != 5 or tuple(input.shape[1:4]) != self.in_shape:
            raise ValueError(f'expected input of shape [batch, {self.in_neurons}, time] or '
                             f'[batch, {", ".join(map(str, self.in_shape))}, time], found {tuple(input.shape)}')
        n, t = input.shape[0], input.shape[-1]
        return self._product(input.reshape(n, self.in_neurons, t)).reshape(n, self.out_neurons, 1, 1, t)

    def _product(self, input):
        if _ops.plain_call():
            return _ops.qdense_fwd(input, self.weight_q, self.weight_scale, self.in_neurons)
        _ops.refuse_tangents('QuantDense', input)
        return _Product.apply(input, self.weight_q, self.weight_scale, self.in_neurons)

    def extra_repr(self):
        return f'{self.in_neurons}, {self.out_neurons}'


class _Product(torch.autograd.Function):
    """For traces, which record a Function as a call."""

    @staticmethod
    def forward(ctx, input, weight, weight_scale, in_neurons):
        return _ops.qdense_fwd(input, weight, weight_scale, in_neurons)
