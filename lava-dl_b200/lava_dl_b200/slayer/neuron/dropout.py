"""Neuron dropout (``src/lava/lib/dl/slayer/neuron/dropout.py``): a dropped neuron stays dropped for
all of its time steps.  The mask comes from a counter-based generator and is never stored: the
backward pass computes it again."""

import torch

from ... import _ops


def dropout(input, p, key, per_step=False):
    """Dropout under a given key; the same key drops the same neurons.

    Parameters
    ----------
    input : torch tensor
        CUDA tensor, time last.
    p : float
        probability of a drop, 0..1; what is kept is multiplied by ``1 / (1 - p)``.
    key : torch tensor
        int64 ``(seed, offset)`` on the input's device.  The mask of a call is a function of the key
        and the shape; the backward pass reads the key again, so it must not be overwritten before.
    per_step : bool
        drop single values instead of whole neurons.

    Returns
    -------
    torch tensor
        shaped like ``input``.
    """
    if not torch.is_grad_enabled():
        return _ops.dropout(input, p, key, per_step)
    return _Dropout.apply(input, key, p, per_step)


class Dropout(torch.nn.Module):
    """Dropout module for the ``dropout`` argument of the neurons.

    Every call in training mode uses a new mask; outside of it the input passes.  The generator's
    state ``(seed, offset)`` lives on the device and is moved on there, so replays of a captured
    training step use new masks as well.

    Parameters
    ----------
    p : float
        probability of a drop, 0..1.
    per_step : bool
        drop single values instead of whole neurons.
    seed : int or None
        seed of the generator; drawn from torch's default generator when ``None``.
    """

    def __init__(self, p=0.5, per_step=False, seed=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f'dropout probability has to be between 0 and 1, but got {p}')
        self.p = float(p)
        self.per_step = per_step
        if seed is None:
            seed = int(torch.randint(0, 2 ** 62, (1,)))
        self.register_buffer('generator', torch.tensor([seed, 0], dtype=torch.int64), persistent=False)

    def forward(self, input):
        if not self.training or self.p == 0.0:
            return input
        if self.generator.device != input.device:
            self.generator = self.generator.to(input.device)
        return dropout(input, self.p, _ops.dropout_next(self.generator), self.per_step)

    def extra_repr(self):
        return f'p={self.p}, per_step={self.per_step}'


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, key, p, per_step):
        ctx.save_for_backward(key)
        ctx.p, ctx.per_step = p, per_step
        return _ops.dropout(input, p, key, per_step)

    @staticmethod
    def backward(ctx, grad_output):
        (key,) = ctx.saved_tensors
        return _Dropout.apply(grad_output, key, ctx.p, ctx.per_step), None, None, None
