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
    if not torch.is_grad_enabled() and _ops.plain_call():
        return _ops.dropout(input, p, key, per_step)
    return _Dropout.apply(input, key, p, per_step)


class Dropout(torch.nn.Module):
    """Dropout module for the ``dropout`` argument of the neurons.

    Every call in training mode uses a new mask; outside of it the input passes.  Without a ``seed`` the
    key of a call comes from torch's generator of the input's device: the masks follow
    ``torch.manual_seed`` and the generator's state (a checkpointed segment that is recomputed repeats
    its masks, a resumed run goes on with them), and replays of a captured training step use new ones.
    With a ``seed`` the n-th call takes the key ``(seed, n)``, counted on the device, whatever else draws
    numbers; a forward that a backward pass recomputes cannot tell which call it repeats, and is refused.

    Parameters
    ----------
    p : float
        probability of a drop, 0..1.
    inplace : bool
        the reference's second argument; ``False`` only.
    per_step : bool
        drop single values instead of whole neurons.
    seed : int or None
        seed of a generator of the module's own, whose state is ``generator``, int64 ``(seed, offset)``; no
        part of ``state_dict()`` and no buffer: ranks that are to drop different neurons take different seeds.
    """

    def __init__(self, p=0.5, inplace=False, *, per_step=False, seed=None):
        super().__init__()
        if inplace:
            raise ValueError('dropout in place is not supported; the mask is never stored, so nothing is saved by it')
        if not 0.0 <= p <= 1.0:
            raise ValueError(f'dropout probability has to be between 0 and 1, but got {p}')
        self.p = float(p)
        self.per_step = per_step
        # no buffer: DistributedDataParallel would give every rank the first one's at each forward
        self.generator = None if seed is None else torch.tensor([seed, 0], dtype=torch.int64)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        if self.generator is not None:
            device = fn(torch.empty(0, device=self.generator.device)).device
            if device.type != 'meta':
                self.generator = self.generator.to(device)
        return self

    def forward(self, input):
        if not self.training or self.p == 0.0:
            return input
        return dropout(input, self.p, self._key(input.device), self.per_step)

    def _key(self, device):
        if self.generator is None:
            return torch.empty(2, dtype=torch.int64, device=device).random_()
        if torch._C._current_graph_task_id() != -1:     # inside a backward pass
            raise RuntimeError('this forward is recomputed by a backward pass, and Dropout with a seed of its own '
                               'cannot repeat its mask; leave seed=None under activation checkpointing')
        if self.generator.device != device:
            self.generator = self.generator.to(device)
        return _ops.dropout_next(self.generator)

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
