"""Linear attention with a decay for each head (no counterpart in lava-dl): a leaky integrator whose
input is the outer product of a key and a value, read out by a query."""

import torch
from torch.autograd.function import once_differentiable

from .... import _ops


def dynamics(query, key, value, decay, state=None, return_state=False, precise=False):
    """Linear attention over whole sequences.

    .. math::
        S[t] &= (1 - \\alpha / 4096)\\,S[t-1] + k[t]\\,v[t]^\\top \\

        o[t] &= S[t]^\\top q[t]

    Differentiable (once) in ``query``, ``key``, ``value`` and ``state``.  ``decay`` is a constant of
    the head: one that requires a gradient is refused.

    An output (gradient, state) is off by less than ``2^-23 (width + 280 + time / 64)`` of the sum of its
    terms' magnitudes, whatever their sizes, as long as the states fit fp32; ``2^-21`` is usual.  Whole
    sequences run in chunks whose vectors are held as pairs of 16-bit numbers with one exponent for each
    step (each row of scores, each column of the state), 22 bits of fp32's 24: an element far below the
    largest of its step keeps fewer (2^20 below, some 17), which adds up to ``2^-28`` of the same sum over the
    largest magnitudes of each step's vectors.  ``precise`` walks step by step in fp32 instead, at about
    0.5 us a step for few heads and many times a chunk's time for many.

    Values that are not finite make outputs of their own step and of later steps not finite (a
    value's in its own channel), never earlier ones; they may make any element of the state so.

    Parameters
    ----------
    query, key : torch tensor
        CUDA tensors ``[batch, heads, width, time]``, width 1 to 128.
    value : torch tensor
        CUDA tensor ``[batch, heads, width of the value, time]``, width 1 to 128.
    decay : torch tensor
        decay (un-scaled value, 0..4096, not rounded), 1 element or one per head.
    state : torch tensor or None
        state before the first step, ``[batch, heads, width, width of the value]``; ``None`` is zero.
    return_state : bool
        also return the state after the last step.
    precise : bool
        fp32 throughout, forward and backward.

    Returns
    -------
    torch tensor or pair of torch tensors
        output, shaped like ``value`` (and the state).
    """
    if not torch.is_grad_enabled() and _ops.plain_call():
        output, final = _ops.linear_attention_fwd(query, key, value, decay, state, return_state, precise)
    elif torch.is_grad_enabled() and decay.requires_grad:
        raise RuntimeError('linear attention has no gradient for its decay; pass decay.detach()')
    else:
        output, final = _LinearAttention.apply(query, key, value, decay, state, return_state, precise)
    return (output, final) if return_state else output


def step(query, key, value, decay, state):
    """One step of :func:`dynamics` on a kept state, for inference.

    The state is rounded to fp32 at each step: a head that loses less than half a rounding in a step
    (a decay below ``2^-13``) forgets nothing this way.

    Parameters
    ----------
    query, key : torch tensor
        CUDA tensors ``[batch, heads, width]``.
    value : torch tensor
        CUDA tensor ``[batch, heads, width of the value]``.
    decay : torch tensor
        as in :func:`dynamics`.
    state : torch tensor
        contiguous ``[batch, heads, width, width of the value]``; UPDATED IN PLACE.

    Returns
    -------
    torch tensor
        output, shaped like ``value``.
    """
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad
                                    or decay.requires_grad or (state is not None and state.requires_grad)):
        raise RuntimeError('linear attention steps update their state in place and have no gradient; use dynamics(), '
                           'or call step() under torch.no_grad()')
    if not _ops.plain_call():
        _ops.refuse_tangents('a linear attention step', query, key, value, decay, state)
        if torch.jit.is_tracing():
            raise RuntimeError('a linear attention step cannot be traced: traces do not see that its state changes; '
                               'capture it in a CUDA graph')
    return _ops.linear_attention_step(query, key, value, decay, state)


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, decay, state, return_state, precise):
        ctx.set_materialize_grads(False)
        ctx.precise = precise
        output, final = _ops.linear_attention_fwd(query, key, value, decay, state, return_state, precise)
        ctx.save_for_backward(query, key, value, decay, state)
        return output, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_final):
        query, key, value, decay, state = ctx.saved_tensors
        if grad_output is None and grad_final is None:
            return None, None, None, None, None, None, None
        if grad_output is None:
            grad_output = torch.zeros_like(value)
        grad_q, grad_k, grad_v, grad_s = _ops.linear_attention_bwd(
            query, key, value, decay, state, grad_output, grad_final, ctx.needs_input_grad[4], ctx.precise)
        return grad_q, grad_k, grad_v, None, grad_s, None, None
