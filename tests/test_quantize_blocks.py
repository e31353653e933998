"""Blocks swapped for their 8-bit forms, without a GPU: what becomes of the mask."""

import pytest
import torch

import lava_dl_b200.slayer as slayer

CUBA = dict(threshold=1.0, current_decay=0.25, voltage_decay=0.03)


def weights(block, neurons):
    q = block.synapse
    return q.weight_q[:, :neurons].float() * q.weight_scale[:, None]


@pytest.mark.parametrize('weight_norm', [False, True])
@pytest.mark.parametrize('hook', ['grid', None])
def test_mask_is_included(weight_norm, hook):
    torch.manual_seed(1)
    mask = torch.rand(4, 6) < 0.5
    options = {} if hook == 'grid' else dict(pre_hook_fx=None)
    block = slayer.block.cuba.Dense(dict(CUBA), 6, 4, weight_scale=4, weight_norm=weight_norm, mask=mask, **options)
    dense = block.synapse
    if weight_norm:
        norm = dense.weight_v.flatten(1).norm(dim=1).view(-1, 1, 1, 1, 1)
        full = (dense.weight_g * dense.weight_v / norm).detach()
    else:
        full = dense.weight.detach().clone()
    want = full * mask.view(4, 6, 1, 1, 1)
    if block.synapse.pre_hook_fx is not None:
        want = block.synapse.pre_hook_fx(want)
    block.quantize()
    got, want = weights(block, 6), want.reshape(4, 6)
    assert not got[~mask].any() and got[mask].any()
    if hook == 'grid':      # exactly; a norm's rounding may move a weight next to the middle to its neighbour
        allowed = 2 / block.neuron.w_scale * (1 if weight_norm else 0)
    else:                   # half a step of 1/127 of the row's largest, 16 roundings of that largest and its norm
        allowed = want.abs().amax(1, keepdim=True) * (0.5 / 127 + 16 * 2.0 ** -24)
    assert ((got - want).abs() <= allowed).all()
    assert block.mask is None


def test_mask_of_zeros():
    block = slayer.block.cuba.Dense(dict(CUBA), 6, 4, weight_norm=True, mask=torch.zeros(4, 6, dtype=torch.bool))
    assert not block.quantize().synapse.weight_q.any()


def test_refusal_leaves_the_block():
    mask = torch.rand(4, 6) < 0.5
    block = slayer.block.rf.Dense(dict(threshold=1.0, period=10, decay=0.1), 6, 4, mask=mask)
    synapse = block.synapse
    with pytest.raises(NotImplementedError):
        block.quantize()
    assert block.synapse is synapse and block.mask is not None
