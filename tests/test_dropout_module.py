"""neuron.Dropout without a GPU: the two device calls are stand-ins that work on CPU tensors."""

import copy

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import lava_dl_b200.slayer as slayer
from lava_dl_b200 import _ops


@pytest.fixture
def on_cpu(monkeypatch):
    def drop(x, p, key, per_step):
        rng = np.random.default_rng([int(k) % 2 ** 64 for k in key])
        shape = x.shape if per_step else x.shape[:-1] + (1,)
        return x * torch.from_numpy(rng.random(shape) >= p).float() / (1 - p)

    def following(state):
        key = state.clone()
        state[1] += 1
        return key

    monkeypatch.setattr(_ops, 'dropout', drop)
    monkeypatch.setattr(_ops, 'dropout_next', following)


def masks(drop, n=1, shape=(8, 16, 3)):
    return [drop(torch.ones(shape)) for _ in range(n)]


@pytest.mark.parametrize('reentrant', [False, True])
def test_recomputed_forward_repeats_its_mask(on_cpu, reentrant):
    drop = slayer.neuron.Dropout(0.5)
    x = torch.ones(8, 16, 3, requires_grad=True)
    first = checkpoint(drop, x, use_reentrant=reentrant)
    second = checkpoint(lambda z: drop(drop(z)), first, use_reentrant=reentrant)
    other = drop(x)
    assert not torch.equal(first, second) and not torch.equal(first, other)
    (g,) = torch.autograd.grad(second.sum(), x) if not reentrant else (backward(second, x),)
    assert torch.equal(g, second.detach())          # three masks' product, the same in both directions


def backward(y, x):
    y.sum().backward()
    return x.grad


def test_masks_follow_torchs_generator(on_cpu):
    drop = slayer.neuron.Dropout(0.5)
    torch.manual_seed(5)
    a, b = masks(drop, 2)
    state = torch.get_rng_state()
    (c,) = masks(drop)
    assert not torch.equal(a, b) and not torch.equal(b, c)
    torch.set_rng_state(state)
    assert torch.equal(masks(drop)[0], c)
    torch.manual_seed(5)
    assert torch.equal(masks(slayer.neuron.Dropout(0.5))[0], a)


@pytest.mark.parametrize('reentrant', [False, True])
def test_seeded_module_refuses_to_be_recomputed(on_cpu, reentrant):
    drop = slayer.neuron.Dropout(0.5, seed=3)
    x = torch.ones(8, 16, 3, requires_grad=True)
    y = checkpoint(drop, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match='recomputed'):
        y.sum().backward()
    y = checkpoint(drop.eval(), x, use_reentrant=reentrant)     # nothing to repeat
    y.sum().backward()


def test_generator_is_no_buffer(on_cpu):
    """DistributedDataParallel broadcasts buffers from rank 0 before each forward."""
    for drop in (slayer.neuron.Dropout(0.5), slayer.neuron.Dropout(0.5, seed=3)):
        assert not list(drop.buffers()) and not drop.state_dict()
    assert slayer.neuron.Dropout(0.5).generator is None
    a, b = masks(drop, 2)
    assert drop.generator.tolist() == [3, 2]
    drop.half()                                     # moves to a device, never to a type
    assert drop.generator.dtype == torch.int64 and drop.generator.tolist() == [3, 2]
    twin = copy.deepcopy(drop)
    assert torch.equal(masks(drop)[0], masks(twin)[0]) and drop.generator is not twin.generator
    drop.generator.copy_(torch.tensor([3, 0]))      # a resumed run sets it back
    assert torch.equal(masks(drop)[0], a) and torch.equal(masks(drop)[0], b)


def test_arguments():
    """The reference's second argument is `inplace`."""
    assert not slayer.neuron.Dropout(0.1, False).per_step
    with pytest.raises(ValueError, match='in place'):
        slayer.neuron.Dropout(0.1, True)
    assert slayer.neuron.Dropout(0.1, per_step=True).per_step
