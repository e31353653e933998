"""neuron.Dropout on the GPU: recomputed segments, captured steps, torch's generator."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import lava_dl_b200.slayer as slayer
from lava_dl_b200 import _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('per_step', [False, True])
@pytest.mark.parametrize('reentrant', [False, True])
def test_recomputed_forward_repeats_its_mask(cuda, reentrant, per_step):
    drop = slayer.neuron.Dropout(0.5, per_step=per_step)
    x = torch.ones(4, 50, 20, device='cuda', requires_grad=True)
    y = checkpoint(drop, x, use_reentrant=reentrant)
    z = checkpoint(lambda a: drop(drop(a)), y, use_reentrant=reentrant)
    drop(x)
    z.sum().backward()
    assert torch.equal(x.grad, z.detach()) and 0 < float((z > 0).float().mean()) < 0.5


def test_recomputed_block(cuda):
    """A neuron's own dropout in a checkpointed block: the gradients of the block that keeps its activations."""
    params = dict(threshold=0.5, current_decay=0.25, voltage_decay=0.03, dropout=slayer.neuron.Dropout(0.3))
    torch.manual_seed(0)
    block = slayer.block.cuba.Dense(params, 24, 32, weight_scale=4).cuda()
    x = (torch.rand(3, 24, 100, device='cuda') < 0.3).float()
    grads = []
    for run in (block, lambda a: checkpoint(block, a, use_reentrant=False)):
        torch.manual_seed(7)
        y = run(x)
        grads.append((y.detach(), torch.autograd.grad((y * torch.arange(100, device='cuda')).sum(), block.synapse.weight)[0]))
    assert torch.equal(grads[0][0], grads[1][0]) and float(grads[0][1].abs().max()) > 0
    # the synapse's own gradient is a library sum whose order may differ: 300 half steps of 2^-24 of the magnitudes
    assert torch.allclose(grads[0][1], grads[1][1], rtol=1e-4, atol=1e-4 * float(grads[0][1].abs().max()))


def test_masks_follow_torchs_generator(cuda):
    drop, x = slayer.neuron.Dropout(0.5), torch.ones(4, 50, 20, device='cuda')
    torch.manual_seed(5)
    a, state, b = drop(x), torch.cuda.get_rng_state(), drop(x)
    assert not torch.equal(a, b)
    torch.cuda.set_rng_state(state)
    assert torch.equal(drop(x), b)


def test_captured_calls_use_new_masks(cuda):
    drop, x = slayer.neuron.Dropout(0.5), torch.ones(4, 50, 20, device='cuda', requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(drop(x).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x)
        (g,) = torch.autograd.grad(y.sum(), x)
    seen = []
    for _ in range(3):
        graph.replay()
        assert torch.equal(y, g)
        seen.append(y.detach().clone())
    assert not any(torch.equal(a, b) for a, b in zip(seen, seen[1:]))


def test_seeded_module_refuses_to_be_recomputed(cuda):
    drop = slayer.neuron.Dropout(0.5, seed=3)
    x = torch.ones(4, 50, 20, device='cuda', requires_grad=True)
    y = checkpoint(drop, x, use_reentrant=False)
    with pytest.raises(RuntimeError, match='recomputed'):
        y.sum().backward()


def test_streams_get_keys_of_their_own(cuda):
    """Branches of a graph run side by side, whatever time the host takes between launches."""
    state, streams, keys = torch.tensor([9, 100], device='cuda'), [torch.cuda.Stream() for _ in range(8)], []
    _ops.dropout_next(state.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                keys += [_ops.dropout_next(state) for _ in range(50)]
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        keys = torch.stack(keys)
    for i in range(5):
        graph.replay()
        assert state.tolist() == [9, 100 + 400 * (i + 1)] and bool((keys[:, 0] == 9).all())
        assert sorted(keys[:, 1].tolist()) == list(range(100 + 400 * i, 500 + 400 * i))
