"""The sequence operators without gradients, under forward-mode differentiation and under tracing: a tangent is
refused as the other operators refuse it, and a trace calls the operator again."""

import warnings

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import lava_dl_b200.slayer as slayer

pytestmark = pytest.mark.gpu
attention = slayer.neuron.dynamics.linear_attention


def operators():
    """name, function of one tensor, input; step() on a state of its own.  (What a trace meets of its example's own
    memory it takes for the input: the other tensors are others.)"""
    gen = torch.Generator(device='cuda').manual_seed(1)
    x, other = (torch.randn(2, 3, 16, 140, generator=gen, device='cuda') for _ in range(2))
    decay = torch.full((3,), 400.0, device='cuda')
    key = torch.tensor([1, 2], device='cuda')
    layer = slayer.synapse.QuantDense(torch.randint(-128, 128, (5, 48), dtype=torch.int8), torch.ones(5)).cuda()
    y, w = x[..., 0].contiguous(), other[..., 0].contiguous()
    return {
        'dynamics': (lambda z: attention.dynamics(z, other, other, decay), x),
        'dynamics with state': (lambda z: attention.dynamics(other, z, other, decay, None, True)[1], x),
        'step': (lambda z: attention.step(z, w, w, decay, torch.ones(2, 3, 16, 16, device='cuda')), y),
        'dense': (lambda z: layer(z.reshape(2, 48, 140)), x),
        'dropout': (lambda z: slayer.neuron.dropout.dropout(z, 0.5, key), x),
    }


NAMES = ['dynamics', 'dynamics with state', 'step', 'dense', 'dropout']


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('name', NAMES)
def test_tangents_are_refused(cuda, name, grad):
    call, x = operators()[name]
    with torch.set_grad_enabled(grad):
        want = call(x)
        with forward_ad.dual_level():
            assert torch.equal(call(x), want)                    # no tangent, nothing to refuse
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(forward_ad.make_dual(x, torch.ones_like(x)))


def test_step_refuses_a_tangent_before_it_steps(cuda):
    y, decay, state = torch.ones(1, 2, 8, device='cuda'), torch.zeros(2, device='cuda'), torch.ones(1, 2, 8, 8, device='cuda')
    with torch.no_grad(), forward_ad.dual_level():
        for i in range(5):
            args = [y, y, y, decay, state]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match='forward-mode'):
                attention.step(*args)
    assert torch.equal(state, torch.ones_like(state))


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('name', NAMES)
def test_traces_call_the_operator(cuda, name, grad):
    call, x = operators()[name]
    with torch.set_grad_enabled(grad), warnings.catch_warnings():
        warnings.simplefilter('ignore')
        if name == 'step':          # its state changes in place, which a trace does not see
            with pytest.raises(RuntimeError, match='traced'):
                torch.jit.trace(call, (x,), check_trace=False)
            return
        traced = torch.jit.trace(call, (x,), check_trace=False)
        assert torch.equal(traced(x), call(x))
        assert torch.equal(traced(2 * x + 1), call(2 * x + 1))
