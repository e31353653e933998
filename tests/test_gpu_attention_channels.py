"""Linear attention whose channels differ in size: chunks with one exponent for each step's vector, and the walk in
fp32 that a caller can ask for instead."""

import numpy as np
import pytest
import torch

import _sequence as O
import lava_dl_b200.slayer as slayer
from lava_dl_b200 import _native
from test_gpu_attention_range import dev, head_tol

pytestmark = pytest.mark.gpu
attention = slayer.neuron.dynamics.linear_attention
SHAPES = [(2, 3, 64, 64, 300), (1, 2, 40, 72, 277), (1, 2, 128, 96, 260), (2, 2, 16, 24, 40), (3, 1, 70, 128, 1284)]


def make(shape, spread):
    """Channels of query and key with exponents against one another, so that small ones of each count; channels of
    value and output gradient with exponents of their own."""
    n, h, dk, dv, T = shape
    rng = np.random.default_rng(31)
    q, k, v, go = (rng.normal(size=(n, h, d, T)) for d in (dk, dk, dv, dv))
    e, f, g = (rng.integers(-spread, spread + 1, size=(n, h, d, 1)) for d in (dk, dv, dv))
    arrays = q * np.exp2(e), k * np.exp2(-e), v * np.exp2(f), go * np.exp2(g)
    s = rng.normal(size=(n, h, dk, dv)) * np.exp2(-e + f.reshape(n, h, 1, dv))
    decay = 4096 * np.geomspace(0.3, 0.001, h)
    return [np.asarray(a, dtype=np.float32) for a in (*arrays, decay, s)]


def fp32_tol(width, T):
    """Step by step: two roundings of 2^-24 a step for the state, one for a product, `width` additions and 8 more to
    join them (a term may be as old as the sequence is long)."""
    return 2.0 ** -24 * (2 * T + width + 12)


def check(shape, spread, precise):
    q, k, v, go, decay, s = make(shape, spread)
    T, width = shape[4], max(shape[2:4])
    leaves = [dev(a).requires_grad_() for a in (q, k, v, s)]
    options = dict(precise=True) if precise else {}
    out, final = attention.dynamics(*leaves[:3], dev(decay), leaves[3], return_state=True, **options)
    grads = torch.autograd.grad(out, leaves, dev(go))
    want = O.attention(q, k, v, decay, s) + O.attention_grads(q, k, v, decay, s, go, None)
    mags = [np.abs(a) for a in (q, k, v, s, go)]
    size = O.attention(*mags[:3], decay, mags[3]) + O.attention_grads(*mags[:3], decay, mags[3], mags[4], None)
    if precise:
        tol, floor = fp32_tol(width, T), [0.0] * 6
    else:
        tol = head_tol(width, T)
        floor = (*O.attention_floor(q, k, v, decay, s), *O.attention_grads_floor(q, k, v, decay, s, go, None))
    names = ('output', 'state', 'query', 'key', 'value', 'start')
    for name, g, w, z, f in zip(names, (out.detach(), final.detach(), *grads), want, size, floor):
        O.assert_sum_close(g, w, z, tol, name, f)
    with torch.no_grad():
        again, state = attention.dynamics(*(a.detach() for a in leaves[:3]), dev(decay), leaves[3].detach(), True, **options)
    assert torch.equal(again, out) and torch.equal(state, final)
    assert _native.device_status() == 0


@pytest.mark.parametrize('spread', [2, 6])
@pytest.mark.parametrize('shape', SHAPES)
def test_channels_of_different_sizes(cuda, shape, spread):
    check(shape, spread, False)


@pytest.mark.parametrize('spread', [0, 6, 20])
@pytest.mark.parametrize('shape', SHAPES)
def test_fp32_when_asked_for(cuda, shape, spread):
    check(shape, spread, True)


def test_fp32_of_nothing(cuda):
    z, s = torch.zeros(2, 3, 8, 0, device='cuda'), torch.randn(2, 3, 8, 8, device='cuda')
    out, final = attention.dynamics(z, z, z, torch.zeros(3, device='cuda'), s, return_state=True, precise=True)
    assert out.shape == z.shape and torch.equal(final, s)
    x = torch.zeros(0, 3, 8, 5, device='cuda')
    assert attention.dynamics(x, x, x, torch.zeros(1, device='cuda'), precise=True).shape == x.shape
