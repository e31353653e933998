"""Linear attention where the sizes of a sequence's steps lie far apart: every finite input whose states
fit fp32 has to come out right, at the steps before a large one as well as at those behind it.

Tolerance, per head, for an element against the sum of its own terms' magnitudes.  fp16 pairs keep an
element to 2^-22, and what a product leaves out is 2^-22: a term passes two such products (scores and
read-out, or growth and read-out), 6 * 2^-22 = 12 * 2^-23.  Additions of the tensor cores lose at most
2^-23 each: width for a score or the state's read-out, 128 for the read-out of a chunk or the state's
growth.  Powers of r and weights: eight roundings of 2^-24.  The state takes two roundings of 2^-24 a
chunk, or a step where the walk goes step by step (fewer than 128 steps), and as many where segments are
joined.  Together, with n = T / 128 chunks (steps below 128):  2^-23 (width + 128 + 16 + 2 n + 8).
Unlike a bound for the slowest head this charges a head's memory once a chunk, and no sequence of less than
2^12 steps gets more than 2^-15 of it, so an operand held in one fp16 (2^-12) does not pass.

Floors: 2^-28 of the sums over the largest magnitudes of each step's vectors (``_sequence.py`` has the
derivation), and what an fp32 state below the normal numbers loses, 2^-150 for each of its updates times
the query's magnitudes.
"""

import numpy as np
import pytest
import torch

import _sequence as O
import lava_dl_b200.slayer as slayer
from lava_dl_b200 import _native

pytestmark = pytest.mark.gpu
attention = slayer.neuron.dynamics.linear_attention


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def head_tol(width, T):
    updates = 2 * (T // 128 + 1) if T >= 128 else T
    return 2.0 ** -23 * (width + 128 + 16 + updates + 8)


def state_floor(reader, T):
    """What the states' subnormal roundings can add to an output read by `reader` [n, h, d, T]."""
    return 2.0 ** -150 * (T + 1) * np.abs(reader.astype(np.float64)).sum(axis=2, keepdims=True)


def exponents(kind, rng, shape, span):
    """One exponent for every step, -span .. span (the step's key times value: twice that)."""
    T = shape[-1]
    if kind == 'rising':          # tiny steps, then large ones from the middle of a chunk on
        e = np.where(np.arange(T) % 128 < 64, -span, span) + np.zeros(shape)
    elif kind == 'falling':
        e = np.where(np.arange(T) % 128 < 64, span, -span) + np.zeros(shape)
    elif kind == 'fading':        # a signal that vanishes over the whole axis
        e = np.linspace(span, -span, T) + np.zeros(shape)
    elif kind == 'growing':
        e = np.linspace(-span, span, T) + np.zeros(shape)
    elif kind == 'last':          # one large step at the end of a chunk
        e = np.where(np.arange(T) % 128 == 127, span, -span) + np.zeros(shape)
    else:
        e = rng.integers(-span, span + 1, size=shape).astype(float)
    return np.rint(e)


def far_apart(seed, n, h, dk, dv, T, kind, span, decay, back=False):
    """Key and value (or, for the walks back in time, query and output gradient) spread by 2^span each way; the
    readers' exponents bring the outputs (or gradients of key and value) back to where fp32 holds them."""
    rng = np.random.default_rng(seed)
    q, k, v, go = (rng.normal(size=(n, h, d, T)) for d in (dk, dk, dv, dv))
    e = exponents(kind, rng, (n, h, 1, T), span)
    r = 1.0 - np.asarray(decay, dtype=np.float64).reshape(1, -1, 1) / 4096.0
    with np.errstate(divide='ignore'):
        log_r = np.maximum(np.log2(r), -1e4)
    size = np.full((n, h, 1), -1e9)
    reach = np.empty((n, h, 1, T))
    for t in (reversed(range(T)) if back else range(T)):      # the exponent of the state's largest part
        size = np.maximum(size + log_r, 2 * e[..., t])
        reach[..., t] = size
    reach = np.clip(np.rint(reach), -110, 110)
    read = np.exp2(-reach)
    part = np.exp2(e)
    if back:
        q, go, k, v = q * part, go * part, k * read, v * read
    else:
        k, v, q, go = k * part, v * part, q * read, go * read
    return [a.astype(np.float32) for a in (q, k, v, go)], np.asarray(decay, dtype=np.float32)


def check_forward(q, k, v, decay):
    T = q.shape[-1]
    with torch.no_grad():
        out, final = attention.dynamics(dev(q), dev(k), dev(v), dev(decay), return_state=True)
    want, ws = O.attention(q, k, v, decay)
    size, ss = O.attention(np.abs(q), np.abs(k), np.abs(v), decay)
    floor, fs = O.attention_floor(q, k, v, decay)
    tol = head_tol(q.shape[2], T)
    O.assert_sum_close(out, want, size, tol, 'output', floor + state_floor(q, T))
    O.assert_sum_close(final, ws, ss, tol, 'state', fs)
    assert _native.device_status() == 0


def check_backward(q, k, v, go, decay, which):
    """`which`: the gradients whose states fit fp32."""
    T = q.shape[-1]
    leaves = [dev(a).requires_grad_() for a in (q, k, v)]
    grads = torch.autograd.grad(attention.dynamics(*leaves, dev(decay)), leaves, dev(go))
    want = O.attention_grads(q, k, v, decay, None, go, None)
    size = O.attention_grads(np.abs(q), np.abs(k), np.abs(v), decay, None, np.abs(go), None)
    floor = O.attention_grads_floor(q, k, v, decay, None, go, None)
    tol = head_tol(max(q.shape[2], v.shape[2]), T)
    for i in which:
        name, reader = (('query', go), ('key', v), ('value', k))[i]
        O.assert_sum_close(grads[i], want[i], size[i], tol, name, floor[i] + state_floor(reader, T))
    assert _native.device_status() == 0


SLOW = [2.048, 40.96, 409.6]             # memories of 2000, 100 and 10 steps
KINDS = ['rising', 'falling', 'fading', 'growing', 'last', 'random']
WIDTHS = [(64, 64, 300), (40, 72, 277), (128, 96, 260), (16, 16, 128), (64, 64, 1284)]


@pytest.mark.parametrize('span', [20, 33, 56])
@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('dk, dv, T', WIDTHS)
def test_forward_of_steps_far_apart(cuda, dk, dv, T, kind, span):
    (q, k, v, _), decay = far_apart(21, 2, 3, dk, dv, T, kind, span, SLOW)
    check_forward(q, k, v, decay)


@pytest.mark.parametrize('span', [33, 56])
@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('dk, dv, T', WIDTHS)
def test_backward_of_steps_far_apart(cuda, dk, dv, T, kind, span):
    for back in (False, True):
        (q, k, v, go), decay = far_apart(22, 2, 3, dk, dv, T, kind, span, SLOW, back)
        check_backward(q, k, v, go, decay, (1, 2) if back else (0,))


FAST = [2048.0, 3300.0, 4055.0, 4095.9, 4096.0]      # r of 0.5, 0.19, 0.01, 2^-15.3 and 0


@pytest.mark.parametrize('span', [33, 56])
@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('dk, dv, T', [(64, 64, 300), (40, 72, 277), (128, 96, 260)])
def test_heads_of_short_memory(cuda, dk, dv, T, kind, span):
    """Powers of r below any float: what decays by them was large enough to be seen all the same."""
    (q, k, v, _), decay = far_apart(23, 1, 5, dk, dv, T, kind, span, FAST)
    check_forward(q, k, v, decay)
    for back in (False, True):
        (q, k, v, go), decay = far_apart(24, 1, 5, dk, dv, T, kind, span, FAST, back)
        check_backward(q, k, v, go, decay, (1, 2) if back else (0,))


@pytest.mark.parametrize('dk, dv, T', [(64, 64, 300), (64, 40, 301), (128, 128, 260), (8, 8, 4096)])
def test_large_states_that_fade(cuda, dk, dv, T):
    """Nothing but a state from before, down to where fp32 ends; in the longest, cut into segments."""
    rng = np.random.default_rng(25)
    decay = np.array([2048.0, 1500.0, 3300.0, 300.0], np.float32)
    r = 1.0 - decay.astype(np.float64).reshape(1, 4, 1, 1) / 4096.0
    s = (rng.normal(size=(1, 4, dk, dv)) * 2.0 ** 120).astype(np.float32)
    gone = 120 + np.log2(r) * np.arange(1, T + 1)                   # exponent of the state
    q = (rng.normal(size=(1, 4, dk, T)) * np.exp2(-np.clip(gone, -110, 120))).astype(np.float32)
    zero_k, zero_v = np.zeros((1, 4, dk, T), np.float32), np.zeros((1, 4, dv, T), np.float32)
    with torch.no_grad():
        out, final = attention.dynamics(*(dev(a) for a in (q, zero_k, zero_v, decay, s)), return_state=True)
    want, ws = O.attention(q, zero_k, zero_v, decay, s)
    size, ss = O.attention(np.abs(q), zero_k, zero_v, decay, np.abs(s))
    floor, _ = O.attention_floor(q, zero_k, zero_v, decay, s)
    assert (np.abs(want[:, :, :, 100]) > 1e-3).any()                # well inside fp32
    O.assert_sum_close(out, want, size, head_tol(dk, T), 'output', floor + state_floor(q, T))
    O.assert_sum_close(final, ws, ss, head_tol(dk, T), 'state')


@pytest.mark.parametrize('n, dk, dv, T', [(50, 16, 20, 260), (41, 24, 70, 131), (33, 70, 40, 128)])
def test_short_memories_side_by_side(cuda, n, dk, dv, T):
    """More heads than multiprocessors: each takes slow and fast ones in turn."""
    (q, k, v, go), decay = far_apart(28, n, 9, dk, dv, T, 'random', 40, FAST + SLOW + [2.048])
    check_forward(q, k, v, decay)
    check_backward(q, k, v, go, decay, (0,))
    (q, k, v, go), decay = far_apart(29, n, 9, dk, dv, T, 'random', 40, FAST + SLOW + [2.048], True)
    check_backward(q, k, v, go, decay, (1, 2))


def test_decay_that_is_not_a_number(cuda):
    """Nothing finite comes out of it, whichever kernel takes the length; other heads do not notice."""
    for T in (20, 300):
        (q, k, v, _), decay = far_apart(26, 2, 3, 16, 24, T, 'random', 3, SLOW)
        with torch.no_grad():
            want = attention.dynamics(dev(q), dev(k), dev(v), dev(decay))
            decay[1] = np.nan
            got = attention.dynamics(dev(q), dev(k), dev(v), dev(decay))
        assert torch.isnan(got[:, 1]).all()
        assert torch.equal(got[:, ::2], want[:, ::2])


@pytest.mark.parametrize('dk', [64, 128])
def test_zero_read_out_of_a_large_state(cuda, dk):
    """A query that meets nothing of a state of the largest numbers reads zero, at any size of its own."""
    q, s = np.zeros((1, 1, dk, 256), np.float32), np.zeros((1, 1, dk, 64), np.float32)
    q[:, :, 0], s[:, :, 1] = 3e38, 3e38
    zero = np.zeros_like(q)
    with torch.no_grad():
        out = attention.dynamics(dev(q), dev(zero), dev(zero[:, :, :64]), dev(np.array([2.048], np.float32)), dev(s))
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize('tiny', [1e-18, 2.0 ** -64, 2.0 ** -65, 1e-20, 1e-22])
@pytest.mark.parametrize('query', [1.0, 1e10])
@pytest.mark.parametrize('dk, dv', [(64, 64), (128, 64)])
def test_tiny_steps_before_a_large_one(cuda, dk, dv, query, tiny):
    """A later step of ordinary size leaves the outputs before it as they are."""
    shape = (1, 1, dk, 256)
    q, k, v = np.full(shape, query, np.float32), np.full(shape, tiny, np.float32), np.full((1, 1, dv, 256), tiny, np.float32)
    k[..., 64:128] = v[..., 64:128] = 1.0
    check_forward(q, k, v, np.array([2.048], np.float32))


def test_single_steps_of_a_slow_head(cuda):
    """Thousands of steps on a kept state decay by r itself, not by r rounded to a float.

    A step rounds an element once, by a relative error of -2^-24 .. 2^-24 (its deviation at most 2^-24 / sqrt 3),
    one step's independent of the next one's as the mantissas are.  Elements are not independent: a step takes a
    mantissa of 2^23 .. 2^24 units down by 2^23 (1 - r) units or more, so that is the least number of different
    courses that mantissas can take (204 for a decay of 0.1), and elements on one course go on alike.  The mean over
    C = 2^23 (1 - r) courses after N steps deviates by 2^-24 sqrt(N / 3 C); six of those are allowed.  r rounded to
    a float moves every element by N times what the rounding loses, the same way."""
    steps, width = 4000, 64
    decay = np.array([0.05, 0.1, 0.3], np.float32)
    r = 1.0 - decay.astype(np.float64) / 4096.0
    lost = np.abs(r - r.astype(np.float32))
    courses = 2.0 ** 23 * (1.0 - r)
    assert (courses < width ** 2).all()
    tol = 6 * 2.0 ** -24 * np.sqrt(steps / 3 / courses)
    assert (steps * lost > 30 * tol).all()
    rng = np.random.default_rng(27)
    start = rng.normal(size=(1, 3, width, width)).astype(np.float32)
    state, zero, d = dev(start), torch.zeros(1, 3, width, device='cuda'), dev(decay)
    for _ in range(steps):
        attention.step(zero, zero, zero, d, state)
    error = (state.cpu().numpy() / (start.astype(np.float64) * (r ** steps).reshape(1, 3, 1, 1)) - 1.0).mean(axis=(0, 2, 3))
    assert (np.abs(error) <= tol).all(), error / tol
