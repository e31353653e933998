"""Linear attention, 8-bit dense synapse and dropout on the GPU against their 64-bit definitions."""

import numpy as np
import pytest
import torch

import _sequence as O
import lava_dl_b200.slayer as slayer
from _util import assert_exact
from lava_dl_b200 import _native

pytestmark = pytest.mark.gpu
attention = slayer.neuron.dynamics.linear_attention
dropout = slayer.neuron.dropout.dropout


def make(seed, n, h, dk, dv, T, spikes=False, state=True, decays=None):
    rng = np.random.default_rng(seed)
    if spikes:
        q, k, v = ((rng.random((n, h, d, T)) < 0.2) for d in (dk, dk, dv))
    else:
        q, k, v = (rng.normal(size=(n, h, d, T)) for d in (dk, dk, dv))
    s = rng.normal(size=(n, h, dk, dv)) if state else None
    decay = 4096 * np.geomspace(0.5, 0.001, h) if decays is None else np.asarray(decays)
    f = [None if a is None else np.asarray(a, dtype=np.float32) for a in (q, k, v, decay, s)]
    return f, rng


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check_walk(arrays, out, final, T):
    q, k, v, decay, s = arrays
    tol = O.attention_tol(q.shape[2], T, decay)
    want, ws = O.attention(q, k, v, decay, s)
    size, ss = O.attention(*(np.abs(a) for a in (q, k, v)), decay, None if s is None else np.abs(s))
    fo, fs = O.attention_floor(*arrays)
    O.assert_sum_close(out, want, size, tol, 'output', fo)
    if final is not None:
        O.assert_sum_close(final, ws, ss, tol, 'state', fs)


SHAPES = [   # n, h, dk, dv, T
    (1, 1, 1, 1, 1), (2, 3, 5, 7, 2), (1, 2, 64, 64, 31), (2, 2, 64, 64, 128), (1, 2, 64, 64, 129), (3, 2, 16, 48, 300),
    (1, 3, 40, 72, 277), (2, 1, 128, 128, 257), (1, 2, 65, 33, 130), (1, 1, 128, 1, 200), (1, 1, 1, 128, 200),
    (2, 2, 64, 64, 1000), (5, 4, 63, 64, 515), (1, 2, 100, 96, 2049),
    (1, 2, 128, 96, 260), (2, 1, 70, 128, 1284), (1, 3, 64, 64, 48), (3, 1, 64, 20, 47), (1, 2, 9, 33, 124)]


@pytest.mark.parametrize('spikes', [False, True])
@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('shape', SHAPES)
def test_attention_forward(cuda, shape, state, spikes):
    arrays, _ = make(1, *shape, spikes=spikes, state=state)
    with torch.no_grad():
        out, final = attention.dynamics(*(dev(a) for a in arrays), return_state=True)
    check_walk(arrays, out, final, shape[-1])
    assert _native.device_status() == 0


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('ends', [False, True])
def test_attention_backward(cuda, shape, ends):
    arrays, rng = make(2, *shape, state=ends)
    q, k, v, decay, s = arrays
    go = rng.normal(size=v.shape).astype(np.float32)
    gf = rng.normal(size=(shape[0], shape[1], shape[2], shape[3])).astype(np.float32) if ends else None
    leaves = [dev(a).requires_grad_() for a in ((q, k, v, s) if ends else (q, k, v))]
    out = attention.dynamics(*leaves[:3], dev(decay), leaves[3] if ends else None, return_state=ends)
    if ends:
        grads = torch.autograd.grad(out, leaves, (dev(go), dev(gf)))
    else:
        grads = torch.autograd.grad(out, leaves, dev(go))
    want = O.attention_grads(q, k, v, decay, s, go, gf)
    size = O.attention_grads(*(np.abs(a) for a in (q, k, v)), decay, None if s is None else np.abs(s), np.abs(go),
                             None if gf is None else np.abs(gf))
    tol = O.attention_tol(max(shape[2:4]), shape[4], decay)
    floor = O.attention_grads_floor(q, k, v, decay, s, go, gf)
    for name, g, w, z, f in zip(('query', 'key', 'value', 'state'), grads, want, size, floor):
        O.assert_sum_close(g, w, z, tol, name, f)


def test_attention_gradient_against_differences(cuda):
    """Linear in each input: the difference over any step is the gradient, up to the two outputs' roundings."""
    arrays, rng = make(3, 2, 2, 24, 40, 200)
    leaves = [dev(arrays[i]).requires_grad_() for i in (0, 1, 2, 4)]
    decay = dev(arrays[3])
    go, gf = dev(rng.normal(size=arrays[2].shape).astype(np.float32)), dev(rng.normal(size=(2, 2, 24, 40)).astype(np.float32))

    def loss(a):
        out, final = attention.dynamics(a[0], a[1], a[2], decay, a[3], return_state=True)
        return (out.double() * go).sum() + (final.double() * gf).sum()

    base = loss(leaves)
    grads = torch.autograd.grad(base, leaves)
    tol = O.attention_tol(40, 200, arrays[3])
    for i, g in enumerate(grads):
        u = torch.from_numpy(rng.normal(size=tuple(g.shape)).astype(np.float32)).cuda()
        moved = [a.detach() + u if j == i else a.detach() for j, a in enumerate(leaves)]
        with torch.no_grad():
            mags = [a.detach().abs() for a in leaves]
            mags[i] = mags[i] + u.abs()
            out, final = attention.dynamics(mags[0], mags[1], mags[2], decay, mags[3], return_state=True)
            bound = 4 * tol * float((out.double() * go.abs()).sum() + (final.double() * gf.abs()).sum())
            assert abs(float(loss(moved) - base) - float((g.double() * u).sum())) <= bound


@pytest.mark.parametrize('decay', [[0.0], [4096.0], [4095.9], [1e-3], [0.0, 4096.0]])
def test_attention_decays(cuda, decay):
    """Nothing forgotten, everything forgotten, one for all heads."""
    arrays, rng = make(4, 2, 2, 16, 24, 400, decays=decay)
    with torch.no_grad():
        out, final = attention.dynamics(*(dev(a) for a in arrays), return_state=True)
    check_walk(arrays, out, final, 400)
    leaves = [dev(a).requires_grad_() for a in arrays[:3]]
    go = rng.normal(size=arrays[2].shape).astype(np.float32)
    grads = torch.autograd.grad(attention.dynamics(*leaves, dev(arrays[3])), leaves, dev(go))
    want = O.attention_grads(*arrays[:4], None, go, None)
    size = O.attention_grads(*(np.abs(a) for a in arrays[:3]), arrays[3], None, np.abs(go), None)
    floor = O.attention_grads_floor(*arrays[:4], None, go, None)
    for g, w, z, f in zip(grads, want, size, floor):
        O.assert_sum_close(g, w, z, O.attention_tol(24, 400, arrays[3]), '', f)


def test_attention_of_sizes_far_apart(cuda):
    """Steps and channels of very different magnitudes keep their relative accuracy: the error of an
    output is measured against its own terms only."""
    arrays, rng = make(5, 2, 2, 32, 32, 300)
    q, k, v, decay, s = arrays
    for a in (q, k, v):
        a *= np.exp2(rng.integers(-30, 30, size=(2, 2, 1, 300))).astype(np.float32)
    with torch.no_grad():
        out = attention.dynamics(*(dev(a) for a in arrays))
    check_walk(arrays, out, None, 300)


MANY = [   # more heads than multiprocessors, several to each: n, h, dk, dv, T
    (50, 16, 16, 20, 260), (41, 19, 24, 64, 131), (5, 80, 70, 128, 130), (31, 13, 64, 100, 129), (4, 13, 16, 12, 4224),
    (90, 9, 8, 12, 128), (15, 10, 8, 12, 2048), (5, 10, 16, 12, 2000)]


@pytest.mark.parametrize('shape', MANY)
def test_attention_of_many_heads(cuda, shape):
    """Heads that a multiprocessor takes one after the other: values, gradients, the same bits again."""
    arrays, rng = make(17, *shape)
    q, k, v, decay, s = arrays
    leaves = [dev(a).requires_grad_() for a in (q, k, v, s)]
    out, final = attention.dynamics(*leaves[:3], dev(decay), leaves[3], return_state=True)
    check_walk(arrays, out.detach(), final.detach(), shape[-1])
    go = rng.normal(size=v.shape).astype(np.float32)
    gf = rng.normal(size=s.shape).astype(np.float32)
    grads = torch.autograd.grad((out, final), leaves, (dev(go), dev(gf)), retain_graph=True)
    want = O.attention_grads(q, k, v, decay, s, go, gf)
    size = O.attention_grads(*(np.abs(a) for a in (q, k, v)), decay, np.abs(s), np.abs(go), np.abs(gf))
    tol = O.attention_tol(max(shape[2:4]), shape[4], decay)
    floor = O.attention_grads_floor(q, k, v, decay, s, go, gf)
    for name, g, w, z, f in zip(('query', 'key', 'value', 'state'), grads, want, size, floor):
        O.assert_sum_close(g, w, z, tol, name, f)
    for a, b in zip(grads, torch.autograd.grad((out, final), leaves, (dev(go), dev(gf)))):
        assert torch.equal(a, b)
    assert _native.device_status() == 0


@pytest.mark.parametrize('shape', [(50, 16, 16, 20, 260), (41, 19, 24, 64, 131), (5, 80, 70, 128, 130),
                                   (15, 10, 8, 12, 2048)])
def test_attention_spoilt_heads_among_many(cuda, shape):
    """What is not finite in some heads leaves every bit of the others as it was."""
    arrays, rng = make(18, *shape)
    with torch.no_grad():
        want, ws = attention.dynamics(*(dev(a) for a in arrays), return_state=True)
        heads = shape[0] * shape[1]
        spoilt = np.zeros(heads, dtype=bool)
        spoilt[rng.choice(heads, heads // 5, replace=False)] = True
        spoilt = spoilt.reshape(shape[:2])
        for i, a in enumerate(arrays[:3]):
            at = np.argwhere(spoilt)[i::3]
            a[at[:, 0], at[:, 1], 3, 100] = (np.nan, np.inf, -np.inf)[i]
        got, gs = attention.dynamics(*(dev(a) for a in arrays), return_state=True)
    keep = dev(~spoilt)
    assert torch.equal(got[keep], want[keep]) and torch.equal(gs[keep], ws[keep])
    assert torch.equal(got[..., :100], want[..., :100])
    assert (~torch.isfinite(got[~keep][..., 100])).any(-1).all()


@pytest.mark.parametrize('bad', [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize('which', [0, 1, 2])
def test_attention_values_that_are_not_finite(cuda, which, bad):
    """They reach their own and later steps (a query's: its own step; a value's: its own channel), no other."""
    arrays, _ = make(6, 1, 2, 48, 40, 300)
    clean = [dev(a) for a in arrays]
    with torch.no_grad():
        want = attention.dynamics(*clean)
        arrays[which][0, 1, 11, 170] = bad
        got = attention.dynamics(*(dev(a) for a in arrays))
    finite = torch.isfinite(got)
    expect = torch.ones_like(finite)
    if which == 0:
        expect[0, 1, :, 170] = False
    elif which == 1:
        expect[0, 1, :, 170:] = False
    else:
        expect[0, 1, 11, 170:] = False
    assert torch.equal(finite, expect)
    tol = O.attention_tol(48, 300, arrays[3])
    size, _ = O.attention(*(np.abs(a.cpu().numpy()) for a in clean[:3]), arrays[3], np.abs(arrays[4]))
    diff = (got - want).abs().double().cpu().numpy()
    mask = expect.cpu().numpy()
    floor, _ = O.attention_floor(*(a.cpu().numpy() for a in clean))
    assert (diff[mask] <= 2 * (tol * size + floor)[mask]).all()


def test_attention_in_pieces_and_steps(cuda):
    """A sequence in pieces, its state handed on, and step by step."""
    arrays, _ = make(7, 3, 4, 64, 64, 300)
    q, k, v, decay, s = (dev(a) for a in arrays)
    with torch.no_grad():
        state, outs = s, []
        for a, b in ((0, 1), (1, 130), (130, 131), (131, 300)):
            o, state = attention.dynamics(q[..., a:b], k[..., a:b], v[..., a:b], decay, state, return_state=True)
            outs.append(o)
        check_walk(arrays, torch.cat(outs, -1), state, 300)
        state, outs = s.clone(), []
        for t in range(300):
            outs.append(attention.step(q[..., t], k[..., t], v[..., t], decay, state))
        check_walk(arrays, torch.stack(outs, -1), state, 300)


@pytest.mark.parametrize('shape', [(1, 1, 1, 1), (3, 5, 7, 9), (2, 4, 64, 64), (2, 2, 128, 128), (1, 3, 33, 100),
                                   (1, 2, 128, 2), (1, 2, 2, 127), (40, 16, 64, 64)])
def test_attention_step(cuda, shape):
    arrays, _ = make(8, *shape, 1)
    q, k, v, decay, s = (dev(a) for a in arrays)
    kept = s.clone()
    out = attention.step(q[..., 0], k[..., 0], v[..., 0], decay, kept)
    check_walk(arrays, out.unsqueeze(-1), kept, 1)


def test_attention_step_replayed(cuda):
    """A captured step moves the state on at each replay."""
    arrays, _ = make(9, 2, 3, 32, 32, 1)
    q, k, v, decay, s = (dev(a) for a in arrays)
    q, k, v = q[..., 0].contiguous(), k[..., 0].contiguous(), v[..., 0].contiguous()
    kept, eager = s.clone(), s.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention.step(q, k, v, decay, kept.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.step(q, k, v, decay, kept)
    for _ in range(3):
        graph.replay()
        want = attention.step(q, k, v, decay, eager)
        assert torch.equal(out, want) and torch.equal(kept, eager)


def test_attention_strides_streams_and_repeats(cuda):
    """Views, shared heads, another stream; the same call gives the same bits."""
    arrays, rng = make(10, 2, 4, 32, 64, 260)
    q, k, v, decay, s = (dev(a) for a in arrays)
    with torch.no_grad():
        want = attention.dynamics(q, k, v, decay, s)
        other = torch.empty(2, 4, 260, 32, device='cuda').transpose(2, 3).copy_(q)
        wide = torch.zeros(2, 4, 64, 263, device='cuda')[..., 2:262].copy_(v)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = attention.dynamics(other, k, wide, decay, s)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want, got)
        assert torch.equal(want, attention.dynamics(q, k, v, decay, s))
    shared = k[:, :1].clone().requires_grad_()
    go = dev(rng.normal(size=arrays[2].shape).astype(np.float32))
    out = attention.dynamics(q, shared.expand(-1, 4, -1, -1), v, decay, s)
    (g,) = torch.autograd.grad(out, shared, go)
    full = k[:, :1].expand(-1, 4, -1, -1).clone().requires_grad_()
    (gf,) = torch.autograd.grad(attention.dynamics(q, full, v, decay, s), full, go)
    assert torch.equal(g, gf.sum(1, keepdim=True))
    assert torch.equal(*(torch.autograd.grad(attention.dynamics(q, full, v, decay, s), full, go)[0] for _ in range(2)))


@pytest.mark.parametrize('shape', [(2, 2, 64, 64, 300), (1, 2, 128, 72, 200), (1, 2, 16, 16, 20)])
def test_attention_unaligned(cuda, shape):
    """Contiguous tensors that start between 16-byte boundaries: other loads, the same values."""
    arrays, rng = make(15, *shape)
    aligned = [dev(a) for a in arrays]

    def moved(t):
        flat = torch.empty(t.numel() + 1, device='cuda')
        return flat[1:].view(t.shape).copy_(t)

    odd = [moved(t) for t in aligned]
    with torch.no_grad():
        for a, b in zip(attention.dynamics(*aligned, return_state=True), attention.dynamics(*odd, return_state=True)):
            assert torch.equal(a, b)
    go = moved(dev(rng.normal(size=arrays[2].shape).astype(np.float32)))
    grads = []
    for args in (aligned, odd):
        leaves = [t.detach().requires_grad_() for t in args[:3]]
        grads.append(torch.autograd.grad(attention.dynamics(*leaves, args[3], args[4]), leaves, go))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    q, k, v = (moved(t[..., 0].contiguous()) for t in aligned[:3])
    kept, want = moved(aligned[4]), aligned[4].clone()
    assert torch.equal(attention.step(q, k, v, odd[3], kept), attention.step(q, k, v, aligned[3], want))
    assert torch.equal(kept, want)


def test_attention_empty(cuda):
    z = torch.zeros(2, 3, 8, 0, device='cuda')
    s = torch.randn(2, 3, 8, 8, device='cuda')
    out, final = attention.dynamics(z, z, z, torch.zeros(3, device='cuda'), s, return_state=True)
    assert out.shape == z.shape and torch.equal(final, s)
    x = torch.zeros(0, 3, 8, 5, device='cuda')
    assert attention.dynamics(x, x, x, torch.zeros(1, device='cuda')).shape == x.shape
    x = torch.zeros(2, 3, 8, 5, device='cuda', requires_grad=True)
    (g,) = torch.autograd.grad(attention.dynamics(x, x, x, torch.zeros(1, device='cuda')).sum(), x)
    assert torch.equal(g, torch.zeros_like(g))


def test_attention_refusals(cuda):
    x = torch.zeros(2, 3, 8, 5, device='cuda')
    d = torch.zeros(3, device='cuda')
    s = torch.zeros(2, 3, 8, 8, device='cuda')
    for args in ((x[0], x[0], x[0], d), (x, x[..., :4], x, d), (x, x, x[..., :4], d), (x, x, x[:1], d), (x, x, x, d[:2]),
                 (x, x, x, d, s[:1]), (x, x, torch.zeros(2, 3, 129, 5, device='cuda'), d)):
        with pytest.raises(ValueError):
            attention.dynamics(*args)
    with pytest.raises(TypeError):
        attention.dynamics(x.double(), x, x, d)
    with pytest.raises(RuntimeError):
        attention.dynamics(x, x, x, d.cpu())
    y = x[..., 0]
    with pytest.raises(ValueError, match='contiguous'):
        attention.step(y, y, y, d, s.transpose(2, 3))
    with pytest.raises(ValueError, match='state'):
        attention.step(y, y, y, d, None)
    g = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(attention.dynamics(g, x, x, d).sum(), g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), g)
    out = attention.dynamics(g, x, x, d, s)      # a state that a graph has saved is stepped on
    attention.step(y, y, y, d, s)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        out.sum().backward()


# --------------------------------------------------------------------------
# 8-bit dense synapse
# --------------------------------------------------------------------------
def make_dense(seed, n, k, o, T, spikes):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(n, k, T)) * np.exp(rng.normal(size=(n, 1, T)))
    if spikes:
        x = (rng.random((n, k, T)) < 0.2) * np.rint(rng.normal(size=(n, k, T)) * 16) / 64
    return (x.astype(np.float32), rng.integers(-128, 128, size=(o, k), dtype=np.int8),
            rng.normal(size=o).astype(np.float32))


DENSE = [(1, 1, 1, 1), (1, 16, 8, 1), (1, 2048, 100, 1), (2, 100, 33, 1), (1, 300, 40, 5), (3, 17, 70, 9), (2, 128, 128, 64),
         (1, 130, 129, 130), (4, 512, 256, 33), (7, 700, 333, 45), (1, 4097, 65, 300), (70, 64, 300, 3),
         (2, 2048, 520, 129), (1, 40000, 20, 3), (1, 131072, 3, 1)]


@pytest.mark.parametrize('spikes', [False, True])
@pytest.mark.parametrize('shape', DENSE)
def test_dense(cuda, shape, spikes):
    x, w, ws = make_dense(11, *shape, spikes)
    layer = slayer.synapse.QuantDense(torch.from_numpy(w), torch.from_numpy(ws)).cuda()
    assert_exact(layer(dev(x)), O.dense(x, w, ws), 'dense')
    assert _native.device_status() == 0


@pytest.mark.parametrize('T', [1, 300])
def test_dense_extremes(cuda, T):
    """Largest sums, borders of the step, zeros, tiny and huge steps, values that are not finite."""
    rng = np.random.default_rng(12)
    n, k, o = 2, 600, 70
    x = rng.normal(size=(n, k, T)).astype(np.float32)
    kinds = np.arange(n * T).reshape(n, T) % 10
    for (i, t), kind in np.ndenumerate(kinds):
        if kind == 0: x[i, :, t] = 0
        if kind == 1: x[i, :, t] = 1
        if kind == 2: x[i, 5, t] = np.float32(127 * 2.0 ** 3)                      # exactly at the border
        if kind == 3: x[i, 5, t] = np.nextafter(np.float32(127 * 2.0 ** 3), np.float32(np.inf))
        if kind == 4: x[i, :, t] *= np.float32(2.0 ** -130)
        if kind == 5: x[i, :, t] = np.float32(3e38) * np.sign(x[i, :, t])
        if kind == 6: x[i, 3, t] = np.nan
        if kind == 7: x[i, 3, t] = -np.inf
        if kind == 8: x[i, :, t] = np.rint(x[i, :, t] * 20) + 0.5                  # ties
    w = rng.integers(-128, 128, size=(o, k), dtype=np.int8)
    w[0], w[1] = -128, 127
    ws = np.full(o, 2.0 ** -10, dtype=np.float32)
    got = slayer.synapse.QuantDense(torch.from_numpy(w), torch.from_numpy(ws)).cuda()(dev(x)).cpu().numpy()
    want = O.dense(x, w, ws)
    assert np.array_equal(got, want, equal_nan=True)


def test_dense_is_the_float_synapse_on_spikes(cuda):
    neuron = slayer.neuron.cuba.Neuron(threshold=1.0, current_decay=0.25, voltage_decay=0.03)
    dense = slayer.synapse.Dense(200, 96, weight_scale=4, pre_hook_fx=neuron.quantize_8bit).cuda()
    layer = slayer.synapse.QuantDense.from_dense(dense, step=2 / neuron.w_scale)
    x = (torch.rand(4, 200, 150, generator=torch.Generator().manual_seed(1)) < 0.3).float()
    want = torch.einsum('ok,nkt->not', dense._hooked_weight().detach().double().cpu().reshape(96, 200), x.double())
    assert_exact(layer(x.cuda()).double(), want)


def test_dense_inputs(cuda):
    """Five dimensions, views, repeats, empty batches, refusals."""
    x, w, ws = make_dense(13, 3, 24, 10, 50, False)
    layer = slayer.synapse.QuantDense(torch.from_numpy(w), torch.from_numpy(ws), (2, 3, 4)).cuda()
    xd = dev(x)
    want = layer(xd)
    assert torch.equal(layer(xd.reshape(3, 2, 3, 4, 50)).reshape(3, 10, 50), want)
    assert layer(xd.reshape(3, 2, 3, 4, 50)).shape == (3, 10, 1, 1, 50)
    assert torch.equal(layer(torch.cat((xd, xd), -1)[..., 50:]), want)
    assert layer(xd[:0]).shape == (0, 10, 50) and layer(xd[..., :0]).shape == (3, 10, 0)
    for bad in (xd[:, :20], xd.reshape(3, 3, 2, 4, 50), xd[0]):
        with pytest.raises(ValueError):
            layer(bad)
    with pytest.raises(TypeError):
        layer(xd.double())
    with pytest.raises(RuntimeError):
        slayer.synapse.QuantDense(torch.from_numpy(w), torch.from_numpy(ws))(xd)
    graphed = slayer.utils.Graphed(layer, xd)
    assert torch.equal(graphed(xd * 2), layer(xd * 2))


# --------------------------------------------------------------------------
# dropout
# --------------------------------------------------------------------------
@pytest.mark.parametrize('per_step', [False, True])
@pytest.mark.parametrize('shape', [(1,), (3, 1), (2, 5, 3), (4, 7, 128), (3, 50, 301), (2, 3, 2, 2, 40), (1, 1, 70001),
                                   (5000, 2)])
@pytest.mark.parametrize('p', [0.0, 0.1, 0.5, 1.0])
def test_dropout(cuda, shape, p, per_step):
    rng = np.random.default_rng(14)
    x, g = (rng.normal(size=shape).astype(np.float32) for _ in range(2))
    x.flat[0] = np.nan
    key = [int(rng.integers(-2 ** 63, 2 ** 63)), int(rng.integers(-2 ** 63, 2 ** 63))]
    xd = dev(x).requires_grad_()
    y = dropout(xd, p, torch.tensor(key, device='cuda'), per_step)
    (gx,) = torch.autograd.grad(y, xd, dev(g))
    unsigned = [k % 2 ** 64 for k in key]
    assert np.array_equal(y.detach().cpu().numpy(), O.dropout(x, p, unsigned, per_step), equal_nan=True)
    assert_exact(gx, O.dropout(g, p, unsigned, per_step), 'gradient')


def test_dropout_views_and_alignment(cuda):
    key = torch.tensor([5, 9], device='cuda')
    x = torch.randn(4099, device='cuda')
    for a in (1, 2, 3):
        for per_step in (False, True):
            view = x[a:].view(2, 1, -1) if (4099 - a) % 2 == 0 else x[a:].view(1, 1, -1)
            assert torch.equal(dropout(view, 0.4, key, per_step), dropout(view.clone(), 0.4, key, per_step))
    t = torch.randn(6, 8, 10, device='cuda')
    assert torch.equal(dropout(t.transpose(0, 1), 0.4, key), dropout(t.transpose(0, 1).contiguous(), 0.4, key))
    y = dropout(t.requires_grad_(), 0.4, key)
    (g,) = torch.autograd.grad(y.sum(), t)          # a broadcast gradient
    assert torch.equal(g, dropout(torch.ones_like(t), 0.4, key))
    assert dropout(x[:0].view(0, 3), 0.4, key).shape == (0, 3)


def test_dropout_refusals(cuda):
    x, key = torch.zeros(2, 3, device='cuda'), torch.zeros(2, dtype=torch.int64, device='cuda')
    for bad in (key.int(), key[:1], key.repeat(2)[::2]):
        with pytest.raises(ValueError):
            dropout(x, 0.5, bad)
    for p in (-0.1, 1.1, float('nan')):
        with pytest.raises(ValueError):
            dropout(x, p, key)
    with pytest.raises(RuntimeError):
        dropout(x, 0.5, key.cpu())
    with pytest.raises(TypeError):
        dropout(x.half(), 0.5, key)


def test_dropout_module(cuda):
    drop = slayer.neuron.Dropout(0.5, seed=3).cuda()
    x = torch.ones(4, 100, 20, device='cuda')
    a, b = drop(x), drop(x)
    assert not torch.equal(a, b) and drop.generator.tolist() == [3, 2]
    assert_exact(a, O.dropout(x.cpu().numpy(), 0.5, [3, 0], False))
    assert_exact(b, O.dropout(x.cpu().numpy(), 0.5, [3, 1], False))
    assert torch.equal(drop.eval()(x), x)
    lazy = slayer.neuron.Dropout(0.5, seed=3)       # moved to its input on first use
    assert torch.equal(lazy(x), a)
    # replays of a captured call use new masks
    drop.train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        drop(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x)
    first = drop.generator.tolist()[1]
    for i in range(3):
        graph.replay()
        assert_exact(y, O.dropout(x.cpu().numpy(), 0.5, [3, first + i], False))


# --------------------------------------------------------------------------
# together: the attention block
# --------------------------------------------------------------------------
CUBA = dict(threshold=0.5, current_decay=0.25, voltage_decay=0.03)


def block(persistent=False, drop=None, **kw):
    torch.manual_seed(0)
    return slayer.block.cuba.Attention(dict(CUBA, persistent_state=persistent, dropout=drop), 24, 32, 4, weight_scale=4,
                                       **kw).cuda()


def plain_block(b, x):
    """The block out of its parts: synapses and neurons as they are, attention in 64 bits, no delay."""
    parts = []
    for name in ('query', 'key', 'value'):
        z = getattr(b, name + '_synapse')(x)
        parts.append(getattr(b, name + '_neuron')(z).reshape(x.shape[0], 4, 8, x.shape[-1]).cpu().numpy())
    o, _ = O.attention(*parts, b.memory_decay.cpu().numpy())
    return o.reshape(x.shape[0], 32, -1)


def test_attention_block_parts(cuda):
    b = block(count_log=True)
    x = (torch.rand(3, 24, 200, generator=torch.Generator().manual_seed(2)) < 0.3).float().cuda()
    spikes, rate = b(x)
    assert spikes.shape == (3, 32, 200) and 0 < float(rate) < 1
    with torch.no_grad():
        read = torch.from_numpy(plain_block(b, x)).float().cuda()
        want = slayer.axon.delay(b.neuron(b.synapse(read)), 1)
    # spikes of rounded currents: a current next to the threshold may fall on the other side
    assert (want != spikes).float().mean() < 1e-3


def test_attention_block_training(cuda):
    b = block(drop=slayer.neuron.Dropout(0.1, seed=1))
    x = (torch.rand(3, 24, 200, generator=torch.Generator().manual_seed(2)) < 0.3).float().cuda()
    b(x).sum().backward()
    for name, p in b.named_parameters():
        if p.requires_grad:
            assert p.grad is not None and torch.isfinite(p.grad).all(), name
    for name in ('query', 'key', 'value'):
        assert getattr(b, name + '_synapse').weight.grad.abs().max() > 0, name
    assert b.neuron.drop.generator.tolist()[1] == 4


def test_attention_block_training_captured(cuda):
    """A captured training step: the gradients of the eager one under the same masks, new masks at each replay."""
    x = (torch.rand(3, 24, 200, generator=torch.Generator().manual_seed(2)) < 0.3).float().cuda()
    b = block(drop=slayer.neuron.Dropout(0.2, seed=1))

    def step(module):
        weights = [p for p in module.parameters() if p.requires_grad]
        return torch.autograd.grad(module(x).sum(), weights, allow_unused=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step(b)
    start = int(b.neuron.drop.generator[1])
    seen = []
    for i in range(2):
        graph.replay()
        got = [g.clone() for g in grads if g is not None]
        fresh = block(drop=slayer.neuron.Dropout(0.2, seed=1))
        fresh.load_state_dict(b.state_dict())
        fresh.neuron.drop.generator.copy_(torch.tensor([1, start + 4 * i]))
        want = [g for g in step(fresh) if g is not None]
        # the synapses' own gradients are library sums over 3 x 200 steps, whose order may differ: 600 half steps
        # of 2^-24 are 4e-5 of the largest
        for g, w in zip(got, want):
            assert torch.allclose(g, w, rtol=1e-4, atol=1e-4 * float(w.abs().max()))
        seen.append(got)
    assert any(not torch.equal(a, c) for a, c in zip(*seen))


def test_attention_block_quantized(cuda):
    """Spikes through weights on the neuron's grid: the 8-bit synapses give the float ones' currents; the
    read-out of the memory is not on a grid and is rounded."""
    b = block()
    x = (torch.rand(3, 24, 200, generator=torch.Generator().manual_seed(2)) < 0.3).float().cuda()
    with torch.no_grad():
        want = [getattr(b, n + '_neuron')(getattr(b, n + '_synapse')(x)) for n in ('query', 'key', 'value')]
        b.quantize()
        got = [getattr(b, n + '_neuron')(getattr(b, n + '_synapse')(x)) for n in ('query', 'key', 'value')]
        for a, c in zip(want, got):
            assert torch.equal(a, c)
        spikes = b(x)
    assert 0 < float(spikes.mean()) < 1
    dense = slayer.block.cuba.Dense(dict(CUBA), 24, 16, weight_scale=4, mask=torch.rand(16, 24) < 0.5).cuda()
    with torch.no_grad():
        want = dense(x)
        assert torch.equal(dense.quantize()(x), want) and dense.quantize() is dense


def test_attention_block_persistent(cuda):
    """Pieces of a sequence, single steps among them, give what the whole gives."""
    x = (torch.rand(2, 24, 60, generator=torch.Generator().manual_seed(4)) < 0.3).float().cuda()
    with torch.no_grad():
        whole = block(persistent=True)(x)
        b = block(persistent=True)
        cuts = [0, 1, 2, 30, 31, 60]
        parts = torch.cat([b(x[..., i:j]) for i, j in zip(cuts, cuts[1:])], -1)
        assert (whole != parts).float().mean() < 1e-3
        assert b(x[:1]).shape == (1, 32, 60)      # another batch size starts anew


@pytest.mark.parametrize('family, params', [
    ('alif', dict(threshold=0.5, threshold_step=0.2, current_decay=0.25, voltage_decay=0.03, threshold_decay=0.1,
                  refractory_decay=0.1)),
    ('rf', dict(threshold=0.5, period=10, decay=0.1)),
    ('adrf', dict(threshold=0.5, threshold_step=0.1, period=10, decay=0.1, threshold_decay=0.1, refractory_decay=0.1))])
def test_attention_block_families(cuda, family, params):
    torch.manual_seed(0)
    b = getattr(slayer.block, family).Attention(params, 24, 32, 4, weight_scale=4, delay=True).cuda()
    x = (torch.rand(2, 24, 100, generator=torch.Generator().manual_seed(2)) < 0.3).float().cuda()
    y = b(x)
    assert y.shape == (2, 32, 100)
    y.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in b.parameters() if p.grad is not None)
