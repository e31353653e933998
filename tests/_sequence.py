"""64-bit oracles of the sequence operators, written from their definitions on numpy arrays.

Tolerances (derived, used by the tests of every kernel):

* linear attention: an element is a sum of signed terms ``r^(i-j) q_i[d] k_j[d] v_j[e]``; its error is
  measured against the same sum over magnitudes (the oracle run on absolute values).  A term passes
  at most the ``Dk`` additions of its score, the additions of a chunk of 128 steps or the additions
  and products of the state, three for each step the head remembers (``min(T, 1 / (1 - r))``), and 32
  roundings of splits, weights and scales, each at most 2^-23 (half a step, 2^-24, for an fp32
  operation; a whole one for the tensor cores' truncating sums):
  ``tol = 2^-23 (Dk + 128 + 3 min(T, 1 / (1 - r)) + 32)``.
  The chunked kernel splits each vector (q, k, v of a step, a row of scores, a row of the state) into
  fp16 pairs: an element is held to 22 bits, or to 2^-25 (half of fp16's smallest step) where that is
  more.  What the second case can add, against sums over the vectors' LARGEST magnitudes q', k', v' (a
  score then is Dk q' k'): q, k, v and state rows are scaled to a largest element of at least 2^13,
  2^-38 relative to it each.  A row of scores is scaled by 2^(15 - u), 2^u >= |q_i| max_j |k_j| r^(i-j)
  2^g_j with u at most 3 too large (three roundings up to a power of two), v to at most 2^14 = 2^-g v':
  2^-25 2^14 2^(u - 15) <= 2^-36 of the largest term, for each of up to 128 terms: 2^-29.  The state's
  growth is a sum of 128 such terms as well, 2^-37 of the largest each.  Together below 2^-28
  (``attention_floor``).
* dense and dropout: the sums are whole numbers and the products are rounded in a stated order, so
  the results are compared bit for bit.
"""

import numpy as np


def attention(q, k, v, decay, state=None):
    """Output and final state of one walk; q, k [N, H, Dk, T], v [N, H, Dv, T]."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    n, h, dk, T = q.shape
    dv = v.shape[2]
    r = np.broadcast_to(1.0 - np.asarray(decay, dtype=np.float64).reshape(-1) / 4096.0, (h,)).reshape(1, h, 1, 1)
    s = np.zeros((n, h, dk, dv)) if state is None else np.array(state, dtype=np.float64)
    o = np.empty((n, h, dv, T))
    for t in range(T):
        s = r * s + k[..., t][..., :, None] * v[..., t][..., None, :]
        o[..., t] = np.einsum('nhd,nhde->nhe', q[..., t], s)
    return o, s


def attention_grads(q, k, v, decay, state, go, gf):
    """Gradients of q, k, v and the initial state for output gradient go and state gradient gf (or None)."""
    q, k, v, go = (np.asarray(a, dtype=np.float64) for a in (q, k, v, go))
    n, h, dk, T = q.shape
    dv = v.shape[2]
    r = np.broadcast_to(1.0 - np.asarray(decay, dtype=np.float64).reshape(-1) / 4096.0, (h,)).reshape(1, h, 1, 1)
    s = np.zeros((n, h, dk, dv)) if state is None else np.array(state, dtype=np.float64)
    gq, gk, gv = np.empty_like(q), np.empty_like(k), np.empty_like(v)
    for t in range(T):
        s = r * s + k[..., t][..., :, None] * v[..., t][..., None, :]
        gq[..., t] = np.einsum('nhe,nhde->nhd', go[..., t], s)
    g = np.zeros((n, h, dk, dv)) if gf is None else np.array(gf, dtype=np.float64)
    for t in reversed(range(T)):
        g = g + q[..., t][..., :, None] * go[..., t][..., None, :]
        gk[..., t] = np.einsum('nhe,nhde->nhd', v[..., t], g)
        gv[..., t] = np.einsum('nhd,nhde->nhe', k[..., t], g)
        g = r * g
    return gq, gk, gv, g


def attention_tol(dk, T, decay):
    """See the module's text; a decay outside 0..4096 forgets nothing."""
    lost = float(np.min(np.abs(np.asarray(decay, dtype=np.float64)))) / 4096.0
    remembered = T if lost <= 0 or lost > 1 else min(T, 1.0 / lost)
    return 2.0 ** -23 * (dk + 128 + 3 * remembered + 32)


def attention_floor(q, k, v, decay, state=None):
    """What the smallest step of an fp16 pair can add up to: the sums (output, state) over the largest
    magnitudes of each step's vectors, times 2^-28."""
    def top(a):
        return np.abs(a).max(axis=2, keepdims=True) + np.zeros_like(a)
    s = None if state is None else np.abs(state).max(axis=(2, 3), keepdims=True) + np.zeros_like(state)
    o, f = attention(top(q), top(k), top(v), decay, s)
    return 2.0 ** -28 * o, 2.0 ** -28 * f


def attention_grads_floor(q, k, v, decay, state, go, gf):
    def top(a):
        return np.abs(a).max(axis=2, keepdims=True) + np.zeros_like(a)
    def whole(a):
        return None if a is None else np.abs(a).max(axis=(2, 3), keepdims=True) + np.zeros_like(a)
    return [2.0 ** -28 * g for g in attention_grads(top(q), top(k), top(v), decay, whole(state), top(go), whole(gf))]


def assert_sum_close(got, want, scale, tol, what='', floor=0.0):
    got = got.detach().cpu().numpy().astype(np.float64)
    assert got.shape == want.shape, f'{what}: shape {got.shape} vs {want.shape}'
    if got.size == 0:
        return
    assert np.isfinite(got).all(), f'{what}: non-finite values'
    err, lim = np.abs(got - want), tol * scale + floor + 1e-37
    assert (err <= lim).all(), f'{what}: worst ratio to the bound {np.max(err / lim):.3g}'


def dense(x, w, ws):
    """Bit-exact 8-bit dense product: x [N, K, T] fp32, w [O, K] int8, ws [O] fp32."""
    x = np.asarray(x, dtype=np.float32)
    top = np.abs(x.astype(np.float64)).max(axis=1, keepdims=True)
    bad = ~np.isfinite(x).all(axis=1, keepdims=True)
    m, e = np.frexp(np.where(bad, 0.0, top))
    p = np.maximum(np.where(m <= 127.0 / 128.0, e - 7, e - 6), -126)
    p = np.where(top == 0, -126, p)
    step = np.ldexp(1.0, p)
    xq = np.rint(np.where(bad, 0.0, x) / step)
    assert np.abs(xq).max(initial=0) <= 127
    acc = np.einsum('ok,nkt->not', w.astype(np.float64), xq)
    with np.errstate(over='ignore', invalid='ignore', under='ignore'):
        y = acc.astype(np.float32) * np.asarray(ws, dtype=np.float32)[None, :, None]
        return y * np.where(bad, np.nan, step).astype(np.float32)


def philox(counter, offset, seed):
    """Philox4x32 with ten rounds on arrays of 64-bit counters -> uint32 words [..., 4]."""
    u = np.uint64
    low = u(0xffffffff)
    counter = np.asarray(counter, dtype=np.uint64)
    c = [counter & low, counter >> u(32), np.full_like(counter, offset & 0xffffffff),
         np.full_like(counter, (offset >> 32) & 0xffffffff)]
    k = [seed & 0xffffffff, (seed >> 32) & 0xffffffff]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return np.stack(c, -1).astype(np.uint32)


def dropout(x, p, key, per_step):
    """Bit-exact dropout of an fp32 array with time last."""
    x = np.asarray(x, dtype=np.float32)
    T = x.shape[-1]
    count = x.size if per_step else (x.size // T if T else 0)
    words = philox(np.arange((count + 3) // 4), key[1], key[0]).reshape(-1)[:count]
    keep = words.astype(np.uint64) >= np.uint64(int(p * 2.0 ** 32))
    keep = keep.reshape(x.shape) if per_step else np.broadcast_to(keep.reshape(x.shape[:-1] + (1,)), x.shape)
    scale = np.float32(1.0 / (1.0 - p)) if p < 1 else np.float32(0)
    return np.where(keep, x * scale, np.float32(0))
