"""What the sequence operators of the framework are timed on.

Three operators that a spiking sequence model runs next to the neurons and synapses:

* ``linear attention``: the leaky integrator whose input is an outer product.  A head keeps
  ``S[t] = r S[t-1] + k[t] v[t]^T`` with ``r = 1 - decay / 4096`` and answers ``o[t] = S[t]^T q[t]``;
  whole sequences forward, forward with backward, and single steps on a kept state;
* ``dense``: the dense synapse with 8-bit weights and 8-bit activations, one scale for each output
  neuron and one power of two for each time step of each sample;
* ``dropout``: of single values or of whole neurons, from a counter-based generator whose mask is
  never stored, forward and backward.

``own`` false runs them in plain torch operations, ``own`` true through the framework's own calls.
"""

import math
import os
import sys

import torch

own = False

DEVICE = 'cuda'


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one new step for one stream of a small model: nothing but latency
        dict(name='attn_step_one', op='attn_step', N=1, H=8, Dk=64, Dv=64),
        # one new step for every stream of a large serving batch
        dict(name='attn_step_batch', op='attn_step', N=128, H=16, Dk=64, Dv=64),
        # a batch of event recordings of 300 steps, spikes in, one decay for each head
        dict(name='attn_prompt', op='attn_prompt', N=64, H=8, Dk=64, Dv=64, T=300, spikes=True, state=False),
        # one long recording, continued from a kept state: few heads, a long axis
        dict(name='attn_prompt_long', op='attn_prompt', N=1, H=8, Dk=64, Dv=64, T=32768, spikes=False, state=True),
        # odd sizes everywhere: heads of unequal widths, a length no vector width divides
        dict(name='attn_prompt_odd', op='attn_prompt', N=5, H=6, Dk=40, Dv=72, T=777, spikes=False, state=True),
        # a training step at the sequence length of the neuron benchmarks
        dict(name='attn_train', op='attn_train', N=16, H=16, Dk=64, Dv=64, T=2000, spikes=True),
        # a training step of few wide heads over a longer axis
        dict(name='attn_train_wide', op='attn_train', N=4, H=8, Dk=128, Dv=128, T=4096, spikes=False),
        # the synapse of one stream, step by step: the weights are all there is to read
        dict(name='dense_step', op='dense', N=1, K=2048, O=2048, T=1, spikes=False),
        # a batch of graded spikes through the projection of a layer
        dict(name='dense_batch', op='dense', N=64, K=2048, O=2048, T=300, spikes=True),
        # odd sizes: neither side a multiple of any tile, rows that start at odd addresses
        dict(name='dense_odd', op='dense', N=7, K=700, O=333, T=451, spikes=False),
        # spikes of a training batch, each value dropped by itself, with the gradient
        dict(name='dropout_values', op='dropout', N=64, C=4096, T=1000, p=0.1, per_step=True),
        # the same for whole neurons over odd sizes
        dict(name='dropout_neurons', op='dropout', N=33, C=2050, T=301, p=0.25, per_step=False),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attn_step', 'attn_prompt', 'attn_prompt', 'attn_train', 'dense', 'dense', 'dropout'])
    if op == 'dropout':
        per_step = rng.random() < 0.5
        T = _log(rng, 1, 2000)
        C = _log(rng, 1, 8192)
        N = min(_log(rng, 1, 64), max(1, 64 * 4096 * 1000 // (C * T)))
        return dict(op=op, N=N, C=C, T=T, p=rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]), per_step=per_step)
    if op == 'dense':
        K, O = _log(rng, 16, 4096), _log(rng, 8, 4096)
        T = 1 if rng.random() < 0.35 else _log(rng, 2, 2000)
        N = _log(rng, 1, 64)
        N = max(1, min(N, int(64 * 300 * 2048 * 2048 / (T * K * O)), 64 * 300 * 2048 // (T * max(K, O))))
        return dict(op=op, N=N, K=K, O=O, T=T, spikes=rng.random() < 0.5)
    widths = [16, 24, 32, 40, 48, 64, 64, 64, 72, 80, 96, 100, 112, 128]
    Dk = rng.choice(widths)
    Dv = Dk if rng.random() < 0.6 else rng.choice(widths)
    H = _log(rng, 1, 16)
    if op == 'attn_step':
        return dict(op=op, N=min(_log(rng, 1, 128), max(1, 128 * 16 * 64 * 64 // (H * Dk * Dv))), H=H, Dk=Dk, Dv=Dv)
    T = _log(rng, 2, 16384)
    budget = 16 * 16 * 2000 * 64 // (H * T * max(Dk, Dv))
    N = max(1, min(_log(rng, 1, 64), budget))
    case = dict(op=op, N=N, H=H, Dk=Dk, Dv=Dv, T=T, spikes=rng.random() < 0.4)
    if op == 'attn_prompt':
        case['state'] = rng.random() < 0.5
    return case


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _spikes(g, rate, *shape):
    return (_rand(g, *shape) < rate).float()


def _decays(g, H):
    """Time constants of about 2 to 1000 steps, spread over the heads as the neurons' decays are."""
    return 4096.0 * torch.exp(math.log(0.5) + (math.log(0.001) - math.log(0.5)) * _rand(g, H))


def prepare(case, seed):
    g = _gen(seed)
    op = case['op']
    st = dict(case=case)
    if op.startswith('attn'):
        N, H, Dk, Dv = case['N'], case['H'], case['Dk'], case['Dv']
        st['decay'] = _decays(g, H)
        if op == 'attn_step':
            st['q'], st['k'] = _randn(g, N, H, Dk) / math.sqrt(Dk), _randn(g, N, H, Dk)
            st['v'] = _randn(g, N, H, Dv)
            st['state'] = 3.0 * _randn(g, N, H, Dk, Dv)
        else:
            T = case['T']
            if case['spikes']:
                st['q'], st['k'] = _spikes(g, 0.15, N, H, Dk, T), _spikes(g, 0.15, N, H, Dk, T)
                st['v'] = _spikes(g, 0.15, N, H, Dv, T)
            else:
                st['q'], st['k'] = _randn(g, N, H, Dk, T) / math.sqrt(Dk), _randn(g, N, H, Dk, T)
                st['v'] = _randn(g, N, H, Dv, T)
            if op == 'attn_prompt':
                st['state'] = 3.0 * _randn(g, N, H, Dk, Dv) if case['state'] else None
            else:
                st['go'] = _randn(g, N, H, Dv, T)
                for name in ('q', 'k', 'v'):
                    st[name].requires_grad_(True)
    elif op == 'dense':
        N, K, O, T = case['N'], case['K'], case['O'], case['T']
        if case['spikes']:      # graded spikes of a sigma-delta layer: sparse multiples of 1/64
            x = _spikes(g, 0.2, N, K, T) * torch.round(16.0 * _randn(g, N, K, T)) / 64.0
        else:                   # values with a different size at each time step
            x = _randn(g, N, K, T) * torch.exp(_randn(g, N, 1, T))
        st['x'] = x
        st['w'] = torch.randint(-127, 128, (O, K), generator=g, device=DEVICE, dtype=torch.int8)
        st['ws'] = (0.5 + _rand(g, O)) / (64.0 * math.sqrt(K))
        if own:
            st['layer'] = _slayer().synapse.QuantDense(st['w'], st['ws'])
    else:
        N, C, T = case['N'], case['C'], case['T']
        st['x'] = _spikes(g, 0.2, N, C, T) * (1.0 + _rand(g, N, C, 1))
        st['x'].requires_grad_(True)
        st['g'] = _randn(g, N, C, T)
        st['key'] = torch.randint(0, 2 ** 62, (2,), generator=g, device=DEVICE, dtype=torch.int64)
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _slayer():
    path = os.path.join(os.getcwd(), 'lava-dl_b200')
    if path not in sys.path:
        sys.path.insert(0, path)
    import lava_dl_b200.slayer as slayer
    return slayer


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    case, op = st['case'], st['case']['op']
    slayer = _slayer()
    attention = slayer.neuron.dynamics.linear_attention
    if op == 'attn_step':
        return attention.step(st['q'], st['k'], st['v'], st['decay'], st['state']), st['state']
    if op == 'attn_prompt':
        with torch.no_grad():
            return attention.dynamics(st['q'], st['k'], st['v'], st['decay'], st['state'], return_state=True)
    if op == 'attn_train':
        o = attention.dynamics(st['q'], st['k'], st['v'], st['decay'])
        return (o.detach(),) + torch.autograd.grad(o, (st['q'], st['k'], st['v']), st['go'])
    if op == 'dense':
        return st['layer'](st['x'])
    y = slayer.neuron.dropout.dropout(st['x'], case['p'], st['key'], per_step=case['per_step'])
    return (y.detach(),) + torch.autograd.grad(y, (st['x'],), st['g'])


def _run_plain(st):
    case, op = st['case'], st['case']['op']
    if op == 'attn_step':
        r = (1.0 - st['decay'].double() / 4096.0).float()
        s = r.view(1, -1, 1, 1) * st['state'] + st['k'].unsqueeze(-1) * st['v'].unsqueeze(-2)
        st['state'].copy_(s)
        return (st['q'].unsqueeze(-1) * s).sum(-2), st['state']
    if op == 'attn_prompt':
        with torch.no_grad():
            return _plain_attention(st['q'], st['k'], st['v'], st['decay'], st['state'])
    if op == 'attn_train':
        o, _ = _plain_attention(st['q'], st['k'], st['v'], st['decay'], None)
        return (o.detach(),) + torch.autograd.grad(o, (st['q'], st['k'], st['v']), st['go'])
    if op == 'dense':
        return _plain_dense(st['x'], st['w'], st['ws'])
    scale, keep = _plain_mask(case, st['key'])
    y = torch.where(keep, st['x'].detach() * scale, 0.0)
    return y, torch.where(keep, st['g'] * scale, 0.0)


def _plain_attention(q, k, v, decay, state, chunk=128):
    """Chunks of `chunk` steps: inside a chunk the steps answer each other through their scores, all
    chunks at once; from chunk to chunk goes the state."""
    N, H, Dk, T = q.shape
    Dv = v.shape[2]
    r = 1.0 - decay.double() / 4096.0
    s = torch.zeros(N, H, Dk, Dv, device=q.device) if state is None else state
    outs = []
    full = T // chunk
    spans = [(0, full, chunk)] if full else []
    if T % chunk:
        spans.append((full * chunk, 1, T % chunk))
    for start, C, L in spans:
        n = torch.arange(L, device=q.device, dtype=torch.float64)
        gap = n.view(-1, 1) - n.view(1, -1)
        inside = torch.where(gap >= 0, r.view(H, 1, 1) ** gap.clamp(min=0), 0.0).float().view(1, H, 1, L, L)
        into = (r.view(H, 1) ** (n + 1.0)).float().view(1, H, 1, L, 1)
        left = (r.view(H, 1) ** (L - 1.0 - n)).float().view(1, H, 1, L, 1)
        over = (r ** float(L)).float().view(1, H, 1, 1)
        part = [x[..., start:start + C * L].reshape(N, H, x.shape[2], C, L).permute(0, 1, 3, 4, 2) for x in (q, k, v)]
        qc, kc, vc = part
        grown = (kc * left).transpose(-1, -2) @ vc
        before = []
        for c in range(C):
            before.append(s)
            s = over * s + grown[:, :, c]
        o = ((qc @ kc.transpose(-1, -2)) * inside) @ vc + into * (qc @ torch.stack(before, 2))
        outs.append(o.reshape(N, H, C * L, Dv))
    return torch.cat(outs, 2).transpose(-1, -2).contiguous(), s


def _plain_dense(x, w, ws):
    """Sums of 8-bit products are whole numbers past 2^24: taken in 64 bits."""
    amax = x.abs().amax(1, keepdim=True)
    m, e = torch.frexp(amax)
    p = torch.where(m <= 127.0 / 128.0, e - 7, e - 6).clamp(min=-126)
    one = torch.ones_like(amax)
    q = torch.round(x * torch.ldexp(one, -p))
    acc = torch.matmul(w.double(), q.double())
    return acc.float() * ws.view(1, -1, 1) * torch.ldexp(one, p)


def _plain_mask(case, key):
    """Philox4x32 with ten rounds (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011)
    in 64-bit integer operations: value i is word i % 4 of counter (i // 4, offset) under key seed."""
    N, C, T, p = case['N'], case['C'], case['T'], case['p']
    count = N * C * (T if case['per_step'] else 1)
    low = 0xffffffff
    i = torch.arange((count + 3) // 4, device=key.device, dtype=torch.int64)
    seed, offset = key[0], key[1]
    c = [i & low, i >> 32, (offset & low).expand_as(i), ((offset >> 32) & low).expand_as(i)]
    k0, k1 = seed & low, (seed >> 32) & low

    def mul(a, m):      # high and low words of a 32 x 32 bit product
        lo, hi = a * (m & 0xffff), a * (m >> 16)
        mid = (lo >> 16) + (hi & low)
        return (hi >> 32 << 16) + (mid >> 16) & low, ((mid & 0xffff) << 16) | (lo & 0xffff)

    for _ in range(10):
        h0, l0 = mul(c[0], 0xD2511F53)
        h1, l1 = mul(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack(c, 1).reshape(-1)[:count]
    keep = (words >= int(p * 2.0 ** 32)).view(N, C, T if case['per_step'] else 1)
    return 1.0 / (1.0 - p), keep


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    op = case['op']
    if op.startswith('attn'):
        N, H, Dk, Dv = case['N'], case['H'], case['Dk'], case['Dv']
        heads = N * H
        if op == 'attn_step':
            return dict(bytes=4 * (heads * (2 * Dk + 2 * Dv + 2 * Dk * Dv) + H), flops=heads * 5 * Dk * Dv)
        T = case['T']
        if op == 'attn_prompt':
            states = heads * Dk * Dv * (2 if case['state'] else 1)
            return dict(bytes=4 * (heads * T * (2 * Dk + 2 * Dv) + states + H), flops=heads * T * 5 * Dk * Dv)
        # q, k, v, the output and its gradient, and the gradients of q, k, v
        return dict(bytes=4 * (heads * T * (4 * Dk + 4 * Dv) + H), flops=heads * T * 15 * Dk * Dv)
    if op == 'dense':
        N, K, O, T = case['N'], case['K'], case['O'], case['T']
        return dict(bytes=4 * N * T * (K + O) + K * O + 4 * O, flops=2 * N * T * K * O)
    count = case['N'] * case['C'] * case['T']
    return dict(bytes=16 * count + 16, flops=2 * count)


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    op = case['op']
    saved = globals()['own']
    globals()['own'] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()['own'] = saved
    if op == 'dense':
        return _exact_dense(st)
    if op == 'dropout':
        return _exact_dropout(case, st)
    q, k, v = (st[n].detach().double() for n in ('q', 'k', 'v'))
    r = (1.0 - st['decay'].double() / 4096.0).view(1, -1, 1, 1)
    if op == 'attn_step':
        s = torch.addcmul(r * st['state'].double(), k[..., :, None], v[..., None, :])
        return torch.einsum('nhd,nhde->nhe', q, s), s
    # the recurrence itself, one step after the other
    q, k, v = (x.permute(3, 0, 1, 2).contiguous() for x in (q, k, v))
    T = q.shape[0]
    start = st.get('state')
    s = q.new_zeros(*q.shape[1:], v.shape[-1]) if start is None else start.double().clone()
    o = torch.empty_like(v)
    train = op == 'attn_train'
    if train:
        go = st['go'].double().permute(3, 0, 1, 2).contiguous()
        gq = torch.empty_like(q)
    for t in range(T):
        s.mul_(r).addcmul_(k[t].unsqueeze(-1), v[t].unsqueeze(-2))
        o[t] = torch.matmul(q[t].unsqueeze(-2), s).squeeze(-2)
        if train:
            gq[t] = torch.matmul(s, go[t].unsqueeze(-1)).squeeze(-1)
    if not train:
        return o.permute(1, 2, 3, 0).contiguous(), s
    gk, gv = torch.empty_like(k), torch.empty_like(v)
    s.zero_()
    for t in reversed(range(T)):
        s.mul_(r).addcmul_(q[t].unsqueeze(-1), go[t].unsqueeze(-2))
        gk[t] = torch.matmul(s, v[t].unsqueeze(-1)).squeeze(-1)
        gv[t] = torch.matmul(k[t].unsqueeze(-2), s).squeeze(-2)
    return tuple(x.permute(1, 2, 3, 0).contiguous() for x in (o, gq, gk, gv))


def _exact_dense(st):
    """The step of a token is the smallest power of two whose 127-fold reaches its largest magnitude
    (2^-126 at least)."""
    x = st['x'].double()
    top = x.abs().max(dim=1, keepdim=True).values
    p = torch.ceil(torch.log2((top / 127.0).clamp(min=2.0 ** -126)))
    p = torch.where(127.0 * 2.0 ** (p - 1.0) >= top, p - 1.0, p)     # a logarithm that rounded up
    p = torch.where(127.0 * 2.0 ** p < top, p + 1.0, p).clamp(min=-126.0)
    step = 2.0 ** p
    whole = torch.round(x / step)
    return torch.einsum('ok,nkt->not', st['w'].double(), whole) * st['ws'].double()[None, :, None] * step


def _exact_dropout(case, st):
    """The generator again, on two-word products of 32-bit halves held as Python-sized integers."""
    N, C, T = case['N'], case['C'], case['T']
    seed, offset = (int(w) for w in st['key'].tolist())
    count = N * C * (T if case['per_step'] else 1)
    keep = torch.empty(count, dtype=torch.bool, device=DEVICE)
    mask = (1 << 32) - 1
    for begin in range(0, count, 1 << 26):
        end = min(count, begin + (1 << 26))
        block = torch.arange(begin // 4, (end + 3) // 4, device=DEVICE, dtype=torch.int64)
        a, b = block & mask, block >> 32
        x, y = torch.full_like(a, offset & mask), torch.full_like(a, (offset >> 32) & mask)
        key = [seed & mask, (seed >> 32) & mask]
        for _ in range(10):
            out = []
            for word, factor in ((a, 0xD2511F53), (x, 0xCD9E8D57)):
                f1, f0 = factor >> 16, factor & 0xffff
                w1, w0 = word >> 16, word & 0xffff
                t0 = w0 * f0
                t1 = w1 * f0 + (t0 >> 16)
                t2 = w0 * f1 + (t1 & 0xffff)
                out.append((w1 * f1 + (t1 >> 16) + (t2 >> 16), (t2 << 16 & mask) | (t0 & 0xffff)))
            (ha, la), (hx, lx) = out
            a, b, x, y = hx ^ b ^ key[0], lx, ha ^ y ^ key[1], la
            key = [(key[0] + 0x9E3779B9) & mask, (key[1] + 0xBB67AE85) & mask]
        words = torch.stack((a, b, x, y), -1).flatten()[:end - begin]
        keep[begin:end] = words >= int(case['p'] * 2.0 ** 32)
    keep = keep.view(N, C, -1)
    factor = 1.0 / (1.0 - case['p'])
    return tuple(torch.where(keep, t.detach().double() * factor, 0.0) for t in (st['x'], st['g']))
