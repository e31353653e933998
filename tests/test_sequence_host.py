"""The sequence operators without a GPU: refusals of the C entry points, of the Python layer, block
construction, and the oracles against each other and against published values."""

import numpy as np
import pytest
import torch

import _sequence as O
import lava_dl_b200.slayer as slayer
from lava_dl_b200 import _native

attention = slayer.neuron.dynamics.linear_attention
CUBA = dict(threshold=1.0, current_decay=0.25, voltage_decay=0.03)


def refused(name, *args):
    lib = _native.load()
    assert getattr(lib, name)(*args) == -1, name
    return _native.last_error()


def att(heads=4, H=2, nd=2, dk=8, dv=8, T=5):
    return (None,) * 4 + (nd, None, None, None, heads, H, dk, dv, T, None, None)


@pytest.mark.parametrize('change, text', [
    (dict(heads=-2), 'negative'), (dict(T=-1), 'negative'), (dict(dk=0), 'widths'), (dict(dk=129), 'widths'),
    (dict(dv=129), 'widths'), (dict(heads=3), 'multiple'), (dict(nd=3), 'decay'), (dict(T=1 << 31), 'large'),
    (dict(), 'null')])
def test_attention_entry_refuses(change, text):
    assert text in refused('sb_linear_attention_fwd', *att(**change))


def test_attention_other_entries_refuse():
    args = (None,) * 4 + (1,) + (None,) * 7 + (4, 2, 8, 8, 5, None, None)
    assert 'null' in refused('sb_linear_attention_bwd', *args)
    assert 'null' in refused('sb_linear_attention_step', *((None,) * 4 + (1, None, None, 4, 2, 8, 8, None)))
    assert 'widths' in refused('sb_linear_attention_step', *((None,) * 4 + (1, None, None, 4, 2, 0, 8, None)))
    lib = _native.load()   # nothing to do is no error
    assert lib.sb_linear_attention_fwd(*att(heads=0)) == 0


@pytest.mark.parametrize('dims, text', [
    ((-1, 4, 16, 4, 4), 'negative'), ((1, 0, 16, 4, 4), 'inputs'), ((1, 131073, 131088, 4, 4), 'inputs'),
    ((1, 4, 17, 4, 4), 'weight rows'), ((1, 4, 32, 4, 4), 'weight rows'), ((1, 4, 16, 4, 4), 'null')])
def test_dense_entry_refuses(dims, text):
    assert text in refused('sb_qdense_fwd', None, None, None, None, *dims, None, None)


@pytest.mark.parametrize('rows, T, p, text', [
    (-1, 4, 0.5, 'negative'), (4, 4, 1.5, 'probability'), (4, 4, -0.1, 'probability'),
    (4, 4, float('nan'), 'probability'), (1 << 40, 1 << 30, 0.5, 'large'), (4, 4, 0.5, 'null')])
def test_dropout_entry_refuses(rows, T, p, text):
    assert text in refused('sb_dropout', None, None, None, rows, T, p, 1, None)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 4, 6)
    with pytest.raises(RuntimeError, match='CUDA'):
        attention.dynamics(x, x, x, torch.zeros(2))
    with pytest.raises(RuntimeError, match='CUDA'):
        attention.step(x[..., 0], x[..., 0], x[..., 0], torch.zeros(2), torch.zeros(1, 2, 4, 4))
    with pytest.raises(RuntimeError, match='CUDA'):
        slayer.neuron.dropout.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='CUDA'):
        slayer.synapse.QuantDense(torch.zeros(3, 2, dtype=torch.int8), torch.ones(3))(torch.zeros(1, 2, 5))


def test_gradients_that_do_not_exist_are_refused():
    x = torch.zeros(1, 2, 4, 6)
    with pytest.raises(RuntimeError, match='decay'):
        attention.dynamics(x, x, x, torch.zeros(2, requires_grad=True))
    with pytest.raises(RuntimeError, match='no gradient'):
        attention.step(x[..., 0].requires_grad_(), x[..., 0], x[..., 0], torch.zeros(2), torch.zeros(1, 2, 4, 4))
    layer = slayer.synapse.QuantDense(torch.zeros(3, 2, dtype=torch.int8), torch.ones(1))
    with pytest.raises(RuntimeError, match='inference'):
        layer(torch.zeros(1, 2, 5, requires_grad=True))


def test_dropout_module():
    with pytest.raises(ValueError, match='probability'):
        slayer.neuron.Dropout(1.5)
    drop = slayer.neuron.Dropout(0.3, seed=7)
    assert drop.generator.tolist() == [7, 0] and not drop.state_dict()
    x = torch.randn(2, 3, 4)
    assert drop.eval()(x) is x
    assert slayer.neuron.Dropout(0.0)(x) is x


def test_quant_dense_construction():
    w = torch.randint(-128, 128, (5, 6), dtype=torch.int8)
    layer = slayer.synapse.QuantDense(w, torch.ones(1), (2, 1, 3))
    assert layer.weight_q.shape == (5, 16) and layer.shape == (5, 2, 1, 3, 1)
    assert torch.equal(layer.weight_q[:, :6], w) and not layer.weight_q[:, 6:].any()
    for bad in (lambda: slayer.synapse.QuantDense(w.float(), torch.ones(5)),
                lambda: slayer.synapse.QuantDense(w[0], torch.ones(5))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: slayer.synapse.QuantDense(w, torch.ones(4)),
                lambda: slayer.synapse.QuantDense(w, torch.ones(5), (2, 2, 2)),
                lambda: slayer.synapse.QuantDense(w[:, :0], torch.ones(5))):
        with pytest.raises(ValueError):
            bad()


def test_quant_dense_from_dense():
    neuron = slayer.neuron.cuba.Neuron(**CUBA)
    dense = slayer.synapse.Dense((3, 2, 4), 7, pre_hook_fx=neuron.quantize_8bit)   # width, height, channels
    layer = slayer.synapse.QuantDense.from_dense(dense, step=2 / neuron.w_scale)
    want = neuron.quantize_8bit(dense.weight).reshape(7, -1)
    assert layer.in_shape == (4, 2, 3)
    assert torch.equal(layer.weight_q[:, :24].float() * layer.weight_scale[:, None], want)
    free = slayer.synapse.QuantDense.from_dense(slayer.synapse.Dense(9, 4))
    assert free.weight_q.abs().amax(1).tolist() == [127] * 4
    normed = slayer.synapse.Dense(9, 4, weight_norm=True)
    with torch.no_grad():
        normed.weight_g *= 3
    q = slayer.synapse.QuantDense.from_dense(normed)
    got = q.weight_q[:, :9].float() * q.weight_scale[:, None]
    want = (normed.weight_g * normed.weight_v / normed.weight_v.flatten(1).norm(dim=1).view(-1, 1, 1, 1, 1)).reshape(4, 9)
    # half a step of the grid, and a few roundings of the norm
    assert ((got - want).abs() <= want.abs().amax(1, keepdim=True) * (0.5 / 127 + 16 * 2 ** -24)).all()
    with pytest.raises(ValueError, match='8 bits'):
        slayer.synapse.QuantDense.from_dense(slayer.synapse.Dense(9, 4), step=1e-6)


def test_attention_block_construction():
    block = slayer.block.cuba.Attention(dict(CUBA), 12, 32, 4, memory_decay=(0.5, 0.004))
    assert block.head_neurons == 8
    assert np.allclose(block.memory_decay.numpy(), 4096 * np.geomspace(0.5, 0.004, 4), rtol=2 ** -23)
    assert slayer.block.cuba.Attention(dict(CUBA), 12, 32, 4, memory_decay=0.1).memory_decay.shape == (4,)
    with pytest.raises(ValueError, match='split'):
        slayer.block.cuba.Attention(dict(CUBA), 12, 30, 4)
    with pytest.raises(ValueError, match='128'):
        slayer.block.cuba.Attention(dict(CUBA), 12, 1024, 4)
    for decay in ((0.5, 0.1, 0.2), 1.5, -0.1):
        with pytest.raises(ValueError, match='fractions'):
            slayer.block.cuba.Attention(dict(CUBA), 12, 32, 4, memory_decay=decay)
    assert isinstance(block.quantize().key_synapse, slayer.synapse.QuantDense)
    rf = slayer.block.rf.Attention(dict(threshold=1.0, period=10, decay=0.1), 12, 32, 4)
    with pytest.raises(NotImplementedError):
        rf.quantize()


def test_oracle_generator_has_the_published_values():
    """Known answers of Philox4x32-10 in the authors' test vectors."""
    ones = (1 << 64) - 1
    assert O.philox(np.array([0]), 0, 0)[0].tolist() == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert O.philox(np.array([ones], dtype=np.uint64), ones, ones)[0].tolist() == \
        [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def test_oracle_gradients_against_differences():
    """The operator is linear in each input: a difference over any distance is its gradient."""
    rng = np.random.default_rng(3)
    q, k, v = rng.normal(size=(1, 2, 3, 9)), rng.normal(size=(1, 2, 3, 9)), rng.normal(size=(1, 2, 4, 9))
    s, decay = rng.normal(size=(1, 2, 3, 4)), np.array([400.0, 3000.0])
    go, gf = rng.normal(size=v.shape), rng.normal(size=s.shape)

    def loss(*a):
        o, f = O.attention(a[0], a[1], a[2], decay, a[3])
        return (o * go).sum() + (f * gf).sum()

    grads = O.attention_grads(q, k, v, decay, s, go, gf)
    args = [q, k, v, s]
    for i, g in enumerate(grads):
        u = rng.normal(size=g.shape)
        moved = [a + u if j == i else a for j, a in enumerate(args)]
        assert np.isclose(loss(*moved) - loss(*args), (g * u).sum(), rtol=1e-10)
