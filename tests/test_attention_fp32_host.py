"""Refusals of the fp32 entry points of the linear attention, without a GPU."""

import pytest

from lava_dl_b200 import _native


def refused(name, *args):
    lib = _native.load()
    assert getattr(lib, name)(*args) == -1, name
    return _native.last_error()


@pytest.mark.parametrize('heads, H, nd, dk, dv, T, text', [
    (-2, 2, 2, 8, 8, 5, 'negative'), (4, 2, 2, 129, 8, 5, 'widths'), (3, 2, 2, 8, 8, 5, 'multiple'),
    (4, 2, 3, 8, 8, 5, 'decay'), (4, 2, 2, 8, 8, 1 << 31, 'large'), (4, 2, 2, 8, 8, 5, 'null')])
def test_entries_refuse(heads, H, nd, dk, dv, T, text):
    shape = (heads, H, dk, dv, T, None)
    assert text in refused('sb_linear_attention_fwd_fp32', *((None,) * 4 + (nd, None, None, None) + shape))
    assert text in refused('sb_linear_attention_bwd_fp32', *((None,) * 4 + (nd,) + (None,) * 7 + shape))


def test_nothing_to_do():
    assert _native.load().sb_linear_attention_fwd_fp32(*((None,) * 4 + (1, None, None, None, 0, 1, 8, 8, 5, None))) == 0
