"""Arguments of the training operators' C side, and what it asks for as workspace."""
import ctypes as C

import pytest

from test_train_cpu import _attention
from turbodeberta_amd import _lib


def workspace(**kw):
    return _lib.load().tdb_attn_train_workspace(C.byref(_attention(**kw)))


NONE = dict(pos_key=None, pos_query=None)


@pytest.mark.parametrize("kw", [dict(span=0), dict(span=-(1 << 30)), dict(span=1 << 30), dict(lut_half=0), dict(delta_lut=None), dict(span=1 << 20, lut_half=1 << 20)])
def test_a_tables_fields_without_tables_change_nothing(kw):
    """The backward pass once looked up what delta_lut points to, by lut_half, and laid out span row starts."""
    assert workspace(**NONE) == workspace(**NONE, **kw) > 0


def test_a_bad_span_needs_no_workspace():
    assert workspace() > 0
    for span in (0, -1, (1 << 20) + 1):
        assert workspace(span=span) == workspace(span=span, pos_key=None) == 0


@pytest.mark.parametrize("total", [1, 63, 200, 5000])
def test_a_loose_bound_of_packed_lengths_costs_no_workspace(total):
    tight = workspace(cu_seqlens=4096, total_tokens=total, max_seqlen=total, lut_half=1 << 20)
    for loose in (total + 1, 32768, 1 << 20):
        assert workspace(cu_seqlens=4096, total_tokens=total, max_seqlen=loose, lut_half=1 << 20) == tight > 0
    if total > 64:
        assert workspace(cu_seqlens=4096, total_tokens=total, max_seqlen=64, lut_half=1 << 20) < tight
