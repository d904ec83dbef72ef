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
