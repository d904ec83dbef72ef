"""Arguments of the training operators' C side, and what it asks for as workspace."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_train_cpu import _attention
from turbodeberta_amd import _lib
from turbodeberta_amd.ops import _launch, trainable_attention


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


def documented(batch, heads, max_seqlen, dtype):
    """The largest workspace that tdb_train.h speaks of for a padded batch, `few` bytes for each row and table included."""
    size, tiles = 4 if dtype == _lib.TDB_F32 else 2, -(-max_seqlen // 64)
    each = batch * tiles * tiles * 64 * 64
    gib2, kib = 2 << 30, 1 << 10
    at_once = max(1, min(heads, gib2 // (each * size)))
    scores = at_once * each * size
    sums = max(at_once * each, 96 * kib * kib, at_once * tiles * 128 * kib)
    one = max(each, tiles * 128 * kib) + each // 4
    few = 32 * batch * tiles * 64 * heads + 17 * 8 + 4 * kib
    return scores + min(sums + at_once * each // 4, max(gib2, one)) + few


@pytest.mark.parametrize("dtype", [_lib.TDB_F32, _lib.TDB_BF16])
@pytest.mark.parametrize("batch,heads,max_seqlen", [(1, 64, 1024), (1, 12, 29), (32, 12, 512), (4, 12, 4096), (1, 65535, 64), (1, 4096, 700), (300, 40, 64), (1, 16, 1 << 15), (1000, 1, 1000),
                                                    (3, 2, 4096), (1, 1, 4160), (2, 1000, 1), (70, 300, 130)])
def test_the_documented_bounds(batch, heads, max_seqlen, dtype):
    need = workspace(batch=batch, heads=heads, max_seqlen=max_seqlen, lut_half=1 << 20, dtype=dtype)
    assert 0 < need <= documented(batch, heads, max_seqlen, dtype)


def test_many_heads_sums_come_in_rounds():
    """One tile for each of 65535 heads: 8 KiB of scores, 64 KiB of sums by relative position."""
    need = workspace(batch=1, heads=65535, max_seqlen=64, lut_half=1 << 20)
    assert need < 2.4 * 2 ** 30


@pytest.mark.parametrize("buckets,max_rel,longest", [(256, 512, None), (0, 64, None), (256, 130, None), (8, 6, None), (256, 129, 129), (256, 64, 129), (32, 16, 17), (32, 17, 17), (4, 3, 3)])
def test_buckets_that_run_backwards_are_refused(buckets, max_rel, longest):
    """Where max_rel - 1 <= buckets / 2 the logarithm's sign turns: rows are met again, and no run of positions has them."""
    table = _lib.delta_table(512, buckets, max_rel).astype(int)
    falls = lambda l: (np.diff(table[511 - (l - 1):511 + l]) < 0).any()
    device = torch.device("cpu")
    _launch.require_rising(device, 512, longest or 512, buckets, max_rel)
    assert not falls(longest or 512)
    if longest:
        assert falls(longest + 1)
        for reach in (longest + 1, 300):
            with pytest.raises(ValueError, match=f"run backwards.* up to {longest} tokens"):
                _launch.require_rising(device, 512, reach, buckets, max_rel)


def odd_tensors():
    """Contiguous, and nothing that the kernels can address: at an odd address; single rows with strides of no size."""
    yield torch.randn(2 * 3 * 5 * 8 + 1)[1:].view(2, 3, 5, 8)
    yield torch.randn(64).as_strided((2, 3, 1, 8), (24, 8, 0, 1))
    yield torch.randn(64).as_strided((2, 3, 1, 8), (24, 8, 3, 1))
    yield torch.randn(64).as_strided((2, 3, 1, 8), (24, 8, 1 << 30, 1))
    yield torch.randn(8).as_strided((1, 1, 1, 8), (1, 5, 0, 1))
    yield torch.randn(41)[1:].view(5, 1, 8)
    yield torch.randn(24).as_strided((1, 3, 8), (0, 8, 1))


@pytest.mark.parametrize("t", odd_tensors(), ids=lambda t: f"{tuple(t.shape)}-{t.stride()}")
def test_contiguous_tensors_that_cannot_be_addressed_are_copied(t):
    assert t.is_contiguous()
    got = trainable_attention._apart(t)
    assert torch.equal(got, t) and _launch.rows_ok(got) and got.shape[-1] <= got.stride(-2 if t.dim() == 4 else 0) <= 64


def test_tables_at_an_odd_address_are_copied():
    t = torch.randn(3 * 16 * 8 + 1)[1:].view(3, 16, 8)
    got = _launch.as_rows(t)
    assert torch.equal(got, t) and _launch.rows_ok(got)


def test_dropout_of_nothing_needs_no_seed():
    """(Without a GPU the launch fails.)"""
    f, name = _lib.load().tdb_dropout, lambda rc: _lib.ERROR_NAMES.get(rc)
    assert name(f(4096, 4096, 5, _lib.TDB_F32, 1, None, None)) == "TDB_ERR_NULL"
    if not torch.cuda.is_available():
        assert name(f(4096, 4096, 5, _lib.TDB_F32, 0, None, None)) not in ("TDB_ERR_NULL", "TDB_OK")
