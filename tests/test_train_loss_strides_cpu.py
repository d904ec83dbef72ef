"""What the C ABI's loss takes as the distance of dweight's rows: a tile's rows are addressed within one buffer of 32 bits, as weight's are."""
import ctypes as C

import pytest

from test_train_loss_cpu import _loss
from turbodeberta_amd import _lib


@pytest.mark.parametrize("dtype,size", [(_lib.TDB_F32, 4), (_lib.TDB_BF16, 2), (_lib.TDB_F16, 2)])
def test_rows_of_dweight_too_far_apart(dtype, size):
    lib = _lib.load()
    most = (1 << 22) // size
    code = lambda **kw: _lib.ERROR_NAMES[lib.tdb_loss_bwd(C.byref(_loss(dtype=dtype, **kw)), None)]
    for stride in (most + 1, 1 << 26, 1 << 31, 1 << 40, 1 << 62):
        assert code(dweight_stride=stride) == "TDB_ERR_STRIDE"
        assert "dweight_stride" in lib.tdb_last_error().decode()
        # not looked at where dweight is not asked for, or forward (nothing is launched: the workspace is too small)
        assert code(dweight_stride=stride, dweight=None, workspace_bytes=0) == "TDB_ERR_SHAPE"
        assert _lib.ERROR_NAMES[lib.tdb_loss_fwd(C.byref(_loss(dtype=dtype, dweight_stride=stride, workspace_bytes=0)), None)] == "TDB_ERR_SHAPE"
    assert code(dweight_stride=most, workspace_bytes=0) == "TDB_ERR_SHAPE"


@pytest.mark.parametrize("dtype,size", [(_lib.TDB_F32, 4), (_lib.TDB_BF16, 2), (_lib.TDB_F16, 2)])
def test_rows_of_weight_too_far_apart(dtype, size):
    """Distances whose bytes wrap around in 64 bits among them."""
    lib = _lib.load()
    for fn in (lib.tdb_loss_fwd, lib.tdb_loss_bwd):
        code = lambda stride: _lib.ERROR_NAMES[fn(C.byref(_loss(dtype=dtype, weight_stride=stride, workspace_bytes=0)), None)]
        for stride in ((1 << 22) // size + 4, 1 << 40, 1 << 61, (1 << 62) + 64, (1 << 63) - 64):
            assert code(stride) == "TDB_ERR_STRIDE"
        assert code((1 << 22) // size) == "TDB_ERR_SHAPE"
