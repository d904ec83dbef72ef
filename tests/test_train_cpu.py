"""The training operators without a GPU: their reference's generator, what the C ABI refuses, CPU tensors."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

import train_reference as R
from turbodeberta_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_generator_gives_the_published_words():
    """Known answers of Philox-4x32 with seven and ten rounds for a counter and key of zeros and of ones (published with the method)."""
    def words(fill, rounds):
        return [int(x) for x in R.philox([np.uint64(fill)] * 4, (fill, fill), rounds)]
    assert words(0, 7) == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]
    assert words(0xffffffff, 7) == [0x5207ddc2, 0x45165e59, 0x4d8ee751, 0x8c52f662]
    assert words(0, 10) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def _declared(name):
    return open(os.path.join(ROOT, "include", name)).read()


def test_header_and_binding_agree():
    header = _declared("tdb_train.h")
    assert set(re.findall(r"^(?:int|int64_t)\s+(tdb_\w+)\s*\(", header, re.M)) == set(_lib.TRAIN_EXPORTS)
    assert all(hasattr(_lib.load(), n) for n in _lib.TRAIN_EXPORTS)
    for cname, cls in (("tdb_norm_args", _lib.NormArgs), ("tdb_train_attn_args", _lib.TrainAttnArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, re.S).group(1)
        names = []
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            decl = re.sub(r"^(const\s+)?(int32_t|int64_t|float|void|tdb_pos_args)\s*\**", "", decl.strip())
            names += [n.strip().lstrip("*").strip() for n in decl.split(",") if n.strip()]
        assert names == [f[0] for f in cls._fields_], cname


def _norm(**kw):
    a = _lib.NormArgs(_lib.TDB_F32, _lib.TDB_F32, 64, 0, 10, 1e-7, 0, *[0x1000] * 11, *[0x2000], *[64] * 6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,err", [
    (dict(dtype=7), "TDB_ERR_DTYPE"), (dict(weight_dtype=_lib.TDB_F16), "TDB_ERR_DTYPE"), (dict(hidden=0), "TDB_ERR_SHAPE"), (dict(hidden=32769), "TDB_ERR_SHAPE"),
    (dict(rows=-1), "TDB_ERR_SHAPE"), (dict(threshold=-1), "TDB_ERR_SHAPE"), (dict(threshold=65537), "TDB_ERR_SHAPE"), (dict(eps=-1.0), "TDB_ERR_SHAPE"),
    (dict(eps=float("nan")), "TDB_ERR_SHAPE"), (dict(threshold=5, seed=None), "TDB_ERR_NULL"), (dict(bias=None), "TDB_ERR_NULL"), (dict(dbias=None), "TDB_ERR_NULL"),
    (dict(x=None), "TDB_ERR_NULL"), (dict(x_stride=-64), "TDB_ERR_STRIDE"), (dict(y_stride=63), "TDB_ERR_STRIDE"), (dict(dx_stride=0), "TDB_ERR_STRIDE")])
def test_norm_refusals(kw, err):
    lib = _lib.load()
    for fn in (lib.tdb_norm_fwd, lib.tdb_norm_bwd):
        assert _lib.ERROR_NAMES[fn(C.byref(_norm(**kw)), None)] == err
    assert _lib.ERROR_NAMES[lib.tdb_norm_bwd(C.byref(_norm(workspace=None)), None)] == "TDB_ERR_NULL"
    assert _lib.ERROR_NAMES[lib.tdb_norm_fwd(None, None)] == "TDB_ERR_NULL"
    assert lib.tdb_norm_fwd(C.byref(_norm(rows=0)), None) == 0


def test_norm_workspace_covers_every_workgroup():
    f = _lib.load().tdb_norm_workspace
    assert f(0, 64) == 128 and f(1, 64) == 128 and f(100, 768) == 100 * 2 * 768 and f(1 << 30, 7) == 512 * 14 and f(-1, 7) == 0


def test_dropout_refusals():
    f = _lib.load().tdb_dropout
    name = lambda *a: _lib.ERROR_NAMES[f(*a, None)]
    assert name(0x1000, 0x1000, 5, 9, 1, 0x1000) == "TDB_ERR_DTYPE"
    assert name(0x1000, 0x1000, -5, 0, 1, 0x1000) == "TDB_ERR_SHAPE"
    assert name(0x1000, 0x1000, 5, 0, 65537, 0x1000) == "TDB_ERR_SHAPE"
    assert name(0x1000, 0x1000, 5, 0, 1, None) == "TDB_ERR_NULL"
    assert f(None, None, 0, 0, 1, None, None) == 0


def test_operators_refuse_cpu_tensors():
    from turbodeberta_amd.ops.dropout import dropout
    from turbodeberta_amd.ops.layer_norm import dropout_add_layer_norm, layer_norm
    x, w, seed = torch.zeros(4, 8), torch.zeros(8), torch.zeros(1, dtype=torch.int64)
    for call in (lambda: dropout(x, 0.1, seed), lambda: layer_norm(x, w, w), lambda: dropout_add_layer_norm(x, x, w, w, 0.1, seed)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
