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


def _attention(**kw):
    """Arguments of a call that would be launched; pointers that nothing looks at."""
    B, H, D, L = 2, 3, 64, 100
    a = dict(dtype=_lib.TDB_BF16, batch=B, heads=H, head_dim=D, max_seqlen=L, threshold=6554, span=8, lut_half=511, sm_scale=0.1, delta_lut=4096, seed=4096, lse=4096, workspace=4096,
             workspace_bytes=1 << 40, pos_key=4096, pos_query=4096, dpos_key=4096, dpos_query=4096, o_rest=4096)
    for t in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        a.update({t: 4096, t + "_stride_b": H * L * D, t + "_stride_h": L * D, t + "_stride_l": D})
    for t in ("pos_key", "pos_query"):
        a.update({t + "_stride_h": 16 * D, t + "_stride_r": D, "d" + t + "_stride_h": 16 * D})
    a.update(kw)
    return _lib.TrainAttnArgs(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(dtype=7), "TDB_ERR_DTYPE"), (dict(batch=-1), "TDB_ERR_SHAPE"), (dict(heads=0), "TDB_ERR_SHAPE"), (dict(heads=65536), "TDB_ERR_SHAPE"),
    (dict(head_dim=60), "TDB_ERR_SHAPE"), (dict(head_dim=0), "TDB_ERR_SHAPE"), (dict(head_dim=72), "TDB_ERR_SHAPE"), (dict(max_seqlen=0), "TDB_ERR_SHAPE"),
    (dict(max_seqlen=(1 << 20) + 1), "TDB_ERR_SHAPE"), (dict(total_tokens=-1), "TDB_ERR_SHAPE"), (dict(threshold=-1), "TDB_ERR_SHAPE"), (dict(threshold=65537), "TDB_ERR_SHAPE"),
    (dict(sm_scale=0.0), "TDB_ERR_SHAPE"), (dict(sm_scale=float("nan")), "TDB_ERR_SHAPE"), (dict(sm_scale=float("inf")), "TDB_ERR_SHAPE"),
    (dict(batch=1 << 21), "TDB_ERR_SHAPE"), (dict(cu_seqlens=4096, total_tokens=1 << 27), "TDB_ERR_SHAPE"),
    (dict(q=None), "TDB_ERR_NULL"), (dict(k=None), "TDB_ERR_NULL"), (dict(v=None), "TDB_ERR_NULL"), (dict(o=None), "TDB_ERR_NULL"), (dict(lse=None), "TDB_ERR_NULL"),
    (dict(seed=None), "TDB_ERR_NULL"), (dict(q=4104), "TDB_ERR_ALIGN"), (dict(pos_key=4098), "TDB_ERR_ALIGN"), (dict(o_rest=4104), "TDB_ERR_ALIGN"),
    (dict(q_stride_b=-64), "TDB_ERR_STRIDE"), (dict(k_stride_h=68), "TDB_ERR_STRIDE"), (dict(v_stride_l=56), "TDB_ERR_STRIDE"), (dict(o_stride_l=1 << 24), "TDB_ERR_STRIDE"),
    (dict(pos_query_stride_r=60), "TDB_ERR_STRIDE"), (dict(pos_key_stride_r=1 << 27), "TDB_ERR_STRIDE"), (dict(span=0), "TDB_ERR_POSITION"), (dict(span=(1 << 20) + 1), "TDB_ERR_POSITION"),
    (dict(delta_lut=None), "TDB_ERR_POSITION"), (dict(lut_half=98), "TDB_ERR_POSITION"),
])
def test_attention_refusals(kw, err):
    lib = _lib.load()
    for fn in (lib.tdb_attn_train_fwd, lib.tdb_attn_train_bwd):
        assert _lib.ERROR_NAMES[fn(C.byref(_attention(**kw)), None)] == err


def test_attention_refusals_of_one_direction_and_calls_with_nothing_to_do():
    lib = _lib.load()
    back = lambda **kw: _lib.ERROR_NAMES[lib.tdb_attn_train_bwd(C.byref(_attention(**kw)), None)]
    for name in ("dout", "dq", "dk", "dv", "workspace", "dpos_key", "dpos_query"):
        assert back(**{name: None}) == "TDB_ERR_NULL"
    assert back(dq_stride_l=56) == "TDB_ERR_STRIDE" and back(dpos_key_stride_h=-64) == "TDB_ERR_STRIDE"
    assert back(dpos_query_stride_h=16 * 64 - 64) == "TDB_ERR_STRIDE"                     # heads' tables that overlap
    for name in ("dq", "dk", "dv"):                                                       # results that do
        assert back(**{name + "_stride_h": 0}) == "TDB_ERR_STRIDE" and back(**{name + "_stride_b": 0}) == "TDB_ERR_STRIDE"
    assert _lib.ERROR_NAMES[lib.tdb_attn_train_fwd(C.byref(_attention(o_stride_h=0)), None)] == "TDB_ERR_STRIDE"
    need = lib.tdb_attn_train_workspace(C.byref(_attention()))
    assert back(workspace_bytes=need - 1) == "TDB_ERR_SHAPE"
    assert _lib.ERROR_NAMES[lib.tdb_attn_train_fwd(None, None)] == _lib.ERROR_NAMES[lib.tdb_attn_train_bwd(None, None)] == "TDB_ERR_NULL"
    for fn in (lib.tdb_attn_train_fwd, lib.tdb_attn_train_bwd):
        assert fn(C.byref(_attention(batch=0, q=None)), None) == 0 and fn(C.byref(_attention(cu_seqlens=4096, total_tokens=0, q=None)), None) == 0


def test_attention_workspace():
    """The scores' gradients of all heads, up to 2 GiB, and of one head at least; nothing for what would be refused."""
    lib = _lib.load()
    need = lambda **kw: lib.tdb_attn_train_workspace(C.byref(_attention(**kw)))
    assert lib.tdb_attn_train_workspace(None) == 0 and need(max_seqlen=0) == 0 and need(head_dim=4) == 0 and need(batch=-1) == 0 and need(heads=0) == 0
    scores = 2 * 3 * 2 * 2 * 64 * 64 * 2            # sequences, heads, tiles of rows, tiles of columns, values, bytes
    assert scores <= need() <= scores + (8 << 20)
    rows = 27 * 2 * 3 * 4 + 256                     # a number for each row more, rounded up
    assert 0 <= need(max_seqlen=128) - need(max_seqlen=101) <= rows and need(max_seqlen=129) > need(max_seqlen=128) + scores
    one = 1 * 512 * 512 * 64 * 64 * 2               # a head of one sequence of 32768 tokens: 2 GiB
    assert one <= need(batch=1, max_seqlen=1 << 15, lut_half=1 << 15) < 1.5 * one
    assert need(batch=1, max_seqlen=1 << 15, lut_half=1 << 15, heads=16) < 1.6 * one
