"""The loss over a vocabulary and the gradient norm without a GPU: what the C ABI refuses, sizes of its buffers, CPU tensors."""
import ctypes as C

import pytest
import torch

from turbodeberta_amd import _lib

BIG = 1 << 50


def _loss(**kw):
    """Arguments of a call that would be launched; pointers that nothing looks at."""
    a = _lib.LossArgs(dtype=_lib.TDB_BF16, bias_dtype=_lib.TDB_F32, hidden=64, reduction=2, rows=100, vocab=1000, ignore_index=-100, x_stride=64, weight_stride=64, dloss_stride=0, dx_stride=64,
                      dweight_stride=64, state_bytes=BIG, workspace_bytes=BIG, **{n: 4096 for n in ("x", "weight", "bias", "labels", "loss", "state", "workspace", "dloss", "dx", "dweight", "dbias")})
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,err", [
    (dict(dtype=7), "TDB_ERR_DTYPE"), (dict(bias_dtype=_lib.TDB_F16), "TDB_ERR_DTYPE"), (dict(hidden=0), "TDB_ERR_SHAPE"), (dict(hidden=32769), "TDB_ERR_SHAPE"), (dict(rows=-1), "TDB_ERR_SHAPE"),
    (dict(rows=(1 << 27) + 1), "TDB_ERR_SHAPE"), (dict(vocab=0), "TDB_ERR_SHAPE"), (dict(vocab=(1 << 27) + 1), "TDB_ERR_SHAPE"), (dict(reduction=3), "TDB_ERR_SHAPE"), (dict(reduction=-1), "TDB_ERR_SHAPE"),
    (dict(weight=None), "TDB_ERR_NULL"), (dict(state=None), "TDB_ERR_NULL"), (dict(workspace=None), "TDB_ERR_NULL"), (dict(weight=4098), "TDB_ERR_ALIGN"), (dict(state=4104), "TDB_ERR_ALIGN"),
    (dict(workspace=4097), "TDB_ERR_ALIGN"), (dict(weight_stride=60), "TDB_ERR_STRIDE"), (dict(weight_stride=67), "TDB_ERR_STRIDE"), (dict(weight_stride=-64), "TDB_ERR_STRIDE"),
    (dict(weight_stride=(1 << 21) + 8), "TDB_ERR_STRIDE"), (dict(hidden=65), "TDB_ERR_STRIDE"), (dict(state_bytes=100), "TDB_ERR_SHAPE"), (dict(workspace_bytes=100), "TDB_ERR_SHAPE"),
])
def test_refusals_of_both_directions(kw, err):
    lib = _lib.load()
    for fn in (lib.tdb_loss_fwd, lib.tdb_loss_bwd):
        assert _lib.ERROR_NAMES[fn(C.byref(_loss(**kw)), None)] == err
        assert _lib.ERROR_NAMES[fn(None, None)] == "TDB_ERR_NULL"


def test_refusals_of_one_direction():
    lib = _lib.load()
    forward = lambda **kw: _lib.ERROR_NAMES[lib.tdb_loss_fwd(C.byref(_loss(**kw)), None)]
    backward = lambda **kw: _lib.ERROR_NAMES[lib.tdb_loss_bwd(C.byref(_loss(**kw)), None)]
    assert forward(x=None) == forward(labels=None) == forward(loss=None) == "TDB_ERR_NULL" and forward(x_stride=-64) == "TDB_ERR_STRIDE"
    assert backward(dloss=None) == backward(bias=None) == "TDB_ERR_NULL"
    assert backward(dloss_stride=-1) == backward(dx_stride=63) == backward(dweight_stride=63) == "TDB_ERR_STRIDE"
    state, work = lib.tdb_loss_state(C.byref(_loss())), [lib.tdb_loss_workspace(C.byref(_loss()), b) for b in (0, 1)]
    assert forward(state_bytes=state - 1) == forward(workspace_bytes=work[0] - 1) == backward(workspace_bytes=work[1] - 1) == "TDB_ERR_SHAPE"


def test_buffers():
    """The state holds the rows and a few words for each and each class; the workspace the logits' gradient up to 2 GiB, or 256 columns of it; nothing for what would be refused."""
    lib = _lib.load()
    state = lambda **kw: lib.tdb_loss_state(C.byref(_loss(**kw)))
    back = lambda **kw: lib.tdb_loss_workspace(C.byref(_loss(**kw)), 1)
    forward = lambda **kw: lib.tdb_loss_workspace(C.byref(_loss(**kw)), 0)
    assert lib.tdb_loss_state(None) == lib.tdb_loss_workspace(None, 0) == 0
    for bad in (dict(hidden=0), dict(vocab=0), dict(rows=-1), dict(dtype=9), dict(vocab=1 << 40)):
        assert state(**bad) == forward(**bad) == back(**bad) == 0
    assert 256 * 128 <= state() <= 256 * 128 + 256 * 7 * 4 + 1024 * 4 + 4096
    parts = 1024 * 256 * 64 * 4             # sums of dx: at most as many compute units
    assert 256 * 1024 * 2 <= back() <= 256 * 1024 * 2 + parts + (1 << 16)
    whole = dict(rows=16384, vocab=128100, hidden=768, dtype=_lib.TDB_BF16)
    assert back(**whole) <= (2 << 30) + (1 << 30) and forward(**whole) <= 1 << 28
    assert back(rows=1 << 24) >= (1 << 24) * 256 * 2
    assert back(reduction=0, dtype=_lib.TDB_F16) >= back(dtype=_lib.TDB_F16) + 256 * 128      # rows shifted by powers of two


def _grads(**kw):
    sizes, kinds = (C.c_int64 * 3)(100, 0, 7), (C.c_int32 * 3)(_lib.TDB_F32, _lib.TDB_BF16, _lib.TDB_F16)
    places = (C.c_void_p * 3)(4096, None, 8192)
    a = _lib.GradsArgs(tensors=3, norm=2, max_norm=1.0, to=C.addressof(places), numel=C.addressof(sizes), from_dtype=C.addressof(kinds), to_dtype=C.addressof(kinds), total=4096, workspace=4096,
                       workspace_bytes=BIG)
    setattr(a, "from", C.addressof(places))
    keep = [sizes, kinds, places]
    for k, v in kw.items():
        if isinstance(v, list):
            v = {"from": C.c_void_p, "to": C.c_void_p, "numel": C.c_int64}.get(k, C.c_int32).__mul__(3)(*v)
            keep.append(v)
            v = C.addressof(v)
        setattr(a, k, v)
    return a, keep


@pytest.mark.parametrize("kw,err", [
    (dict(tensors=-1), "TDB_ERR_SHAPE"), (dict(tensors=(1 << 20) + 1), "TDB_ERR_SHAPE"), (dict(norm=3), "TDB_ERR_SHAPE"), (dict(norm=-1), "TDB_ERR_SHAPE"), (dict(total=None), "TDB_ERR_NULL"),
    (dict(workspace=None), "TDB_ERR_NULL"), (dict(workspace=4100), "TDB_ERR_ALIGN"), (dict(workspace_bytes=8), "TDB_ERR_SHAPE"), ({"from": None}, "TDB_ERR_NULL"), (dict(numel=None), "TDB_ERR_NULL"),
    (dict(from_dtype=None), "TDB_ERR_NULL"), (dict(from_dtype=[0, 1, 5]), "TDB_ERR_DTYPE"), (dict(numel=[100, 0, -1]), "TDB_ERR_SHAPE"), (dict(numel=[100, 0, (1 << 40) + 1]), "TDB_ERR_SHAPE"),
    ({"from": [None, None, 8192]}, "TDB_ERR_NULL"), ({"from": [4098, None, 8192]}, "TDB_ERR_ALIGN"), ({"from": [4096, None, 8193]}, "TDB_ERR_ALIGN"),
])
def test_refusals_of_norm_and_clipping(kw, err):
    lib = _lib.load()
    for fn in (lib.tdb_grads_norm, lib.tdb_grads_clip):
        a, keep = _grads(**kw)
        assert _lib.ERROR_NAMES[fn(C.byref(a), None)] == err
        assert _lib.ERROR_NAMES[fn(None, None)] == "TDB_ERR_NULL"


@pytest.mark.parametrize("kw,err", [
    (dict(max_norm=-1.0), "TDB_ERR_SHAPE"), (dict(max_norm=float("nan")), "TDB_ERR_SHAPE"), (dict(to=None), "TDB_ERR_NULL"), (dict(to_dtype=None), "TDB_ERR_NULL"), (dict(to_dtype=[0, 1, 9]), "TDB_ERR_DTYPE"),
    (dict(to=[None, None, 8192]), "TDB_ERR_NULL"), (dict(to=[4097, None, 8192]), "TDB_ERR_ALIGN"), (dict(to=[4096, None, 4100]), "TDB_ERR_STRIDE"),      # a result on another one's input
    (dict(to=[20000, None, 20396]), "TDB_ERR_STRIDE"), (dict(to=[4100, None, 8192]), "TDB_ERR_STRIDE"), (dict(to_dtype=[1, 1, 2]), "TDB_ERR_STRIDE"),      # each other, shifted, of another type in place
    ({"from": [4096, None, 4200], "to": [4096, None, 30000]}, "TDB_ERR_STRIDE"),
])
def test_refusals_of_clipping(kw, err):
    a, keep = _grads(**kw)
    assert _lib.ERROR_NAMES[_lib.load().tdb_grads_clip(C.byref(a), None)] == err


def test_workspace_of_the_norm():
    lib = _lib.load()

    def need(**kw):
        a, keep = _grads(**kw)
        return lib.tdb_grads_workspace(C.byref(a))
    assert lib.tdb_grads_workspace(None) == 0 and need(tensors=-1) == 0 and need(numel=None) == 0 and need(numel=[5, -1, 5]) == 0
    assert need(numel=[0, 0, 0]) == 16 and need() == 32 and need(numel=[8193, 1, 8192]) == 16 + 8 * 4 and need(numel=[1 << 30, 1 << 30, 5]) <= 16 + 8 * 4100


def test_operators_refuse_cpu_tensors():
    from turbodeberta_amd.ops.grad_norm import clip_grad_norm_, clip_grads, grad_norm
    from turbodeberta_amd.ops.linear_cross_entropy import linear_cross_entropy
    x, w, labels = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    for call in (lambda: linear_cross_entropy(x, w, labels), lambda: grad_norm([x]), lambda: grad_norm(x), lambda: clip_grads([x], 1.0), lambda: clip_grads([x], 1.0, out=[x]),
                 lambda: clip_grad_norm_([p], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    assert grad_norm([]).item() == 0
