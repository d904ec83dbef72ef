"""Calls of the training operators' C side that the Python one does not make."""
import ctypes as C

import pytest
import torch

from test_train_attention_gpu import TYPES, Case
from test_train_paths_gpu import python_path  # noqa: F401
import turbodeberta_amd.ops.trainable_attention as T
from turbodeberta_amd import _lib

pytestmark = pytest.mark.gpu


def random(*shape, dtype=torch.float32, n=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()


def attention(fields, dtype):
    """Results and gradients of one call without tables, with these fields set."""
    q, k, v, dout = (random(2, 3, 150, 32, dtype=dtype, n=n) for n in range(4))
    o, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
    lse = torch.empty(3, 300, device="cuda")
    a = T._args(q, k, v, o, None, lse, None, None, None, None, 150, 0.2, 0, 0, 0, None)
    T._fill(a, dout=dout, dq=dq, dk=dk, dv=dv)
    for name, x in fields.items():
        setattr(a, name, x)
    a.workspace_bytes = _lib.load().tdb_attn_train_workspace(C.byref(a))
    work = torch.empty(a.workspace_bytes, dtype=torch.uint8, device="cuda")
    a.workspace = work.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.load().tdb_attn_train_fwd(C.byref(a), stream))
    _lib.check(_lib.load().tdb_attn_train_bwd(C.byref(a), stream))
    return o, lse, dq, dk, dv


@pytest.mark.parametrize("dtype", TYPES)
def test_a_tables_fields_without_tables_change_nothing(dtype):
    lut = torch.arange(4096, dtype=torch.int32, device="cuda")
    want = attention({}, dtype)
    for fields in ({"delta_lut": lut.data_ptr(), "lut_half": 2047}, {"delta_lut": lut.data_ptr(), "lut_half": 0, "span": -5}):
        assert all(torch.equal(a, b) for a, b in zip(attention(fields, dtype), want))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_loose_bound_of_packed_lengths_changes_nothing(dtype):
    c = Case([100, 0, 70], dtype=dtype, p=0.1, seed=31)
    tight = c.packed(170)
    for loose in (171, 5000, 1 << 17):
        got = c.packed(loose)
        assert all(torch.equal(got[n], tight[n]) for n in tight)
    c.check(tight)


@pytest.mark.parametrize("path", ["native", "python"])
def test_buckets_that_run_backwards(path, python_path):  # noqa: F811
    """Taken where no sequence is long enough to meet them, refused else."""
    if path == "python":
        python_path()
    c = Case([129, 40], dtype=torch.float32, buckets=256, max_rel=129, p=0.1, seed=32)
    c.check(c.packed(129))
    c.check(c.unpad(c.padded(129), 129))
    short = Case([40, 60], buckets=256, max_rel=129, seed=33)
    short.check(short.packed(1000))                     # 100 tokens in all
    for refused in (lambda: c.packed(130), lambda: c.padded(130), lambda: c.packed(5000)):
        with pytest.raises(ValueError, match="up to 129 tokens"):
            refused()


@pytest.mark.parametrize("dtype", TYPES)
def test_contiguous_tensors_that_cannot_be_addressed(dtype):
    """Inputs, tables and the gradient at odd addresses, and rows of one token with strides of no size: as their copies."""
    def odd(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return room.copy_(t)

    def grads(*t):
        leaves = [x.detach().requires_grad_() for x in t[:5]]
        o = T.trainable_attention_with_disentangled(*leaves, 0.2, 8, 32)
        return [o.detach(), *torch.autograd.grad(o, leaves, t[5])]

    for length, change in ((33, odd), (1, odd), (1, lambda t: t.as_strided(t.shape, (*t.stride()[:2], 0, 1)) if t.dim() == 4 else t)):
        t = [random(2, 3, length, 16, dtype=dtype, n=n) for n in range(3)] + [random(3, 16, 16, dtype=dtype, n=n) for n in (3, 4)] + [random(2, 3, length, 16, dtype=dtype, n=5)]
        want = grads(*t)
        for some in ([0], [1], [2], [3], [4], [5], range(6)):
            got = grads(*(change(x) if n in some else x for n, x in enumerate(t)))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (length, some)


@pytest.mark.parametrize("path", ["native", "python"])
def test_tables_with_a_leading_1_are_the_operators_own_leaves(path, python_path):  # noqa: F811
    """Nothing stands between such a leaf and the operator's node, which looks at the streams of its leaves; gradients have the leaf's shape."""
    if path == "python":
        python_path()
    q = random(2, 3, 40, 16)
    tables = [random(1, 3, rows, 16, n=rows).requires_grad_() for rows in (16, 19)]
    plain = [t.detach()[0].requires_grad_() for t in tables]
    call = lambda pk, pq: T.trainable_attention_with_disentangled(q, q, q, pk, pq, 0.2, 8, 32)
    o = call(*tables)
    leaves = [f.variable for f, _ in o.grad_fn.next_functions if f is not None]
    assert len(leaves) == 2 and all(a is b for a, b in zip(leaves, tables))
    want = torch.autograd.grad(call(*plain), plain, random(2, 3, 40, 16, n=9))
    got = torch.autograd.grad(o, tables, random(2, 3, 40, 16, n=9))
    assert all(a.shape == t.shape and torch.equal(a[0], b) for a, b, t in zip(got, want, tables))
    none = T.trainable_attention_with_disentangled(q[:0], q[:0], q[:0], *tables, 0.2, 8, 32)
    assert all(g.shape == t.shape and not g.any() for g, t in zip(torch.autograd.grad(none.sum(), tables), tables))


@pytest.mark.parametrize("path", ["native", "python"])
def test_capture_while_an_eager_graph_of_a_table_with_a_leading_1_lives(path, python_path):  # noqa: F811
    """Refused, as for any other leaf, before autograd's engine meets the other stream."""
    if path == "python":
        python_path()
    q, dy = random(2, 3, 40, 16), random(2, 3, 40, 16, n=9)
    table = random(1, 3, 16, 16, n=1).requires_grad_()
    call = lambda: T.trainable_attention_with_disentangled(q, q, q, table, None, 0.2, 8, 32)
    earlier = call()
    want, = torch.autograd.grad(call(), table, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call()
        with pytest.raises(RuntimeError, match="holds the same leaves"):
            torch.autograd.grad(o, table, dy)
    del o, earlier
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call()
        got, = torch.autograd.grad(o, table, dy)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_of_nothing_reads_no_seed(dtype):
    x = random(1003, dtype=dtype)
    y = torch.empty_like(x)
    code = {torch.float32: _lib.TDB_F32, torch.bfloat16: _lib.TDB_BF16, torch.float16: _lib.TDB_F16}[dtype]
    _lib.check(_lib.load().tdb_dropout(x.data_ptr(), y.data_ptr(), x.numel(), code, 0, None, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(x, y)
