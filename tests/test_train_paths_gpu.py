"""The training operators' native front and the Python path behind it, and calls that reach their corners: gradients of some inputs only, gradients that arrive in odd shapes, hooks."""
import pytest
import torch

import turbodeberta_amd._lib as _lib
from test_train_attention_gpu import Case, TYPES
from turbodeberta_amd.ops.dropout import dropout
from turbodeberta_amd.ops.layer_norm import dropout_add_layer_norm, layer_norm
from turbodeberta_amd.ops.trainable_attention import trainable_attention_with_disentangled as fixed
from turbodeberta_amd.ops.trainable_attention import trainable_attention_with_disentangled_varlen as varlen

pytestmark = pytest.mark.gpu
SEED = 1234567890123


class PythonOnly:
    """The native front, taking none of the training operators' calls."""

    def __getattr__(self, name):
        return (lambda *a: None) if name.startswith("train_") else getattr(_host, name)


_host = None


@pytest.fixture
def python_path(monkeypatch):
    global _host
    _host = _lib.host()
    return lambda: monkeypatch.setattr(_lib, "host", lambda: PythonOnly())


def seed():
    return torch.tensor([SEED], device="cuda")


def random(*shape, dtype=torch.float32, n=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()


def calls(dtype):
    """name -> (function, inputs)"""
    s = seed()
    x, r, w, b = random(37, 96, dtype=dtype), random(37, 96, dtype=dtype, n=1), random(96, dtype=dtype, n=2), random(96, dtype=dtype, n=3)
    q, k, v = (random(2, 3, 90, 24, dtype=dtype, n=n) for n in (4, 5, 6))
    pk, pq = (random(3, 16, 24, dtype=dtype, n=n) for n in (7, 8))
    lens = torch.tensor([90, 41], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 50, 50, 180], dtype=torch.int32).cuda()
    tokens = lambda t: t.transpose(1, 2).reshape(180, 3, 24)
    return {
        "dropout": (lambda x: dropout(x, 0.3, s), [x]),
        "layer_norm": (layer_norm, [x, w, b]),
        "plain_layer_norm": (layer_norm, [x]),
        "add_norm": (lambda *a: dropout_add_layer_norm(*a, p=0.3, seed=s), [x, r, w, b]),
        "attention": (lambda *a: fixed(*a, 0.2, 8, 32, seqlens_k=lens, dropout_p=0.2, seed=s), [q, k, v, pk, pq]),
        "packed_attention": (lambda *a: varlen(*a, cu, 130, 0.2, 8, 32, dropout_p=0.2, seed=s), [*map(tokens, (q, k, v)), pk, pq]),
    }


NAMES = ["dropout", "layer_norm", "plain_layer_norm", "add_norm", "attention", "packed_attention"]


def run(name, dtype, wanted=None, gradient=None):
    """(result, gradients, None where not wanted)"""
    fn, inputs = calls(dtype)[name]
    inputs = [t.clone().requires_grad_(wanted is None or wanted[i]) for i, t in enumerate(inputs)]
    y = fn(*inputs)
    dy = random(*y.shape, dtype=dtype, n=9) if gradient is None else gradient(y)
    y.backward(dy)
    return y.detach(), [t.grad for t in inputs]


def same(a, b):
    return torch.equal(a[0], b[0]) and all(x is y is None or torch.equal(x, y) for x, y in zip(a[1], b[1]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", NAMES)
def test_both_paths_give_the_same_bits(name, dtype, python_path):
    native = run(name, dtype)
    python_path()
    assert same(native, run(name, dtype))


@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("name", ["layer_norm", "add_norm", "attention"])
def test_gradients_of_some_inputs(name, path, python_path):
    y, grads = run(name, torch.float32)
    if path == "python":
        python_path()
    for mask in range(1, 1 << len(grads)):
        wanted = [bool(mask >> i & 1) for i in range(len(grads))]
        got = run(name, torch.float32, wanted)
        assert same(got, (y, [g if w else None for g, w in zip(grads, wanted)]))


@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("name", NAMES)
def test_gradients_that_arrive_in_odd_shapes(name, path, python_path):
    if path == "python":
        python_path()
    flat = lambda y: torch.full(y.shape, 0.5, device="cuda")
    expanded = lambda y: torch.full((1,) * y.dim(), 0.5, device="cuda").expand(y.shape)
    assert same(run(name, torch.float32, gradient=flat), run(name, torch.float32, gradient=expanded))
    turned = lambda y: random(*y.shape, n=9).transpose(0, -1).contiguous().transpose(0, -1)
    apart = lambda y: torch.nn.functional.pad(random(*y.shape, n=9), (1, 2))[..., 1:-2]
    want = run(name, torch.float32)
    assert same(run(name, torch.float32, gradient=turned), want)
    # Rows at odd addresses go to another kernel of LayerNorm's, which adds up in another order.  A sum of n <= 96 terms is off by n U of their sizes' sum, a gradient has three of
    # them and ten roundings, and the sizes' sum of 37 random terms is sqrt(37) times theirs: 300 x 2^-24 x 6 of the norm.
    y, grads = run(name, torch.float32, gradient=apart)
    assert torch.equal(y, want[0])
    for got, ref in zip(grads, want[1]):
        assert torch.equal(got, ref) if "norm" not in name else (got - ref).norm() <= 1.1e-4 * ref.norm()


@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("name", NAMES)
def test_a_second_gradient_is_refused(name, path, python_path):
    if path == "python":
        python_path()
    fn, inputs = calls(torch.float32)[name]
    inputs = [t.requires_grad_() for t in inputs]
    grads = torch.autograd.grad(fn(*inputs).square().sum(), inputs, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        sum(g.sum() for g in grads).backward()


@pytest.mark.parametrize("name", NAMES)
def test_hooks_of_saved_tensors(name):
    want = run(name, torch.bfloat16)
    with torch.autograd.graph.save_on_cpu():
        assert same(run(name, torch.bfloat16), want)

    class Refused(Exception):
        pass

    def refuse(t):
        raise Refused("what a hook raises passes through")

    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t), pytest.raises(Refused):
        run(name, torch.bfloat16)


def test_graphs_used_more_than_once():
    """Two calls of the same inputs alive at once, and a backward pass run again."""
    for name in NAMES:
        fn, inputs = calls(torch.float32)[name]
        inputs = [t.requires_grad_() for t in inputs]
        a, b = fn(*inputs), fn(*inputs)
        dy = random(*a.shape, n=9)
        first = torch.autograd.grad(b, inputs, dy, retain_graph=True)
        assert all(torch.equal(x, y) for x, y in zip(first, torch.autograd.grad(a, inputs, dy)))
        assert all(torch.equal(x, y) for x, y in zip(first, torch.autograd.grad(b, inputs, dy)))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(b, inputs, dy)


def test_the_same_tensor_in_several_places():
    x = random(20, 64, n=1)
    a = x.clone().requires_grad_()
    y = dropout_add_layer_norm(a, a, p=0.25, seed=seed())
    dy = random(20, 64, n=2)
    y.backward(dy)
    b, c = x.clone().requires_grad_(), x.clone().requires_grad_()
    dropout_add_layer_norm(b, c, p=0.25, seed=seed()).backward(dy)
    assert torch.equal(a.grad, b.grad + c.grad)
    q, pos = random(1, 2, 50, 16, n=3), random(2, 8, 16, n=4)
    one, table = q.clone().requires_grad_(), pos.clone().requires_grad_()
    fixed(one, one, one, table, table, 0.2, 4, 16).sum().backward()
    three, two = [q.clone().requires_grad_() for _ in range(3)], [pos.clone().requires_grad_() for _ in range(2)]
    fixed(*three, *two, 0.2, 4, 16).sum().backward()
    # each a sum of the same three or two numbers in some order: two roundings of partial sums, none larger than the sum of the sizes
    for got, parts in ((one.grad, three), (table.grad, two)):
        bound = 2 * 2 ** -24 * sum(t.grad.abs() for t in parts)
        assert ((got.double() - sum(t.grad.double() for t in parts)).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,buckets,max_rel", [([1000], 8, 4000), ([1000, 130], 16, 4000), ([330, 0, 450, 64, 129], 16, 64), ([64] * 9 + [300], 4, 16), ([500], 0, 1)])
def test_tiles_of_one_table_row(lens, buckets, max_rel, dtype):
    """In the middle of the tables as well as past their ends; several sequences of a diagonal for a workgroup and the other way round."""
    c = Case(lens, H=1 if lens[0] > 900 else 2, dtype=dtype, buckets=buckets, max_rel=max_rel, p=0.1, seed=21)
    c.check(c.packed())
    c.check(c.unpad(c.padded(max(lens)), max(lens)))


class Look(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, seen):
        ctx.seen = seen
        return x.clone()

    @staticmethod
    def backward(ctx, dy):
        ctx.seen.append(_lib.host().backward_begins())
        return dy, None


def test_a_leaf_that_belongs_to_another_stream_is_seen():
    side = torch.cuda.Stream()
    for alive in (False, True):
        x = random(8, 64).requires_grad_()
        earlier = x * 2 if alive else None
        side.wait_stream(torch.cuda.current_stream())
        seen = []
        with torch.cuda.stream(side):
            Look.apply(x, seen).sum().backward()
        torch.cuda.synchronize()
        assert seen == [alive] and (earlier is not None) == alive


@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("name", ["dropout", "layer_norm", "attention"])
def test_capture_while_an_eager_graph_of_the_same_leaves_lives(name, path, python_path):
    """Refused before autograd's engine meets the other stream; possible once that graph is gone, also by the same leaves."""
    if path == "python":
        python_path()
    want = run(name, torch.float32)
    fn, inputs = calls(torch.float32)[name]
    inputs = [t.requires_grad_() for t in inputs]
    earlier = fn(*inputs)
    dy = random(*earlier.shape, n=9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fn(*inputs)
        with pytest.raises(RuntimeError, match="holds the same leaves"):
            torch.autograd.grad(y, inputs, dy)
    del y, earlier
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fn(*inputs)
        grads = torch.autograd.grad(y, inputs, dy)
    for _ in range(3):
        for t in (y, *grads):
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same((y.detach(), list(grads)), want)


def test_offsets_past_32_bits():
    """Tensors of more than 2^32 bytes and 2^31 values; what is not looked at is not written first."""
    n = (1 << 31) + 72
    x = torch.empty(n, dtype=torch.float16, device="cuda")
    y = torch.empty_like(x)
    ends = [slice(0, 64), slice((1 << 31) - 64, n)]
    for e in ends:
        x[e] = 1.0
    _lib.check(_lib.load().tdb_dropout(x.data_ptr(), y.data_ptr(), n, _lib.TDB_F16, 1 << 15, seed().data_ptr(), torch.cuda.current_stream().cuda_stream))
    import numpy as np
    import train_reference as R
    for e in ends:
        at = np.arange(e.start, e.stop)
        u = R.numbers(((at // 8 & 0xffffffff).astype(np.uint64), (at // 8 >> 32).astype(np.uint64), np.zeros(len(at), np.uint64), np.zeros(len(at), np.uint64)), SEED)
        assert torch.equal(y[e].cpu().double(), R.factors(u[np.arange(len(at)), at % 8], 0.5))
    del x, y
    rows, hidden = (1 << 31) // 2048 + 5, 2048
    x = torch.empty(rows, hidden, dtype=torch.float16, device="cuda")
    x[-7:] = random(7, hidden, dtype=torch.float16)
    assert torch.equal(layer_norm(x)[-7:], layer_norm(x[-7:].clone()))
    del x
    torch.cuda.empty_cache()


def test_attention_offsets_past_32_bits():
    """A batch of 2100 whose first and last sequence have tokens: 4.4 GB for q alone; the last one's results are those it has by itself."""
    B, H, L, D = 2100, 8, 2048, 64
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens[0], lens[-1] = 100, 130
    big = [torch.empty(B, H, L, D, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    small = [random(1, H, 130, D, dtype=torch.bfloat16, n=n) for n in range(4)]
    for t, s in zip(big, small):
        t[0, :, :100], t[-1, :, :130] = s[0, :, :100], s[0]
    tables = [random(H, 32, D, dtype=torch.bfloat16, n=n) for n in (5, 6)]

    def grads(q, k, v, dout, n):
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        o = fixed(q, k, v, *tables, 0.1, 16, 64, seqlens_k=n)
        return [o, *torch.autograd.grad(o, (q, k, v), dout)]

    got = [t[-1, :, :130].clone() for t in grads(*big, lens)]
    want = grads(*(s.clone() for s in small), lens[-1:].clone())
    assert all(torch.equal(a, b[0]) for a, b in zip(got, want))
    del big
    torch.cuda.empty_cache()


def test_threads_with_streams_of_their_own():
    """Two calls of every operator at once."""
    import threading
    want = {name: run(name, torch.bfloat16) for name in NAMES}
    torch.cuda.synchronize()
    wrong = []

    def work(names):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for name in names:
                got = run(name, torch.bfloat16)
                stream.synchronize()
                if not same(got, want[name]):
                    wrong.append(name)

    threads = [threading.Thread(target=work, args=(names,)) for names in (NAMES * 5, NAMES[::-1] * 5)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
