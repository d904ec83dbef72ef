"""The norm of many gradients and clipping, against 64 bits."""
import math
import threading

import pytest
import torch

import turbodeberta_amd._lib as _lib
from test_train_loss_gpu import PythonOnly
from turbodeberta_amd.ops.grad_norm import clip_grad_norm_, clip_grads, grad_norm

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        host = _lib.host()
        monkeypatch.setattr(_lib, "host", lambda: PythonOnly(host))


def _rand(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _norm64(tensors, kind):
    each = torch.stack([torch.linalg.vector_norm(t.detach().double().flatten(), kind) for t in tensors if t.numel()] or [torch.zeros((), dtype=torch.float64)])
    return torch.linalg.vector_norm(each, kind).item()


def _check_norm(got, tensors, kind):
    """Sums in 64 bits: half a step of the float32 result is all that is off (and 2^-40 for the sums)."""
    ref = _norm64(tensors, kind)
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    assert abs(got.double().item() - ref) <= (U + 2.0 ** -40) * ref + 2.0 ** -149


def _check_clipped(out, grads, norm, max_norm):
    """The factor and the product, each rounded to float32, and the result to its type."""
    factor = min(1.0, max_norm / (norm + 1e-6))
    for o, t in zip(out, grads):
        ref, info = t.double() * factor, torch.finfo(o.dtype)
        assert o.shape == t.shape
        assert ((o.double() - ref).abs() <= ref.abs() * (info.eps / 2 + 2.01 * U) * (1 + 2 * U) + info.smallest_normal * info.eps).all()


SHAPES = [(1,), (3, 5), (8191,), (8192,), (8193,), (0,), (7, 0, 3), (130, 257), (), (1 << 20,), (1 << 16, 33)]


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_and_clipping(dtype, kind, path):
    grads = [_rand(n, *shape, dtype=dtype, scale=1 + n % 3) for n, shape in enumerate(SHAPES)]
    _check_norm(grad_norm(grads, kind), grads, kind)
    norm = _norm64(grads, kind)
    for to in TYPES:
        for max_norm in (0.3 * norm, 2 * norm, 0.0):
            out = [torch.full(t.shape, torch.nan, dtype=to, device="cuda") for t in grads]
            got, same = clip_grads(grads, max_norm, kind, out=out)
            _check_norm(got, grads, kind)
            assert all(a is b for a, b in zip(same, out))
            _check_clipped(out, grads, norm, max_norm)
    got, new = clip_grads(grads, 0.5 * norm, kind)
    assert all(o.dtype == t.dtype for o, t in zip(new, grads))
    _check_clipped(new, grads, norm, 0.5 * norm)


@pytest.mark.parametrize("count", [1, 127, 128, 129, 175, 176, 177, 400])
def test_many_tensors_of_mixed_types(count, path):
    """Around the number of tensors of a launch of each kind; sizes and alignments that differ from tensor to tensor."""
    flat = {t: _rand(1, 400 * 101 + 7, dtype=t) for t in TYPES}
    grads, at = [], 1
    for n in range(count):
        size = 1 + (37 * n) % 100
        grads.append(flat[TYPES[n % 3]][at:at + size])
        at += size
    grads.append(_rand(2, 123457))
    _check_norm(grad_norm(grads), grads, 2.0)
    norm = _norm64(grads, 2.0)
    out = [torch.empty(t.shape, dtype=TYPES[(n + n // 3) % 3], device="cuda") for n, t in enumerate(grads)]
    clip_grads(grads, 0.01 * norm, out=out)
    _check_clipped(out, grads, norm, 0.01 * norm)


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place(dtype, path):
    params = [torch.nn.Parameter(_rand(n, *shape, dtype=dtype)) for n, shape in enumerate(SHAPES)]
    grads = [_rand(50 + n, *shape, dtype=dtype) for n, shape in enumerate(SHAPES)]
    params.append(torch.nn.Parameter(torch.zeros(5, device="cuda")))               # without a gradient
    for p, t in zip(params, grads):
        p.grad = t.clone()
    norm = _norm64(grads, 2.0)
    before = [p.grad._version for p in params[:-1]]
    got = clip_grad_norm_(iter(params + params[:2]), 2 * norm)         # healthy; a parameter that comes twice counts once
    _check_norm(got, grads, 2.0)
    assert all(torch.equal(p.grad, t) for p, t in zip(params, grads)) and params[-1].grad is None
    got = clip_grad_norm_(params, 0.1 * norm)
    _check_norm(got, grads, 2.0)
    _check_clipped([p.grad for p in params[:-1]], grads, norm, 0.1 * norm)
    assert all(p.grad._version > v for p, v in zip(params, before))
    one = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    one.grad = torch.tensor([3.0, 0.0, 4.0], device="cuda")
    assert clip_grad_norm_(one, 1.0).item() == 5.0
    _check_clipped([one.grad], [torch.tensor([3.0, 0.0, 4.0], device="cuda")], 5.0, 1.0)


def test_as_in_pytorch(path):
    model = torch.nn.Sequential(torch.nn.Linear(70, 50), torch.nn.LayerNorm(50), torch.nn.Linear(50, 3)).cuda()
    model(_rand(1, 20, 70)).square().sum().backward()
    for kind in (2.0, 1.0, math.inf):
        mine, theirs = ([torch.nn.Parameter(p.detach().clone()) for p in model.parameters()] for _ in range(2))
        for a, b, p in zip(mine, theirs, model.parameters()):
            a.grad, b.grad = p.grad.clone(), p.grad.clone()
        a, b = clip_grad_norm_(mine, 0.7, kind), torch.nn.utils.clip_grad_norm_(theirs, 0.7, kind)
        torch.testing.assert_close(a, b, rtol=1e-6, atol=0)
        for p, q in zip(mine, theirs):
            torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)


def test_layouts(path):
    base = _rand(3, 65, 130)
    odd = [base[:, 1:], base.t(), base[::2, ::3], base[0].expand(4, 130), base.flatten()[3:2000], _rand(4, 6, 5, 4, 3).to(memory_format=torch.channels_last)]
    for kind in (2.0, 1.0, math.inf):
        _check_norm(grad_norm(odd, kind), odd, kind)
        for t in odd:
            _check_norm(grad_norm(t, kind), [t], kind)
    norm = _norm64(odd, 2.0)
    outs = [torch.empty_like(t) for t in odd]
    outs[1] = torch.empty(odd[1].shape, device="cuda")              # another order of dimensions than the gradient's
    outs[2] = torch.empty(outs[2].shape[0], 2 * outs[2].shape[1], device="cuda")[:, ::2]                  # values that lie apart
    clip_grads(odd, 0.5 * norm, out=outs)
    _check_clipped(outs, odd, norm, 0.5 * norm)
    # in place: rows that lie apart keep what is between them
    big = _rand(5, 40, 64)
    kept = big.clone()
    p = torch.nn.Parameter(torch.zeros(40, 30, device="cuda"))
    p.grad = big[:, 3:33]
    norm = _norm64([p.grad], 2.0)
    clip_grad_norm_([p], 0.25 * norm)
    _check_clipped([big[:, 3:33]], [kept[:, 3:33]], norm, 0.25 * norm)
    assert torch.equal(big[:, :3], kept[:, :3]) and torch.equal(big[:, 33:], kept[:, 33:])


def test_large_and_small_values(path):
    """No overflow and no underflow of squares; infinities and NaN as in PyTorch's."""
    for scale in (1e30, 1e-30, 2.0 ** -149):
        t = [torch.full((1000,), scale, device="cuda"), torch.full((7,), -scale, device="cuda")]
        for kind in (2.0, 1.0, math.inf):
            _check_norm(grad_norm(t, kind), t, kind)
    big = [torch.full((1 << 21,), 3e38, device="cuda")]
    assert grad_norm(big).item() == math.inf and grad_norm(big, math.inf).item() == torch.tensor(3e38).item()
    a, b = torch.tensor([1.0, math.inf, 2.0], device="cuda"), torch.tensor([1.0, 2.0], device="cuda")
    for kind in (2.0, 1.0, math.inf):
        norm, (x, y) = clip_grads([a, b], 1.0, kind)
        assert norm.item() == math.inf and x.tolist()[::2] == [0.0, 0.0] and x[1].isnan() and not y.any()
        a2 = a.clone()
        a2[0] = math.nan
        norm, out = clip_grads([a2, b], 1.0, kind)
        assert norm.isnan() and all(o.isnan().all() for o in out)
        for bad in (a, a2):
            kept = [bad.clone(), b.clone()]
            with pytest.raises(RuntimeError, match="nothing is clipped"):
                clip_grads(kept, 1.0, kind, out=kept, error_if_nonfinite=True)
            assert torch.equal(kept[1], b) and torch.equal(kept[0].isnan(), bad.isnan())
    clip_grads([b], 0.5, out=[b], error_if_nonfinite=True)
    _check_clipped([b], [torch.tensor([1.0, 2.0], device="cuda")], 5 ** 0.5, 0.5)


def test_nothing(path):
    assert grad_norm([]).item() == 0 and clip_grad_norm_([], 1.0).item() == 0 and clip_grads([], 1.0)[1] == []
    empty = [torch.zeros(0, 3, device="cuda")]
    assert grad_norm(empty).item() == 0 and clip_grads(empty, 1.0)[0].item() == 0
    zero = [torch.zeros(10, device="cuda")]
    norm, out = clip_grads(zero, 1.0)
    assert norm.item() == 0 and not out[0].any()


def test_more_than_4_gib(path):
    t = torch.zeros((1 << 31) + 77, dtype=torch.bfloat16, device="cuda")
    t[-70:], t[:3] = 2.0, -3.0
    norm = math.sqrt(70 * 4 + 27)
    assert abs(grad_norm(t).item() - norm) <= 1e-6 * norm
    assert grad_norm(t, math.inf).item() == 3 and grad_norm(t, 1.0).item() == 149
    clip_grads([t], 0.5 * norm, out=[t])
    assert t[-70:].eq(1.0).all() and t[:3].eq(-1.5).all() and not t[3:1000].any()


def test_same_bits_every_time_other_streams_and_threads():
    grads = [_rand(n, 100003, dtype=TYPES[n % 3]) for n in range(30)]
    first = [clip_grads(grads, 0.5, k) for k in (2.0, 1.0)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[k] = clip_grads(grads, 0.5, (2.0, 1.0)[k])
            torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for (norm, out), (n, o) in zip(got, first):
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(out, o))


def test_captured_and_replayed():
    grads = [_rand(n, 5000 + n, dtype=TYPES[n % 3]) for n in range(200)]
    step = lambda: clip_grads(grads, 100.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
    for n in range(4):
        for t in grads:
            t.mul_(0.5 if n % 2 else 1.5)
        norm, out = step()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, (a, b) in graphs:
            assert torch.equal(a, norm) and all(torch.equal(x, y) for x, y in zip(b, out))


def test_refusals(path):
    t = _rand(1, 100)
    for bad in (lambda: grad_norm([t], 3.0), lambda: grad_norm([t], "fro"), lambda: grad_norm([t.double()]), lambda: grad_norm([t.to_sparse()]), lambda: grad_norm([t, t.cpu()]),
                lambda: grad_norm([t, 5]), lambda: clip_grads([t], -1.0), lambda: clip_grads([t], math.nan), lambda: clip_grads([t], 1.0, out=[]), lambda: clip_grads([t], 1.0, out=[t[:50]]),
                lambda: clip_grads([t], 1.0, out=[t.double()]), lambda: clip_grads([t[:60], t[40:]], 1.0, out=[t[:60], t[40:]]), lambda: clip_grads([t, t], 1.0, out=[t, t]),
                lambda: clip_grads([t[:50], t[50:]], 1.0, out=[t[50:], t[:50]]), lambda: clip_grads([t[:50]], 1.0, out=[t[10:60]]), lambda: clip_grads([t.half()], 1.0, out=[t.cpu()])):
        kept = t.clone()
        with pytest.raises(ValueError):
            bad()
        assert torch.equal(t, kept)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        grad_norm([t.cpu()])
