"""Dropout, LayerNorm and dropout + residual + LayerNorm with their gradients, against 64 bits."""
import pytest
import torch

import train_reference as R
from turbodeberta_amd.ops.dropout import dropout, new_seed
from turbodeberta_amd.ops.layer_norm import dropout_add_layer_norm, layer_norm

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-7


def _rand(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _seed(value):
    return torch.tensor([value], dtype=torch.int64, device="cuda")


# sizes around a chunk of eight, a workgroup's 2048 values and several of them
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2049, 100003])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout(n, p, dtype):
    x, dy = _rand(1, n, dtype=dtype).requires_grad_(), _rand(2, n, dtype=dtype)
    seed = _seed(-(1 << 62) + n)
    y = dropout(x, p, seed)
    dx, = torch.autograd.grad(y, x, dy)
    keep = R.keep_of((n,), p, seed.item())
    for name, got, ref in (("y", y, x.detach().cpu().double() * keep), ("dx", dx, dy.cpu().double() * keep)):
        R.check(name, got, ref, 2 * R.U * ref.abs())        # the factor and the product, each rounded to float32
    assert torch.equal(y == 0, (keep.cuda() == 0) | (x == 0))


def test_dropout_of_views_and_ends():
    base = _rand(3, 65, 130)
    seed = _seed(5)
    for x in (base[:, 1:], base.t(), base.flatten()[3:2000], base[::2, ::3], base[0].expand(4, 130), base[:0]):
        keep = R.keep_of(tuple(x.shape), 0.3, 5)
        got = dropout(x, 0.3, seed)
        assert got.shape == x.shape and got.is_contiguous()
        R.check("y", got, x.cpu().double() * keep, 2 * R.U * x.cpu().double().abs() * keep)
    assert dropout(base, 0.0, seed) is base and not dropout(base, 1.0, seed).any()
    bad = torch.full((4096,), float("nan"), device="cuda")
    got = dropout(bad, 0.5, seed)
    assert torch.equal(got.isnan(), R.keep_of((4096,), 0.5, 5).cuda() != 0) and not got.nan_to_num().any()


def test_dropout_share_and_independence():
    """Shares of 2^20 values within five standard deviations; two seeds agree as often as chance has it."""
    n, p = 1 << 20, 0.1
    x = torch.ones(n, device="cuda")
    a, b = ((dropout(x, p, _seed(s)) != 0).double() for s in (1, 2))
    for t in (a, b):
        assert abs(t.mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5 + 2 ** -17
    assert abs((a * b).mean().item() - (1 - p) ** 2) < 5 * 0.4 / n ** 0.5


def _norm_case(rows, hidden, dtype, p=None, wide=False, weighted=True, shape=None, offset=3.0):
    shape = shape or (rows, hidden)
    x = (_rand(1, *shape) + offset).to(dtype).requires_grad_()
    res = _rand(2, *shape, dtype=dtype).requires_grad_() if p is not None else None
    wt = torch.float32 if wide else dtype
    w = (1 + 0.2 * _rand(3, hidden)).to(wt).requires_grad_() if weighted else None
    b = _rand(4, hidden, dtype=wt, scale=0.3).requires_grad_() if weighted else None
    return x, res, w, b, _rand(5, *shape, dtype=dtype)


def _check_norm(x, res, w, b, dy, p, seed, eps=EPS):
    y = layer_norm(x, w, b, eps) if res is None else dropout_add_layer_norm(x, res, w, b, p, seed, eps)
    leaves = [t for t in (x, res, w, b) if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dres", "dw", "db"), (x, res, w, b)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    c = lambda t: None if t is None else t.detach().cpu().double()
    keep = R.keep_of(tuple(x.shape), p, seed.item()) if p else torch.ones((), dtype=torch.float64)
    ref, off = R.norm(c(x), c(res), c(w), c(b), c(dy), keep, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    R.check("y", y, ref["y"], off["y"])
    R.check("dx", grads["dx"], ref["dz"] * keep, off["dz"] * keep + 2 * R.U * (ref["dz"] * keep).abs())
    if res is not None:
        R.check("dres", grads["dres"], ref["dz"], off["dz"])
    if w is not None:
        assert grads["dw"].dtype == w.dtype
        R.check("dw", grads["dw"], ref["dw"], off["dw"])
        R.check("db", grads["db"], ref["db"], off["db"])


# widths at the edges of a wave's chunks (512, 1024, 2048), of the row kernels, odd ones; rows at the edges of the workgroups' shares
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 8), (9, 512), (4100, 520), (33, 1024), (17, 1032), (5, 2048), (3, 2056), (7, 4096), (1, 1), (6, 3), (515, 255),
                                         (1030, 771), (2, 20000), (2, 32768)])
def test_layer_norm(rows, hidden, dtype):
    _check_norm(*_norm_case(rows, hidden, dtype), None, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 16), (70, 768), (4099, 64), (19, 1536), (12, 2040), (5, 2304), (11, 773)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.6])
def test_dropout_add_layer_norm(rows, hidden, p, dtype):
    _check_norm(*_norm_case(rows, hidden, dtype, p), p, _seed(rows * 7919 - (1 << 40)))


@pytest.mark.parametrize("hidden", [768, 771])
def test_weights_in_float32_and_none(hidden):
    for dtype in (torch.bfloat16, torch.float16):
        _check_norm(*_norm_case(30, hidden, dtype, 0.1, wide=True), 0.1, _seed(3))
        _check_norm(*_norm_case(30, hidden, dtype, 0.1, weighted=False), 0.1, _seed(3))
    _check_norm(*_norm_case(30, hidden, torch.float32, weighted=False), None, None)


@pytest.mark.parametrize("hidden", [64, 61])
def test_layouts(hidden):
    """More dimensions, rows that lie apart, transposed and repeated ones, and bases that are not aligned."""
    seed = _seed(11)
    for dtype in (torch.float32, torch.bfloat16):
        for make in (lambda t: t.clone()[:, :, :hidden], lambda t: t[:, :, 1:hidden + 1], lambda t: t.transpose(0, 1)[:, :, :hidden],
                     lambda t: t[:1, :, :hidden].expand(5, 7, hidden), lambda t: t[..., :1].expand(5, 7, hidden),
                     lambda t: t.transpose(1, 2)[:, :hidden].transpose(1, 2)):
            x, res, dy = (make(_rand(s, 5, 7, hidden + 3, dtype=dtype)) for s in (1, 2, 3))
            w, b = (1 + _rand(4, hidden, dtype=dtype, scale=0.1)).requires_grad_(), _rand(5, hidden, dtype=dtype).requires_grad_()
            _check_norm(x.detach().requires_grad_(), res.detach().requires_grad_(), w, b, dy, 0.2, seed)
            _check_norm(x.detach().requires_grad_(), None, w, b, dy, None, None, 1e-3)


def test_large_means_and_extremes():
    """A mean a thousand times the deviation: the variance is taken around it.  Infinities spoil their own row, dropped ones not even that."""
    _check_norm(*_norm_case(40, 768, torch.float32, offset=1000.0), None, None)
    x, res, w, b, dy = _norm_case(64, 768, torch.bfloat16, 0.5)
    clean = dropout_add_layer_norm(x, res, w, b, 0.5, _seed(1))
    spoiled = x.detach().clone()
    gone = R.keep_of((64, 768), 0.5, 1).cuda() == 0
    spoiled[gone] = float("inf")
    assert torch.equal(dropout_add_layer_norm(spoiled, res, w, b, 0.5, _seed(1)), clean)
    spoiled[3, ~gone[3]] = float("inf")
    out = dropout_add_layer_norm(spoiled, res, w, b, 0.5, _seed(1))
    other = torch.arange(64, device="cuda") != 3
    assert torch.equal(out[other], clean[other]) and out[3].isnan().all()


def test_only_some_gradients_and_none_of_rows():
    x, res, w, b, dy = _norm_case(20, 96, torch.float32, 0.1)
    full = torch.autograd.grad(dropout_add_layer_norm(x, res, w, b, 0.1, _seed(2), EPS), (x, res, w, b), dy)
    for k in range(4):
        some = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, res, w, b))]
        got, = torch.autograd.grad(dropout_add_layer_norm(*some, 0.1, _seed(2), EPS), some[k], dy)
        assert torch.equal(got, full[k])
    for hidden in (96, 5):
        x, w, b = torch.zeros(0, hidden, device="cuda", requires_grad=True), torch.ones(hidden, device="cuda", requires_grad=True), torch.zeros(hidden, device="cuda", requires_grad=True)
        y = layer_norm(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert y.shape == dx.shape == (0, hidden) and not dw.any() and not db.any()


def test_gradients_against_differences():
    """Central differences of the float32 operator in random directions; the step's own error is h^2 times third derivatives, the rounding's U |L| / h."""
    x, res, w, b, dy = _norm_case(6, 40, torch.float32, 0.3, offset=0.0)
    seed, h = _seed(8), 2.0 ** -6
    loss = lambda *t: (dropout_add_layer_norm(*t, 0.3, seed, 1e-2).double() * dy.double()).sum().item()
    grads = torch.autograd.grad(dropout_add_layer_norm(x, res, w, b, 0.3, seed, 1e-2), (x, res, w, b), dy)
    plain = [t.detach() for t in (x, res, w, b)]
    for k, g in enumerate(grads):
        d = _rand(20 + k, *plain[k].shape)
        d /= d.norm()
        moved = lambda s: loss(*(t + s * d if i == k else t for i, t in enumerate(plain)))
        slope = (8 * (moved(h) - moved(-h)) - (moved(2 * h) - moved(-2 * h))) / (12 * h)
        assert abs(slope - (g.double() * d.double()).sum().item()) <= 1e-3 * g.double().norm().item()


@pytest.mark.parametrize("hidden", [768, 771])
def test_same_bits_every_time_and_other_streams(hidden):
    x, res, w, b, dy = _norm_case(3000, hidden, torch.bfloat16, 0.1)
    run = lambda: torch.autograd.grad(dropout_add_layer_norm(x, res, w, b, 0.1, _seed(4)), (x, res, w, b), dy)
    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = [run() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for o in other for a, c in zip(first, o))


def test_captured_and_replayed_with_other_seeds():
    """A graph of forward and backward: every replay drops what its seed says, beside eager work and a second graph of the same inputs."""
    x, res, w, b, dy = _norm_case(200, 768, torch.float32, 0.1)
    seed = _seed(0)

    def step(s):
        leaves = [t.detach().requires_grad_() for t in (x, res, w, b)]
        y = dropout(dropout_add_layer_norm(*leaves, 0.1, s, EPS), 0.2, s)
        return (y,) + torch.autograd.grad(y, leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step(seed)))
    for n in range(4):
        seed.fill_(1000 + n)
        expect = [t.clone() for t in step(_seed(1000 + n))]
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, expect))


def test_seeds_come_from_the_generator():
    torch.manual_seed(7)
    a, b = new_seed("cuda"), new_seed("cuda")
    torch.manual_seed(7)
    assert torch.equal(new_seed("cuda"), a) and not torch.equal(a, b)


def test_a_seed_changed_before_the_backward_pass_raises():
    x, seed = _rand(1, 64).requires_grad_(), _seed(1)
    y = dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals():
    x, w, seed = _rand(1, 4, 16), _rand(2, 16), _seed(1)
    for bad in (lambda: dropout(x, -0.1, seed), lambda: dropout(x, 1.5, seed), lambda: dropout(x, float("nan"), seed), lambda: dropout(x.double(), 0.1, seed),
                lambda: dropout(x, 0.1, seed.int()), lambda: dropout(x, 0.1, torch.cat([seed, seed])), lambda: dropout(x, 0.1, 5), lambda: dropout(x, 0.1, seed.cpu()),
                lambda: layer_norm(x, w), lambda: layer_norm(x, w[:8], w[:8]), lambda: layer_norm(x, w.double(), w.double()), lambda: layer_norm(x, w, w, -1.0),
                lambda: layer_norm(x[:, :0]), lambda: layer_norm(x.half(), w.bfloat16(), w.bfloat16()), lambda: layer_norm(x, w, w.cpu()),
                lambda: layer_norm(_rand(1, 2, 32769)), lambda: dropout_add_layer_norm(x, x[:2], w, w), lambda: dropout_add_layer_norm(x, x.half(), w, w),
                lambda: dropout_add_layer_norm(x, x, w, w, 0.1), lambda: dropout_add_layer_norm(x, None, w, w)):
        with pytest.raises(ValueError):
            bad()
