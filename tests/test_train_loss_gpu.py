"""The loss over a vocabulary with its gradient, against 64 bits."""
import threading

import pytest
import torch

import loss_reference as R
import turbodeberta_amd._lib as _lib
from turbodeberta_amd.ops.linear_cross_entropy import linear_cross_entropy

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IGNORED = -100


def _rand(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _inputs(rows, hidden, vocab, dtype, share=1.0, bias="same", scale=2.0):
    """x, weight, labels, bias: logits of a few units, labels of the first rows among them the first and last class."""
    x, w = _rand(1, rows, hidden, dtype=dtype), _rand(2, vocab, hidden, dtype=dtype, scale=scale / hidden ** 0.5)
    g = torch.Generator().manual_seed(3)
    labels = torch.randint(0, vocab, (rows,), generator=g)
    labels[:2] = torch.tensor([0, vocab - 1])[:len(labels)]
    labels[torch.rand(rows, generator=g) >= share] = IGNORED
    b = None if bias is None else _rand(4, vocab, dtype=torch.float32 if bias == "fp32" else dtype, scale=0.5)
    return x, w, labels.cuda(), b


def _step(x, w, labels, b, reduction, dloss=None, ignore=IGNORED):
    """(loss, {name: gradient}) of fresh leaves."""
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2], ignore, reduction)
    there = [t for t in leaves if t is not None]
    return loss.detach(), dict(zip([n for n, t in zip(("dx", "dweight", "dbias"), leaves) if t is not None], torch.autograd.grad(loss, there, dloss)))


def _check(x, w, labels, b, reduction="mean", dloss=None, ignore=IGNORED):
    loss, grads = _step(x, w, labels, b, reduction, dloss, ignore)
    assert loss.dtype == torch.float32
    flat = lambda t: t if t is None or reduction != "none" else t.reshape(-1)
    ref = R.loss(x.reshape(-1, x.shape[-1]), w, labels.reshape(-1), b, ignore, reduction, flat(dloss), x.dtype)
    R.check("loss", loss.reshape(ref["loss"][0].shape), *ref["loss"])
    assert grads["dx"].shape == x.shape
    for name, got in grads.items():
        assert got.dtype == {"dx": x, "dweight": w, "dbias": b}[name].dtype
        R.check(name, got.reshape(ref[name][0].shape), *ref[name])
    return loss, grads


# rows, columns and classes at and around the tiles' 256 and the steps' 64 (32 in float32), single ones, odd ones
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden,vocab,share", [(1, 8, 1, 1.0), (1, 64, 257, 1.0), (3, 1, 5, 1.0), (2, 7, 300, 1.0), (31, 72, 255, 1.0), (33, 40, 64, 1.0), (65, 64, 1000, 1.0), (255, 128, 513, 1.0),
                                                     (256, 256, 256, 1.0), (257, 264, 700, 1.0), (600, 771, 1025, 0.5), (1500, 96, 2049, 0.15), (300, 1032, 300, 0.02), (129, 32, 5000, 1.0)])
def test_sizes(rows, hidden, vocab, share, dtype):
    x, w, labels, b = _inputs(rows, hidden, vocab, dtype, share)
    _check(x, w, labels, b, "mean", torch.tensor(0.7, device="cuda"))


# every height of tiles, one and several of them, up to where the next one takes over
@pytest.mark.parametrize("rows", [1, 16, 17, 32, 60, 96, 97, 128, 160, 161, 192, 193, 257, 288, 320, 480, 481, 512, 760, 1024, 1025])
@pytest.mark.parametrize("dtype", TYPES)
def test_heights_of_tiles(dtype, rows):
    x, w, labels, b = _inputs(rows, 160, 900, dtype)
    _check(x, w, labels, b, "mean")
    _check(x, w, labels, b, "none", _rand(5, rows))


# many rows of a small vocabulary: several workgroups share a tile of dweight, some of them without any row
@pytest.mark.parametrize("rows,hidden,vocab,share", [(1025, 64, 100, 1.0), (1100, 130, 300, 0.01), (2100, 257, 515, 0.6), (4199, 96, 2010, 1.0), (6000, 33, 7, 0.9), (1600, 200, 9000, 1.0), (1500, 64, 300, 0.0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_of_few_classes(dtype, rows, hidden, vocab, share):
    x, w, labels, b = _inputs(rows, hidden, vocab, dtype, share)
    if share == 0.0:
        loss, grads = _step(x, w, labels, b, "sum")
        assert not loss.any() and all(not g.any() for g in grads.values())
        return
    first = _check(x, w, labels, b, "mean")
    again = _step(x, w, labels, b, "mean")
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[1][k], again[1][k]) for k in first[1])
    _check(x, w, labels, None, "none", _rand(5, rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("bias", [None, "same", "fp32"])
def test_reductions_and_biases(reduction, bias, dtype):
    x, w, labels, b = _inputs(200, 96, 900, dtype, 0.6, bias)
    dloss = _rand(5, 200) if reduction == "none" else torch.tensor(-3.0, device="cuda")
    _check(x, w, labels, b, reduction, dloss)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_very_different_weight(dtype):
    """Each row's gradient is as exact as its own size, however small it is beside the others'."""
    x, w, labels, b = _inputs(90, 64, 600, dtype, 0.9)
    size = 2.0 ** torch.linspace(0, -12, 90, device="cuda")
    _check(x, w, labels, b, "none", _rand(5, 90) * size)
    zero = torch.zeros(90, device="cuda")
    loss, grads = _step(x, w, labels, b, "none", zero)
    assert all(not t.any() for t in grads.values())
    zero[7] = -2.0
    _check(x, w, labels, b, "none", zero)


@pytest.mark.parametrize("dtype", TYPES)
def test_sure_and_flat_logits(dtype):
    """Logits up to several tens: losses near 0 and large ones; and all the same."""
    x, w, labels, b = _inputs(120, 64, 700, dtype, scale=16.0)
    s = x.double() @ w.double().t() + b.double()
    labels[:60] = s[:60].argmax(-1)
    loss, _ = _check(x, w, labels, b, "none", _rand(5, 120).abs())
    assert (loss >= -1e-5).all()
    _check(torch.zeros_like(x), w, labels, None, "sum")


def test_small_probabilities_in_float16():
    """Probabilities of 2^-20 and less are none of float16's own; their gradients are those of the formula to a hundredth."""
    x, w, labels, _ = _inputs(64, 64, 512, torch.float16)
    b = torch.zeros(512, device="cuda")
    b[256:] = -16.0
    _, grads = _step(x, w, labels % 256, b, "sum", torch.tensor(512.0, device="cuda"))
    ref = R.loss(x, w, labels % 256, b, IGNORED, "sum", torch.tensor(512.0, device="cuda"), torch.float16)["dweight"][0][256:]
    assert (grads["dweight"][256:].double() - ref).norm() <= 1e-2 * ref.norm()


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_classes(dtype):
    """Biases of minus infinity and of the type's lowest value take classes out; where a row's label is such a class the loss is infinite; where all of them are, that of equal ones."""
    x, w, labels, b = _inputs(70, 48, 600, dtype)
    labels.clamp_(min=0)
    for lowest in (-torch.inf, torch.finfo(dtype).min):
        gone = b.clone()
        gone[300:590] = lowest
        keep = torch.where((labels >= 300) & (labels < 590), 0, labels)
        loss, grads = _step(x, w, keep, gone, "mean")
        there = [*range(300), *range(590, 600)]
        small = _step(x, w[there], torch.where(keep >= 590, keep - 290, keep), b[there], "mean")
        assert (loss - small[0]).abs() <= 1e-5 * small[0].abs() and not grads["dweight"][300:590].any() and not grads["dbias"][300:590].any()
        torch.testing.assert_close(grads["dweight"][there].float(), small[1]["dweight"].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
    bad = keep.clone()
    bad[3] = 400
    gone[300:590] = -torch.inf
    rows = linear_cross_entropy(x, w, bad, gone, reduction="none")
    assert rows[3] == torch.inf and rows[:3].isfinite().all() and rows[4:].isfinite().all()
    if dtype != torch.float16:      # (lowest and any logit is lowest again; float16's lowest value is one like others in float32)
        loss, grads = _step(x, w, labels, torch.full_like(b, torch.finfo(dtype).min), "mean")
        torch.testing.assert_close(loss, torch.log(torch.tensor(600.0, device="cuda")), rtol=1e-5, atol=0)
        assert all(t.isfinite().all() for t in grads.values())
    assert linear_cross_entropy(x, w, labels, torch.full_like(b, -torch.inf)).isnan()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count(dtype):
    x, w, labels, b = _inputs(300, 64, 400, dtype, 0.4)
    clean = _step(x, w, labels, b, "mean")
    spoiled = x.clone()
    spoiled[labels == IGNORED] = torch.tensor([torch.nan, torch.inf, -torch.inf] * 22, device="cuda")[:64].to(dtype)
    got = _step(spoiled, w, labels, b, "mean")
    assert torch.equal(got[0], clean[0]) and all(torch.equal(got[1][k], clean[1][k]) for k in clean[1])
    assert not got[1]["dx"][labels == IGNORED].any()
    none = torch.full_like(labels, IGNORED)
    for reduction in ("mean", "sum", "none"):
        loss, grads = _step(spoiled, w, none, b, reduction, torch.ones(300, device="cuda") if reduction == "none" else None)
        assert loss.isnan() if reduction == "mean" else not loss.any()
        assert all(not t.any() for t in grads.values())
    # another number that does not count, one that is a class
    some = torch.where(labels == IGNORED, 7, labels)
    _check(x, w, some, b, "mean", ignore=7)
    _check(x, w, torch.where(labels == IGNORED, (1 << 40) + 5, labels), b, "sum", ignore=(1 << 40) + 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [-1, 400, 1 << 40, -(1 << 40)])
def test_labels_that_are_none(bad, dtype):
    x, w, labels, b = _inputs(40, 64, 400, dtype)
    labels[11] = bad
    loss, grads = _step(x, w, labels, b, "none", torch.ones(40, device="cuda"))
    assert loss[11].isnan() and loss.isnan().sum() == 1 and grads["dx"][11].isnan().all() and grads["dx"].isnan().any(-1).sum() == 1
    assert grads["dweight"].isnan().all() and grads["dbias"].isnan().all()
    assert linear_cross_entropy(x, w, labels, b).isnan()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_spoil_their_own_row(dtype):
    x, w, labels, b = _inputs(300, 64, 400, dtype)
    clean = linear_cross_entropy(x, w, labels, b, reduction="none")
    x[5, 3], x[290, 60] = torch.inf, torch.nan
    got = linear_cross_entropy(x, w, labels, b, reduction="none")
    other = [i for i in range(300) if i not in (5, 290)]
    assert got[[5, 290]].isnan().all() and torch.equal(got[other], clean[other])


def test_no_rows():
    x, w, _, b = _inputs(2, 16, 30, torch.float32)
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.zeros(shape, device="cuda")
        labels = torch.zeros(shape[:-1], dtype=torch.int64, device="cuda")
        for reduction in ("mean", "sum", "none"):
            loss, grads = _step(x, w, labels, b, reduction, torch.zeros(shape[:-1], device="cuda") if reduction == "none" else None)
            assert loss.shape == (shape[:-1] if reduction == "none" else ()) and (loss.isnan() if reduction == "mean" else not loss.any())
            assert grads["dx"].shape == shape and not grads["dweight"].any() and not grads["dbias"].any()
    one = linear_cross_entropy(_rand(1, 16), w, torch.tensor(5, device="cuda"), b)     # a vector and its label
    R.check("loss", one, *R.loss(_rand(1, 16)[None], w, torch.tensor([5], device="cuda"), b, IGNORED, "mean", None, torch.float32)["loss"])


@pytest.mark.parametrize("hidden", [64, 61])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(hidden, dtype):
    """More dimensions, rows that lie apart, transposed and repeated ones, addresses that are not aligned, strided labels, biases and gradients."""
    _, w, labels, b = _inputs(35, hidden, 300, dtype, 0.7)
    labels = labels.view(5, 7)
    wide = _rand(9, 300, hidden + 8, dtype=dtype, scale=0.2)
    weights = [w, wide[:, :hidden], wide[:, 8:], wide[:, 1:hidden + 1], _rand(10, hidden, 300, dtype=dtype, scale=0.2).t(), w[:1].expand(300, hidden)]
    for make in (lambda t: t.clone()[:, :, :hidden], lambda t: t[:, :, 1:hidden + 1], lambda t: t.transpose(0, 1)[:, :, :hidden].transpose(0, 1),
                 lambda t: t[:1, :, :hidden].expand(5, 7, hidden), lambda t: t[..., :1].expand(5, 7, hidden), lambda t: t.transpose(1, 2)[:, :hidden].transpose(1, 2)):
        x = make(_rand(1, 5, 7, hidden + 3, dtype=dtype))
        _check(x, w, labels, b)
    x = _rand(1, 5, 7, hidden, dtype=dtype)
    for weight in weights:
        _check(x, weight, labels, b, "sum")
    both = torch.stack([b, b], 1)[:, 0]
    strided = torch.stack([labels.view(-1), labels.view(-1) * 0], 1)[:, 0].view(5, 7)
    _check(x, w, strided, both, "none", _rand(3, 7, 5).t())
    _check(x, w, strided, both, "none", torch.ones(1, 1, device="cuda").expand(5, 7))
    loss, grads = _step(x, w, labels.flip(0), b, "none", _rand(3, 5, 7))
    again, _ = _step(x, w, labels.flip(0).contiguous(), b, "none", _rand(3, 5, 7))
    assert torch.equal(loss, again)


# few rows and many; rows that end 0, 2, 4 ... bytes into 16, one step and several
@pytest.mark.parametrize("rows", [20, 600])
@pytest.mark.parametrize("hidden", [8, 21, 66, 127, 130, 301])
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_among_other_values(dtype, hidden, rows):
    """Rows at multiples of 4 bytes inside a wider matrix whose other values are NaN, and inside one whose rows are at odd places."""
    x, w, labels, b = _inputs(rows, hidden, 700, dtype)
    want = _check(x, w, labels, b)
    for pad in (3, 4):
        wide = torch.full((702, hidden + pad + (hidden + pad) % 2), torch.nan, dtype=dtype, device="cuda")
        view = wide[1:701, 2:2 + hidden]
        view.copy_(w)
        got = _check(x, view, labels, b)
        assert torch.equal(got[0], want[0]) and all(torch.equal(want[1][k], got[1][k]) for k in want[1])
    wide = torch.full((700, hidden + 1 + hidden % 2), torch.nan, dtype=dtype, device="cuda")
    view = wide[:, 1:1 + hidden]
    view.copy_(w)
    got = _check(x, view, labels, b)
    assert torch.equal(got[0], want[0]) and all(torch.equal(want[1][k], got[1][k]) for k in want[1])


@pytest.mark.parametrize("hidden", [6, 7])
@pytest.mark.parametrize("dtype", TYPES)
def test_one_class_of_many(dtype, hidden):
    """A single row of a matrix whose rows lie an odd number of values or very far apart."""
    x, _, labels, _ = _inputs(20, hidden, 1, dtype)
    for apart in (hidden + 2, hidden + 3, (1 << 22) + 1):
        _check(x, torch.as_strided(_rand(2, hidden + 9, dtype=dtype), (1, hidden), (apart, 1)), labels, None, "sum")


@pytest.mark.parametrize("rows,hidden,vocab", [(5, 32768, 300), (140, 32767, 70), (300, 20000, 300), (3, 4, 1 << 20), (1030, 2, 1 << 17)])
@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_shapes(dtype, rows, hidden, vocab):
    x, w, labels, b = _inputs(rows, hidden, vocab, dtype, 0.9)
    if rows * vocab < 1 << 24:
        _check(x, w, labels, b)
        return
    loss, grads = _step(x, w, labels, b, "sum")         # (64 bits of 10^8 logits: some of the rows by themselves, and what all of them add up to)
    each, _ = _step(x, w, labels, b, "none", torch.ones(rows, device="cuda"))
    few = R.loss(x[:50], w, labels[:50], b, IGNORED, "none", None, x.dtype)
    R.check("loss", each[:50], *few["loss"])
    R.check("dx", grads["dx"][:50], *few["dx"])
    assert torch.isclose(loss.double(), each.double().sum(), rtol=1e-6)


def test_backward_twice():
    """What is kept for the backward pass is not used up by it."""
    for dtype, reduction in ((torch.float16, "none"), (torch.bfloat16, "mean"), (torch.float32, "sum")):
        x, w, labels, b = _inputs(150, 72, 700, dtype, 0.8)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        loss = linear_cross_entropy(x, w, labels, b, reduction=reduction)
        weight = torch.ones_like(loss)
        first = torch.autograd.grad(loss, leaves, weight, retain_graph=True)
        torch.autograd.grad(loss, leaves, 3 * weight, retain_graph=True)
        again = torch.autograd.grad(loss, leaves, weight)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_only_some_gradients():
    x, w, labels, b = _inputs(90, 96, 500, torch.bfloat16, 0.8)
    _, full = _step(x, w, labels, b, "mean")
    for mask in range(1, 8):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        linear_cross_entropy(some[0], some[1], labels, some[2]).backward()
        for t, name in zip(some, ("dx", "dweight", "dbias")):
            assert torch.equal(t.grad, full[name]) if t.requires_grad else t.grad is None
    assert not linear_cross_entropy(x, w, labels, b).requires_grad
    with torch.no_grad():
        assert not linear_cross_entropy(x.requires_grad_(), w, labels, b).requires_grad


def test_gradients_against_differences():
    """Central differences of the float32 operator in random directions; the step's own error is h^4 times fifth derivatives, the rounding's U |L| / h."""
    x, w, labels, b = _inputs(12, 40, 90, torch.float32, 0.8)
    dy, h = _rand(8, 12), 2.0 ** -5
    value = lambda *t: (linear_cross_entropy(t[0], t[1], labels, t[2], reduction="none").double() * dy.double()).sum().item()
    _, grads = _step(x, w, labels, b, "none", dy)
    for k, g in enumerate(grads.values()):
        d = _rand(20 + k, *(x, w, b)[k].shape)
        d /= d.norm()
        moved = lambda s: value(*(t + s * d if i == k else t for i, t in enumerate((x, w, b))))
        slope = (8 * (moved(h) - moved(-h)) - (moved(2 * h) - moved(-2 * h))) / (12 * h)
        assert abs(slope - (g.double() * d.double()).sum().item()) <= 1e-3 * g.double().norm().item()


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_pieces_of_the_vocabulary(reduction):
    """So many rows that a piece of the logits' gradient is a part of the vocabulary, and a workgroup takes several column tiles together; few of them count."""
    x, w, labels, b = _inputs(70000, 16, 80001, torch.bfloat16, 0.004)
    a = _lib.LossArgs(_lib.TDB_BF16, _lib.TDB_BF16, 16, 2, 70000, 80001)
    assert _lib.load().tdb_loss_workspace(a, 1) < 3 << 30 < 70000 * 80001 * 2
    dloss = _rand(5, 70000) if reduction == "none" else None
    loss, grads = _step(x, w, labels, b, reduction, dloss)
    counts = labels != IGNORED
    ref = R.loss(x[counts], w, labels[counts], b, IGNORED, reduction, dloss if dloss is None else dloss[counts], torch.bfloat16)
    R.check("loss", loss[counts] if reduction == "none" else loss, *ref["loss"])
    R.check("dx", grads["dx"][counts], *ref["dx"])
    assert not grads["dx"][~counts].any()
    R.check("dweight", grads["dweight"], *ref["dweight"])
    R.check("dbias", grads["dbias"], *ref["dbias"])


def test_offsets_past_32_bits():
    """A weight and hidden states of more than 4 GiB, of which the last rows and classes matter."""
    hidden, vocab, rows = 2304, 1 << 20, 9
    w = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    w[-300:] = _rand(2, 300, hidden, dtype=torch.bfloat16, scale=0.05)
    wide = torch.zeros(40000, 65536, dtype=torch.bfloat16, device="cuda")
    x = wide[:, -hidden:]
    x[-rows:] = _rand(1, rows, hidden, dtype=torch.bfloat16)
    labels = torch.full((40000,), IGNORED, device="cuda")
    labels[-rows:] = vocab - 1 - torch.arange(rows, device="cuda") * 30
    loss, grads = _step(x, w, labels, None, "sum")
    # The classes without weights: each has the exponential of 0.
    s = x[-rows:].double() @ w[-300:].double().t()
    total = s.exp().sum(-1, keepdim=True) + (vocab - 300)
    p = s.exp() / total
    d = p.clone()
    d[torch.arange(rows), 299 - torch.arange(rows) * 30] -= 1
    expect = (total.log().squeeze(-1) - s[torch.arange(rows), 299 - torch.arange(rows) * 30]).sum()
    assert abs(loss.double() - expect) <= 1e-4 * expect
    for got, ref in ((grads["dx"][-rows:], d @ w[-300:].double()), (grads["dweight"][-300:], d.t() @ x[-rows:].double()),
                     (grads["dweight"][:5], (1 / total).expand(rows, 5).t() @ x[-rows:].double())):
        assert (got.double() - ref).norm() <= 2.0 ** -7 * ref.norm()
    assert not grads["dx"][:-rows].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_same_bits_every_time_and_other_streams(dtype, reduction):
    x, w, labels, b = _inputs(700, 264, 3000, dtype, 0.5)
    dloss = _rand(5, 700) if reduction == "none" else None
    first = _step(x, w, labels, b, reduction, dloss)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = [_step(x, w, labels, b, reduction, dloss) for _ in range(3)]
    torch.cuda.synchronize()
    for loss, grads in other:
        assert torch.equal(loss, first[0]) and all(torch.equal(grads[k], first[1][k]) for k in grads)


def test_two_threads_at_once():
    x, w, labels, b = _inputs(300, 96, 2000, torch.bfloat16, 0.5)
    alone = [_step(x * k, w, labels, b, "mean") for k in (1, 2)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[k] = _step(x * (k + 1), w, labels, b, "mean")
            torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for (loss, grads), (l, g) in zip(got, alone):
        assert torch.equal(loss, l) and all(torch.equal(grads[k], g[k]) for k in g)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_captured_and_replayed_with_other_inputs(reduction):
    """Two graphs of forward and backward; every replay sees the inputs, and as many rows that count, as there are then."""
    x, w, labels, b = _inputs(300, 96, 1500, torch.bfloat16, 0.5)
    dloss = _rand(5, 300) if reduction == "none" else None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(x, w, labels, b, reduction, dloss)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, _step(x, w, labels, b, reduction, dloss)))
    for n, share in enumerate((0.1, 1.0, 0.0, 0.7)):
        x.copy_(_rand(50 + n, 300, 96))
        labels.copy_(torch.where(torch.rand(300, generator=torch.Generator().manual_seed(n)).cuda() < share, torch.arange(300, device="cuda") * 5, IGNORED))
        loss, grads = _step(x.clone(), w, labels.clone(), b, reduction, dloss)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, (l, d) in graphs:
            assert torch.equal(l, loss) or (l.isnan() and loss.isnan())
            assert all(torch.equal(d[k], grads[k]) for k in grads)


class PythonOnly:
    def __init__(self, host):
        self.host = host

    def __getattr__(self, name):
        return (lambda *a: None) if name.startswith("train_") else getattr(self.host, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_both_paths_give_the_same_bits(dtype, reduction, monkeypatch):
    host = _lib.host()
    for bias in ("same", None):
        x, w, labels, b = _inputs(75, 64, 700, dtype, 0.5, bias)
        dloss = _rand(5, 75) if reduction == "none" else None
        assert host.train_loss(x, w, labels, b, IGNORED, 2) is not None
        native = _step(x, w, labels, b, reduction, dloss)
        with monkeypatch.context() as m:
            m.setattr(_lib, "host", lambda: PythonOnly(host))
            python = _step(x, w, labels, b, reduction, dloss)
        assert torch.equal(native[0], python[0]) and native[1].keys() == python[1].keys() and all(torch.equal(native[1][k], python[1][k]) for k in native[1])


@pytest.mark.parametrize("native", [True, False])
def test_differentiable_once_and_saved_inputs(native, monkeypatch):
    host = _lib.host()
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: PythonOnly(host))
    x, w, labels, b = _inputs(20, 64, 300, torch.float32)
    x.requires_grad_()
    grad, = torch.autograd.grad(linear_cross_entropy(x, w, labels, b), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once|does not require grad"):
        grad.sum().backward()
    v = w.clone().requires_grad_()
    loss = linear_cross_entropy(x, v, labels, b)
    with torch.no_grad():
        v.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals():
    x, w, labels, b = _inputs(10, 32, 50, torch.float32)
    for bad in (lambda: linear_cross_entropy(x.double(), w.double(), labels), lambda: linear_cross_entropy(x, w.half(), labels), lambda: linear_cross_entropy(x, w[:, :16], labels),
                lambda: linear_cross_entropy(x, w, labels.int()), lambda: linear_cross_entropy(x, w, labels[:5]), lambda: linear_cross_entropy(x, w, labels, b[:5]),
                lambda: linear_cross_entropy(x, w, labels, b.half()), lambda: linear_cross_entropy(x, w, labels, b, reduction="max"), lambda: linear_cross_entropy(x, w, labels, b, ignore_index=1.5),
                lambda: linear_cross_entropy(x, w, labels, b, ignore_index=1 << 63), lambda: linear_cross_entropy(x, w, labels.cpu()), lambda: linear_cross_entropy(x, w.cpu(), labels),
                lambda: linear_cross_entropy(x, w[:0], labels), lambda: linear_cross_entropy(x, w, labels, 0.5), lambda: linear_cross_entropy(x, w, None), lambda: linear_cross_entropy(x, w.flatten(), labels)):
        with pytest.raises(ValueError):
            bad()
