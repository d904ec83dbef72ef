"""float16, each row's loss with a gradient of its own: rows whose gradients are far smaller than the largest keep what float16 holds of theirs."""
import pytest
import torch

import loss_reference as R
from test_train_loss_gpu import IGNORED, _inputs, _rand, _step

pytestmark = pytest.mark.gpu
H = 2.0 ** -11      # half a step of float16, relative


# gradients of 2^12 and of 2^(12 - apart); few and many rows, values of x of several sizes
@pytest.mark.parametrize("rows,size", [(20, 1.0), (300, 1.0), (700, 1.0), (90, 2.0 ** -6), (90, 2.0 ** 3)])
@pytest.mark.parametrize("apart", [0, 10, 14, 18, 22, 24])
def test_lightly_weighted_rows(apart, rows, size):
    """Each light row's label is a class of its own, which a bias of -45 takes out of all other rows: dweight there is -g x and a sum of others' g p x, p < 2^-55.

    Off by: D's rounding, H; the result's, H or half its smallest step 2^-25; x's at the row's power of two: the largest of all |g x| is brought to 2^15 at least, so it is half of float16's smallest
    step there, 2^-25 2^-15 max |g x|, times |g| up to twice its power of two; p of those classes, below 2^-55 of the largest |g x|, for each row; 8 U of arithmetic."""
    vocab = 1000
    x, w, labels, _ = _inputs(rows, 72, vocab, torch.float16)
    x *= size
    light = torch.arange(0, rows, 2, device="cuda")
    labels = labels % 400
    labels[light] = 600 + torch.arange(len(light), device="cuda")
    b = torch.zeros(vocab, device="cuda")
    b[600:] = -45.0
    dloss = (1 + torch.rand(rows, generator=torch.Generator().manual_seed(6)).cuda() * 0.9) * 2.0 ** 12
    dloss[light] *= 2.0 ** -apart
    s = x.double() @ w.double().t() + b.double()
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - lse)
    d = p.clone()
    d[torch.arange(rows), labels] -= 1
    d *= dloss.double()[:, None]
    ref = (d.t() @ x.double())[600:600 + len(light)]
    largest = (dloss.double()[:, None] * x.double()).abs().max()
    _, grads = _step(x, w, labels, b, "none", dloss)
    own = (dloss.double()[:, None] * x.double()).abs()[light]
    bound = own * (2 * H + 8 * 2.0 ** -24) * (1 + H) + 2.0 ** -25 + 2 * 2.0 ** -40 * largest + rows * 2.0 ** -55 * largest
    got = grads["dweight"][600:600 + len(light)].double()
    bad = ~((got - ref).abs() <= bound) & ~((got * ref.sign() == torch.inf) & (ref.abs() + bound >= 65520.0))       # (what is as large as that is float16's infinity)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, by up to {((got - ref).abs() / bound).max().item():.3g} of the bound"
    full = R.loss(x, w, labels, b, IGNORED, "none", dloss, torch.float16)
    for name in ("dx", "dbias"):
        R.check(name, grads[name], *full[name])


def test_extreme_gradients_and_rows():
    """Zero and subnormal gradients, rows of zeros, of float16's largest and of its smallest values among ordinary ones; rows that are infinite spoil dweight and their own dx alone."""
    x, w, labels, b = _inputs(60, 40, 300, torch.float16, 0.9, "fp32")
    dloss = _rand(5, 60)
    dloss[::7] = 0.0
    dloss[3], dloss[4] = 2.0 ** -140, 2.0 ** -60
    x[10], x[11], x[12] = 0.0, 2.0 ** -24, 2.0 ** -14
    x[13], dloss[13] = 65504.0 * torch.sign(x[13].float()), 0.25
    w[:] *= 2.0 ** -10                                  # (so that logits of the largest row are of some units)
    ref = R.loss(x, w, labels, b, IGNORED, "none", dloss, torch.float16)
    loss, grads = _step(x, w, labels, b, "none", dloss)
    R.check("loss", loss, *ref["loss"])
    for name, got in grads.items():
        R.check(name, got, *ref[name])
    for tiny in (torch.full_like(dloss, 2.0 ** -149), torch.full_like(dloss, -(2.0 ** -110))):          # nothing that float16 holds; float32 does
        ref = R.loss(x, w, labels, b, IGNORED, "none", tiny, torch.float16)
        _, grads = _step(x, w, labels, b, "none", tiny)
        assert not grads["dx"].any() and not grads["dweight"].any()
        R.check("dbias", grads["dbias"], *ref["dbias"])
    x[20, 3], x[21, 5], labels[20], labels[21] = torch.inf, torch.nan, 7, 8
    dloss[20] = dloss[21] = 1.0
    _, grads = _step(x, w, labels, b, "none", dloss)
    spoiled = grads["dx"].isnan().any(-1)
    assert spoiled[[20, 21]].all() and spoiled.sum() == 2 and grads["dweight"].isnan().all()


def test_same_bits_in_a_graph():
    """The rows' powers of two are found on the device: a captured pass follows other gradients and values."""
    x, w, labels, b = _inputs(130, 64, 500, torch.float16, 0.8)
    dloss = _rand(5, 130)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(x, w, labels, b, "none", dloss)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = _step(x, w, labels, b, "none", dloss)
    for n, scale in enumerate((1.0, 2.0 ** -20, 0.0, 2.0 ** 9)):
        x.copy_(_rand(30 + n, 130, 64))
        dloss.copy_(_rand(40 + n, 130) * scale)
        dloss[::2] *= 2.0 ** -12
        wanted = _step(x.clone(), w, labels, b, "none", dloss.clone())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], wanted[0]) and all(torch.equal(kept[1][k], wanted[1][k]) for k in wanted[1])
