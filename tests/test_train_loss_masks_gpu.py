"""Losses and gradients where a row's label is a class that a bias of the type's lowest value has taken out, and of biases of the largest value."""
import pytest
import torch

import loss_reference as R
from test_train_loss_gpu import TYPES, _inputs, _rand, _step

pytestmark = pytest.mark.gpu
U, HIDDEN = 2.0 ** -24, 48


# few and many rows; biases of x's type and of float32
@pytest.mark.parametrize("rows", [7, 150, 700])
@pytest.mark.parametrize("bias", ["same", "fp32"])
@pytest.mark.parametrize("dtype", TYPES)
def test_labels_of_masked_classes(dtype, bias, rows):
    """A masked class has no probability, and as a label a loss of the mask's size.

    Off by: such a loss by the roundings of a sum of HIDDEN products and the mask, and of two differences, relative; the others and all gradients as loss_reference has it, over the classes that are left:
    E of a logit, rho of a probability, D's rounding to the type (float16: half of its smallest step at 2^14 / g, g up to twice its power of two) and the sums'; in float16 x's, at its row's power
    of two, half of the smallest step, 2^-25, relative to the largest of all g."""
    x, w, labels, b = _inputs(rows, HIDDEN, 600, dtype, 0.9, bias)
    b[300:590] = lowest = torch.finfo(b.dtype).min
    counts = labels != -100
    labels[counts] %= 300
    hidden = [r for r in range(0, rows, 3) if counts[r]]
    labels[hidden] += 290 + (labels[hidden] < 10) * 10                 # 300 to 589
    dloss = _rand(5, rows)
    loss, grads = _step(x, w, labels, b, "none", dloss)
    X, W = x.double(), w.double()
    s = X @ W.t() + b.double()
    left = torch.ones(600, dtype=torch.bool, device="cuda")
    left[300:590] = False
    size = (X.abs() @ W.abs().t() + b.double().abs())[:, left].amax(-1)
    lse = torch.logsumexp(s, -1)
    ref = torch.where(counts, lse - s.gather(-1, labels.clamp(min=0)[:, None]).squeeze(-1), 0.0)
    E = (HIDDEN + 6) * U * size
    off = 2 * E + 8 * U * (lse.abs() + size + 1) + 608 * U
    off[hidden] = (HIDDEN + 14) * U * ref[hidden]
    R.check("loss", loss, ref, off)
    assert (loss[hidden] >= 0.999 * -lowest).all()
    total, _ = _step(x, w, labels, b, "sum")
    expect = loss.double().sum()
    assert abs(total.double() - expect) <= 2 * U * expect or total.isinf() and expect > torch.finfo(torch.float32).max

    g = (dloss.double() * counts)[:, None]
    p = torch.exp(s - lse[:, None])
    one = torch.zeros_like(p).scatter_(-1, labels.clamp(min=0)[:, None], 1.0)
    D = g * (p - one)
    D_off = g.abs() * (p * (2 * E + 630 * U)[:, None] + 4 * U * (p + one))
    u = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    stored = D_off + u * (D.abs() + D_off) + (2.0 ** -38 * g.abs() if dtype == torch.float16 else 0.0)
    lost = (2.0 ** -24 * g.abs().max() * (p + one) * counts[:, None]).sum(0)[:, None] if dtype == torch.float16 else 0.0
    R.check("dx", grads["dx"], D @ W, stored @ W.abs() + 608 * U * (D.abs() @ W.abs()))
    R.check("dweight", grads["dweight"], D.t() @ X, stored.t() @ X.abs() + (rows + 8) * U * (D.abs().t() @ X.abs()) + lost)
    R.check("dbias", grads["dbias"], D.sum(0), D_off.sum(0) + (rows + 8) * U * D.abs().sum(0))


@pytest.mark.parametrize("dtype", TYPES)
def test_largest_biases(dtype):
    """One class at the type's largest value has all of the probability, and every other label a loss of that size."""
    x, w, labels, b = _inputs(70, HIDDEN, 600, dtype)
    b[123] = torch.finfo(dtype).max
    ones = torch.ones(70, device="cuda")
    loss, grads = _step(x, w, torch.full_like(labels, 123), b, "none", ones)
    assert not loss.any() and all(not t.any() for t in grads.values())
    loss, grads = _step(x, w, torch.full_like(labels, 5), b, "none", ones)
    s = x.double() @ w.double().t() + b.double()
    R.check("loss", loss, s[:, 123] - s[:, 5], (HIDDEN + 14) * U * s[:, 123])
    want = torch.zeros(600, device="cuda")
    want[123], want[5] = 70.0, -70.0
    assert torch.equal(grads["dbias"].float(), want)
