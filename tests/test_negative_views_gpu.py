"""Tensors whose values are the negatives of what their memory holds, as the imaginary part of a conjugate is: the operators take the values."""
import pytest
import torch

from test_grad_norm_gpu import _check_clipped, _check_norm, _norm64, _rand, path      # noqa: F401
from turbodeberta_amd.ops.grad_norm import clip_grad_norm_, clip_grads, grad_norm
from turbodeberta_amd.ops.linear_cross_entropy import linear_cross_entropy

pytestmark = pytest.mark.gpu


def _negative(values):
    """Dense or not, as the values are."""
    t = torch._neg_view(-values)
    assert t.is_neg() and torch.equal(t, values)
    return t


def test_norm_and_clipping(path):       # noqa: F811
    a, b = _rand(1, 30, 50), _rand(2, 77)
    norm = _norm64([a, b], 2.0)
    for x in (_negative(a), _negative(a.t().contiguous()).t(), torch.complex(a, -a).conj().imag):
        assert x.is_neg()
        _check_norm(grad_norm([x, b]), [a, b], 2.0)
        _check_clipped(clip_grads([x, b], 0.5 * norm)[1], [a, b], norm, 0.5 * norm)
        out = [torch.empty(30, 50, dtype=torch.bfloat16, device="cuda"), torch.empty(77, device="cuda")]
        clip_grads([x, b], 0.5 * norm, out=out)
        _check_clipped(out, [a, b], norm, 0.5 * norm)
        out = [_negative(torch.ones(30, 50, device="cuda")), _negative(torch.ones(77, device="cuda"))]
        clip_grads([a, b], 0.5 * norm, out=out)
        _check_clipped(out, [a, b], norm, 0.5 * norm)
        p = torch.nn.Parameter(torch.zeros(30, 50, device="cuda"))
        p.grad = x
        one = _norm64([a], 2.0)
        clip_grad_norm_([p], 0.5 * one)
        _check_clipped([p.grad], [a], one, 0.5 * one)


@pytest.mark.parametrize("which", range(4))
def test_loss(which, request, path):       # noqa: F811
    """The same bits as of the values themselves: x, weight, bias and the loss's gradient, which the native host path refuses like any that is not an ordinary tensor."""
    given = [_rand(1, 20, 32), _rand(2, 300, 32), _rand(3, 300), _rand(4, 20)]
    labels = torch.arange(20, device="cuda") * 7

    def step(x, w, b, dloss):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2], reduction="none")
        return loss.detach(), *torch.autograd.grad(loss, leaves, dloss)
    wanted = step(*given)
    given[which] = _negative(given[which])
    if which == 3 and request.node.callspec.params["path"] == "native":
        with pytest.raises(RuntimeError, match="ordinary tensor"):
            step(*given)
        return
    got = step(*given)
    assert all(torch.equal(a, b) for a, b in zip(got, wanted))
