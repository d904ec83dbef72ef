"""A step of masked language modelling with the training operators together: loss without logits, backward pass, clipping, update."""
import copy

import pytest
import torch
from transformers import DebertaV2Config
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2ForMaskedLM

from turbodeberta_amd.model import patch_model
from turbodeberta_amd.ops.grad_norm import clip_grad_norm_, clip_grads, grad_norm
from turbodeberta_amd.ops.layer_norm import dropout_add_layer_norm
from turbodeberta_amd.ops.linear_cross_entropy import linear_cross_entropy

pytestmark = pytest.mark.gpu


def config(p=0.0, **other):
    return DebertaV2Config(**dict(dict(vocab_size=1003, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, intermediate_size=96, relative_attention=True, position_buckets=8,
                                       max_relative_positions=24, pos_att_type=["c2p", "p2c"], norm_rel_ebd="layer_norm", share_att_key=True, hidden_dropout_prob=p,
                                       attention_probs_dropout_prob=p, initializer_range=0.1), **other))


def batch(share=0.3):
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(1, 1003, (3, 70), generator=g)
    mask = (torch.arange(70) < torch.tensor([70, 1, 33])[:, None]).long()
    labels = torch.where((torch.rand(3, 70, generator=g) < share) & mask.bool(), ids, -100)
    return dict(input_ids=(ids * mask).cuda(), attention_mask=mask.cuda(), labels=labels.cuda())


@pytest.mark.parametrize("legacy", [True, False])
def test_loss_and_gradients_are_those_of_the_logits(legacy):
    """Against the model without the operator, in float32: the output layer's sums in another order (U = 2^-24; logits of some units, 64 and 1003 terms): 1e-5 of each gradient's norm."""
    stock = DebertaV2ForMaskedLM(config(legacy=legacy))
    plain = patch_model(copy.deepcopy(stock), training=True).cuda().train()
    fused = patch_model(copy.deepcopy(stock), training=True, fused_loss=True).cuda().train()
    a, b = plain(**batch()), fused(**batch())
    assert a.logits is not None and b.logits is None and b.loss.dtype == torch.float32
    torch.testing.assert_close(b.loss, a.loss, rtol=1e-5, atol=0)
    a.loss.backward()
    b.loss.backward()
    for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
        assert (p.grad is None) == (q.grad is None), name
        if p.grad is not None:
            assert (p.grad - q.grad).norm() <= 1e-5 * q.grad.norm() + 1e-8, name
    with torch.no_grad():
        for model in (plain, fused):
            model.eval()
        a, b = plain(**batch()), fused(**batch())
    assert torch.equal(a.logits, b.logits) and torch.equal(a.loss, b.loss)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, "autocast"])
def test_in_16_bits(dtype):
    """The loss in float32 from the same hidden states and weights: that of the model in 16 bits, whose logits and loss are rounded, within their rounding."""
    stock = DebertaV2ForMaskedLM(config())
    models = [patch_model(copy.deepcopy(stock), training=True, fused_loss=f).cuda().train() for f in (False, True)]
    if dtype != "autocast":
        models = [m.to(dtype) for m in models]
    with torch.autocast("cuda", torch.bfloat16, enabled=dtype == "autocast"):
        a, b = (m(**batch()) for m in models)
    eps = torch.finfo(torch.bfloat16 if dtype == "autocast" else dtype).eps
    assert b.loss.dtype == torch.float32 and abs(a.loss.float() - b.loss) <= 2 * eps * (b.loss + a.logits.abs().max())
    for model, loss in zip(models, (a.loss, b.loss)):
        loss.backward()
    assert all(p.grad is None or (p.grad.isfinite().all() and p.grad.dtype == p.dtype) for p in models[1].parameters())


def test_steps_with_clipping():
    """Three steps beside PyTorch's loss and clipping, from the same start: the same weights but for the sums' order."""
    stock = DebertaV2ForMaskedLM(config())
    ours, theirs = (patch_model(copy.deepcopy(stock), training=True, fused_loss=f).cuda().train() for f in (True, False))
    optimizers = [torch.optim.SGD(m.parameters(), 0.1) for m in (ours, theirs)]
    for _ in range(3):
        for model, optimizer, clip in zip((ours, theirs), optimizers, (clip_grad_norm_, torch.nn.utils.clip_grad_norm_)):
            optimizer.zero_grad()
            model(**batch()).loss.backward()
            model.norm = clip(model.parameters(), 0.5)
            optimizer.step()
        torch.testing.assert_close(ours.norm, theirs.norm, rtol=1e-4, atol=0)
    assert ours.norm > 0.5                              # (so that something was clipped)
    for (name, p), q in zip(ours.named_parameters(), theirs.named_parameters()):
        torch.testing.assert_close(p, q[1], rtol=1e-3, atol=1e-5, msg=name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_operators_together_in_two_graphs(dtype):
    """The end of a step, captured twice: dropout, residual and LayerNorm, the loss, all gradients, clipping into float32.  Each replay, with other inputs and labels, has the eager bits."""
    g = torch.Generator().manual_seed(2)
    make = lambda *shape: torch.randn(shape, generator=g).to(dtype).cuda()
    x, r, w, b, vocab, bias = make(150, 64), make(150, 64), make(64), make(64), make(1003, 64), make(1003)
    labels, seed = torch.randint(0, 1003, (150,), generator=g).cuda(), torch.tensor([5], device="cuda")

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, r, w, b, vocab, bias)]
        loss = linear_cross_entropy(dropout_add_layer_norm(*leaves[:4], 0.1, seed), leaves[4], labels, leaves[5])
        grads = torch.autograd.grad(loss, leaves)
        return loss.detach(), *grads, *clip_grads(grads[2:], 0.05, out=[torch.empty(t.shape, device="cuda") for t in grads[2:]])[1], grad_norm(grads[:2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for n in range(4):
        x.mul_(0.9)
        seed.add_(1)
        labels.copy_(torch.where(torch.rand(150, generator=g).cuda() < 0.3 * n, labels, -100) if n else labels)
        wanted = [t.clone() for t in step()]
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(a, c) or (a.isnan().all() and c.isnan().all()) for a, c in zip(got, wanted))
