"""The gradients of a masked language model in 16 bits whose loss is the operator's, against 64 bits at its output layer and against the model with logits behind it."""
import copy

import pytest
import torch
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2ForMaskedLM

import loss_reference as R
from test_training_step_gpu import batch, config
from turbodeberta_amd.model import patch_model

pytestmark = pytest.mark.gpu
WAYS = [torch.bfloat16, torch.float16, "autocast"]


def _run(model, way):
    with torch.autocast("cuda", torch.bfloat16, enabled=way == "autocast"):
        return model(**batch())


@pytest.mark.parametrize("way", WAYS)
def test_output_layer(way):
    """Loss, hidden states' gradient and, of an output layer with weights of its own, their gradients: those of the formula on what the layer was given.  (Under autocast the weights' gradient, in the
    operator's type, is widened to float32.)"""
    model = patch_model(DebertaV2ForMaskedLM(config(tie_word_embeddings=False)), training=True, fused_loss=True).cuda().train()
    torch.nn.init.normal_(model.cls.predictions.decoder.bias, std=0.3)
    if way != "autocast":
        model.to(way)
    seen = []
    model.cls.predictions.transform.register_forward_hook(lambda module, args, out: (out.retain_grad(), seen.append(out))[0])
    out = _run(model, way)
    assert out.logits is None and len(seen) == 1
    out.loss.backward()
    decoder, dtype = model.cls.predictions.decoder, torch.bfloat16 if way == "autocast" else way
    x, w = seen[0].detach().to(dtype).reshape(-1, 64), decoder.weight.detach().to(dtype)
    ref = R.loss(x, w, batch()["labels"].reshape(-1), decoder.bias.detach(), -100, "mean", None, dtype)
    R.check("loss", out.loss, *ref["loss"])
    for name, got in (("dx", seen[0].grad.reshape(-1, 64)), ("dweight", decoder.weight.grad)):
        assert got.to(dtype).to(got.dtype).equal(got)           # (no more bits than the operator's type)
        R.check(name, got.to(dtype), *ref[name])
    R.check("dbias", decoder.bias.grad, *ref["dbias"])


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("legacy", [True, False])
def test_all_parameters(legacy, way):
    """The same parameters have gradients as in the model with logits, and those of the tied embedding, the head and its bias agree.  26 operators lie behind the loss on the longest way (4 of the
    head, 10 of a layer, 2 of the embeddings); each rounds its result by half a step at most in either model: 52 half steps of the norm."""
    stock = DebertaV2ForMaskedLM(config(legacy=legacy))
    models = [patch_model(copy.deepcopy(stock), training=True, fused_loss=f).cuda().train() for f in (False, True)]
    for model in models:
        if way != "autocast":
            model.to(way)
        _run(model, way).loss.backward()
    plain, fused = (dict(m.named_parameters()) for m in models)
    assert all((fused[n].grad is None) == (plain[n].grad is None) for n in plain)
    head = "cls.predictions." if legacy else "lm_predictions.lm_head."
    looked_at = [n for n in plain if n == "deberta.embeddings.word_embeddings.weight" or n.startswith(head) and plain[n].grad is not None]
    assert len(looked_at) >= 6
    half = torch.finfo(torch.float16 if way == torch.float16 else torch.bfloat16).eps / 2
    for n in looked_at:
        p, q = fused[n].grad.double(), plain[n].grad.double()
        assert q.norm() > 0 and (p - q).norm() <= 52 * half * q.norm(), n
    assert all(p.grad is None or p.grad.isfinite().all() for p in fused.values())
