"""A trained model whose modules have been replaced or have hooks, against Hugging Face's own modules in 64 bits with the same ones."""
import copy

import pytest
import torch
from torch import nn
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2Model

from test_training_gpu import BFLOAT16, FLOAT32, compare, config, gradients, inputs
from turbodeberta_amd.model import patch_model

pytestmark = pytest.mark.gpu


class Halved(nn.Dropout):
    def forward(self, x):
        return 0.5 * x


def identities(model):
    for m in list(model.modules()):
        for name in ("dropout", "pos_dropout"):
            if name in m._modules:
                setattr(m, name, nn.Identity())


def classes(model):
    for layer in model.encoder.layer:
        layer.attention.self.dropout = layer.output.dropout = Halved(0.25)


def hooks(model):
    for layer in model.encoder.layer:
        layer.output.LayerNorm.register_forward_hook(lambda module, args, out: 2 * out)
        layer.attention.output.LayerNorm.register_full_backward_pre_hook(lambda module, grads: tuple(0.5 * g for g in grads))
        layer.attention.self.dropout.register_forward_hook(lambda module, args, out: 0.75 * out)


# (Halving what leaves a softmax, or doubling what leaves a LayerNorm, is exact and changes no relative error.)
@pytest.mark.parametrize("change,p", [(identities, 0.25), (classes, 0.0), (hooks, 0.0)])
def test_a_models_gradients(change, p):
    torch.manual_seed(11)
    stock = DebertaV2Model(config(p))
    exact = copy.deepcopy(stock).double().train()
    model = patch_model(copy.deepcopy(stock), training=True).cuda().train()
    for m in (exact, model):
        change(m)
    ids, mask, dout = inputs()
    out = gradients(model, ids.cuda(), mask.cuda(), dout.cuda())
    compare(model, exact, out, gradients(exact, ids, mask, dout), mask, FLOAT32)


@pytest.mark.parametrize("change", [classes, hooks])
@pytest.mark.parametrize("autocast", [False, True])
def test_in_bfloat16_and_under_autocast(change, autocast):
    torch.manual_seed(11)
    stock = DebertaV2Model(config(0.0)).to(torch.float32 if autocast else torch.bfloat16)
    exact = copy.deepcopy(stock).double().train()
    model = patch_model(copy.deepcopy(stock), training=True).cuda().train()
    for m in (exact, model):
        change(m)
    ids, mask, dout = inputs()
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        out = gradients(model, ids.cuda(), mask.cuda(), dout.cuda())
    compare(model, exact, out, gradients(exact, ids, mask, dout), mask, BFLOAT16)
