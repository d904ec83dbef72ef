"""What patch_model(training=True) does to a model, and the modules where autograd does not record or the CPU has the tensors."""
import pytest
import torch
from torch import nn
from transformers import DebertaV2Config
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2ForSequenceClassification, DebertaV2Model, DebertaV2SelfOutput

from turbodeberta_amd.model import FlashDisentangledSelfAttention, FlashDebertaV2Model, patch_model
from turbodeberta_amd.training import FlashDebertaV2Output, FlashDebertaV2SelfOutput, FlashDropout, FlashLayerNorm


def config(**other):
    return DebertaV2Config(**dict(dict(vocab_size=60, hidden_size=32, num_hidden_layers=2, num_attention_heads=4, intermediate_size=48, relative_attention=True, position_buckets=8,
                                       max_relative_positions=16, pos_att_type=["c2p", "p2c"], norm_rel_ebd="layer_norm", share_att_key=True), **other))


def test_what_is_switched():
    model = DebertaV2ForSequenceClassification(config())
    keys = list(model.state_dict())
    patch_model(model, training=True)
    assert list(model.state_dict()) == keys
    inner = model.deberta
    assert type(inner) is FlashDebertaV2Model and type(inner.embeddings.LayerNorm) is FlashLayerNorm and type(inner.embeddings.dropout) is FlashDropout
    assert type(inner.encoder.LayerNorm) is FlashLayerNorm
    for layer in inner.encoder.layer:
        att = layer.attention
        assert type(att.self) is FlashDisentangledSelfAttention and att.self.trainable and type(att.self.pos_dropout) is FlashDropout
        assert type(att.output) is FlashDebertaV2SelfOutput and type(layer.output) is FlashDebertaV2Output
    assert type(model.dropout) is nn.Dropout                    # the task head's
    model = patch_model(DebertaV2Model(config()))
    assert not any(isinstance(m, (FlashDropout, FlashLayerNorm, FlashDebertaV2SelfOutput)) for m in model.modules())
    assert not any(getattr(m, "trainable", False) for m in model.modules())
    patch_model(model, training=True)                           # a model that has been switched before
    assert all(m.trainable for m in model.modules() if isinstance(m, FlashDisentangledSelfAttention))


def test_head_dimensions_without_a_gradient():
    model = DebertaV2Model(config(hidden_size=48))              # 12
    with pytest.raises(ValueError, match="head dimension 12"):
        patch_model(model, training=True)
    assert not any(isinstance(m, FlashDisentangledSelfAttention) for m in model.modules())      # left as it was


def test_position_terms_without_relative_attention():
    model = DebertaV2Model(config(relative_attention=False, norm_rel_ebd="none"))
    with pytest.raises(ValueError, match="pos_att_type"):
        patch_model(model, training=True)


@pytest.mark.parametrize("train", [False, True])
def test_the_parents_code_on_the_cpu(train):
    torch.manual_seed(0)
    ours, theirs = FlashDebertaV2SelfOutput(config()), DebertaV2SelfOutput(config())
    theirs.load_state_dict(ours.state_dict())
    ours.dropout.__class__, ours.LayerNorm.__class__ = FlashDropout, FlashLayerNorm
    x, r = torch.randn(3, 5, 32), torch.randn(3, 5, 32)
    out = []
    for m in (ours, theirs):
        m.train(train)
        torch.manual_seed(1)
        y = m(x, r)
        y.square().sum().backward()
        out.append([y] + [p.grad for p in m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*out))
