"""A masked language model whose loss is the operator's: what patch_model(fused_loss=True) does, and when the operator stands for the head.  The operator and the check of the device are
stood in for."""
import copy

import pytest
import torch
from torch import nn
from transformers import DebertaV2Config
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2ForMaskedLM, DebertaV2Model

import turbodeberta_amd.training as training
from turbodeberta_amd.model import FlashDebertaV2ForMaskedLM, patch_model


def config(**other):
    return DebertaV2Config(**dict(dict(vocab_size=60, hidden_size=32, num_hidden_layers=2, num_attention_heads=4, intermediate_size=48, relative_attention=True, position_buckets=8,
                                       max_relative_positions=16, pos_att_type=["c2p", "p2c"], hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0), **other))


def batch():
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(1, 60, (3, 7), generator=g)
    labels = torch.where(torch.rand(3, 7, generator=g) < 0.4, ids, -100)
    labels[0, 0] = 5
    return ids, labels


@pytest.fixture
def calls(monkeypatch):
    """The operator's calls; attention and the blocks are the parent's."""
    seen = []

    def loss(x, weight, labels, bias):
        seen.append(x.shape)
        return nn.functional.cross_entropy(nn.functional.linear(x, weight, bias).view(-1, len(weight)).float(), labels.view(-1))
    monkeypatch.setattr(training, "operators_take", lambda module, *t: isinstance(module, FlashDebertaV2ForMaskedLM) and torch.is_grad_enabled())
    monkeypatch.setattr(training, "linear_cross_entropy", loss)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    return seen


def fused(model):
    """The class and flag that patch_model gives, with the parent's attention inside."""
    model.__class__, model.fused_loss = FlashDebertaV2ForMaskedLM, True
    return model


def test_what_is_switched():
    model = DebertaV2ForMaskedLM(config())
    keys = list(model.state_dict())
    patch_model(model, training=True, fused_loss=True)
    assert type(model) is FlashDebertaV2ForMaskedLM and model.fused_loss and list(model.state_dict()) == keys
    assert not patch_model(FlashDebertaV2ForMaskedLM(config())).fused_loss
    with pytest.raises(ValueError, match="no DebertaV2ForMaskedLM"):
        patch_model(DebertaV2Model(config()), fused_loss=True)


@pytest.mark.parametrize("legacy", [True, False])
def test_the_loss_without_logits(legacy, calls):
    stock = DebertaV2ForMaskedLM(config(legacy=legacy))
    ids, labels = batch()
    wanted = stock(ids, labels=labels)
    model = fused(copy.deepcopy(stock))
    got = model(ids, labels=labels, output_hidden_states=True)
    assert calls == [(3, 7, 32)] and got.logits is None and len(got.hidden_states) == 3
    torch.testing.assert_close(got.loss, wanted.loss)
    got.loss.backward()
    wanted.loss.backward()
    for (name, p), q in zip(model.named_parameters(), stock.parameters()):
        torch.testing.assert_close(p.grad, q.grad, msg=name)
    loss, logits = model(ids, labels=labels, return_dict=False)
    torch.testing.assert_close(loss, wanted.loss)
    assert logits is None and len(calls) == 2


def test_calls_of_the_parent(calls):
    stock = DebertaV2ForMaskedLM(config())
    ids, labels = batch()
    model = fused(copy.deepcopy(stock))
    assert torch.equal(model(ids).logits, stock(ids).logits)
    with torch.no_grad():
        got = model(ids, labels=labels)
    assert got.logits is not None
    model.fused_loss = False
    assert model(ids, labels=labels).logits is not None
    assert not calls


@pytest.mark.parametrize("legacy", [True, False])
@pytest.mark.parametrize("change", ["hook", "replaced", "forward", "subclass"])
def test_a_head_that_is_watched_or_replaced(change, legacy, calls):
    model = fused(DebertaV2ForMaskedLM(config(legacy=legacy)))
    seen = []
    head = model.cls.predictions if legacy else model.lm_predictions.lm_head
    if change == "hook":
        head.register_forward_hook(lambda *a: seen.append(1))
    elif change == "replaced":
        class Head(type(head)):
            pass
        head.__class__ = Head
    elif change == "forward":
        own = head.forward
        head.forward = lambda *a: own(*a)
    elif legacy:
        model.cls.predictions.decoder = nn.Sequential(nn.Linear(32, 60))
    else:
        model.lm_predictions.register_forward_pre_hook(lambda *a: seen.append(1))
    ids, labels = batch()
    assert model(ids, labels=labels).logits is not None and not calls
    assert change != "hook" or seen


def test_on_the_cpu_the_parents_code():
    stock = DebertaV2ForMaskedLM(config())
    ids, labels = batch()
    model = copy.deepcopy(stock)
    model.__class__, model.fused_loss = FlashDebertaV2ForMaskedLM, True
    got, wanted = model(ids, labels=labels), stock(ids, labels=labels)
    assert torch.equal(got.loss, wanted.loss) and torch.equal(got.logits, wanted.logits)
