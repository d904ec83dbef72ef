"""Modules that an operator of the training mode stands for, replaced or watched: they are called then.  The check of the device and the operators are stood in for."""
import copy

import pytest
import torch
from torch import nn
from transformers import DebertaV2Config

import turbodeberta_amd.model as model_module
import turbodeberta_amd.training as training
from turbodeberta_amd.model import FlashDisentangledSelfAttention
from turbodeberta_amd.training import FlashDebertaV2Output, FlashDebertaV2SelfOutput, FlashDropout, FlashLayerNorm

CONFIG = DebertaV2Config(hidden_size=32, num_attention_heads=4, intermediate_size=48, relative_attention=True, position_buckets=8, max_relative_positions=16, pos_att_type=["c2p", "p2c"],
                         hidden_dropout_prob=0.25, attention_probs_dropout_prob=0.25)


@pytest.fixture
def calls(monkeypatch):
    """The operators' calls, as (operator, probability); the modules that call an operator of their own do not here."""
    seen = []

    def joined(x, residual, weight, bias, p, seed, eps):
        seen.append(("dropout_add_layer_norm", p))
        return nn.functional.layer_norm(x + residual, x.shape[-1:], weight, bias, eps)

    def attention(q, k, v, *args, dropout_p=0.0, **kw):
        seen.append(("attention", dropout_p))
        return v.clone()

    monkeypatch.setattr(training, "operators_take", lambda module, *t: not isinstance(module, (FlashDropout, FlashLayerNorm)))
    monkeypatch.setattr(training, "dropout_add_layer_norm", joined)
    monkeypatch.setattr(model_module, "trainable_attention_with_disentangled", attention)
    return seen


def block(cls, drop=None):
    m = cls(CONFIG).train()
    m.dropout.__class__, m.LayerNorm.__class__ = FlashDropout, FlashLayerNorm
    if drop is not None:
        m.dropout = drop
    return m, torch.randn(2, 5, m.dense.in_features), torch.randn(2, 5, 32)


BLOCKS = [FlashDebertaV2SelfOutput, FlashDebertaV2Output]


@pytest.mark.parametrize("cls", BLOCKS)
def test_an_output_block_by_itself_is_one_operator(cls, calls):
    m, x, r = block(cls)
    m(x, r)
    m.eval()(x, r)
    assert calls == [("dropout_add_layer_norm", 0.25), ("dropout_add_layer_norm", 0.0)]


@pytest.mark.parametrize("cls", BLOCKS)
def test_dropout_switched_off_by_an_identity(cls, calls):
    m, x, r = block(cls, nn.Identity())
    torch.testing.assert_close(m(x, r), m.LayerNorm(m.dense(x) + r))
    assert calls == [("dropout_add_layer_norm", 0.0)]


class Doubled(nn.LayerNorm):
    def forward(self, x):
        return 2 * super().forward(x)


class Halved(nn.Dropout):
    def forward(self, x):
        return 0.5 * x


@pytest.mark.parametrize("cls", BLOCKS)
def test_classes_of_their_own_are_called(cls, calls):
    m, x, r = block(cls, Halved(0.25))
    torch.testing.assert_close(m(x, r), m.LayerNorm(0.5 * m.dense(x) + r))
    m, x, r = block(cls, nn.Identity())
    m.LayerNorm.__class__ = Doubled
    torch.testing.assert_close(m(x, r), 2 * nn.functional.layer_norm(m.dense(x) + r, (32,), m.LayerNorm.weight, m.LayerNorm.bias, m.LayerNorm.eps))
    m, x, r = block(cls, nn.Identity())
    m.LayerNorm.forward = lambda x: x
    torch.testing.assert_close(m(x, r), m.dense(x) + r)
    assert not calls


@pytest.mark.parametrize("cls", BLOCKS)
@pytest.mark.parametrize("name", ["dropout", "LayerNorm"])
@pytest.mark.parametrize("kind", ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"])
def test_hooks_fire(cls, name, kind, calls):
    m, x, r = block(cls)
    fired = []
    handle = getattr(m.get_submodule(name), kind)(lambda *a: fired.append(name))
    m(x.requires_grad_(), r).sum().backward()
    assert fired == [name] and not calls
    handle.remove()
    m(x, r)
    assert fired == [name] and len(calls) == 1


def test_what_a_hook_returns_is_the_result(calls):
    m, x, r = block(FlashDebertaV2Output)
    m.LayerNorm.register_forward_hook(lambda module, args, out: torch.zeros_like(out))
    assert not m(x, r).any() and not calls


def test_hooks_of_all_modules_fire(calls):
    m, x, r = block(FlashDebertaV2Output)
    fired = []
    handle = nn.modules.module.register_module_forward_hook(lambda module, args, out: fired.append(type(module).__name__))
    try:
        m(x, r)
    finally:
        handle.remove()
    assert {"FlashDropout", "FlashLayerNorm"} <= set(fired) and not calls


def attention(drop=None):
    m = FlashDisentangledSelfAttention(CONFIG).train()
    m.trainable, m.pos_dropout = True, nn.Identity()
    if drop is not None:
        m.dropout = drop
    mask = torch.ones(2, 1, 6, 6, dtype=torch.long)
    return m, lambda relative_pos=None, mask=mask: m(x, mask, rel_embeddings=rel, relative_pos=relative_pos)[0]


x, rel = torch.randn(2, 6, 32), torch.randn(16, 32)


def test_attentions_dropout(calls):
    attention()[1]()
    attention(nn.Identity())[1]()
    m, run = attention()
    m.eval()
    run()
    assert calls == [("attention", 0.25), ("attention", 0.0), ("attention", 0.0)]


def test_attentions_dropout_of_another_class_or_with_a_hook_is_called(calls):
    m, run = attention(Halved(0.25))
    whole = attention(nn.Identity())[0]
    whole.load_state_dict(m.state_dict())
    want = super(FlashDisentangledSelfAttention, whole).forward(x, torch.ones(2, 1, 6, 6), rel_embeddings=rel)[0]
    for relative_pos in (None, x.new_empty(0)):              # what a direct call and the encoder pass
        torch.testing.assert_close(run(relative_pos), 0.5 * want)
    torch.testing.assert_close(run(None, None), 0.5 * want)
    m, run = attention()
    shapes = []
    m.dropout.register_forward_hook(lambda module, args, out: shapes.append(tuple(out.shape)))
    run()
    assert shapes == [(2, 4, 6, 6)] and not calls


def test_a_norm_without_weights_takes_rows_of_its_width():
    """Other rows go to the parent's code, which raises."""
    norm = FlashLayerNorm(8, elementwise_affine=False)
    assert training._norm_arguments(norm, torch.zeros(2, 8)) is not None
    assert all(training._norm_arguments(norm, torch.zeros(shape)) is None for shape in ((2, 6), (8, 1), ()))
    with pytest.raises(RuntimeError):
        norm(torch.zeros(2, 6))


@pytest.mark.parametrize("cls", BLOCKS)
def test_inputs_that_broadcast(cls, calls):
    """The parent's sum takes them, the operator does not."""
    m, x, r = block(cls, nn.Identity())
    torch.testing.assert_close(m(x, r[:1]), m.LayerNorm(m.dense(x) + r[:1]))
    torch.testing.assert_close(m(x[:1], r), m.LayerNorm(m.dense(x[:1]) + r))
    assert not calls


@pytest.mark.parametrize("lengths", [(6, 6), (6, 2), (0, 5)])
@pytest.mark.parametrize("terms", [["c2p", "p2c"], ["c2p"], ["p2c"], []])
def test_attention_by_its_probabilities(terms, lengths, calls):
    """Hugging Face's module where tokens are valid, zeros behind them; gradients too."""
    config = copy.deepcopy(CONFIG)
    config.pos_att_type, config.relative_attention = terms, bool(terms)
    m = FlashDisentangledSelfAttention(config).double().train()
    m.trainable, m.pos_dropout, m.dropout = True, nn.Identity(), Halved(0.25)
    valid = torch.arange(6) < torch.tensor(lengths)[:, None]
    mask = (valid[:, None, :, None] & valid[:, None, None, :]).long()
    dy = torch.randn(2, 6, 32, dtype=torch.float64) * valid[..., None]
    out = []
    for forward in (m, super(FlashDisentangledSelfAttention, m).forward):
        m.zero_grad()
        h = x.double().requires_grad_()
        y = forward(h, mask, rel_embeddings=rel.double())[0]
        y.backward(dy)
        out.append([y[valid], h.grad] + [p.grad for p in m.parameters() if p.grad is not None])
        if forward is m:
            assert not y[~valid].any()
    # float32 products of 8 and 6 terms, their roundings' sum and a softmax between them: 50 steps of 2^-24
    assert len(out[0]) == len(out[1]) and all((a - b).norm() <= 50 * 2.0 ** -24 * max(b.norm(), 1) for a, b in zip(*out))
    assert not calls
