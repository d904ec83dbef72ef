"""A model trained with the operators together, against Hugging Face's own modules in 64 bits with the same masks."""
import copy

import pytest
import torch
from torch import nn
from transformers import DebertaV2Config
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2Model

import turbodeberta_amd.training as training
from train_reference import drop, keep_of, keep_of_probabilities
from turbodeberta_amd.model import patch_model

pytestmark = pytest.mark.gpu
B, L, LENGTHS = 3, 70, (70, 1, 33)


def config(p, **other):
    return DebertaV2Config(**dict(dict(vocab_size=60, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, intermediate_size=96, relative_attention=True, position_buckets=8,
                                       max_relative_positions=24, pos_att_type=["c2p", "p2c"], norm_rel_ebd="layer_norm", share_att_key=True, position_biased_input=False,
                                       type_vocab_size=0, hidden_dropout_prob=p, attention_probs_dropout_prob=p, initializer_range=0.2), **other))


class Kept(nn.Module):
    """A dropout of the model in 64 bits, with the masks of the seeds that its counterpart has drawn."""

    def __init__(self, p, seeds):
        super().__init__()
        self.p, self.seeds = p, list(seeds)

    def forward(self, x):
        if not self.seeds:
            return x
        seed = self.seeds.pop(0)
        if x.shape[-1] == x.shape[-2] == L and x.numel() == B * 4 * L * L:
            keep = torch.stack([keep_of_probabilities(L, n, self.p, seed) for n in range(B * 4)]).reshape(x.shape)
        else:
            keep = keep_of(tuple(x.shape), self.p, seed)
        return drop(x, keep)


def inputs():
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(1, 60, (B, L), generator=g)
    mask = (torch.arange(L) < torch.tensor(LENGTHS)[:, None]).long()
    return ids * mask, mask, torch.randn(B, L, 64, generator=g, dtype=torch.float64) * mask[..., None]


def gradients(model, ids, mask, dout):
    out = model(input_ids=ids, attention_mask=mask).last_hidden_state
    (out * dout.to(out.dtype)).sum().backward()
    return out.detach()


def compare(model, exact, out, wanted, mask, tol):
    valid = mask.bool().cpu()
    err = lambda a, b: (a.double().cpu() - b).norm().item() / b.norm().item()
    assert err(out.cpu()[valid], wanted[valid]) <= tol
    ours, theirs = dict(model.named_modules()), dict(exact.named_modules())
    seen = 0
    for name, module in theirs.items():
        params = [n for n, p in module.named_parameters(recurse=False) if p.grad is not None]
        if params:          # a module's together: a bias whose gradient all but cancels is measured by its weight's
            flat = lambda m: torch.cat([getattr(m, n).grad.double().cpu().flatten() for n in params])
            assert err(flat(ours[name]), flat(module)) <= tol, name
            seen += 1
    assert seen >= 15


def run(p, monkeypatch, dtype=torch.float32, autocast=False, **other):
    """(model on the GPU, its result, the model in 64 bits, its result, the mask), both with gradients."""
    torch.manual_seed(11)
    stock = DebertaV2Model(config(p, **other)).to(dtype)
    exact = copy.deepcopy(stock).double().train()
    model = patch_model(copy.deepcopy(stock), training=True).cuda().train()
    names = {m: n for n, m in model.named_modules()}
    seeds = {}

    def draw(module, device):
        seed = training.new_seed(device)
        seeds.setdefault(names[module], []).append(seed.item())
        return seed

    monkeypatch.setattr(training, "draw_seed", draw)
    ids, mask, dout = inputs()
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        out = gradients(model, ids.cuda(), mask.cuda(), dout.cuda())
    for name, module in list(exact.named_modules()):
        if type(module) is nn.Dropout:
            parent = name.rsplit(".", 1)[0]
            own = seeds.pop(name, None) or (seeds.pop(parent, []) if name.endswith(".dropout") and not name.endswith("pos_dropout") else [])
            setattr(exact.get_submodule(parent), name.rsplit(".", 1)[1], Kept(module.p, own))
    assert not seeds
    wanted = gradients(exact, ids, mask, dout)
    assert all(not m.seeds for m in exact.modules() if isinstance(m, Kept))
    return model, out, exact, wanted, mask


# Tolerances, relative to the norm of a result or of a module's gradients.  Between the loss and the embeddings lie two layers, forward and backward, of some 20 operations each,
# a rounding or the sum of up to 96 terms: 80 steps.  float32: a sum of n terms is off by n U at most, 96 x 2^-24, and 80 of them by 4.6e-4 where each adds to the last; random
# signs make it the root of both: 10 x 9 U = 5e-6, and the LayerNorms and softmaxes in between, whose inputs have a spread of up to 10, ten times as much.  bfloat16: 80 roundings of
# 2^-9 on average, root 9, and ten times as much: 0.18.
FLOAT32, BFLOAT16 = 5e-5, 0.18


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("other", [{}, {"share_att_key": False}, {"pos_att_type": ["p2c"]}, {"relative_attention": False, "norm_rel_ebd": "none", "pos_att_type": []}])
def test_a_models_gradients(p, other, monkeypatch):
    model, out, exact, wanted, mask = run(p, monkeypatch, **other)
    compare(model, exact, out, wanted, mask, FLOAT32)


def test_in_bfloat16_and_under_autocast(monkeypatch):
    for kind in ({"dtype": torch.bfloat16}, {"autocast": True}):
        model, out, exact, wanted, mask = run(0.25, monkeypatch, **kind)
        compare(model, exact, out, wanted, mask, BFLOAT16)


# (The reentrant kind runs a layer without gradients first.  Hugging Face's own modules fail with it where the relative embeddings have a LayerNorm, whose graph
# all layers share.)
@pytest.mark.parametrize("reentrant,norm", [(False, "layer_norm"), (False, "none"), (True, "none")])
def test_the_generator_decides_and_checkpointing_finds_the_masks_again(reentrant, norm):
    torch.manual_seed(11)
    model = patch_model(DebertaV2Model(config(0.25, norm_rel_ebd=norm)), training=True).cuda().train()
    ids, mask, dout = (t.cuda() for t in inputs())

    def grads(seed):
        model.zero_grad()
        torch.manual_seed(seed)
        out = gradients(model, ids, mask, dout)
        return [out] + [p.grad.clone() for p in model.parameters() if p.grad is not None]

    first, again, other = grads(1), grads(1), grads(2)
    near = lambda a, b: all((x - y).norm() <= FLOAT32 * y.norm() for x, y in zip(a, b))
    assert near(first, again) and not near(first, other)
    model.gradient_checkpointing_enable(gradient_checkpointing_kwargs={"use_reentrant": reentrant})
    assert near(grads(1), first)


def test_training_mode_without_gradients_drops_the_same():
    torch.manual_seed(11)
    model = patch_model(DebertaV2Model(config(0.25)), training=True).cuda().train()
    ids, mask, _ = (t.cuda() for t in inputs())
    out = []
    for grad in (True, False):
        torch.manual_seed(3)
        with torch.set_grad_enabled(grad):
            out.append(model(input_ids=ids, attention_mask=mask).last_hidden_state.detach())
    assert torch.equal(*out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_evaluation_is_as_before(dtype):
    torch.manual_seed(11)
    stock = DebertaV2Model(config(0.25)).to(dtype)
    ids, mask, _ = (t.cuda() for t in inputs())
    out = []
    for training_too in (False, True):
        model = patch_model(copy.deepcopy(stock), training=training_too).cuda().eval()
        with torch.no_grad():
            out.append([model(input_ids=ids, attention_mask=m).last_hidden_state for m in (mask, torch.ones_like(mask))])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_a_model_that_has_been_evaluated_before():
    torch.manual_seed(11)
    model = patch_model(DebertaV2Model(config(0.25))).cuda().eval()
    ids, mask, dout = (t.cuda() for t in inputs())
    evaluate = lambda: [model(input_ids=ids, attention_mask=m).last_hidden_state for m in (mask, torch.ones_like(mask))]
    with torch.no_grad():
        before = evaluate()
    patch_model(model, training=True)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(before, evaluate()))
    gradients(model.train(), ids, mask, dout)
    model.eval()
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(before, evaluate()))


def test_gradients_reach_the_embeddings_of_a_model_in_eval_mode():
    """Without dropout, whatever the mode: the gradient of inputs."""
    torch.manual_seed(11)
    model = patch_model(DebertaV2Model(config(0.25)), training=True).cuda().eval()
    ids, mask, dout = (t.cuda() for t in inputs())
    x = model.embeddings.word_embeddings(ids).detach().requires_grad_()
    run = lambda: (model(inputs_embeds=x, attention_mask=mask).last_hidden_state * dout.float()).sum()
    a, = torch.autograd.grad(run(), x)
    b, = torch.autograd.grad(run(), x)
    assert torch.equal(a, b) and a[0].abs().sum() > 0 and not a[2, LENGTHS[2]:].any()
