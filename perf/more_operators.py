"""The two ends of a training step, as cases that can be timed and checked.

What a masked-language-model step needs beside its encoder: the loss over the vocabulary with its gradient, and the norm of all gradients
with clipping.  A case is a dict of plain values; ``prepare`` makes what a program has in hand before the call, ``run`` makes one
pass and returns its results: in plain torch operations, or, with ``own`` set, through this package's operators.

Loss: logits s = x W^T + b; rows whose label is IGNORED do not count; of the others log(sum(exp(s))) - s[label], as they are, or their sum or mean."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCAB = 128100
IGNORED = -100
MASKED = 0.15       # share of the tokens that masked language modelling predicts


def listed():
    return [
        # One short text: seven of its tokens are predicted.
        {"name": "loss_one_text", "op": "loss", "dtype": "bf16", "rows": 48, "hidden": 768, "vocab": VOCAB, "share": MASKED, "gap": 0, "bias": "same", "reduction": "mean", "grad": True},
        # A small batch of 8 x 128 tokens in float16.
        {"name": "loss_small_batch_fp16", "op": "loss", "dtype": "fp16", "rows": 1024, "hidden": 768, "vocab": VOCAB, "share": MASKED, "gap": 0, "bias": "same", "reduction": "mean", "grad": True},
        # The same in float32, the type that checkpoints are loaded in.
        {"name": "loss_small_batch_fp32", "op": "loss", "dtype": "fp32", "rows": 1024, "hidden": 768, "vocab": VOCAB, "share": MASKED, "gap": 0, "bias": "same", "reduction": "mean", "grad": True},
        # Sizes that are no multiple of anything, rows that lie apart, each row's loss weighted by the caller.
        {"name": "loss_odd_fp32", "op": "loss", "dtype": "fp32", "rows": 1013, "hidden": 771, "vocab": 30011, "share": 0.5, "gap": 5, "bias": "none", "reduction": "none", "grad": True},
        # A full batch of 32 x 512 tokens.
        {"name": "loss_batch", "op": "loss", "dtype": "bf16", "rows": 16384, "hidden": 768, "vocab": VOCAB, "share": MASKED, "gap": 0, "bias": "same", "reduction": "mean", "grad": True},
        # The same batch in evaluation: the loss of every token, no gradient.
        {"name": "loss_evaluation", "op": "loss", "dtype": "bf16", "rows": 16384, "hidden": 768, "vocab": VOCAB, "share": MASKED, "gap": 0, "bias": "fp32", "reduction": "none", "grad": False},
        # A large-sized model where every token of 16 x 512 is predicted.
        {"name": "loss_every_token", "op": "loss", "dtype": "bf16", "rows": 8192, "hidden": 1024, "vocab": VOCAB, "share": 1.0, "gap": 0, "bias": "same", "reduction": "mean", "grad": True},
        # The norm of a small model's gradients, to be logged.
        {"name": "norm_small_model", "op": "norm", "dtype": "fp32", "layers": 2, "hidden": 128, "vocab": 1000, "norm": 2.0},
        # The norm of a large-sized model's gradients, a healthy step: they stay as they are.
        {"name": "clip_healthy_fp32", "op": "clip", "dtype": "fp32", "layers": 24, "hidden": 1024, "vocab": VOCAB, "norm": 2.0, "share": 1.5},
        # Gradients in bfloat16 of a middle-sized model that are clipped into the float32 ones that its optimizer takes.
        {"name": "clip_into_fp32", "op": "clip_out", "dtype": "bf16", "out": "fp32", "layers": 12, "hidden": 512, "vocab": VOCAB, "norm": 2.0, "share": 0.25},
        # The same of a large-sized one in float16, into their own type.
        {"name": "clip_large_fp16", "op": "clip_out", "dtype": "fp16", "out": "fp16", "layers": 24, "hidden": 1024, "vocab": VOCAB, "norm": 2.0, "share": 0.5},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    if rng.random() < 0.3:
        op = rng.choice(["norm", "clip", "clip_out"])
        case = {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "layers": _log_int(rng, 1, 24), "hidden": rng.choice([8 * rng.randint(2, 128), rng.randint(5, 1024)]),
                "vocab": _log_int(rng, 100, VOCAB), "norm": rng.choice([2.0, 2.0, 2.0, 1.0, math.inf])}
        if op != "norm":
            case["share"] = round(rng.uniform(0.05, 0.95), 3) if op == "clip_out" else round(rng.uniform(1.05, 3.0), 3)
        return {**case, "out": rng.choice([case["dtype"], "fp32"])} if op == "clip_out" else case
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hidden = rng.choice([384, 768, 1024, 8 * rng.randint(4, 160), rng.randint(20, 1300)])
    vocab = rng.choice([VOCAB, VOCAB, _log_int(rng, 500, VOCAB), _log_int(rng, 500, VOCAB)])
    share = rng.choice([MASKED, MASKED, 1.0, round(rng.uniform(0.01, 1.0), 3)])
    budget = 8192 * 1024 * VOCAB // (12 if dtype == "fp32" else 1)
    rows = _log_int(rng, 1, max(1, min(16384, (1 << 31) // vocab, int(budget / (hidden * vocab * share)))))
    return {"op": "loss", "dtype": dtype, "rows": rows, "hidden": hidden, "vocab": vocab, "share": share, "gap": rng.choice([0, 0, 3, 8]),
            "bias": rng.choice(["same", "same", "fp32", "none"]), "reduction": rng.choice(["mean", "mean", "sum", "none"]), "grad": rng.random() < 0.85}


def _counting(case):
    """Rows that have a label: their number does not depend on the seed."""
    return max(1, round(case["rows"] * case["share"]))


def _shapes(case):
    """Parameters of an encoder with embeddings, as a model lists them."""
    h, inner = case["hidden"], 4 * case["hidden"]
    layer = [(h, h), (h,)] * 4 + [(h,), (h,), (inner, h), (inner,), (h, inner), (h,), (h,), (h,)]
    return [(case["vocab"], h), (h,), (h,), (512, h)] + layer * case["layers"]


def _bucket(case, dtype):
    """Memory for all gradients, and each one's part of it: how data-parallel training keeps them."""
    shapes = _shapes(case)
    sizes = [math.prod(shape) for shape in shapes]
    flat = torch.empty(sum(sizes), dtype=dtype, device="cuda")
    return flat, [t.view(shape) for t, shape in zip(flat.split(sizes), shapes)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    s = {"op": case["op"]}
    if case["op"] != "loss":
        # Layers' gradients differ in size; in float16 they are those of a scaled loss.
        size = 3e-2 if case["dtype"] == "fp16" else 1e-4
        s["flat"], s["grads"] = _bucket(case, dtype)
        for n, t in enumerate(s["grads"]):
            t.copy_(make(*t.shape) * (size * (1 + n % 7)))
        s["norm"] = case["norm"]
        if case["op"] == "norm":
            return s
        s["max"] = case["share"] * float(_plain_norm(s["grads"], case["norm"]))
        if case["op"] == "clip":
            s["params"] = [torch.nn.Parameter(torch.empty_like(t)) for t in s["grads"]]
            for p, t in zip(s["params"], s["grads"]):
                p.grad = t
        else:
            s["flat"], s["out"] = _bucket(case, DTYPES[case["out"]])
        return s
    rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
    weight = make(vocab, hidden) * (1.4 / math.sqrt(hidden))
    labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    # What the model believes of the right answer, from nothing to almost certain.
    sure = torch.rand(rows, 1, generator=g, device="cuda") * 12
    right = weight[labels]
    wide = make(rows, hidden + case["gap"])
    wide[:, :hidden] += sure * right / right.square().sum(-1, keepdim=True).clamp(min=1e-3)
    gone = torch.randperm(rows, generator=g, device="cuda")[_counting(case):]
    labels[gone] = IGNORED
    s["x"] = wide.to(dtype)[:, :hidden].requires_grad_(case["grad"])
    s["weight"] = weight.to(dtype).requires_grad_(case["grad"])
    s["labels"] = labels
    bias = make(vocab) * 0.3
    s["bias"] = None if case["bias"] == "none" else bias.to(torch.float32 if case["bias"] == "fp32" else dtype).requires_grad_(case["grad"])
    s["reduction"] = case["reduction"]
    s["grad"] = case["grad"]
    s["dy"] = torch.rand(rows, generator=g, device="cuda") / rows if case["reduction"] == "none" and case["grad"] else None
    return s


_LEAVES = (("dx", "x"), ("dweight", "weight"), ("dbias", "bias"))


def run(s):
    if own:
        return _run_own(s)
    return _loss(s) if s["op"] == "loss" else _norm(s)


def _run_own(s):
    if s["op"] == "norm":
        from turbodeberta_amd.ops.grad_norm import grad_norm
        return {"norm": grad_norm(s["grads"], s["norm"])}
    if s["op"] == "clip":
        from turbodeberta_amd.ops.grad_norm import clip_grad_norm_
        return {"norm": clip_grad_norm_(s["params"], s["max"], s["norm"]), "grads": s["flat"]}
    if s["op"] == "clip_out":
        from turbodeberta_amd.ops.grad_norm import clip_grads
        norm, _ = clip_grads(s["grads"], s["max"], s["norm"], out=s["out"])
        return {"norm": norm, "grads": s["flat"]}
    from turbodeberta_amd.ops.linear_cross_entropy import linear_cross_entropy
    loss = linear_cross_entropy(s["x"], s["weight"], s["labels"], s["bias"], ignore_index=IGNORED, reduction=s["reduction"])
    if not s["grad"]:
        return {"loss": loss}
    names, leaves = zip(*((n, s[k]) for n, k in _LEAVES if s[k] is not None))
    return {"loss": loss.detach(), **dict(zip(names, torch.autograd.grad(loss, leaves, s["dy"])))}


def _plain_norm(grads, kind):
    """In 64 bits: sums over hundreds of millions of values."""
    if kind == math.inf:
        return torch.stack([t.abs().amax() for t in grads]).amax().double()
    if kind == 1.0:
        return torch.stack([t.abs().sum(dtype=torch.float64) for t in grads]).sum()
    return torch.stack([t.float().square().sum(dtype=torch.float64) for t in grads]).sum().sqrt()


def _norm(s):
    norm = _plain_norm(s["grads"], s["norm"])
    if s["op"] == "norm":
        return {"norm": norm.float()}
    factor = (s["max"] / (norm + 1e-6)).clamp(max=1.0).float()
    if s["op"] == "clip":
        for p in s["params"]:
            p.grad.copy_(p.grad.float() * factor)
    else:
        for o, t in zip(s["out"], s["grads"]):
            o.copy_(t.float() * factor)
    return {"norm": norm.float(), "grads": s["flat"]}


def _loss(s):
    with torch.no_grad():
        x, weight, labels = s["x"].float(), s["weight"].float(), s["labels"]
        counts = labels != IGNORED
        at = labels.clamp(min=0)[:, None]
        logits = x @ weight.t()
        if s["bias"] is not None:
            logits += s["bias"].float()
        top = logits.amax(-1, keepdim=True)
        right = logits.gather(-1, at) - top
        logits = logits.sub_(top).exp_()
        sums = logits.sum(-1, keepdim=True)
        rows = ((sums.log() - right).squeeze(-1)).masked_fill_(~counts, 0.0)
        n = counts.sum()
        loss = rows if s["reduction"] == "none" else rows.sum(dtype=torch.float64) if s["reduction"] == "sum" else rows.sum(dtype=torch.float64) / n
        out = {"loss": loss.float()}
        if not s["grad"]:
            return out
        each = s["dy"] if s["reduction"] == "none" else counts.float() / (n.clamp(min=1) if s["reduction"] == "mean" else 1)
        d = logits.div_(sums)
        d.scatter_add_(-1, at, torch.full_like(right, -1.0))
        d *= (each * counts)[:, None]
        out["dx"] = (d @ weight).to(s["x"].dtype)
        out["dweight"] = (d.t() @ x).to(s["weight"].dtype)
        if s["bias"] is not None:
            out["dbias"] = d.sum(0).to(s["bias"].dtype)
        return out


def work(case):
    """Loss: every input that counts read once, every result written once; a product for the logits and two for the gradients.  Norms: every gradient
    read once, and written once where it is clipped."""
    size = lambda t: 4 if t == "fp32" else 2
    if case["op"] != "loss":
        n = float(sum(math.prod(shape) for shape in _shapes(case)))
        if case["op"] == "clip_out":
            return {"bytes": n * (size(case["dtype"]) + size(case["out"])), "flops": 3 * n}
        return {"bytes": n * size(case["dtype"]), "flops": 2 * n}
    n, h, v = _counting(case), case["hidden"], case["vocab"]
    e = size(case["dtype"])
    bias = 0 if case["bias"] == "none" else 4 if case["bias"] == "fp32" else e
    moved = e * (n * h + v * h) + bias * v + 8 * case["rows"] + (4 * case["rows"] if case["reduction"] == "none" else 4)
    if not case["grad"]:
        return {"bytes": float(moved), "flops": 2.0 * n * h * v}
    moved += e * (case["rows"] * h + v * h) + bias * v + (4 * case["rows"] if case["reduction"] == "none" else 0)
    return {"bytes": float(moved), "flops": 6.0 * n * h * v}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_loss(s) if s["op"] == "loss" else _exact_norm(s)


def _exact_norm(s):
    each = torch.stack([torch.linalg.vector_norm(t.flatten(), s["norm"], dtype=torch.float64) for t in s["grads"]])
    norm = torch.linalg.vector_norm(each, s["norm"])
    if s["op"] == "norm":
        return {"norm": norm}
    factor = min(1.0, s["max"] / (norm.item() + 1e-6))
    return {"norm": norm, "grads": torch.cat([t.flatten() for t in s["grads"]]).double() * factor}


def _exact_loss(s):
    """The rows that count, some at a time."""
    x, weight, labels = s["x"].double(), s["weight"].double(), s["labels"]
    bias = 0.0 if s["bias"] is None else s["bias"].double()
    index = (labels != IGNORED).nonzero().flatten()
    n = len(index)
    each = s["dy"].double() if s["reduction"] == "none" and s["grad"] else torch.full((len(labels),), 1.0 / max(n, 1) if s["reduction"] == "mean" else 1.0, dtype=torch.float64, device=x.device)
    rows = torch.zeros(len(labels), dtype=torch.float64, device=x.device)
    dx, dweight = torch.zeros_like(x), torch.zeros_like(weight)
    dbias = torch.zeros(len(weight), dtype=torch.float64, device=x.device)
    for part in index.split(max(1, (1 << 28) // len(weight))):
        score = torch.log_softmax(x[part] @ weight.t() + bias, -1)
        rows[part] = -score[torch.arange(len(part), device=x.device), labels[part]]
        if not s["grad"]:
            continue
        d = score.exp_()
        d[torch.arange(len(part), device=x.device), labels[part]] -= 1.0
        d *= each[part, None]
        dx[part] = d @ weight
        dweight += d.t() @ x[part]
        dbias += d.sum(0)
    out = {"loss": rows if s["reduction"] == "none" else rows.sum() if s["reduction"] == "sum" else rows.sum() / n}
    if s["grad"]:
        out |= {"dx": dx, "dweight": dweight}
        if s["bias"] is not None:
            out["dbias"] = dbias
    return out
