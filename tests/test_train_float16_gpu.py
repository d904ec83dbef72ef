"""float16: the scores' gradients are brought into the type's range by a power of two for each sequence and head, whatever its neighbours' sizes."""
import numpy as np
import pytest
import torch

import train_reference as R
from oracle import hf_eager as O
from test_train_attention_gpu import Case
from test_train_rounds_gpu import grads

pytestmark = pytest.mark.gpu


def alone(c, b, h=None):
    """The case of one sequence, or of one sequence and head."""
    rows, heads = slice(int(c.cu[b]), int(c.cu[b + 1])), slice(None) if h is None else slice(h, h + 1)
    one = Case([c.lens[b]], H=c.H if h is None else 1, dtype=c.dtype, buckets=c.buckets, max_rel=c.max_rel)
    for n in ("q", "k", "v", "dout"):
        setattr(one, n, getattr(c, n)[rows, heads].contiguous())
    one.pk, one.pq, one.scale = c.pk[heads].contiguous(), c.pq[heads].contiguous(), c.scale
    return one


# (64 .. 127 tokens: lengths that share the power of two of the probabilities)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** -8, 0.0, float("inf"), float("nan")])
def test_a_sequences_gradients_are_its_own(size):
    c = Case([100, 80, 64, 127], dtype=torch.float16, buckets=8, max_rel=32, seed=51)
    for b in (0, 2):
        c.dout[int(c.cu[b]):int(c.cu[b + 1])] *= size
    whole = c.packed(127)
    padded = c.unpad(c.padded(127), 127)
    for b in (1, 3):
        got, rows = alone(c, b).packed(), slice(int(c.cu[b]), int(c.cu[b + 1]))
        for n in ("o", "dq", "dk", "dv"):
            assert torch.equal(whole[n][rows], got[n]) and torch.equal(padded[n][rows], got[n]), (b, n)


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** -8, float("inf")])
def test_a_heads_gradients_are_its_own(size):
    c = Case([100, 80], H=3, dtype=torch.float16, buckets=8, max_rel=32, seed=52)
    c.dout[:, 1] *= size
    whole = c.packed()
    for h in (0, 2):
        parts = [alone(c, b, h).packed() for b in range(2)]
        for n in ("o", "dq", "dk", "dv"):
            assert torch.equal(whole[n][:, h], torch.cat([p[n] for p in parts])[:, 0]), (h, n)


# Seven sequences are dealt to four workgroups of a diagonal: 0 and 4, 1 and 5, 2 and 6, 3.  Long ones have positions that no short one has.
@pytest.mark.parametrize("sizes", [[10, -6, 4, 0, -6, 10, -4], [-6, 10, 0, 4, 10, -6, 8], [-20, -2, 0, -20, 10, -20, -8]])
@pytest.mark.parametrize("buckets,max_rel", [(0, 300), (8, 32), (0, 1)])
def test_table_gradients_of_sequences_of_any_size(sizes, buckets, max_rel):
    """Bounds as everywhere (train_reference.attention), with the largest |dout| |v| of the sequence and head in the place of the call's."""
    c = Case([150, 40, 77, 130, 150, 30, 64], dtype=torch.float16, buckets=buckets, max_rel=max_rel, seed=53)
    for b, e in enumerate(sizes):
        rows = slice(int(c.cu[b]), int(c.cu[b + 1]))
        c.dout[rows] *= 2.0 ** max(e, -8)
        c.v[rows] *= 2.0 ** (e - max(e, -8))
    got = c.packed()
    d = lambda t: t.detach().cpu().double()
    ref = {n: [torch.zeros_like(d(x)) for _ in range(2)] for n, x in (("o", c.q), ("dq", c.q), ("dk", c.q), ("dv", c.q), ("dpk", c.pk), ("dpq", c.pq))}
    for b, l in enumerate(c.lens):
        table = torch.from_numpy(O.delta_table(l, buckets, max_rel)).long()
        rows = table[torch.arange(l)[:, None] - torch.arange(l)[None] + l - 1]
        for h in range(c.H):
            at = lambda x: x[int(c.cu[b]):int(c.cu[b + 1]), h]
            most = (d(at(c.dout)).norm(dim=-1).max() * d(at(c.v)).norm(dim=-1).max()).item()
            one = R.attention(*(d(at(t)) for t in (c.q, c.k, c.v)), d(c.pk[h]), d(c.pq[h]), d(at(c.dout)), rows, c.scale, torch.ones(l, l, dtype=torch.float64), 1.0, c.dtype, most)
            for n, pair in one.items():
                for into, x in zip(ref[n], pair):
                    (into[h] if n in ("dpk", "dpq") else at(into)).add_(x)
    for n, (x, off) in ref.items():
        R.check(n, got[n], x, off + (len(c.lens) * R.U * off.max().item() if n in ("dpk", "dpq") else 0.0))


@pytest.mark.parametrize("heads,length,some", [(18, 8192, slice(15, 18)), (40000, 64, slice(32700, 32800))])
def test_rounds_of_heads(heads, length, some):
    """Each head's results are those it has in a call of few heads, bit for bit, whatever size the others have."""
    g = torch.Generator(device="cuda").manual_seed(43)
    make = lambda *shape: torch.randn(*shape, generator=g, device="cuda").half()
    tensors = [*(make(1, heads, length, 8) for _ in range(3)), make(heads, 32, 8), make(heads, 32, 8), make(1, heads, length, 8)]
    tensors[5] *= torch.from_numpy(2.0 ** np.random.RandomState(1).randint(-8, 9, heads)).half().cuda()[None, :, None, None]
    whole = grads(slice(None), tensors, 16)
    for n, (a, b) in enumerate(zip(whole, grads(some, tensors, 16))):
        assert torch.equal(a[..., some, :, :], b), n
