"""Backward passes of attention that take several rounds of heads, and diagonals that are dealt to several workgroups within one sequence."""
import math

import pytest
import torch

import train_reference as R
from oracle import hf_eager as O
from test_train_attention_gpu import TYPES, Case
from turbodeberta_amd.ops.trainable_attention import trainable_attention_with_disentangled as fixed

pytestmark = pytest.mark.gpu


def strip(x, rows, n):
    """[l, l] summed along its columns by the table row of each, which do not decrease: [l, n]."""
    ends = torch.searchsorted(rows, torch.arange(n, device=x.device).expand(len(x), n).contiguous(), right=True)
    sums = torch.nn.functional.pad(x.cumsum(1), (1, 0)).gather(1, ends)
    return sums.diff(dim=1, prepend=torch.zeros_like(sums[:, :1]))


def attention(q, k, v, pk, pq, dout, rows, scale, dtype, most):
    """train_reference.attention without dropout, its formulas and bounds, by products of [l, l] and [l, table rows] arrays."""
    u, half, U, l, n = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0, dtype == torch.float16, R.U, len(q), len(pk)
    steps = 100 + l / 8
    sums_q, sums_k = (lambda x: strip(x.flip(1), rows.flip(1).contiguous(), n)), (lambda x: strip(x.t().contiguous(), rows.t().contiguous(), n))
    score = lambda q, k, pk, pq: q @ k.t() + (q @ pk.t()).gather(1, rows) + (k @ pq.t()).gather(1, rows.t()).t()
    A = scale * score(*(t.abs() for t in (q, k, pk, pq)))
    p = torch.softmax(scale * score(q, k, pk, pq), -1)
    rho = 100 * U * (1 + A + A.amax(-1, keepdim=True))
    p_off = (u + rho + steps * U) * p
    o, o_off = p @ v, (p_off + (p.amax(-1, keepdim=True) * 2.0 ** -25 if half else 0)) @ v.abs()
    dv, dv_off = p.t() @ dout, (p_off + (2.0 ** -25 / 2 ** int(math.log2(l)) if half else 0)).t() @ dout.abs()
    dp = dout @ v.t()
    D = (p * dp).sum(-1, keepdim=True)
    D_off = (dout.abs() * (u * o.abs() + o_off + 70 * U * o.abs())).sum(-1, keepdim=True)
    ds = p * (dp - D)
    ds_off = (rho + u) * ds.abs() + p * (72 * U * (dout.abs() @ v.abs().t()) + D_off + 4 * U * (dp.abs() + D.abs())) * (1 + u) + (2.0 ** -25 / 2 ** 14 * 4 * most if half else 0)
    ds_off = ds_off + steps * U * ds.abs()
    by_q, by_k, by_q_off, by_k_off = sums_q(ds), sums_k(ds), sums_q(ds_off), sums_k(ds_off)
    got = {"o": (o, o_off), "dv": (dv, dv_off)}
    for name, x, off in (("dq", ds @ k + by_q @ pk, ds_off @ k.abs() + by_q_off @ pk.abs()), ("dk", ds.t() @ q + by_k @ pq, ds_off.t() @ q.abs() + by_k_off @ pq.abs()),
                         ("dpk", by_q.t() @ q, by_q_off.t() @ q.abs()), ("dpq", by_k.t() @ k, by_k_off.t() @ k.abs())):
        got[name] = (scale * x, scale * off)
    return got


def reference(c):
    """{name: (value, bound)} of a case without dropout."""
    d = lambda t: t.detach().double()
    most = (d(c.dout).norm(dim=-1).max() * d(c.v).norm(dim=-1).max()).item()
    ref = {n: [torch.zeros_like(d(x)) for _ in range(2)] for n, x in (("o", c.q), ("dq", c.q), ("dk", c.q), ("dv", c.q), ("dpk", c.pk), ("dpq", c.pq))}
    first = 0
    for l in c.lens:
        table = torch.from_numpy(O.delta_table(l, c.buckets, c.max_rel)).long().cuda()
        i = torch.arange(l, device="cuda")
        rows = table[i[:, None] - i[None] + l - 1]
        for h in range(c.H):
            at = lambda x: x[first:first + l, h]
            got = attention(*(d(at(t)) for t in (c.q, c.k, c.v)), d(c.pk[h]), d(c.pq[h]), d(at(c.dout)), rows, c.scale, c.dtype, most)
            for n, pair in got.items():
                for into, x in zip(ref[n], pair):
                    (into[h] if n in ("dpk", "dpq") else at(into)).add_(x)
        first += l
    return {n: [t.cpu() for t in pair] for n, pair in ref.items()}


def test_the_reference_is_the_other_ones():
    c = Case([200, 33], dtype=torch.float16, buckets=16, max_rel=64, seed=40)
    ours, theirs = reference(c), c.reference()
    for n in theirs:
        for a, b in zip(ours[n], theirs[n]):
            assert (a - b).abs().max() <= 1e-9 * b.abs().max(), n


# More than 64 tiles of rows and a batch that is too small to deal them out by sequences: 65 tiles of one, 64 each of three.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,buckets,max_rel", [([4160], 32, 128), ([4096] * 3, 16, 4000)])
def test_diagonals_dealt_out_within_a_sequence(lens, buckets, max_rel, dtype):
    c = Case(lens, H=1, D=16, dtype=dtype, buckets=buckets, max_rel=max_rel, seed=41)
    got = c.packed()
    for n, (ref, off) in reference(c).items():
        R.check(n, got[n], ref, off + (len(lens) * R.U * off.max().item() if n in ("dpk", "dpq") else 0.0))       # (sums over sequences)
    if len(set(lens)) == 1:
        same = c.padded(lens=False)
        assert all(torch.equal(same[n], got[n]) for n in ("dpk", "dpq"))


def grads(heads, tensors, buckets):
    q, k, v, pk, pq = (t[..., heads, :, :].detach().requires_grad_() for t in tensors[:5])
    o = fixed(q, k, v, pk, pq, 0.3, buckets, 64)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v, pk, pq), tensors[5][:, heads])]


# By the scores' gradients, 128 MiB a head, and by the positions' sums, 64 KiB a head: 2 GiB at a time of either.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,length,alone", [(18, 8192, [slice(0, 1), slice(7, 9), slice(15, 18)]), (40000, 64, [slice(0, 9), slice(32700, 32800), slice(39990, 40000)])])
def test_rounds_of_heads(heads, length, alone, dtype):
    """Each head's results are those it has in a call of few heads, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(43)
    make = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dtype)
    tensors = [*(make(1, heads, length, 8) for _ in range(3)), make(heads, 32, 8), make(heads, 32, 8), make(1, heads, length, 8)]
    whole = grads(slice(None), tensors, 16)
    for some in alone:
        for n, (a, b) in enumerate(zip(whole, grads(some, tensors, 16))):
            assert torch.equal(a[..., some, :, :], b), (some, n)
