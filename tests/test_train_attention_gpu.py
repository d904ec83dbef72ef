"""Attention with its gradient against 64 bits, sequence by sequence and head by head."""
import math

import pytest
import torch

import train_reference as R
from oracle import hf_eager as O
from turbodeberta_amd.ops.flash_attention import flash_attention_with_disentangled
from turbodeberta_amd.ops.trainable_attention import trainable_attention_with_disentangled as fixed
from turbodeberta_amd.ops.trainable_attention import trainable_attention_with_disentangled_varlen as varlen

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _seed(value):
    return torch.tensor([value], dtype=torch.int64, device="cuda")


class Case:
    """Inputs on the GPU: packed [T, H, D] in order, boundaries, tables."""

    def __init__(self, lens, H=2, D=64, dtype=torch.bfloat16, terms="both", buckets=32, max_rel=64, p=0.0, size=0.6, dsize=0.1, seed=1):
        self.lens, self.H, self.D, self.dtype, self.p, self.buckets, self.max_rel = list(lens), H, D, dtype, p, buckets, max_rel
        self.g = torch.Generator().manual_seed(seed)
        T, span = sum(lens), buckets if buckets > 0 else max_rel
        make = lambda s, *shape: (torch.randn(*shape, generator=self.g) * s).to(dtype).cuda()
        self.q, self.k, self.v, self.dout = make(size, T, H, D), make(size, T, H, D), make(size, T, H, D), make(dsize, T, H, D)
        self.pk = make(size, H, 2 * span, D) if terms in ("both", "c2p") else None
        self.pq = make(size, H, 2 * span, D) if terms in ("both", "p2c") else None
        self.scale = 1 / math.sqrt(D * (1 + (self.pk is not None) + (self.pq is not None)))
        self.seed = _seed(-987654321987 + seed)
        self.cu = torch.tensor([0] + list(torch.tensor(self.lens).cumsum(0)), dtype=torch.int32).cuda()

    @property
    def names(self):
        return ["dq", "dk", "dv"] + ["dpk"] * (self.pk is not None) + ["dpq"] * (self.pq is not None)

    def grads(self, call, q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, self.pk, self.pq) if t is not None]
        rest = leaves[3:]
        pk = rest.pop(0) if self.pk is not None else None
        pq = rest.pop(0) if self.pq is not None else None
        o = call(*leaves[:3], pk, pq)
        return {"o": o.detach(), **dict(zip(self.names, torch.autograd.grad(o, leaves, dout)))}

    def packed(self, longest=None):
        call = lambda q, k, v, pk, pq: varlen(q, k, v, pk, pq, self.cu, longest or max(self.lens + [1]), self.scale, self.buckets, self.max_rel, dropout_p=self.p, seed=self.seed)
        return self.grads(call, self.q, self.k, self.v, self.dout)

    def pad(self, t, L, fill=0.0):
        out = torch.full((len(self.lens), L, self.H, self.D), fill, dtype=t.dtype, device=t.device)
        for b, n in enumerate(self.lens):
            out[b, :n] = t[int(self.cu[b]):int(self.cu[b]) + n]
        return out.transpose(1, 2)

    def padded(self, L=None, fill=0.0, lens=True):
        L = L or max(self.lens + [1])
        n = torch.tensor(self.lens, dtype=torch.int32).cuda() if lens else None
        call = lambda q, k, v, pk, pq: fixed(q, k, v, pk, pq, self.scale, self.buckets, self.max_rel, seqlens_k=n, dropout_p=self.p, seed=self.seed)
        return self.grads(call, *(self.pad(t, L, fill) for t in (self.q, self.k, self.v, self.dout)))

    def unpad(self, got, L):
        out = dict(got)
        for n in ("o", "dq", "dk", "dv"):
            t = got[n].transpose(1, 2)
            out[n] = torch.cat([t[b, :m] for b, m in enumerate(self.lens)])
            for b, m in enumerate(self.lens):
                assert not t[b, m:].any(), f"{n}: padding of sequence {b}"
        return out

    def reference(self):
        c = lambda t: None if t is None else t.detach().cpu().double()
        q, k, v, dout, pk, pq = (c(t) for t in (self.q, self.k, self.v, self.dout, self.pk, self.pq))
        t = round(65536 * self.p)
        factor = 65536 / (65536 - t) if t else 1.0
        most = (dout.norm(dim=-1).max() * v.norm(dim=-1).max()).item() if len(q) else 0.0
        ref = {n: [torch.zeros_like(x), torch.zeros_like(x)] for n, x in (("o", q), ("dq", q), ("dk", q), ("dv", q), ("dpk", pk), ("dpq", pq)) if x is not None}
        first = 0
        for b, l in enumerate(self.lens):
            if l == 0:
                continue
            rows = None
            if pk is not None or pq is not None:
                table = torch.from_numpy(O.delta_table(l, self.buckets, self.max_rel)).long()
                i = torch.arange(l)
                rows = table[i[:, None] - i[None] + l - 1]
            for h in range(self.H):
                keep = R.keep_of_probabilities(l, b * self.H + h, self.p, self.seed.item()) if t else torch.ones(l, l, dtype=torch.float64)
                at = lambda x: x[first:first + l, h]
                got = R.attention(at(q), at(k), at(v), None if pk is None else pk[h], None if pq is None else pq[h], at(dout), rows, self.scale, keep, factor, self.dtype, most)
                for n, pair in got.items():
                    for into, x in zip(ref[n], pair):
                        (into[h] if n in ("dpk", "dpq") else at(into)).add_(x)
            first += l
        return ref

    def check(self, got):
        for n, (ref, off) in self.reference().items():
            more = len(self.lens) * R.U * off.max().item() if n in ("dpk", "dpq") else 0.0      # (sums over sequences)
            R.check(n, got[n], ref, off + more)


# lengths at the edges of the 16-row blocks, the 64-row steps and the 128-row tiles
LENGTHS = [[1], [2], [15, 17], [63], [64], [65, 1, 3], [100, 128], [129], [190, 0, 7, 64], [257]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", LENGTHS)
def test_packed(lens, dtype):
    c = Case(lens, dtype=dtype)
    c.check(c.packed())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", LENGTHS)
def test_padded_with_dropout(lens, dtype):
    c = Case(lens, dtype=dtype, p=0.2, seed=2)
    L = max(lens) + 9
    c.check(c.unpad(c.padded(L), L))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("terms", ["both", "c2p", "p2c", "none"])
@pytest.mark.parametrize("buckets,max_rel", [(256, 512), (8, 100), (0, 40), (0, 300)])
def test_terms_and_buckets(buckets, max_rel, terms, dtype):
    c = Case([150, 37], dtype=dtype, terms=terms, buckets=buckets, max_rel=max_rel, p=0.1, seed=3)
    c.check(c.packed())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 56])
def test_head_dimensions(D, dtype):
    c = Case([70, 130], D=D, H=3, dtype=dtype, p=0.3, seed=4)
    c.check(c.packed())


@pytest.mark.parametrize("dtype", TYPES)
def test_longer(dtype):
    """Offsets beyond the tables' ends, several rounds of the rings, rows shared by hundreds of offsets."""
    c = Case([700], H=1, dtype=dtype, buckets=32, max_rel=128, p=0.1, seed=5)
    c.check(c.packed())


@pytest.mark.parametrize("dtype", TYPES)
def test_sharp_and_large_scores(dtype):
    """Scores of some hundreds: probabilities of 0 and 1, maxima that move."""
    c = Case([140], dtype=dtype, size=4.0, seed=6)
    c.check(c.packed())


@pytest.mark.parametrize("dsize", [1e-4, 200.0])
def test_float16_gradients_of_any_size(dsize):
    """The scores' gradients are brought into float16's range, whatever the size of the result's."""
    c = Case([200], dtype=torch.float16, dsize=dsize, seed=7)
    c.check(c.packed())


@pytest.mark.parametrize("dtype", TYPES)
def test_padded_equals_packed(dtype):
    c = Case([129, 64, 0, 31], dtype=dtype, p=0.1, seed=8)
    a, b = c.packed(), c.unpad(c.padded(140), 140)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", TYPES)
def test_padding_is_not_read(dtype):
    """Infinities and NaN behind the valid rows, in the inputs and in the result's gradient."""
    c = Case([100, 1, 65], dtype=dtype, p=0.1, seed=9)
    clean = c.padded(131)
    for fill in (float("nan"), float("inf"), torch.finfo(dtype).min):
        got = c.padded(131, fill)
        assert all(torch.equal(got[n], clean[n]) for n in got)


def test_unpadded_batch_without_lengths():
    c = Case([96, 96, 96], p=0.1, seed=10)
    a, b = c.padded(96), c.padded(96, lens=False)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_with_gaps(dtype):
    """Tokens in front of, between and behind the sequences, and what max_seqlen cuts off: zeros, whatever they hold; the others as without them."""
    c = Case([50, 90, 20], dtype=dtype, seed=11)
    T, spread = 230, {}
    for n in ("q", "k", "v", "dout"):
        spread[n] = torch.full((T, c.H, c.D), float("nan"), dtype=dtype, device="cuda")
        for start, first, l in zip((3, 60, 190), (0, 50, 140), c.lens):
            spread[n][start:start + l] = getattr(c, n)[first:first + l]
    for start, first, l in zip((3, 60, 190), (0, 50, 140), c.lens):        # one sequence at a time among rows of none
        cu = torch.tensor([start, start + l], dtype=torch.int32).cuda()
        run = lambda cu, *t: c.grads(lambda q, k, v, pk, pq: varlen(q, k, v, pk, pq, cu, l, c.scale, c.buckets, c.max_rel), *t)
        got, want = run(cu, *spread.values()), run(cu - start, *(getattr(c, n)[first:first + l] for n in spread))
        for n in ("o", "dq", "dk", "dv"):
            assert torch.equal(got[n][start:start + l], want[n])
            assert not got[n][:start].any() and not got[n][start + l:].any()
    cut = Case([40, 90], dtype=dtype, seed=12)
    got = cut.packed(64)
    short = Case([40, 64], dtype=dtype, seed=13)
    for n in ("q", "k", "v", "dout"):
        setattr(short, n, torch.cat([getattr(cut, n)[:40], getattr(cut, n)[40:104]]))
    short.pk, short.pq = cut.pk, cut.pq
    ref = short.packed(64)
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n][:104], ref[n]) and not got[n][104:].any()
    assert torch.equal(got["dpk"], ref["dpk"]) and torch.equal(got["dpq"], ref["dpq"])


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Views of one projection, contiguous heads, rows that are not aligned, an expanded gradient, shared heads, tables with more rows and a leading 1."""
    c = Case([77, 77], dtype=dtype, p=0.1, seed=14)
    base = c.padded(77, lens=False)
    B, L, H, D = 2, 77, c.H, c.D
    q, k, v, dout = (c.pad(t, L) for t in (c.q, c.k, c.v, c.dout))
    call = lambda q, k, v, pk, pq: fixed(q, k, v, pk, pq, c.scale, c.buckets, c.max_rel, dropout_p=c.p, seed=c.seed)
    fused = torch.stack([t.transpose(1, 2) for t in (q, k, v)], 2).permute(2, 0, 3, 1, 4).unbind(0)
    for got in (c.grads(call, *fused, dout), c.grads(call, *(t.contiguous() for t in (q, k, v)), dout.contiguous())):
        assert all(torch.equal(got[n], base[n]) for n in got)
    wide = [torch.empty(B, H, L, D + 1, dtype=dtype, device="cuda")[..., 1:] for _ in range(3)]
    for w, t in zip(wide, (q, k, v)):
        w.copy_(t)
    got = c.grads(call, *wide, dout)
    assert all(torch.equal(got[n], base[n]) for n in got)
    ones = c.grads(call, q, k, v, torch.ones(1, dtype=dtype, device="cuda").expand(B, H, L, D))
    full = c.grads(call, q, k, v, torch.ones(B, H, L, D, dtype=dtype, device="cuda"))
    assert all(torch.equal(ones[n], full[n]) for n in ones)
    k1 = k[:, :1].detach().clone().requires_grad_()         # one head of keys for all queries' heads
    qs = q.detach().requires_grad_()
    dk1, = torch.autograd.grad(call(qs, k1.expand(B, H, L, D), v, c.pk, c.pq), k1, dout)
    ks = k1.detach().expand(B, H, L, D).contiguous().requires_grad_()
    dks, = torch.autograd.grad(call(qs, ks, v, c.pk, c.pq), ks, dout)
    assert torch.equal(dk1, dks.sum(1, keepdim=True))
    more = torch.cat([c.pk, torch.full_like(c.pk[:, :3], float("nan"))], 1)[None].requires_grad_()
    d, = torch.autograd.grad(call(q, k, v, more, c.pq), more, dout)
    assert d.shape == more.shape and torch.equal(d[0, :, :-3], base["dpk"]) and not d[0, :, -3:].any()


def test_same_result_as_the_forward_operator():
    """Both round the probabilities once; the forward operator its position terms as well, so: twice the bound."""
    for dtype in TYPES:
        c = Case([90, 200], dtype=dtype, buckets=256, max_rel=512, seed=15)
        q, k, v = (c.pad(t, 200) for t in (c.q, c.k, c.v))
        lens = torch.tensor(c.lens, dtype=torch.int32).cuda()
        a = fixed(q, k, v, c.pk, c.pq, c.scale, 256, 512, seqlens_k=lens)
        b = flash_attention_with_disentangled(q, k, v, None, None, False, c.scale, 256, 512, pos_key_layer=c.pk, pos_query_layer=c.pq, seqlens_k=lens)
        assert (a.float() - b.float()).abs().max().item() <= (1e-5 if dtype == torch.float32 else 2e-2)


def test_gradients_against_differences():
    c = Case([40], H=1, dtype=torch.float32, p=0.2, dsize=1.0, seed=16)
    got, h = c.packed(), 2.0 ** -6
    for name, leaf in (("dq", "q"), ("dk", "k"), ("dv", "v"), ("dpk", "pk"), ("dpq", "pq")):
        at = getattr(c, leaf)
        d = torch.randn(at.shape, generator=c.g).cuda()
        d /= d.norm()

        def loss(s):
            t = {n: getattr(c, n) for n in ("q", "k", "v", "pk", "pq")}
            t[leaf] = at + s * d
            o = varlen(t["q"], t["k"], t["v"], t["pk"], t["pq"], c.cu, 40, c.scale, c.buckets, c.max_rel, dropout_p=c.p, seed=c.seed)
            return (o.double() * c.dout.double()).sum().item()
        slope = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
        assert abs(slope - (got[name].double() * d.double()).sum().item()) <= 1e-3 * got[name].double().norm().item(), name


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_time_and_other_streams(dtype):
    c = Case([300, 77, 128], H=4, dtype=dtype, p=0.1, seed=17)
    first = c.packed()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = [c.packed() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(first[n], o[n]) for o in other for n in first)


def test_captured_and_replayed():
    """Forward and backward in two graphs of the same inputs, replayed beside eager work with other values and seeds."""
    c = Case([130, 60], p=0.1, seed=18)
    q, seed = c.q.clone(), c.seed.clone()

    def step(q, seed):
        c.seed = seed
        call = lambda q, k, v, pk, pq: varlen(q, k, v, pk, pq, c.cu, 130, c.scale, c.buckets, c.max_rel, dropout_p=c.p, seed=seed)
        return c.grads(call, q, c.k, c.v, c.dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, seed)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step(q, seed)))
    for n in range(4):
        q.copy_(c.q * (1 + 0.25 * n))
        seed.fill_(500 + n)
        want = {k: t.clone() for k, t in step(q.clone(), _seed(500 + n)).items()}
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], want[k]) for _, out in graphs for k in want)


def test_nothing_to_do():
    empty = torch.zeros(5, 2, 64, device="cuda", requires_grad=True)
    pk = torch.zeros(2, 64, 64, device="cuda", requires_grad=True)
    for cu in ([0], [0, 0], [0, 0, 0, 0]):
        o = varlen(empty, empty, empty, pk, None, torch.tensor(cu, dtype=torch.int32).cuda(), 8, None, 32, 64)
        d, dp = torch.autograd.grad(o, (empty, pk), torch.ones_like(o))
        assert not o.any() and not d.any() and not dp.any()
    none = torch.zeros(0, 2, 64, device="cuda", requires_grad=True)
    o = varlen(none, none, none, pk, None, torch.tensor([0, 0], dtype=torch.int32).cuda(), 8, None, 32, 64)
    d, dp = torch.autograd.grad(o, (none, pk), torch.ones_like(o))
    assert o.shape == d.shape == (0, 2, 64) and not dp.any()
    for shape in ((0, 2, 9, 64), (2, 2, 0, 64)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        o = fixed(x, x, x, pk, None, None, 32, 64)
        d, dp = torch.autograd.grad(o, (x, pk), torch.ones_like(o))
        assert o.shape == d.shape == shape and not dp.any()
    x = torch.randn(3, 2, 9, 64, device="cuda", requires_grad=True)
    o = fixed(x, x, x, pk, None, None, 32, 64, seqlens_k=torch.zeros(3, dtype=torch.int32, device="cuda"))
    d, dp = torch.autograd.grad(o, (x, pk), torch.ones_like(o))
    assert not o.any() and not d.any() and not dp.any()


def test_everything_dropped():
    c = Case([70], p=1.0, seed=19)
    got = c.packed()
    assert not any(t.any() for t in got.values())


def test_refusals():
    x, t, cu, seed = torch.randn(2, 2, 9, 64, device="cuda"), torch.randn(2, 64, 64, device="cuda"), torch.tensor([0, 9], dtype=torch.int32).cuda(), _seed(1)
    y = x[0].transpose(0, 1)
    for bad in (lambda: fixed(x[0], x[0], x[0]), lambda: fixed(x, x[:1], x), lambda: fixed(x, x, x.half()), lambda: fixed(x.double(), x.double(), x.double()),
                lambda: fixed(x[..., :12], x[..., :12], x[..., :12]), lambda: fixed(*[torch.randn(1, 1, 4, 72, device="cuda")] * 3), lambda: fixed(x, x, x, sm_scale=0.0),
                lambda: fixed(x, x, x, sm_scale=-1.0), lambda: fixed(x, x, x, sm_scale=float("nan")), lambda: fixed(x, x, x, t), lambda: fixed(x, x, x, t.half(), None, None, 32, 64),
                lambda: fixed(x, x, x, t[:1], None, None, 32, 64), lambda: fixed(x, x, x, t[:, :63], None, None, 32, 64), lambda: fixed(x, x, x, dropout_p=0.1),
                lambda: fixed(x, x, x, dropout_p=2.0, seed=seed), lambda: fixed(x, x, x, seqlens_k=cu[:1]), lambda: fixed(x, x, x, seqlens_k=cu.cpu()),
                lambda: varlen(x, x, x, None, None, cu, 9), lambda: varlen(y, y, y, None, None, cu[None], 9), lambda: varlen(y, y, y, None, None, cu[:0], 9),
                lambda: varlen(y, y, y, None, None, cu, (1 << 20) + 1)):
        with pytest.raises(ValueError):
            bad()
