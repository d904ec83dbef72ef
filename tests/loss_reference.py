"""The loss over a vocabulary in 64 bits, from its formulas, with what the operator may be off by."""
import torch

U = 2.0 ** -24      # half a step of float32, relative


def loss(x, weight, labels, bias, ignore, reduction, dloss, dtype):
    """{name: (value, bound)} of loss, dx, dweight, dbias; inputs as the operator has them, [rows, hidden] and so on, dloss: the loss's gradient (None: 1).

    Bounds, u half a step of `dtype`, U of float32.  A logit is a sum of `hidden` products and the bias, however it is taken: off by E = (hidden + 3) U of its terms' sizes,
    and by two roundings of its own size where it goes to base 2 and back.  Largest logits are exact differences' ends, so an exponential is off by as much, relative, and by its
    own 4 U; a sum of exponentials by that and (vocab + 8) U if it were taken one after another.  rho: all of this, relative, of a probability.  D = g (p - [label]) has p's error, its
    own rounding to float32 and to the type (float16: or half the smallest step, 2^-25, of 2^14 max|g| / max|g| at most 2: a row's own power of two is 2^14 |g| or more).
    A product's sum is off by as many U of its terms' sizes as it has terms; a row of x is divided by a power of two in float16, exactly but for values below the smallest
    normal one (2^-25 relative to the largest |g|, a power of two: at most 2 max|g|).  Check adds the rounding of the result."""
    x, weight = x.double(), weight.double()
    counts = labels != ignore
    n = int(counts.sum())
    bias_ = torch.zeros(len(weight), dtype=torch.float64, device=x.device) if bias is None else bias.double()
    x = torch.where(counts[:, None], x, 0.0)
    hidden, vocab = x.shape[1], len(weight)
    half = dtype == torch.float16
    u = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    s = x @ weight.t() + bias_
    size = x.abs() @ weight.abs().t() + bias_.abs()
    finite = size.isfinite()
    E = torch.where(finite, (hidden + 3) * U * size + 3 * U * s.abs(), 0.0).amax(-1, keepdim=True)
    top = torch.where(finite, s.abs(), 0.0).amax(-1, keepdim=True)
    at = labels.clamp(0, vocab - 1)[:, None]
    good = (labels >= 0) & (labels < vocab)
    lse = torch.logsumexp(s, -1, keepdim=True)
    rows = torch.where(counts, torch.where(good, (lse - s.gather(-1, at)).squeeze(-1), torch.nan), 0.0)
    rows_off = ((2 * E + 8 * U * (lse.abs() + top + 1) + (vocab + 8) * U).squeeze(-1)) * counts
    g0 = torch.ones(rows.shape if reduction == "none" else (), device=x.device) if dloss is None else dloss
    if reduction == "none":
        got = {"loss": (rows, rows_off)}
        g = g0.double() * counts
    else:
        by = n if reduction == "mean" else 1
        got = {"loss": (rows.sum() / by if by else rows.sum() * torch.nan, rows_off.sum() / max(by, 1) + 2 * U * rows.abs().sum() / max(by, 1))}
        g = (g0.double() / max(by, 1)).expand(rows.shape) * counts
    p = torch.exp(s - lse)
    one = torch.zeros_like(p).scatter_(-1, at, 1.0)
    D = torch.where(counts[:, None], g[:, None] * (p - one), 0.0)
    D = torch.where((counts & ~good)[:, None], torch.nan, D)
    G = g.abs()[:, None]
    rho = 2 * E + (vocab + 30) * U
    D_off = G * (p * rho + 4 * U * (p + one))
    stored = D_off + u * (D.abs() + D_off) + (2 * 2.0 ** -25 * 2.0 ** -14 * G if half else 0.0)
    W, X = weight.abs(), x.abs()
    rounding = lambda terms, m: (terms + 8) * U * m
    got["dx"] = (D @ weight, stored @ W + rounding(vocab, D.abs() @ W))
    lost = 2.0 ** -24 * g.abs().max() if half and len(g) else 0.0         # of each value of x, relative to its row's g
    got["dweight"] = (D.t() @ x, stored.t() @ X + rounding(max(n, 1), D.abs().t() @ X) + (lost * (D.abs() / G.clamp(min=1e-300)).sum(0)[:, None] if half else 0.0))
    got["dbias"] = (D.sum(0), D_off.sum(0) + rounding(max(n, 1), D.abs().sum(0)))
    return got


def check(name, got, ref, off):
    """Half a step of the result's type, and what the arithmetic may be off by (with a subnormal result's step).  NaN and infinities where the reference has them."""
    info = torch.finfo(got.dtype)
    ref, off = ref.to(got.device), off.to(got.device)
    assert got.shape == ref.shape, f"{name}: {tuple(got.shape)}, {tuple(ref.shape)}"
    bound = ref.abs() * info.eps / 2 + off * (1 + info.eps) + info.smallest_normal * info.eps
    far = (got.detach().double() - ref).abs()
    bad = ~(far <= bound) & ~(got.isnan() & ref.isnan()) & ~(got.isinf() & (got.double() == ref))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values, by up to {(far / bound)[bad].max().item():.3g} of the bound"
