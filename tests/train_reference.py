"""The training operators in 64 bits, from their formulas: what the GPU tests compare with."""
import numpy as np
import torch

U = 2.0 ** -24      # half a step of float32, relative


def philox(counter, key, rounds=7):
    """Philox-4x32 of numpy arrays (uint64 holding 32 bits): counter [4, ..], key (low, high)."""
    a, b, c, d = (np.asarray(x, dtype=np.uint64) for x in counter)
    k0, k1 = (int(k) for k in key)
    low = np.uint64(0xffffffff)
    for _ in range(rounds):
        x, y = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (y >> np.uint64(32)) ^ b ^ np.uint64(k0), y & low, (x >> np.uint64(32)) ^ d ^ np.uint64(k1), x & low
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return np.stack(np.broadcast_arrays(a, b, c, d))


def numbers(counter, seed):
    """The eight 16-bit numbers of each counter, along a last axis."""
    seed = int(seed) & (1 << 64) - 1
    w = philox(counter, (seed & 0xffffffff, seed >> 32))
    return np.stack([h for x in w for h in (x & np.uint64(0xffff), x >> np.uint64(16))], axis=-1).astype(np.int64)


def factors(u, p):
    t = round(65536 * p)
    return torch.from_numpy(np.where(u >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0, 0.0))


def keep_of(shape, p, seed):
    """What dropout multiplies the values of a tensor by (float64, on the CPU)."""
    n = int(np.prod(shape))
    chunk = np.arange((n + 7) // 8, dtype=np.uint64)
    zero = np.zeros_like(chunk)
    u = numbers((chunk & np.uint64(0xffffffff), chunk >> np.uint64(32), zero, zero), seed)
    return factors(u.reshape(-1)[:n].reshape(shape), p)


def keep_of_probabilities(length, which, p, seed):
    """The same for the probabilities [query, key] of head and sequence number `which`."""
    j, i = np.arange(length), np.arange(length)
    octet = np.arange(4 * -(-length // 32))
    u = numbers((octet[None].astype(np.uint64), i[:, None].astype(np.uint64), np.uint64(which), np.uint64(1)), seed)
    return factors(u[:, 4 * (j // 32) + j // 4 % 4, 4 * (j // 16 % 2) + j % 4], p)


def drop(x, keep):
    """Dropped values are 0 whatever they were."""
    return torch.where(keep == 0, 0.0, x * keep)


def norm(x, residual, weight, bias, dy, keep, eps):
    """(results, bounds of the error of float32 arithmetic) of LayerNorm(x keep + residual): y, dz, dw, db, all in 64 bits.

    Bounds.  A sum of n terms taken in k steps one after another is off by at most k U times the sum of its terms' sizes.  Steps here: 8 in a
    lane for each 512 columns (a column in 256 otherwise), up to 8 over the wave and waves, the mean's division and the terms' own
    roundings (dropout's product, the residual): k below.  The mean is off by k U mean|z|, the reciprocal of the standard
    deviation by k U relative and what the mean adds, xhat by k U X with X below, and the gradient's three terms by as much relative to
    each.  Rows: up to rows / 512 one after another, 64 workgroups' parts in a lane and 8 twice."""
    hidden, rows = x.shape[-1], x.reshape(-1, x.shape[-1]).shape[0]
    k = 20 + max(32, hidden // 256)
    z = drop(x, keep) + (0 if residual is None else residual)
    size = drop(x, keep).abs() + (0 if residual is None else residual.abs())
    w, b = (torch.ones(hidden), torch.zeros(hidden)) if weight is None else (weight, bias)
    w, b = w.double(), b.double()
    var, mean = torch.var_mean(z, -1, correction=0, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    hat = (z - mean) * rstd
    X = hat.abs() + rstd * (size + size.mean(-1, keepdim=True))
    got, off = {"y": hat * w + b}, {"y": 3 * k * U * (w.abs() * X + b.abs())}
    if dy is not None:
        g = dy * w
        dot = (g * hat).mean(-1, keepdim=True)
        got["dz"] = rstd * (g - g.mean(-1, keepdim=True) - hat * dot)
        off["dz"] = 4 * k * U * rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + X * (g.abs() * X).mean(-1, keepdim=True)) * (1 + (X * X).mean(-1, keepdim=True))
        flat = lambda t: t.reshape(-1, hidden)
        steps = rows // 512 + 90
        got |= {"dw": flat(dy * hat).sum(0), "db": flat(dy).sum(0)}
        off |= {"dw": (steps + 4 * k) * U * flat(dy.abs() * X).sum(0), "db": steps * U * flat(dy.abs()).sum(0)}
    return got, off


def check(name, got, ref, off):
    """Half a step of the result's type, and what float32 arithmetic may be off by (with a subnormal result's step)."""
    info = torch.finfo(got.dtype)
    bound = ref.abs() * info.eps / 2 + off * (1 + info.eps) + info.smallest_normal * info.eps
    far = (got.detach().cpu().double() - ref).abs()
    bad = ~(far <= bound)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values, by up to {(far / bound).max().item():.3g} of the bound"


def attention(q, k, v, pk, pq, dout, rows, scale, keep, factor, dtype, most):
    """One sequence and head in 64 bits: {name: (value, bound)} of o, dq, dk, dv and, where there are tables, dpk, dpq.  q, k, v, dout [l, D]; rows: table row of
    (query, key); keep: what the probabilities are multiplied by (factor or 0); most: the largest |dout| |v| of the whole call (float16).

    Bounds, u half a step of the type, U of float32.  A score is a sum of 64 products for each of three terms: off by 70 U of its terms' sizes A.  A probability is
    off by that, by its exponent's rounding and by its sum's, relative: rho = 100 U (1 + A + max A).  Rounded to the type where it enters a product: u, or in float16, for
    small ones, half the smallest step: 2^-25 of a row's largest forward, 2^-25 / 2^floor(log2 l) backward.  D comes from the rounded result.  A gradient of a score is off by what
    its factors are, and rounded to the type (float16: or half the smallest step after a scaling that brings 2 most factor below 2^15, to 2^14 at least).  The
    sums that follow have `steps` terms one after another."""
    u, half = torch.finfo(dtype).eps / 2, dtype == torch.float16
    if dtype == torch.float32:
        u = 0.0
    l = q.shape[0]
    steps = 100 + l / 8
    K, Q = (k[None] + pk[rows] if pk is not None else k[None].expand(l, -1, -1)), (q[:, None] + pq[rows] if pq is not None else q[:, None].expand(-1, l, -1))
    size = lambda *t: sum(x.abs() for x in t if x is not None)
    sizeK, sizeQ = size(k[None], None if pk is None else pk[rows]), size(q[:, None], None if pq is None else pq[rows])
    s, A = q @ k.t(), q.abs() @ k.abs().t()
    if pk is not None:
        s, A = s + torch.einsum("id,ijd->ij", q, pk[rows]), A + torch.einsum("id,ijd->ij", q.abs(), pk[rows].abs())
    if pq is not None:
        s, A = s + torch.einsum("jd,ijd->ij", k, pq[rows]), A + torch.einsum("jd,ijd->ij", k.abs(), pq[rows].abs())
    p, A = torch.softmax(s * scale, -1), A * scale
    rho = 100 * U * (1 + A + A.amax(-1, keepdim=True))
    kept = p * keep
    o = kept @ v
    low = p.amax(-1, keepdim=True) * 2.0 ** -25 * (keep != 0) * factor if half else 0
    o_off = ((u + rho + steps * U) * kept + low) @ v.abs()
    dv = kept.t() @ dout
    low = 2.0 ** -25 / 2 ** int(np.log2(l)) * factor if half else 0
    dv_off = ((u + rho + steps * U) * kept + low).t() @ dout.abs()
    dp = dout @ v.t() * keep
    D = (p * dp).sum(-1, keepdim=True)
    D_off = (dout.abs() * (u * o.abs() + o_off + 70 * U * o.abs())).sum(-1, keepdim=True)
    ds = p * (dp - D) * (l > 1)
    ds_off = (rho + u) * ds.abs() + p * (72 * U * (dout.abs() @ v.abs().t()) * keep + D_off + 4 * U * (dp.abs() + D.abs())) * (1 + u)
    if half:
        ds_off = ds_off + 2.0 ** -25 / 2 ** 14 * 2 * 2 * most * factor
    ds_off = ds_off * (l > 1) + steps * U * ds.abs()
    got = {"o": (o, o_off), "dv": (dv, dv_off),
           "dq": tuple(scale * torch.einsum("ij,ijd->id", x, y) for x, y in ((ds, K), (ds_off, sizeK))),
           "dk": tuple(scale * torch.einsum("ij,ijd->jd", x, y) for x, y in ((ds, Q), (ds_off, sizeQ)))}
    for name, table, rows_of in (("dpk", pk, q[:, None].expand(l, l, -1)), ("dpq", pq, k[None].expand(l, l, -1))):
        if table is not None:
            got[name] = tuple(scale * torch.zeros_like(table).index_add_(0, rows.flatten(), (x[..., None] * y).flatten(0, 1))
                              for x, y in ((ds, rows_of), (ds_off, rows_of.abs())))
    return got
