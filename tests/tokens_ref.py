"""Plain 64-bit forms (torch and numpy on the CPU) of the token operators, and the error each
result may have.  U is fp32's unit (2^-24); see experts_ref for `unit`, `tiny` and `close`."""

import math

import numpy as np
import torch

from tests.experts_ref import U, f64, tiny, unit


def rounded(dt, v):
    """What rounding v to dt may cost."""
    return unit(dt) * v.abs() * 1.01 + tiny(dt)


# --- embedding --------------------------------------------------------------------

def embed(table, index, scale, dy=None):
    """{name: (value, bound)} of out and, given dy, dtable."""
    dt = table.dtype
    t, i = f64(table), index.cpu().long().reshape(-1)
    v, d = t.shape
    there = (i >= 0) & (i < v)
    at = torch.where(there, i, 0)
    y = torch.where(there[:, None], t[at] * scale, torch.zeros(()).double())
    # the scale's rounding to fp32 and the product's
    out = {"out": (y.reshape(*index.shape, d), (2 * U * y.abs() + rounded(dt, y)).reshape(*index.shape, d))}
    if dy is not None:
        g = f64(dy).reshape(-1, d)[there]
        total = torch.zeros((v, d), dtype=torch.float64).index_add_(0, at[there], g)
        size = torch.zeros((v, d), dtype=torch.float64).index_add_(0, at[there], g.abs())
        count = torch.bincount(at[there], minlength=v)[:, None].double()
        # no chain of additions is longer than the token's places and a level of partial sums above them
        bound = (count + 8) * U * size * abs(scale) + 2 * U * (total * scale).abs()
        out["dtable"] = (total * scale, torch.where(count > 0, bound + rounded(dt, total * scale), 0.0))
    return out


# --- dropout ------------------------------------------------------------------------

def words(count, seed, offset=0, rounds=10):
    """The first words of Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, 2011), by Python's own integers where the
    constants are concerned and numpy's 64-bit ones for the products."""
    low = np.uint64(0xFFFFFFFF)
    i = np.arange(-(-count // 4), dtype=np.uint64)
    c = [i & low, i >> np.uint64(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    return _philox(c, [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF], rounds)[:count]


def _philox(c, key, rounds=10):
    low = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]),
             a & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)


def dropout(x, p, seed, offset=0, residual=None):
    """(value, bound, kept)"""
    border = round(p * 2.0 ** 32)
    keep = torch.from_numpy((words(x.numel(), seed, offset) >= np.uint64(border)).reshape(tuple(x.shape)))
    v = torch.where(keep, f64(x) / (1.0 - p) if p < 1.0 else 0.0, 0.0)
    y = v if residual is None else v + f64(residual)
    # the factor's rounding and the product's; the sum's
    return y, 2 * U * v.abs() + U * y.abs() + rounded(x.dtype, y), keep


# --- log probabilities -----------------------------------------------------------------

def log_probs(scores, index, k=0, dchosen=None, dentropy=None, dtop=None):
    """{name: (value, bound)} of chosen, entropy, top, top_index (whole numbers, bound None) and, given gradients,
    dscores.

    The error of one e^d: d is rounded (relative error |d| U), d log2(e) is rounded and its factor is (|d| U each),
    the exponential is good to 2 U; and a sum is brought to a larger maximum at most once a vector, whose
    exponents add up to at most |d|: another 3 |d| U, and 4 U for each of them.  The reference may lie below the largest
    score by up to 7: 6 |d| is 42 more.  `adds` bounds a thread's vectors (which also are the additions of its
    chain, but for 8 in a vector, 10 levels and 64 parts above them)."""
    dt = scores.dtype
    s, t = f64(scores), index.cpu().long()
    n, v = s.shape
    there = s > -math.inf
    x = torch.where(there, s, -math.inf)
    m = x.max(1, keepdim=True).values
    some = m > -math.inf
    d = torch.where(x == m, torch.zeros(()).double(), x - m)
    d = torch.where(there, d, -math.inf)
    w = torch.where(there, torch.exp(d), 0.0)
    z = torch.where(some, w.sum(1, keepdim=True), 1.0)
    logz = torch.log(z)
    p = w / z
    size = torch.where(p > 0, d.abs(), 0.0)
    mean, square = (p * size).sum(1, keepdim=True), (p * size * size).sum(1, keepdim=True)
    entropy = torch.where(some, logz + mean, 0.0)
    adds = -(-v // 512) + 90.0
    dz = U * (6 * mean + 42 + 5 * adds + 8)                   # relative error of Z, so absolute of log Z
    dlogz = dz + 4 * U * logz.abs()
    dh = dlogz + U * (6 * square + (42 + 5 * adds + 8) * (mean + 7)) + (mean + 7) * dz + 4 * U * entropy.abs()
    counts = (t >= 0) & (t < v)
    at = torch.where(counts, t, 0)[:, None]

    def log_p(c):
        dc = d.gather(1, c)
        lp = dc - logz
        b = U * (dc.abs() + lp.abs() + logz.abs()) + dlogz
        return lp, torch.where(torch.isfinite(lp), b, 0.0)

    chosen, dchosen_err = log_p(at)
    out = {"chosen": (torch.where(counts, chosen[:, 0], 0.0), torch.where(counts, dchosen_err[:, 0], 0.0)),
           "entropy": (entropy[:, 0], torch.where(some, dh, 0.0)[:, 0])}
    place = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    real = there.gather(1, place)
    top, dtop_err = log_p(place) if k else (torch.zeros((n, 0)).double(),) * 2
    out["top"] = (torch.where(real, top, -math.inf), dtop_err)
    out["top_index"] = (torch.where(real, place, -1), None)
    if dchosen is None and dentropy is None and dtop is None:
        return out
    zero = torch.zeros(n, dtype=torch.float64)
    gc = torch.where(counts, f64(dchosen) if dchosen is not None else zero, zero)[:, None]
    gh = (f64(dentropy) if dentropy is not None else zero)[:, None]
    gt = torch.where(real, f64(dtop), 0.0) if dtop is not None else torch.zeros((n, k)).double()
    c = -gc - gt.sum(1, keepdim=True)
    csize = gc.abs() + gt.abs().sum(1, keepdim=True)
    lp = torch.where(p > 0, d - logz, 0.0)
    far = lp + entropy
    ds = p * (c - gh * far)
    dlp = U * (torch.where(p > 0, d.abs(), 0.0) + lp.abs()) + dlogz
    dp = p * (dlp + 3 * U * lp.abs() + 4 * U)
    err = csize * (dp + (k + 3) * U * p) + gh.abs() * (dp * far.abs() + p * (dlp + dh + 2 * U * far.abs()))
    err = err + 4 * U * p * (csize + (gh * far).abs())
    # (p below 2^-126 comes out as 0: what it is multiplied by is no more than this)
    err = err + 2.0 ** -126 * (csize + gh.abs() * (far.abs() + 110))
    extra = torch.zeros_like(ds).scatter_add_(1, at, torch.where(there.gather(1, at), gc, 0.0))
    extra_size = extra.abs()
    if k:
        extra = extra.scatter_add(1, place, gt)
        extra_size = extra_size.scatter_add(1, place, gt.abs())
    err = err + 3 * U * (extra_size + ds.abs() * (extra_size > 0))
    ds = torch.where(some, ds + extra, 0.0)
    out["dscores"] = (ds, torch.where(there, err + rounded(dt, ds), 0.0))
    return out


# --- 8-bit integers ----------------------------------------------------------------------

def quantize(x):
    """(values, scales) by fp32 arithmetic, as they are defined (numpy's, which rounds each operation)."""
    x = x.detach().float().cpu().numpy()
    finite = np.isfinite(x).all(1)
    x = np.where(finite[:, None], x, np.float32(0))
    most = np.abs(x).max(1)
    lift = np.where(most < np.float32(2.0 ** -100), np.float32(2.0 ** 100), np.float32(1))
    with np.errstate(divide="ignore"):
        by = np.where(most > 0, np.float32(1) / (most * lift) * np.float32(127), np.float32(0))
    q = np.rint((x * lift[:, None]) * by[:, None])
    scales = np.where(finite, most * (np.float32(1) / np.float32(127)), np.float32(math.nan))
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(scales.astype(np.float32))


def quantized_matmul(qx, sx, qw, sw, bias, dt):
    """(value, bound): the sum is exact; its conversion to fp32, the scales' product and the product with it round once
    each, and so does the sum with the bias."""
    total = (qx.cpu().long().double() @ qw.cpu().long().double().t())
    y = total * f64(sx)[:, None] * f64(sw)
    out = y if bias is None else y + f64(bias)
    # (the scales' product may be subnormal: half of fp32's spacing there, times the sum)
    bound = 3 * U * y.abs() + U * out.abs() + 2.0 ** -150 * total.abs() + 2.0 ** -149 + rounded(dt, out)
    # half a step past the type's largest value, a result rounds to infinity
    most = torch.finfo(dt).max * (1 + unit(dt) / 2)
    return torch.where(out.abs() >= most, out.sign() * math.inf, out), bound
