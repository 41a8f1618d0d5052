"""Plain 64-bit forms (numpy-style torch on the CPU) of the sparsely gated layer's
operators, and the error each result may have.

Rounding: U is fp32's unit (2^-24), `unit(dtype)` that of the stored type.  A sum
formed in fp32 differs from the exact one by at most `adds` U times the sum of its
terms' absolute values, `adds` being the longest chain of additions.
"""

import math

import torch

U = 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    # the spacing of the type's subnormals: what rounding there may cost
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def f64(t):
    return t.detach().double().cpu()


def close(got, want, bound, what):
    """got (any dtype, GPU) against want within bound (both 64-bit CPU); equal where not finite."""
    got = f64(got)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} and not {tuple(want.shape)}"
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: other values are finite"
    off = torch.where(fine, (got - want).abs() - bound, torch.zeros_like(want))
    bad = off > 0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by up to {float(off.max())} over the bound"


# --- layer norm -------------------------------------------------------------------

def norm(x, w, b, eps, dy=None):
    """{name: (value, bound)} of y and, given dy, dx, dw, db."""
    dt, n, d = x.dtype, x.shape[0], x.shape[1]
    pt = dt if w is None and b is None else (w if w is not None else b).dtype
    x = f64(x)
    w = torch.ones(d, dtype=torch.float64) if w is None else f64(w)
    b = torch.zeros(d, dtype=torch.float64) if b is None else f64(b)
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    h = c * rstd
    y = h * w + b
    # a thread adds at most 64 elements, a row's sum at most 1024 threads (10 levels, or 6 and 16 in turn)
    adds = 64 + 24
    dmean = adds * U * x.abs().mean(1, keepdim=True) + U * mean.abs()
    # the variance: its own sum, the rounding of (x - mean), and the shifted mean (which enters squared)
    drel = 0.5 * ((adds + 4) * U + (dmean * rstd) ** 2) + 4 * U
    dh = dmean * rstd + h.abs() * drel + 2 * U * h.abs()
    out = {"y": (y, w.abs() * dh + 3 * U * ((h * w).abs() + b.abs()) + unit(dt) * y.abs() * 1.01 + tiny(dt))}
    if dy is not None:
        dy = f64(dy)
        g = dy * w
        mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
        dx = rstd * (g - mg - h * mgh)
        dmg = (adds + 2) * U * g.abs().mean(1, keepdim=True)
        dmgh = (adds + 3) * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * dh).mean(1, keepdim=True)
        parts = g.abs() + mg.abs() + (h * mgh).abs()
        ddx = rstd * (dmg + h.abs() * dmgh + dh * mgh.abs() + 6 * U * parts) + drel * rstd * parts
        out["dx"] = (dx, ddx + unit(dt) * dx.abs() * 1.01 + tiny(dt))
        rows = n + 16      # no chain is longer than the rows and the levels above them
        out["dw"] = ((dy * h).sum(0), rows * U * (dy * h).abs().sum(0) + (dy.abs() * dh).sum(0)
                     + unit(pt) * (dy * h).sum(0).abs() * 1.01 + tiny(pt))
        out["db"] = (dy.sum(0), rows * U * dy.abs().sum(0) + unit(pt) * dy.sum(0).abs() * 1.01 + tiny(pt))
    return out


# --- routing ------------------------------------------------------------------------

def route(scores, k, renormalize):
    """(experts, gates, offsets, rows, slots) by loops over the rows, gates in 64 bits."""
    s = f64(scores)
    n, e = s.shape
    experts = torch.full((n, k), -1, dtype=torch.int64)
    gates = torch.zeros((n, k), dtype=torch.float64)
    for r in range(n):
        row = s[r].tolist()
        there = [i for i in range(e) if row[i] == row[i] and row[i] > -math.inf]
        best = sorted(there, key=lambda i: (-row[i], i))[:k]
        if not best:
            continue
        top = row[best[0]]
        weigh = lambda i: 1.0 if row[i] == top else math.exp(row[i] - top) if top < math.inf else 0.0   # noqa: E731
        whole = sum(weigh(i) for i in (best if renormalize else there))
        for j, i in enumerate(best):
            experts[r, j] = i
            gates[r, j] = weigh(i) / whole
    flat = torch.where(experts < 0, e, experts).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    offsets = torch.tensor([int((flat < i).sum()) for i in range(e + 1)])
    slots = torch.empty_like(order)
    slots[order] = torch.arange(n * k)
    return experts, gates, offsets, order // k, slots.reshape(n, k)


def route_grad(scores, k, renormalize, dgates):
    experts, gates, *_ = route(scores, k, renormalize)
    s, dg = f64(scores), f64(dgates)
    ds = torch.zeros_like(s)
    for r in range(s.shape[0]):
        there = experts[r] >= 0
        if not there.any():
            continue
        mean = float((gates[r] * dg[r])[there].sum())
        if not renormalize:
            row = torch.where(s[r] == s[r], s[r], -math.inf)
            top = float(row.max())
            p = torch.where(row == top, 1.0, torch.exp(row - top) if top < math.inf else 0.0)
            ds[r] = -mean * p / p.sum()
        for j in range(k):
            if there[j]:
                ds[r, experts[r, j]] += gates[r, j] * (dg[r, j] - (mean if renormalize else 0.0))
    return ds


# --- grouped products -----------------------------------------------------------------

def grouped(x, w, b, offsets, rows, slots=None, dy=None):
    """{name: (value, bound)} of out and, given dy, dx, dw, db."""
    dt = x.dtype
    x, w = f64(x), f64(w)
    b = torch.zeros(w.shape[0], w.shape[2], dtype=torch.float64) if b is None else f64(b)
    ends = [int(v) for v in offsets]
    m = x.shape[0] if rows is None else rows.numel()
    src = torch.arange(m) if rows is None else rows.cpu().long()
    e, d, f = w.shape
    y, my = torch.zeros(m, f, dtype=torch.float64), torch.zeros(m, f, dtype=torch.float64)
    dp, mdp = torch.zeros(m, d, dtype=torch.float64), torch.zeros(m, d, dtype=torch.float64)
    dw, mdw, ddw = (torch.zeros_like(w) for _ in range(3))
    db, mdb = torch.zeros_like(b), torch.zeros_like(b)
    g = None if dy is None else f64(dy)
    for i in range(e):
        at = slice(ends[i], ends[i + 1])
        xe = x[src[at]]
        y[at] = xe @ w[i] + b[i]
        my[at] = xe.abs() @ w[i].abs() + b[i].abs()
        if g is not None:
            ge = g[at]
            dp[at] = ge @ w[i].t()
            mdp[at] = ge.abs() @ w[i].t().abs()
            dw[i], mdw[i] = xe.t() @ ge, xe.t().abs() @ ge.abs()
            ddw[i] = (xe.shape[0] + 16) * U * mdw[i]
            db[i], mdb[i] = ge.sum(0), (ge.shape[0] + 16) * U * ge.abs().sum(0)
    rnd = lambda v: unit(dt) * v.abs() * 1.01 + tiny(dt)   # noqa: E731
    out = {"out": (y, (d + 2) * U * my + rnd(y))}
    if g is not None:
        if rows is None:
            out["dx"] = (dp, (f + 2) * U * mdp + rnd(dp))
        else:
            picked, size = dp[slots.cpu().long()], mdp[slots.cpu().long()]
            dx = picked.sum(1)
            out["dx"] = (dx, (f + 2 + slots.shape[1]) * U * size.sum(1) + rnd(dx))
        out["dw"] = (dw, ddw + rnd(dw))
        out["db"] = (db, mdb + rnd(db))
    return out


# --- combination -------------------------------------------------------------------------

def combine(y, gates, slots, taken, dout=None):
    """{name: (value, bound)}; positions from `taken` on add nothing."""
    dt = y.dtype
    y, g, s = f64(y), f64(gates), slots.cpu().long()
    k = s.shape[1]
    there = (s < taken)
    picked = torch.where(there[:, :, None], y[s], torch.zeros(()).double())
    g = torch.where(there, g, torch.zeros(()).double())
    out = (picked * g[:, :, None]).sum(1)
    size = (picked * g[:, :, None]).abs().sum(1)
    rnd = lambda v: unit(dt) * v.abs() * 1.01 + tiny(dt)   # noqa: E731
    res = {"out": (out, (k + 1) * U * size + rnd(out))}
    if dout is not None:
        d = f64(dout)
        dy = torch.zeros_like(y)
        dy[s.reshape(-1)] = torch.where(there[:, :, None], g[:, :, None] * d[:, None, :],
                                        torch.zeros(()).double()).reshape(y.shape)
        dots = (picked * d[:, None, :])
        res["dy"] = (dy, U * dy.abs() + rnd(dy))
        res["dgates"] = (dots.sum(2), (y.shape[1] + 8) * U * dots.abs().sum(2))
    return res
