"""layer_norm of rows whose mean is large beside their spread: the mean is taken out to the
precision of the spread, not of the mean.  The bounds hold no term of a unit of the mean
times a sum's length."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = ref.U


def closely(x, w, b, eps, dy):
    """{name: (value, bound)}.  The first mean is off by e0 (a sum of the row); the second, of what is left after
    taking it out, by a sum of those; the one that the backward pass reads is rounded to fp32 besides."""
    dt = x.dtype
    exact = {k: v[0] for k, v in ref.norm(x, w, b, eps, dy).items()}
    x, w, b, dy = (ref.f64(t) for t in (x, w, b, dy))
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    h = c * rstd
    adds = 64 + 24                      # as in ref.norm
    e0 = adds * U * x.abs().mean(1, keepdim=True) + U * mean.abs()
    spread = (c.abs() + e0).mean(1, keepdim=True)
    dmean = (adds + 3) * U * spread     # of the sum of x - first mean, each of which has one rounding
    # the variance: its sum, the squares of what the first mean left in, and the second mean's error squared
    drel = 0.5 * (adds + 8) * U * (1 + (e0 * rstd) ** 2) + 0.5 * (dmean * rstd) ** 2 + 6 * U
    dh = dmean * rstd + h.abs() * drel + 3 * U * (h.abs() + e0 * rstd)
    out = {"y": w.abs() * dh + 3 * U * ((h * w).abs() + b.abs())}
    dh = dh + U * (mean.abs() + dmean) * rstd
    g = dy * w
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dmg = (adds + 2) * U * g.abs().mean(1, keepdim=True)
    dmgh = (adds + 3) * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * dh).mean(1, keepdim=True)
    parts = g.abs() + mg.abs() + (h * mgh).abs()
    out["dx"] = rstd * (dmg + h.abs() * dmgh + dh * mgh.abs() + 6 * U * parts) + drel * rstd * parts
    rows = x.shape[0] + 16
    out["dw"] = rows * U * (dy * h).abs().sum(0) + (dy.abs() * dh).sum(0)
    return {k: (exact[k], v + 1.01 * ref.unit(dt) * exact[k].abs() + ref.tiny(dt)) for k, v in out.items()}


# (every size of group; four or eight elements a thread)
@pytest.mark.parametrize("d", [100, 129, 300, 520, 1100, 4100, 9000, 20001])
@pytest.mark.parametrize("offset", [1000.0, 30000.0])
def test_mean_beside_spread(hip, offset, d):
    g = torch.Generator().manual_seed(d)
    x = torch.randn((12, d), generator=g) + offset * (1 + torch.rand((12, 1), generator=g))
    w, b, dy = 1 + 0.2 * torch.randn(d, generator=g), 0.2 * torch.randn(d, generator=g), torch.randn((12, d), generator=g)
    x, w, b, dy = (t.to(DEV) for t in (x, w, b, dy))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = gmmxx_amd.layer_norm(*leaves)
    dx, dw, _ = torch.autograd.grad(y, leaves, dy)
    want = closely(x, w, b, 1e-5, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        ref.close(got, *want[name], name)


def test_rows_of_one_value(hip):
    """What a mean's rounding leaves of a constant row is taken out too."""
    x = torch.full((5, 1000), 0.1, device=DEV) * torch.arange(1, 6, device=DEV)[:, None]
    y = gmmxx_amd.layer_norm(x, eps=1e-12)
    # each x differs from the first mean alike: the second leaves its own sum's rounding, a part of that difference
    first = 89 * U * x.double().abs().amax(1, keepdim=True)
    assert (y.double().abs() <= 92 * U * first / 1e-6).all()
