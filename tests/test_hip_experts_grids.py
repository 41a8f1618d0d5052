"""Calls within the documented sizes whose workgroups or threads pass what one dimension of
a grid counts: many rows, many experts of wide matrices.  Operands are small whole numbers
where results are sums of products, so those are exact in any order."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def whole(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g, device=DEV).bfloat16()


def ends(e, m, seed=0):
    """Offsets of e groups of m positions, many empty."""
    cuts = torch.randint(0, m + 1, (e - 1,), generator=torch.Generator().manual_seed(seed)).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.full((1,), m)]).to(torch.int32).to(DEV)


def test_gradient_of_many_rows(hip):
    """2^29 rows and some, gates over both candidates: d gate = gate (1 - gate) where the row's best is, and minus
    that elsewhere."""
    n, part = (1 << 29) + 37, 1 << 26
    print(f"[grids] route n={n}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(0)
    scores = torch.empty((n, 2), dtype=torch.float16, device=DEV).normal_(generator=g).requires_grad_()
    dgates = torch.empty((n, 1), device=DEV).normal_(generator=g)
    r = gmmxx_amd.route_rows(scores, 1, renormalize=False)
    ds, = torch.autograd.grad(r.gates, scores, dgates)
    for i in range(0, n, part):
        s, d = scores.detach()[i:i + part].double(), dgates[i:i + part].double()
        p = torch.softmax(s, 1)
        best = (s[:, 1:] > s[:, :1])
        slope = (p[:, :1] * p[:, 1:]) * d
        want = torch.where(best, torch.cat([-slope, slope], 1), torch.cat([slope, -slope], 1))
        # exponentials, sum, products and differences of fp32 values up to |d|, then one rounding
        bound = 32 * ref.U * d.abs() + ref.unit(torch.float16) * want.abs() * 1.01 + ref.tiny(torch.float16)
        assert ((ds[i:i + part].double() - want).abs() <= bound).all(), i
        assert torch.equal(r.experts[i:i + part, 0].long(), best[:, 0].long())


@pytest.mark.parametrize("adjacent", ["columns", "reduction"])
def test_tiles_of_many_experts(hip, adjacent):
    e, m, d, f = 4096, 40, 8, 4096 * 128 + 8
    print(f"[grids] rows e={e} f={f}", flush=True)
    x, w = whole(m, d), whole(1, d, f, seed=1)
    if adjacent == "reduction":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    y = gmmxx_amd.grouped_matmul(x, w.expand(e, d, f), ends(e, m))
    assert torch.equal(y, (x.float() @ w[0].float()).bfloat16())


@pytest.mark.parametrize("adjacent", ["columns", "reduction"])
def test_few_rows_of_many_experts(hip, adjacent):
    e, m, d, f = 4096, 8192, 7, 1366 * 64 + 3
    print(f"[grids] few e={e} f={f}", flush=True)
    x, w = whole(m, d), whole(1, d, f, seed=1)
    if adjacent == "reduction":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    off = ends(e, m - 5)             # the last positions: zeros
    y = gmmxx_amd.grouped_matmul(x, w.expand(e, d, f), off)
    assert torch.equal(y[:m - 5], (x[:m - 5].float() @ w[0].float()).bfloat16())
    assert not y[m - 5:].any()


def test_weight_gradient_of_many_experts(hip):
    e, m, f = 4096, 24, 4096 * 128 + 8
    print(f"[grids] dw e={e} f={f}", flush=True)
    x, dy, off = whole(m, 1), whole(m, f, seed=1), ends(e, m)
    w = torch.zeros((e, 1, f), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    dw, = torch.autograd.grad(gmmxx_amd.grouped_matmul(x, w, off), w, dy)
    group = torch.searchsorted(off[1:].contiguous(), torch.arange(m, device=DEV, dtype=torch.int32), right=True)
    used = group.unique()
    for i in used.tolist():
        at = group == i
        assert torch.equal(dw[i, 0], (x[at].float() * dy[at].float()).sum(0).bfloat16()), i
    dw[used] = 0
    assert not dw.any()
