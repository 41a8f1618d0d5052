"""route_rows against a row-by-row form in 64 bits: ties, masks that leave a row little
or nothing, the type's lowest value, infinities and NaN, odd expert counts, many blocks,
and the gates' gradient."""

import math

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(n, e, dtype, seed=0, levels=None):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn((n, e), generator=g)
    if levels:      # few different values: ties everywhere
        s = torch.round(s * levels) / levels
    return s.to(dtype)


def check(scores, k, renormalize, dgates=None):
    s = scores.to(DEV)
    want = ref.route(scores, k, renormalize)
    got = gmmxx_amd.route_rows(s, k, renormalize=renormalize)
    assert got.gates.dtype == torch.float32
    for name, w in zip(gmmxx_amd.Routing._fields, want):
        g = getattr(got, name)
        if name == "gates":
            # exp to 4 units, a sum of E terms, a division
            ref.close(g, w, (scores.shape[1] + 16) * ref.U * w + 1e-37, "gates")
        else:
            assert g.dtype == torch.int32
            assert torch.equal(g.cpu().long(), w), name
    if dgates is None:
        g = torch.Generator().manual_seed(5)
        dgates = torch.randn((scores.shape[0], k), generator=g)
    leaf = s.detach().requires_grad_()
    r = gmmxx_amd.route_rows(leaf, k, renormalize=renormalize)
    assert torch.equal(r.gates.detach(), got.gates) and torch.equal(r.slots, got.slots)
    ds, = torch.autograd.grad(r.gates, leaf, dgates.to(DEV))
    assert ds.dtype == scores.dtype
    wd = ref.route_grad(scores, k, renormalize, dgates)
    # every term g dg and p Σ g dg to (E + k + 24) units of the row's Σ |g dg| + max |dg|
    size = dgates.double().abs().amax(1, keepdim=True) * 2
    ref.close(ds, wd, (scores.shape[1] + k + 24) * ref.U * size + ref.unit(scores.dtype) * wd.abs() * 1.01
              + ref.tiny(scores.dtype), "dscores")


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("e,k", [(1, 1), (2, 1), (3, 3), (8, 2), (9, 4), (16, 16), (63, 5), (64, 8), (65, 2), (100, 64),
                                 (255, 3), (256, 1), (257, 7), (500, 4), (512, 2), (513, 2), (1000, 8), (1024, 2),
                                 (1025, 3), (4096, 2)])
def test_experts(hip, e, k, dtype, renormalize):
    print(f"[route] e={e} k={k} {dtype} renormalize={renormalize}", flush=True)
    check(make(37, e, dtype, seed=e), k, renormalize)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 129, 1000, 2049])
@pytest.mark.parametrize("e,k", [(7, 2), (64, 3), (300, 1)])
def test_rows(hip, n, e, k):
    check(make(n, e, torch.float32, seed=n), k, True)


@pytest.mark.parametrize("renormalize", [True, False])
def test_many_blocks(hip, renormalize):
    """More rows than one scan part holds, against a vectorised form."""
    n, e, k = 70_001, 33, 2
    s = make(n, e, torch.bfloat16, seed=1)
    got = gmmxx_amd.route_rows(s.to(DEV), k, renormalize=renormalize)
    ranked, index = torch.sort(s.float(), dim=1, descending=True, stable=True)
    flat = index[:, :k].reshape(-1)
    assert torch.equal(got.experts.cpu().long().reshape(-1), flat)
    order = torch.sort(flat, stable=True).indices
    assert torch.equal(got.rows.cpu().long(), order // k)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(n * k)
    assert torch.equal(got.slots.cpu().long().reshape(-1), slots)
    assert torch.equal(got.offsets.cpu().long()[1:], torch.bincount(flat, minlength=e).cumsum(0))


def test_blocks_of_more_rows(hip):
    """Past 4096 blocks of 64 rows a block takes more of them."""
    n, e, k = 300_001, 5, 1
    s = make(n, e, torch.float16, seed=2)
    got = gmmxx_amd.route_rows(s.to(DEV), k)
    flat = torch.sort(s.float(), dim=1, descending=True, stable=True).indices[:, 0]
    assert torch.equal(got.rows.cpu().long(), torch.sort(flat, stable=True).indices)
    assert torch.equal(got.gates.cpu(), torch.ones(n, 1))


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("e,k", [(8, 3), (64, 8), (300, 5)])
def test_ties(hip, e, k, dtype):
    check(make(50, e, dtype, levels=2), k, True)
    check(torch.zeros((9, e), dtype=dtype), k, False)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("e,k", [(6, 4), (64, 8), (200, 7)])
def test_masks(hip, e, k, dtype, renormalize):
    s = make(60, e, dtype, seed=4)
    s[1] = -math.inf                                   # nothing is left
    s[2, 1:] = -math.inf                               # one is left
    s[3] = torch.finfo(dtype).min                      # the lowest value is a candidate
    s[4, 2:] = torch.finfo(dtype).min
    s[5, ::2] = math.nan                               # NaN is none
    s[6] = math.nan
    s[7, 3] = math.inf                                 # takes all
    s[8, :3] = math.inf                                # share
    s[9] = math.inf
    s[10, 0], s[10, 1:] = math.inf, -math.inf
    s[11, 0], s[11, 1:] = torch.finfo(dtype).max, torch.finfo(dtype).min
    s[59] = -math.inf
    check(s, k, renormalize)


def test_all_rows_masked(hip):
    r = gmmxx_amd.route_rows(torch.full((70, 12), -math.inf, device=DEV), 3)
    assert (r.experts == -1).all() and not r.gates.any() and not r.offsets.any()
    assert torch.equal(r.rows.cpu().long(), torch.arange(70).repeat_interleave(3))


def test_strides(hip):
    wide = make(40, 90, torch.bfloat16).to(DEV)
    want = gmmxx_amd.route_rows(wide[:, 7:50].contiguous(), 4)
    for view in (wide[:, 7:50], wide[:, 7:50].t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(gmmxx_amd.route_rows(view, 4), want))
    leaf = wide[:, 7:50].detach().requires_grad_()
    ds, = torch.autograd.grad(gmmxx_amd.route_rows(leaf, 4, renormalize=False).gates.sum(), leaf)
    assert ds.shape == (40, 43)


def test_no_rows(hip):
    leaf = torch.zeros((0, 6), device=DEV, requires_grad=True)
    r = gmmxx_amd.route_rows(leaf, 2)
    assert r.experts.shape == r.slots.shape == (0, 2) and r.rows.shape == (0,) and not r.offsets.any()
    ds, = torch.autograd.grad(r.gates.sum(), leaf)
    assert ds.shape == (0, 6)


@pytest.mark.parametrize("renormalize", [True, False])
def test_differences(hip, renormalize):
    s = make(11, 20, torch.float32, seed=8)
    dg = torch.randn((11, 4), generator=torch.Generator().manual_seed(1))
    leaf = s.to(DEV).requires_grad_()
    ds, = torch.autograd.grad(gmmxx_amd.route_rows(leaf, 4, renormalize=renormalize).gates, leaf, dg.to(DEV))
    # a direction small enough to leave the choices as they are
    v = torch.randn(s.shape, generator=torch.Generator().manual_seed(2))
    h = 2.0 ** -10
    ends = [gmmxx_amd.route_rows((s + t * h * v).to(DEV), 4, renormalize=renormalize) for t in (1, -1)]
    assert torch.equal(ends[0].experts, ends[1].experts)
    slope = float(((ref.f64(ends[0].gates) - ref.f64(ends[1].gates)) * dg.double()).sum()) / (2 * h)
    want = float((ref.f64(ds) * v.double()).sum())
    scale = float((ref.f64(ds) * v.double()).abs().sum())
    # h² of third derivatives (1e-6 of the terms), rounding of the gates over h: 44 · 2^-24 · 4 / h
    assert abs(slope - want) <= 1e-4 * scale + 44 * 4 * ref.U / h


def test_row_constants_cancel(hip):
    """A mixture's log joint densities and its log responsibilities choose and weigh alike."""
    s = make(30, 12, torch.float32)
    a = gmmxx_amd.route_rows(s.to(DEV), 3, renormalize=False)
    b = gmmxx_amd.route_rows(torch.log_softmax(s.double(), 1).float().to(DEV), 3, renormalize=False)
    assert torch.equal(a.experts, b.experts)
    assert torch.allclose(a.gates, b.gates, rtol=1e-5)


def test_refusals(hip):
    s = torch.zeros((4, 10), device=DEV)
    f = gmmxx_amd.route_rows
    for err, call in [
        (TypeError, lambda: f([1.0], 1)),
        (ValueError, lambda: f(s.cpu(), 1)),
        (TypeError, lambda: f(s.double(), 1)),
        (ValueError, lambda: f(s[0], 1)),
        (ValueError, lambda: f(s, 0)),
        (ValueError, lambda: f(s, 11)),
        (ValueError, lambda: f(s[:, :0], 1)),
        (ValueError, lambda: f(torch.zeros((1, 4097), device=DEV), 1)),
        (ValueError, lambda: f(torch.zeros((1, 100), device=DEV), 65)),
    ]:
        with pytest.raises(err):
            call()
