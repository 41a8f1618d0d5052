"""grouped_matmul and combine_rows against their definitions in 64 bits: empty and uneven
groups, rows without an expert, odd widths, strides and both weight layouts, and all
gradients; the layer of all four operators."""

import math

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def routing(n, e, k, seed=0, absent=0.0, only=None):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn((n, e), generator=g)
    if only is not None:       # the other experts stay empty
        keep = torch.zeros(e, dtype=torch.bool)
        keep[only] = True
        s[:, ~keep] = -math.inf
    if absent:
        s[torch.rand(n, generator=g) < absent] = -math.inf
    return gmmxx_amd.route_rows(s.to(DEV), k)


def operands(n, e, d, f, m, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 100)
    x = torch.randn((n, d), generator=g).to(dtype)
    w = (torch.randn((e, d, f), generator=g) / math.sqrt(d)).to(dtype)
    b = torch.randn((e, f), generator=g).to(dtype)
    dy = torch.randn((m, f), generator=g).to(dtype)
    return tuple(t.to(DEV) for t in (x, w, b, dy))


def check(x, w, b, dy, groups):
    routed = isinstance(groups, gmmxx_amd.Routing)
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = gmmxx_amd.grouped_matmul(leaves[0], leaves[1], groups, bias=leaves[2])
    assert y.dtype == x.dtype
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    offsets = groups.offsets if routed else groups
    want = ref.grouped(x, w, b, offsets, groups.rows if routed else None, groups.slots if routed else None, dy)
    ref.close(y, *want["out"], "out")
    for nm, got in zip(["dx", "dw"] + ["db"] * (b is not None), grads):
        ref.close(got, *want[nm], nm)
    assert torch.equal(gmmxx_amd.grouped_matmul(x, w, groups, bias=b), y.detach())


SIZES = [(1, 1), (1, 40), (40, 1), (16, 16), (17, 33), (64, 64), (65, 63), (100, 77), (128, 256), (136, 264),
         (192, 320), (512, 128), (130, 514)]


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("d,f", SIZES)
def test_sizes(hip, d, f, dtype):
    print(f"[grouped] d={d} f={f} {dtype}", flush=True)
    r = routing(150, 5, 2, seed=d)
    check(*operands(150, 5, d, f, 300, dtype), r)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (1, 8, 2), (3, 70, 3), (16, 4, 4), (63, 2, 1), (64, 1, 1), (257, 3, 1),
                                   (1000, 6, 2), (700, 130, 2), (2500, 2, 1)])
def test_rows_and_experts(hip, n, e, k, dtype):
    print(f"[grouped] n={n} e={e} k={k} {dtype}", flush=True)
    r = routing(n, e, k, seed=n)
    check(*operands(n, e, 72, 96, n * k, dtype), r)
    check(*operands(n, e, 128, 128, n * k, dtype), r)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("d,f", [(64, 128), (50, 30)])
def test_empty_groups_and_absent_choices(hip, d, f, dtype):
    for r in (routing(200, 9, 2, only=[4], absent=0.3), routing(200, 9, 3, only=[0, 8]),
              routing(40, 9, 2, absent=1.0), routing(200, 9, 2, absent=0.5)):
        x, w, b, dy = operands(200 if r.slots.shape[0] == 200 else 40, 9, d, f, r.slots.numel(), dtype)
        check(x, w, b, dy, r)
        check(x, w, None, dy, r)


@pytest.mark.parametrize("bits", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("ends", [[0, 5, 5, 130, 200, 300], [0, 0, 0, 0, 0, 300], [0, 300, 300, 300, 300, 300],
                                  [0, 1, 2, 3, 4, 5], [0, 0, 0, 0, 0, 0], [0, 64, 128, 192, 256, 300]])
def test_offsets(hip, ends, bits):
    for dtype in ref.DTYPES:
        off = torch.tensor(ends, dtype=bits, device=DEV)
        x, w, b, dy = operands(300, 5, 80, 144, 300, dtype)
        check(x, w, b, dy, off)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("d,f", [(64, 192), (39, 70)])
def test_layouts(hip, d, f, dtype):
    r = routing(120, 4, 2)
    x, w, b, dy = operands(120, 4, d, f, 240, dtype)
    turned = w.transpose(1, 2).contiguous().transpose(1, 2)      # (E, F, D) in memory
    check(x, turned, b, dy, r)
    padded = torch.zeros((4, d + 3, f + 5), dtype=dtype, device=DEV)
    padded[:, 1:d + 1, 3:f + 3] = w
    check(x, padded[:, 1:d + 1, 3:f + 3], b, dy, r)
    spread = torch.zeros((4, 2 * d, 2 * f), dtype=dtype, device=DEV)
    spread[:, ::2, ::2] = w
    check(x, spread[:, ::2, ::2], b, dy, r)                      # neither dimension adjacent: copied
    wide = torch.zeros((120, d + 9), dtype=dtype, device=DEV)
    wide[:, 5:d + 5] = x
    wide_dy = torch.zeros((240, f + 7), dtype=dtype, device=DEV)
    wide_dy[:, 1:f + 1] = dy
    check(wide[:, 5:d + 5], w, b, wide_dy[:, 1:f + 1], r)
    check(x.t().contiguous().t(), w, b, dy.t().contiguous().t(), r)
    one = w[:1].expand(4, d, f)                                  # the same matrix for every expert
    check(x, one, b, dy, r)


def test_broadcast_gradients(hip):
    """A matrix shared by all experts gets the sum of theirs."""
    r = routing(90, 3, 2)
    x, w, b, dy = operands(90, 3, 40, 48, 180, torch.float32)
    leaf = w[0].detach().requires_grad_()
    y = gmmxx_amd.grouped_matmul(x, leaf.expand(3, 40, 48), r)
    g, = torch.autograd.grad(y, leaf, dy)
    want, bound = ref.grouped(x, leaf.expand(3, 40, 48), None, r.offsets, r.rows, r.slots, dy)["dw"]
    ref.close(g, want.sum(0), bound.sum(0) + 4 * ref.U * want.abs().sum(0), "dw")


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_rows_that_are_not_finite(hip, dtype):
    """A row's infinities and NaN stay in its own results (forward)."""
    r = routing(100, 4, 2)
    x, w, b, dy = operands(100, 4, 64, 64, 200, dtype)
    want = gmmxx_amd.grouped_matmul(x, w, r, bias=b)
    x[10, 3], x[20, 5], x[30, 7] = math.inf, -math.inf, math.nan
    got = gmmxx_amd.grouped_matmul(x, w, r, bias=b)
    hit = torch.zeros(200, dtype=torch.bool, device=DEV)
    for row in (10, 20, 30):
        hit[r.slots[row].long()] = True
    assert torch.equal(got[~hit], want[~hit])
    assert not torch.isfinite(got[hit]).any()


def test_group_that_is_not_finite(hip):
    """An expert's non-finite weights and gradients stay its own."""
    off = torch.tensor([0, 50, 81, 200], dtype=torch.int32, device=DEV)
    for dtype in ref.DTYPES:
        x, w, b, dy = operands(200, 3, 64, 64, 200, dtype)
        w[1] = math.nan
        y = gmmxx_amd.grouped_matmul(x, w, off)
        assert torch.isnan(y[50:81]).all() and torch.isfinite(y[:50]).all() and torch.isfinite(y[81:]).all()
        x[60], dy[70] = math.nan, math.inf
        lw = w.detach().requires_grad_()
        lb = b.detach().requires_grad_()
        gw, gb = torch.autograd.grad(gmmxx_amd.grouped_matmul(x, lw, off, bias=lb), (lw, lb), dy)
        assert torch.isfinite(gw[0]).all() and torch.isfinite(gw[2]).all() and torch.isnan(gw[1]).all()
        assert torch.isfinite(gb[0]).all() and torch.isfinite(gb[2]).all() and not torch.isfinite(gb[1]).any()


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_values_out_of_range(hip, dtype):
    """Offsets and rows out of range stay in bounds."""
    x, w, b, _ = operands(100, 3, 64, 64, 100, dtype)
    off = torch.tensor([0, 40, 1000, -5], dtype=torch.int64, device=DEV)
    y = gmmxx_amd.grouped_matmul(x, w, off, bias=b)
    assert torch.equal(y[:40], gmmxx_amd.grouped_matmul(x[:40], w, off.clamp(0, 40), bias=b))
    r = routing(50, 3, 2)
    wild = r._replace(rows=(r.rows.long() * 1000 - 7).int())
    assert gmmxx_amd.grouped_matmul(x[:50], w, wild).shape == (100, 64)


def test_one_expert_is_a_plain_product(hip):
    x, w, _, _ = operands(513, 1, 96, 80, 513, torch.float32)
    off = torch.tensor([0, 513], dtype=torch.int32, device=DEV)
    y = gmmxx_amd.grouped_matmul(x, w, off)
    want = ref.f64(x) @ ref.f64(w[0])
    ref.close(y, want, 98 * ref.U * (ref.f64(x).abs() @ ref.f64(w[0]).abs()) + ref.U * want.abs(), "out")


def test_no_positions(hip):
    x, w, b, _ = operands(4, 3, 16, 16, 4, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x[:0], w, b)]
    y = gmmxx_amd.grouped_matmul(leaves[0], leaves[1], torch.zeros(4, dtype=torch.int32, device=DEV), bias=leaves[2])
    dx, dw, db = torch.autograd.grad(y.sum(), leaves)
    assert y.shape == (0, 16) and dx.shape == (0, 16) and not dw.any() and not db.any()


def test_differences(hip):
    r = routing(40, 4, 2, absent=0.1)
    x, w, b, dy = operands(40, 4, 24, 20, 80, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(gmmxx_amd.grouped_matmul(leaves[0], leaves[1], r, bias=leaves[2]), leaves, dy)
    g = torch.Generator().manual_seed(9)
    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=g).to(DEV)
        ends = []
        for sign in (1, -1):
            args = [t.detach() for t in leaves]
            args[i] = args[i] + sign * v
            ends.append((ref.f64(gmmxx_amd.grouped_matmul(args[0], args[1], r, bias=args[2])) * ref.f64(dy)).sum())
        want = float((ref.f64(grads[i]) * ref.f64(v)).sum())
        scale = float((ref.f64(grads[i]) * ref.f64(v)).abs().sum())
        # bilinear: the difference over a whole step has no error but rounding, of 1600 results and of x + v
        assert abs(float(ends[0] - ends[1]) / 2 - want) <= 1e-5 * scale + 1600 * 32 * ref.U


def test_grouped_same_bits_again(hip):
    r = routing(3000, 7, 2)
    leaves = [t.requires_grad_() for t in operands(3000, 7, 128, 192, 6000, torch.bfloat16)[:3]]
    dy = operands(3000, 7, 128, 192, 6000, torch.bfloat16)[3]
    runs = [torch.autograd.grad(gmmxx_amd.grouped_matmul(leaves[0], leaves[1], r, bias=leaves[2]), leaves, dy)
            for _ in range(3)]
    for g in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(g, runs[0]))


# --- combination ------------------------------------------------------------------------

def check_combine(y, r, gates, dout):
    ly, lg = y.detach().requires_grad_(), gates.detach().requires_grad_()
    out = gmmxx_amd.combine_rows(ly, r, lg)
    assert out.dtype == y.dtype
    dy, dg = torch.autograd.grad(out, (ly, lg), dout)
    want = ref.combine(y, gates, r.slots, int(r.offsets[-1]), dout)
    ref.close(out, *want["out"], "out")
    ref.close(dy, *want["dy"], "dy")
    ref.close(dg, *want["dgates"], "dgates")
    assert torch.equal(gmmxx_amd.combine_rows(y, r, gates), out.detach())


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("f", [1, 5, 8, 31, 64, 100, 256, 257, 1000, 2048, 4099])
@pytest.mark.parametrize("k", [1, 2, 3, 4, 7, 9])
def test_combine(hip, f, k, dtype):
    r = routing(33, 9, k, seed=f, absent=0.2)
    g = torch.Generator().manual_seed(f)
    y = torch.randn((33 * k, f), generator=g).to(dtype).to(DEV)
    dout = torch.randn((33, f), generator=g).to(dtype).to(DEV)
    check_combine(y, r, r.gates, dout)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_combine_strides(hip, dtype):
    r = routing(50, 6, 2)
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((100, 90), generator=g).to(dtype).to(DEV)
    dout = torch.randn((50, 80), generator=g).to(dtype).to(DEV)
    gates = torch.randn((50, 2), generator=g).to(DEV)
    check_combine(wide[:, 3:70], r, gates, dout[:, 5:72])
    check_combine(wide[:, 3:70].t().contiguous().t(), r, gates.t().contiguous().t(), dout[:, 5:72].t().contiguous().t())


def test_combine_ignores_positions_without_expert(hip):
    r = routing(30, 4, 2, absent=0.5)
    y = torch.randn((60, 40), generator=torch.Generator().manual_seed(0)).to(DEV)
    taken = int(r.offsets[-1])
    assert taken < 60
    want = gmmxx_amd.combine_rows(y, r)
    y[taken:] = math.nan
    assert torch.equal(gmmxx_amd.combine_rows(y, r), want)
    ly, lg = y.requires_grad_(), r.gates.detach().requires_grad_()
    dy, dg = torch.autograd.grad(gmmxx_amd.combine_rows(ly, r, lg).sum(), (ly, lg))
    assert not dy[taken:].any() and torch.isfinite(dg).all()


def test_combine_no_rows(hip):
    r = gmmxx_amd.route_rows(torch.zeros((0, 4), device=DEV), 2)
    y = torch.zeros((0, 8), device=DEV, requires_grad=True)
    out = gmmxx_amd.combine_rows(y, r)
    assert out.shape == (0, 8) and torch.autograd.grad(out.sum(), y)[0].shape == (0, 8)


def test_combine_out_of_range(hip):
    r = routing(20, 3, 2)
    y = torch.ones((40, 16), device=DEV)
    wild = r._replace(slots=r.slots * 1000 - 3)
    assert torch.isfinite(gmmxx_amd.combine_rows(y, wild)).all()


# --- the layer ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_layer(hip, dtype):
    """norm, gate, experts and sum with gradients through all of them, against 64 bits."""
    n, e, k, d, f = 300, 6, 2, 48, 40
    g = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    base = [make(n, d), 1 + 0.1 * make(d), 0.1 * make(d), make(d, e) / 7, make(e, d, f) / 7, 0.1 * make(e, f)]
    dout = make(n, f)
    own = [t.to(dtype).to(DEV).requires_grad_() for t in base]
    h = gmmxx_amd.layer_norm(own[0], own[1], own[2])
    r = gmmxx_amd.route_rows(h.float() @ own[3].float(), k)
    out = gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(h, own[4], r, bias=own[5]), r)
    got = torch.autograd.grad(out, own, dout.to(dtype).to(DEV))
    # 64 bits, with the same choices
    lv = [t.to(dtype).double().requires_grad_() for t in base]
    var, mean = torch.var_mean(lv[0], dim=1, keepdim=True, unbiased=False)
    h64 = (lv[0] - mean) / torch.sqrt(var + 1e-5) * lv[1] + lv[2]
    s64 = h64 @ lv[3]
    pick = r.experts.cpu().long()
    gates = torch.softmax(s64.gather(1, pick), 1)
    out64 = sum(gates[:, j, None] * (torch.matmul(h64[:, None, :], lv[4][pick[:, j]])[:, 0] + lv[5][pick[:, j]])
                for j in range(k))
    want = torch.autograd.grad(out64, lv, dout.to(dtype).double())
    # five roundings to the type in a row, each a unit of values whose sums are no larger than 32 of them
    tol = 32 * 5 * ref.unit(dtype) if dtype != torch.float32 else 2e-5
    for a, b in zip((out, *got), (out64, *want)):
        err = float((ref.f64(a) - b.detach()).norm() / b.detach().norm())
        assert err <= tol, err


def test_mixture_as_gate(hip):
    """A fitted mixture's responsibilities route its rows: the best expert is predict()'s label."""
    g = torch.Generator().manual_seed(0)
    centers = 6 * torch.randn((5, 8), generator=g)
    x = (centers[torch.randint(0, 5, (2000,), generator=g)] + torch.randn((2000, 8), generator=g)).to(DEV)
    model = gmmxx_amd.GMMXX(n_components=5, covariance_type="diag", max_iter=10, device=DEV).fit(x)
    r = gmmxx_amd.route_rows(torch.log(model.predict_proba(x)), 1, renormalize=False)
    assert torch.equal(r.experts[:, 0].long(), model.predict(x).long())
    counts = torch.bincount(model.predict(x), minlength=5)
    assert torch.equal((r.offsets[1:] - r.offsets[:-1]).long(), counts)


def test_refusals(hip):
    r = routing(10, 3, 2)
    x, w, b, _ = operands(10, 3, 16, 8, 20, torch.float32)
    off = torch.tensor([0, 3, 5, 10], dtype=torch.int32, device=DEV)
    y = torch.zeros((20, 8), device=DEV)
    f, c = gmmxx_amd.grouped_matmul, gmmxx_amd.combine_rows
    for err, call in [
        (TypeError, lambda: f([1.0], w, r)),
        (ValueError, lambda: f(x.cpu(), w, r)),
        (TypeError, lambda: f(x.double(), w.double(), r)),
        (TypeError, lambda: f(x, w.bfloat16(), r)),
        (ValueError, lambda: f(x, w.cpu(), r)),
        (ValueError, lambda: f(x[0], w, r)),
        (ValueError, lambda: f(x, w[0], r)),
        (ValueError, lambda: f(x[:, :15], w, r)),
        (ValueError, lambda: f(x[:9], w, r)),
        (ValueError, lambda: f(x, w[:2], r)),
        (ValueError, lambda: f(x, w[:, :, :0], r)),
        (ValueError, lambda: f(x, w, r, bias=b[:2])),
        (TypeError, lambda: f(x, w, r, bias=b.half())),
        (TypeError, lambda: f(x, w, off.float())),
        (ValueError, lambda: f(x, w, off[:3])),
        (ValueError, lambda: f(x, w, off.cpu())),
        (TypeError, lambda: f(x, w, None)),
        (TypeError, lambda: f(x, w, r._replace(rows=r.rows.long()))),
        (ValueError, lambda: f(x, w, r._replace(rows=r.rows[:-1]))),
        (TypeError, lambda: c(y, tuple(r))),
        (ValueError, lambda: c(y[:19], r)),
        (ValueError, lambda: c(y[0], r)),
        (ValueError, lambda: c(y[:, :0], r)),
        (TypeError, lambda: c(y, r, r.gates.half())),
        (ValueError, lambda: c(y, r, r.gates[:, :1])),
        (ValueError, lambda: c(y.cpu(), r)),
        (TypeError, lambda: c(y.int(), r)),
    ]:
        with pytest.raises(err):
            call()
