"""log_probs against its definition in 64 bits: row lengths, counts and alternatives at which the kernels change
their ways, ties, masked and empty rows, infinities and NaN, places that do not count, and the gradients of all
three results against the formula and against differences."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref, tokens_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = experts_ref.DTYPES
INF = float("inf")


def make(n, v, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    s = (spread * torch.randn((n, v), generator=g)).to(dtype)
    t = torch.randint(0, v, (n,), generator=g)
    t[3::7] = -1
    return s.to(DEV), t.to(DEV)


def compare(got, want):
    for name in ("chosen", "entropy", "top"):
        experts_ref.close(getattr(got, name), *want[name], name)
    assert got.top_index.dtype == torch.int32
    assert torch.equal(got.top_index.cpu().long(), want["top_index"][0]), "top_index"


def check(s, t, k, seed=0):
    n = s.shape[0]
    g = torch.Generator().manual_seed(seed)
    dc, dh, dt = (torch.randn(sh, generator=g).to(DEV) for sh in ((n,), (n,), (n, k)))
    leaf = s.detach().requires_grad_()
    r = gmmxx_amd.log_probs(leaf, t, top_k=k)
    outs, grads = (r.chosen, r.entropy, r.top), (dc, dh, dt)
    if k == 0:
        outs, grads = outs[:2], grads[:2]
    ds, = torch.autograd.grad(outs, leaf, grads)
    want = ref.log_probs(s, t, k, dc, dh, dt if k else None)
    compare(r, want)
    assert ds.dtype == s.dtype
    experts_ref.close(ds, *want["dscores"], "dscores")
    plain = gmmxx_amd.log_probs(s, t, top_k=k)
    assert all(torch.equal(a, b) for a, b in zip(plain, r))


LENGTHS = [1, 2, 3, 4, 7, 8, 9, 31, 63, 100, 127, 128, 129, 500, 512, 513, 1000, 2047, 2048, 2049, 4095, 4097, 8193, 20001,
           65536, 131073]


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("v", LENGTHS)
def test_lengths(hip, v, dtype):
    for k in sorted({0, 1, min(v, 5), min(v, 64)}):
        print(f"[log_probs] v={v} k={k} {dtype}", flush=True)
        check(*make(5, v, dtype, seed=v), k)


@pytest.mark.parametrize("n", [1, 2, 3, 17, 64, 257, 1025, 3000])
@pytest.mark.parametrize("v,k", [(77, 0), (77, 3), (300, 0), (2100, 0), (5001, 4)])
def test_counts(hip, n, v, k):
    print(f"[log_probs] n={n} v={v} k={k}", flush=True)
    check(*make(n, v, BF16, seed=n), k)


@pytest.mark.parametrize("n", [4095, 4097])
@pytest.mark.parametrize("v", [2049, 4099, 32768, 32769])
@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_many_long_rows(hip, n, v, dtype):
    """Both sides of the counts and lengths from which a wave takes a row; masked rows and far scores among them.
    A lane adds 128 vectors of fp32 at most, 8 in a vector and 6 levels: 142 additions, the bound counts 154."""
    print(f"[log_probs] n={n} v={v} {dtype}", flush=True)
    s, t = make(61, v, dtype)
    s, t = s.repeat(n // 61 + 1, 1)[:n], t.repeat(n // 61 + 1)[:n]
    s[7], s[8], s[9] = -INF, torch.finfo(dtype).min, float("nan")
    s[10, v - 1], s[11, :v - 1], s[12] = 2.0 ** 101, -INF, torch.finfo(dtype).max
    got = gmmxx_amd.log_probs(s, t)
    at = torch.cat([torch.arange(30), torch.arange(n - 30, n)]).to(DEV)
    want = ref.log_probs(s[at], t[at])
    experts_ref.close(got.chosen[at], *want["chosen"], "chosen")
    experts_ref.close(got.entropy[at], *want["entropy"], "entropy")


@pytest.mark.parametrize("v", [6, 700, 3000, 40_000])
@pytest.mark.parametrize("k", [0, 4])
@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
def test_masks(hip, v, k, dtype):
    """Masks of -inf, of the type's lowest value and of NaN; rows of each alone; one candidate; some +inf."""
    print(f"[log_probs] masks v={v} k={k} {dtype}", flush=True)
    s, t = make(13, v, dtype)
    low = torch.finfo(dtype).min
    off = torch.rand((13, v), generator=torch.Generator().manual_seed(1)).to(DEV) < 0.4
    s[0][off[0]] = -INF
    s[1][off[1]] = low
    s[2][off[2]] = float("nan")
    s[3], s[4], s[5] = -INF, low, float("nan")
    s[6] = -INF
    s[6, v - 1] = 2.0
    s[7, 1], s[7, v - 1] = INF, INF
    s[8] = INF
    s[9], s[9, 2] = -INF, low
    s[10, v // 2] = INF
    s[11] = -INF
    s[11, ::2] = float("nan")
    s[12] = 0.0
    t[:] = torch.arange(13, device=DEV) % min(v, 5)
    t[8] = -5
    t[9] = 2
    check(s, t, k)


@pytest.mark.parametrize("v", [200, 10_000, 100_000])
@pytest.mark.parametrize("order", ["equal", "ascending", "descending", "two values", "few"])
def test_orders(hip, v, order):
    """Rows whose order or ties fill the list of alternatives: the lower index comes first."""
    print(f"[log_probs] {order} v={v}", flush=True)
    i = torch.arange(v, dtype=torch.float32)
    row = {"equal": torch.zeros(v), "ascending": i / v, "descending": -i / v, "two values": (i % 7 == 3).float(),
           "few": torch.where(i % (v // 5) == 9, i / v, torch.full((v,), -INF))}[order]
    s = torch.stack([row, row.flip(0)]).to(DEV)
    for k in (1, 64):
        check(s, torch.tensor([v - 1, 9], device=DEV), k)


def test_many_rows_of_ties(hip):
    s = torch.randint(0, 3, (2000, 9000), generator=torch.Generator().manual_seed(0)).to(BF16).to(DEV)
    r = gmmxx_amd.log_probs(s, torch.zeros(2000, dtype=torch.int64, device=DEV), top_k=20)
    want = torch.sort(s.float(), dim=1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(r.top_index.long(), want)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0, 1000.0])
@pytest.mark.parametrize("v", [400, 9000])
def test_spreads(hip, scale, v):
    check(*make(6, v, F32, spread=scale), 3)
    s, t = make(6, v, F32, spread=scale)
    check(s + 5000.0, t, 0)                # far from zero


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("v", [150, 5000])
def test_strides_and_types(hip, dtype, v):
    s, t = make(12, v, dtype)
    wide = torch.full((12, v + 50), 30.0, dtype=dtype, device=DEV)
    wide[:, 33:33 + v] = s
    for k in (0, 3):
        check(wide[:, 33:33 + v], t.int(), k)
        check(s.t().contiguous().t(), torch.stack([t, t], 1)[:, 0], k)
    r = gmmxx_amd.log_probs(s.reshape(3, 4, v), t.reshape(3, 4), top_k=2)
    want = gmmxx_amd.log_probs(s, t, top_k=2)
    assert r.top.shape == (3, 4, 2) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(r, want))
    one = gmmxx_amd.log_probs(s[0], t[0], top_k=2)
    assert one.chosen.shape == () and torch.equal(one.top_index, want.top_index[0])


def test_some_gradients(hip):
    """Each result's gradient alone."""
    s, t = make(9, 300, F32)
    dc, dh, dt = torch.randn(9), torch.randn(9), torch.randn(9, 3)
    for which in ("chosen", "entropy", "top"):
        leaf = s.detach().requires_grad_()
        r = gmmxx_amd.log_probs(leaf, t, top_k=3)
        g = {"chosen": dc, "entropy": dh, "top": dt}[which]
        ds, = torch.autograd.grad(getattr(r, which), leaf, g.to(DEV))
        experts_ref.close(ds, *ref.log_probs(s, t, 3, **{"d" + which: g})["dscores"], which)
    leaf = s.detach().requires_grad_()
    gmmxx_amd.log_probs(leaf, t).chosen.sum().backward()          # a gradient with strides of zero
    experts_ref.close(leaf.grad, *ref.log_probs(s, t, 0, dchosen=torch.ones(9))["dscores"], "ones")


def test_differences(hip):
    """Gradients against central differences of the 64-bit form."""
    s, t = make(4, 11, F32)
    leaf = s.detach().requires_grad_()
    r = gmmxx_amd.log_probs(leaf, t, top_k=2)
    w = [torch.randn(sh, generator=torch.Generator().manual_seed(5)) for sh in ((4,), (4,), (4, 2))]
    ds, = torch.autograd.grad((r.chosen, r.entropy, r.top), leaf, [x.to(DEV) for x in w])

    def value(x):
        o = ref.log_probs(x, t, 2)
        return sum(float((o[name][0] * wi.double()).sum()) for name, wi in zip(("chosen", "entropy", "top"), w))

    base, h = s.double().cpu(), 1e-5
    for r0 in range(4):
        for c in range(11):
            up, down = base.clone(), base.clone()
            up[r0, c] += h
            down[r0, c] -= h
            # the difference's own error: h^2 / 6 times third derivatives (of order 10), and the values' rounding over h
            assert abs((value(up) - value(down)) / (2 * h) - float(ds[r0, c])) < 1e-4


def test_no_rows(hip):
    s, t = make(3, 20, F32)
    leaf = s[:0].detach().requires_grad_()
    r = gmmxx_amd.log_probs(leaf, t[:0], top_k=2)
    assert r.chosen.shape == (0,) and r.top.shape == (0, 2)
    assert torch.autograd.grad(r.chosen.sum() + r.entropy.sum(), leaf)[0].shape == (0, 20)


def test_tokens_outside(hip):
    s, t = make(6, 50, F32)
    for bad in (-1, -100, 50, 1 << 40, -(1 << 40)):
        t[:] = bad
        leaf = s.detach().requires_grad_()
        r = gmmxx_amd.log_probs(leaf, t)
        assert not r.chosen.any()
        assert not torch.autograd.grad(r.chosen.sum(), leaf)[0].any()


def test_past_32_bits(hip):
    """Scores past 2^31 elements and 2^32 bytes, at the far rows."""
    n, v = 36_000, 65_536
    s = torch.empty((n, v), dtype=BF16, device=DEV)
    for i in range(0, n, 4000):
        s[i:i + 4000].normal_()
    t = torch.randint(0, v, (n,), device=DEV)
    leaf = s.requires_grad_()
    r = gmmxx_amd.log_probs(leaf, t, top_k=2)
    far = torch.tensor([0, 1, n // 2, n - 1], device=DEV)
    want = ref.log_probs(s.detach()[far], t[far], 2, dchosen=torch.ones(4))
    compare(gmmxx_amd.LogProbs(*(x[far] for x in r)), want)
    ds, = torch.autograd.grad(r.chosen.sum(), leaf)
    experts_ref.close(ds[far], *want["dscores"], "dscores")


@pytest.mark.parametrize("v,k", [(4096, 64), (5000, 4), (9000, 33)])
def test_few_candidates_among_nan(hip, v, k):
    """Candidates in a few places only, the rest NaN: a bound from some of the scores must not pass any of them."""
    g = torch.Generator().manual_seed(v)
    s = torch.full((40, v), float("nan"))
    for r in range(40):
        at = torch.randperm(v, generator=g)[:1 + 2 * r]
        s[r, at] = torch.randn(at.numel(), generator=g)
    check(s.to(DEV), torch.randint(0, v, (40,), generator=g).to(DEV), k)


@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("v", [9, 600, 5000, 40_000])
@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_far_scores(hip, v, k, dtype):
    """Rows around 2^100 in size and at the type's ends, among ordinary scores and alone."""
    big = torch.finfo(dtype).max
    s, t = make(12, v, dtype)
    for r, x in enumerate((2.0 ** 99, 2.0 ** 100, 2.0 ** 101, big)):
        s[r, v // 3] = x
        s[r, v // 2] = x
        s[4 + r] = -x
        s[4 + r, v // 4] = -x / 2
    s[8], s[9, 5], s[10], s[11, 1::2] = big, -big, -big, -2.0 ** 100
    t[:] = torch.tensor([v // 3, 0, v // 2, v // 3, 1, v // 4, v // 4, 2, 3, 5, 0, 1], device=DEV)
    check(s, t, k)


@pytest.mark.parametrize("dtype", (F32, F16), ids=str)
@pytest.mark.parametrize("n", [300, 600])
@pytest.mark.parametrize("v", [2, 5, 32, 33, 64, 65, 128, 129, 256, 257, 512, 513, 1024, 1025, 2048, 2049])
def test_short_rows_with_alternatives(hip, n, v, dtype):
    """Every group of lanes, more rows than a workgroup's, ties and masks among them."""
    g = torch.Generator().manual_seed(v)
    s = (torch.randint(-6, 7, (n, v), generator=g) / 2.0).to(dtype)
    s[torch.rand((n, v), generator=g) < 0.3] = -INF
    s[7], s[8] = -INF, torch.finfo(dtype).min
    s[9, v // 2] = INF
    s[10, ::2] = float("nan")
    t = torch.randint(0, v, (n,), generator=g)
    t[::13] = -1
    for k in sorted({1, min(v, 7), min(v, 33), min(v, 64)}):
        check(s.to(DEV), t.to(DEV), k)


FAR = [-1e30, -1e20, -1e12, -1e10, -3e9, -1.2e9, -1e9, -5e8, -3.1e7, -1.5e7, 1.5e7, 3.1e7, 5e8, 1e9, 1.2e9, 3e9, 1e10, 1e12, 1e20,
       1e30]


def far_rows(v, dtype):
    """For each far value rows of it alone, of numbers around it, of ordinary scores of which it takes the place of a third, or of
    most of those in front, and a row of which it is the only candidate."""
    g = torch.Generator().manual_seed(v)
    rows = []
    for x in FAR:
        some = 3.0 * torch.randn((5, v), generator=g)
        some[0] = x
        some[1] = x + some[1] * abs(x) * 2.0 ** -23
        some[2][torch.rand(v, generator=g) < 0.3] = x
        some[3, :v - v // 4] = x
        some[4], some[4, v // 2] = -INF, x
        rows.append(some)
    s = torch.cat(rows).to(dtype)
    t = torch.randint(0, v, (s.shape[0],), generator=g)
    t[4::5] = v // 2
    return s.to(DEV), t.to(DEV)


@pytest.mark.parametrize("v,k", [(3, 0), (9, 0), (9, 3), (100, 0), (600, 0), (600, 3), (600, 9), (2000, 0), (5000, 0), (5000, 3),
                                 (40_000, 0), (40_000, 3)])
@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_values_of_far_scores(hip, v, k, dtype):
    """Scores of sizes at which log2(e) times them is rounded by more than exponents hold, as fill values often are."""
    print(f"[log_probs] far values v={v} k={k} {dtype}", flush=True)
    s, t = far_rows(v, dtype)
    compare(gmmxx_amd.log_probs(s, t, top_k=k), ref.log_probs(s, t, k))


@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_values_of_far_scores_in_many_rows(hip, dtype):
    s, t = far_rows(2500, dtype)
    n = s.shape[0]
    got = gmmxx_amd.log_probs(s.repeat(42, 1), t.repeat(42))
    want = ref.log_probs(s, t)
    for part in (slice(0, n), slice(41 * n, 42 * n)):
        experts_ref.close(got.chosen[part], *want["chosen"], "chosen")
        experts_ref.close(got.entropy[part], *want["entropy"], "entropy")


@pytest.mark.parametrize("v,k", [(3, 0), (9, 0), (9, 3), (600, 0), (600, 3), (600, 9), (5000, 0), (5000, 3), (40_000, 0), (40_000, 3)])
@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_gradients_of_far_scores(hip, v, k, dtype):
    print(f"[log_probs] far gradients v={v} k={k} {dtype}", flush=True)
    check(*far_rows(v, dtype), k)


@pytest.mark.parametrize("n,v,lanes,k", [(2000, 64, 4, 0), (2000, 512, 16, 0), (2000, 2000, 64, 0), (4100, 4096, 256, 0),
                                         (2000, 5000, 256, 0), (2000, 5000, 256, 1), (2000, 9000, 1024, 0), (2000, 9000, 1024, 1)])
@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_confident_rows(hip, n, v, lanes, k, dtype):
    """Two candidates, 3.1 to 9.8 powers of two apart, the likelier in a vector that the same lane takes later, p from 0.89
    to 0.999.  The sums are beside the likelier then, whose 2^l is 1 within 2 U; the other's, at most 0.117, is good to 8 U,
    and their sum is rounded by U: log Z is good to 4 U, and so is log p (of at most 0.12, which is rounded by less than U).
    The entropy is log Z less a term of at most 0.25, whose own sum is good to 9 U of itself and whose divisor to 6 U: 4 U."""
    step = lanes * (16 // dtype.itemsize)
    g = torch.Generator().manual_seed(v)
    low = 8.0 * torch.rand(n, generator=g) - 4.0
    s = torch.full((n, v), -INF)
    s[:, 1], s[:, step + 2] = low, low + 2.2 + 4.5 * torch.rand(n, generator=g)
    s, t = s.to(dtype).to(DEV), torch.full((n,), step + 2, device=DEV)
    got, want = gmmxx_amd.log_probs(s, t, top_k=k), ref.log_probs(s, t, k)
    chosen, entropy = want["chosen"][0], want["entropy"][0]
    u = experts_ref.U
    experts_ref.close(got.chosen, chosen, torch.full_like(chosen, 5 * u), "chosen")
    experts_ref.close(got.entropy, entropy, torch.full_like(entropy, 9 * u), "entropy")


@pytest.mark.parametrize("v", [5, 64, 500, 2000, 5000, 40_000])
@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
def test_no_probability_past_one(hip, v, dtype):
    n = 1000
    s, t = make(n, v, dtype, spread=1.0)
    t = t.clamp(min=0)
    s.scatter_(1, t[:, None], 14.0 + 6.0 * torch.rand((n, 1), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV))
    for k in (0, 2):
        r = gmmxx_amd.log_probs(s, t, top_k=k)
        assert (r.chosen <= 0).all() and (r.top <= 0).all() and (r.entropy >= 0).all()


@pytest.mark.parametrize("v,k", [(3, 0), (9, 0), (9, 3), (600, 0), (600, 3), (5000, 0), (5000, 3), (40_000, 0), (40_000, 3)])
@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
def test_gradients_that_are_not_finite(hip, v, k, dtype):
    """They reach the row's candidates and nothing else."""
    print(f"[log_probs] gradients not finite v={v} k={k} {dtype}", flush=True)
    n, nan = 12, float("nan")
    s, t = make(n, v, dtype)
    g = torch.Generator().manual_seed(2)
    s[torch.rand((n, v), generator=g).to(DEV) < 0.3] = -INF
    s[torch.rand((n, v), generator=g).to(DEV) < 0.2] = nan
    s[:, v // 2] = 1.0
    s[9] = -INF
    t[:] = v // 2
    dc, dh, dt = (torch.randn(sh, generator=g) for sh in ((n,), (n,), (n, k)))
    dc[0], dc[1], dc[2], dc[9] = nan, INF, -INF, nan
    dh[3], dh[4], dh[5], dh[6] = nan, INF, -INF, 3e38
    if k:
        dt[7, 0], dt[8, 0] = nan, INF
    leaf = s.detach().requires_grad_()
    r = gmmxx_amd.log_probs(leaf, t, top_k=k)
    some = 3 if k else 2
    ds, = torch.autograd.grad((r.chosen, r.entropy, r.top)[:some], leaf, [x.to(DEV) for x in (dc, dh, dt)[:some]])
    assert not ds[~(s > -INF)].any()
    fine = [10, 11]
    want = ref.log_probs(s[fine], t[fine], k, dc[fine], dh[fine], dt[fine] if k else None)
    experts_ref.close(ds[fine], *want["dscores"], "dscores")
    for row in range(6):
        assert not torch.isfinite(ds[row, v // 2])


@pytest.mark.parametrize("n", [999, 1000])
@pytest.mark.parametrize("v", [2049, 9216, 9217])
@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_long_rows_by_count(hip, n, v, dtype):
    """Both sides of the count from which a wave takes a row of these lengths."""
    print(f"[log_probs] n={n} v={v} {dtype}", flush=True)
    s, t = make(43, v, dtype)
    s, t = s.repeat(n // 43 + 1, 1)[:n], t.repeat(n // 43 + 1)[:n]
    s[7], s[8], s[9] = -INF, torch.finfo(dtype).min, float("nan")
    s[10, v - 1], s[11, :v - 1], s[12] = 3e12, -INF, -1e10
    got = gmmxx_amd.log_probs(s, t)
    at = torch.cat([torch.arange(20), torch.arange(n - 20, n)]).to(DEV)
    want = ref.log_probs(s[at], t[at])
    experts_ref.close(got.chosen[at], *want["chosen"], "chosen")
    experts_ref.close(got.entropy[at], *want["entropy"], "entropy")
