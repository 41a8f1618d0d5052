"""quantize_rows and quantized_matmul: 8-bit values equal to their definition in fp32, products within the
rounding of an exact sum, at sizes around every tile, odd and strided layouts."""

import pytest
import torch

import gmmxx_amd
from gmmxx_amd import Quantized
from tests import experts_ref, tokens_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = experts_ref.DTYPES
U = experts_ref.U


def rand(*shape, seed=0, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def same(q, x):
    values, scales = ref.quantize(x)
    assert q.values.dtype == torch.int8 and torch.equal(q.values.cpu(), values)
    assert torch.equal(q.scales.cpu().isnan(), scales.isnan())
    assert torch.equal(q.scales.cpu().nan_to_num(7.0), scales.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("d", [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 64, 100, 128, 129, 511, 513, 1000, 1024, 1025, 4096, 8193, 40_000,
                               131_072])
def test_values(hip, d, dtype):
    print(f"[quantize] d={d} {dtype}", flush=True)
    for n in (1, 5, 33):
        same(gmmxx_amd.quantize_rows(rand(n, d, seed=n, dtype=dtype)), rand(n, d, seed=n, dtype=dtype))


def test_values_at_the_ends(hip):
    x = rand(12, 200)
    x[0] = 0.0
    x[1] *= 1e-44                      # subnormal
    x[2] *= 1e-38
    x[3] *= 1e37
    x[4, 7] = float("inf")
    x[5, 8] = float("nan")
    x[6] = 0.0
    x[6, 3] = -5.0
    x[7] = torch.arange(200, device=DEV) / 2.0 - 50          # ties
    x[8] *= 2.0 ** -100
    x[9] = 3.0
    x[10, 199] = float("-inf")
    same(gmmxx_amd.quantize_rows(x), x)
    y = gmmxx_amd.quantized_matmul(x, gmmxx_amd.quantize_rows(rand(9, 200, seed=1)))
    bad = torch.tensor([4, 5, 10], device=DEV)
    # (row 3's results have a deviation of 1e37 sqrt(200) = 1.4e38: some pass fp32's largest, 3.4e38)
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[[0, 1, 2, 6, 7, 8, 9, 11]]).all() and not y[0].any()


def test_layout(hip):
    x = rand(6, 300)
    q = gmmxx_amd.quantize_rows(x)
    assert q.values.shape == (6, 300) and q.values.stride() == (384, 1)
    wide = torch.zeros((6, 400), device=DEV)
    wide[:, 51:351] = x
    assert torch.equal(gmmxx_amd.quantize_rows(wide[:, 51:351]).values, q.values)
    assert torch.equal(gmmxx_amd.quantize_rows(x.t().contiguous().t()).values, q.values)
    assert gmmxx_amd.quantize_rows(x[:0]).values.shape == (0, 300)


def check(n, d, f, dtype, bias=True, seed=0):
    x = rand(n, d, seed=seed, dtype=dtype)
    w = rand(f, d, seed=seed + 1, scale=d ** -0.5)
    b = rand(f, seed=seed + 2, dtype=dtype) if bias else None
    q = gmmxx_amd.quantize_rows(w)
    y = gmmxx_amd.quantized_matmul(x, q, b)
    assert y.dtype == dtype and y.shape == (n, f)
    qx, sx = ref.quantize(x)
    want, bound = ref.quantized_matmul(qx, sx, q.values, q.scales, b, dtype)
    experts_ref.close(y, want, bound, f"{n} x {d} x {f}")


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("n", [1, 2, 4, 15, 16, 17, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300])
def test_rows(hip, n, dtype):
    print(f"[int8] n={n} {dtype}", flush=True)
    check(n, 200, 144, dtype, seed=n)


@pytest.mark.parametrize("n", [3, 40, 70, 200])
@pytest.mark.parametrize("d", [1, 2, 15, 16, 17, 31, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 383, 1000, 1025, 2048])
def test_depths(hip, n, d):
    print(f"[int8] n={n} d={d}", flush=True)
    check(n, d, 50, BF16, seed=d)


@pytest.mark.parametrize("n", [2, 20, 150])
@pytest.mark.parametrize("f", [1, 3, 15, 16, 17, 64, 127, 128, 129, 255, 257, 1000])
def test_columns(hip, n, f):
    print(f"[int8] n={n} f={f}", flush=True)
    check(n, 96, f, F16, bias=f % 2 == 0, seed=f)


@pytest.mark.parametrize("n,f", [(40, 2100), (200, 1100)])
@pytest.mark.parametrize("d", [1, 15, 16, 17, 64, 100, 127, 128, 129, 257, 383, 1000, 1025])
def test_depths_of_tiles(hip, n, f, d):
    """More groups of 32 rows and 16 columns than the card holds at once."""
    print(f"[int8] n={n} d={d} f={f}", flush=True)
    check(n, d, f, BF16, seed=d)


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("n", [33, 64, 65, 96, 1000, 4095, 8190, 8193])
@pytest.mark.parametrize("f", [1, 16, 17])
def test_groups_of_rows(hip, n, f, dtype):
    """256 groups of 32 rows and 16 columns, one more, and fewer."""
    print(f"[int8] n={n} f={f} {dtype}", flush=True)
    check(n, 70, f, dtype, bias=n % 2 == 0, seed=n)


def test_longest_sums_of_tiles(hip):
    d = 131_072
    x = Quantized(torch.full((200, d), 127, dtype=torch.int8, device=DEV), torch.ones(200, device=DEV))
    w = Quantized(torch.full((1100, d), -127, dtype=torch.int8, device=DEV), torch.ones(1100, device=DEV))
    # (-127^2 2^17 needs 14 bits: fp32 holds it)
    assert (gmmxx_amd.quantized_matmul(x, w) == -127.0 ** 2 * d).all()


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("n,d,f", [(4096, 128, 4096), (4099, 300, 4100), (5000, 1000, 3500), (2048, 513, 16_384)])
def test_large_tiles(hip, n, d, f, dtype):
    """Sizes that take the widest tiles, against exact sums in 64 bits on the card."""
    print(f"[int8] {n} x {d} x {f} {dtype}", flush=True)
    x, q = rand(n, d, dtype=dtype), gmmxx_amd.quantize_rows(rand(f, d, seed=1))
    b = rand(f, seed=2, dtype=dtype)
    y = gmmxx_amd.quantized_matmul(x, q, b).double()
    qx = gmmxx_amd.quantize_rows(x)
    same(Quantized(qx.values[:50], qx.scales[:50]), x[:50])
    prod = (qx.values.double() @ q.values.double().t()) * qx.scales.double()[:, None] * q.scales.double()
    want = prod + b.double()
    bound = 3 * U * prod.abs() + U * want.abs() + experts_ref.unit(dtype) * want.abs() * 1.01 + experts_ref.tiny(dtype)
    assert ((y - want).abs() <= bound).all()


def whole(*shape, seed=0, low=-127):
    return torch.randint(low, 128, shape, generator=torch.Generator().manual_seed(seed)).to(torch.int8).to(DEV)


@pytest.mark.parametrize("n", [1, 30, 200])
@pytest.mark.parametrize("d", [131_072, 131_071])
def test_longest_sums(hip, n, d):
    """Sums up to 2^31: all values 127, and of both signs."""
    ones = torch.ones
    x = torch.full((n, d), 127, dtype=torch.int8, device=DEV)
    w = torch.full((20, d), 127, dtype=torch.int8, device=DEV)
    w[1::2] = -127
    y = gmmxx_amd.quantized_matmul(Quantized(x, ones(n, device=DEV)), Quantized(w, ones(20, device=DEV)))
    assert y.dtype == F32
    want = torch.full((n, 20), 127.0 * 127.0 * d, dtype=torch.float64)
    want[:, 1::2] *= -1
    experts_ref.close(y, want, U * want.abs(), "sums")


@pytest.mark.parametrize("n", [5, 90])
def test_quantized_on_both_sides(hip, n):
    x, w = whole(n, 100), whole(60, 100, seed=1)
    sx, sw = rand(n, seed=2).abs(), rand(60, seed=3).abs()
    b = rand(60, seed=4, dtype=F16)
    for dtype, bias in ((F32, None), (BF16, None), (F16, b)):
        y = gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(w, sw), bias, dtype=dtype)
        experts_ref.close(y, *ref.quantized_matmul(x, sx, w, sw, bias, dtype), str(dtype))
    lowest = whole(60, 100, low=-128)       # -128 too
    experts_ref.close(gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(lowest, sw)),
                      *ref.quantized_matmul(x, sx, lowest, sw, None, F32), "-128")


@pytest.mark.parametrize("n", [5, 90])
def test_layouts_of_values(hip, n):
    """Whatever lies behind a row's values does not count, and rows that are not whole 16 bytes are copied."""
    d = 75
    x, w = whole(n, d), whole(40, d, seed=1)
    sx, sw = rand(n, seed=2).abs(), rand(40, seed=3).abs()
    want = gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(w, sw))
    experts_ref.close(want, *ref.quantized_matmul(x, sx, w, sw, None, F32), "contiguous")

    def laid(t, ld, first):
        room = torch.full((t.shape[0] * ld + first + 64,), 99, dtype=torch.int8, device=DEV)
        view = room[first:first + t.shape[0] * ld].reshape(t.shape[0], ld)[:, :t.shape[1]]
        view.copy_(t)
        return view

    end = torch.full(((n - 1) * 80 + d,), 99, dtype=torch.int8, device=DEV)       # the last row ends the storage
    end = torch.as_strided(end, (n, d), (80, 1))
    end.copy_(x)
    for a in (laid(x, 80, 0), laid(x, 128, 16), laid(x, 77, 0), laid(x, 96, 5), x.t().contiguous().t(), end):
        for b in (laid(w, 80, 0), laid(w, 160, 32), laid(w, 81, 3), w.t().contiguous().t()):
            assert torch.equal(gmmxx_amd.quantized_matmul(Quantized(a, sx), Quantized(b, sw)), want)
    rows = x[:1].expand(n, d)
    assert torch.equal(gmmxx_amd.quantized_matmul(Quantized(rows, sx[:1].expand(n)), Quantized(w, sw)),
                       want[:1].expand(n, 40))


def test_layouts_of_values_in_tiles(hip):
    n, d, f = 90, 75, 1600
    x, w = whole(n, d), whole(f, d, seed=1)
    sx, sw = rand(n, seed=2).abs(), rand(f, seed=3).abs()
    want = gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(w, sw))
    experts_ref.close(want, *ref.quantized_matmul(x, sx, w, sw, None, F32), "contiguous")
    for ld, first in ((80, 0), (128, 16), (77, 0), (96, 5)):
        views = []
        for t in (x, w):
            room = torch.full((t.shape[0] * ld + first + 64,), 99, dtype=torch.int8, device=DEV)
            views.append(room[first:first + t.shape[0] * ld].reshape(t.shape[0], ld)[:, :d])
            views[-1].copy_(t)
        assert torch.equal(gmmxx_amd.quantized_matmul(Quantized(views[0], sx), Quantized(views[1], sw)), want)


def test_no_rows(hip):
    q = gmmxx_amd.quantize_rows(rand(8, 40))
    assert gmmxx_amd.quantized_matmul(rand(0, 40), q).shape == (0, 8)


def test_past_32_bits(hip):
    """Values and results past 2^32 bytes."""
    d, f = 8192, 600_000                       # 4.9 GB of values
    w = torch.zeros((f, d), dtype=torch.int8, device=DEV)
    w[f - 1, 3], w[f - 1, d - 1] = 2, 3
    ones = torch.ones(f, device=DEV)
    for n in (3, 200):
        x = whole(n, d)
        y = gmmxx_amd.quantized_matmul(Quantized(x, torch.ones(n, device=DEV)), Quantized(w, ones))
        assert torch.equal(y[:, f - 1], 2.0 * x[:, 3] + 3.0 * x[:, d - 1]) and not y[:, :f - 1].any()
    n, d, f = 40_000, 32, 30_000               # 4.8 GB of results
    x = whole(n, d)
    w = whole(f, d, seed=1)
    y = gmmxx_amd.quantized_matmul(Quantized(x, torch.ones(n, device=DEV)), Quantized(w, ones[:f]))
    assert torch.equal(y[-3:], x[-3:].float() @ w.float().t())


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("d", [4, 7, 8, 9, 500, 1000, 4096, 4100, 8192, 16_000, 16_400, 32_768, 40_000])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9])
def test_few_rows(hip, n, d, dtype):
    """Rows that are brought into 8 bits by the product's own workgroups, up to where they are too many or too long."""
    print(f"[int8] few n={n} d={d} {dtype}", flush=True)
    check(n, d, 40, dtype, seed=d)


@pytest.mark.parametrize("n", [4, 30, 100])
def test_other_result_types(hip, n):
    q = gmmxx_amd.quantize_rows(rand(50, 333, seed=1))
    for dtype in experts_ref.DTYPES:
        x = rand(n, 333, dtype=dtype)
        qx, sx = ref.quantize(x)
        for out in experts_ref.DTYPES:
            b = rand(50, seed=2, dtype=out)
            y = gmmxx_amd.quantized_matmul(x, q, b, dtype=out)
            assert y.dtype == out
            experts_ref.close(y, *ref.quantized_matmul(qx, sx, q.values, q.scales, b, out), f"{dtype} {out}")


@pytest.mark.parametrize("n", [1, 2, 4, 7, 20, 100])
def test_rows_of_zeros_and_not_finite(hip, n):
    x, q = rand(n, 300, dtype=F32), gmmxx_amd.quantize_rows(rand(70, 300, seed=1))
    want = gmmxx_amd.quantized_matmul(x, q)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[n // 2, 299] = bad
        y = gmmxx_amd.quantized_matmul(y, q)
        assert torch.isnan(y[n // 2]).all()
        keep = [i for i in range(n) if i != n // 2]
        assert torch.equal(y[keep], want[keep])
    x[n // 2] = 0.0
    y = gmmxx_amd.quantized_matmul(x, q, rand(70, seed=3))
    assert torch.equal(y[n // 2], rand(70, seed=3))
    wide = torch.zeros((n, 411), dtype=F16, device=DEV)
    wide[:, 7:307] = rand(n, 300, dtype=F16)
    assert torch.equal(gmmxx_amd.quantized_matmul(wide[:, 7:307], q), gmmxx_amd.quantized_matmul(rand(n, 300, dtype=F16), q))


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("n,f", [(5, 60), (60, 70), (90, 1600), (300, 4100)])
def test_scales_whose_product_passes_fp32(hip, n, f, dtype):
    """Scales of every size: what counts is the whole product.  Beside scales whose product has fp32's precision a result is
    rounded three times before the bias (the sum, the scales' product, the product); the others are as good."""
    print(f"[int8] scales n={n} f={f} {dtype}", flush=True)
    x, w = whole(n, 96), whole(f, 96, seed=1)
    x[::7], x[3::7] = 0, 1                        # sums of 0, of which a scale makes nothing else
    sx, sw = rand(n, seed=2).abs() + 0.1, rand(f, seed=3).abs() + 0.1
    for i, p in enumerate((100.0, -70.0, 40.0, -120.0, 120.0, -148.0, 124.0)):
        sx[i % n::11] *= 2.0 ** p
    for i, p in enumerate((-75.0, 40.0, -100.0, 120.0, 100.0, -20.0, -140.0)):
        sw[i::13] *= 2.0 ** p
    b = rand(f, seed=4, dtype=dtype)
    for bias in (None, b):
        y = gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(w, sw), bias, dtype=dtype)
        want, _ = ref.quantized_matmul(x, sx, w, sw, bias, dtype)
        prod = (x.cpu().double() @ w.cpu().double().t()) * sx.cpu().double()[:, None] * sw.cpu().double()
        bound = 3 * U * prod.abs() + U * want.abs() + 2.0 ** -149 + ref.rounded(dtype, want)
        # (no result lies so near the border of infinity that fp32's error decides)
        out = prod if bias is None else prod + bias.cpu().double()
        border = torch.finfo(dtype).max * (1 + experts_ref.unit(dtype) / 2)
        assert ((out.abs() / border - 1).abs() > 5 * U).all()
        experts_ref.close(y, want, bound.nan_to_num(0.0, 0.0, 0.0), f"{n} x {f}")


def test_scales_of_other_rows_change_nothing(hip):
    """A row's results are those that it has alone beside scales of any size."""
    for n, f in ((20, 60), (90, 1600)):
        x, w = whole(n, 96), whole(f, 96, seed=1)
        sx, sw = rand(n, seed=2).abs() + 0.1, rand(f, seed=3).abs() + 0.1
        b = rand(f, seed=4)
        want = gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(w, sw), b)
        sx[::3] *= 2.0 ** 100
        sw[5::9] *= 2.0 ** -120
        y = gmmxx_amd.quantized_matmul(Quantized(x, sx), Quantized(w, sw), b)
        rows, cols = torch.arange(n) % 3 != 0, torch.arange(f) % 9 != 5
        assert torch.equal(y.cpu()[rows][:, cols], want.cpu()[rows][:, cols])


@pytest.mark.parametrize("n", [1, 30, 100])
def test_rows_of_any_size(hip, n):
    """Rows and matrices of small and of large numbers, brought into 8 bits on the way."""
    x, w, b = rand(n, 300), rand(70, 300, seed=1), rand(70, seed=3)
    x[::2] *= 2.0 ** 110
    x[1::2] *= 2.0 ** -110
    w[::2] *= 2.0 ** 30
    w[1::2] *= 2.0 ** -60
    x[n // 2] = 0.0
    q = gmmxx_amd.quantize_rows(w)
    qx, sx = ref.quantize(x)
    want, _ = ref.quantized_matmul(qx, sx, q.values, q.scales, b, F32)
    prod = (qx.double() @ q.values.cpu().double().t()) * sx.double()[:, None] * q.scales.cpu().double()
    y = gmmxx_amd.quantized_matmul(x, q, b)
    experts_ref.close(y, want, (3 * U * prod.abs() + U * want.abs() + 2.0 ** -149 + ref.rounded(F32, want)).nan_to_num(0.0, 0.0, 0.0),
                      "rows")
    assert torch.equal(y[n // 2], b)


@pytest.mark.parametrize("n,f", [(1, 20), (30, 20), (200, 20), (20, 4100), (200, 1100), (300, 9000)])
@pytest.mark.parametrize("d", [131_072, 131_071])
def test_longest_sums_of_the_lowest_value(hip, n, d, f):
    """-128 on both sides, as a user's values may have it: a sum of 2^31 at the longest."""
    print(f"[int8] -128 n={n} d={d} f={f}", flush=True)
    x = Quantized(torch.full((n, d), -128, dtype=torch.int8, device=DEV), torch.ones(n, device=DEV))
    w = torch.full((f, d), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    b = torch.full((f,), 5.0, device=DEV)
    y = gmmxx_amd.quantized_matmul(x, Quantized(w, torch.full((f,), 0.5, device=DEV)), b)
    # (the sum, its product and the sum with the bias are rounded)
    want = torch.tensor([8192.0 * d, -8128.0 * d], dtype=torch.float64) + 5.0
    for i in range(2):
        assert ((y[:, i::2].double() - want[i]).abs() <= 3 * U * want[i].abs()).all()
