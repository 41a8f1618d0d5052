"""layer_norm against its definition in 64 bits: widths around every group size, odd
widths and strides, rows whose mean is large beside their spread, non-finite rows, and
its gradients against the formulas and against differences."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(n, d, dtype, seed=0, ptype=None, spread=1.0, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn((n, d), generator=g) + offset * torch.randn((n, 1), generator=g)).to(dtype)
    w = (1.0 + 0.2 * torch.randn(d, generator=g)).to(ptype or dtype)
    b = (0.2 * torch.randn(d, generator=g)).to(ptype or dtype)
    dy = torch.randn((n, d), generator=g).to(dtype)
    return tuple(t.to(DEV) for t in (x, w, b, dy))


def check(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = gmmxx_amd.layer_norm(*leaves, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    want = ref.norm(x, w, b, eps, dy)
    ref.close(y, *want["y"], "y")
    names = [nm for nm, t in zip(("dx", "dw", "db"), leaves) if t is not None]
    for nm, got in zip(names, grads):
        ref.close(got, *want[nm], nm)
    plain = gmmxx_amd.layer_norm(x, w, b, eps=eps)
    assert torch.equal(plain, y.detach())


# every group size, one element less and more; one column; the widest
WIDTHS = [1, 2, 7, 8, 16, 100, 127, 128, 129, 255, 256, 257, 512, 513, 1000, 1024, 1025, 4096, 4097, 8192, 8193, 20001,
          65536]


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("d", WIDTHS)
def test_widths(hip, d, dtype):
    print(f"[layer_norm] d={d} {dtype}", flush=True)
    check(*make(5, d, dtype, seed=d))


@pytest.mark.parametrize("n", [1, 2, 31, 33, 257, 1025, 5000])
@pytest.mark.parametrize("d,dtype", [(24, torch.float32), (100, torch.bfloat16), (1100, torch.float16)])
def test_rows(hip, n, d, dtype):
    check(*make(n, d, dtype, seed=n))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16), ids=str)
def test_fp32_parameters(hip, dtype):
    check(*make(9, 200, dtype, ptype=torch.float32))


@pytest.mark.parametrize("which", ["neither", "weight", "bias"])
def test_without_parameters(hip, which):
    x, w, b, dy = make(17, 70, torch.float32)
    check(x, w if which == "weight" else None, b if which == "bias" else None, dy)


def test_mean_beside_spread(hip):
    # mean 1000, spread 1: E[x²] - E[x]² would keep one digit of the variance
    check(*make(40, 300, torch.float32, offset=1000.0))


def test_constant_rows(hip):
    x = torch.full((3, 64), 2.5, device=DEV)
    y = gmmxx_amd.layer_norm(x, eps=1e-5)
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_strides(hip, dtype):
    x, w, b, dy = make(12, 150, dtype)
    wide = torch.zeros((12, 200), dtype=dtype, device=DEV)
    wide[:, 33:183] = x
    wide_dy = torch.zeros((12, 171), dtype=dtype, device=DEV)
    wide_dy[:, 5:155] = dy
    check(wide[:, 33:183], w, b, wide_dy[:, 5:155])          # odd starts, row strides that are no multiple of 16 bytes
    check(x.t().contiguous().t(), w, b, dy)                  # columns adjacent instead
    every = torch.zeros(300, dtype=w.dtype, device=DEV)
    every[::2] = w
    check(x, every[::2], b, dy)


def test_leading_dimensions(hip):
    x, w, b, dy = make(24, 50, torch.float32)
    y = gmmxx_amd.layer_norm(x.reshape(2, 3, 4, 50), w, b)
    assert torch.equal(y.reshape(24, 50), gmmxx_amd.layer_norm(x, w, b))
    assert torch.equal(gmmxx_amd.layer_norm(x[0], w, b), y.reshape(24, 50)[0])


def test_broadcast_gradient(hip):
    x, w, b, _ = make(6, 40, torch.float32)
    leaf = x.requires_grad_()
    gmmxx_amd.layer_norm(leaf, w, b).sum().backward()        # dy with strides of zero
    ref.close(leaf.grad, *ref.norm(x, w, b, 1e-5, torch.ones(6, 40))["dx"], "dx")


def test_no_rows(hip):
    x, w, b, dy = make(3, 20, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x[:0], w, b)]
    y = gmmxx_amd.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy[:0])
    assert y.shape == dx.shape == (0, 20)
    assert not dw.any() and not db.any()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_row_that_is_not_finite(hip, bad):
    x, w, b, _ = make(8, 90, torch.float32)
    want = gmmxx_amd.layer_norm(x, w, b)
    x[3, 17] = bad
    y = gmmxx_amd.layer_norm(x, w, b)
    assert torch.isnan(y[3]).any()
    keep = [0, 1, 2, 4, 5, 6, 7]
    assert torch.equal(y[keep], want[keep])


def test_differences(hip):
    x, w, b, dy = make(7, 33, torch.float32, seed=3)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(gmmxx_amd.layer_norm(*leaves), leaves, dy)
    g = torch.Generator().manual_seed(9)
    h = 2.0 ** -7
    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=g).to(DEV)
        ends = []
        for sign in (1, -1):
            args = [t.detach() for t in leaves]
            args[i] = args[i] + sign * h * v
            ends.append((ref.f64(gmmxx_amd.layer_norm(*args)) * ref.f64(dy)).sum())
        slope = float(ends[0] - ends[1]) / (2 * h)
        want = float((ref.f64(grads[i]) * ref.f64(v)).sum())
        scale = float((ref.f64(grads[i]) * ref.f64(v)).abs().sum())
        # third derivatives times h² / 6 (h = 2^-7: 1e-5 of O(1) terms), rounding of y over h: 231 · 2^-24 / h
        assert abs(slope - want) <= 1e-3 * scale + 231 * ref.U / h


def test_same_bits_again(hip):
    x, w, b, dy = make(3000, 100, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    runs = [torch.autograd.grad(gmmxx_amd.layer_norm(*leaves), leaves, dy) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r, runs[0]))


def test_another_stream(hip):
    x, w, b, dy = make(2000, 256, torch.float32)
    want = gmmxx_amd.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = gmmxx_amd.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)


def test_refusals(hip):
    x, w, b, _ = make(4, 10, torch.float32)
    f = gmmxx_amd.layer_norm
    for err, call in [
        (TypeError, lambda: f([1.0])),
        (ValueError, lambda: f(x.cpu())),
        (TypeError, lambda: f(x.double())),
        (TypeError, lambda: f(x.int())),
        (ValueError, lambda: f(x[:, :0])),
        (ValueError, lambda: f(torch.zeros((1, 65537), device=DEV))),
        (ValueError, lambda: f(x, w[:9])),
        (ValueError, lambda: f(x, w.reshape(1, 10))),
        (TypeError, lambda: f(x, w.bfloat16())),
        (TypeError, lambda: f(x.bfloat16(), w.bfloat16(), b)),
        (TypeError, lambda: f(x.bfloat16(), w.half())),
        (ValueError, lambda: f(x, w.cpu())),
        (ValueError, lambda: f(x, w, b, eps=-1.0)),
        (ValueError, lambda: f(x, w, b, eps=float("nan"))),
    ]:
        with pytest.raises(err):
            call()
