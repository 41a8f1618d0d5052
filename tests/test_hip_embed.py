"""embed_rows against its definition in 64 bits: widths, counts and tokens at which the lookup, the
sort and the sums change their ways, tokens outside the table, strides and types."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref, tokens_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = experts_ref.DTYPES


def make(n, v, d, dtype, seed=0, kind="skewed", index_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    table, dy = torch.randn((v, d), generator=g).to(dtype), torch.randn((n, d), generator=g).to(dtype)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    if kind == "skewed":
        index = torch.floor((v + 1.0) ** u - 1.0).long().clamp_(0, v - 1)
    elif kind == "uniform":
        index = torch.floor(u * v).long()
    elif kind == "one":
        index = torch.full((n,), v // 2)
    elif kind == "none":
        index = torch.full((n,), -1)
    else:                                # a fifth outside, at both ends
        index = torch.floor(u * v * 1.25 - v * 0.125).long()
    return table.to(DEV), index.to(index_dtype).to(DEV), dy.to(DEV)


def check(table, index, dy, scale=1.0):
    leaf = table.detach().requires_grad_()
    y = gmmxx_amd.embed_rows(leaf, index, scale=scale)
    assert y.dtype == table.dtype and y.shape == (*index.shape, table.shape[1])
    dtable, = torch.autograd.grad(y, leaf, dy.reshape(y.shape) if dy.is_contiguous() else dy)
    want = ref.embed(table, index, scale, dy)
    experts_ref.close(y, *want["out"], "out")
    experts_ref.close(dtable, *want["dtable"], "dtable")
    with torch.no_grad():
        assert torch.equal(gmmxx_amd.embed_rows(leaf, index, scale=scale), y)
    again, = torch.autograd.grad(gmmxx_amd.embed_rows(leaf, index, scale=scale), leaf, dy.reshape(y.shape))
    assert torch.equal(again, dtable)


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("d", [1, 2, 3, 7, 8, 9, 31, 64, 100, 255, 257, 1000, 2048, 2056, 4100])
def test_widths(hip, d, dtype):
    print(f"[embed] d={d} {dtype}", flush=True)
    check(*make(200, 50, d, dtype, seed=d), scale=0.37)


@pytest.mark.parametrize("kind", ["skewed", "uniform", "one", "none", "outside"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 257, 2047, 2049, 5000, 20011])
def test_counts(hip, n, kind):
    print(f"[embed] n={n} {kind}", flush=True)
    check(*make(n, 300, 40, BF16, seed=n, kind=kind))


@pytest.mark.parametrize("v", [1, 2, 3, 63, 64, 65, 255, 256, 2047, 2048, 4095, 4097, 65535, 65536, 300000])
@pytest.mark.parametrize("kind", ["skewed", "outside"])
def test_tables(hip, v, kind):
    """Every number of passes and digits of the sort; rows that no token has."""
    print(f"[embed] v={v} {kind}", flush=True)
    check(*make(3001, v, 12, F32, seed=v, kind=kind), scale=2.0)


@pytest.mark.parametrize("v", [(1 << 18) - 1, 1 << 18, (1 << 18) + 1, 700_001])
@pytest.mark.parametrize("n", [1, 1024, 1025, 2048, 2049])
def test_few_tokens_of_large_tables(hip, n, v):
    """Both sides of the size from which workgroups do nothing but clear marks."""
    print(f"[embed] n={n} v={v}", flush=True)
    check(*make(n, v, 5, F32, seed=n, kind="outside"))


def test_largest_table(hip):
    """Tokens of 24 bits."""
    v = 1 << 24
    table = torch.zeros((v, 8), dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(0)
    index = torch.randint(0, v, (70_001,), generator=g)
    index[::1000] = v - 1
    index[1::1000] = 0
    index[2::1000] = v
    dy = torch.randint(-2, 3, (70_001, 8), generator=g).to(BF16)
    leaf = table.requires_grad_()
    y = gmmxx_amd.embed_rows(leaf, index.to(DEV))
    dtable, = torch.autograd.grad(y, leaf, dy.to(DEV))
    there = index < v
    want = torch.zeros((v, 8)).index_add_(0, index[there], dy[there].float())       # whole numbers: exact in any order
    assert torch.equal(dtable.float().cpu(), want)


@pytest.mark.parametrize("n", [40_000, 150_000, 300_017])
def test_long_runs(hip, n):
    """One token in most places: a run over thousands of tiles, in whole numbers."""
    g = torch.Generator().manual_seed(n)
    index = torch.where(torch.rand(n, generator=g) < 0.9, 7, torch.randint(0, 20, (n,), generator=g))
    dy = torch.randint(-1, 2, (n, 100), generator=g).float()
    leaf = torch.zeros((20, 100), device=DEV, requires_grad=True)
    dtable, = torch.autograd.grad(gmmxx_amd.embed_rows(leaf, index.to(DEV)), leaf, dy.to(DEV))
    assert torch.equal(dtable.cpu(), torch.zeros((20, 100)).index_add_(0, index, dy))


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
def test_strides_and_types(hip, dtype):
    table, index, dy = make(130, 40, 70, dtype, kind="outside", index_dtype=torch.int32)
    wide = torch.full((40, 100), 7.0, dtype=dtype, device=DEV)
    wide[:, 13:83] = table
    wide_dy = torch.full((130, 91), 7.0, dtype=dtype, device=DEV)
    wide_dy[:, 5:75] = dy
    check(wide[:, 13:83], index, wide_dy[:, 5:75])
    check(table.t().contiguous().t(), index, dy)
    every = torch.stack([index, index + 1], 1)[:, 0]
    assert not every.is_contiguous()
    check(table, every, dy)
    check(table, index.reshape(2, 5, 13), dy)
    check(table, index[:1].reshape(()), dy[:1])


def test_broadcast_gradient(hip):
    table, index, _ = make(50, 9, 24, F32)
    leaf = table.requires_grad_()
    gmmxx_amd.embed_rows(leaf, index).sum().backward()
    want = ref.embed(table, index, 1.0, torch.ones(50, 24))["dtable"]
    experts_ref.close(leaf.grad, *want, "dtable")


def test_no_places(hip):
    table, index, dy = make(4, 9, 24, F16)
    leaf = table.requires_grad_()
    y = gmmxx_amd.embed_rows(leaf, index[:0])
    assert y.shape == (0, 24)
    dtable, = torch.autograd.grad(y, leaf, dy[:0])
    assert dtable.shape == (9, 24) and not dtable.any()


def test_values_that_are_not_finite(hip):
    table, index, dy = make(40, 9, 24, F32, kind="uniform")
    table[3] = float("nan")
    index[index == 3] = 4
    index[::7] = -1
    assert torch.isfinite(gmmxx_amd.embed_rows(table, index)).all()
    dy[::7] = float("inf")                     # at places without a token
    leaf = table.requires_grad_()
    dtable, = torch.autograd.grad(gmmxx_amd.embed_rows(leaf, index), leaf, dy)
    assert torch.isfinite(dtable).all()
    index[0] = 3
    assert torch.isnan(gmmxx_amd.embed_rows(table, index)[0]).all()


def test_routing_as_tokens(hip):
    """A row for each expert that a row of scores goes to; a choice without an expert has none."""
    scores = torch.full((3, 4), float("-inf"), device=DEV)
    scores[0, 2], scores[1, :] = 1.0, torch.arange(4.0)
    r = gmmxx_amd.route_rows(scores, 2)
    table = torch.arange(1.0, 13.0, device=DEV).reshape(4, 3)
    y = gmmxx_amd.embed_rows(table, r.experts)
    assert torch.equal(y[0, 0], table[2]) and torch.equal(y[1], table[[3, 2]])
    assert not y[0, 1].any() and not y[2].any()


def test_past_32_bits(hip):
    """A table and places past 2^32 bytes and 2^31 elements."""
    v, d = 1_100_000, 2056
    table = torch.empty((v, d), dtype=BF16, device=DEV)
    for i in range(0, v, 100_000):
        table[i:i + 100_000].normal_()
    index = torch.tensor([v - 1, 0, v - 2, v // 2, v], device=DEV)
    y = gmmxx_amd.embed_rows(table, index)
    assert torch.equal(y[:4], table[index[:4]]) and not y[4].any()
    leaf = table.detach().requires_grad_()
    dy = torch.ones((5, d), dtype=BF16, device=DEV)
    dtable, = torch.autograd.grad(gmmxx_amd.embed_rows(leaf, index), leaf, dy)
    rows = dtable.any(1).nonzero()[:, 0].tolist()
    assert rows == [0, v // 2, v - 2, v - 1] and torch.equal(dtable[rows], dy[:4])


@pytest.mark.parametrize("v", [1, 3, 255, 511, 512, 1023, 2047, 2048, 4095, 65_535, 1 << 20, (1 << 21) - 1, (1 << 22) - 1, 1 << 22])
@pytest.mark.parametrize("n", [2047, 2048, 2049, 4097, 20_001, 32_768, 32_769, 34_000])
def test_sorts(hip, n, v):
    """Every width of the sort's digits, with one workgroup, few and many: whole numbers, exact in any order."""
    print(f"[embed] sort n={n} v={v}", flush=True)
    g = torch.Generator().manual_seed(v)
    index = torch.floor((v + 1.0) ** torch.rand(n, generator=g, dtype=torch.float64) - 1.0).long().clamp_(0, v - 1)
    index[::9] = torch.randint(0, v, (index[::9].numel(),), generator=g)
    index[4::50] = v
    index[5::50] = -7
    index[-1] = v - 1
    dy = torch.randint(-3, 4, (n, 4), generator=g).float()
    leaf = torch.zeros((v, 4), device=DEV, requires_grad=True)
    dtable, = torch.autograd.grad(gmmxx_amd.embed_rows(leaf, index.to(DEV)), leaf, dy.to(DEV))
    there = (index >= 0) & (index < v)
    assert torch.equal(dtable.cpu(), torch.zeros((v, 4)).index_add_(0, index[there], dy[there]))
