"""dropout against its definition: the generator's published words, masks that are the same in every type,
layout and direction, all probabilities, and its gradients."""

import numpy as np
import pytest
import torch

import gmmxx_amd
from tests import experts_ref, tokens_ref as ref

DEV = "cuda:0"
F32, BF16, F16 = experts_ref.DTYPES
gpu = pytest.mark.gpu


def rand(*shape, seed=0, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def test_published_words():
    """The generator's known answers (counter, key, words), for the reference that the others compare with."""
    one = lambda *c: [np.array([v], dtype=np.uint64) for v in c]      # noqa: E731
    ones = 0xFFFFFFFF
    for counter, key, words in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(ref._philox(one(*counter), list(key)).tolist()) == words


@gpu
@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("n", [1, 3, 4, 5, 7, 8, 9, 255, 2047, 2048, 2049, 100_003])
def test_counts(hip, n, dtype):
    print(f"[dropout] n={n} {dtype}", flush=True)
    x, r, dy = rand(n, seed=1, dtype=dtype), rand(n, seed=2, dtype=dtype), rand(n, seed=3, dtype=dtype)
    for residual in (None, r):
        leaves = [t.detach().requires_grad_() for t in (x, residual) if t is not None]
        y = gmmxx_amd.dropout(leaves[0], 0.3, 1234567890123456789, offset=77,
                              residual=leaves[1] if residual is not None else None)
        grads = torch.autograd.grad(y, leaves, dy)
        want, bound, keep = ref.dropout(x, 0.3, 1234567890123456789, 77, residual)
        experts_ref.close(y, want, bound, "y")
        want, bound, _ = ref.dropout(dy, 0.3, 1234567890123456789, 77)
        experts_ref.close(grads[0], want, bound, "dx")
        assert torch.equal(grads[0].cpu() != 0, keep & (dy.cpu() != 0))
        if residual is not None:
            assert torch.equal(grads[1], dy)


@gpu
@pytest.mark.parametrize("p", [0.0, 2.0 ** -33, 2.0 ** -32, 1e-6, 0.1, 0.5, 0.999, 1.0 - 2.0 ** -32, 1.0 - 2.0 ** -34, 1.0])
def test_probabilities(hip, p):
    x = rand(40_000)
    y = gmmxx_amd.dropout(x, p, 5)
    want, bound, keep = ref.dropout(x, p, 5)
    if round(p * 2.0 ** 32) == 2 ** 32:
        assert not y.any()
    else:
        experts_ref.close(y, want, bound, "y")
        assert torch.equal((y != 0).cpu(), keep)
    if p == 0.0:
        assert torch.equal(y, x)


@gpu
def test_share(hip):
    """The share of kept elements: within five standard deviations."""
    n = 1 << 22
    for p in (0.1, 0.5, 0.9):
        kept = int((gmmxx_amd.dropout(torch.ones(n, device=DEV), p, 99) != 0).sum())
        assert abs(kept - n * (1 - p)) < 5 * (n * p * (1 - p)) ** 0.5


@gpu
def test_one_mask_for_types_and_layouts(hip):
    x = torch.ones((60, 35), device=DEV)
    want = gmmxx_amd.dropout(x, 0.5, 3) != 0
    for t in (x.bfloat16(), x.half(), x.t().contiguous().t(), torch.ones((60, 70), device=DEV)[:, ::2]):
        assert torch.equal(gmmxx_amd.dropout(t, 0.5, 3) != 0, want)
    room = torch.ones(2101, device=DEV)
    assert torch.equal((gmmxx_amd.dropout(room[1:], 0.5, 3) != 0).reshape(60, 35), want)       # 4 bytes off
    half = torch.ones(2101, device=DEV, dtype=F16)
    assert torch.equal((gmmxx_amd.dropout(half[1:], 0.5, 3, residual=half[1:]) > 1).reshape(60, 35), want)


@gpu
@pytest.mark.parametrize("seed", [0, -1, (1 << 63) - 1, -(1 << 63), (1 << 64) - 1])
@pytest.mark.parametrize("offset", [0, 1, 1 << 32, (1 << 63) - 1])
def test_seeds(hip, seed, offset):
    x = torch.ones(1000, device=DEV)
    y = gmmxx_amd.dropout(x, 0.5, seed, offset=offset)
    keep = torch.from_numpy(ref.words(1000, seed % (1 << 64), offset) >= np.uint64(1 << 31))
    assert torch.equal((y != 0).cpu(), keep)
    if seed < 1 << 63:
        at = torch.tensor([seed], device=DEV)
        assert torch.equal(gmmxx_amd.dropout(x, 0.5, at, offset=offset), y)


@gpu
def test_seed_that_changes_before_the_backward_pass(hip):
    seed = torch.tensor(4, device=DEV)
    x = rand(100).requires_grad_()
    y = gmmxx_amd.dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_dropped_values_that_are_not_finite(hip):
    x = rand(4096)
    keep = ref.dropout(x, 0.5, 8)[2].to(DEV)
    x[~keep] = float("nan")
    assert torch.isfinite(gmmxx_amd.dropout(x, 0.5, 8)).all()
    x = torch.full((10,), float("inf"), device=DEV)
    assert not gmmxx_amd.dropout(x, 1.0, 8).any()
    r = rand(10)
    assert torch.equal(gmmxx_amd.dropout(x, 1.0, 8, residual=r), r)


@gpu
def test_shapes(hip):
    assert gmmxx_amd.dropout(rand(0, 5), 0.5, 1).shape == (0, 5)
    assert gmmxx_amd.dropout(rand(1)[0], 0.0, 1).shape == ()
    x = rand(2, 3, 50)
    assert torch.equal(gmmxx_amd.dropout(x, 0.4, 1).reshape(-1), gmmxx_amd.dropout(x.reshape(-1), 0.4, 1))
    leaf = x.requires_grad_()
    gmmxx_amd.dropout(leaf, 0.4, 1).sum().backward()        # a gradient with strides of zero
    assert torch.equal(leaf.grad != 0, gmmxx_amd.dropout(torch.ones_like(x), 0.4, 1) != 0)


@gpu
def test_past_32_bits(hip):
    """Elements from 2^32 on: the counter's second word, and bytes past 2^32."""
    n = (1 << 34) + 12
    x = torch.ones(n, dtype=BF16, device=DEV)
    y = gmmxx_amd.dropout(x, 0.5, 21)
    low = np.uint64(0xFFFFFFFF)
    for first in (0, 1 << 32, 1 << 34):
        i = np.arange(first // 4, first // 4 + 3, dtype=np.uint64)
        zero = np.zeros_like(i)
        w = ref._philox([i & low, i >> np.uint64(32), zero, zero], [21, 0])
        assert torch.equal((y[first:first + 12] != 0).cpu(), torch.from_numpy(w >= np.uint64(1 << 31)))
