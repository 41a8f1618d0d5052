"""grouped_matmul in 16 bits where its tiles are 256 x 256: forward, for x and for the
weights, both weight layouts, ragged rows, columns and ends of the reduction, uneven and
empty groups, positions without an expert, rows far apart.  Each case first asks the
library's own rule whether it takes these tiles."""

import math
import os
import re

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref
from tests.test_hip_grouped import check, operands, routing

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = (torch.bfloat16, torch.float16)


def rule():
    """larger_tiles() of csrc/grouped.hip, whose expression reads the same in Python."""
    path = os.path.join(os.path.dirname(os.path.abspath(gmmxx_amd.__file__)), "csrc", "grouped.hip")
    text = open(path).read()
    body = re.search(r"bool larger_tiles\(double tiles256, double tiles128\) \{\s*return (.*?);\s*\}", text, re.S)[1]
    return lambda a, b: eval(body, {"ceil": math.ceil, "tiles256": a, "tiles128": b})   # noqa: S307


def tiles(n, size):
    return -(-n // size)


def rows_by_256(m, e, columns):
    return rule()(*((m / s + 0.5 * e) * tiles(columns, s) for s in (256, 128)))


def weights_by_256(e, d, f):
    return rule()(*(e * tiles(d, s) * tiles(f, s) for s in (256, 128)))


def turned(w):
    return w.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("layout", ["columns adjacent", "reduction adjacent"])
@pytest.mark.parametrize("d", [8, 56, 64, 72, 128, 200])
def test_forward(hip, d, layout, dtype):
    n, e, k, f = 4100, 16, 2, 1416
    assert rows_by_256(n * k, e, f)
    x, w, b, dy = operands(n, e, d, f, n * k, dtype, seed=d)
    check(x, w if layout.startswith("columns") else turned(w), b, dy, routing(n, e, k, seed=d, absent=0.1))


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("layout", ["columns adjacent", "reduction adjacent"])
@pytest.mark.parametrize("f", [24, 64, 136, 192, 264])
def test_gradient_for_rows(hip, f, layout, dtype):
    """For x, whose parts are fp32 where a row has several choices."""
    n, e, k, d = 4100, 16, 2, 1416
    assert rows_by_256(n * k, e, d)
    x, w, b, dy = operands(n, e, d, f, n * k, dtype, seed=f)
    check(x, w if layout.startswith("columns") else turned(w), b, dy, routing(n, e, k, seed=f, absent=0.05))


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_offsets(hip, dtype):
    """Groups of one row, whole tiles, one row past a tile, none; the last positions belong to none."""
    sizes = [1, 255, 256, 257, 0, 0, 511, 512, 513, 2, 1000, 1500, 0, 2300, 3, 700]
    m, d, f = 8213, 1400, 1352
    assert sum(sizes) < m - 300 and rows_by_256(m, len(sizes), d) and rows_by_256(m, len(sizes), f)
    ends = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).to(DEV)
    x, w, b, dy = operands(m, len(sizes), d, f, m, dtype, seed=1)
    check(x, w, b, dy, ends)


# every end of a step of 64 positions and of its four products, one step and several
SIZES = [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 79, 81, 95, 96, 97, 111, 127, 128, 129, 160, 191, 192,
         193, 255, 257, 300, 0, 450]


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("d,f", [(1000, 504), (776, 512), (504, 1000)])
def test_gradient_for_weights(hip, d, f, dtype):
    assert weights_by_256(len(SIZES), d, f)
    ends = torch.tensor([0] + SIZES).cumsum(0)
    m = int(ends[-1]) + 70
    x, w, b, dy = operands(m, len(SIZES), d, f, m, dtype, seed=d)
    check(x, w, b, dy, ends.to(DEV))


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_gradient_for_weights_of_a_routing(hip, dtype):
    n, e, k, d, f = 1500, 32, 2, 1000, 504
    assert weights_by_256(e, d, f)
    x, w, b, dy = operands(n, e, d, f, n * k, dtype, seed=5)
    check(x, w, b, dy, routing(n, e, k, seed=5, absent=0.1))


@pytest.mark.parametrize("layout", ["columns adjacent", "reduction adjacent"])
def test_rows_far_apart(hip, layout):
    """Rows that begin past 2^32 bytes: other offsets, the same products."""
    n, e, d, f, apart = 8300, 8, 1000, 1416, 1 << 18
    assert rows_by_256(n, e, f) and weights_by_256(32, 1000, 504)
    store = torch.empty((n, apart), dtype=torch.bfloat16, device=DEV)
    x, w, b, _ = operands(n, e, d, f, n, torch.bfloat16, seed=6)
    if layout.startswith("reduction"):
        w = turned(w)
    far = store[:, :d]
    far.copy_(x)
    r = routing(n, e, 1, seed=6)
    assert torch.equal(gmmxx_amd.grouped_matmul(far, w, r, bias=b), gmmxx_amd.grouped_matmul(x, w, r, bias=b))
    r = routing(n, 32, 1, seed=7)
    w, dy = operands(1, 32, d, 504, n, torch.bfloat16, seed=7)[1::2]
    grads = []
    for rows in (far, x):
        leaf = w.detach().requires_grad_()
        grads += torch.autograd.grad(gmmxx_amd.grouped_matmul(rows, leaf, r), leaf, dy)
    assert torch.equal(*grads)
    ref.close(grads[1][5:6], *(t[5:6] for t in ref.grouped(x, w, None, r.offsets, r.rows, r.slots, dy)["dw"]), "dw")
