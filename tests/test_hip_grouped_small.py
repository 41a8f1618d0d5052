"""grouped_matmul in fp32 with groups of few rows, whose tiles are wide and low: every end
of the reduction within a step, ragged columns, both weight layouts, empty and full tiles,
rows far apart; the bias's gradient alone."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref
from tests.test_hip_grouped import check, operands, routing

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("f", [4, 77, 252, 256, 260, 600])
@pytest.mark.parametrize("d", [4, 31, 32, 33, 36, 41, 68, 100, 128])
def test_ends(hip, d, f):
    x, w, b, dy = operands(200, 20, d, f, 400, torch.float32, seed=d + f)
    check(x, w, b, dy, routing(200, 20, 2, seed=d))


@pytest.mark.parametrize("ends", [[0, 1, 33, 33, 65, 96, 128, 191, 200], [0, 0, 0, 0, 0, 0, 0, 0, 130],
                                  [0, 32, 64, 96, 128, 160, 192, 224, 256], [0, 31, 31, 62, 93, 93, 124, 155, 155]],
                         ids=str)
@pytest.mark.parametrize("d,f", [(64, 256), (50, 130)])
def test_groups(hip, ends, d, f):
    m = max(ends[-1], 140)           # (past the last group: zeros)
    x, w, b, dy = operands(m, 8, d, f, m, torch.float32, seed=3)
    check(x, w, b, dy, torch.tensor(ends, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("d,f", [(64, 256), (37, 300)])
def test_transposed_weights(hip, d, f):
    x, w, b, dy = operands(150, 12, d, f, 300, torch.float32, seed=4)
    check(x, w.transpose(1, 2).contiguous().transpose(1, 2), b, dy, routing(150, 12, 2, seed=1, absent=0.1))


@pytest.mark.parametrize("e", [64, 2], ids=["small groups", "large groups"])
def test_rows_far_apart(hip, e):
    """Rows of fp32 that begin past 2^32 bytes."""
    n, d, f, apart = 1100, 64, 256, 1 << 20
    store = torch.empty((n, apart), device=DEV)
    x, w, b, _ = operands(n, e, d, f, n, torch.float32, seed=5)
    far = store[:, :d]
    far.copy_(x)
    r = routing(n, e, 1, seed=6)
    assert torch.equal(gmmxx_amd.grouped_matmul(far, w, r, bias=b), gmmxx_amd.grouped_matmul(x, w, r, bias=b))


def test_bias_gradient_alone(hip):
    for dtype in ref.DTYPES:
        x, w, b, dy = operands(300, 5, 64, 72, 600, dtype, seed=7)
        r = routing(300, 5, 2, seed=8)
        leaf = b.detach().requires_grad_()
        got, = torch.autograd.grad(gmmxx_amd.grouped_matmul(x, w, r, bias=leaf), leaf, dy)
        ref.close(got, *ref.grouped(x, w, b, r.offsets, r.rows, r.slots, dy)["db"], "db")
