"""The composed layer's gradients in 16 bits by a bound that a missing term would break, and
the sum's gradients where only one of them is asked for."""

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
N, E, K, D, F = 300, 6, 2, 48, 40


def exact(leaves, dout, pick, gate_has_gradient=True):
    """Result and gradients of the layer in 64 bits for given choices."""
    lv = [t.detach().requires_grad_() for t in leaves]
    var, mean = torch.var_mean(lv[0], dim=1, keepdim=True, unbiased=False)
    h = (lv[0] - mean) / torch.sqrt(var + 1e-5) * lv[1] + lv[2]
    gates = torch.softmax((h @ lv[3]).gather(1, pick), 1)
    if not gate_has_gradient:
        gates = gates.detach()
    out = sum(gates[:, j, None] * (torch.matmul(h[:, None, :], lv[4][pick[:, j]])[:, 0] + lv[5][pick[:, j]])
              for j in range(K))
    return out.detach(), torch.autograd.grad(out, lv, dout, allow_unused=True)


def error(got, want):
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_layer(hip, dtype):
    """Up to eight roundings to the type lie between the inputs and a gradient: of h, y, out, dy, the two parts of dh,
    their sum, and the result.  Each is at most a unit of what it rounds and independent of the others, so in the
    norm they add up as squares, and no term is much larger than the gradients that it is part of: eight units.
    Sums of up to 300 fp32 terms, several in a row, add 64 of fp32's."""
    g = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    base = [make(N, D), 1 + 0.1 * make(D), 0.1 * make(D), make(D, E) / 7, make(E, D, F) / 7, 0.1 * make(E, F)]
    base, dout = [t.to(dtype) for t in base], make(N, F).to(dtype)
    own = [t.to(DEV).requires_grad_() for t in base]
    h = gmmxx_amd.layer_norm(own[0], own[1], own[2])
    r = gmmxx_amd.route_rows(h.float() @ own[3].float(), K)
    out = gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(h, own[4], r, bias=own[5]), r)
    got = torch.autograd.grad(out, own, dout.to(DEV))
    pick = r.experts.cpu().long()
    leaves = [t.double() for t in base]
    want_out, want = exact(leaves, dout.double(), pick)
    bound = 8 * ref.unit(dtype) + 64 * ref.U
    assert error(ref.f64(out), want_out) <= bound
    for name, a, b in zip(("x", "scale", "shift", "gate", "maps", "offsets"), got, want):
        assert error(ref.f64(a), b) <= bound, name
    # what the bound is there to see: without the gate's share the gradient for x would be far off
    assert error(exact(leaves, dout.double(), pick, gate_has_gradient=False)[1][0], want[0]) > 4 * bound


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("k,f", [(1, 40), (2, 100), (4, 512), (6, 37)])
def test_one_gradient_of_the_sum(hip, k, f, dtype):
    """dy or dgates alone has the bits that it has beside the other."""
    g = torch.Generator().manual_seed(f)
    scores = torch.randn((90, 7), generator=g)
    scores[::9] = -float("inf")
    r = gmmxx_amd.route_rows(scores.to(DEV), k)
    y = torch.randn((90 * k, f), generator=g).to(dtype).to(DEV)
    dout = torch.randn((90, f), generator=g).to(dtype).to(DEV)
    both = [y.detach().requires_grad_(), r.gates.detach().requires_grad_()]
    want = torch.autograd.grad(gmmxx_amd.combine_rows(both[0], r, both[1]), both, dout)
    exact_sum = ref.combine(y, r.gates, r.slots, int(r.offsets[-1]), dout)
    for i, name in enumerate(("dy", "dgates")):
        args = [t.detach().requires_grad_(i == j) for j, t in enumerate(both)]
        got, = torch.autograd.grad(gmmxx_amd.combine_rows(args[0], r, args[1]), [args[i]], dout)
        assert torch.equal(got, want[i])
        ref.close(got, *exact_sum[name], name)
