"""The sparsely gated layer's operators beyond single calls: what autograd asks of them,
other streams, captured graphs, arrays past 2^31 elements and 2^32 bytes, and the
example that runs them together."""

import os
import sys

import pytest
import torch

import gmmxx_amd
from tests import experts_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(*shape, seed=0, dtype=torch.float32, grad=False):
    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    return t.requires_grad_() if grad else t


def layer(x, scale, shift, gate, maps, bias, k=2):
    h = gmmxx_amd.layer_norm(x, scale, shift)
    r = gmmxx_amd.route_rows(h @ gate, k)
    return gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(h, maps, r, bias=bias), r)


def parameters(d=64, e=5, f=40, dtype=torch.float32, grad=False):
    return [rand(*s, seed=i, dtype=dtype, grad=grad) for i, s in
            enumerate([(d,), (d,), (d, e), (e, d, f), (e, f)])]


def test_differentiable_once(hip):
    x = rand(20, 64, grad=True)
    p = parameters(grad=True)
    g, = torch.autograd.grad(layer(x, *p).sum(), x, create_graph=True)
    assert torch.isfinite(g).all()
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


def test_gradients_of_some_inputs(hip):
    x, (scale, shift, gate, maps, bias) = rand(30, 64), parameters()
    r = gmmxx_amd.route_rows(rand(30, 5, seed=9), 2)
    full = [t.detach().requires_grad_() for t in (x, maps, bias)]
    dy = rand(60, 40, seed=11)
    want = torch.autograd.grad(gmmxx_amd.grouped_matmul(full[0], full[1], r, bias=full[2]), full, dy)
    for some in ((0,), (1,), (2,), (0, 2), (1, 2)):
        args = [t.detach().requires_grad_(i in some) for i, t in enumerate((x, maps, bias))]
        y = gmmxx_amd.grouped_matmul(args[0], args[1], r, bias=args[2])
        got = torch.autograd.grad(y, [args[i] for i in some], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, some))
    leaves = [t.detach().requires_grad_() for t in (x, scale, shift)]
    want = torch.autograd.grad(gmmxx_amd.layer_norm(*leaves), leaves, rand(30, 64, seed=12))
    for i in range(3):
        args = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, scale, shift))]
        got, = torch.autograd.grad(gmmxx_amd.layer_norm(*args), [args[i]], rand(30, 64, seed=12))
        assert torch.equal(got, want[i])
    y, gates = rand(60, 40, seed=13), r.gates
    for i in range(2):
        args = [t.detach().requires_grad_(i == j) for j, t in enumerate((y, gates))]
        got, = torch.autograd.grad(gmmxx_amd.combine_rows(args[0], r, args[1]).sum(), [args[i]])
        assert torch.isfinite(got).all()


def test_a_choice_that_is_not_used(hip):
    """Gradients through the integer outputs do not exist; unused gates have none to give."""
    s = rand(12, 6, grad=True)
    r = gmmxx_amd.route_rows(s, 2)
    assert r.gates.requires_grad and not r.experts.requires_grad and not r.slots.requires_grad
    y = gmmxx_amd.grouped_matmul(rand(12, 64, grad=True), parameters(e=6)[3], r)
    y.sum().backward()
    assert s.grad is None


def test_no_grad(hip):
    x, p = rand(10, 64, grad=True), parameters(grad=True)
    with torch.no_grad():
        assert not layer(x, *p).requires_grad
    with torch.inference_mode():
        out = layer(x, *p)
    assert torch.equal(out, layer(x, *p).detach())


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_other_streams(hip, dtype):
    """A layer and its gradients on a stream of its own, workspaces included, beside other work."""
    x = rand(3000, 64, dtype=dtype)
    p = parameters(dtype=dtype)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, *p)]
        out = layer(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))]

    want = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_captured_graph(hip):
    """The operators hold no host state: a captured layer gives the eager results on every replay, new inputs
    included."""
    p = parameters(dtype=torch.bfloat16)
    x = rand(500, 64, dtype=torch.bfloat16)

    def run(x):
        h = gmmxx_amd.layer_norm(x, p[0], p[1])
        r = gmmxx_amd.route_rows(h[:, :5], 2)
        return gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(h, p[3], r, bias=p[4]), r), r.offsets

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        out, offsets = run(static)
    for seed in range(5):
        fresh = rand(500, 64, seed=seed, dtype=torch.bfloat16)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want, want_offsets = run(fresh)
        assert torch.equal(out, want) and torch.equal(offsets, want_offsets)
        torch.zeros(1000, device=DEV).sum().item()


def test_past_32_bits(hip):
    """2.3e9 elements, 4.6 GB: offsets past 2^31 elements and 2^32 bytes, at the far rows."""
    n, d, f, e = 1_120_000, 2056, 64, 3
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty((n, d), dtype=torch.bfloat16, device=DEV)
    for i in range(0, n, 140_000):
        x[i:i + 140_000].normal_(generator=g)
    far = torch.tensor([0, 1, n // 2, n - 2, n - 1])
    y = gmmxx_amd.layer_norm(x)
    ref.close(y[far], *ref.norm(x[far], None, None, 1e-5)["y"], "layer_norm")
    del y
    r = gmmxx_amd.route_rows(x[:, :e], 1)
    w = (torch.randn((e, d, f), generator=g, device=DEV) / 45).to(torch.bfloat16)
    out = gmmxx_amd.grouped_matmul(x, w, r)
    pick = r.experts[far, 0].cpu().long()
    for i, row in enumerate(far.tolist()):
        xr, wr = ref.f64(x[row]), ref.f64(w[pick[i]])
        want = xr @ wr
        bound = (d + 2) * ref.U * (xr.abs() @ wr.abs()) + ref.unit(torch.bfloat16) * want.abs() * 1.01
        ref.close(out[int(r.slots[row, 0])], want, bound, f"row {row}")
    # the weight's gradient reads every row: one column of dy for each of a few rows counts them
    dy = torch.zeros((n, f), dtype=torch.bfloat16, device=DEV)
    for i, row in enumerate(far.tolist()):
        dy[int(r.slots[row, 0]), i] = 1.0
    wl = w.detach().requires_grad_()
    dw, = torch.autograd.grad(gmmxx_amd.grouped_matmul(x, wl, r), wl, dy)
    for i, row in enumerate(far.tolist()):
        assert torch.equal(dw[int(pick[i]), :, i], x[row])
    del dy, out
    # combination of as many elements
    back = gmmxx_amd.combine_rows(x, gmmxx_amd.Routing(r.experts, r.gates, r.offsets, r.rows, r.slots))
    assert torch.equal(back[far], x[r.slots[far, 0].long()])


def test_weights_past_32_bits(hip):
    """Experts whose matrices begin past 2^32 bytes."""
    e, d, f = 40, 8192, 8192                     # 5.4 GB of bf16
    w = torch.zeros((e, d, f), dtype=torch.bfloat16, device=DEV)
    w[e - 1, 5, 7] = 2.0
    w[e - 1, d - 1, f - 1] = 3.0
    x = rand(300, d, dtype=torch.bfloat16)
    ends = torch.full((e + 1,), 0, dtype=torch.int32, device=DEV)
    ends[e] = 300
    y = gmmxx_amd.grouped_matmul(x, w, ends)
    assert torch.equal(y[:, 7], 2 * x[:, 5]) and torch.equal(y[:, f - 1], 3 * x[:, d - 1])
    assert int((y != 0).any(0).sum()) == 2
    few = torch.zeros_like(ends)
    few[e] = 3
    assert torch.equal(gmmxx_amd.grouped_matmul(x[:3], w, few), y[:3])


def test_example(hip):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")
    sys.path.insert(0, path)
    try:
        import local_experts
    finally:
        sys.path.remove(path)
    errors, trained, x = local_experts.run(rows=4000, width=16, outputs=8, clusters=5, steps=60)
    assert errors[-1] < 0.2 * errors[0]
    with torch.no_grad():
        many, one = trained(x[:64]), trained(x[7:8])
    # one row alone takes other kernels: the same sums in another order, of 16 terms
    assert torch.allclose(one, many[7:8], rtol=1e-4, atol=1e-4)
