"""The token operators together, as a model uses them: what autograd asks of them, other streams, captured graphs,
and the example."""

import os
import sys

import pytest
import torch

import gmmxx_amd
from tests import experts_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
V, D, E = 300, 72, 4


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (scale * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def parameters(dtype):
    return [rand(V, D, seed=1, dtype=dtype), rand(D, E, seed=2, dtype=dtype, scale=D ** -0.5),
            rand(E, D, D, seed=3, dtype=dtype, scale=D ** -0.5), rand(V, D, seed=4, dtype=dtype, scale=D ** -0.5)]


def tokens(n, seed=0):
    t = torch.randint(0, V, (n + 1,), generator=torch.Generator().manual_seed(seed)).to(DEV)
    t[5::11] = -1
    return t[:-1].contiguous(), t[1:].contiguous()


def forward(p, t, seed, keep=None):
    """The model's hidden rows and scores; `keep` collects what passes between the operators."""
    keep = [] if keep is None else keep
    h = gmmxx_amd.embed_rows(p[0], t, scale=1.5)
    x = gmmxx_amd.layer_norm(h)
    r = gmmxx_amd.route_rows(x @ p[1], 2)
    b = gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(x, p[2], r), r)
    y = gmmxx_amd.dropout(b, 0.25, seed, offset=3, residual=h)
    s = gmmxx_amd.layer_norm(y) @ p[3].t()
    keep += [h, b, y, s]
    return s


def step(p, t, following, seed):
    leaves = [w.detach().requires_grad_() for w in p]
    o = gmmxx_amd.log_probs(forward(leaves, t, seed), following, top_k=2)
    total = -(o.chosen.sum() + 0.1 * o.entropy.sum()) + 0.01 * o.top.sum()
    return [o.chosen.detach(), o.entropy.detach(), o.top.detach(), o.top_index, *torch.autograd.grad(total, leaves)]


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
def test_gradients_pass_through(hip, dtype):
    """Each operator's gradient within the model is that of the operator alone on the same rows (and those are
    compared with the formulas in the operators' own tests): equal, since it is the same arithmetic."""
    t, following = tokens(700)
    p = [w.requires_grad_() for w in parameters(dtype)]
    keep = []
    o = gmmxx_amd.log_probs(forward(p, t, 9, keep), following, top_k=2)
    h, b, y, s = keep
    dc, de, dt = rand(700, seed=5), rand(700, seed=6), rand(700, 2, seed=7)
    dtable, dh, db, dy, ds = torch.autograd.grad((o.chosen, o.entropy, o.top), (p[0], h, b, y, s), (dc, de, dt))
    alone = s.detach().requires_grad_()
    r = gmmxx_amd.log_probs(alone, following, top_k=2)
    assert torch.equal(r.chosen, o.chosen)
    assert torch.equal(torch.autograd.grad((r.chosen, r.entropy, r.top), alone, (dc, de, dt))[0], ds)
    alone = [b.detach().requires_grad_(), h.detach().requires_grad_()]
    z = gmmxx_amd.dropout(alone[0], 0.25, 9, offset=3, residual=alone[1])
    gb, gh = torch.autograd.grad(z, alone, dy)
    assert torch.equal(z, y) and torch.equal(gb, db) and torch.equal(gh, dy)
    alone = p[0].detach().requires_grad_()
    z = gmmxx_amd.embed_rows(alone, t, scale=1.5)
    assert torch.equal(z, h) and torch.equal(torch.autograd.grad(z, alone, dh)[0], dtable)
    assert not dtable[[i for i in range(V) if not (t == i).any()]].any()


def test_differentiable_once(hip):
    for call in (lambda x: gmmxx_amd.embed_rows(x, torch.tensor([1, 2], device=DEV)),
                 lambda x: gmmxx_amd.dropout(x, 0.5, 1),
                 lambda x: gmmxx_amd.log_probs(x, torch.zeros(6, dtype=torch.int64, device=DEV)).chosen):
        x = rand(6, 8).requires_grad_()
        g, = torch.autograd.grad(call(x).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()


def test_gradients_of_some_inputs(hip):
    x, r, dy = rand(30, 40), rand(30, 40, seed=1), rand(30, 40, seed=2)
    full = [x.detach().requires_grad_(), r.detach().requires_grad_()]
    want = torch.autograd.grad(gmmxx_amd.dropout(full[0], 0.3, 1, residual=full[1]), full, dy)
    for i in range(2):
        args = [v.detach().requires_grad_(i == j) for j, v in enumerate((x, r))]
        got, = torch.autograd.grad(gmmxx_amd.dropout(args[0], 0.3, 1, residual=args[1]), [args[i]], dy)
        assert torch.equal(got, want[i])
    o = gmmxx_amd.log_probs(x.detach().requires_grad_(), torch.zeros(30, dtype=torch.int32, device=DEV), top_k=2)
    assert not o.top_index.requires_grad and o.top.requires_grad


def test_no_grad(hip):
    t, following = tokens(50)
    p = [w.requires_grad_() for w in parameters(torch.float32)]
    with torch.no_grad():
        a = gmmxx_amd.log_probs(forward(p, t, 1), following)
    assert not a.chosen.requires_grad
    with torch.inference_mode():
        b = gmmxx_amd.log_probs(forward(p, t, 1), following)
    assert torch.equal(a.chosen, b.chosen)


@pytest.mark.parametrize("dtype", experts_ref.DTYPES, ids=str)
@pytest.mark.parametrize("n", [900, 6000])
def test_other_streams(hip, n, dtype):
    p, (t, following) = parameters(dtype), tokens(n)
    want = step(p, t, following, 4)
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(p, t, following, 4))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def capture(run):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    return graph, out


@pytest.mark.parametrize("n", [900, 6000])
def test_captured_training_step(hip, n):
    """Forward and backward passes in a graph: the eager results at every replay, with new tokens and a new seed on the
    device, beside other work; two graphs in turn share no workspace."""
    p = parameters(torch.bfloat16)
    first, second = tokens(n), tokens(n, seed=1)
    t, following, seed = first[0].clone(), first[1].clone(), torch.tensor([7], device=DEV)
    graphs = [capture(lambda: step(p, t, following, seed)) for _ in range(2)]
    for i, (new, s) in enumerate(((first, 7), (second, 8), (first, -9), (second, 8))):
        t.copy_(new[0])
        following.copy_(new[1])
        seed.fill_(s)
        want = step(p, t, following, s)
        for graph, _ in graphs:
            graph.replay()
        torch.zeros(1000, device=DEV).sum().item()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


@pytest.mark.parametrize("n", [1, 5, 30, 200])
def test_captured_serving_step(hip, n):
    p = parameters(torch.bfloat16)
    head = gmmxx_amd.quantize_rows(p[3])
    t = tokens(n)[0].clamp(min=0)

    def serve():
        with torch.no_grad():
            h = gmmxx_amd.layer_norm(gmmxx_amd.embed_rows(p[0], t))
            return gmmxx_amd.log_probs(gmmxx_amd.quantized_matmul(h, head), t, top_k=4)

    graph, out = capture(serve)
    for seed in range(4):
        t.copy_(tokens(n, seed=seed)[0].clamp(min=0))
        graph.replay()
        torch.zeros(1000, device=DEV).sum().item()
        assert all(torch.equal(a, b) for a, b in zip(out, serve()))


def test_example(hip):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")
    sys.path.insert(0, path)
    try:
        import code_model
    finally:
        sys.path.remove(path)
    losses, model, codes = code_model.run(rows=3000, clusters=9, steps=5)
    assert all(v == v and abs(v) < float("inf") for v in losses)
    for w in model.parameters():
        assert w.grad is not None and torch.isfinite(w.grad).all() and w.grad.any()
    one, many = model.answer(codes[:1]), model.answer(codes[:40])
    assert one.top.shape == (1, 3) and many.top_index.shape == (40, 3)
    assert ((many.top_index >= 0) & (many.top_index < 9)).all() and not many.chosen.any()
    assert (many.top[:, :-1] >= many.top[:, 1:]).all()


def test_example_answers_with_its_present_head(hip):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")
    sys.path.insert(0, path)
    try:
        import code_model
    finally:
        sys.path.remove(path)
    _, model, codes = code_model.run(rows=2000, clusters=9, steps=2)
    before = model.answer(codes[:50])
    with torch.no_grad():
        model.head.copy_(model.head.flip(0))                 # as training further or loading does
    after = model.answer(codes[:50])
    # (the same scores at the mirrored tokens; their probabilities' sum is added in another order)
    assert torch.equal(after.top_index, 8 - before.top_index)
    head = model.quantized_head()
    given = model.answer(codes[:50], head=head)
    assert all(torch.equal(a, b) for a, b in zip(given, after))
