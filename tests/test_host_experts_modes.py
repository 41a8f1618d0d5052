"""What the sparsely gated layer's operators cannot give is refused, never left out of the
result: forward-mode derivatives, and traces, which would record the results' allocation
without the launch that writes them.

The native module is called with no rows, so no kernel is launched and no GPU is needed.
"""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from gmmxx_amd import experts

INTS = dict(dtype=torch.int32)


def layer_norm(ops, t):
    return ops.layer_norm(t(0, 4), t(4), t(4), 1e-5)


def route(ops, t):
    return ops.route(t(0, 4), 2, True)[1]


def grouped(ops, t):
    return ops.grouped(t(0, 4), t(3, 4, 5), t(3, 5), torch.zeros(4, **INTS), None, None)


def combine(ops, t):
    return ops.combine(t(0, 5), t(0, 2), torch.zeros((0, 2), **INTS), torch.zeros(4, **INTS))


OPERANDS = [(layer_norm, 3), (route, 1), (grouped, 3), (combine, 2)]
EACH = [(call, i) for call, count in OPERANDS for i in range(count)]


@pytest.fixture(scope="module")
def ops():
    return experts._native()


def operands(change):
    """A maker of zeros that counts them: change(number, tensor) replaces it."""
    made = []

    def make(*shape):
        made.append(torch.zeros(shape))
        return change(len(made) - 1, made[-1])
    return make


@pytest.mark.parametrize("grad", [False, True], ids=["plain", "another requires grad"])
@pytest.mark.parametrize("call,which", EACH, ids=lambda v: getattr(v, "__name__", str(v)))
def test_forward_mode_is_refused(ops, call, which, grad):
    def change(i, t):
        if i == which:
            return forward_ad.make_dual(t, torch.ones_like(t))
        return t.requires_grad_() if grad else t

    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(ops, operands(change))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(ops, operands(change))
        # (switched off, tangents are not asked for)
        with torch.no_grad(), forward_ad._set_fwd_grad_enabled(False):
            call(ops, operands(change))
    call(ops, operands(lambda i, t: t))


@pytest.mark.parametrize("call", [c for c, _ in OPERANDS], ids=lambda c: c.__name__)
def test_traces_are_refused(ops, call):
    from torch.fx.experimental.proxy_tensor import make_fx

    def run(first):
        return call(ops, operands(lambda i, t: first if i == 0 else t))

    call(ops, operands(lambda i, t: t))
    first = []
    call(ops, operands(lambda i, t: first.append(t) or t))
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(run, (first[0],), check_trace=False)
    for mode in ("real", "fake"):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(run, tracing_mode=mode)(first[0])
    # other modes are no traces
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):
        run(first[0])


@pytest.mark.parametrize("call", [c for c, _ in OPERANDS], ids=lambda c: c.__name__)
def test_backward_passes_refuse_them_too(ops, call):
    """A gradient is linear in the results' gradients: a tangent of theirs must not be dropped."""
    leaves = []

    def change(i, t):
        leaves.append(t.requires_grad_())
        return leaves[-1]

    out = call(ops, operands(change))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, leaves, dual, retain_graph=True)
    grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert all(g.shape == t.shape for g, t in zip(grads, leaves))
