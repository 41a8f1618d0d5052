"""Operands whose memory does not hold their values.  Views of the negatives of it, as the
imaginary part of a conjugate is: the values count, in every operand and in the results'
gradients.  Tensors without memory: refused, optional operands among them."""

import pytest
import torch

import gmmxx_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(*shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def negated(t):
    """t, as a view of -t."""
    view = torch._neg_view(-t)
    assert view.is_neg() and torch.equal(view, t)
    return view


def layer_norm(x, w, b):
    return gmmxx_amd.layer_norm(x, w, b)


def gates(scores):
    return gmmxx_amd.route_rows(scores, 2, renormalize=False).gates


def grouped(x, w, b):
    return gmmxx_amd.grouped_matmul(x, w, torch.tensor([0, 3, 9], dtype=torch.int32, device=DEV), bias=b)


def combine(y, g):
    return gmmxx_amd.combine_rows(y, gmmxx_amd.route_rows(rand(6, 3, seed=9), 2), g)


CALLS = [(layer_norm, [(5, 24), (24,), (24,)]), (gates, [(7, 6)]), (grouped, [(9, 16), (2, 16, 24), (2, 24)]),
         (combine, [(12, 8), (6, 2)])]


@pytest.mark.parametrize("call,shapes", CALLS, ids=[c.__name__ for c, _ in CALLS])
def test_negated_views(hip, call, shapes):
    args = [rand(*s, seed=i) for i, s in enumerate(shapes)]
    leaves = [t.clone().requires_grad_() for t in args]
    want = call(*leaves)
    dout = rand(*want.shape, seed=7)
    grads = torch.autograd.grad(want, leaves, dout)
    with torch.no_grad():
        for i in range(len(args)):
            assert torch.equal(call(*[negated(t) if i == j else t for j, t in enumerate(args)]), want), i
    leaves = [negated(t).requires_grad_() for t in args]
    got = call(*leaves)
    assert torch.equal(got, want)
    for g, w in zip(torch.autograd.grad(got, leaves, negated(dout)), grads):
        assert torch.equal(g, w)


def test_imaginary_part_of_a_conjugate(hip):
    z = torch.complex(rand(6, 1, seed=1), rand(6, 1, seed=2))
    x = z.conj().imag
    assert x.is_neg()
    w, off = rand(2, 1, 8, seed=3), torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
    assert torch.equal(gmmxx_amd.grouped_matmul(x, w, off), gmmxx_amd.grouped_matmul(-z.imag.contiguous(), w, off))


@pytest.mark.parametrize("call,shapes", CALLS, ids=[c.__name__ for c, _ in CALLS])
def test_operands_without_memory(hip, call, shapes):
    """None of them is taken for an operand that was left out."""
    args = [rand(*s, seed=i) for i, s in enumerate(shapes)]
    for i, t in enumerate(args):
        zeros = torch._efficientzerotensor(t.shape, device=DEV)
        with pytest.raises(NotImplementedError, match="hold their values"):
            call(*[zeros if i == j else a for j, a in enumerate(args)])
        with pytest.raises(NotImplementedError, match="hold their values"):
            torch.func.functionalize(lambda v: call(*[v if i == j else a for j, a in enumerate(args)]))(t)
