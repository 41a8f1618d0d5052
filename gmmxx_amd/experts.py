"""A sparsely gated layer of experts on the HIP library.

A fitted mixture says how responsible each component is for a row.  These four
operators make the components into experts with maps of their own, and train
them:

    h = layer_norm(x, weight, bias)             # rows on one scale
    routing = route_rows(scores, top_k)         # each row's best experts, rows grouped by expert
    y = grouped_matmul(h, experts, routing, b)  # every expert's matrix on its own rows
    out = combine_rows(y, routing)              # added up by gate

``scores`` are a gate's outputs or the logarithms of a mixture's responsibilities
(``torch.log(mixture.predict_proba(x))``).  Every function runs on the caller's
current stream, never synchronises, and is differentiable (once) by torch's
autograd; where no gradient is wanted, nothing is saved.  Forward-mode
derivatives, traces (``torch.jit.trace``, ``make_fx``) and tensors that hold no
values of their own are refused with ``NotImplementedError``.  Elements are
float32, bfloat16 or float16; sums and statistics are float32 and results are
rounded once.  Results are the same from run to run: no sum depends on the order
in which workgroups finish.

The kernels are hand-written HIP behind the C ABI (include/gmmxx_hip.h); the
autograd functions around it are the native module ``gmmxx_amd._autograd``
(csrc/autograd.cpp), whose backward passes run without the interpreter.  There is
no PyTorch fallback.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Union

import torch

from . import _hip

_ELEMS = (torch.float32, torch.bfloat16, torch.float16)
MAX_EXPERTS = 4096
MAX_TOP_K = 64
MAX_NORM_WIDTH = 65536
MAX_WIDTH = 1 << 22
_MAX_POSITIONS = 1 << 30


class Routing(NamedTuple):
    """Which experts each of N rows goes to, and the rows grouped by expert.

    Position p of the grouped order runs from 0 to N * top_k - 1; expert e's rows
    are at positions ``offsets[e]`` to ``offsets[e + 1] - 1``, in ascending order.
    Choices that found no candidate come after all groups.
    """

    experts: torch.Tensor   #: (N, top_k) int32, best first; -1: no candidate was left
    gates: torch.Tensor     #: (N, top_k) float32
    offsets: torch.Tensor   #: (E + 1,) int32
    rows: torch.Tensor      #: (N * top_k,) int32, the row at each position
    slots: torch.Tensor     #: (N, top_k) int32, the position of each choice


# --- arguments ----------------------------------------------------------------

def _tensor(t, name: str) -> torch.Tensor:
    if not torch.is_tensor(t):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: must be on a GPU device, got {t.device}")
    return t


def _operand(t, name: str) -> torch.Tensor:
    if _tensor(t, name).dtype not in _ELEMS:
        raise TypeError(f"{name}: dtype must be float32, bfloat16 or float16, got {t.dtype}")
    return t


def _like(t, name: str, dtype, index: int) -> torch.Tensor:
    if _tensor(t, name).dtype != dtype:
        raise TypeError(f"{name}: dtype must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: must be on the same device as the rows, got {t.device}")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix whose rows' elements are adjacent: itself, or a copy."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


_ENTRY_POINTS = ("last_error", "layer_norm", "layer_norm_workspace_bytes", "layer_norm_backward",
                 "route_workspace_bytes", "route", "route_backward", "grouped_matmul", "grouped_workspace_bytes",
                 "grouped_weight_grad", "combine", "combine_backward")
_ops = None


def _native():
    """The autograd functions, bound (once) to the loaded library's entry points."""
    global _ops
    if _ops is None:
        lib = _hip.load_library()
        try:
            from . import _autograd
        except ImportError as exc:
            raise _hip.HipBackendUnavailable(
                f"cannot load gmmxx_amd._autograd: {exc}. Build it with `python -m gmmxx_amd.build`.") from exc
        _autograd.bind({name: ctypes.cast(getattr(lib, "gmmxx_hip_" + name), ctypes.c_void_p).value
                        for name in _ENTRY_POINTS})
        _ops = _autograd
    return _ops


def _failed(exc: RuntimeError):
    """A library call's failure as the package's own error; any other as it is."""
    if not str(exc).startswith("gmmxx_hip_"):
        raise exc
    cls = _hip.HipRuntimeError if _hip.no_fallback() else _hip.HipRuntimeFallback
    raise cls(str(exc).split("\n", 1)[0]) from exc


# --- layer norm -----------------------------------------------------------------

def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension.

    ``x`` is (..., D) with 1 <= D <= 65536; ``weight`` and ``bias`` are (D,), both of
    x's dtype or both float32, and may be left out.  Differentiable in all three."""
    _operand(x, "x")
    index = x.get_device()
    if x.ndim < 1 or not 1 <= x.shape[-1] <= MAX_NORM_WIDTH:
        raise ValueError(f"x must have shape (..., D) with 1 <= D <= {MAX_NORM_WIDTH}, got {tuple(x.shape)}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("eps must be non-negative")
    d = x.shape[-1]
    for p, name in ((weight, "weight"), (bias, "bias")):
        if p is None:
            continue
        if _operand(p, name).dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name}: dtype must be {x.dtype} or torch.float32, got {p.dtype}")
        if p.get_device() != index:
            raise ValueError(f"{name}: must be on the same device as the rows, got {p.device}")
        if p.ndim != 1 or p.shape[0] != d:
            raise ValueError(f"{name} must have shape {(d,)}, got {tuple(p.shape)}")
    if weight is not None:
        if bias is not None and weight.dtype != bias.dtype:
            raise TypeError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    try:
        y = _native().layer_norm(_rows(x if x.ndim == 2 else x.reshape(-1, d)), weight, bias, eps)
    except RuntimeError as exc:
        _failed(exc)
    return y if x.ndim == 2 else y.reshape(x.shape)


# --- routing --------------------------------------------------------------------

def route_rows(scores: torch.Tensor, top_k: int, *, renormalize: bool = True) -> Routing:
    """Each row's ``top_k`` best of E experts, and the rows grouped by expert.

    ``scores`` is (N, E), E <= 4096 and top_k <= 64.  Equal scores go to the lower
    index.  Scores of -inf or NaN are no candidates (mask an expert with -inf); where
    fewer than ``top_k`` candidates are left, the remaining choices are expert -1 with
    gate 0.  ``gates`` are the softmax of the scores over the chosen experts, or, with
    ``renormalize=False``, over all candidates (the mixture's responsibilities where
    the scores are their logarithms); candidates of +inf share the whole weight.
    ``gates`` is differentiable in ``scores``."""
    _operand(scores, "scores")
    if scores.ndim != 2 or not 1 <= scores.shape[1] <= MAX_EXPERTS:
        raise ValueError(f"scores must have shape (N, E) with 1 <= E <= {MAX_EXPERTS}, got {tuple(scores.shape)}")
    n, e = scores.shape
    k = int(top_k)
    if not 1 <= k <= min(e, MAX_TOP_K):
        raise ValueError(f"top_k must satisfy 1 <= top_k <= {min(e, MAX_TOP_K)}, got {top_k}")
    if n * k >= _MAX_POSITIONS:
        raise ValueError(f"N * top_k must be less than {_MAX_POSITIONS}, got {n * k}")
    try:
        return Routing(*_native().route(_rows(scores), k, bool(renormalize)))
    except RuntimeError as exc:
        _failed(exc)


# --- grouped products -----------------------------------------------------------

def _matrices(w: torch.Tensor) -> torch.Tensor:
    """(E, K, N) matrices of which one dimension's elements are adjacent (or its only ones): itself, a stack of
    transposed matrices included, or a copy."""
    _, sk, sn = w.stride()
    return w if sn == 1 or sk == 1 else w.contiguous()


def _int_tensor(t, name, index, shape, dtypes=(torch.int32,)):
    if _tensor(t, name).dtype not in dtypes:
        raise TypeError(f"{name}: dtype must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: must be on the same device as the rows, got {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, groups: Union[Routing, torch.Tensor],
                   bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x[p] @ weight[e] + bias[e]`` for every position p of every expert e's group.

    ``weight`` is (E, D, F) with E <= 4096 and D and F <= 2^22, contiguous or a transposed view of
    (E, F, D), ``bias`` (E, F), both of x's dtype.  ``groups`` is

    * a ``Routing``: ``x`` is (N, D), its rows are read where the routing sends them,
      and the result is (N * top_k, F) in grouped order;
    * offsets (E + 1,), int32 or int64, ascending from 0 to at most M: ``x`` is (M, D)
      with expert e's rows at offsets[e] to offsets[e + 1] - 1.

    Positions past the last group get zeros, an empty group's gradient is zero.
    The offsets stay on the device and are not checked: values out of range act as the
    nearest valid ones.  Differentiable in x, weight and bias."""
    _operand(x, "x")
    index = x.get_device()
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError(f"x must have shape (rows, D) with D >= 1, got {tuple(x.shape)}")
    _like(weight, "weight", x.dtype, index)
    if x.shape[1] > MAX_WIDTH:
        raise ValueError(f"x must have shape (rows, D) with D <= {MAX_WIDTH}, got {tuple(x.shape)}")
    if weight.ndim != 3 or weight.shape[1] != x.shape[1] or not 1 <= weight.shape[0] <= MAX_EXPERTS \
            or not 1 <= weight.shape[2] <= MAX_WIDTH:
        raise ValueError(f"weight must have shape (E, {x.shape[1]}, F) with 1 <= E <= {MAX_EXPERTS} and "
                         f"1 <= F <= {MAX_WIDTH}, got {tuple(weight.shape)}")
    e, _, f = weight.shape
    if bias is not None:
        if tuple(_like(bias, "bias", x.dtype, index).shape) != (e, f):
            raise ValueError(f"bias must have shape {(e, f)}, got {tuple(bias.shape)}")
        bias = bias.contiguous()
    if isinstance(groups, Routing):
        offsets = _int_tensor(groups.offsets, "groups.offsets", index, (e + 1,))
        if _tensor(groups.slots, "groups.slots").ndim != 2 or not 1 <= groups.slots.shape[1] <= MAX_TOP_K:
            raise ValueError(f"groups.slots must have shape (N, top_k) with 1 <= top_k <= {MAX_TOP_K}, "
                             f"got {tuple(groups.slots.shape)}")
        slots = _int_tensor(groups.slots, "groups.slots", index, (x.shape[0], groups.slots.shape[1]))
        rows = _int_tensor(groups.rows, "groups.rows", index, (slots.numel(),))
        m = slots.numel()
    else:
        offsets = _int_tensor(groups, "groups", index, (e + 1,), (torch.int32, torch.int64))
        rows = slots = None
        m = x.shape[0]
    if m >= _MAX_POSITIONS:
        raise ValueError(f"there must be fewer than {_MAX_POSITIONS} positions, got {m}")
    try:
        return _native().grouped(_rows(x), _matrices(weight), bias, offsets, rows, slots)
    except RuntimeError as exc:
        _failed(exc)


# --- combination ----------------------------------------------------------------

def combine_rows(y: torch.Tensor, routing: Routing, gates: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[n] = sum over j of gates[n, j] * y[routing.slots[n, j]]``: the experts' results
    of each row, added up.

    ``y`` is (N * top_k, F) in grouped order, F <= 2^22, ``gates`` (N, top_k) float32,
    by default ``routing.gates``.  Choices without an expert add nothing.  Differentiable in y
    and the gates."""
    _operand(y, "y")
    index = y.get_device()
    if not isinstance(routing, Routing):
        raise TypeError("routing must be a Routing")
    slots, offsets = _tensor(routing.slots, "routing.slots"), _tensor(routing.offsets, "routing.offsets")
    if slots.ndim != 2 or not 1 <= slots.shape[1] <= MAX_TOP_K:
        raise ValueError(f"routing.slots must have shape (N, top_k) with 1 <= top_k <= {MAX_TOP_K}, "
                         f"got {tuple(slots.shape)}")
    slots = _int_tensor(slots, "routing.slots", index, slots.shape)
    if offsets.ndim != 1 or offsets.shape[0] < 2:
        raise ValueError(f"routing.offsets must have shape (E + 1,), got {tuple(offsets.shape)}")
    offsets = _int_tensor(offsets, "routing.offsets", index, offsets.shape)
    if y.ndim != 2 or y.shape[0] != slots.numel() or not 1 <= y.shape[1] <= MAX_WIDTH:
        raise ValueError(f"y must have shape ({slots.numel()}, F) with 1 <= F <= {MAX_WIDTH}, got {tuple(y.shape)}")
    if y.shape[0] >= _MAX_POSITIONS:
        raise ValueError(f"there must be fewer than {_MAX_POSITIONS} positions, got {y.shape[0]}")
    gates = routing.gates if gates is None else gates
    if _like(gates, "gates", torch.float32, index).shape != slots.shape:
        raise ValueError(f"gates must have shape {tuple(slots.shape)}, got {tuple(gates.shape)}")
    try:
        return _native().combine(_rows(y), gates.contiguous(), slots, offsets)
    except RuntimeError as exc:
        _failed(exc)
