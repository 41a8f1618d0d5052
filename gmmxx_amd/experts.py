"""A sparsely gated layer of experts on the HIP library.

A fitted mixture says how responsible each component is for a row.  These four
operators make the components into experts with maps of their own, and train
them:

    h = layer_norm(x, weight, bias)             # rows on one scale
    routing = route_rows(scores, top_k)         # each row's best experts, rows grouped by expert
    y = grouped_matmul(h, experts, routing, b)  # every expert's matrix on its own rows
    out = combine_rows(y, routing)              # added up by gate

``scores`` are a gate's outputs or a mixture's log joint densities (log
responsibilities serve as well: a row's constant cancels).  Every function runs
on the caller's current stream, never synchronises, and is differentiable (once)
by torch's autograd; without a gradient to keep, nothing is saved.  Elements are
float32, bfloat16 or float16; sums and statistics are float32 and results are
rounded once.  Results are the same from run to run: no sum depends on the order
in which workgroups finish.

The kernels are hand-written HIP behind the C ABI (include/gmmxx_hip.h); there is
no PyTorch fallback.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _hip

_ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_EXPERTS = 4096
MAX_TOP_K = 64
MAX_NORM_WIDTH = 65536
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
    if _tensor(t, name).dtype not in _ELEM:
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


def _call(name: str, index: int, *args) -> None:
    """One library call on device ``index``, on its current stream."""
    lib = _hip._lib or _hip.load_library()
    if torch.cuda.current_device() == index:
        rc = getattr(lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _hip._check(rc, name)


def _workspace(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    # (the caching allocator's blocks are 512-byte aligned; the library checks)
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --- layer norm -----------------------------------------------------------------

def _norm_forward(x, weight, bias, eps, stats):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n, d = x.shape
    param = weight if weight is not None else bias
    if n:
        mean = stats.data_ptr() if stats is not None else None
        _call("gmmxx_hip_layer_norm", x.get_device(), _ELEM[x.dtype],
              _ELEM[x.dtype if param is None else param.dtype], n, d, x.data_ptr(), x.stride(0),
              None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), eps,
              y.data_ptr(), mean, mean + 4 * n if mean is not None else None)
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        stats = torch.empty(2 * x.shape[0], dtype=torch.float32, device=x.device)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return _norm_forward(x, weight, bias, eps, stats)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        n, d = x.shape
        _, need_w, need_b, _ = ctx.needs_input_grad
        param = weight.dtype if weight is not None else ctx.bias_dtype or x.dtype
        make = torch.empty if n else torch.zeros
        dx = torch.empty((n, d), dtype=x.dtype, device=x.device)
        dw = make(d, dtype=param, device=x.device) if need_w else None
        db = make(d, dtype=param, device=x.device) if need_b else None
        if n:
            dy = _rows(dy)
            need = _hip._lib.gmmxx_hip_layer_norm_workspace_bytes(n, d) if need_w or need_b else 0
            ws = _workspace(need, x) if need else None
            mean = stats.data_ptr()
            _call("gmmxx_hip_layer_norm_backward", x.get_device(), _ELEM[x.dtype], _ELEM[param], n, d, x.data_ptr(),
                  x.stride(0), dy.data_ptr(), dy.stride(0), None if weight is None else weight.data_ptr(), mean,
                  mean + 4 * n, dx.data_ptr(), dw.data_ptr() if need_w else None, db.data_ptr() if need_b else None,
                  ws.data_ptr() if need else None, need)
        return dx, dw, db, None


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
    flat = _rows(x if x.ndim == 2 else x.reshape(-1, d))
    if _wants_grad(x, weight, bias):
        y = _LayerNorm.apply(flat, weight, bias, eps)
    else:
        y = _norm_forward(flat, weight, bias, eps, None)
    return y if x.ndim == 2 else y.reshape(x.shape)


# --- routing --------------------------------------------------------------------

def _route_forward(scores, k, renormalize, want_norm):
    n, e = scores.shape
    dev, m = scores.device, n * k
    # experts, rows, slots and offsets in one allocation, and the gates (and the rows' normalisers) in another
    ints = torch.empty(3 * m + e + 1, dtype=torch.int32, device=dev) if n else torch.zeros(e + 1, dtype=torch.int32,
                                                                                           device=dev)
    experts, rows, slots, offsets = ints.split([m, m, m, e + 1])
    gates = torch.empty((n, k), dtype=torch.float32, device=dev)
    norm = torch.empty((n, 2), dtype=torch.float32, device=dev) if want_norm else None
    if n:
        lib = _hip._lib or _hip.load_library()
        need = lib.gmmxx_hip_route_workspace_bytes(n, e, k)
        ws = _workspace(need, scores)
        _call("gmmxx_hip_route", scores.get_device(), _ELEM[scores.dtype], n, e, k, int(renormalize),
              scores.data_ptr(), scores.stride(0), experts.data_ptr(), gates.data_ptr(), offsets.data_ptr(),
              rows.data_ptr(), slots.data_ptr(), norm.data_ptr() if want_norm else None, ws.data_ptr(), need)
    return experts.view(n, k), gates, offsets, rows, slots.view(n, k), norm


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, k, renormalize):
        experts, gates, offsets, rows, slots, norm = _route_forward(scores, k, renormalize, not renormalize)
        ctx.save_for_backward(experts, gates, *(() if renormalize else (scores, norm)))
        ctx.renormalize, ctx.shape, ctx.dtype = renormalize, scores.shape, scores.dtype
        ctx.mark_non_differentiable(experts, offsets, rows, slots)
        ctx.set_materialize_grads(False)
        return experts, gates, offsets, rows, slots

    @staticmethod
    @once_differentiable
    def backward(ctx, _experts, dgates, *_others):
        if dgates is None:
            return None, None, None
        experts, gates = ctx.saved_tensors[:2]
        scores, norm = (None, None) if ctx.renormalize else ctx.saved_tensors[2:]
        n, e = ctx.shape
        ds = torch.empty((n, e), dtype=ctx.dtype, device=gates.device)
        if n:
            dgates = dgates.contiguous()
            _call("gmmxx_hip_route_backward", gates.get_device(), _ELEM[ctx.dtype], n, e, gates.shape[1],
                  int(ctx.renormalize), None if scores is None else scores.data_ptr(),
                  0 if scores is None else scores.stride(0), experts.data_ptr(), gates.data_ptr(),
                  None if norm is None else norm.data_ptr(), dgates.data_ptr(), ds.data_ptr())
        return ds, None, None


def route_rows(scores: torch.Tensor, top_k: int, *, renormalize: bool = True) -> Routing:
    """Each row's ``top_k`` best of E experts, and the rows grouped by expert.

    ``scores`` is (N, E), E <= 4096 and top_k <= 64.  Equal scores go to the lower
    index.  Scores of -inf or NaN are no candidates (mask an expert with -inf); where
    fewer than ``top_k`` candidates are left, the remaining choices are expert -1 with
    gate 0.  ``gates`` are the softmax of the scores over the chosen experts, or, with
    ``renormalize=False``, over all candidates (the mixture's responsibilities where
    the scores are its log joint densities); candidates of +inf share the whole weight.
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
    renormalize = bool(renormalize)
    if _wants_grad(scores):
        return Routing(*_Route.apply(_rows(scores), k, renormalize))
    return Routing(*_route_forward(_rows(scores), k, renormalize, False)[:5])


# --- grouped products -----------------------------------------------------------

def _matrices(w: torch.Tensor) -> torch.Tensor:
    """(E, K, N) matrices of which one dimension's elements are adjacent: itself (a stack of transposed
    matrices included), or a copy."""
    se, sk, sn = w.stride()
    return w if sn == 1 or sk == 1 else w.contiguous()


def _strides(w: torch.Tensor, a: int, b: int):
    """The element strides of dimensions (0, a, b); a dimension of one element counts as adjacent where the
    other is not."""
    sa, sb = w.stride(a), w.stride(b)
    if sa != 1 and sb != 1:
        return (w.stride(0), 1, sb) if w.shape[a] == 1 else (w.stride(0), sa, 1)
    return w.stride(0), sa, sb


def _grouped(x, w, reduce_dim, out_dim, bias, offsets, rows, m, out_dtype):
    """out (M, w.shape[out_dim]): rows of x by w's matrices, summed over ``reduce_dim``."""
    out = torch.empty((m, w.shape[out_dim]), dtype=out_dtype, device=x.device)
    if m:
        we, wk, wn = _strides(w, reduce_dim, out_dim)
        _call("gmmxx_hip_grouped_matmul", x.get_device(), _ELEM[x.dtype], m, x.shape[0], w.shape[0],
              w.shape[reduce_dim], w.shape[out_dim], x.data_ptr(), x.stride(0),
              None if rows is None else rows.data_ptr(), w.data_ptr(), we, wk, wn,
              None if bias is None else bias.data_ptr(), offsets.data_ptr(), 8 * offsets.element_size(),
              out.data_ptr(), _ELEM[out_dtype])
    return out


def _combine(y, gates, slots, offsets, dtype):
    n, k = slots.shape
    out = torch.empty((n, y.shape[1]), dtype=dtype, device=y.device)
    if n:
        _call("gmmxx_hip_combine", y.get_device(), _ELEM[dtype], n, k, offsets.shape[0] - 1, y.shape[1],
              y.data_ptr(), _ELEM[y.dtype], y.stride(0), None if gates is None else gates.data_ptr(),
              slots.data_ptr(), offsets.data_ptr(), out.data_ptr())
    return out


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, rows, slots):
        ctx.save_for_backward(x, weight, offsets, rows, slots)
        m = x.shape[0] if rows is None else rows.shape[0]
        return _grouped(x, weight, 1, 2, bias, offsets, rows, m, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, offsets, rows, slots = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = _rows(dy)
        m, f = dy.shape
        e, d = weight.shape[:2]
        dx = dw = db = None
        if need_x and rows is None:
            dx = _grouped(dy, weight, 2, 1, None, offsets, None, m, x.dtype)
        elif need_x:
            # A row's choices are added in fp32 and rounded once; a single choice needs no sum.
            single = slots.shape[1] == 1
            parts = _grouped(dy, weight, 2, 1, None, offsets, None, m, x.dtype if single else torch.float32)
            dx = _combine(parts, None, slots, offsets, x.dtype)
        if need_w or need_b:
            make = torch.empty if m else torch.zeros
            dw = make((e, d, f), dtype=x.dtype, device=x.device)
            db = make((e, f), dtype=x.dtype, device=x.device) if need_b else None
            if m:
                need = _hip._lib.gmmxx_hip_grouped_workspace_bytes(m, e, d, f)
                ws = _workspace(need, x) if need else None
                _call("gmmxx_hip_grouped_weight_grad", x.get_device(), _ELEM[x.dtype], m, x.shape[0], e, d, f,
                      x.data_ptr(), x.stride(0), None if rows is None else rows.data_ptr(), dy.data_ptr(),
                      dy.stride(0), offsets.data_ptr(), 8 * offsets.element_size(), dw.data_ptr(),
                      db.data_ptr() if need_b else None, ws.data_ptr() if need else None, need)
        return dx, dw if need_w else None, db, None, None, None


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

    ``weight`` is (E, D, F) with E <= 4096, contiguous or a transposed view of
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
    if weight.ndim != 3 or weight.shape[1] != x.shape[1] or not 1 <= weight.shape[0] <= MAX_EXPERTS \
            or weight.shape[2] < 1:
        raise ValueError(f"weight must have shape (E, {x.shape[1]}, F) with 1 <= E <= {MAX_EXPERTS}, "
                         f"got {tuple(weight.shape)}")
    e, _, f = weight.shape
    if bias is not None:
        if tuple(_like(bias, "bias", x.dtype, index).shape) != (e, f):
            raise ValueError(f"bias must have shape {(e, f)}, got {tuple(bias.shape)}")
        bias = bias.contiguous()
    if isinstance(groups, Routing):
        offsets = _int_tensor(groups.offsets, "groups.offsets", index, (e + 1,))
        if _tensor(groups.slots, "groups.slots").ndim != 2:
            raise ValueError(f"groups.slots must have shape (N, top_k), got {tuple(groups.slots.shape)}")
        slots = _int_tensor(groups.slots, "groups.slots", index, (x.shape[0], groups.slots.shape[1]))
        rows = _int_tensor(groups.rows, "groups.rows", index, (slots.numel(),))
        m = slots.numel()
        if slots.shape[1] > MAX_TOP_K:
            raise ValueError(f"groups: top_k must be at most {MAX_TOP_K}, got {slots.shape[1]}")
    else:
        offsets = _int_tensor(groups, "groups", index, (e + 1,), (torch.int32, torch.int64))
        rows = slots = None
        m = x.shape[0]
    if m >= _MAX_POSITIONS:
        raise ValueError(f"there must be fewer than {_MAX_POSITIONS} positions, got {m}")
    x, weight = _rows(x), _matrices(weight)
    if _wants_grad(x, weight, bias):
        return _Grouped.apply(x, weight, bias, offsets, rows, slots)
    return _grouped(x, weight, 1, 2, bias, offsets, rows, m, x.dtype)


# --- combination ----------------------------------------------------------------

class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, gates, slots, offsets):
        ctx.save_for_backward(y, gates, slots, offsets)
        return _combine(y, gates, slots, offsets, y.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, gates, slots, offsets = ctx.saved_tensors
        n, k = slots.shape
        dout = _rows(dout)
        dy = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        dgates = torch.empty((n, k), dtype=torch.float32, device=y.device)
        if n:
            _call("gmmxx_hip_combine_backward", y.get_device(), _ELEM[y.dtype], n, k, offsets.shape[0] - 1,
                  y.shape[1], y.data_ptr(), y.stride(0), gates.data_ptr(), slots.data_ptr(), offsets.data_ptr(),
                  dout.data_ptr(), dout.stride(0), dy.data_ptr(), dgates.data_ptr())
        need_y, need_g = ctx.needs_input_grad[:2]
        return dy if need_y else None, dgates if need_g else None, None, None


def combine_rows(y: torch.Tensor, routing: Routing, gates: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[n] = sum over j of gates[n, j] * y[routing.slots[n, j]]``: the experts' results
    of each row, added up.

    ``y`` is (N * top_k, F) in grouped order, ``gates`` (N, top_k) float32, by default
    ``routing.gates``.  Choices without an expert add nothing.  Differentiable in y
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
    if y.ndim != 2 or y.shape[0] != slots.numel() or y.shape[1] < 1:
        raise ValueError(f"y must have shape ({slots.numel()}, F) with F >= 1, got {tuple(y.shape)}")
    if y.shape[0] >= _MAX_POSITIONS:
        raise ValueError(f"there must be fewer than {_MAX_POSITIONS} positions, got {y.shape[0]}")
    gates = routing.gates if gates is None else gates
    if _like(gates, "gates", torch.float32, index).shape != slots.shape:
        raise ValueError(f"gates must have shape {tuple(slots.shape)}, got {tuple(gates.shape)}")
    y, gates = _rows(y), gates.contiguous()
    if _wants_grad(y, gates):
        return _Combine.apply(y, gates, slots, offsets)
    return _combine(y, gates, slots, offsets, y.dtype)
