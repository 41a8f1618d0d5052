"""Tokens in and tokens out, on the HIP library.

A fitted mixture turns rows into labels.  These operators take labels (or any codes)
as tokens: rows in front of a layer of experts, what regularises it in training, the loss on
the scores over the tokens that it answers with, and the large product of serving in 8 bits:

    h = embed_rows(table, mixture.predict(x))             # a row for every token
    h = dropout(branch(h), 0.1, seed, residual=h)         # a mask that is never stored
    p = log_probs(h @ head, targets, top_k=5)             # chosen, entropy, alternatives
    q = quantize_rows(head.t())                           # once
    scores = quantized_matmul(h, q)                       # 8-bit products, a scale for each row and column

Every function runs on the caller's current stream, never synchronises, and is
differentiable (once) by torch's autograd but for the 8-bit products, which are for serving.
Elements are float32, bfloat16 or float16; sums and statistics are float32 (of 8-bit values:
exact integers) and results are rounded to their type at the end.  Results are the same from run to run.
Forward-mode derivatives, traces and tensors that hold no values of their own are refused
with ``NotImplementedError``, as in ``gmmxx_amd.experts``.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from .experts import _ELEMS, _MAX_POSITIONS, MAX_WIDTH, _failed, _native, _operand, _rows, _tensor

MAX_TOKENS = 1 << 24        # rows of an embedding's table
MAX_SCORES = 1 << 22        # scores in a row
MAX_ALTERNATIVES = 64
MAX_QUANTIZED = 1 << 17     # the longest sum of 8-bit products that 32 bits tell from every other
_FP32_MAX = torch.finfo(torch.float32).max


class LogProbs(NamedTuple):
    """Log probabilities of N tokens."""

    chosen: torch.Tensor      #: (N,) float32, log p of the given tokens; 0 where none is given
    entropy: torch.Tensor     #: (N,) float32, of each row's distribution
    top: torch.Tensor         #: (N, top_k) float32, the largest log p, best first; -inf: none was left
    top_index: torch.Tensor   #: (N, top_k) int32, their tokens; -1: none was left


class Quantized(NamedTuple):
    """A matrix in 8-bit integers: ``values * scales[:, None]``."""

    values: torch.Tensor      #: (rows, D) int8
    scales: torch.Tensor      #: (rows,) float32


# --- arguments ----------------------------------------------------------------

def _tokens(t, name: str, index: int) -> torch.Tensor:
    if _tensor(t, name).dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: dtype must be torch.int32 or torch.int64, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: must be on the same device as the other operands, got {t.device}")
    if t.numel() >= _MAX_POSITIONS:
        raise ValueError(f"{name}: there must be fewer than {_MAX_POSITIONS} positions, got {t.numel()}")
    return t.reshape(-1).contiguous()


# --- embedding ----------------------------------------------------------------

def embed_rows(table: torch.Tensor, index: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[index]``: a row of the table for every token.

    ``table`` is (V, D) with V <= 2^24 and D <= 2^22, ``index`` int32 or int64 of any shape; the
    result is (*index.shape, D).  A token outside 0 .. V - 1 (-1 for padding, or for a
    choice of ``Routing.experts`` without an expert) gives zeros and no gradient.  ``scale`` is
    a finite number.  Differentiable in the table: the gradient is dense, and each row's sum is
    taken over the places of its token in their order."""
    _operand(table, "table")
    if table.ndim != 2 or not 1 <= table.shape[0] <= MAX_TOKENS or not 1 <= table.shape[1] <= MAX_WIDTH:
        raise ValueError(f"table must have shape (V, D) with 1 <= V <= {MAX_TOKENS} and 1 <= D <= {MAX_WIDTH}, "
                         f"got {tuple(table.shape)}")
    flat = _tokens(index, "index", table.get_device())
    scale = float(scale)
    if not abs(scale) <= _FP32_MAX:
        raise ValueError(f"scale must be finite in float32, got {scale}")
    try:
        y = _native().embed(_rows(table), flat, scale)
    except RuntimeError as exc:
        _failed(exc)
    return y if index.ndim == 1 else y.reshape(*index.shape, table.shape[1])


# --- dropout ------------------------------------------------------------------

def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], *, offset: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` with a share p of its elements zero and the others times 1 / (1 - p), plus ``residual``.

    Element i, in the order of x's shape, is dropped where word i of the counter-based generator
    Philox 4x32-10 with key ``seed`` at ``offset`` is less than p 2^32 (rounded): the mask
    is a function of seed, offset and i, the same for every dtype and layout, and the backward
    pass computes it again.  ``seed`` is an integer of 64 bits, or an int64 tensor of one
    element on x's device, which is read when the kernel runs (so a captured graph can draw a
    new mask at every replay) and must stay as it is until the backward pass has run;
    0 <= ``offset`` < 2^63 tells the calls of one seed apart.  A dropped element is zero
    whatever x holds.  ``residual`` has x's shape and dtype.  Differentiable in x and residual;
    x and residual that are not contiguous are copied first."""
    _operand(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must satisfy 0 <= p <= 1, got {p}")
    if x.numel() > 1 << 40:
        raise ValueError(f"x must have at most 2^40 elements, got {x.numel()}")
    offset = int(offset)
    if not 0 <= offset < 1 << 63:
        raise ValueError(f"offset must satisfy 0 <= offset < 2^63, got {offset}")
    seed_at = None
    if torch.is_tensor(seed):
        if _tensor(seed, "seed").dtype != torch.int64 or seed.numel() != 1:
            raise TypeError(f"seed must be an integer or an int64 tensor of one element, got {seed.dtype} of shape "
                            f"{tuple(seed.shape)}")
        if seed.get_device() != x.get_device():
            raise ValueError(f"seed: must be on the same device as x, got {seed.device}")
        seed, seed_at = 0, seed
    else:
        seed = int(seed)
        if not -(1 << 63) <= seed < 1 << 64:
            raise ValueError(f"seed must be an integer of 64 bits, got {seed}")
        seed = seed - (1 << 64) if seed >= 1 << 63 else seed
    if residual is not None:
        if _operand(residual, "residual").dtype != x.dtype:
            raise TypeError(f"residual: dtype must be {x.dtype}, got {residual.dtype}")
        if residual.get_device() != x.get_device():
            raise ValueError(f"residual: must be on the same device as x, got {residual.device}")
        if residual.shape != x.shape:
            raise ValueError(f"residual must have shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        residual = residual.contiguous()
    try:
        return _native().dropout(x.contiguous(), residual, p, seed, seed_at, offset)
    except RuntimeError as exc:
        _failed(exc)


# --- log probabilities ----------------------------------------------------------

def log_probs(scores: torch.Tensor, index: torch.Tensor, *, top_k: int = 0) -> LogProbs:
    """Log probabilities of given tokens under softmax(scores), with entropies and alternatives.

    ``scores`` is (..., V) with V <= 2^22, ``index`` (...) int32 or int64, ``top_k`` <= 64.  Scores
    of -inf or NaN are no candidates (mask a token with -inf); of several +inf each weighs the
    same.  ``chosen`` is log p of the row's token: -inf where it is no candidate, 0 without a
    gradient where the token is outside 0 .. V - 1 (a place that does not count).  ``entropy``
    is -sum p log p, 0 in a row without candidates.  ``top`` and ``top_index`` are the
    ``top_k`` likeliest tokens, the lower first among equals; where fewer candidates are left, -inf
    and -1.  ``chosen``, ``entropy`` and ``top`` are differentiable in scores, whose gradient
    is zero at what is no candidate."""
    _operand(scores, "scores")
    if scores.ndim < 1 or not 1 <= scores.shape[-1] <= MAX_SCORES:
        raise ValueError(f"scores must have shape (..., V) with 1 <= V <= {MAX_SCORES}, got {tuple(scores.shape)}")
    v = scores.shape[-1]
    flat = _tokens(index, "index", scores.get_device())
    if index.shape != scores.shape[:-1]:
        raise ValueError(f"index must have shape {tuple(scores.shape[:-1])}, got {tuple(index.shape)}")
    k = int(top_k)
    if not 0 <= k <= min(v, MAX_ALTERNATIVES):
        raise ValueError(f"top_k must satisfy 0 <= top_k <= {min(v, MAX_ALTERNATIVES)}, got {top_k}")
    try:
        r = _native().log_probs(_rows(scores if scores.ndim == 2 else scores.reshape(-1, v)), flat, k)
    except RuntimeError as exc:
        _failed(exc)
    if scores.ndim == 2:
        return LogProbs(*r)
    at = scores.shape[:-1]
    return LogProbs(r[0].reshape(at), r[1].reshape(at), r[2].reshape(*at, k), r[3].reshape(*at, k))


# --- products in 8-bit integers -------------------------------------------------

def _quantizable(x, name: str) -> torch.Tensor:
    if _operand(x, name).ndim != 2 or not 1 <= x.shape[1] <= MAX_QUANTIZED:
        raise ValueError(f"{name} must have shape (rows, D) with 1 <= D <= {MAX_QUANTIZED}, got {tuple(x.shape)}")
    if x.shape[0] >= _MAX_POSITIONS:
        raise ValueError(f"{name} must have fewer than {_MAX_POSITIONS} rows, got {x.shape[0]}")
    return x


def _quantized(q: Quantized, name: str, index: Optional[int]) -> Quantized:
    values, scales = _tensor(q.values, f"{name}.values"), _tensor(q.scales, f"{name}.scales")
    if values.dtype != torch.int8:
        raise TypeError(f"{name}.values: dtype must be torch.int8, got {values.dtype}")
    if scales.dtype != torch.float32:
        raise TypeError(f"{name}.scales: dtype must be torch.float32, got {scales.dtype}")
    if values.ndim != 2 or not 1 <= values.shape[1] <= MAX_QUANTIZED or values.shape[0] >= _MAX_POSITIONS:
        raise ValueError(f"{name}.values must have shape (rows, D) with 1 <= D <= {MAX_QUANTIZED} and fewer than "
                         f"{_MAX_POSITIONS} rows, got {tuple(values.shape)}")
    if scales.shape != values.shape[:1]:
        raise ValueError(f"{name}.scales must have shape {tuple(values.shape[:1])}, got {tuple(scales.shape)}")
    for t, what in ((values, "values"), (scales, "scales")):
        if t.get_device() != (values.get_device() if index is None else index):
            raise ValueError(f"{name}.{what}: must be on the same device as the other operands, got {t.device}")
    return Quantized(values, scales.contiguous())


def quantize_rows(x: torch.Tensor) -> Quantized:
    """The rows of a matrix in 8 bits, with a scale each.

    With a the largest absolute value of a row: ``values = round(x * (127 * (1 / a)))`` (ties to
    even), ``scales = a * (1 / 127)``, each operation rounded to float32.  ``x`` is (rows, D) with
    D <= 131072.  A row of zeros has scale 0; a row with a NaN or an infinity has scale NaN, and so
    have its products.  For a product's
    matrix, whose columns have the scales, take the rows of its transpose.  The rows of
    ``values`` are laid out in whole 128 bytes, as ``quantized_matmul`` reads them.  Has no gradient."""
    _quantizable(x, "x")
    try:
        return Quantized(*_native().quantize(_rows(x)))
    except RuntimeError as exc:
        _failed(exc)


def quantized_matmul(x: Union[torch.Tensor, Quantized], weight: Quantized, bias: Optional[torch.Tensor] = None, *,
                     dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x @ weight.T + bias`` by products of 8-bit integers, with a scale for each row and column.

    ``x`` is (rows, D), quantized here by rows, or ``Quantized`` already; ``weight`` is
    ``Quantized`` of (F, D), F <= 2^22, one row for each column of the result (``quantize_rows`` lays it
    out; values in rows that are not whole, aligned 16 bytes are copied at every call).
    ``bias`` is (F,) of the result's dtype, which is x's, float32 where x is ``Quantized``, or
    ``dtype``.  Sums are exact.  Each is rounded to float32, so is the product of its two scales, so
    is theirs with the bias added, and so to ``dtype`` is the result; with a scale below 2^-60 or above 2^60 in size
    it is formed in 64 bits instead, so no size of the scales loses it.  Has no gradient:
    operands that require one are refused outside ``torch.no_grad()``."""
    if not isinstance(weight, Quantized):
        raise TypeError("weight must be a Quantized (see quantize_rows)")
    if isinstance(x, Quantized):
        values, scales = _quantized(x, "x", None)
    else:
        values, scales = _quantizable(x, "x"), None
    index = values.get_device()
    weight = _quantized(weight, "weight", index)
    f, d = weight.values.shape
    if d != values.shape[1] or not 1 <= f <= MAX_WIDTH:
        raise ValueError(f"weight.values must have shape (F, {values.shape[1]}) with 1 <= F <= {MAX_WIDTH}, "
                         f"got {tuple(weight.values.shape)}")
    if dtype is None:
        dtype = torch.float32 if scales is not None else values.dtype
    if dtype not in _ELEMS:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    if bias is not None:
        if _operand(bias, "bias").dtype != dtype:
            raise TypeError(f"bias: dtype must be {dtype}, got {bias.dtype}")
        if bias.get_device() != index:
            raise ValueError(f"bias: must be on the same device as the other operands, got {bias.device}")
        if bias.shape != (f,):
            raise ValueError(f"bias must have shape {(f,)}, got {tuple(bias.shape)}")
        bias = bias.contiguous()
    try:
        return _native().quantized_matmul(values if scales is not None else _rows(values), scales, weight.values,
                                          weight.scales, bias, dtype)
    except RuntimeError as exc:
        _failed(exc)
