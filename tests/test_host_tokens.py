"""The token operators' arguments, without a GPU: what the C ABI refuses and with which status, that calls without
rows return at once, what the Python functions refuse, and that forward-mode derivatives, traces and gradients of what has
none are refused.

No kernel is launched: every call here returns before any device work.
"""

import ctypes
import os
import re

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import gmmxx_amd
from gmmxx_amd import Quantized, _hip, experts

F32, BF16, F16 = 0, 1, 2
OK = 0
P = ctypes.c_void_p(4096)      # never read: the call ends before
NULL = ctypes.c_void_p(0)
INVALID, UNSUPPORTED, WORKSPACE = "GMMXX_ERR_INVALID_ARGUMENT", "GMMXX_ERR_UNSUPPORTED", "GMMXX_ERR_WORKSPACE"


@pytest.fixture(scope="module")
def lib():
    return _hip.load_library()


@pytest.fixture(scope="module")
def codes():
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "gmmxx_hip.h")).read()
    return {m[0]: int(m[1]) for m in re.findall(r"(GMMXX_[A-Z0-9_]+)\s*=\s*(-?\d+)", text)}


def embed(lib, elem=F32, n=3, v=9, d=8, table=P, ldt=8, index=P, bits=64, scale=1.0, out=P):
    return lib.gmmxx_hip_embed(elem, n, v, d, table, ldt, index, bits, scale, out, NULL)


def embed_back(lib, elem=F32, n=3, v=9, d=8, dy=P, lddy=8, index=P, bits=64, scale=1.0, out=P, ws=P, size=1 << 30):
    return lib.gmmxx_hip_embed_backward(elem, n, v, d, dy, lddy, index, bits, scale, out, ws, size, NULL)


def drop(lib, elem=F32, n=3, p=0.5, x=P, out=P):
    return lib.gmmxx_hip_dropout(elem, n, p, 1, NULL, 0, x, NULL, out, NULL)


def logp(lib, elem=F32, n=3, v=9, k=2, scores=P, ld=9, index=P, bits=64, chosen=P, entropy=P, top=P, top_index=P, ws=P,
         size=1 << 40):
    return lib.gmmxx_hip_log_probs(elem, n, v, k, scores, ld, index, bits, chosen, entropy, top, top_index, NULL, ws,
                                   size, NULL)


def logp_back(lib, elem=F32, n=3, v=9, k=2, scores=P, ld=9, index=P, bits=64, top_index=P, stats=P, dtop=P, ds=P):
    return lib.gmmxx_hip_log_probs_backward(elem, n, v, k, scores, ld, index, bits, top_index, stats, P, P, dtop, ds,
                                            NULL)


def quantize(lib, elem=F32, n=3, d=8, x=P, ldx=8, values=P, ldv=16, scales=P):
    return lib.gmmxx_hip_quantize(elem, n, d, x, ldx, values, ldv, scales, NULL)


def matmul(lib, elem=F32, n=3, f=5, d=8, x=P, ldx=16, xs=P, w=P, ldw=16, ws=P, out=P):
    return lib.gmmxx_hip_quantized_matmul(elem, n, f, d, x, ldx, xs, w, ldw, ws, NULL, out, NULL)


def linear(lib, elem=F32, out_elem=F32, n=30, f=5, d=8, x=P, ldx=8, w=P, ldw=16, ws=P, out=P, work=P, size=1 << 30):
    return lib.gmmxx_hip_quantized_linear(elem, out_elem, n, f, d, x, ldx, w, ldw, ws, NULL, out, work, size, NULL)


ODD = ctypes.c_void_p(4100)
CASES = [
    (embed, dict(elem=7), INVALID, "elem"), (embed, dict(n=-1), INVALID, "N"), (embed, dict(v=0), INVALID, "V"),
    (embed, dict(d=0), INVALID, "D"), (embed, dict(bits=16), INVALID, "index_bits"),
    (embed, dict(scale=float("nan")), INVALID, "scale"), (embed, dict(scale=float("inf")), INVALID, "scale"),
    (embed, dict(scale=1e39), INVALID, "scale"), (embed, dict(v=(1 << 24) + 1), UNSUPPORTED, "2^24"),
    (embed, dict(d=(1 << 22) + 1), UNSUPPORTED, "2^22"), (embed, dict(n=1 << 30), UNSUPPORTED, "2^30"),
    (embed, dict(n=1 << 29, d=1 << 12), UNSUPPORTED, "2^40"), (embed, dict(table=NULL), INVALID, "NULL"),
    (embed, dict(index=NULL), INVALID, "NULL"), (embed, dict(out=NULL), INVALID, "NULL"),
    (embed, dict(ldt=-1), INVALID, "strides"),
    (embed_back, dict(elem=-1), INVALID, "elem"), (embed_back, dict(dy=NULL), INVALID, "NULL"),
    (embed_back, dict(index=NULL), INVALID, "NULL"), (embed_back, dict(out=NULL), INVALID, "NULL"),
    (embed_back, dict(lddy=-8), INVALID, "strides"), (embed_back, dict(ws=NULL), WORKSPACE, "NULL"),
    (embed_back, dict(size=64), WORKSPACE, "small"), (embed_back, dict(ws=ODD), WORKSPACE, "aligned"),
    (embed_back, dict(scale=float("-inf")), INVALID, "scale"), (embed_back, dict(bits=8), INVALID, "index_bits"),
    (drop, dict(elem=3), INVALID, "elem"), (drop, dict(n=-1), INVALID, "n must"), (drop, dict(p=-0.1), INVALID, "p must"),
    (drop, dict(p=1.5), INVALID, "p must"), (drop, dict(p=float("nan")), INVALID, "p must"),
    (drop, dict(n=(1 << 40) + 1), UNSUPPORTED, "2^40"), (drop, dict(x=NULL), INVALID, "NULL"),
    (drop, dict(out=NULL), INVALID, "NULL"),
    (logp, dict(elem=4), INVALID, "elem"), (logp, dict(n=-1), INVALID, "N"), (logp, dict(v=0), INVALID, "V"),
    (logp, dict(bits=0), INVALID, "index_bits"), (logp, dict(k=-1), INVALID, "k must"), (logp, dict(k=10), INVALID, "k must"),
    (logp, dict(v=100, k=65), UNSUPPORTED, "64"), (logp, dict(v=(1 << 22) + 1), UNSUPPORTED, "2^22"),
    (logp, dict(n=1 << 30), UNSUPPORTED, "2^30"), (logp, dict(scores=NULL), INVALID, "NULL"),
    (logp, dict(index=NULL), INVALID, "NULL"), (logp, dict(chosen=NULL), INVALID, "NULL"),
    (logp, dict(entropy=NULL), INVALID, "NULL"), (logp, dict(top=NULL), INVALID, "NULL"),
    (logp, dict(top_index=NULL), INVALID, "NULL"), (logp, dict(ld=-9), INVALID, "strides"),
    (logp, dict(v=100_000, ld=100_000, ws=NULL), WORKSPACE, "NULL"),
    (logp, dict(v=100_000, ld=100_000, size=16), WORKSPACE, "small"),
    (logp_back, dict(stats=NULL), INVALID, "NULL"), (logp_back, dict(ds=NULL), INVALID, "NULL"),
    (logp_back, dict(scores=NULL), INVALID, "NULL"), (logp_back, dict(index=NULL), INVALID, "NULL"),
    (logp_back, dict(top_index=NULL), INVALID, "NULL"), (logp_back, dict(ld=-1), INVALID, "strides"),
    (logp_back, dict(k=65, v=99), UNSUPPORTED, "64"),
    (quantize, dict(elem=9), INVALID, "elem"), (quantize, dict(n=-1), INVALID, "N"), (quantize, dict(d=0), INVALID, "D"),
    (quantize, dict(d=(1 << 17) + 1), UNSUPPORTED, "131072"), (quantize, dict(n=1 << 30), UNSUPPORTED, "2^30"),
    (quantize, dict(x=NULL), INVALID, "NULL"), (quantize, dict(values=NULL), INVALID, "NULL"),
    (quantize, dict(scales=NULL), INVALID, "NULL"), (quantize, dict(ldx=-1), INVALID, "strides"),
    (quantize, dict(ldv=24), INVALID, "16"), (quantize, dict(d=40, ldv=32), INVALID, "16"),
    (quantize, dict(values=ODD), INVALID, "16"),
    (matmul, dict(elem=9), INVALID, "elem"), (matmul, dict(n=-1), INVALID, "N"), (matmul, dict(f=0), INVALID, "F"),
    (matmul, dict(d=0), INVALID, "D"), (matmul, dict(d=(1 << 17) + 1), UNSUPPORTED, "131072"),
    (matmul, dict(f=(1 << 22) + 1), UNSUPPORTED, "2^22"), (matmul, dict(n=1 << 30), UNSUPPORTED, "2^30"),
    (matmul, dict(x=NULL), INVALID, "NULL"), (matmul, dict(w=NULL), INVALID, "NULL"),
    (matmul, dict(xs=NULL), INVALID, "NULL"), (matmul, dict(ws=NULL), INVALID, "NULL"),
    (matmul, dict(out=NULL), INVALID, "NULL"), (matmul, dict(ldx=24), INVALID, "16"), (matmul, dict(ldw=-16), INVALID, "16"),
    (matmul, dict(x=ODD), INVALID, "16"), (matmul, dict(w=ODD), INVALID, "16"),
    (matmul, dict(ldw=1 << 24), UNSUPPORTED, "2^23"),
    (linear, dict(elem=9), INVALID, "elem"), (linear, dict(out_elem=4), INVALID, "out_elem"),
    (linear, dict(n=-1), INVALID, "N"), (linear, dict(f=0), INVALID, "F"), (linear, dict(d=0), INVALID, "D"),
    (linear, dict(d=(1 << 17) + 1), UNSUPPORTED, "131072"), (linear, dict(f=(1 << 22) + 1), UNSUPPORTED, "2^22"),
    (linear, dict(x=NULL), INVALID, "NULL"), (linear, dict(w=NULL), INVALID, "NULL"),
    (linear, dict(ws=NULL), INVALID, "NULL"), (linear, dict(out=NULL), INVALID, "NULL"),
    (linear, dict(ldx=-8), INVALID, "strides"), (linear, dict(ldw=40), INVALID, "16"), (linear, dict(w=ODD), INVALID, "16"),
    (linear, dict(work=NULL), WORKSPACE, "NULL"), (linear, dict(size=100), WORKSPACE, "small"),
    (linear, dict(work=ODD), WORKSPACE, "aligned"),
]


@pytest.mark.parametrize("call,change,status,says", CASES,
                         ids=[f"{c[0].__name__}-{'-'.join(c[1])}-{i}" for i, c in enumerate(CASES)])
def test_refused(lib, codes, call, change, status, says):
    assert call(lib, **change) == codes[status]
    assert says in lib.gmmxx_hip_last_error().decode()


def test_no_rows(lib):
    assert embed(lib, n=0, table=NULL, index=NULL, out=NULL) == OK
    assert embed_back(lib, n=0, dy=NULL, out=NULL, ws=NULL, size=0) == OK
    assert drop(lib, n=0, x=NULL, out=NULL) == OK
    assert logp(lib, n=0, scores=NULL, index=NULL, chosen=NULL, ws=NULL, size=0) == OK
    assert logp_back(lib, n=0, stats=NULL, ds=NULL) == OK
    assert quantize(lib, n=0, x=NULL, values=NULL, scales=NULL) == OK
    assert matmul(lib, n=0, x=NULL, out=NULL) == OK
    assert linear(lib, n=0, x=NULL, out=NULL, work=NULL, size=0) == OK


def test_workspace_sizes(lib):
    assert lib.gmmxx_hip_embed_workspace_bytes(3, 0, 8) == -1
    assert lib.gmmxx_hip_embed_workspace_bytes(0, 9, 8) == 0
    for n in (1, 33, 5000, 10 ** 6):
        # two copies of tokens and positions
        assert lib.gmmxx_hip_embed_workspace_bytes(n, 1000, 8) >= 16 * n
    assert lib.gmmxx_hip_log_probs_workspace_bytes(3, 9, 10) == -1
    assert lib.gmmxx_hip_log_probs_workspace_bytes(0, 9, 2) == 0
    assert lib.gmmxx_hip_log_probs_workspace_bytes(100_000, 500, 0) == 0
    # rows of whole 128 bytes and a scale each, none where one kernel does it all
    assert lib.gmmxx_hip_quantized_linear_workspace_bytes(F32, 30, 0) == -1
    assert lib.gmmxx_hip_quantized_linear_workspace_bytes(BF16, 4, 4096) == 0
    assert lib.gmmxx_hip_quantized_linear_workspace_bytes(BF16, 300, 129) >= 300 * 260
    # a long row in parts: three statistics and the alternatives of each
    assert lib.gmmxx_hip_log_probs_workspace_bytes(1, 1 << 20, 5) >= 2 * (12 + 40)


def test_host_tensors_are_refused():
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    q = Quantized(torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3))
    for call in (lambda: gmmxx_amd.embed_rows(x, i), lambda: gmmxx_amd.dropout(x, 0.5, 1),
                 lambda: gmmxx_amd.log_probs(x, i), lambda: gmmxx_amd.quantize_rows(x),
                 lambda: gmmxx_amd.quantized_matmul(x, q)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: gmmxx_amd.embed_rows([1.0], i), lambda: gmmxx_amd.dropout(None, 0.5, 1),
                 lambda: gmmxx_amd.log_probs(3.0, i), lambda: gmmxx_amd.quantize_rows("x")):
        with pytest.raises(TypeError, match="torch.Tensor"):
            call()
    with pytest.raises(TypeError, match="Quantized"):
        gmmxx_amd.quantized_matmul(x, x)


# --- the native functions, with no rows -----------------------------------------------

LONGS = dict(dtype=torch.int64)


def native_embed(ops, t):
    return ops.embed(t(3, 4), torch.zeros(0, **LONGS), 1.0)


def native_dropout(ops, t):
    return ops.dropout(t(0, 4), t(0, 4), 0.5, 1, None, 0)


def native_log_probs(ops, t):
    return ops.log_probs(t(0, 4), torch.zeros(0, **LONGS), 2)[0]


OPERANDS = [(native_embed, 1), (native_dropout, 2), (native_log_probs, 1)]


@pytest.fixture(scope="module")
def ops():
    return experts._native()


def operands(change):
    made = []

    def make(*shape):
        made.append(torch.zeros(shape))
        return change(len(made) - 1, made[-1])
    return make


@pytest.mark.parametrize("call,which", [(c, i) for c, n in OPERANDS for i in range(n)],
                         ids=lambda v: getattr(v, "__name__", str(v)))
def test_forward_mode_is_refused(ops, call, which):
    with forward_ad.dual_level():
        dual = operands(lambda i, t: forward_ad.make_dual(t, torch.ones_like(t)) if i == which else t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(ops, dual)
    call(ops, operands(lambda i, t: t))


@pytest.mark.parametrize("call", [c for c, _ in OPERANDS], ids=lambda c: c.__name__)
def test_traces_are_refused(ops, call):
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(lambda first: call(ops, operands(lambda i, t: first if i == 0 else t)))(torch.zeros(0, 4))


def test_products_without_a_gradient_are_refused(ops):
    q, s = torch.zeros((3, 4), dtype=torch.int8), torch.zeros(3)
    x = torch.zeros((0, 4), requires_grad=True)
    for call in (lambda: ops.quantize(x), lambda: ops.quantized_matmul(x, None, q, s, None, torch.float32),
                 lambda: ops.quantized_matmul(x.detach(), None, q, s.clone().requires_grad_(), None, torch.float32),
                 lambda: ops.quantized_matmul(x.detach(), None, q, s, torch.zeros(3, requires_grad=True),
                                              torch.float32)):
        with pytest.raises(NotImplementedError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
