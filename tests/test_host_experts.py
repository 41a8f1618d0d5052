"""The sparsely gated layer's arguments, without a GPU: what the C ABI refuses and with
which status, that calls without rows return at once, what the Python functions refuse,
and that the native module of the autograd functions loads and binds.

No kernel is launched: every call here returns before any device work.
"""

import ctypes

import pytest
import torch

import gmmxx_amd
from gmmxx_amd import _hip, experts

F32, BF16, F16 = 0, 1, 2
OK = 0


@pytest.fixture(scope="module")
def lib():
    return _hip.load_library()


@pytest.fixture(scope="module")
def codes():
    import os
    import re
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "gmmxx_hip.h")).read()
    return {m[0]: int(m[1]) for m in re.findall(r"(GMMXX_[A-Z0-9_]+)\s*=\s*(-?\d+)", text)}


P = ctypes.c_void_p(4096)      # never read: the call ends before
NULL = ctypes.c_void_p(0)


def norm(lib, elem=F32, param=F32, n=3, d=8, x=P, ldx=8, eps=1e-5, y=P, mean=P, rstd=P):
    return lib.gmmxx_hip_layer_norm(elem, param, n, d, x, ldx, NULL, NULL, eps, y, mean, rstd, NULL)


def norm_back(lib, elem=F32, n=3, d=8, x=P, dy=P, lddy=8, dx=P, dw=P, ws=P, size=1 << 30):
    return lib.gmmxx_hip_layer_norm_backward(elem, elem, n, d, x, 8, dy, lddy, NULL, P, P, dx, dw, NULL, ws, size, NULL)


def route(lib, elem=F32, n=3, e=8, k=2, scores=P, ld=8, out=P, ws=P, size=1 << 30):
    return lib.gmmxx_hip_route(elem, n, e, k, 1, scores, ld, out, out, out, out, out, NULL, ws, size, NULL)


def route_back(lib, elem=F32, n=3, e=8, k=2, renormalize=1, scores=P, norm=P, ld=8, dgates=P):
    return lib.gmmxx_hip_route_backward(elem, n, e, k, renormalize, scores, ld, P, P, norm, dgates, P, NULL)


def grouped(lib, elem=F32, m=6, nx=3, e=4, k=8, n=8, x=P, ldx=8, rows=P, w=P, we=64, wk=8, wn=1, offsets=P, bits=32,
            out=P, out_elem=F32):
    return lib.gmmxx_hip_grouped_matmul(elem, m, nx, e, k, n, x, ldx, rows, w, we, wk, wn, NULL, offsets, bits, out,
                                        out_elem, NULL)


def grouped_back(lib, elem=F32, m=6, nx=3, e=4, k=8, n=8, rows=P, ldx=8, lddy=8, bits=32, dw=P, db=P, ws=P,
                 size=1 << 40):
    return lib.gmmxx_hip_grouped_weight_grad(elem, m, nx, e, k, n, P, ldx, rows, P, lddy, P, bits, dw, db, ws, size,
                                             NULL)


def combine(lib, elem=F32, n=3, k=2, e=4, f=8, y=P, y_elem=F32, ldy=8, slots=P, out=P):
    return lib.gmmxx_hip_combine(elem, n, k, e, f, y, y_elem, ldy, NULL, slots, P, out, NULL)


def combine_back(lib, elem=F32, n=3, k=2, e=4, f=8, ldy=8, gates=P, dout=P, lddout=8, dy=P):
    return lib.gmmxx_hip_combine_backward(elem, n, k, e, f, P, ldy, gates, P, P, dout, lddout, dy, P, NULL)


INVALID, UNSUPPORTED, WORKSPACE = "GMMXX_ERR_INVALID_ARGUMENT", "GMMXX_ERR_UNSUPPORTED", "GMMXX_ERR_WORKSPACE"

CASES = [
    (norm, dict(elem=7), INVALID, "elem"), (norm, dict(param=BF16), INVALID, "param_elem"),
    (norm, dict(n=-1), INVALID, "N"), (norm, dict(d=0), INVALID, "D"), (norm, dict(d=65537), UNSUPPORTED, "65536"),
    (norm, dict(eps=-1.0), INVALID, "eps"), (norm, dict(eps=float("nan")), INVALID, "eps"),
    (norm, dict(x=NULL), INVALID, "NULL"), (norm, dict(y=NULL), INVALID, "NULL"),
    (norm, dict(mean=NULL), INVALID, "NULL"), (norm, dict(ldx=-1), INVALID, "strides"),
    (norm_back, dict(dy=NULL), INVALID, "NULL"), (norm_back, dict(dx=NULL), INVALID, "NULL"),
    (norm_back, dict(lddy=-1), INVALID, "strides"), (norm_back, dict(ws=NULL), WORKSPACE, "NULL"),
    (norm_back, dict(size=8), WORKSPACE, "small"),
    (norm_back, dict(ws=ctypes.c_void_p(4100)), WORKSPACE, "aligned"),
    (route, dict(elem=-1), INVALID, "elem"), (route, dict(n=-1), INVALID, "N"), (route, dict(e=0), INVALID, "E"),
    (route, dict(k=0), INVALID, "k"), (route, dict(k=9), INVALID, "k"), (route, dict(e=4097), UNSUPPORTED, "4096"),
    (route, dict(e=100, k=65), UNSUPPORTED, "64"), (route, dict(n=1 << 29), UNSUPPORTED, "2^30"),
    (route, dict(scores=NULL), INVALID, "NULL"), (route, dict(out=NULL), INVALID, "NULL"),
    (route, dict(ld=-8), INVALID, "strides"), (route, dict(ws=NULL), WORKSPACE, "NULL"),
    (route, dict(size=1), WORKSPACE, "small"),
    (route_back, dict(dgates=NULL), INVALID, "NULL"), (route_back, dict(renormalize=0, norm=NULL), INVALID, "norm"),
    (route_back, dict(renormalize=0, scores=NULL), INVALID, "scores"), (route_back, dict(ld=-1), INVALID, "strides"),
    (grouped, dict(elem=3), INVALID, "elem"), (grouped, dict(out_elem=BF16), INVALID, "out_elem"),
    (grouped, dict(m=-1), INVALID, "M"), (grouped, dict(e=0), INVALID, "E"), (grouped, dict(k=0), INVALID, "K"),
    (grouped, dict(n=0), INVALID, "N"), (grouped, dict(nx=0), INVALID, "rows"),
    (grouped, dict(bits=16), INVALID, "offset_bits"), (grouped, dict(e=4097), UNSUPPORTED, "4096"),
    (grouped, dict(m=1 << 30), UNSUPPORTED, "2^30"), (grouped, dict(nx=1 << 31), UNSUPPORTED, "2^31"),
    (grouped, dict(k=(1 << 22) + 1), UNSUPPORTED, "2^22"), (grouped, dict(n=(1 << 22) + 1), UNSUPPORTED, "2^22"),
    (grouped, dict(x=NULL), INVALID, "NULL"), (grouped, dict(w=NULL), INVALID, "NULL"),
    (grouped, dict(offsets=NULL), INVALID, "NULL"), (grouped, dict(out=NULL), INVALID, "NULL"),
    (grouped, dict(wk=-8), INVALID, "strides"), (grouped, dict(wk=8, wn=2), INVALID, "1"),
    (grouped, dict(rows=NULL), INVALID, "fewer rows"),
    (grouped_back, dict(dw=NULL, db=NULL), INVALID, "NULL"), (grouped_back, dict(lddy=-1), INVALID, "strides"),
    (grouped_back, dict(rows=NULL), INVALID, "fewer rows"), (grouped_back, dict(bits=0), INVALID, "offset_bits"),
    (grouped_back, dict(m=4096, nx=4096, ws=NULL), WORKSPACE, "NULL"),
    (grouped_back, dict(m=4096, nx=4096, size=16), WORKSPACE, "small"),
    (combine, dict(elem=5), INVALID, "elem"), (combine, dict(y_elem=F16), INVALID, "y_elem"),
    (combine, dict(n=-1), INVALID, "N"), (combine, dict(k=0), INVALID, "k"), (combine, dict(k=65), UNSUPPORTED, "64"),
    (combine, dict(f=0), INVALID, "F"), (combine, dict(f=(1 << 22) + 1), UNSUPPORTED, "2^22"),
    (combine, dict(n=1 << 29), UNSUPPORTED, "2^30"), (combine, dict(y=NULL), INVALID, "NULL"),
    (combine, dict(slots=NULL), INVALID, "NULL"), (combine, dict(out=NULL), INVALID, "NULL"),
    (combine, dict(ldy=-1), INVALID, "strides"),
    (combine_back, dict(gates=NULL), INVALID, "NULL"), (combine_back, dict(dout=NULL), INVALID, "NULL"),
    (combine_back, dict(dy=NULL), INVALID, "NULL"), (combine_back, dict(lddout=-2), INVALID, "strides"),
]


@pytest.mark.parametrize("call,change,status,says", CASES,
                         ids=[f"{c[0].__name__}-{'-'.join(c[1])}-{i}" for i, c in enumerate(CASES)])
def test_refused(lib, codes, call, change, status, says):
    assert call(lib, **change) == codes[status]
    assert says in lib.gmmxx_hip_last_error().decode()


def test_no_rows(lib):
    assert norm(lib, n=0, x=NULL, y=NULL) == OK
    assert norm_back(lib, n=0, x=NULL, dy=NULL, dx=NULL, ws=NULL, size=0) == OK
    assert route(lib, n=0, scores=NULL, out=NULL, ws=NULL, size=0) == OK
    assert route_back(lib, n=0, dgates=NULL) == OK
    assert grouped(lib, m=0, nx=0, x=NULL, out=NULL) == OK
    assert grouped_back(lib, m=0, nx=0, dw=NULL, db=NULL, ws=NULL, size=0) == OK
    assert combine(lib, n=0, y=NULL, out=NULL) == OK
    assert combine_back(lib, n=0, dout=NULL, dy=NULL) == OK


def test_workspace_sizes(lib):
    assert lib.gmmxx_hip_layer_norm_workspace_bytes(3, 0) == -1
    assert lib.gmmxx_hip_layer_norm_workspace_bytes(3, 65537) == -1
    assert lib.gmmxx_hip_route_workspace_bytes(3, 8, 9) == -1
    assert lib.gmmxx_hip_grouped_workspace_bytes(3, 0, 8, 8) == -1
    for n in (0, 1, 1000, 10 ** 6):
        # partial sums of weight and bias: two floats a column for each workgroup
        assert lib.gmmxx_hip_layer_norm_workspace_bytes(n, 100) % 800 == 0
        assert lib.gmmxx_hip_route_workspace_bytes(n, 8, 2) >= 8 * 4
    # one product needs none; many rows of one small matrix are cut into parts
    assert lib.gmmxx_hip_grouped_workspace_bytes(64, 4096, 8, 8) == 0
    assert lib.gmmxx_hip_grouped_workspace_bytes(1 << 20, 1, 8, 8) >= 2 * 8 * 8 * 4


def test_native_module_binds(lib):
    ops = experts._native()
    assert ops.__file__.endswith("_autograd.so") and ops is experts._native()


def test_host_tensors_are_refused():
    x = torch.zeros(4, 8)
    ints = torch.zeros(4, 2, dtype=torch.int32)
    routing = gmmxx_amd.Routing(ints, torch.zeros(4, 2), torch.zeros(9, dtype=torch.int32), ints.view(-1), ints)
    for call in (lambda: gmmxx_amd.layer_norm(x), lambda: gmmxx_amd.route_rows(x, 2),
                 lambda: gmmxx_amd.grouped_matmul(x, torch.zeros(8, 8, 8), routing),
                 lambda: gmmxx_amd.combine_rows(torch.zeros(8, 8), routing)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: gmmxx_amd.layer_norm([1.0]), lambda: gmmxx_amd.route_rows(None, 1)):
        with pytest.raises(TypeError, match="torch.Tensor"):
            call()


def test_failures_are_the_packages_own():
    with pytest.raises((_hip.HipRuntimeError, _hip.HipRuntimeFallback), match="status 3"):
        experts._failed(RuntimeError("gmmxx_hip_route failed (status 3): x\nException raised from check"))
    with pytest.raises(RuntimeError, match="out of memory"):
        experts._failed(RuntimeError("out of memory"))


def test_library_without_the_entry_points(tmp_path):
    import subprocess
    src = tmp_path / "old.c"
    src.write_text("int gmmxx_hip_abi_version(void) { return 2; }\n")
    old = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(old), str(src)], check=True)
    with pytest.raises(_hip.HipBackendUnavailable, match="Build it"):
        _hip.load_library(str(old))
