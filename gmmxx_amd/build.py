"""Builds libgmmxx_hip.so for gfx950 in-tree with hipcc.

    python -m gmmxx_amd.build          # or: from gmmxx_amd.build import build; build()

Each translation unit is compiled separately (in parallel) and linked into a
shared library next to this file, where ``gmmxx_amd._hip`` loads it.  The
autograd functions of ``gmmxx_amd.experts`` are a Python extension beside it,
``_autograd.so``, compiled against the installed torch; where a C++ compiler, torch
or Python's headers are missing, the library is built without it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from typing import Optional

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
BUILD_DIR = os.path.join(PKG_DIR, "_build")
LIB_PATH = os.path.join(PKG_DIR, "libgmmxx_hip.so")
AUTOGRAD_PATH = os.path.join(PKG_DIR, "_autograd.so")
SOURCES = ("em_tile.hip", "em_sph_bf16.hip", "em_fused.hip", "em_coop.hip", "em_one.hip", "em_label.hip", "em_full_wide.hip", "em_full_stats.hip", "em_full_infer.hip",
           "params.hip",
           "kmeans.hip", "abi.hip",
           "layer_norm.hip", "route.hip", "grouped.hip", "grouped_bf16.hip", "grouped_f16.hip", "grouped_f32.hip", "grouped_few.hip", "combine.hip", "experts_abi.hip")
ARCH = os.environ.get("GMMXX_HIP_ARCH", "gfx950")

# -packed-fp32-ops: keep the compiler from emitting packed fp32 VALU ops.
COMMON_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I", CSRC, "-I", os.path.join(ROOT, "include"),
]
# The tile kernels' logits are finite or -inf: no NaN canonicalisation around
# min/max there.  Kept off elsewhere (the Cholesky kernel tests for NaN pivots).
EXTRA_FLAGS = {"em_tile.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"],
               "em_sph_bf16.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"],
               "em_fused.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"],
               "em_coop.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"],
               "em_one.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"],
               "em_label.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"]}


def _hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found; the HIP library cannot be built")
    return path


def _compile(src: str) -> str:
    obj = os.path.join(BUILD_DIR, os.path.splitext(src)[0] + ".o")
    cmd = [_hipcc(), *COMMON_FLAGS, *EXTRA_FLAGS.get(src, []), "-c", os.path.join(CSRC, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{res.stderr}")
    return obj


def _cxx() -> Optional[str]:
    return shutil.which("g++") or shutil.which("c++")


def _autograd_lacks() -> Optional[str]:
    """What the autograd extension needs and this host does not have."""
    if _cxx() is None:
        return "a C++ compiler"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers"
    try:
        import torch.utils.cpp_extension  # noqa: F401
    except ImportError:
        return "torch"
    return None


def _build_autograd() -> None:
    """Compile csrc/autograd.cpp (host code only) into _autograd.so."""
    import torch
    from torch.utils import cpp_extension

    tmp = AUTOGRAD_PATH + ".tmp"
    cmd = [_cxx(), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(ROOT, "include"),
           *(a for p in cpp_extension.include_paths() for a in ("-isystem", p)),
           "-isystem", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"),
           "-isystem", sysconfig.get_paths()["include"], os.path.join(CSRC, "autograd.cpp"), "-o", tmp,
           *("-L" + p for p in cpp_extension.library_paths()),
           "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on autograd.cpp:\n{res.stderr}")
    os.replace(tmp, AUTOGRAD_PATH)


def build(verbose: bool = False) -> str:
    """Compile every HIP translation unit and link libgmmxx_hip.so, and the autograd
    extension; returns the library's path.

    The library does not depend on the extension: it is in place before an error of the
    extension's is raised, and a host that lacks what only the extension needs gets a
    warning.  An extension of an earlier build is taken away then: it may not fit."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    lacks = _autograd_lacks()
    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        extension = None if lacks else ex.submit(_build_autograd)
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB_PATH + ".tmp"
    cmd = [_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    if (extension is None or extension.exception()) and os.path.exists(AUTOGRAD_PATH):
        os.remove(AUTOGRAD_PATH)
    if extension is None:
        warnings.warn(f"{os.path.basename(AUTOGRAD_PATH)} is not built for want of {lacks}; gmmxx_amd.experts needs it",
                      RuntimeWarning, stacklevel=2)
    else:
        extension.result()
    if verbose:
        print(f"built {LIB_PATH}" + ("" if lacks else f" and {AUTOGRAD_PATH}"))
    return LIB_PATH


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
