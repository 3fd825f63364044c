"""Build recipe for libb2attn.so (sm_100a only) and the Python module _serving
that binds its serving operators to torch tensors, written next to this file.

    python -m npu_b200.build            # build if sources are newer
    python -m npu_b200.build --force    # rebuild
    python -m npu_b200.build --verbose  # also print ptxas register/smem usage

The library is compiled ahead of time into the package directory so that it
travels with the source tree; nothing is JIT-compiled at import time.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libb2attn.so"
BUILD_DIR = PKG / "_build"
BINDING = PKG / "_serving.so"
BINDING_SOURCE = CSRC / "serving_binding.cpp"

SOURCES = ["capi.cu", "capi_serving.cu", "prefill.cu", "prefill_pair.cu", "prefill_d256.cu",
           "prefill_packed_d64.cu", "decode.cu", "decode_noalloc.cu", "rope_append.cu", "rope_append_paged.cu",
           "decode_paged.cu", "sample.cu", "diag.cu", "host_pipeline.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FAST_MATH = ["--use_fast_math"]
# The same without its replacement of expf and the like by approximations.
FLUSH_ONLY = ["--ftz=true", "--prec-div=false", "--prec-sqrt=false"]
MATH_FLAGS = {"sample.cu": FLUSH_ONLY}
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-I", str(INCLUDE), "-I", str(CSRC),
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put CUDA's bin directory on PATH")


def _stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h")) + [Path(__file__)]
    return any(p.stat().st_mtime > t for p in deps)


def _build_binding(force: bool) -> None:
    """Compile the torch binding against libb2attn.so (found beside it at run time)."""
    deps = [BINDING_SOURCE, INCLUDE / "b2attn.h", Path(__file__)]
    if not force and BINDING.exists() and all(p.stat().st_mtime <= BINDING.stat().st_mtime for p in deps):
        return
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    nvcc = Path(_nvcc()).resolve()
    tmp = BINDING.with_suffix(".so.tmp")
    # The host compiler that nvcc takes, and torch's libstdc++: a compiler whose own is static would put a second
    # C++ runtime into the process (CXX named one here), whose locale nobody sets up.
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w",
           "-I", str(INCLUDE), "-isystem", str(root / "include"),
           "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(nvcc.parent.parent / "include"),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           str(BINDING_SOURCE), "-o", str(tmp), "-L", str(PKG), "-l:libb2attn.so", "-L", str(root / "lib"),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-l:libstdc++.so.6",
           "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building {BINDING.name} failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every .cu under csrc/ for sm_100a, link libb2attn.so and build the torch binding."""
    if force or _stale():
        _build_library(verbose)
    _build_binding(force)
    return LIB


def _build_library(verbose: bool) -> None:
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []
    for src in SOURCES:
        obj = BUILD_DIR / (Path(src).stem + ".o")
        cmd = [nvcc, *ARCH, *NVCC_FLAGS, *MATH_FLAGS.get(src, FAST_MATH), "-c", str(CSRC / src), "-o", str(obj)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, file=sys.stderr)
        objs.append(str(obj))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH, "-shared", "-o", str(tmp), *objs, "-Xcompiler", "-fPIC"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
