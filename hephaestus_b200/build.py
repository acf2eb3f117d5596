"""Build ``libheph_b200.so`` in-tree with nvcc for sm_100a.

Every translation unit under ``csrc/`` is compiled to an object in
``_build/`` (in parallel, skipping up-to-date objects) and linked into
``hephaestus_b200/libheph_b200.so``; ``csrc/torch_rows.cpp`` is compiled with
the host compiler against torch's headers and linked with that library into
the CPython module ``hephaestus_b200/_torch_rows.so``.  Runs without a GPU (nvcc
cross-compiles).  ``python hephaestus_b200/build.py [--verbose-ptxas]``.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libheph_b200.so")
TORCH_MODULE = os.path.join(PKG, "_torch_rows.so")
INCLUDE = os.path.join(ROOT, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++20", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-Wall", "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    inc = os.path.join(INCLUDE, "heph")
    hs += [os.path.join(inc, f) for f in os.listdir(inc)]
    return hs


def _compile(src: str, verbose_ptxas: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    newest_dep = max(os.path.getmtime(p) for p in [src, __file__] + headers())
    if os.path.exists(obj) and os.path.getmtime(obj) >= newest_dep and not verbose_ptxas:
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", src, "-o", obj]
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stderr}")
    if verbose_ptxas:
        sys.stderr.write(res.stderr)
    return obj


def build_torch_module(force: bool = False) -> str | None:
    """``_torch_rows.so``: the torch boundary of the row operators, beside LIB.

    None, and no module, without a CUDA build of torch: LIB does not need one.
    Where it does not compile, none is left of older sources either."""
    src = os.path.join(CSRC, "torch_rows.cpp")
    spec = importlib.util.find_spec("torch")
    torch_dir = os.path.dirname(spec.origin) if spec else ""
    if not os.path.exists(os.path.join(torch_dir, "include", "c10", "cuda", "CUDAStream.h")):
        return None
    newest_dep = max(os.path.getmtime(p) for p in [src, __file__, spec.origin] + headers())
    if os.path.exists(TORCH_MODULE) and os.path.getmtime(TORCH_MODULE) >= newest_dep and not force:
        return TORCH_MODULE
    import torch

    cuda_home = os.path.dirname(os.path.dirname(nvcc()))
    lib_dir = os.path.join(torch_dir, "lib")
    tmp = TORCH_MODULE + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++20", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-I", INCLUDE, "-isystem", os.path.join(torch_dir, "include"),
           "-isystem", os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda_home, "include"),
           src, "-o", tmp, "-L", PKG, "-l:libheph_b200.so", "-L", lib_dir, "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{lib_dir}"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        if os.path.exists(TORCH_MODULE):
            os.remove(TORCH_MODULE)
        raise RuntimeError(f"{cmd[0]} failed on {src}:\n{res.stderr}")
    os.replace(tmp, TORCH_MODULE)
    return TORCH_MODULE


def _torch_module_or_note(force: bool = False) -> None:
    """build_torch_module, or a line on stderr that says why it is left out: LIB is complete without it."""
    try:
        made = build_torch_module(force)
        why = "no CUDA build of torch is installed"
    except (RuntimeError, OSError, ImportError) as e:
        made, why = None, str(e)
    if made is None:
        sys.stderr.write(f"{os.path.basename(TORCH_MODULE)} (torch_ops' row operators) is left out: {why}\n")


def build(verbose_ptxas: bool = False, force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    if force:
        for f in os.listdir(BUILD):
            os.remove(os.path.join(BUILD, f))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose_ptxas), srcs))
    if (os.path.exists(LIB) and not force and
            os.path.getmtime(LIB) >= max(os.path.getmtime(o) for o in objs)):
        _torch_module_or_note()
        return LIB
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB)
    _torch_module_or_note(force)
    return LIB


if __name__ == "__main__":
    print(build(verbose_ptxas="--verbose-ptxas" in sys.argv, force="--force" in sys.argv))
