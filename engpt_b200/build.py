"""Build ``libengpt_b200.so`` (all CUDA sources under ``csrc/``) for sm_100a and the torch binding ``_native.so``.

The library is built in-tree next to this file so that it travels with the
source tree.  ``python -m engpt_b200.build`` (or ``build()``) recompiles the
objects whose sources or headers changed and relinks.  Without torch (``python
engpt_b200/build.py``) the library alone is built.
"""

from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libengpt_b200.so")
NATIVE = os.path.join(HERE, "_native.so")     # Python module of csrc/bindings.cpp, linked against LIB

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-rdc=true",
    "-I" + INCLUDE,
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build engpt_b200")
    return path


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _compile(src: str, verbose_ptxas: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src).replace(".cu", ".o"))
    cmd = [nvcc(), *NVCC_FLAGS, "-c", src, "-o", obj]
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    if verbose_ptxas:
        sys.stderr.write(res.stderr)
    return obj


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    newest_header = max((os.path.getmtime(h) for h in _headers()), default=0.0)
    todo = []
    for s in srcs:
        obj = os.path.join(BUILD, os.path.basename(s).replace(".cu", ".o"))
        if force or verbose_ptxas or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(s),
                                                                                           newest_header):
            todo.append(s)
    with cf.ThreadPoolExecutor(max_workers=max(1, min(len(todo), os.cpu_count() or 1))) as ex:
        list(ex.map(lambda s: _compile(s, verbose_ptxas), todo))
    objs = [os.path.join(BUILD, os.path.basename(s).replace(".cu", ".o")) for s in srcs]
    if todo or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", tmp, *objs,
               "-Xcompiler", "-fPIC"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    if importlib.util.find_spec("torch") is not None:   # the library alone, for callers of the C ABI, needs no torch
        build_native(force)
    return LIB


def build_native(force: bool = False) -> str:
    """The torch binding ``engpt_b200._native`` (host code only), for the running interpreter and its torch."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    src = os.path.join(CSRC, "bindings.cpp")
    newest = max(os.path.getmtime(p) for p in (src, os.path.join(INCLUDE, "engpt_b200.h"), torch.__file__))
    if not force and os.path.exists(NATIVE) and os.path.getmtime(NATIVE) >= newest:
        return NATIVE
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda_include = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    includes = [*cpp_extension.include_paths(), cuda_include, sysconfig.get_paths()["include"]]
    tmp = NATIVE + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in includes), src, "-o", tmp,
           f"-L{HERE}", "-l:libengpt_b200.so", f"-L{torch_lib}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, NATIVE)
    return NATIVE


if __name__ == "__main__":
    force = "--force" in sys.argv
    print(build(force=force, verbose_ptxas="-v" in sys.argv))
