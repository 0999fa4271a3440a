"""Builds libstlq_b200.so in-tree for sm_100a (nvcc; no JIT cache, so the library travels with the repo).

    python -m stlq_b200.build            # incremental
    python -m stlq_b200.build --force    # rebuild everything

It also builds _operators.so, the Python binding of the routed 8-bit operators, against the installed torch.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libstlq_b200.so")
BINDING = os.path.join(HERE, "binding", "operators.cpp")
BINDING_OUT = os.path.join(HERE, "_operators.so")
OBJDIR = os.path.join(HERE, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC = os.environ.get("NVCC", shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc")
HOST_CXX = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
# No --use_fast_math: the kernels rely on IEEE division / square root and on denormals, like
# the reference's host build.
NVFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-ccbin", HOST_CXX, "--expt-relaxed-constexpr"]


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cpp")))


def _stale(obj, deps):
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJDIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(HERE, "..", "include", "stlq_b200.h"))
    objs = []
    for src in sources():
        path = os.path.join(CSRC, src)
        obj = os.path.join(OBJDIR, src + ".o")
        objs.append(obj)
        if force or _stale(obj, [path] + headers):
            cmd = [NVCC, *ARCH, *NVFLAGS, "-c", path, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
    if force or _stale(OUT, objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", OUT, *objs, "-ccbin", HOST_CXX]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    return OUT


def built_for() -> str:
    """The torch and the Python that a binding built now is for; it shares C++ objects with the one and the ABI of the other."""
    from importlib import metadata

    try:
        torch_version = metadata.version("torch")
    except metadata.PackageNotFoundError:  # a torch that was not installed as a package
        from torch import __version__ as torch_version
    return f"torch {torch_version}, {sys.implementation.cache_tag}"


def _read(path):
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return None


def build_binding(force: bool = False, verbose: bool = False) -> str:
    header = os.path.join(HERE, "..", "include", "stlq_b200.h")
    os.makedirs(OBJDIR, exist_ok=True)
    stamp = os.path.join(OBJDIR, "operators.for")
    if force or _stale(BINDING_OUT, [BINDING, header]) or _read(stamp) != built_for():
        import importlib.util

        torch_dir = os.path.dirname(importlib.util.find_spec("torch").origin)
        inc, lib = os.path.join(torch_dir, "include"), os.path.join(torch_dir, "lib")
        cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(NVCC))), "include")
        cmd = [HOST_CXX, "-O2", "-std=c++17", "-shared", "-fPIC", f'-DSTLQ_BUILT_FOR="{built_for()}"', BINDING, "-o", BINDING_OUT, "-I", inc, "-I",
               os.path.join(inc, "torch", "csrc", "api", "include"), "-I", sysconfig.get_path("include"), "-I", cuda, "-L", lib,
               "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,-rpath," + lib]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        with open(stamp, "w") as f:
            f.write(built_for())
    return BINDING_OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    build_binding(force="--force" in sys.argv, verbose=True)
