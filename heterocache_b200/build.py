"""Build the sm_100a shared library in-tree (``heterocache_b200/libhcb200.so``)
and the Python binding of the paged operators (``heterocache_b200/_paged.so``).

    python -m heterocache_b200.build

Compiles every ``csrc/*.cu`` for ``sm_100a`` with nvcc (one object per source,
compiled in parallel) and links them into one shared library exporting the C
ABI of ``include/heterocache_b200.h``; then ``csrc/binding.cpp`` with the host
compiler, against torch's headers and that library (found beside it when it is
loaded).  No GPU is needed to build.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(PKG, "libhcb200.so")
BINDING = os.path.join(CSRC, "binding.cpp")
BINDING_OUT = os.path.join(PKG, "_paged.so")
BINDING_NOTE = os.path.join(PKG, "_paged.built")  # what _paged.so was built for
OBJ_DIR = os.path.join(PKG, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMPILE_FLAGS = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + [os.path.join(INCLUDE, "heterocache_b200.h"),
                                                                  os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("build failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
    return res


def _binding_for() -> str:
    """What a binding belongs to: the torch and the Python it is built with."""
    import torch
    return (f"torch {torch.__version__} {torch.version.git_version} cxx11_abi {int(torch.compiled_with_cxx11_abi())} "
            f"{sys.implementation.cache_tag}\n")


def binding_built_for_another() -> bool:
    """Whether the note beside the binding names another torch or Python."""
    try:
        with open(BINDING_NOTE) as f:
            return f.read() != _binding_for()
    except OSError:
        return False  # no note


def _binding_stale() -> bool:
    if not os.path.exists(BINDING_OUT) or not os.path.exists(BINDING_NOTE) or binding_built_for_another():
        return True
    t = os.path.getmtime(BINDING_OUT)
    deps = [BINDING, os.path.join(INCLUDE, "heterocache_b200.h"), os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def _build_binding(verbose: bool) -> None:
    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    system = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
              os.path.join(cuda, "include")]
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I" + INCLUDE,
          "-I" + sysconfig.get_paths()["include"], *(x for d in system for x in ("-isystem", d)), BINDING,
          "-o", BINDING_OUT + ".tmp", "-L" + os.path.join(base, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
          "-ltorch_python", "-L" + PKG, "-l:" + os.path.basename(OUT), "-Wl,-rpath,$ORIGIN"], verbose)
    if os.path.exists(BINDING_NOTE):
        os.remove(BINDING_NOTE)  # (a build that is cut off here leaves a stale binding, not a wrong note)
    os.replace(BINDING_OUT + ".tmp", BINDING_OUT)
    with open(BINDING_NOTE, "w") as f:
        f.write(_binding_for())


def build(force: bool = False, verbose: bool = False) -> str:
    if force or _stale():
        _build_library(verbose)
    if force or _binding_stale():
        _build_binding(verbose)
    return OUT


def _build_library(verbose: bool) -> None:
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sources()
    objs = [os.path.join(OBJ_DIR, os.path.basename(s)[:-3] + ".o") for s in srcs]
    cmds = [[nvcc, *COMPILE_FLAGS, "-I" + INCLUDE, "-c", s, "-o", o] for s, o in zip(srcs, objs)]
    with ThreadPoolExecutor(max_workers=max(1, min(len(cmds), os.cpu_count() or 1))) as ex:
        list(ex.map(lambda c: _run(c, verbose), cmds))
    _run([nvcc, *ARCH, "-shared", "-o", OUT + ".tmp", *objs], verbose)
    os.replace(OUT + ".tmp", OUT)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
