"""Builds ``libmeshb200.so`` (sm_100a) in-tree with nvcc, and ``_serving``, the
Python binding of its serving operators, with the host compiler where torch is
installed.

Usage: ``python -m grokking_abmod_b200.build`` (or ``build()`` from Python).
The library exports the C ABI declared in ``include/meshb200.h``.
"""

import glob
import hashlib
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmeshb200.so")
HEADER = os.path.join(ROOT, "include", "meshb200.h")
BINDING_SOURCE = os.path.join(CSRC, "binding.cpp")

SOURCES = ["gpt_model.cu", "mesh_ops.cu", "gemm_tc.cu", "simple_model.cu", "config.cpp", "data.cpp",
           "simple_config.cpp", "checkpoint.cpp", "cache_ops.cu", "cache_attention.cu", "logprobs.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def _older(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _stale():
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != "binding.cpp"]
    deps.append(HEADER)
    return _older(LIB, deps)


def _header_key():
    """What library and binding hold of the header that they were built from."""
    with open(HEADER, "rb") as f:
        return f"-DMB_HEADER_KEY=0x{hashlib.sha256(f.read()).hexdigest()[:16]}ull"


def _run(cmd, target, verbose):
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + res.stdout + res.stderr)
    os.replace(cmd[cmd.index("-o") + 1], target)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the library and the binding if any source is newer than them;
    returns the library's path.  Without torch there is no binding, which only
    ``ops`` of torch tensors needs."""
    build_library(force, verbose)
    try:
        import torch  # noqa: F401
    except ImportError:
        print("no torch: the library is built, its Python binding is not", file=sys.stderr)
        return LIB
    build_binding(force, verbose)
    return LIB


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compiles the library if any source is newer than it; returns its path."""
    if force or _stale():
        cmd = [_nvcc(), "-std=c++17", "-O3", "-lineinfo", "--threads", "0", *ARCH, "-shared", "-Xcompiler",
               "-fPIC,-ffp-contract=off",
               _header_key(), "-I", os.path.join(ROOT, "include"), "-o", LIB + ".tmp"]
        cmd += [os.path.join(CSRC, s) for s in SOURCES]
        cmd += ["-ldl"]
        _run(cmd, LIB, verbose)
    return LIB


def binding_path() -> str:
    """Where the binding of these sources, this torch and this Python is: its
    name says what it was built from, so another one is never taken for it."""
    import torch
    made = hashlib.sha256(f"{torch.__version__} {sysconfig.get_config_var('SOABI')}".encode())
    for name in (BINDING_SOURCE, HEADER):
        with open(name, "rb") as f:
            made.update(f.read())
    return os.path.join(HERE, f"_serving_{made.hexdigest()[:16]}.so")


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compiles the binding against the installed torch and the library (found
    beside it at run time) unless it is there; returns its path."""
    target = binding_path()
    if os.path.exists(target) and not force:
        return target
    import torch
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", _header_key(),
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(home, "include"),
           "-I", os.path.join(home, "include", "torch", "csrc", "api", "include"),
           "-I", os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"],
           BINDING_SOURCE, "-o", f"{target}.{os.getpid()}.o", "-L", HERE, "-l:libmeshb200.so", "-Wl,-rpath,$ORIGIN",
           "-L", os.path.join(home, "lib"), "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    _run(cmd, target, verbose)
    for old in glob.glob(os.path.join(HERE, "_serving*.so")):
        if old != target:
            os.remove(old)
    return target


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
