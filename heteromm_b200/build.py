"""Builds the native libraries of heteromm_b200 in-tree.

  lib/libheteromm_cuda.so   the C ABI (include/heteromm_cuda.h) and its sm_100a
                            kernels, compiled by nvcc from csrc/*.cu
  lib/libheteromm_steps.so  the C++17 heteromm step API (include/heteromm/dev),
                            CPU bodies and GPU adapters (src/*.cpp), linked
                            to the former
  lib/heteromm_cpp_kernels<ext>  Python bindings of the steps under the names the
                            reference's pipeline generator calls
                            (src/py/heteromm_cpp_kernels.cpp, pybind11)
  lib/heteromm_serve_calls-<torch>-<sources><ext>  the serving entry points called with
                            torch tensors (src/py/serve_calls.cpp, torch's headers)

nvcc cross-compiles for sm_100a without a GPU; the built .so files travel with
the repository snapshot to the GPU machine.
"""
from __future__ import annotations

import contextlib
import glob
import hashlib
import os
import subprocess
import sys
import threading

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
INC = os.path.join(ROOT, "include")
LIB_DIR = os.path.join(PKG, "lib")
CUDA_LIB = os.path.join(LIB_DIR, "libheteromm_cuda.so")
STEPS_LIB = os.path.join(LIB_DIR, "libheteromm_steps.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _newer(target: str, sources: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _run(cmd: list[str]) -> None:
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout)
        raise RuntimeError(f"build failed: {' '.join(cmd[:3])} ... (exit {r.returncode})")


def build_cuda(force: bool = False, verbose: bool = False) -> str:
    srcs = sorted(glob.glob(os.path.join(PKG, "csrc", "*.cu")))
    deps = srcs + glob.glob(os.path.join(PKG, "csrc", "*.cuh")) + [os.path.join(INC, "heteromm_cuda.h")]
    if force or _newer(CUDA_LIB, deps):
        os.makedirs(LIB_DIR, exist_ok=True)
        cmd = [NVCC, f"--threads={os.cpu_count() or 1}", *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
               f"-I{INC}", "-o", CUDA_LIB, *srcs]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        _run(cmd)
    return CUDA_LIB


def build_steps(force: bool = False) -> str:
    srcs = sorted(glob.glob(os.path.join(PKG, "src", "*.cpp")))
    if not srcs:
        return ""
    deps = srcs + glob.glob(os.path.join(PKG, "src", "*.h")) + \
        glob.glob(os.path.join(INC, "heteromm", "**", "*.h"), recursive=True) + [CUDA_LIB]
    if force or _newer(STEPS_LIB, deps):
        cmd = ["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-fPIC", "-shared", "-Wall",
               "-Wextra", f"-I{INC}",
               "-I/usr/local/cuda/include", "-o", STEPS_LIB, *srcs, f"-L{LIB_DIR}",
               "-lheteromm_cuda", "-Wl,-rpath,$ORIGIN", "-L/usr/local/cuda/lib64", "-lcudart"]
        _run(cmd)
    return STEPS_LIB


def py_kernels_path() -> str:
    import sysconfig
    return os.path.join(LIB_DIR, "heteromm_cpp_kernels" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_py_kernels(force: bool = False) -> str:
    """The pybind11 module heteromm_cpp_kernels, linked to the step library."""
    import sysconfig
    try:
        import pybind11
    except ImportError:   # bindings are optional; the C ABI and step API stand alone
        return ""
    src = os.path.join(PKG, "src", "py", "heteromm_cpp_kernels.cpp")
    out = py_kernels_path()
    deps = [src, STEPS_LIB, os.path.join(PKG, "src", "packed.h")] + \
        glob.glob(os.path.join(INC, "heteromm", "**", "*.h"), recursive=True)
    if force or _newer(out, deps):
        cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden",
               f"-I{pybind11.get_include()}", f"-I{sysconfig.get_paths()['include']}",
               f"-I{INC}", f"-I{os.path.join(PKG, 'src')}", "-o", out, src, f"-L{LIB_DIR}",
               "-lheteromm_steps", "-Wl,-rpath,$ORIGIN"]
        _run(cmd)
    return out


def _serve_calls_sources() -> list[str]:
    return [os.path.join(PKG, "src", "py", "serve_calls.cpp"), os.path.join(INC, "heteromm_cuda.h")]


def _serve_calls_name(digest: str) -> str:
    """The module's file for this torch, this Python and sources of this digest: one built for
    or from others has another name."""
    import sysconfig
    import torch
    return os.path.join(LIB_DIR, f"heteromm_serve_calls-torch{torch.__version__.replace('+', '_')}-"
                                 f"{digest}{sysconfig.get_config_var('EXT_SUFFIX')}")


def _built_serve_calls() -> list[str]:
    """Those built for this torch and Python, from whatever sources."""
    before, after = _serve_calls_name("*").split("*")
    return sorted(glob.glob(glob.escape(before) + "*" + glob.escape(after)))


def serve_calls_path() -> str:
    """Where the module for this torch, this Python and these sources is or will be; without
    the sources, the one that was built ("" if there is none)."""
    if not all(map(os.path.exists, _serve_calls_sources())):
        return (_built_serve_calls() or [""])[-1]
    digest = hashlib.sha256()
    for f in _serve_calls_sources():
        with open(f, "rb") as src:
            digest.update(src.read())
    return _serve_calls_name(digest.hexdigest()[:12])


def build_serve_calls(force: bool = False) -> str:
    """The module heteromm_serve_calls; torch's own libraries are loaded when it is.  "" where
    torch's headers or its CUDA library are not: the C ABI does not need them."""
    import sysconfig
    try:
        import torch
    except ImportError:
        return ""
    out = serve_calls_path()
    if out == "" or (not force and os.path.exists(out)):
        return out
    home = os.path.dirname(torch.__file__)
    include, lib = os.path.join(home, "include"), os.path.join(home, "lib")
    if not os.path.exists(os.path.join(include, "torch", "csrc", "Exceptions.h")) or \
            not os.path.exists(os.path.join(lib, "libc10_cuda.so")):
        return ""
    os.makedirs(LIB_DIR, exist_ok=True)
    # (renamed when it is whole: another process may look for it, or build it too)
    part = f"{out}.{os.getpid()}.{threading.get_ident()}"
    try:
        _run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall",
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
              f"-isystem{include}", f"-isystem{os.path.join(include, 'torch', 'csrc', 'api', 'include')}",
              "-I/usr/local/cuda/include", f"-I{sysconfig.get_paths()['include']}", f"-I{INC}", "-o", part,
              _serve_calls_sources()[0], f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10",
              "-lc10_cuda"])
        os.replace(part, out)
    finally:
        if os.path.exists(part):
            os.remove(part)
    for old in _built_serve_calls():   # from older sources
        if old != out:
            with contextlib.suppress(FileNotFoundError):
                os.remove(old)
    return out


def build(force: bool = False) -> None:
    build_cuda(force)
    build_steps(force)
    build_py_kernels(force)
    build_serve_calls(force)


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(CUDA_LIB)
