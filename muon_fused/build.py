"""Build the native library ``muon_fused/libfused_muon.so`` for sm_100a, and
``muon_fused/_step_ext.so``, which reads torch's tensors for it.

The library is plain CUDA C++ behind the C ABI of ``include/fused_muon.h``;
it links only the CUDA runtime (the tensor-map encoder is fetched from the
driver at run time), so it is built with nvcc directly rather than as a torch
extension.  The build is in-tree so the .so travels with the source tree.

Usage: ``python -m muon_fused.build`` (or ``build()`` from Python).
"""

from __future__ import annotations

import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfused_muon.so")
EXT = os.path.join(HERE, "_step_ext.so")
EXT_SOURCE = os.path.join(CSRC, "step_ext.cpp")
SOURCES = ["ns_capi.cu"]
DEPS = SOURCES + ["fm_ptx.cuh", "ns_gemm_sm100.cuh", "ns_gemm2_sm100.cuh", "ns_prep.cuh", "ns_fused_sm100.cuh", "ns_fused2_sm100.cuh",
                  "muon_elementwise.cuh", "adamw_list.cuh", "normed_update.cuh",
                  "ns_heads_sm100.cuh"]
HEADER = os.path.join(os.path.dirname(HERE), "include", "fused_muon.h")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-shared",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the fused_muon library needs the CUDA toolkit to build")
    return cand


def _stale(lib: str, deps) -> bool:
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(d) > t for d in [*deps, HEADER] if os.path.exists(d))


def _run(cmd, verbose: bool) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}):\n"
                           f"{res.stdout}\n{res.stderr}")
    if verbose:
        print(res.stdout + res.stderr)


def _build_ext(verbose: bool) -> None:
    """The CPython extension: C++ against the installed torch's headers."""
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    includes = [os.path.join(root, "include"),
                os.path.join(root, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    libs = os.path.join(root, "lib")
    tmp = EXT + ".tmp"
    _run([shutil.which("g++") or "c++", "-O2", "-std=c++20", "-fPIC", "-shared",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(f"-I{i}" for i in includes), EXT_SOURCE, "-o", tmp, f"-L{libs}", f"-Wl,-rpath,{libs}",
          "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"], verbose)
    os.replace(tmp, EXT)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile what is older than its sources; return the library's path."""
    if force or _stale(EXT, [EXT_SOURCE]):
        _build_ext(verbose)
    if force or _stale(LIB, [os.path.join(CSRC, d) for d in DEPS]):
        tmp = LIB + ".tmp"
        _run([_nvcc(), *NVCC_FLAGS, "-o", tmp] + [os.path.join(CSRC, s) for s in SOURCES], verbose)
        os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
