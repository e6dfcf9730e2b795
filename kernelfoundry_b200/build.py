"""Build libkf_attn.so (sm_100a only) and _kf_host-*.so in-tree.

    python -m kernelfoundry_b200.build [--verbose]

nvcc cross-compiles for B200 without a GPU.  The library links the static CUDA
runtime and reaches the driver only through cudaGetDriverEntryPoint, so it
loads (and its argument checks run) on machines without a GPU driver.  _kf_host-*.so is the
host side of the small operators' Python calls (csrc/kf_host.cpp), built against the installed
torch.  It needs Python's and torch's headers; the library does not, and is built (and used from C)
without them.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

import torch

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.environ.get("KF_LIB_PATH") or os.path.join(LIB_DIR, "libkf_attn.so")
# Beside the library; named after the torch and the Python whose binary interfaces it is built against.
HOST_PATH = os.path.join(os.path.dirname(os.path.abspath(LIB_PATH)),
                         f"_kf_host-torch{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}")
HOST_SOURCE = os.path.join(CSRC, "kf_host.cpp")
SOURCES = ["kf_api.cu"]
HEADERS = ["kf_ptx.cuh", "prefill_sm100.cuh", "decode_sm100.cuh", "pointwise_sm100.cuh", "peer_sm100.cuh",
           "synth_sm100.cuh", "cache_sm100.cuh", "decode_q4_sm100.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    "-cudart", "static",
]


def _nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def needs_rebuild() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS]
    deps += [os.path.join(REPO_DIR, "include", h) for h in ("kf_attn.h", "kf_cache.h", "kf_pointwise.h", "kf_synth.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build_host(force: bool = False) -> str:
    built = os.path.exists(HOST_PATH)
    if built and os.path.getmtime(HOST_PATH) < os.path.getmtime(HOST_SOURCE):
        os.remove(HOST_PATH)                               # never loaded again, even if the build fails
    elif built and not force:
        return HOST_PATH
    os.makedirs(os.path.dirname(HOST_PATH), exist_ok=True)
    base, tmp = os.path.dirname(torch.__file__), HOST_PATH + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I" + sysconfig.get_paths()["include"],
           "-isystem", os.path.join(base, "include"),
           "-isystem", os.path.join(base, "include", "torch", "csrc", "api", "include"),
           "-o", tmp, HOST_SOURCE, "-L" + os.path.join(base, "lib"), "-lc10", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"g++ failed ({res.returncode}): {' '.join(cmd)}")
    os.replace(tmp, HOST_PATH)
    return HOST_PATH


def build_library(verbose: bool = False, force: bool = False) -> str:
    if not force and not needs_rebuild():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    cmd = [_nvcc(), *NVCC_FLAGS]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += ["-o", tmp] + [os.path.join(CSRC, s) for s in SOURCES]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}): {' '.join(cmd)}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build(verbose: bool = False, force: bool = False) -> str:
    """The library, then _kf_host-*.so; where that cannot be built, a warning (the calls that need it raise ImportError)."""
    path = build_library(verbose, force)
    try:
        build_host(force)
    except (OSError, RuntimeError) as e:
        sys.stderr.write(f"warning: {path} is built, _kf_host-*.so is not, so the Python calls that need it will raise: {e}\n")
    return path


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv, force=True))
