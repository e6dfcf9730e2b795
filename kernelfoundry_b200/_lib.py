"""ctypes binding of libkf_attn.so (the C ABI declared in include/kf_attn.h,
include/kf_cache.h, include/kf_pointwise.h and include/kf_synth.h).

There is no fallback: if the library is missing this module raises, and every
compute entry point goes through the CUDA kernels in the library.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import struct

import torch

from .build import HOST_PATH, LIB_DIR, LIB_PATH

KF_OK = 0
KF_ERR_INVALID_ARG = 1
KF_ERR_UNSUPPORTED_HEAD_DIM = 2
KF_ERR_MISALIGNED = 3
KF_ERR_CUDA = 4
KF_ERR_DEVICE_TIMEOUT = 5
KF_ERR_UNSUPPORTED_DEVICE = 6
KF_ERR_WORKSPACE = 7

KF_FLAG_CAUSAL = 1
KF_FLAG_OUT_F16 = 2
KF_FLAG_OUT_BF16 = 4

KF_PW_BF16 = 1
KF_ROPE_GPTJ = 2

KF_CACHE_BF16 = 1
KF_FLAG_Q_BF16 = 8

# Every symbol include/kf_attn.h, include/kf_pointwise.h and include/kf_synth.h declare.
EXPORTED = [
    "kf_strerror", "kf_last_cuda_error", "kf_version",
    "kf_attn_fwd", "kf_attn_fwd_lse", "kf_attn_fwd_ex", "kf_attn_fwd_paged", "kf_attn_paged_workspace_bytes", "kf_attn_fwd_partial", "kf_attn_combine", "kf_attn_combine_packed",
    "kf_attn_workspace_bytes", "kf_attn_workspace_init", "kf_attn_plan",
    "kf_launch_flash_attn", "kf_attn_fwd_noalloc", "kf_device_error", "kf_set_wait_timeout_ns",
    "kf_selftest_wait_timeout",
    "kf_rmsnorm", "kf_rope", "kf_qk_norm_rope", "kf_swiglu",
    "kf_peer_window_bytes", "kf_peer_window_alloc", "kf_peer_window_open", "kf_peer_window_close",
    "kf_peer_window_free", "kf_attn_exchange_combine", "kf_attn_fwd_exchange", "kf_attn_exchange_workspace_bytes",
    "kf_fill_normal_f16",
]

# Every symbol include/kf_cache.h declares.
EXPORTED_CACHE = ["kf_kv_write_q4", "kf_kv_read_q4", "kf_attn_fwd_paged_q4", "kf_attn_paged_q4_workspace_bytes"]

KF_PEER_HANDLE_BYTES = 64
KF_MAX_PEERS = 8


class KFError(RuntimeError):
    def __init__(self, code: int, what: str = ""):
        self.code = code
        msg = lib().kf_strerror(code).decode()
        if code == KF_ERR_CUDA:
            msg += f" (cudaError {lib().kf_last_cuda_error()})"
        super().__init__(f"{what}: {msg}" if what else msg)


_lib = None
_host = None


def host():
    """Load _kf_host-*.so once (csrc/kf_host.cpp; beside the library, or the package's own); raise if it has not been built."""
    global _host
    if _host is None:
        path = next((p for p in (HOST_PATH, os.path.join(LIB_DIR, os.path.basename(HOST_PATH))) if os.path.exists(p)), None)
        if path is None:
            raise ImportError(f"{HOST_PATH} is missing: run `python -m kernelfoundry_b200.build`")
        loader = importlib.machinery.ExtensionFileLoader("_kf_host", path)
        _host = importlib.util.module_from_spec(importlib.util.spec_from_loader("_kf_host", loader))
        loader.exec_module(_host)
    return _host



def lib():
    """Load libkf_attn.so once; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: run `python -m kernelfoundry_b200.build` "
                          "(the package has no CPU fallback)")
    L = ctypes.CDLL(LIB_PATH)
    P, I, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    FP = ctypes.POINTER(ctypes.c_float)
    L.kf_strerror.argtypes = [I]
    L.kf_strerror.restype = ctypes.c_char_p
    L.kf_last_cuda_error.argtypes = []
    L.kf_last_cuda_error.restype = I
    L.kf_version.argtypes = []
    L.kf_version.restype = ctypes.c_char_p
    L.kf_attn_fwd.argtypes = [P, P, P, P, I, I, I, I, I, I, P, Z, P]
    L.kf_attn_fwd.restype = I
    L.kf_attn_fwd_lse.argtypes = [P, P, P, P, P, P, I, I, I, I, I, I, P, Z, P]
    L.kf_attn_fwd_lse.restype = I
    L.kf_attn_fwd_ex.argtypes = [P, P, P, P, P, P, I, I, I, I, I, I, ctypes.c_uint, P, Z, P]
    L.kf_attn_fwd_ex.restype = I
    L.kf_attn_fwd_paged.argtypes = [P, P, P, P, P, P, P, P, I, I, I, I, I, I, I, I, P, Z, P]
    L.kf_attn_fwd_paged.restype = I
    L.kf_attn_paged_workspace_bytes.argtypes = [I, I, I, I, I, I, I]
    L.kf_attn_paged_workspace_bytes.restype = Z
    L.kf_attn_fwd_partial.argtypes = [P, P, P, P, P, P, I, I, I, I, I, I, P, Z, P]
    L.kf_attn_fwd_partial.restype = I
    L.kf_attn_combine.argtypes = [P, P, P, I, P, P, P, I, I, I, I, P]
    L.kf_attn_combine.restype = I
    L.kf_attn_combine_packed.argtypes = [P, ctypes.c_longlong, I, P, P, P, I, I, I, I, P]
    L.kf_attn_combine_packed.restype = I
    L.kf_attn_workspace_bytes.argtypes = [I, I, I, I, I, I]
    L.kf_attn_workspace_bytes.restype = Z
    L.kf_attn_workspace_init.argtypes = [P, Z, P]
    L.kf_attn_workspace_init.restype = I
    L.kf_attn_plan.argtypes = [I, I, I, I, I, I, Z, ctypes.POINTER(I), ctypes.POINTER(I), ctypes.POINTER(I)]
    L.kf_attn_plan.restype = I
    L.kf_launch_flash_attn.argtypes = [P, P, P, P, I, I, I, I, I, P]
    L.kf_launch_flash_attn.restype = I
    L.kf_attn_fwd_noalloc.argtypes = [P, P, P, P, I, I, I, I, I, I, P]
    L.kf_attn_fwd_noalloc.restype = I
    L.kf_device_error.argtypes = [I, ctypes.POINTER(ctypes.c_uint)]
    L.kf_device_error.restype = I
    L.kf_set_wait_timeout_ns.argtypes = [ctypes.c_ulonglong]
    L.kf_set_wait_timeout_ns.restype = None
    L.kf_selftest_wait_timeout.argtypes = [ctypes.c_ulonglong, P]
    L.kf_selftest_wait_timeout.restype = I
    LL, U, F = ctypes.c_longlong, ctypes.c_uint, ctypes.c_float
    L.kf_peer_window_bytes.argtypes = [I, LL, I]
    L.kf_peer_window_bytes.restype = Z
    L.kf_peer_window_alloc.argtypes = [Z, ctypes.POINTER(P), P]
    L.kf_peer_window_alloc.restype = I
    L.kf_peer_window_open.argtypes = [P, ctypes.POINTER(P)]
    L.kf_peer_window_open.restype = I
    L.kf_peer_window_close.argtypes = [P]
    L.kf_peer_window_close.restype = I
    L.kf_peer_window_free.argtypes = [P]
    L.kf_peer_window_free.restype = I
    L.kf_attn_exchange_combine.argtypes = [ctypes.POINTER(P), I, I, LL, I, P, P, P, I, I, I, I, P]
    L.kf_attn_exchange_combine.restype = I
    L.kf_attn_fwd_exchange.argtypes = [P, P, P, ctypes.POINTER(P), I, I, LL, P, P, P, I, I, I, I, I, I, P, Z, P]
    L.kf_attn_fwd_exchange.restype = I
    L.kf_attn_exchange_workspace_bytes.argtypes = [I, I, I, I, I, I]
    L.kf_attn_exchange_workspace_bytes.restype = Z
    L.kf_rmsnorm.argtypes = [P, P, P, P, LL, I, F, U, P]
    L.kf_rmsnorm.restype = I
    L.kf_rope.argtypes = [P, P, P, P, I, I, I, I, I, I, F, LL, LL, LL, LL, LL, LL, U, P]
    L.kf_rope.restype = I
    L.kf_qk_norm_rope.argtypes = [P] * 8 + [I] * 6 + [F] * 3 + [P, U, P]
    L.kf_qk_norm_rope.restype = I
    L.kf_kv_write_q4.argtypes = [P] * 4 + [I] * 6 + [P, U, P]
    L.kf_kv_write_q4.restype = I
    L.kf_kv_read_q4.argtypes = [P] * 4 + [I] * 6 + [P, U, P]
    L.kf_kv_read_q4.restype = I
    L.kf_attn_fwd_paged_q4.argtypes = [P] * 7 + [I] * 8 + [F, U, P, Z, P]
    L.kf_attn_fwd_paged_q4.restype = I
    L.kf_attn_paged_q4_workspace_bytes.argtypes = [I] * 7
    L.kf_attn_paged_q4_workspace_bytes.restype = Z
    L.kf_swiglu.argtypes = [P, P, LL, I, U, P]
    L.kf_swiglu.restype = I
    L.kf_fill_normal_f16.argtypes = [P, LL, ctypes.c_ulonglong, LL, P]
    L.kf_fill_normal_f16.restype = I
    del FP
    _lib = L
    return _lib


def check(rc: int, what: str = "") -> None:
    if rc != KF_OK:
        raise KFError(rc, what)


class CallPlans:
    """What a wrapper worked out for tensors of one set of shapes, strides, types and devices (its key,
    _kf_host.form), so that a decode loop pays for the checks of a call's form once.  Pointers and
    values are never part of a plan.  (The host's part of a call: attention over the 4-bit cache with its
    result's allocation 10.6 us with the key and 24 ctypes arguments made in Python, 6.0 with _kf_host.)"""

    def __init__(self, limit: int = 512):
        self._plans, self._limit = {}, limit

    def get(self, key):
        return self._plans.get(key)

    def put(self, key, plan):
        if len(self._plans) >= self._limit:
            self._plans.clear()
        self._plans[key] = plan
        return plan


def host_plan(fn, strides, dims, flags) -> bytes:
    """A plan of _kf_host's calls: the C function, its strides, sizes and flags (kf_host.cpp's structs)."""
    return struct.pack(f"<Q{len(strides)}q{len(dims)}iIi", ctypes.cast(fn, ctypes.c_void_p).value, *strides, *dims, flags, 0)


def on_device(index: int, fn, what: str, *args) -> None:
    """``fn(*args, current stream of device index)`` with that device current; raises KFError on a status.

    The two torch calls are the ones behind torch.cuda.current_stream / current_device, without
    the Stream object and the lazy-initialisation check (a tensor on the device exists): the
    small operators' host cost is mostly this."""
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != KF_OK:
        raise KFError(rc, what)
