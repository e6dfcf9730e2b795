"""Host API of the paged KV cache held in 4 bits (include/kf_cache.h).

* :func:`q4_cache` -- a zeroed cache: one uint8 tensor
  ``[n_blocks, H_kv, block_size / 16, 16 * (D + 8)]`` (the format is in kf_cache.h;
  the shape carries block size and head dimension, so no other handle is needed).
* :func:`kv_write_q4` / :func:`kv_read_q4` -- tokens into slots and back.
* :func:`flash_attn_paged_q4` -- decode attention over the pages, which stay in 4 bits.

No counterpart in the reference (sviraaj/kernelfoundry has no KV cache of its own).
Calls are asynchronous on the current stream and run in libkf_attn.so; there is no
CPU path.
"""
from __future__ import annotations

import torch

from ._lib import (KF_CACHE_BF16, KF_FLAG_CAUSAL, KF_FLAG_OUT_BF16, KF_FLAG_OUT_F16, KF_FLAG_Q_BF16,
                   CallPlans, host, host_plan, lib, on_device)

__all__ = ["q4_cache", "kv_write_q4", "kv_read_q4", "flash_attn_paged_q4"]

_ws: dict[tuple[int, int], torch.Tensor] = {}    # (device, stream) -> zero-filled workspace, grown on demand
_ws_outgrown: list[torch.Tensor] = []            # kept (a few MB at most): a captured graph may hold their addresses

_IO_FLAGS = {torch.float16: 0, torch.bfloat16: KF_CACHE_BF16}
_OUT_FLAGS = {torch.float32: 0, torch.float16: KF_FLAG_OUT_F16, torch.bfloat16: KF_FLAG_OUT_BF16}


def q4_cache(n_blocks: int, n_kv_heads: int, block_size: int, head_dim: int, device=None) -> torch.Tensor:
    """A zeroed 4-bit cache for ``n_blocks`` pages of ``block_size`` tokens (every slot reads zeros)."""
    if head_dim not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    if block_size not in (16, 32, 64, 128, 256):
        raise ValueError("block_size must be a power of two in [16, 256]")
    return torch.zeros(n_blocks, n_kv_heads, block_size // 16, 16 * (head_dim + 8), dtype=torch.uint8,
                       device=device or torch.device("cuda"))


def _cache_dims(cache):
    """(n_blocks, H_kv, block_size, D) of a cache tensor."""
    if not cache.is_cuda or cache.dtype != torch.uint8 or cache.dim() != 4 or not cache.is_contiguous():
        raise ValueError("cache must be a contiguous 4-D uint8 CUDA tensor made by q4_cache (no CPU path)")
    n_blocks, H_kv, groups, nbytes = cache.shape
    D = nbytes // 16 - 8
    if nbytes % 16 or D not in (64, 128, 256):
        raise ValueError("cache's last dimension must be 16 * (D + 8) bytes with D = 64, 128 or 256")
    return n_blocks, H_kv, 16 * groups, D


def _tokens(t, name, layout, device):
    """(B, H, S, D) and (batch, head, token) strides of a 16-bit tensor in `layout`."""
    if t.dtype not in _IO_FLAGS or t.dim() != 4 or t.device != device or t.stride(3) != 1:
        raise ValueError(f"{name} must be a 4-D float16 or bfloat16 tensor on {device} with a contiguous head dimension")
    if layout == "bhsd":
        (B, H, S, D), (sb, sh, ss, _) = t.shape, t.stride()
    elif layout == "bshd":
        (B, S, H, D), (sb, ss, sh, _) = t.shape, t.stride()
    else:
        raise ValueError("layout must be 'bhsd' or 'bshd'")
    return (B, H, S, D), (sb, sh, ss)


def _check_slots(slots, B, S, device):
    if slots.dtype != torch.int32 or tuple(slots.shape) != (B, S) or not slots.is_contiguous() or slots.device != device:
        raise ValueError(f"slots must be a contiguous int32 [{B}, {S}] tensor on {device}")


def _workspace(device, nbytes):
    """The current stream's workspace: calls on different streams may overlap, those on one cannot."""
    key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
    ws = _ws.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        if not torch.cuda.is_current_stream_capturing():   # memory of a graph's pool stays with the graph
            if key in _ws:
                _ws_outgrown.append(_ws[key])
            _ws[key] = ws
    return ws


def _check_workspace(workspace, device):
    if workspace.device != device or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on {device}")


def kv_write_q4(k, v, cache, slots, *, layout: str = "bhsd") -> None:
    """Quantise ``k`` and ``v`` to 4 bits into ``cache``: token (b, s) goes to slot ``slots[b, s]``.

    k, v: fp16 or bf16, ``[B, H_kv, S, D]`` ("bhsd") or ``[B, S, H_kv, D]`` ("bshd"), any
    strides (multiples of 8) with a contiguous head dimension.  slots: int32 ``[B, S]``; slot
    t is row ``t % block_size`` of block ``t // block_size``; one outside the cache (-1) is
    skipped, one named twice holds anything.  Each head row is quantised by itself (scale and zero point per row)."""
    h = host()
    key = (layout, h.form(k, v, cache, slots))
    index, plan = _write_plans.get(key) or _write_plans.put(key, _plan_io(lib().kf_kv_write_q4, cache, slots, k, v, layout))
    on_device(index, h.kv_io, "kf_kv_write_q4", plan, k, v, cache, slots)


_write_plans, _read_plans, _attn_plans = CallPlans(), CallPlans(), CallPlans()


def _plan_io(fn, cache, slots, k, v, layout):
    """Checks of a write or read (`fn`) and the arguments that follow from its tensors' form."""
    n_blocks, H_kv, bs, D = _cache_dims(cache)
    dev = cache.device
    (B, H, S, Dk), ks = _tokens(k, "k", layout, dev)
    dims_v, vs = _tokens(v, "v", layout, dev)
    if dims_v != (B, H, S, Dk) or v.dtype != k.dtype:
        raise ValueError("k and v must have one shape and type")
    if (H, Dk) != (H_kv, D):
        raise ValueError(f"k and v must have the cache's {H_kv} heads of {D}")
    _check_slots(slots, B, S, dev)
    return dev.index, host_plan(fn, (*ks, *vs), (B, S, H, D, n_blocks, bs), _IO_FLAGS[k.dtype])


def kv_read_q4(cache, slots, *, dtype=torch.float16, layout: str = "bhsd", out=None):
    """``(k, v)`` of the tokens in ``slots`` (int32 ``[B, S]``) as fp16 or bf16 tensors.

    ``[B, H_kv, S, D]`` ("bhsd", in fp16 what :func:`flash_attn_fwd` takes) or ``[B, S, H_kv, D]``
    ("bshd").  A slot outside the cache reads zeros.  ``out``: (k, v) to write into."""
    h = host()
    if out is None:
        key = (layout, dtype, h.form(cache, slots))
        shape, device, index, plan = _read_plans.get(key) or _read_plans.put(key, _plan_read(cache, slots, dtype, layout))
        k = torch.empty(shape, dtype=dtype, device=device)
        v = torch.empty_like(k)
    else:
        k, v = out
        key = (layout, h.form(cache, slots, k, v))
        index, plan = _read_plans.get(key) or _read_plans.put(key, _plan_io(lib().kf_kv_read_q4, cache, slots, k, v, layout))
    on_device(index, h.kv_io, "kf_kv_read_q4", plan, cache, slots, k, v)
    return k, v


def _plan_read(cache, slots, dtype, layout):
    """Shape of a read's results and the plan of reading into such tensors."""
    n_blocks, H_kv, bs, D = _cache_dims(cache)
    if slots.dim() != 2 or layout not in ("bhsd", "bshd") or dtype not in _IO_FLAGS:
        raise ValueError("slots must be [B, S], layout 'bhsd' or 'bshd', dtype float16 or bfloat16")
    B, S = slots.shape
    _check_slots(slots, B, S, cache.device)
    if layout == "bhsd":
        shape, strides = (B, H_kv, S, D), (H_kv * S * D, S * D, D)
    else:
        shape, strides = (B, S, H_kv, D), (H_kv * S * D, D, H_kv * D)
    return shape, cache.device, cache.device.index, host_plan(lib().kf_kv_read_q4, strides + strides,
                                                              (B, S, H_kv, D, n_blocks, bs), _IO_FLAGS[dtype])


def flash_attn_paged_q4(q, cache, block_table, seq_lens, *, causal=False, scale=None, out=None, out_dtype=None,
                        return_lse=False, workspace=None):
    """Attention of ``q`` ``[B, H_q, S_q, D]`` (fp16 or bf16) over the 4-bit pages of ``cache``.

    block_table int32 ``[B, max_blocks]``: pool block of each logical block; seq_lens int32
    ``[B]``: keys per sequence (0 gives O = 0).  ``causal``: query i sees keys
    ``j <= seq_len - S_q + i`` (drafted tokens whose keys are already in the cache); a row
    that sees no key is 0.  ``scale`` defaults to 1/sqrt(D); 0 weighs all keys alike.  Decode shapes:
    ``H_q / H_kv * S_q <= 64``.  O has ``out_dtype`` (or ``out``'s; default q's dtype);
    with ``return_lse`` also (Mi, Li), the row max of the scaled scores and sum of exp(s - Mi).
    Each stream has its workspace; ``workspace`` (zero-filled uint8,
    ``kf_attn_paged_q4_workspace_bytes``) replaces it: a captured graph that may run beside other
    calls, or other graphs captured on its stream, needs one of its own."""
    if out is None:
        out = torch.empty_like(q, dtype=out_dtype) if out_dtype is not None else torch.empty_like(q)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    h = host()
    key = (bool(causal), h.form(q, cache, block_table, seq_lens, out))
    device, index, need, plan = (_attn_plans.get(key) or
                                 _attn_plans.put(key, _plan_attn(q, cache, block_table, seq_lens, out, causal)))
    if workspace is None:
        workspace = _workspace(device, need)
    else:
        _check_workspace(workspace, device)
    Mi = Li = None
    if return_lse:
        Mi = torch.empty(q.shape[:3], dtype=torch.float32, device=device)
        Li = torch.empty_like(Mi)
    on_device(index, h.attn_q4, "kf_attn_fwd_paged_q4", plan, q, cache, block_table, seq_lens, out, Mi, Li,
              scale, workspace)
    return (out, Mi, Li) if return_lse else out


def _plan_attn(q, cache, block_table, seq_lens, out, causal):
    """Checks of :func:`flash_attn_paged_q4` and the arguments that follow from its tensors' form."""
    n_blocks, H_kv, bs, D = _cache_dims(cache)
    dev = cache.device
    if q.dtype not in _IO_FLAGS or q.dim() != 4 or not q.is_contiguous() or q.device != dev or q.shape[3] != D:
        raise ValueError(f"q must be a contiguous [B, H_q, S_q, {D}] float16 or bfloat16 tensor on {dev}")
    B, H_q, S_q, _ = q.shape
    for t, name, nd in ((block_table, "block_table", 2), (seq_lens, "seq_lens", 1)):
        if t.dtype != torch.int32 or t.dim() != nd or t.shape[0] != B or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {nd}-D int32 tensor with {B} rows on {dev}")
    if out.dtype not in _OUT_FLAGS:
        raise ValueError("output dtype must be float32, float16 or bfloat16")
    if out.shape != q.shape or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be a contiguous {tuple(q.shape)} tensor on {dev}")
    max_blocks = block_table.shape[1]
    flags = (KF_FLAG_CAUSAL if causal else 0) | _OUT_FLAGS[out.dtype] | (KF_FLAG_Q_BF16 if q.dtype == torch.bfloat16 else 0)
    with torch.cuda.device(dev):
        need = lib().kf_attn_paged_q4_workspace_bytes(B, H_q, H_kv, S_q, D, bs, max_blocks)
    return dev, dev.index, max(need, 16), host_plan(lib().kf_attn_fwd_paged_q4, (),
                                                    (B, H_q, H_kv, S_q, D, n_blocks, bs, max_blocks), flags)
