"""NumPy oracle for the 4-bit KV cache, the attention over it and the query/key norm with RoPE.

TEST INFRASTRUCTURE ONLY.  The reference has no counterpart; the format and the
quantiser are defined in ``include/kf_cache.h``.  The quantiser's steps are fp32
operations by definition and are restated in fp32; everything else is fp64.
"""
from __future__ import annotations

import numpy as np

from .pointwise_oracle import rope, round_to

__all__ = ["quantise", "values", "empty_cache", "write", "read", "attention", "qk_norm_rope"]

BAD = np.uint32(0x7FC00000)


def quantise(x):
    """x [..., D] -> (codes uint8 [..., D], words uint32 [...])."""
    f = np.float32
    x = np.asarray(x).astype(f)
    fin = np.isfinite(x).all(-1)
    x = np.where(fin[..., None], x, f(0))
    lo, hi = np.minimum(x.min(-1), f(0)), np.maximum(x.max(-1), f(0))
    s = hi * f(1 / 15) - lo * f(1 / 15)
    s = ((s.view(np.uint32).astype(np.uint64) + 0x80) & 0xFFFFFF00).astype(np.uint32).view(f)
    s = np.where(s < f(2.0 ** -100), f(0), s)
    inv = np.zeros_like(s)
    np.divide(f(1), s, out=inv, where=s > 0)
    z = np.clip(np.rint(-lo * inv), 0, 15)
    n = np.clip(np.rint(x * inv[..., None]) + z[..., None], 0, 15).astype(np.uint8)
    return n, np.where(fin, s.view(np.uint32) | z.astype(np.uint32), BAD)


def values(codes, words):
    """What codes stand for, in fp64."""
    s = (words & np.uint32(0xFFFFFF00)).view(np.float32).astype(np.float64)
    z = (words & np.uint32(15)).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return s[..., None] * (codes.astype(np.float64) - z[..., None])


def empty_cache(n_blocks, H, bs, D):
    return np.zeros((n_blocks, H, bs // 16, 16 * (D + 8)), np.uint8)


def _fields(cache):
    D = cache.shape[-1] // 16 - 8
    lead = cache.shape[:3]
    k = cache[..., :8 * D].reshape(*lead, 16, D // 2)
    v = cache[..., 8 * D:16 * D].reshape(*lead, 16, D // 2)
    words = np.ascontiguousarray(cache[..., 16 * D:]).view(np.uint32)
    return k, v, words[..., :16], words[..., 16:]


def write(cache, slots, k, v):
    """k, v [B, H, S, D] into slots [B, S]; returns the new cache."""
    cache = cache.copy()
    n_blocks, H, groups, nbytes = cache.shape
    D = nbytes // 16 - 8
    rows = cache.reshape(n_blocks, H, groups, nbytes)
    for which, x in ((0, k), (1, v)):
        codes, words = quantise(x)
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        for b, s in np.ndindex(*slots.shape):
            t = int(slots[b, s])
            if 0 <= t < n_blocks * groups * 16:
                blk, g, r = t // (16 * groups), t % (16 * groups) // 16, t % 16
                at = which * 8 * D + r * (D // 2)
                rows[blk, :, g, at:at + D // 2] = packed[b, :, s]
                at = 16 * D + which * 64 + 4 * r
                rows[blk, :, g, at:at + 4] = np.ascontiguousarray(words[b, :, s]).view(np.uint8).reshape(H, 4)
    return cache


def read(cache, slots):
    """(k, v) [B, H, S, D] fp64 of the slots; zeros outside the cache."""
    n_blocks, H, groups, nbytes = cache.shape
    D = nbytes // 16 - 8
    kc, vc, kw, vw = _fields(cache)
    ok = (slots >= 0) & (slots < n_blocks * groups * 16)
    t = np.where(ok, slots, 0)
    at = (t // (16 * groups), slice(None), t % (16 * groups) // 16, t % 16)
    outs = []
    for c, w in ((kc, kw), (vc, vw)):
        n = c[at]                                              # [B, S, H, D / 2]
        codes = np.stack((n & 15, n >> 4), -1).reshape(*n.shape[:-1], D)
        x = np.where(ok[..., None, None], values(codes, w[at]), 0.0)
        outs.append(np.moveaxis(x, 2, 1))
    return tuple(outs)


def attention(q, cache, table, lens, causal=False, scale=None):
    """(O, Mi, Li, A) in fp64: A[d] = sum_j p_j |v_jd| / l, the scale of O's rounding errors.

    q [B, H_q, S_q, D]; a key in a block outside the pool is zeros (so is its value)."""
    B, H_q, S_q, D = q.shape
    n_blocks, H, groups, _ = cache.shape
    bs, G = 16 * groups, H_q // H
    scale = 1 / np.sqrt(D) if scale is None else scale
    O, A = np.zeros((2, B, H_q, S_q, D))
    Mi, Li = np.full((B, H_q, S_q), -np.inf), np.zeros((B, H_q, S_q))
    for b in range(B):
        n = int(np.clip(lens[b], 0, table.shape[1] * bs))
        if n == 0:
            continue
        j = np.arange(n)
        blk = table[b, j // bs]
        slots = np.where((blk >= 0) & (blk < n_blocks), blk.astype(np.int64) * bs + j % bs, -1)
        k, v = (x[0] for x in read(cache, slots[None]))        # [H, n, D]
        for i in range(S_q):
            m = n - S_q + i + 1 if causal else n
            if m <= 0:
                continue
            qi = q[b, :, i].astype(np.float64).reshape(H, G, D)
            s = np.einsum("hgd,hjd->hgj", qi, k[:, :m]) * scale
            mx = s.max(-1)
            with np.errstate(invalid="ignore"):
                p = np.exp(s - mx[..., None])
            l = p.sum(-1)
            O[b, :, i] = (np.einsum("hgj,hjd->hgd", p, v[:, :m]) / l[..., None]).reshape(H_q, D)
            A[b, :, i] = (np.einsum("hgj,hjd->hgd", p, np.abs(v[:, :m])) / l[..., None]).reshape(H_q, D)
            Mi[b, :, i], Li[b, :, i] = mx.reshape(H_q), l.reshape(H_q)
    return O, Mi, Li, A


def qk_norm_rope(x, w, positions, eps, dtype, theta=10000.0, rot_dim=None, interleaved=False, inv_freq=None,
                 rot_scale=1.0):
    """x [B, H, S, D]: norm over D, rotation, one rounding; also the un-rounded normalised rows."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    rot = D if rot_dim is None else rot_dim
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    y = y if w is None else y * np.asarray(w, np.float64)
    out = y
    if rot:
        out = rope(y, positions, None, theta=theta, rot_dim=rot, interleaved=interleaved, inv_freq=inv_freq)
        out = np.concatenate((out[..., :rot] * rot_scale, out[..., rot:]), -1)
    return round_to(out, dtype), y
