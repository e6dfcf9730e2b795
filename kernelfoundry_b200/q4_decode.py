"""A decoder layer's attention block served over the 4-bit KV cache.

    python -m kernelfoundry_b200.q4_decode [--batch 16 --prompt 2048 --steps 64]

Runs the block as a server would: prompts of different lengths are prefilled, in two
chunks (the second attends the first as read back from the cache), then tokens are
decoded from a captured CUDA graph.  Prints the time of a decode step and how far its
output is from attention over the un-quantised keys and values.

The block: RMSNorm, the fused query/key/value projection, :func:`qk_norm_rope`,
:func:`kv_write_q4`, attention (:func:`flash_attn_fwd` over the chunk and what
:func:`kv_read_q4` returns, or :func:`flash_attn_paged_q4`), the output projection, the
residual.  The projections are plain matrix products (cuBLAS, through torch).
"""
from __future__ import annotations

import argparse

import torch

from ._lib import lib
from .attention import flash_attn_fwd
from .kv_cache import flash_attn_paged_q4, kv_read_q4, kv_write_q4, q4_cache
from .pointwise import qk_norm_rope, rms_norm

__all__ = ["Q4AttentionBlock"]


class Q4AttentionBlock:
    """Attention block with random fp16 weights, its 4-bit cache and the block table of ``batch`` sequences."""

    def __init__(self, batch: int, max_len: int, hidden: int = 4096, H_q: int = 32, H_kv: int = 8, D: int = 128,
                 block_size: int = 16, theta: float = 10000.0, eps: float = 1e-6, device=None, seed: int = 0):
        self.device = torch.device(device or "cuda")
        self.H_q, self.H_kv, self.D, self.block_size, self.theta, self.eps = H_q, H_kv, D, block_size, theta, eps
        g = torch.Generator(device=self.device).manual_seed(seed)

        def weight(*shape, scale):
            return (torch.randn(*shape, generator=g, device=self.device) * scale).half()

        self.w_norm = torch.ones(hidden, device=self.device).half()
        self.w_qkv = weight(hidden, (H_q + 2 * H_kv) * D, scale=hidden ** -0.5)
        self.w_o = weight(H_q * D, hidden, scale=(H_q * D) ** -0.5)
        self.w_q, self.w_k = ((1 + weight(D, scale=0.1)).contiguous() for _ in range(2))
        per = -(-max_len // block_size)
        self.cache = q4_cache(batch * per, H_kv, block_size, D, self.device)
        self.table = torch.randperm(batch * per, generator=g, device=self.device).to(torch.int32).view(batch, per)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.capacity = per * block_size                   # tokens of a sequence that the table has room for
        self._most = 0                                     # what the longest sequence has, or more: the lengths are on the device
        self._captured = False                             # a graph's replays may have moved them since
        # The attention's workspace, one for eager and captured steps alike (they share the cache, so they never overlap).
        # Without it a call captured on a stream of the graph's own records a zero-fill of a new one.
        most = max(1, 64 // max(1, H_q // H_kv))           # tokens of a step, at most
        need = max(lib().kf_attn_paged_q4_workspace_bytes(batch, H_q, H_kv, s, D, block_size, per) for s in (1, most))
        self._workspace = torch.zeros(need, dtype=torch.uint8, device=self.device)

    def slots(self, positions, valid=None):
        """Cache slots of ``positions`` [B, S] (int64); -1 where not valid and past the table (padding may be there)."""
        page = positions // self.block_size
        outside = page >= self.table.shape[1]
        if valid is not None:
            outside = outside | ~valid
        blocks = self.table.gather(1, page.clamp(max=self.table.shape[1] - 1)).long()
        return (blocks * self.block_size + positions % self.block_size).masked_fill(outside, -1).to(torch.int32)

    def _check_room(self, n):
        if n > self.capacity:
            raise ValueError(f"a sequence would have {n} tokens, the block table has room for {self.capacity}")

    def _project(self, x, positions):
        """Rotated queries and keys, and values, all [B, H, S, D]."""
        B, S, _ = x.shape
        Hq, Hk, D = self.H_q, self.H_kv, self.D
        qkv = rms_norm(x.contiguous(), self.w_norm, self.eps) @ self.w_qkv
        q = qkv[..., :Hq * D].view(B, S, Hq, D)
        k = qkv[..., Hq * D:(Hq + Hk) * D].view(B, S, Hk, D)
        v = qkv[..., (Hq + Hk) * D:].view(B, S, Hk, D)
        q_out, k_out = (torch.empty(B, h, S, D, dtype=x.dtype, device=x.device) for h in (Hq, Hk))
        qk_norm_rope(q, k, self.w_q, self.w_k, positions.to(torch.int32).contiguous(), eps=self.eps, theta=self.theta,
                     layout="bshd", out=(q_out.transpose(1, 2), k_out.transpose(1, 2)))
        return q_out, k_out, v.transpose(1, 2)

    def _output(self, x, o):
        B, H, S, D = o.shape
        return x + o.transpose(1, 2).reshape(B, S, H * D) @ self.w_o

    def prefill(self, x, lens=None, past: int = 0):
        """A chunk ``x`` [B, S, hidden] at positions past ..; ``lens`` [B]: tokens of each (the rest is padding).

        Every sequence has ``past`` tokens in the cache already; they are read back and attended.  Padding may go
        past the table, a token may not (ValueError)."""
        B, S, _ = x.shape
        if past + S > self.capacity:
            self._check_room(past + (S if lens is None else int(lens.max())))
        self._most = past + S
        positions = past + torch.arange(S, device=x.device).expand(B, S)
        lens = torch.full((B,), S, dtype=torch.int32, device=x.device) if lens is None else lens
        q, k, v = self._project(x, positions)
        kv_write_q4(k, v, self.cache, self.slots(positions, positions - past < lens[:, None]))
        k_all, v_all = k, v.contiguous()
        if past:
            before = self.slots(torch.arange(past, device=x.device).expand(B, past)).contiguous()
            k_past, v_past = kv_read_q4(self.cache, before, dtype=x.dtype)
            k_all, v_all = torch.cat((k_past, k), 2), torch.cat((v_past, v_all), 2)
        o = flash_attn_fwd(q, k_all, v_all, causal=True, out_dtype=x.dtype)      # padding comes after every real token
        self.lens.copy_(lens + past)
        return self._output(x, o)

    def step(self, x):
        """``x`` [B, S, hidden]: the next S tokens of every sequence (S > 1: drafts, causal among themselves).

        ValueError if they do not fit the table.  Replays of a captured step are the caller's to count: nothing on
        the host sees them, and a token past the table is not kept."""
        B, S, _ = x.shape
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            self._captured = True
        else:
            if self._captured or self._most + S > self.capacity:
                self._most = int(self.lens.max())
                self._check_room(self._most + S)
            self._most += S
        positions = self.lens.long()[:, None] + torch.arange(S, device=x.device)
        q, k, v = self._project(x, positions)
        kv_write_q4(k, v, self.cache, self.slots(positions))
        self.lens += S
        o = flash_attn_paged_q4(q, self.cache, self.table, self.lens, causal=S > 1, workspace=self._workspace)
        return self._output(x, o)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args(argv)
    if a.batch < 1 or a.prompt < 2 or a.steps < 1:
        ap.error("--batch and --steps must be at least 1, --prompt (two chunks) at least 2")
    torch.manual_seed(0)
    hidden, half = 4096, a.prompt // 2
    block = Q4AttentionBlock(a.batch, a.prompt + a.steps + 8, hidden)
    x = torch.randn(a.batch, a.prompt, hidden, device="cuda").half()
    lens = torch.randint(1, a.prompt - half + 1, (a.batch,), device="cuda", dtype=torch.int32)
    block.prefill(x[:, :half])
    block.prefill(x[:, half:], lens, past=half)

    # one step against un-quantised keys and values of the same tokens
    token = torch.randn(a.batch, 1, hidden, device="cuda").half()
    b = int(lens.argmax())
    n = half + int(lens[b])
    q, k, v = block._project(torch.cat((x[b:b + 1, :n], token[b:b + 1]), 1), torch.arange(n + 1, device="cuda")[None])
    want = block._output(token[b:b + 1], flash_attn_fwd(q[:, :, -1:].contiguous(), k, v.contiguous(), out_dtype=torch.float16))
    got = block.step(token)[b:b + 1]
    print(f"4-bit cache against fp16 keys and values: {((got - want).norm() / (want - token[b:b + 1]).norm()).item():.3f} "
          "of the attention's contribution")

    static = token.clone()
    block.step(static)                                     # warm-up: plans of the calls, cuBLAS
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.step(static)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(a.steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"decode: {start.elapsed_time(end) * 1e3 / a.steps:.1f} us a step, batch {a.batch}, "
          f"{int(block.lens.min())}..{int(block.lens.max())} keys, cache {block.cache.numel() / 1e6:.1f} MB "
          f"(fp16: {block.cache.numel() * 4 * block.D / (block.D + 8) / 1e6:.1f} MB)")


if __name__ == "__main__":
    main()
