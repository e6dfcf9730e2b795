/*
 * kf_cache.h -- C ABI of the paged KV cache held in 4 bits: tokens quantised as they
 * are written, read back as 16-bit tensors, and attended without leaving their 4 bits.
 *
 * No counterpart in the reference (its paged benchmark gathers fp16 pages,
 * reference_benchmarks/bench_flash_attn2.py:153-215); conventions are those of kf_attn.h:
 * device pointers, plain C types, asynchronous on `stream` (a cudaStream_t, NULL = legacy
 * default stream), no allocation, KF_OK or a KF_ERR_* code, argument checks before any
 * CUDA call.
 *
 * The cache is [n_blocks][H_kv][block_size / 16] groups.  A group holds 16 tokens of one
 * head in KF_Q4_GROUP_BYTES(D) = 16 * (D + 8) bytes:
 *   K codes [16][D / 2]    byte j of a row: dim 2j in the low, dim 2j + 1 in the high half
 *   V codes [16][D / 2]
 *   K words [16] uint32    fp32 scale, its low 8 bits replaced by the zero point 0..15
 *   V words [16] uint32
 * A code n of a row with scale s and zero point z stands for s * (n - z), exact in fp32.
 * Slot t is row t % block_size of block t / block_size.
 *
 * A row x is quantised by single fp32 operations (bit-reproducible):
 *   lo = min(0, min x), hi = max(0, max x), s = hi * (1/15) - lo * (1/15), rounded to 16
 *   significant bits (half up); s = 0 below 2^-100 (the row reads back as zeros);
 *   z = rint(-lo * (1/s)) in [0, 15], n = clamp(rint(x * (1/s)) + z, 0, 15).
 * So |x - s (n - z)| <= s / 2 (and a few ulp), and 0 is held exactly.  A row with a NaN or
 * an infinity gets a NaN scale: all of it reads back as NaN.
 *
 * D: 64, 128 or 256.  block_size: a power of two in [16, 256].  The cache, q, k, v, O and
 * the 16-bit tensors' rows are 16-byte aligned.
 */
#ifndef KF_CACHE_H_
#define KF_CACHE_H_

#include <stddef.h>

#include "kf_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KF_Q4_GROUP_BYTES(D) (16 * ((D) + 8))

#define KF_CACHE_BF16 1u     /* kf_kv_*_q4: k and v are bf16 (default fp16) */
#define KF_FLAG_Q_BF16 8u    /* kf_attn_fwd_paged_q4: Q is bf16 (default fp16) */

/* Quantises k and v (both [B, H_kv, S, D] by element strides, head dimension contiguous)
 * into the cache: token (b, s) goes to slot slots[b * S + s].  A slot outside
 * [0, n_blocks * block_size) is skipped (padding: -1).  If one slot is named twice, what ends there
 * is undefined (it may be made of both tokens).  strides: 6 values in host memory, the batch, head and token
 * strides of k, then of v; multiples of 8, >= 0 (of a dimension of one element: any).
 * B * S == 0 is a no-op. */
int kf_kv_write_q4(const void* k, const void* v, void* cache, const int* slots, int B, int S, int H_kv, int D,
                   int n_blocks, int block_size, const long long* strides, unsigned flags, void* stream);

/* Reads slots back into k and v (layout and strides as kf_kv_write_q4, outputs distinct
 * and without overlap): rnd(s * (n - z)), one rounding.  A slot outside
 * [0, n_blocks * block_size) reads zeros. */
int kf_kv_read_q4(const void* cache, const int* slots, void* k, void* v, int B, int S, int H_kv, int D,
                  int n_blocks, int block_size, const long long* strides, unsigned flags, void* stream);

/* Attention over the cache: O[b, h, i] = softmax_j(scale * q . k_j) v_j over the keys
 * j < seq_lens[b] of sequence b, whose logical block n is pool block
 * block_table[b * max_blocks + n].  Q and O [B, H_q, S_q, D] contiguous and without overlap, query head h uses
 * cache head h / (H_q / H_kv); H_q / H_kv * S_q at most 64 (longer chunks: kf_kv_read_q4 and
 * kf_attn_fwd_ex).  seq_lens is clamped to [0, max_blocks * block_size].
 * flags: KF_FLAG_CAUSAL: query i sees keys j <= seq_lens[b] - S_q + i; KF_FLAG_Q_BF16;
 * KF_FLAG_OUT_F16 / KF_FLAG_OUT_BF16 (default fp32 O).  A query row that sees no key gets
 * O = 0 (Mi = -inf, Li = 0).  Mi / Li (optional) as kf_attn_fwd_lse.  scale == 0: 1/sqrt(D).
 * Table entries past a sequence's last block are not read; an entry outside
 * [0, n_blocks) reads zeros.  Probabilities times the values' scales enter the second
 * product as fp16 for a bf16 O (2^-11 a key, relative) and as two fp16 for fp16 and fp32 (2^-22),
 * in both cases to no finer than 2^-23 of the row's largest; everything else is exact or fp32
 * (for queries below 2^120: beyond, scores may overflow that would not have to).  max_blocks * block_size < 2^31 - 64.
 * workspace: required, kf_attn_paged_q4_workspace_bytes(), handled as kf_attn_fwd's
 * (zero-filled once, left ready by every call, not shared by overlapping calls);
 * KF_ERR_WORKSPACE if it is too small. */
int kf_attn_fwd_paged_q4(const void* Q, const void* cache, const int* block_table, const int* seq_lens,
                         void* O, float* Mi, float* Li, int B, int H_q, int H_kv, int S_q, int D,
                         int n_blocks, int block_size, int max_blocks, float scale, unsigned flags,
                         void* workspace, size_t workspace_bytes, void* stream);
size_t kf_attn_paged_q4_workspace_bytes(int B, int H_q, int H_kv, int S_q, int D, int block_size, int max_blocks);

#ifdef __cplusplus
}
#endif

#endif /* KF_CACHE_H_ */
