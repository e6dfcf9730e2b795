// The 4-bit paged KV cache for B200 (sm_100a): quantise tokens into it, read them back.
//
// Format, quantiser and their guarantees: include/kf_cache.h.  The quantiser's steps are
// single IEEE fp32 operations (written with the __f*_rn intrinsics so that none is
// contracted), which makes the stored bytes reproducible from the inputs alone.
#pragma once

#include <stdint.h>

#include "kf_ptx.cuh"
#include "pointwise_sm100.cuh"

namespace kf {

constexpr int kQ4GroupTokens = 16;
template <int D>
struct Q4 {
    static constexpr int ROW = D / 2;                       // bytes of one row of codes
    static constexpr int V_CODES = 16 * ROW;                // offsets inside a group
    static constexpr int K_WORDS = 2 * V_CODES;
    static constexpr int V_WORDS = K_WORDS + 64;
    static constexpr int GROUP = 16 * (D + 8);
};

constexpr uint32_t kQ4BadRow = 0x7FC00000u;                 // word of a row with a NaN or an infinity

__device__ __forceinline__ float q4_scale(uint32_t w) { return __uint_as_float(w & 0xFFFFFF00u); }

// Parameter word of a row from its extremes (lo <= 0 <= hi, NaN if the row has one) and what
// the codes need: the reciprocal scale and the zero point (both 0 for a spoiled row).
__device__ __forceinline__ uint32_t q4_params(float lo, float hi, float* inv, float* zp) {
    const float c = 1.0f / 15.0f;
    float s = __fsub_rn(__fmul_rn(hi, c), __fmul_rn(lo, c));
    if (!(fabsf(s) <= 3.402823466e38f)) {                   // finite exactly when the row is
        *inv = *zp = 0.0f;
        return kQ4BadRow;
    }
    s = __uint_as_float((__float_as_uint(s) + 0x80u) & 0xFFFFFF00u);
    if (s < 7.888609052210118e-31f) s = 0.0f;               // 2^-100: keeps 1/s finite
    *inv = s == 0.0f ? 0.0f : __frcp_rn(s);
    *zp = fminf(fmaxf(rintf(__fmul_rn(-lo, *inv)), 0.0f), 15.0f);
    return __float_as_uint(s) | static_cast<uint32_t>(*zp);
}

// Eight codes, clamp(rint(x * inv) + zp, 0, 15), in a word.  Adding 1.5 * 2^23 rounds to an integer
// (ties to even); the clamp is taken around it, and the nibbles are put together by exact FMAs.
__device__ __forceinline__ uint32_t q4_codes8(const float (&x)[8], float inv, float zp) {
    const float m = 12582912.0f, lo = m - zp, hi = lo + 15.0f;
    float n[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        // (not packed: a packed product and sum of explicit rounding were still fused into one FMA)
        const float q0 = __fadd_rn(__fmul_rn(x[e], inv), m), q1 = __fadd_rn(__fmul_rn(x[e + 1], inv), m);
        const float2 y = fadd2(make_float2(fminf(fmaxf(q0, lo), hi), fminf(fmaxf(q1, lo), hi)), make_float2(-lo, -lo));
        n[e] = y.x;
        n[e + 1] = y.y;
    }
    float h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        h[i] = fmaf(fmaf(n[4 * i + 3], 16.0f, n[4 * i + 2]), 256.0f, fmaf(n[4 * i + 1], 16.0f, n[4 * i]));
    return __float2uint_rz(h[0]) | __float2uint_rz(h[1]) << 16;
}

__device__ __forceinline__ float fmax_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

struct Q4IoParams {
    uint8_t* cache;
    const int* slots;             // [B, S]
    uint4* k;
    uint4* v;
    long long k_sb, k_sh, k_ss;   // strides in 16-byte vectors
    long long v_sb, v_sh, v_ss;
    long long n_tokens;           // B * S
    int S, H;
    int bs_log2;                  // log2(block_size)
    int TPB;                      // tokens per block
    int splits, rows_per_split;   // blocks per token group, and their rows (K and V of each head) of it
    long long n_slots;            // n_blocks * block_size
};

constexpr int kQ4IoTokens = 16;                            // the largest TPB

// Both kernels below are bound by HBM.  A block takes a few tokens (their slots and offsets are
// looked up once, in shared memory) and all their rows, K and V of each head; a thread has UNR
// rows in flight.  Rows of one token are neighbours in the 16-bit tensors ([B, S, H, D]) or
// (token by token) in their head ([B, H, S, D]): either way every access is whole sectors.
struct Q4Tokens {
    long long k[kQ4IoTokens], v[kQ4IoTokens];              // offsets in the 16-bit tensors, vectors
    long long group[kQ4IoTokens];                          // byte offset of head 0's group; -1: no such slot
    int row[kQ4IoTokens];                                  // row in it
};

template <int D>
__device__ __forceinline__ int q4_tokens(const Q4IoParams& p, Q4Tokens& tok, long long tok0) {
    const int n = p.n_tokens - tok0 < p.TPB ? static_cast<int>(p.n_tokens - tok0) : p.TPB;
    const int tid = threadIdx.x;
    if (tid < n) {
        const long long t = tok0 + tid, b = t / p.S, s = t - b * p.S;
        const long long slot = p.slots[t];
        const long long groups = 1ll << (p.bs_log2 - 4);
        tok.k[tid] = b * p.k_sb + s * p.k_ss;
        tok.v[tid] = b * p.v_sb + s * p.v_ss;
        tok.group[tid] = slot < 0 || slot >= p.n_slots
                             ? -1 : ((slot >> p.bs_log2) * p.H * groups + ((slot >> 4) & (groups - 1))) * Q4<D>::GROUP;
        tok.row[tid] = slot & 15;
    }
    __syncthreads();
    return n;
}

// A row belongs to D / 16 threads with the vectors u and u + D / 16: a store of their words is a
// whole sector.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 3) q4_write_kernel(const Q4IoParams p) {
    constexpr int GS = D / 16, RG = 256 / GS, UNR = 4;
    __shared__ Q4Tokens tok;
    const int tid = threadIdx.x, u = tid % GS, H2 = 2 * p.H, split = blockIdx.x % p.splits;
    const int n = q4_tokens<D>(p, tok, static_cast<long long>(blockIdx.x / p.splits) * p.TPB);
    const int end = min((split + 1) * p.rows_per_split, n * H2);
    const size_t head = static_cast<size_t>(Q4<D>::GROUP) << (p.bs_log2 - 4);   // bytes from a head to the next
    int row = split * p.rows_per_split + tid / GS;
    int t = row / H2, r = row - t * H2;                                  // token, row of it: K of each head, then V
    for (; row - tid / GS < end; row += UNR * RG) {
        uint4 x4[UNR][2];
        uint8_t* dst[UNR];
        int at[UNR];
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            dst[i] = nullptr;
            x4[i][0] = x4[i][1] = make_uint4(0u, 0u, 0u, 0u);
            if (row + i * RG < end && tok.group[t] >= 0) {
                const bool is_v = r >= p.H;
                const int h = is_v ? r - p.H : r;
                const uint4* src = is_v ? p.v + tok.v[t] + h * p.v_sh : p.k + tok.k[t] + h * p.k_sh;
                x4[i][0] = ld_stream(src + u);
                x4[i][1] = ld_stream(src + u + GS);
                dst[i] = p.cache + tok.group[t] + h * head + (is_v ? Q4<D>::V_CODES : 0);
                at[i] = tok.row[t];
                if (is_v) at[i] |= 16;
            }
            for (r += RG; r >= H2; r -= H2) ++t;
        }
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            float x[2][8], lo = 0.f, hi = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                unpack8<BF16>(x4[i][c], x[c]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    lo = fminf(lo, x[c][e]);
                    hi = fmax_nan(hi, x[c][e]);
                }
            }
#pragma unroll
            for (int o = GS / 2; o > 0; o >>= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmax_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            if (!dst[i]) continue;
            float inv, zp;
            const uint32_t word = q4_params(lo, hi, &inv, &zp);
            const int rr = at[i] & 15;
            uint32_t* w = reinterpret_cast<uint32_t*>(dst[i] + rr * Q4<D>::ROW);
            if (word == kQ4BadRow) {
                w[u] = w[u + GS] = 0u;
            } else {
                w[u] = q4_codes8(x[0], inv, zp);
                w[u + GS] = q4_codes8(x[1], inv, zp);
            }
            if (u == 0)
                reinterpret_cast<uint32_t*>(dst[i] + (at[i] & 16 ? Q4<D>::V_WORDS - Q4<D>::V_CODES : Q4<D>::K_WORDS))[rr] = word;
        }
    }
}

// Eight values s * (n - z) of a word.  A nibble in place, at bit 4e, under the exponent of 2^23 is
// 2^23 + n 16^e; taking away 2^23 + z 16^e is exact, and s 16^-e puts the product back (exact
// powers of two, so each value is rounded once, as s * (n - z) is).  Nibbles 5..7 come from the
// word shifted by 20.  zc, sc: {2^23 + z 16^e}, {s 16^-e} for e = 0..4.
__device__ __forceinline__ void q4_values8(uint32_t w, const float (&zc)[5], const float (&sc)[5], float (&x)[8]) {
    const uint32_t v = w >> 20;
    float n[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int at = e < 5 ? e : e - 5;
        n[e] = __uint_as_float(((e < 5 ? w : v) & (15u << (4 * at))) | 0x4B000000u);
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const int a = e < 5 ? e : e - 5, b = e + 1 < 5 ? e + 1 : e + 1 - 5;
        const float2 y = fmul2(fadd2(make_float2(n[e], n[e + 1]), make_float2(-zc[a], -zc[b])), make_float2(sc[a], sc[b]));
        x[e] = y.x;
        x[e + 1] = y.y;
    }
}

// A row belongs to D / 16 threads with the words (8 codes, one 16-byte vector) u and u + D / 16.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 4) q4_read_kernel(const Q4IoParams p) {
    constexpr int GS = D / 16, RG = 256 / GS, UNR = 4;
    __shared__ Q4Tokens tok;
    const int tid = threadIdx.x, u = tid % GS, H2 = 2 * p.H, split = blockIdx.x % p.splits;
    const int n = q4_tokens<D>(p, tok, static_cast<long long>(blockIdx.x / p.splits) * p.TPB);
    const int end = min((split + 1) * p.rows_per_split, n * H2);
    const size_t head = static_cast<size_t>(Q4<D>::GROUP) << (p.bs_log2 - 4);
    int row = split * p.rows_per_split + tid / GS;
    int t = row / H2, r = row - t * H2;
    for (; row < end; row += UNR * RG) {
        uint32_t w[UNR][2], word[UNR];
        uint4* dst[UNR];
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            dst[i] = nullptr;
            w[i][0] = w[i][1] = word[i] = 0u;
            if (row + i * RG < end) {
                const bool is_v = r >= p.H;
                const int h = is_v ? r - p.H : r;
                dst[i] = (is_v ? p.v + tok.v[t] + h * p.v_sh : p.k + tok.k[t] + h * p.k_sh) + u;
                if (tok.group[t] >= 0) {
                    const uint8_t* g = p.cache + tok.group[t] + h * head;
                    const int rr = tok.row[t];
                    const uint32_t* c = reinterpret_cast<const uint32_t*>(g + (is_v ? Q4<D>::V_CODES : 0) + rr * Q4<D>::ROW) + u;
                    w[i][0] = __ldg(c);
                    w[i][1] = __ldg(c + GS);
                    word[i] = __ldg(reinterpret_cast<const uint32_t*>(g + (is_v ? Q4<D>::V_WORDS : Q4<D>::K_WORDS)) + rr);
                }
            }
            for (r += RG; r >= H2; r -= H2) ++t;
        }
#pragma unroll
        for (int i = 0; i < UNR; ++i) {
            if (!dst[i]) continue;
            const float s = q4_scale(word[i]), z = __uint_as_float(0x4B000000u | (word[i] & 15u)) - 8388608.0f;
            float zc[5], sc[5];
#pragma unroll
            for (int e = 0; e < 5; ++e) {
                zc[e] = fmaf(z, static_cast<float>(1 << (4 * e)), 8388608.0f);
                sc[e] = s * (1.0f / static_cast<float>(1 << (4 * e)));
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[8];
                q4_values8(w[i][c], zc, sc, x);
                st_stream(dst[i] + c * GS, pack8<BF16>(x));
            }
        }
    }
}

}  // namespace kf
