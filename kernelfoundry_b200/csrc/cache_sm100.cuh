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
// the codes need: the reciprocal scale (0 for a spoiled row); its low bits are the zero point.
__device__ __forceinline__ uint32_t q4_params(float lo, float hi, float* inv) {
    const float c = 1.0f / 15.0f;
    float s = __fsub_rn(__fmul_rn(hi, c), __fmul_rn(lo, c));
    if (!(fabsf(s) <= 3.402823466e38f)) {                   // finite exactly when the row is
        *inv = 0.0f;
        return kQ4BadRow;
    }
    s = __uint_as_float((__float_as_uint(s) + 0x80u) & 0xFFFFFF00u);
    if (s < 7.888609052210118e-31f) s = 0.0f;               // 2^-100: keeps 1/s finite
    *inv = s == 0.0f ? 0.0f : __frcp_rn(s);
    return __float_as_uint(s) | static_cast<uint32_t>(rintf(__fmul_rn(-lo, *inv)));
}

// Eight codes, clamp(rint(x * inv) + zp, 0, 15), in a word.  Adding 1.5 * 2^23 rounds to an integer
// r (ties to even) and leaves it as 0x4B400000 + r, so the sum of these words times 16^e, less the
// constants', is the sum of r 16^e; zp goes in eight times at once.  The lower clamp never acts:
// rint(x inv) >= rint(lo inv) = -zp, and zp needs none, as s >= (hi - lo) / 15 * (1 - 2^-16).
__device__ __forceinline__ uint32_t q4_codes8(const float (&x)[8], float inv, uint32_t zp) {
    const float top = 12582912.0f + static_cast<float>(15 - static_cast<int>(zp));
    uint32_t w = 0;
#pragma unroll
    for (int e = 7; e >= 0; --e)        // (not packed: a packed product and sum, both rounded, were still fused into an FMA)
        w = w * 16u + __float_as_uint(fminf(__fadd_rn(__fmul_rn(x[e], inv), 12582912.0f), top));
    return w + zp * 0x11111111u - 0x4B400000u * 0x11111111u;
}

// Larger of two packed pairs, NaN if either is.
template <bool BF16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// n / d for n < 2^31 by a multiplication: d <= 2^shift, mul = floor(2^32 (2^shift - d) / d) + 1.
struct FastDiv {
    unsigned mul, shift;
    __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct Q4IoParams {
    uint8_t* cache;
    const int* slots;             // [B, S]
    uint4* k;
    uint4* v;
    unsigned k_sb, k_sh, k_ss;    // strides in 16-byte vectors
    unsigned v_sb, v_sh, v_ss;
    int S, H;
    unsigned rows;                // B * S * 2 H < 2^31
    int head_major;               // order of a sequence's rows: head by head (K, then V), or token by token
    int n_in, n_out;              // S and 2 H, or 2 H and S
    FastDiv by_in, by_out;
    int passes;                   // rows a thread takes, at most UNR
    int bs_log2;                  // log2(block_size)
    long long n_slots;            // n_blocks * block_size
};

// Both kernels below are bound by HBM.  Rows are numbered as they lie in the 16-bit tensors: token
// by token ([B, S, H, D]) or head by head ([B, H, S, D], where neighbours also share the cache's
// groups).  A block takes up to four passes of neighbouring rows, all in flight; one pass where
// that still leaves SMs idle.
struct Q4Row {
    bool is_v;
    int h;
    unsigned tok;
    unsigned long long at;         // offset in the 16-bit tensor, vectors
};
__device__ __forceinline__ Q4Row q4_row(const Q4IoParams& p, unsigned row) {
    Q4Row r;
    const unsigned q = p.by_in.div(row), in = row - q * p.n_in, b = p.by_out.div(q), out = q - b * p.n_out;
    const int hh = p.head_major ? out : in, s = p.head_major ? in : out;
    r.tok = b * p.S + s;
    r.is_v = hh >= p.H;
    r.h = r.is_v ? hh - p.H : hh;
    const unsigned sb = r.is_v ? p.v_sb : p.k_sb, sh = r.is_v ? p.v_sh : p.k_sh, ss = r.is_v ? p.v_ss : p.k_ss;
    r.at = static_cast<unsigned long long>(b) * sb + static_cast<unsigned long long>(r.h) * sh +
           static_cast<unsigned long long>(s) * ss;
    return r;
}
// The group that holds `slot` of a head; nullptr outside the cache.
template <int D>
__device__ __forceinline__ uint8_t* q4_group(const Q4IoParams& p, int slot, int h) {
    if (slot < 0 || slot >= p.n_slots) return nullptr;
    const unsigned gs = p.bs_log2 - 4, block = static_cast<unsigned>(slot) >> p.bs_log2;   // (fewer than 2^32 groups)
    return p.cache + static_cast<unsigned long long>(((block * p.H + h) << gs) + ((slot >> 4) & ((1u << gs) - 1))) * Q4<D>::GROUP;
}

// A row belongs to D / 32 threads with four neighbouring vectors each: their words are one 16-byte
// store, and the row's parameters are worked out by few threads.  The extremes are found on packed
// pairs, the largest value and the largest negated one in the halves of one word.  (Two vectors a
// thread and fp32 extremes: 87 us for 65536 tokens, at 15 instructions an element.)
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 3) q4_write_kernel(const Q4IoParams p) {
    constexpr int GS = D / 32, RG = 256 / GS, UNR = 2;
    const int u = threadIdx.x % GS;
    const unsigned row0 = blockIdx.x * (p.passes * RG) + threadIdx.x / GS;
    uint4 x4[UNR][4];
    int slot[UNR], h[UNR];                                           // head; V's have bit 30 set
#pragma unroll
    for (int i = 0; i < UNR; ++i) {
        const unsigned row = row0 + i * RG;
        slot[i] = -1;
        h[i] = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) x4[i][c] = make_uint4(0u, 0u, 0u, 0u);
        if (i < p.passes && row < p.rows) {
            const Q4Row r = q4_row(p, row);
            const uint4* src = (r.is_v ? p.v : p.k) + r.at + 4 * u;
#pragma unroll
            for (int c = 0; c < 4; ++c) x4[i][c] = src[c];
            slot[i] = p.slots[r.tok];
            h[i] = r.is_v ? r.h | 1 << 30 : r.h;
        }
    }
#pragma unroll
    for (int i = 0; i < UNR; ++i) {
        if (i >= p.passes) break;
        uint32_t mx = 0u, mn = 0u;                                   // (0 is always within the row's range)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t w[4] = {x4[i][c].x, x4[i][c].y, x4[i][c].z, x4[i][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mx = max2_nan<BF16>(mx, w[e]);
                mn = min2_nan<BF16>(mn, w[e]);
            }
        }
        mn ^= 0x80008000u;
        uint32_t ext = max2_nan<BF16>(__byte_perm(mx, mn, 0x5410), __byte_perm(mx, mn, 0x7632));
#pragma unroll
        for (int o = GS / 2; o > 0; o >>= 1) ext = max2_nan<BF16>(ext, __shfl_xor_sync(0xffffffffu, ext, o));
        const bool is_v = h[i] >> 30;
        uint8_t* g = q4_group<D>(p, slot[i], h[i] & 0xFFFF);
        if (!g) continue;
        float inv;
        const uint32_t word = q4_params(-to_f32<BF16>(ext >> 16), to_f32<BF16>(ext & 0xFFFFu), &inv);
        const int rr = slot[i] & 15;
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (word != kQ4BadRow) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float x[8];
                unpack8<BF16>(x4[i][c], x);
                w[c] = q4_codes8(x, inv, word & 15u);
            }
        }
        reinterpret_cast<uint4*>(g + (is_v ? Q4<D>::V_CODES : 0) + rr * Q4<D>::ROW)[u] = make_uint4(w[0], w[1], w[2], w[3]);
        if (u == 0) reinterpret_cast<uint32_t*>(g + (is_v ? Q4<D>::V_WORDS : Q4<D>::K_WORDS))[rr] = word;
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
// 65536 tokens of 8 heads of 128: 57.1 us, 5.95 TB/s of results and codes (write: 61.7 us, 5.5 TB/s); a long
// read is bound by its writes to memory, 8192 tokens (9.7 us) by instructions and by starting and draining.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 4) q4_read_kernel(const Q4IoParams p) {
    constexpr int GS = D / 16, RG = 256 / GS, UNR = 4;
    const int u = threadIdx.x % GS;
    const unsigned row0 = blockIdx.x * (p.passes * RG) + threadIdx.x / GS;
    uint32_t w[UNR][2], word[UNR];
    uint4* dst[UNR];
    int slot[UNR], h[UNR];                                           // head; V's have bit 30 set
#pragma unroll
    for (int i = 0; i < UNR; ++i) {
        const unsigned row = row0 + i * RG;
        dst[i] = nullptr;
        slot[i] = -1;
        h[i] = 0;
        if (i < p.passes && row < p.rows) {
            const Q4Row r = q4_row(p, row);
            dst[i] = (r.is_v ? p.v : p.k) + r.at + u;
            slot[i] = p.slots[r.tok];
            h[i] = r.is_v ? r.h | 1 << 30 : r.h;
        }
    }
#pragma unroll
    for (int i = 0; i < UNR; ++i) {
        w[i][0] = w[i][1] = word[i] = 0u;
        if (const uint8_t* g = q4_group<D>(p, slot[i], h[i] & 0xFFFF)) {
            const bool is_v = h[i] >> 30;
            const int rr = slot[i] & 15;
            const uint32_t* c = reinterpret_cast<const uint32_t*>(g + (is_v ? Q4<D>::V_CODES : 0) + rr * Q4<D>::ROW) + u;
            w[i][0] = __ldg(c);
            w[i][1] = __ldg(c + GS);
            word[i] = __ldg(reinterpret_cast<const uint32_t*>(g + (is_v ? Q4<D>::V_WORDS : Q4<D>::K_WORDS)) + rr);
        }
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

}  // namespace kf
