// Attention over the 4-bit paged KV cache (include/kf_cache.h) for B200 (sm_100a).
//
//   x_j = scale * s_j (q . n_j - z_j sum(q)),  O = sum_j e^(x_j - m) t_j (n'_j - z'_j) / sum_j e^(x_j - m)
// with (s, z, n) a key's scale, zero point and codes and (t, z', n') a value's.
//
// What bounds it: a key and value of one head are D + 8 bytes, read once; at 6.5 TB/s an SM
// receives 46 codes per clock, so the codes have to become MMA operands in about two
// instructions per eight.  mma.m16n8k16 with the KEYS as its 16 rows and the queries as its 8
// columns (S^T = K Q^T, O^T = V^T P^T) wastes nothing for up to 8 query rows a cache head; a
// 128-row tcgen05 tile would be 1/16 filled by 8 rows (half by the 64 that are accepted) and wants
// its operands expanded in memory.  Beyond 8 NT rows every group of them copies and unpacks the
// cache for itself (B=32, 4096 keys of 128: 8 rows 40.1 us, 16 60.1, 32 109, 64 203).
//
// Codes to operands.  A 4-bit integer in bits 2..5 of an fp16 is the subnormal n * 2^-22, in bits
// 6..9 it is n * 2^-18, and the tensor core multiplies subnormals exactly.  For K two shifts and
// four ands therefore make four half2 operands of a word's eight codes; the factor 16 goes into the
// query operand, 2^22 into the score's factor, and the zero point enters once per score.  The
// tensor core aligns a sum by its operands' exponent fields, which for subnormals are too large by
// up to 2^8: the low bits this costs leave scores off by 2^-20 (from bits 0..3 and 4..7, with one
// shift, it was 2^-18; made normal by an FMA each, 2^-21, and 5 % slower).
// For V two keys' words are interleaved by halves (prmt), masked in place (bits 0..3 and 4..7), and
// one half2 FMA makes (n - z) * 2^-9 of each pair, exact and normal: sums of p t (n - z) keep the
// value's own size, where sum(p t n) - sum(p t z) would cancel.
// Queries are scaled by a power of two per row to a maximum in [2^13, 2^14), every other operand
// by 1/16 of it.  fp16's last bit is then 2^-37 of the row's largest element, or 2^-33 in those:
// what is lost of an element is at most half of that.
// p t enters the second product as fp16, times a power of two (norm) of its query row: the one that
// keeps the largest t seen below 2^7, or a larger one if the row's largest p t would then be below
// 2^-2 (a value far beyond the others with next to no probability, or hidden from the row, must not
// push the others out of fp16).  For a bf16 output this rounding is the only one below fp32 in the
// sum, 2^-11 relative per key (or 2^-23 of the row's largest p t); for fp16 and fp32 outputs (SPLIT)
// what it leaves goes in as a second fp16 operand, which leaves 2^-22 (or the same 2^-23).
// The running maximum is lazy: p = 2^(x - m) with an integer m that is raised only when a score passes
// m + 8 (p <= 2^8 then, which fp16 and fp32 hold as well as p <= 1), so a tile needs one vote
// instead of a maximum across the warp, and the same vote finds a t beyond what the norms allow.
// The true maximum is kept per thread and put in at the end.
//
// Work split.  Every (sequence, cache head, group of 8 NT query rows) is a unit of 32-key
// tiles; all units' tiles in a row (and kQ4UnitTiles more for each unit) are cut evenly over the CTAs (one per SM) and each CTA's
// share over its warps.  A warp is on its own: it copies its tiles (cp.async.bulk, one or two
// 16-token groups each) into its ring, waits, computes and refills, with no CTA barrier, and
// carries (m, l, O) in registers.  Lengths are read on the device, so the split is even
// whatever they are.  A unit that one warp covers is written straight to O; parts are merged
// at the CTA's end in shared memory, and units that cross CTAs by the last CTA to arrive
// (at most two parts per CTA in the workspace, merged in CTA order: results do not depend on
// timing).
//
// Measured, 32 query and 8 cache heads of 128 (bytes of codes and words over time; 6.55 TB/s is a copy):
// B=64, KV=4096 69.9 us (4.1 TB/s; bf16 65.9), B=16 25.7 (2.8), B=1, KV=131072, bf16 38.2 (3.7), B=1, KV=512
// 8.3.  The copies alone take 46 us at B=64 and 24.6 at KV=131072.  The rest is latency inside a warp: 296
// instructions for 16 keys form one chain (scores, exponentials, transposition, values' products), and 3 warps
// a scheduler issue 1.9 of 4 a clock at B=16 with no pipe more than 42 % busy (ALU; tensor 27 %); for few
// sequences it is the chain of loads before the first tile (about 6000 clocks) and the merges.
#pragma once

#include "cache_sm100.cuh"

namespace kf {

struct Q4AttnParams {
    const uint8_t* cache;
    const uint16_t* Q;            // [B, H_q, S_q, D]
    void* O;                      // [B, H_q, S_q, D]
    float* Mi;                    // nullable
    float* Li;                    // nullable
    const int* table;             // [B, max_blocks]
    const int* lens;              // [B]
    unsigned* tickets;            // [grid], zero between calls
    float* parts;                 // [grid][2][PART_FLOATS]
    int B, H_kv, S_q;
    int R;                        // query rows of a cache head: H_q / H_kv * S_q
    int n_rg;                     // row groups of 8 NT of them
    int n_blocks, bs_log2, max_blocks;
    int causal, q_bf16, out_type;
    float scale_log2;             // scale * log2(e)
    unsigned long long timeout_ns;
};

template <int D_, int NT_>
struct Q4AttnCfg {
    static constexpr int D = D_, NT = NT_;
    // As many warps as the registers allow without spills in the loop (D = 64 with 12 warps: 51.2 us instead of
    // 45.8 at B=32, KV=8192; D = 128 with 16: 128 registers, which spill; D = 64 with 16 rows and two operands
    // of p spills 4 bytes).  Two stages hide the copies; a third
    // costs 0 to 2 % at 12 warps of 8 rows and gains 2 % at 8 warps of 16.
    static constexpr int W = D == 256 ? 8 : NT == 1 ? (D == 64 ? 16 : 12) : (D == 64 ? 12 : 8);   // warps
    static constexpr int STAGES = NT == 2 || D == 64 ? 3 : 2;
    static constexpr int THREADS = 32 * W;
    static constexpr int GROUP = Q4<D>::GROUP;
    static constexpr int STAGE_BYTES = 2 * GROUP;                // a tile: 32 keys
    static constexpr int MT = D / 16;                            // 16-dim output tiles
    static constexpr int SETS = D == 256 ? 2 : 1;                // sets of 8 of them (4 for D = 64)
    static constexpr int IV = D == 64 ? 4 : 8;                   // tiles in a set
    static constexpr int V4 = IV / 4;
    static constexpr int KW = D / 32;                            // words of a key's row a thread holds
    static constexpr int ROWS = 8 * NT;
    static constexpr int O_FLOATS = ROWS * D;
    static constexpr int PART_FLOATS = O_FLOATS + 2 * ROWS;      // O, m, l
    static constexpr int RING_BYTES = W * STAGES * STAGE_BYTES;
    static constexpr int SMEM_BYTES = RING_BYTES + W * PART_FLOATS * 4;
    static_assert(STAGES <= 16 && STAGES * STAGE_BYTES >= PART_FLOATS * 4, "a warp's last part is kept in its ring");
    static_assert(SMEM_BYTES <= 225 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// mma_16816 with a zero C.
__device__ __forceinline__ void mma_16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
constexpr uint32_t kNibLo = 0x000F000Fu, kNibHi = 0x00F000F0u;
constexpr uint32_t kHalf2Exp15 = 0x78007800u, kHalf2Exp11 = 0x68006800u;   // half2 of 2^15, 2^11

// -z * 2^-9 of two zero points (integers in the low bits of each half).
__device__ __forceinline__ uint32_t q4_negz(uint32_t z) { return hfma2_u(z, kHalf2Exp15 | 0x80008000u, 0u); }

// Two codes in bits 0..3 (lo) or 4..7 (hi) of each half -> half2 (n - z) * 2^-9.
__device__ __forceinline__ uint32_t q4_lo(uint32_t x, uint32_t negz) { return hfma2_u(x & kNibLo, kHalf2Exp15, negz); }
__device__ __forceinline__ uint32_t q4_hi(uint32_t x, uint32_t negz) { return hfma2_u(x & kNibHi, kHalf2Exp11, negz); }

// Four codes of two keys (x: key 0 in the low, key 1 in the high half).
__device__ __forceinline__ void q4_unpack4(uint32_t x, uint32_t negz, uint32_t (&a)[4]) {
    a[0] = q4_lo(x, negz);
    a[1] = q4_hi(x, negz);
    x >>= 8;
    a[2] = q4_lo(x, negz);
    a[3] = q4_hi(x, negz);
}

// A warp's position in the row of tiles.
struct Q4Cursor {
    int b, h, rg, tile;            // sequence, cache head, row group, tile of 32 keys
    int nt, len;                   // the sequence's tiles and keys
};

constexpr float kQ4NoMax = -3.402823466e38f;                    // below every finite score

template <int D, int NT>
struct Q4Warp {                    // a warp's running state of one unit; pairs: columns 2t, 2t + 1
    float o[NT][Q4AttnCfg<D, NT>::MT][4];
    float2 m[NT], l[NT];           // reference of the exponent (kQ4NoMax before the first key), sum of p
    float2 mt[NT];                 // this thread's largest score
    uint32_t q[NT][Q4AttnCfg<D, NT>::KW][4];
    float2 qs[NT], cq[NT];         // -sum(q) * 2^-22, and a column's factor of the scores
    float2 norm[NT];               // a column's factor of p t, a power of two
    float tlim;                    // value scales up to tlim times this thread's norms stay within 2^7
};

__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }   // 2^(e - 127)
constexpr int kQ4NormMin = 6, kQ4NormMax = 233;                  // biased exponents of norm: 2^-121, 2^106

__device__ __forceinline__ float2 fmax2(float2 a, float2 b) { return make_float2(fmaxf(a.x, b.x), fmaxf(a.y, b.y)); }

__device__ __forceinline__ int q4_len(const Q4AttnParams& p, int b) {
    const int cap = p.max_blocks << p.bs_log2;
    const int n = p.lens[b];
    return n < 0 ? 0 : n > cap ? cap : n;
}
// Tiles of a sequence: an empty one keeps one (masked) tile, whose unit writes the zeros.
__device__ __forceinline__ int q4_tiles(int len) { return len <= 32 ? 1 : (len + 31) >> 5; }

__device__ __forceinline__ void q4_next_unit(const Q4AttnParams& p, Q4Cursor& c) {
    c.tile = 0;
    if (++c.rg < p.n_rg) return;
    c.rg = 0;
    if (++c.h < p.H_kv) return;
    c.h = 0;
    if (++c.b < p.B) {
        c.len = q4_len(p, c.b);
        c.nt = q4_tiles(c.len);
    }
}
__device__ __forceinline__ int q4_unit(const Q4AttnParams& p, const Q4Cursor& c) {
    return (c.b * p.H_kv + c.h) * p.n_rg + c.rg;
}

// The unit's query rows, raw (lane (g, t): row g of each 8, its chunks of 8 dims).
template <int D, int NT>
__device__ __forceinline__ void q4_load_q(const Q4AttnParams& p, uint4 (&raw)[NT][Q4AttnCfg<D, NT>::KW], const Q4Cursor& c,
                                          int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int g = lane >> 2, t = lane & 3;
    const uint16_t* q = p.Q + (static_cast<size_t>(c.b) * p.H_kv + c.h) * p.R * D;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = c.rg * C::ROWS + 8 * n + g;
#pragma unroll
        for (int i = 0; i < C::KW; ++i) {
            const int chunk = D == 64 ? 2 * t + i : (i >> 2) * 16 + 4 * t + (i & 3);
            raw[n][i] = r < p.R ? reinterpret_cast<const uint4*>(q + static_cast<size_t>(r) * D)[chunk] : make_uint4(0u, 0u, 0u, 0u);
        }
    }
}

// Unit start: queries to MMA operands (B fragments: column = query g, k = dims of lane t).
template <int D, int NT>
__device__ __forceinline__ void q4_begin(const Q4AttnParams& p, Q4Warp<D, NT>& s, const uint4 (&raw)[NT][Q4AttnCfg<D, NT>::KW],
                                         const Q4Cursor& c, int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int t = lane & 3;
    s.tlim = pow2_biased(261 - kQ4NormMax);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float x[C::KW][8], mx = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < C::KW; ++i) {
            if (p.q_bf16) unpack8<true>(raw[n][i], x[i]);
            else unpack8<false>(raw[n][i], x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[i][e]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int ex = static_cast<int>(__float_as_uint(mx) >> 23);            // biased exponent of the row's maximum
        ex = ex < 14 ? 14 : ex;
        const float f = __uint_as_float(static_cast<uint32_t>(267 - ex) << 23);   // 2^13 / 2^(ex - 127)
#pragma unroll
        for (int i = 0; i < C::KW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = x[i][e] * f, b = x[i][e + 4] * f;
                sum += a + b;
                s.q[n][i][e] = e & 1 ? pack_half2(a * 0.0625f, b * 0.0625f) : pack_half2(a, b);
            }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const float qs = sum * -0x1p-22f;
        const float cq = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(ex - 13) << 23) * 0x1p22f;
        s.qs[n].x = __shfl_sync(0xffffffffu, qs, 8 * t);
        s.qs[n].y = __shfl_sync(0xffffffffu, qs, 8 * t + 4);
        s.cq[n].x = __shfl_sync(0xffffffffu, cq, 8 * t);
        s.cq[n].y = __shfl_sync(0xffffffffu, cq, 8 * t + 4);
        s.m[n] = make_float2(kQ4NoMax, kQ4NoMax);
        s.mt[n] = make_float2(-INFINITY, -INFINITY);
        s.l[n] = make_float2(0.f, 0.f);
        s.norm[n] = make_float2(pow2_biased(kQ4NormMax), pow2_biased(kQ4NormMax));
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s.o[n][i][e] = 0.f;
    }
}

// One tile of 32 keys from shared memory.  MASKED: some key is outside the sequence, hidden
// from a row, or in a page outside the pool (valid: bit j set when group j was copied).
template <int D, int NT, bool SPLIT, bool MASKED>
__device__ __forceinline__ void q4_tile(const Q4AttnParams& p, Q4Warp<D, NT>& s, const uint8_t* st, const Q4Cursor& c,
                                        uint32_t valid, int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int g = lane >> 2, t = lane & 3, key0 = c.tile * 32, len = c.len;
    int lim[NT][2];                // keys the column's query sees
    if (MASKED) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                lim[n][k] = len - (p.causal ? p.S_q - 1 - (c.rg * C::ROWS + 8 * n + 2 * t + k) % p.S_q : 0);
    }
    float2 x[2][NT][2];            // scores [group][query tile][row g or g + 8]
    float tv[2][2];                // value scales of the same rows
    // S^T = K Q^T, in two chains per 128 dims, added up in fp32
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint8_t* gr = st + j * C::GROUP;
        constexpr int NW = D == 64 ? 2 : 4;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(gr + Q4<D>::K_WORDS);
        const uint32_t wk[2] = {words[g], words[g + 8]};
#pragma unroll
        for (int hf = 0; hf < (D == 256 ? 2 : 1); ++hf) {
            uint32_t wa[NW], wb[NW];
            if constexpr (D == 64) {
                const uint2 a = *reinterpret_cast<const uint2*>(gr + g * 32 + t * 8);
                const uint2 b = *reinterpret_cast<const uint2*>(gr + (g + 8) * 32 + t * 8);
                wa[0] = a.x; wa[1] = a.y; wb[0] = b.x; wb[1] = b.y;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(gr + g * (D / 2) + hf * 64 + t * 16);
                const uint4 b = *reinterpret_cast<const uint4*>(gr + (g + 8) * (D / 2) + hf * 64 + t * 16);
                wa[0] = a.x; wa[1] = a.y; wa[2] = a.z; wa[3] = a.w;
                wb[0] = b.x; wb[1] = b.y; wb[2] = b.z; wb[3] = b.w;
            }
            float acc[2][NT][4];
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int w = hf * 4 + i;
                const uint32_t ua = wa[i] << 2, ub = wb[i] << 2, va = wa[i] >> 6, vb = wb[i] >> 6;
                const uint32_t a0 = ua & 0x003C003Cu, a1 = ub & 0x003C003Cu, a2 = ua & 0x03C003C0u, a3 = ub & 0x03C003C0u;
                const uint32_t c0 = va & 0x003C003Cu, c1 = vb & 0x003C003Cu, c2 = va & 0x03C003C0u, c3 = vb & 0x03C003C0u;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (i == 0) {
                        mma_16816_first(acc[0][n], a0, a1, a2, a3, s.q[n][w][0], s.q[n][w][1]);
                        mma_16816_first(acc[1][n], c0, c1, c2, c3, s.q[n][w][2], s.q[n][w][3]);
                    } else {
                        mma_16816(acc[0][n], a0, a1, a2, a3, s.q[n][w][0], s.q[n][w][1]);
                        mma_16816(acc[1][n], c0, c1, c2, c3, s.q[n][w][2], s.q[n][w][3]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 v = fadd2(make_float2(acc[0][n][2 * h], acc[0][n][2 * h + 1]),
                                           make_float2(acc[1][n][2 * h], acc[1][n][2 * h + 1]));
                    x[j][n][h] = hf == 0 ? v : fadd2(x[j][n][h], v);
                }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key = key0 + 16 * j + 8 * h + g;
            const float sc = q4_scale(wk[h]), z = __uint_as_float(0x4B000000u | (wk[h] & 15u)) - 8388608.0f;
            tv[j][h] = q4_scale(words[16 + g + 8 * h]);
            if (MASKED && (!((valid >> j) & 1u) || key >= len)) tv[j][h] = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float2 v = fmul2(ffma2(make_float2(z, z), s.qs[n], x[j][n][h]), fmul2(make_float2(sc, sc), s.cq[n]));
                if (MASKED) {
                    if (!((valid >> j) & 1u)) v = make_float2(0.f, 0.f);     // a page outside the pool reads zeros
                    if (key >= lim[n][0]) v.x = -INFINITY;
                    if (key >= lim[n][1]) v.y = -INFINITY;
                }
                x[j][n][h] = v;
            }
        }
    }
    // Does a score pass m + 8, or a value scale what the norms are good for?  Rarely.
    const float tm = fmax3f(fmax3f(tv[0][0], tv[0][1], tv[1][0]), tv[1][1], 0.f);   // (a spoiled row's NaN is ignored)
    bool up = tm > s.tlim;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        s.mt[n].x = fmax3f(fmax3f(s.mt[n].x, x[0][n][0].x, x[0][n][1].x), x[1][n][0].x, x[1][n][1].x);
        s.mt[n].y = fmax3f(fmax3f(s.mt[n].y, x[0][n][0].y, x[0][n][1].y), x[1][n][0].y, x[1][n][1].y);
        up = up || s.mt[n].x > s.m[n].x + 8.0f || s.mt[n].y > s.m[n].y + 8.0f;
    }
    if (__any_sync(0xffffffffu, up)) {
        const int et = static_cast<int>(__reduce_max_sync(0xffffffffu, __float_as_uint(tm)) >> 23);
        int top = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float v[2] = {s.mt[n].x, s.mt[n].y}, a[2], r[2], nm[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float m = k ? s.m[n].y : s.m[n].x;
                v[k] = fmaxf(v[k], __shfl_xor_sync(0xffffffffu, v[k], 4));
                v[k] = fmaxf(v[k], __shfl_xor_sync(0xffffffffu, v[k], 8));
                v[k] = fmaxf(v[k], __shfl_xor_sync(0xffffffffu, v[k], 16));
                v[k] = fmaxf(ceilf(v[k]), m);                                // (no key seen by this column yet: kQ4NoMax)
                float pt = 0.f;                                              // the tile's largest p t that the column sees
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        pt = fmaxf(pt, ex2_approx((k ? x[j][n][h].y : x[j][n][h].x) - v[k]) * tv[j][h]);
                pt = fmaxf(pt, __shfl_xor_sync(0xffffffffu, pt, 4));
                pt = fmaxf(pt, __shfl_xor_sync(0xffffffffu, pt, 8));
                pt = fmaxf(pt, __shfl_xor_sync(0xffffffffu, pt, 16));
                const int d = static_cast<int>(fminf(v[k] - m, 512.0f));     // m moves by whole powers of two
                const int was = static_cast<int>(__float_as_uint(k ? s.norm[n].y : s.norm[n].x) >> 23);
                int e = 260 - et;                                            // t norm < 2^7 ...
                e = max(e, pt > 0.f ? 252 - static_cast<int>(__float_as_uint(pt) >> 23) : 0);   // ... but p t norm >= 2^-2
                e = max(min(min(e, was + d), kQ4NormMax), kQ4NormMin);       // O is never scaled up
                const int er = 127 - d + e - was;
                top = max(top, e);
                nm[k] = pow2_biased(e);
                a[k] = d < 127 ? pow2_biased(127 - d) : 0.f;
                r[k] = er > 0 ? pow2_biased(er) : 0.f;
            }
            s.m[n] = make_float2(v[0], v[1]);
            s.norm[n] = make_float2(nm[0], nm[1]);
            s.l[n] = make_float2(s.l[n].x * a[0], s.l[n].y * a[1]);
#pragma unroll
            for (int i = 0; i < C::MT; ++i) {
                s.o[n][i][0] *= r[0];
                s.o[n][i][1] *= r[1];
                s.o[n][i][2] *= r[0];
                s.o[n][i][3] *= r[1];
            }
        }
        s.tlim = pow2_biased(261 - top);                                     // 2^7 / the larger norm
    }
    // O^T += V^T P^T
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint8_t* gr = st + j * C::GROUP;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(gr + Q4<D>::V_WORDS);
        uint32_t pb[NT][2], pl[NT][2];                                       // p t, and (SPLIT) what its rounding left
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 d = fadd2(x[j][n][h], make_float2(-s.m[n].x, -s.m[n].y));
                const float2 pr = make_float2(ex2_approx(d.x), ex2_approx(d.y));
                s.l[n] = fadd2(s.l[n], pr);
                float2 pt = fmul2(fmul2(pr, make_float2(tv[j][h], tv[j][h])), s.norm[n]);
                if (MASKED) {                                                // 0 * a spoiled row's NaN
                    const int key = key0 + 16 * j + 8 * h + g;
                    if (key >= lim[n][0]) pt.x = 0.f;
                    if (key >= lim[n][1]) pt.y = 0.f;
                }
                const uint32_t hi = pack_half2(pt.x, pt.y);
                pb[n][h] = movmatrix_trans(hi);
                if (SPLIT) {
                    const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                    const float2 lo = fadd2(pt, make_float2(-back.x, -back.y));
                    pl[n][h] = movmatrix_trans(pack_half2(lo.x, lo.y));
                }
            }
        }
        const uint2 z01 = *reinterpret_cast<const uint2*>(words + 2 * t);
        const uint2 z89 = *reinterpret_cast<const uint2*>(words + 8 + 2 * t);
        const uint32_t za = q4_negz(__byte_perm(z01.x, z01.y, 0x5410) & kNibLo);
        const uint32_t zb = q4_negz(__byte_perm(z89.x, z89.y, 0x5410) & kNibLo);
        const uint8_t* vr = gr + Q4<D>::V_CODES + 2 * t * (D / 2);
        constexpr int R1 = D / 2, R8 = 8 * (D / 2);                      // next key, eighth next key
        if constexpr (D == 64) {
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(vr + g * 4);
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(vr + R1 + g * 4);
            const uint32_t w8 = *reinterpret_cast<const uint32_t*>(vr + R8 + g * 4);
            const uint32_t w9 = *reinterpret_cast<const uint32_t*>(vr + R8 + R1 + g * 4);
            uint32_t a0[4], a1[4], a2[4], a3[4];
            q4_unpack4(__byte_perm(w0, w1, 0x5410), za, a0);
            q4_unpack4(__byte_perm(w0, w1, 0x7632), za, a1);
            q4_unpack4(__byte_perm(w8, w9, 0x5410), zb, a2);
            q4_unpack4(__byte_perm(w8, w9, 0x7632), zb, a3);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_16816(s.o[n][i], a0[i], a1[i], a2[i], a3[i], pb[n][0], pb[n][1]);
                    if (SPLIT) mma_16816(s.o[n][i], a0[i], a1[i], a2[i], a3[i], pl[n][0], pl[n][1]);
                }
        } else {
#pragma unroll
            for (int set = 0; set < C::SETS; ++set) {
                const int at = g * (8 * C::SETS) + 8 * set;
                const uint2 w0 = *reinterpret_cast<const uint2*>(vr + at);
                const uint2 w1 = *reinterpret_cast<const uint2*>(vr + R1 + at);
                const uint2 w8 = *reinterpret_cast<const uint2*>(vr + R8 + at);
                const uint2 w9 = *reinterpret_cast<const uint2*>(vr + R8 + R1 + at);
#pragma unroll
                for (int q = 0; q < 2; ++q) {                            // codes 0..3, then 4..7 of each word
                    const uint32_t sel = q == 0 ? 0x5410u : 0x7632u;
                    uint32_t a0[4], a1[4], a2[4], a3[4];
                    q4_unpack4(__byte_perm(w0.x, w1.x, sel), za, a0);
                    q4_unpack4(__byte_perm(w0.y, w1.y, sel), za, a1);
                    q4_unpack4(__byte_perm(w8.x, w9.x, sel), zb, a2);
                    q4_unpack4(__byte_perm(w8.y, w9.y, sel), zb, a3);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float(&o)[4] = s.o[n][set * 8 + q * 4 + i];
                            mma_16816(o, a0[i], a1[i], a2[i], a3[i], pb[n][0], pb[n][1]);
                            if (SPLIT) mma_16816(o, a0[i], a1[i], a2[i], a3[i], pl[n][0], pl[n][1]);
                        }
                }
            }
        }
    }
}

// Parts keep the accumulators' own order: float4 v of item (n, set, e) of lane (g, t) holds
// column 8n + 2t + (e & 1) and four neighbouring dims from q4_dim().
template <int D>
__device__ __forceinline__ int q4_dim(int set, int e, int v, int g) {
    if constexpr (D == 64) return 8 * g + 4 * (e >> 1);
    return (D / 8) * g + 16 * set + 8 * (e >> 1) + 4 * v;
}

// A unit's output rows.
struct Q4Unit {
    int u;                         // unit number (sequence, head, row group); -1: no part here
    int start, nt;                 // its first tile in the row of all tiles, and their count
};

// End of a warp's share of a unit: O, m and l in true units, to the output or to a part.
template <int D, int NT>
__device__ __forceinline__ void q4_emit(const Q4AttnParams& p, Q4Warp<D, NT>& s, const Q4Cursor& c, bool whole, float* part,
                                        int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int g = lane >> 2, t = lane & 3;
    const int row0 = c.rg * C::ROWS;
    const size_t rbase = (static_cast<size_t>(c.b) * p.H_kv + c.h) * p.R;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float2 l = s.l[n], m = s.mt[n];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l = fadd2(l, make_float2(__shfl_xor_sync(0xffffffffu, l.x, o), __shfl_xor_sync(0xffffffffu, l.y, o)));
            m = fmax2(m, make_float2(__shfl_xor_sync(0xffffffffu, m.x, o), __shfl_xor_sync(0xffffffffu, m.y, o)));
        }
        // From the exponent's reference to the true maximum (at most 8 above it).
        const float2 a = make_float2(m.x == -INFINITY ? 1.0f : ex2_approx(s.m[n].x - m.x),
                                     m.y == -INFINITY ? 1.0f : ex2_approx(s.m[n].y - m.y));
        l = fmul2(l, a);
        float2 f = fmul2(a, make_float2(pow2_biased(254 - static_cast<int>(__float_as_uint(s.norm[n].x) >> 23)),
                                        pow2_biased(254 - static_cast<int>(__float_as_uint(s.norm[n].y) >> 23))));
        if (whole) f = fmul2(f, make_float2(l.x == 0.f ? 0.f : 1.0f / l.x, l.y == 0.f ? 0.f : 1.0f / l.y));
        const int col = 8 * n + 2 * t;
#pragma unroll
        for (int set = 0; set < C::SETS; ++set)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int v = 0; v < C::V4; ++v) {
                    float2 y[4];                                             // 2^9 by itself: with f it could leave fp32's range
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float(&o)[4] = s.o[n][set * 8 + 4 * v + i];
                        y[i] = fmul2(fmul2(make_float2(o[2 * h], o[2 * h + 1]), make_float2(0x1p9f, 0x1p9f)), f);
                    }
                    const float4 y0 = make_float4(y[0].x, y[1].x, y[2].x, y[3].x), y1 = make_float4(y[0].y, y[1].y, y[2].y, y[3].y);
                    if (!whole) {
                        float4* at = reinterpret_cast<float4*>(part) + (((n * C::SETS + set) * 4 + 2 * h) * C::V4 + v) * 32 + lane;
                        at[0] = y0;
                        at[C::V4 * 32] = y1;
                    } else {
                        const size_t at = (rbase + row0 + col) * D + q4_dim<D>(set, 2 * h, v, g);
                        if (row0 + col < p.R) store_out4(p.O, at, y0, p.out_type);
                        if (row0 + col + 1 < p.R) store_out4(p.O, at + D, y1, p.out_type);
                    }
                }
        if (g == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float mk = k ? m.y : m.x, lk = k ? l.y : l.x;
                if (!whole) {
                    part[C::O_FLOATS + col + k] = mk;
                    part[C::O_FLOATS + C::ROWS + col + k] = lk;
                } else if (row0 + col + k < p.R) {
                    if (p.Mi) p.Mi[rbase + row0 + col + k] = mk * 0.6931471805599453f;
                    if (p.Li) p.Li[rbase + row0 + col + k] = lk;
                }
            }
        }
    }
}

// What the merge of a unit across CTAs costs, in tiles of one CTA.  Fitted at D = 128 and good for the others:
// B=16, 8 cache heads, with 0 (an even split whenever it is shorter) / 32 / 64, in us:
//   rows x D    KV=2048              KV=4096              KV=8192
//   4 x 64      15.0 / 13.5 / 13.3   19.5 / 18.5 / 18.4   28.7 / 28.4 / 28.7
//   4 x 128     17.9 / 16.8 / 16.9   25.6 / 25.2 / 25.1   39.8 / 39.8 / 41.9
//   4 x 256     26.9 / 25.4 / 25.2   39.9 / 40.5 / 40.4   65.4 / 65.6 / 71.0
//   16 x 64     19.1 / 16.4 / 16.4   26.4 / 24.1 / 24.1   40.3 / 40.0 / 40.2
//   16 x 128    24.9 / 23.1 / 23.1   36.3 / 36.6 / 36.6   59.2 / 59.0 / 63.6
constexpr unsigned kQ4MergeTiles = 32;
// What a unit costs a warp besides its tiles (queries in, results out), in tiles.  (With 0: 48 sequences
// of 1 to 8192 keys 24.6 us instead of 18.3.)
constexpr int kQ4UnitTiles = 2;

__device__ __forceinline__ float q4_weight(float m, float M) { return m == -INFINITY ? 0.f : ex2_approx(m - M); }

// One thread's share of a merge: the V4 float4 of item idx / 32, lane idx % 32 (q4_emit's order),
// over parts 0..count-1.  Part i is at first (i = 0), last (i = count - 1) or mid + i * stride.
template <int D, int NT>
struct Q4Merged {
    float4 a[Q4AttnCfg<D, NT>::V4];
    float M, L;
    int col, dim;
    bool stats;                    // this thread also writes the column's M and L
};
template <int D, int NT, bool GLOBAL>
__device__ __forceinline__ Q4Merged<D, NT> q4_merge(int idx, int count, const float* first, const float* mid, size_t stride,
                                                    const float* last) {
    using C = Q4AttnCfg<D, NT>;
    constexpr int U = GLOBAL ? (C::V4 == 1 ? 16 : 10) : 4;               // parts in flight
    const int ln = idx & 31, item = idx >> 5;
    const int e = item & 3, set = (item >> 2) % C::SETS, n = item / (4 * C::SETS);
    Q4Merged<D, NT> r;
    r.col = 8 * n + 2 * (ln & 3) + (e & 1);
    r.dim = q4_dim<D>(set, e, 0, ln >> 2);
    r.stats = (ln >> 2) == 0 && set == 0 && (e >> 1) == 0;
    r.M = -INFINITY;
    r.L = 0.f;
#pragma unroll
    for (int v = 0; v < C::V4; ++v) r.a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int st = C::O_FLOATS + r.col, at = item * (C::V4 * 128) + ln * 4;
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += U) {
        float m[U], l[U], M = r.M;
        float4 y[U][C::V4];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            m[i] = -INFINITY;
            if (i0 + i >= count) continue;
            const float* part = i0 + i == 0 ? first : i0 + i == count - 1 ? last : mid + (i0 + i) * stride;
            m[i] = GLOBAL ? __ldcg(part + st) : part[st];
            l[i] = GLOBAL ? __ldcg(part + st + C::ROWS) : part[st + C::ROWS];
#pragma unroll
            for (int v = 0; v < C::V4; ++v) {
                const float4* src = reinterpret_cast<const float4*>(part + at) + v * 32;
                y[i][v] = GLOBAL ? __ldcg(src) : *src;
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) M = fmaxf(M, m[i]);
        const float w0 = q4_weight(r.M, M);
        r.M = M;
        r.L *= w0;
#pragma unroll
        for (int v = 0; v < C::V4; ++v) { r.a[v].x *= w0; r.a[v].y *= w0; r.a[v].z *= w0; r.a[v].w *= w0; }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (i0 + i >= count) continue;
            const float w = q4_weight(m[i], M);
            r.L = fmaf(w, l[i], r.L);
#pragma unroll
            for (int v = 0; v < C::V4; ++v) {
                r.a[v].x = fmaf(w, y[i][v].x, r.a[v].x); r.a[v].y = fmaf(w, y[i][v].y, r.a[v].y);
                r.a[v].z = fmaf(w, y[i][v].z, r.a[v].z); r.a[v].w = fmaf(w, y[i][v].w, r.a[v].w);
            }
        }
    }
    return r;
}
template <int D, int NT>
__device__ __forceinline__ void q4_write(const Q4AttnParams& p, const Q4Merged<D, NT>& r, int u) {
    using C = Q4AttnCfg<D, NT>;
    const int h = p.n_rg == 1 ? u : u / p.n_rg, row = (u - h * p.n_rg) * C::ROWS + r.col;
    if (row >= p.R) return;
    const size_t at = static_cast<size_t>(h) * p.R + row;
    const float inv = r.L == 0.f ? 0.f : 1.0f / r.L;
#pragma unroll
    for (int v = 0; v < C::V4; ++v)
        store_out4(p.O, at * D + r.dim + 4 * v,
                   make_float4(r.a[v].x * inv, r.a[v].y * inv, r.a[v].z * inv, r.a[v].w * inv), p.out_type);
    if (r.stats && p.Mi) p.Mi[at] = r.M * 0.6931471805599453f;
    if (r.stats && p.Li) p.Li[at] = r.L;
}

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(Q4AttnCfg<D, NT>::THREADS, 1) q4_attn_kernel(const __grid_constant__ Q4AttnParams p) {
    using C = Q4AttnCfg<D, NT>;
    constexpr int W = C::W, STAGES = C::STAGES;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[W][STAGES];
    __shared__ int s_abort, s_drop[W], s_last[2];
    __shared__ uint32_t s_valid[W][STAGES];                              // groups copied, 2 bits
    __shared__ Q4Unit s_ent[2 * W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* heads = reinterpret_cast<float*>(smem + C::RING_BYTES);
    uint8_t* ring = smem + warp * STAGES * C::STAGE_BYTES;

    if (tid == 0) s_abort = 0;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&bars[warp][i], 1);
        s_ent[2 * warp].u = s_ent[2 * warp + 1].u = -1;
        fence_mbar_init();
    }
    __syncthreads();
    grid_dep_launch_dependents();
    grid_dep_wait();

    // ---- the row of slots: a unit's tiles and kQ4UnitTiles empty slots for what a unit costs by
    // itself.  Totals, this CTA's share, this warp's place (every warp for itself: lane i counts
    // sequences i * per ...).
    constexpr int OV = kQ4UnitTiles;
    const int HR = p.H_kv * p.n_rg;
    const int per = (p.B + 31) >> 5;
    const int b0 = lane * per < p.B ? lane * per : p.B, b1 = b0 + per < p.B ? b0 + per : p.B;
    const int nt0 = q4_tiles(q4_len(p, 0));
    int mine = 0;
    bool same = true;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int nt = q4_tiles(q4_len(p, b));
        mine += nt + OV;
        same = same && nt == nt0;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    const unsigned T = __shfl_sync(0xffffffffu, incl, 31) * HR;          // < 2^31, the host sees to it
    // CTAs that take part: about a slot for every warp of theirs at least.  CTA c has the slots from
    // c * quot + min(c, rem), its warps even shares of them; where there are fewer slots than warps, the
    // last warps are the ones without (the merge below relies on a unit's warps being neighbours).
    const unsigned want = (T + W - 1) / W;
    unsigned act = want < gridDim.x ? want : gridDim.x, quot = T / act, rem = T - quot * act;
    // Sequences of one length: whole units to each CTA, if that takes no longer than an even
    // split and the merge across CTAs that it needs.
    if (__all_sync(0xffffffffu, same)) {
        const unsigned units = p.B * HR, each = units <= gridDim.x ? 1 : (units + gridDim.x - 1) / gridDim.x;
        if (each * (nt0 + OV) <= quot + kQ4MergeTiles) {
            act = each == 1 ? units : (units + each - 1) / each;
            quot = each * (nt0 + OV);
            rem = 0;
        }
    }
    if (blockIdx.x >= act) return;
    const int x0 = blockIdx.x * quot + (blockIdx.x < rem ? blockIdx.x : rem);
    const int x1 = blockIdx.x == act - 1 ? T : x0 + quot + (blockIdx.x < rem ? 1 : 0);
    const int wq = (x1 - x0) / W, wr = (x1 - x0) % W;
    const int z0 = x0 + warp * wq + (warp < wr ? warp : wr), z1 = z0 + wq + (warp < wr ? 1 : 0);

    // The tile at slot z (of an empty slot: the next unit's first) and its number among all tiles.
    auto locate = [&](int z, Q4Cursor& c) {
        const int lo = (incl - mine) * HR;
        const bool here = z >= lo && z < incl * HR;
        int b = b0, at = lo;
        if (here)
            for (; b < b1 - 1; ++b) {
                const int next = at + (q4_tiles(q4_len(p, b)) + OV) * HR;
                if (z < next) break;
                at = next;
            }
        const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
        c.b = __shfl_sync(0xffffffffu, b, from);
        at = __shfl_sync(0xffffffffu, at, from);
        c.len = q4_len(p, c.b);
        c.nt = q4_tiles(c.len);
        const unsigned off = z - at, hr = off / (c.nt + OV), o = off - hr * (c.nt + OV);
        c.tile = static_cast<int>(o) < c.nt ? o : c.nt;
        c.h = hr;
        c.rg = 0;
        if (p.n_rg > 1) {
            c.h = hr / p.n_rg;
            c.rg = hr - c.h * p.n_rg;
        }
        const int y = at - OV * HR * c.b + hr * c.nt + c.tile;
        if (c.tile == c.nt) q4_next_unit(p, c);
        return y;
    };
    Q4Cursor cur, next;
    const int y0 = z0 < z1 ? locate(z0, cur) : 0;
    const int y1 = z0 == z1 ? 0 : z1 == static_cast<int>(T) ? z1 - OV * HR * p.B : locate(z1, next);

    if (y0 < y1) {
        int y_cur = y0;                                                  // the tile in work
        uint4 raw[NT][C::KW];
        q4_load_q<D, NT>(p, raw, cur, lane);                             // ahead of the copies

        // Copies.  Lane i holds what tile win0 + i needs and issues its copy.  The window moves on
        // every 32 tiles; the table entries of the next one are loaded when it does (a load waits
        // behind the copies in flight for microseconds).
        int issued = y0, win0 = y0;
        const uint8_t* src0 = nullptr;                                   // the window's groups, and which are in the pool
        const uint8_t* src1 = nullptr;
        uint32_t bytes = 0, valid = 0;
        const bool paired = p.bs_log2 == 4;
        unsigned e0 = 0, e1 = 0, e_at = 0;                               // the next one's; at: head << 4 | group in the page
        auto fetch = [&](int y) {                                        // for the window that begins at tile y
            e0 = e1 = 0xffffffffu;
            if (y + lane < y1) {
                int b = cur.b, len = cur.len, nt = cur.nt;
                unsigned off = (cur.h * p.n_rg + cur.rg) * nt + cur.tile + (y - y_cur) + lane;
                while (off >= static_cast<unsigned>(HR * nt)) {
                    off -= HR * nt;
                    len = q4_len(p, ++b);
                    nt = q4_tiles(len);
                }
                const unsigned hr = off / nt, tile = off - hr * nt, h = p.n_rg == 1 ? hr : hr / p.n_rg;
                const int left = len - static_cast<int>(tile) * 32;
                const unsigned page = (tile * 32) >> p.bs_log2;
                const int* row = p.table + static_cast<size_t>(b) * p.max_blocks + page;
                e_at = h << 4 | ((tile * 32) & ((1u << p.bs_log2) - 1)) >> 4;
                if (left > 0) e0 = row[0];
                if (left > 16) e1 = row[paired ? 1 : 0];
                // A unit that begins here: its queries on their way to L2, for the same reason.
                if (tile == 0 && y + lane != y0) {
                    const unsigned rg = hr - h * p.n_rg, rows = p.R - rg * C::ROWS;
                    const char* q = reinterpret_cast<const char*>(
                        p.Q + ((static_cast<size_t>(b) * p.H_kv + h) * p.R + rg * C::ROWS) * D);
                    for (unsigned at = 0; at < (rows < C::ROWS ? rows : C::ROWS) * D * 2; at += 128)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(q + at));
                }
            }
        };
        auto move_on = [&](int y) {
            win0 = y;
            const uint32_t page_bytes = static_cast<uint32_t>(C::GROUP) << (p.bs_log2 - 4);
            src0 = p.cache + static_cast<uint64_t>(e0 * p.H_kv + (e_at >> 4)) * page_bytes + (e_at & 15u) * C::GROUP;
            src1 = p.cache + static_cast<uint64_t>(e1 * p.H_kv + (e_at >> 4)) * page_bytes;
            valid = (e0 < static_cast<unsigned>(p.n_blocks) ? 1u : 0u) | (e1 < static_cast<unsigned>(p.n_blocks) ? 2u : 0u);
            bytes = __popc(valid) * C::GROUP;
            if (win0 + 32 < y1) fetch(win0 + 32);
        };
        auto issue = [&](int stage) {                                    // by the lane that holds the tile
            uint64_t* bar = &bars[warp][stage];
            uint8_t* dst = ring + stage * C::STAGE_BYTES;
            s_valid[warp][stage] = valid;
            mbar_arrive_expect_tx(bar, bytes);
            if (!paired) {
                if (valid) bulk_g2s(dst, src0, bytes, bar);              // both groups lie in one page
            } else {
                if (valid & 1u) bulk_g2s(dst, src0, C::GROUP, bar);
                if (valid & 2u) bulk_g2s(dst + C::GROUP, src1, C::GROUP, bar);
            }
        };

        fetch(y0);
        move_on(y0);
        issued = y0 + STAGES < y1 ? y0 + STAGES : y1;
        if (lane < issued - y0) issue(lane);
        __syncwarp();
        Q4Warp<D, NT> s;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
#pragma unroll 1
        while (y_cur < y1) {                                             // a unit, or the warp's share of it
            q4_begin<D, NT>(p, s, raw, cur, lane);
            const int first = cur.tile, n = cur.nt - first < y1 - y_cur ? cur.nt - first : y1 - y_cur;
            const int plain_end = cur.len - (p.causal ? p.S_q - 1 : 0) - 32;   // key0 up to here: all rows see all keys
#pragma unroll 1
            for (int i = 0; i < n && ok; ++i) {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bars[warp][stage], phase, &s_abort, p.timeout_ns))) {
                    // The copies in flight still land in this ring: wait for them (bounded) before leaving it.
                    if (lane == 0) atomicOr(&g_kf_dev_error, KF_DEVERR_TIMEOUT_TMA);
                    for (int z = y_cur, sz = stage, pz = phase; z < issued; ++z) {
                        s_drop[warp] = 0;
                        __syncwarp();
                        mbar_wait_bounded(&bars[warp][sz], pz, &s_drop[warp], p.timeout_ns + 1000000000ull);
                        __syncwarp();
                        if (++sz == STAGES) { sz = 0; pz ^= 1; }
                    }
                    ok = false;
                    break;
                }
                const uint32_t got = s_valid[warp][stage];
                const uint8_t* st = ring + stage * C::STAGE_BYTES;
                if (got != 3u || cur.tile * 32 > plain_end) q4_tile<D, NT, SPLIT, true>(p, s, st, cur, got, lane);
                else q4_tile<D, NT, SPLIT, false>(p, s, st, cur, got, lane);
                ++cur.tile;
                ++y_cur;
                __syncwarp();
                if (issued < y1) {
                    if (issued - win0 == 32) move_on(issued);
                    if (lane == issued - win0) issue(stage);
                    ++issued;
                }
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) {                                                   // (the parts still go through the merge)
                y_cur += first + n - cur.tile;
                cur.tile = first + n;
            }
            const bool whole = n == cur.nt, last = y_cur >= y1;
            // A part that ends inside the warp's share goes to the warp's head slot, the last one to its ring.
            float* part = last ? reinterpret_cast<float*>(ring) : heads + warp * C::PART_FLOATS;
            __syncwarp();
            const Q4Cursor done = cur;
            if (!last) {
                q4_next_unit(p, cur);
                q4_load_q<D, NT>(p, raw, cur, lane);
            }
            q4_emit<D, NT>(p, s, done, whole, part, lane);
            if (!whole && lane == 0)
                s_ent[2 * warp + (last ? 1 : 0)] = Q4Unit{q4_unit(p, done), y_cur - done.tile, done.nt};
        }
    }
    __syncthreads();

    // ---- merge the CTA's parts: runs of equal units in the entries' order
    constexpr int items = NT * C::SETS * 4;                              // warps that merge a run
    constexpr int teams = W / items > 0 ? W / items : 1;                 // runs merged side by side
    const int team = warp / items, in_team = tid - team * items * 32;
    int run_no = 0;
    const Q4Unit mine_u = lane < 2 * W ? s_ent[lane] : Q4Unit{-1, 0, 0};
    int cross_u[2] = {-1, -1}, cross_first[2] = {0, 0}, cross_n[2] = {0, 0};
    for (uint32_t todo = __ballot_sync(0xffffffffu, mine_u.u >= 0); todo;) {
        const int lead = __ffs(todo) - 1;
        const int u = __shfl_sync(0xffffffffu, mine_u.u, lead);
        const int us = __shfl_sync(0xffffffffu, mine_u.start, lead), unt = __shfl_sync(0xffffffffu, mine_u.nt, lead);
        const uint32_t run = __ballot_sync(0xffffffffu, mine_u.u == u);
        todo &= ~run;
        // A unit's first part here is in slot `lead`; the others are the last parts (odd slots) of
        // the warps that follow, but for the run's end, which may be a head (even) slot.
        const int count = __popc(run), end = 31 - __clz(run);
        auto entry = [&](int f) {
            return reinterpret_cast<const float*>(f & 1 ? smem + (f >> 1) * (STAGES * C::STAGE_BYTES)
                                                        : smem + C::RING_BYTES + (f >> 1) * (C::PART_FLOATS * 4));
        };
        const int ws = us + OV * u;                                      // the unit's first slot
        const bool inside = ws >= x0 && ws + unt <= x1;
        const int slot = ws >= x0 ? 1 : 0;
        float* out = p.parts + (static_cast<size_t>(blockIdx.x) * 2 + slot) * C::PART_FLOATS;
        const bool ours = teams == 1 || run_no % teams == team;
        ++run_no;
#pragma unroll 1
        for (int idx = teams == 1 ? tid : in_team; ours && idx < items * 32; idx += teams == 1 ? C::THREADS : items * 32) {
            const Q4Merged<D, NT> r = q4_merge<D, NT, false>(idx, count, entry(lead), entry(lead | 1),
                                                             STAGES * C::STAGE_BYTES / 4, entry(end));
            if (inside) {
                q4_write(p, r, u);
            } else {
                float4* o = reinterpret_cast<float4*>(out) + (idx >> 5) * (C::V4 * 32) + (idx & 31);
#pragma unroll
                for (int v = 0; v < C::V4; ++v) o[v * 32] = r.a[v];
                if (r.stats) {
                    out[C::O_FLOATS + r.col] = r.M;
                    out[C::O_FLOATS + C::ROWS + r.col] = r.L;
                }
            }
        }
        if (!inside) {
            auto cta_of = [&](unsigned x) {
                const unsigned big = rem * (quot + 1);
                return static_cast<int>(x < big ? x / (quot + 1) : rem + (x - big) / quot);
            };
            const int cf = slot ? static_cast<int>(blockIdx.x) : cta_of(ws), cl = cta_of(ws + unt - 1);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (k == slot) {
                    cross_u[k] = u;
                    cross_first[k] = cf;
                    cross_n[k] = cl - cf + 1;
                }
        }
    }
    if (cross_u[0] < 0 && cross_u[1] < 0) return;

    // ---- units that cross CTAs: the last CTA to arrive merges the parts, in CTA order
    __syncthreads();
    if (warp < 2 && lane == 0) {                                         // (its release covers what the barrier ordered before)
        const int u = warp ? cross_u[1] : cross_u[0], first = warp ? cross_first[1] : cross_first[0];
        const unsigned others = (warp ? cross_n[1] : cross_n[0]) - 1;
        s_last[warp] = 0;
        if (u >= 0 && atom_add_acq_rel_gpu(p.tickets + first, 1u) == others) {
            p.tickets[first] = 0u;
            s_last[warp] = 1;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        if (!s_last[k] || (teams > 1 && team != k)) continue;
        const int cf = k ? cross_first[1] : cross_first[0], u = k ? cross_u[1] : cross_u[0];
        const int count = k ? cross_n[1] : cross_n[0];
        const float* mid = p.parts + static_cast<size_t>(cf) * 2 * C::PART_FLOATS;   // its first CTA's second slot, then first slots
#pragma unroll 1
        for (int idx = teams == 1 ? tid : in_team; idx < items * 32; idx += teams == 1 ? C::THREADS : items * 32)
            q4_write(p, q4_merge<D, NT, true>(idx, count, mid + C::PART_FLOATS, mid, 2 * C::PART_FLOATS,
                                              mid + (count - 1) * 2 * C::PART_FLOATS), u);
    }
}

}  // namespace kf
