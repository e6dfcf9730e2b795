// Attention over the 4-bit paged KV cache (include/kf_cache.h) for B200 (sm_100a).
//
//   x_j = scale * s_j q . (n_j - z_j),  O = sum_j e^(x_j - m) t_j (n'_j - z'_j) / sum_j e^(x_j - m)
// with (s, z, n) a key's scale, zero point and codes and (t, z', n') a value's.
//
// What bounds it: a key and value of one head are D + 8 bytes, read once; at 6.5 TB/s an SM
// receives 46 codes per clock, so the codes have to become MMA operands in about two
// instructions per eight.  mma.m16n8k16 with the KEYS as its 16 rows and the queries as its 8
// columns (S^T = K Q^T, O^T = V^T P^T) wastes nothing for up to 8 query rows a cache head; the
// 128-row tcgen05 tiles would be 1/16 filled and want their operands expanded in memory.
//
// Codes to operands.  A 4-bit integer in the low bits of an fp16 is the subnormal n * 2^-24,
// so `word & 0x000F000F` is a half2 of codes 0 and 4 of eight, `word & 0x00F000F0` of 16 times
// codes 1 and 5, and a shift by 8 gives the other two.  One half2 FMA (on the FMA pipe, which
// is idle beside the integer work) makes (n - z) * 2^-9 of each, exact.  Subnormal operands
// would be exact products too, but the tensor core aligns its sums by the operands' exponent
// fields and drops their low bits (measured: scores off by 2^-18 instead of 2^-21); and sums of
// p t (n - z) keep the value's own size, where sum(p t n) - sum(p t z) would cancel.
// Queries are scaled by a power of two per row to a maximum in [2^13, 2^14), which holds fp16
// rows exactly, and bf16 ones but for elements below 2^-28 of the row's largest.
// p t enters the second product as fp16, scaled by a power of two such that the largest t seen
// is below 2^14 (t spans any range; small ones lose bits only against the largest).  This
// rounding, 2^-11 relative per key, is the only one below fp32 in the sum.
//
// Work split.  Every (sequence, cache head, group of 8 NT query rows) is a unit of 32-key
// tiles; all units' tiles in a row are cut evenly over the CTAs (one per SM) and each CTA's
// share over its warps.  A warp is on its own: it copies its tiles (cp.async.bulk, one or two
// 16-token groups each) into its ring, waits, computes and refills, with no CTA barrier, and
// carries (m, l, O) in registers.  Lengths are read on the device, so the split is even
// whatever they are.  A unit that one warp covers is written straight to O; parts are merged
// at the CTA's end in shared memory, and units that cross CTAs by the last CTA to arrive
// (at most two parts per CTA in the workspace, merged in CTA order: results do not depend on
// timing).
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
    static constexpr int W = D == 256 ? 8 : NT == 1 ? (D == 64 ? 16 : 12) : (D == 64 ? 12 : 8);   // warps
    static constexpr int STAGES = D == 256 ? 2 : D == 64 ? 4 : NT == 1 ? 3 : 4;
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
    static_assert(STAGES * STAGE_BYTES >= PART_FLOATS * 4, "a warp's last part is kept in its ring");
    static_assert(SMEM_BYTES <= 225 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
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
    int b, hr, tile, nt, len;
};

template <int D, int NT>
struct Q4Warp {                    // a warp's running state of one unit
    float o[NT][Q4AttnCfg<D, NT>::MT][4];
    float m[NT][2], ms[NT][2], l[NT][2];       // ms: m, or 0 while m is -inf
    uint32_t q[NT][Q4AttnCfg<D, NT>::KW][4];
    float cq[NT][2];               // a column's factor of the scores
    int lim[NT][2];                // keys the column's query sees
    uint32_t tmax;                 // bits of the largest value scale seen
    float tnorm, tinv;             // 2^13 / 2^exponent(tmax), and its inverse
};

__device__ __forceinline__ int q4_len(const Q4AttnParams& p, int b) {
    const int cap = p.max_blocks << p.bs_log2;
    const int n = p.lens[b];
    return n < 0 ? 0 : n > cap ? cap : n;
}
// Tiles of a sequence: an empty one keeps one (masked) tile, whose unit writes the zeros.
__device__ __forceinline__ int q4_tiles(int len) { return len <= 32 ? 1 : (len + 31) >> 5; }

__device__ __forceinline__ void q4_advance(const Q4AttnParams& p, Q4Cursor& c, int HR) {
    if (++c.tile < c.nt) return;
    c.tile = 0;
    if (++c.hr < HR) return;
    c.hr = 0;
    if (++c.b < p.B) {
        c.len = q4_len(p, c.b);
        c.nt = q4_tiles(c.len);
    }
}

// Unit start: queries to MMA operands (B fragments: column = query g, k = dims of lane t).
template <int D, int NT>
__device__ __forceinline__ void q4_begin(const Q4AttnParams& p, Q4Warp<D, NT>& s, const Q4Cursor& c, int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int g = lane >> 2, t = lane & 3;
    const int h = c.hr / p.n_rg, row0 = (c.hr % p.n_rg) * C::ROWS;
    const size_t qbase = (static_cast<size_t>(c.b) * p.H_kv + h) * p.R;
    s.tmax = 0u;
    s.tnorm = s.tinv = 1.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + 8 * n + g;
        float x[C::KW][8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < C::KW; ++i) {
            const int chunk = D == 64 ? 2 * t + i : (i >> 2) * 16 + 4 * t + (i & 3);
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < p.R) v = reinterpret_cast<const uint4*>(p.Q + (qbase + r) * D)[chunk];
            if (p.q_bf16) unpack8<true>(v, x[i]);
            else unpack8<false>(v, x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[i][e]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int ex = static_cast<int>(__float_as_uint(mx) >> 23);            // biased exponent of the row's maximum
        ex = ex < 14 ? 14 : ex;
        const float f = __uint_as_float(static_cast<uint32_t>(267 - ex) << 23);   // 2^13 / 2^(ex - 127)
#pragma unroll
        for (int i = 0; i < C::KW; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s.q[n][i][e] = pack_half2(x[i][e] * f, x[i][e + 4] * f);
        }
        const float cq = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(ex - 13) << 23) * 0x1p9f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            s.cq[n][k] = __shfl_sync(0xffffffffu, cq, 4 * (2 * t + k));
            const int i = (row0 + 8 * n + 2 * t + k) % p.S_q;
            s.lim[n][k] = c.len - (p.causal ? p.S_q - 1 - i : 0);
            s.m[n][k] = -INFINITY;
            s.ms[n][k] = 0.f;
            s.l[n][k] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s.o[n][i][e] = 0.f;
    }
}

// One tile of 32 keys from shared memory.  valid: bit j set when group j was copied.
template <int D, int NT>
__device__ __forceinline__ void q4_tile(const Q4AttnParams& p, Q4Warp<D, NT>& s, const uint8_t* st, int key0, int len,
                                        uint32_t valid, bool masked, int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int g = lane >> 2, t = lane & 3;
    float x[2][NT][4], mx[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) mx[n][0] = mx[n][1] = -INFINITY;
    // S^T = K Q^T.  Every word of 8 dims has its own accumulator (the chains of two MMAs do not
    // wait on one another), added up in fp32.
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint8_t* gr = st + j * C::GROUP;
        constexpr int NW = D == 64 ? 2 : 4;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(gr + Q4<D>::K_WORDS);
        const uint32_t wk[2] = {words[g], words[g + 8]};
        const uint32_t za = q4_negz((wk[0] & 15u) * 0x00010001u), zb = q4_negz((wk[1] & 15u) * 0x00010001u);
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
            float acc[NW][NT][4];
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int w = hf * 4 + i;
                const uint32_t ua = wa[i] >> 8, ub = wb[i] >> 8;
                const uint32_t a0 = q4_lo(wa[i], za), a1 = q4_lo(wb[i], zb), a2 = q4_hi(wa[i], za), a3 = q4_hi(wb[i], zb);
                const uint32_t c0 = q4_lo(ua, za), c1 = q4_lo(ub, zb), c2 = q4_hi(ua, za), c3 = q4_hi(ub, zb);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.f;
                    mma_16816(acc[i][n], a0, a1, a2, a3, s.q[n][w][0], s.q[n][w][1]);
                    mma_16816(acc[i][n], c0, c1, c2, c3, s.q[n][w][2], s.q[n][w][3]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = acc[0][n][e] + acc[1][n][e];
                    if constexpr (NW == 4) v += acc[2][n][e] + acc[3][n][e];
                    x[j][n][e] = hf == 0 ? v : x[j][n][e] + v;
                }
        }
        // Scores, masks and the tile's maxima (rows g and g + 8; columns 2t, 2t + 1).
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float sc = q4_scale(wk[h]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float v = x[j][n][2 * h + k] * (sc * s.cq[n][k]);
                    if (masked) {
                        if (!((valid >> j) & 1u)) v = 0.f;               // a page outside the pool reads zeros
                        if (key0 + 16 * j + 8 * h + g >= s.lim[n][k]) v = -INFINITY;
                    }
                    x[j][n][2 * h + k] = v;
                    mx[n][k] = fmaxf(mx[n][k], v);
                }
        }
    }
    // The largest value scale so far sets the fp16 range of p t.
    {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(st + (lane >> 4) * C::GROUP + Q4<D>::V_WORDS);
        uint32_t u = words[lane & 15] & 0xFFFFFF00u;
        if (u >= 0x7F800000u) u = 0u;                                    // a spoiled row sets no range
        if (masked && (!((valid >> (lane >> 4)) & 1u) || key0 + lane >= len)) u = 0u;
        u = __reduce_max_sync(0xffffffffu, u);
        if (u > s.tmax) {
            s.tmax = u;
            int ex = static_cast<int>(u >> 23);
            ex = ex < 27 ? 27 : ex;                                      // scales are 0 or at least 2^-100
            const float norm = __uint_as_float(static_cast<uint32_t>(267 - ex) << 23);
            const float r = norm * s.tinv;
            s.tnorm = norm;
            s.tinv = __uint_as_float(static_cast<uint32_t>(ex - 13) << 23);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < C::MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s.o[n][i][e] *= r;
        }
    }
    bool grew = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mx[n][k] = fmaxf(mx[n][k], __shfl_xor_sync(0xffffffffu, mx[n][k], 4));
            mx[n][k] = fmaxf(mx[n][k], __shfl_xor_sync(0xffffffffu, mx[n][k], 8));
            mx[n][k] = fmaxf(mx[n][k], __shfl_xor_sync(0xffffffffu, mx[n][k], 16));
            grew = grew || mx[n][k] > s.m[n][k];
        }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float m = fmaxf(s.m[n][k], mx[n][k]);
                const float ms = m == -INFINITY ? 0.f : m;
                const float a = ex2_approx(s.m[n][k] - ms);
                s.m[n][k] = m;
                s.ms[n][k] = ms;
                s.l[n][k] *= a;
#pragma unroll
                for (int i = 0; i < C::MT; ++i) {
                    s.o[n][i][k] *= a;
                    s.o[n][i][2 + k] *= a;
                }
            }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint8_t* gr = st + j * C::GROUP;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(gr + Q4<D>::V_WORDS);
        uint32_t pb[NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float tv = q4_scale(words[g + 8 * h]) * s.tnorm;
            if (masked && (!((valid >> j) & 1u) || key0 + 16 * j + 8 * h + g >= len)) tv = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float pt[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float pr = ex2_approx(x[j][n][2 * h + k] - s.ms[n][k]);
                    s.l[n][k] += pr;
                    pt[k] = pr * tv;
                    if (masked && key0 + 16 * j + 8 * h + g >= s.lim[n][k]) pt[k] = 0.f;   // 0 * a spoiled row's NaN
                }
                pb[n][h] = movmatrix_trans(pack_half2(pt[0], pt[1]));
            }
        }
        const uint2 z01 = *reinterpret_cast<const uint2*>(words + 2 * t);
        const uint2 z89 = *reinterpret_cast<const uint2*>(words + 8 + 2 * t);
        const uint32_t za = q4_negz((z01.x & 15u) | ((z01.y & 15u) << 16)), zb = q4_negz((z89.x & 15u) | ((z89.y & 15u) << 16));
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
                for (int n = 0; n < NT; ++n) mma_16816(s.o[n][i], a0[i], a1[i], a2[i], a3[i], pb[n][0], pb[n][1]);
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
                        for (int n = 0; n < NT; ++n)
                            mma_16816(s.o[n][set * 8 + q * 4 + i], a0[i], a1[i], a2[i], a3[i], pb[n][0], pb[n][1]);
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
__device__ __forceinline__ void q4_emit(const Q4AttnParams& p, Q4Warp<D, NT>& s, int u, bool whole, float* part, int lane) {
    using C = Q4AttnCfg<D, NT>;
    const int g = lane >> 2, t = lane & 3;
    const int row0 = (u % p.n_rg) * C::ROWS;
    const size_t rbase = static_cast<size_t>(u / p.n_rg) * p.R;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float l = s.l[n][k];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int col = 8 * n + 2 * t + k, r = row0 + col;
            // 2^9 first: with the scales' power in one factor it could leave fp32's range
            const float f = whole ? s.tinv * (l == 0.f ? 0.f : 1.0f / l) : s.tinv;
#pragma unroll
            for (int set = 0; set < C::SETS; ++set)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int v = 0; v < C::V4; ++v) {
                        float y[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            y[i] = s.o[n][set * 8 + 4 * v + i][2 * h + k] * 0x1p9f * f;
                        const float4 y4 = make_float4(y[0], y[1], y[2], y[3]);
                        const int e = 2 * h + k;
                        if (!whole)
                            reinterpret_cast<float4*>(part)[(((n * C::SETS + set) * 4 + e) * C::V4 + v) * 32 + lane] = y4;
                        else if (r < p.R)
                            store_out4(p.O, (rbase + r) * D + q4_dim<D>(set, e, v, g), y4, p.out_type);
                    }
            if (g == 0) {
                if (!whole) {
                    part[C::O_FLOATS + col] = s.m[n][k];
                    part[C::O_FLOATS + C::ROWS + col] = l;
                } else if (r < p.R) {
                    if (p.Mi) p.Mi[rbase + r] = s.m[n][k] * 0.6931471805599453f;
                    if (p.Li) p.Li[rbase + r] = l;
                }
            }
        }
}

__device__ __forceinline__ float q4_weight(float m, float M) { return m == -INFINITY ? 0.f : ex2_approx(m - M); }

template <int D, int NT>
__global__ void __launch_bounds__(Q4AttnCfg<D, NT>::THREADS, 1) q4_attn_kernel(const __grid_constant__ Q4AttnParams p) {
    using C = Q4AttnCfg<D, NT>;
    constexpr int W = C::W, STAGES = C::STAGES;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[W][STAGES];
    __shared__ int s_abort, s_drop[W], s_last[2];
    __shared__ int s_sum[W];
    __shared__ int s_b[W], s_base[W];
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
    grid_dep_launch_dependents();
    grid_dep_wait();

    // ---- the row of tiles: totals, this CTA's share, each warp's first sequence
    const int HR = p.H_kv * p.n_rg;
    const int per = (p.B + C::THREADS - 1) / C::THREADS;
    const int b0 = tid * per < p.B ? tid * per : p.B, b1 = b0 + per < p.B ? b0 + per : p.B;
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += q4_tiles(q4_len(p, b));
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int total = 0, before = incl - mine;
    for (int w = 0; w < W; ++w) {
        before += w < warp ? s_sum[w] : 0;
        total += s_sum[w];
    }
    const long long T = static_cast<long long>(total) * HR;
    // CTAs that take part: every warp of theirs gets at least a tile.
    long long act = (T + W - 1) / W;
    if (act > gridDim.x) act = gridDim.x;
    if (blockIdx.x >= act) return;
    const long long x0 = blockIdx.x * T / act, x1 = (blockIdx.x + 1) * T / act;
    if (mine > 0) {
        const long long lo = static_cast<long long>(before) * HR, hi = lo + static_cast<long long>(mine) * HR;
        for (int w = 0; w < W; ++w) {
            const long long y = x0 + w * (x1 - x0) / W;
            if (y >= lo && y < hi) {
                long long at = lo;
                int b = b0;
                for (; b < b1 - 1; ++b) {
                    const long long next = at + static_cast<long long>(q4_tiles(q4_len(p, b))) * HR;
                    if (y < next) break;
                    at = next;
                }
                s_b[w] = b;
                s_base[w] = static_cast<int>(at);
            }
        }
    }
    __syncthreads();

    const int y0 = static_cast<int>(x0 + warp * (x1 - x0) / W), y1 = static_cast<int>(x0 + (warp + 1) * (x1 - x0) / W);
    if (y0 < y1) {
        Q4Cursor cur;
        cur.b = s_b[warp];
        cur.len = q4_len(p, cur.b);
        cur.nt = q4_tiles(cur.len);
        cur.hr = (y0 - s_base[warp]) / cur.nt;
        cur.tile = (y0 - s_base[warp]) % cur.nt;
        Q4Cursor pre = cur;                                              // next tile to copy
        int win = -1, win_b = -1, win_p = 0;                             // 32 table entries, one per lane
        uint32_t vbits = 0;                                              // 2 validity bits per stage
        const size_t page_bytes = static_cast<size_t>(C::GROUP) << (p.bs_log2 - 4);

        auto copy = [&](int stage) {
            const int key0 = pre.tile * 32, rem = pre.len - key0;
            const int ng = rem <= 0 ? 0 : rem <= 16 ? 1 : 2;
            const int p0 = key0 >> p.bs_log2, p1 = p.bs_log2 == 4 && ng == 2 ? p0 + 1 : p0;
            if (ng && (pre.b != win_b || p0 < win_p || p1 >= win_p + 32)) {
                win_b = pre.b;
                win_p = p0;
                const int used = (pre.len + (1 << p.bs_log2) - 1) >> p.bs_log2;
                win = p0 + lane < used ? p.table[static_cast<size_t>(pre.b) * p.max_blocks + p0 + lane] : -1;
            }
            const int e0 = __shfl_sync(0xffffffffu, win, (p0 - win_p) & 31);
            const int e1 = __shfl_sync(0xffffffffu, win, (p1 - win_p) & 31);
            const bool v0 = ng >= 1 && static_cast<unsigned>(e0) < static_cast<unsigned>(p.n_blocks);
            const bool v1 = ng == 2 && static_cast<unsigned>(e1) < static_cast<unsigned>(p.n_blocks);
            vbits = (vbits & ~(3u << (2 * stage))) | ((v0 ? 1u : 0u) | (v1 ? 2u : 0u)) << (2 * stage);
            uint64_t* bar = &bars[warp][stage];
            uint8_t* dst = ring + stage * C::STAGE_BYTES;
            if (lane == 0) mbar_arrive_expect_tx(bar, ((v0 ? 1u : 0u) + (v1 ? 1u : 0u)) * C::GROUP);
            __syncwarp();
            const int h = pre.hr / p.n_rg;
            if (p.bs_log2 == 4) {                                        // a group is a page: two copies
                if (lane == 0 ? v0 : lane == 1 && v1)
                    bulk_g2s(dst + lane * C::GROUP,
                             p.cache + (static_cast<size_t>(lane ? e1 : e0) * p.H_kv + h) * page_bytes, C::GROUP, bar);
            } else if (lane == 0 && v0) {                                // both groups lie in one page
                const int gr = (key0 & ((1 << p.bs_log2) - 1)) >> 4;
                bulk_g2s(dst, p.cache + (static_cast<size_t>(e0) * p.H_kv + h) * page_bytes + static_cast<size_t>(gr) * C::GROUP,
                         ng * C::GROUP, bar);
            }
            q4_advance(p, pre, HR);
        };

        int issued = y0;
        for (int i = 0; i < STAGES && issued < y1; ++i, ++issued) copy(i);
        Q4Warp<D, NT> s;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true, fresh = true;
        int first = 0;
        for (int y = y0; y < y1; ++y) {
            if (fresh) {
                q4_begin<D, NT>(p, s, cur, lane);
                first = cur.tile;
                fresh = false;
            }
            if (ok) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars[warp][stage], phase, &s_abort, p.timeout_ns));
                if (ok) {
                    const uint32_t valid = (vbits >> (2 * stage)) & 3u;
                    const int key0 = cur.tile * 32;
                    const bool masked = valid != 3u || key0 + 32 > cur.len - (p.causal ? p.S_q - 1 : 0);
                    q4_tile<D, NT>(p, s, ring + stage * C::STAGE_BYTES, key0, cur.len, valid, masked, lane);
                    __syncwarp();
                    if (issued < y1) {
                        copy(stage);
                        ++issued;
                    }
                } else {
                    // The copies in flight still land in this ring: wait for them (bounded) before leaving it.
                    if (lane == 0) atomicOr(&g_kf_dev_error, KF_DEVERR_TIMEOUT_TMA);
                    for (int z = y, sz = stage, pz = phase; z < issued; ++z) {
                        s_drop[warp] = 0;
                        __syncwarp();
                        mbar_wait_bounded(&bars[warp][sz], pz, &s_drop[warp], p.timeout_ns);
                        __syncwarp();
                        if (++sz == STAGES) { sz = 0; pz ^= 1; }
                    }
                }
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            const bool unit_end = cur.tile == cur.nt - 1, last = y == y1 - 1;
            if (unit_end || last) {
                const bool whole = unit_end && first == 0;
                const int u = cur.b * HR + cur.hr;
                // A part that ends inside the warp's share goes to the warp's head slot, the last one to its ring.
                float* part = last ? reinterpret_cast<float*>(ring) : heads + warp * C::PART_FLOATS;
                __syncwarp();
                q4_emit<D, NT>(p, s, u, whole, part, lane);
                if (!whole && lane == 0) s_ent[2 * warp + (last ? 1 : 0)] = Q4Unit{u, y - cur.tile, cur.nt};
                fresh = true;
            }
            q4_advance(p, cur, HR);
        }
    }
    __syncthreads();

    // ---- merge the CTA's parts: runs of equal units in the entries' order
    const int n4 = NT * C::SETS * 4 * C::V4;
    Q4Unit mine_u = lane < 2 * W ? s_ent[lane] : Q4Unit{-1, 0, 0};
    uint32_t todo = __ballot_sync(0xffffffffu, mine_u.u >= 0);
    int cross_u[2] = {-1, -1}, cross_first[2] = {0, 0}, cross_n[2] = {0, 0};
    while (todo) {
        const int lead = __ffs(todo) - 1;
        const int u = __shfl_sync(0xffffffffu, mine_u.u, lead);
        const int us = __shfl_sync(0xffffffffu, mine_u.start, lead), unt = __shfl_sync(0xffffffffu, mine_u.nt, lead);
        const uint32_t run = __ballot_sync(0xffffffffu, mine_u.u == u);
        todo &= ~run;
        const bool inside = us >= x0 && us + unt <= x1;
        const int slot = us >= x0 ? 1 : 0;
        float* out = p.parts + (static_cast<size_t>(blockIdx.x) * 2 + slot) * C::PART_FLOATS;
        const int row0 = (u % p.n_rg) * C::ROWS;
        const size_t rbase = static_cast<size_t>(u / p.n_rg) * p.R;
        for (int idx = tid; idx < n4 * 32; idx += C::THREADS) {
            const int ln = idx & 31, q4 = idx >> 5, v = q4 % C::V4, item = q4 / C::V4;
            const int e = item & 3, set = (item >> 2) % C::SETS, n = item / (4 * C::SETS);
            const int col = 8 * n + 2 * (ln & 3) + (e & 1), r = row0 + col;
            auto entry = [&](int i) {
                return i & 1 ? reinterpret_cast<const float*>(smem + (i >> 1) * STAGES * C::STAGE_BYTES)
                             : heads + (i >> 1) * C::PART_FLOATS;
            };
            float M = -INFINITY, L = 0.f;
            for (uint32_t b = run; b; b &= b - 1) M = fmaxf(M, entry(__ffs(b) - 1)[C::O_FLOATS + col]);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t b = run; b; b &= b - 1) {
                const float* part = entry(__ffs(b) - 1);
                const float w = q4_weight(part[C::O_FLOATS + col], M);
                const float4 y = reinterpret_cast<const float4*>(part)[q4 * 32 + ln];
                L = fmaf(w, part[C::O_FLOATS + C::ROWS + col], L);
                a.x = fmaf(w, y.x, a.x); a.y = fmaf(w, y.y, a.y); a.z = fmaf(w, y.z, a.z); a.w = fmaf(w, y.w, a.w);
            }
            const bool stats = (ln >> 2) == 0 && set == 0 && v == 0 && (e >> 1) == 0;
            if (inside) {
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                if (r < p.R) {
                    store_out4(p.O, (rbase + r) * D + q4_dim<D>(set, e, v, ln >> 2),
                               make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv), p.out_type);
                    if (stats && p.Mi) p.Mi[rbase + r] = M * 0.6931471805599453f;
                    if (stats && p.Li) p.Li[rbase + r] = L;
                }
            } else {
                reinterpret_cast<float4*>(out)[q4 * 32 + ln] = a;
                if (stats) {
                    out[C::O_FLOATS + col] = M;
                    out[C::O_FLOATS + C::ROWS + col] = L;
                }
            }
        }
        if (!inside) {
            // CTA of tile x: the largest c with floor(c T / act) <= x.
            const int cf = static_cast<int>(((us + 1ll) * act - 1) / T);
            const int cl = static_cast<int>((static_cast<long long>(us + unt) * act - 1) / T);
            cross_u[slot] = u;
            cross_first[slot] = cf;
            cross_n[slot] = cl - cf + 1;
        }
    }
    if (cross_u[0] < 0 && cross_u[1] < 0) return;

    // ---- units that cross CTAs: the last CTA to arrive merges the parts, in CTA order
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        for (int k = 0; k < 2; ++k) {
            s_last[k] = 0;
            if (cross_u[k] >= 0 &&
                atom_add_acq_rel_gpu(p.tickets + cross_first[k], 1u) == static_cast<unsigned>(cross_n[k] - 1)) {
                p.tickets[cross_first[k]] = 0u;
                s_last[k] = 1;
            }
        }
    }
    __syncthreads();
    float* wm = reinterpret_cast<float*>(smem);                          // [parts][ROWS] m, then weights; [parts][ROWS] l; totals
    for (int k = 0; k < 2; ++k) {
        if (!s_last[k]) continue;
        const int nparts = cross_n[k], cf = cross_first[k], u = cross_u[k];
        float* wl = wm + nparts * C::ROWS;
        float* tot = wl + nparts * C::ROWS;                              // M, L per column
        auto part = [&](int i) { return p.parts + (static_cast<size_t>(cf + i) * 2 + (i == 0 ? 1 : 0)) * C::PART_FLOATS; };
        __syncthreads();
        for (int i = tid; i < nparts * C::ROWS; i += C::THREADS) {
            const float* src = part(i / C::ROWS) + C::O_FLOATS + i % C::ROWS;
            wm[i] = __ldcg(src);
            wl[i] = __ldcg(src + C::ROWS);
        }
        __syncthreads();
        for (int col = warp; col < C::ROWS; col += W) {
            float M = -INFINITY, L = 0.f;
            for (int i = lane; i < nparts; i += 32) M = fmaxf(M, wm[i * C::ROWS + col]);
            for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            for (int i = lane; i < nparts; i += 32) {
                const float w = q4_weight(wm[i * C::ROWS + col], M);
                wm[i * C::ROWS + col] = w;
                L = fmaf(w, wl[i * C::ROWS + col], L);
            }
            for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
            if (lane == 0) {
                tot[2 * col] = M;
                tot[2 * col + 1] = L;
            }
        }
        __syncthreads();
        const int row0 = (u % p.n_rg) * C::ROWS;
        const size_t rbase = static_cast<size_t>(u / p.n_rg) * p.R;
        for (int idx = tid; idx < n4 * 32; idx += C::THREADS) {
            const int ln = idx & 31, q4 = idx >> 5, v = q4 % C::V4, item = q4 / C::V4;
            const int e = item & 3, set = (item >> 2) % C::SETS, n = item / (4 * C::SETS);
            const int col = 8 * n + 2 * (ln & 3) + (e & 1), r = row0 + col;
            if (r >= p.R) continue;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int i = 0; i < nparts; ++i) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(part(i)) + q4 * 32 + ln);
                const float w = wm[i * C::ROWS + col];
                a.x = fmaf(w, y.x, a.x); a.y = fmaf(w, y.y, a.y); a.z = fmaf(w, y.z, a.z); a.w = fmaf(w, y.w, a.w);
            }
            const float L = tot[2 * col + 1], inv = L == 0.f ? 0.f : 1.0f / L;
            store_out4(p.O, (rbase + r) * D + q4_dim<D>(set, e, v, ln >> 2),
                       make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv), p.out_type);
            if ((ln >> 2) == 0 && set == 0 && v == 0 && (e >> 1) == 0) {
                if (p.Mi) p.Mi[rbase + r] = tot[2 * col] * 0.6931471805599453f;
                if (p.Li) p.Li[rbase + r] = L;
            }
        }
    }
}

}  // namespace kf
