// RMSNorm, rotary position embedding (RoPE) and SwiGLU for B200 (sm_100a).
//
// The reference lists these three kernels as planned with no code
// (README.md:16-18), so the arithmetic follows the Llama-family convention
// used by transformers' Llama modules:
//   rmsnorm : y = rnd(rnd(x * r) * w),  r = 1 / sqrt(mean(x^2) + eps)
//             (fused residual form: s = rnd(x + res) is written back to res
//             and normalised in place of x)
//   rope    : pairs (x0, x1) -> (x0 c - x1 s, x1 c + x0 s), c/s of
//             pos * theta^(-2i/rot_dim); NeoX pairing (i, i + rot_dim/2) or
//             GPT-J pairing (2i, 2i+1); one rounding at the end
//   swiglu  : y = rnd(rnd(silu(g)) * u),  silu(g) = g / (1 + e^-g)
// where rnd() rounds to the 16-bit storage type (fp16 or bf16).  Arithmetic is
// fp32 except the RoPE angle, which is formed and reduced modulo 2*pi in fp64
// so that positions up to 2^31 keep the fp32 accuracy of sincosf.
//
// The query/key norm with the rotation (qk_norm_rope) rounds once, at the end.
//
// All are HBM-streaming kernels: 16-byte vector loads and stores,
// inputs read once with the evict-first hint, grids sized from the occupancy
// of the 148 SMs.  Nothing here is GEMM-shaped, so no tensor-core path.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "kf_ptx.cuh"

namespace kf {

// ---- 8 x 16-bit <-> 8 x fp32 -------------------------------------------------
template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4 v, float (&f)[8]) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 p;
        if constexpr (BF16) {
            __nv_bfloat162 h;
            *reinterpret_cast<unsigned*>(&h) = w[i];
            p = __bfloat1622float2(h);
        } else {
            __half2 h;
            *reinterpret_cast<unsigned*>(&h) = w[i];
            p = __half22float2(h);
        }
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

template <bool BF16>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    unsigned u;
    if constexpr (BF16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        u = *reinterpret_cast<unsigned*>(&h);
    } else {
        __half2 h = __floats2half2_rn(a, b);
        u = *reinterpret_cast<unsigned*>(&h);
    }
    return u;
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]),
                      pack2<BF16>(f[6], f[7]));
}

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t u) {
    if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
    return __half2float(__ushort_as_half(u));
}
template <bool BF16>
__device__ __forceinline__ uint16_t from_f32(float x) {
    if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
    return __half_as_ushort(__float2half_rn(x));
}

// Rounds 8 fp32 values to the storage type and back.
template <bool BF16>
__device__ __forceinline__ void round8(float (&f)[8]) {
    unpack8<BF16>(pack8<BF16>(f), f);
}

__device__ __forceinline__ uint4 ld_stream(const uint4* p) { return __ldcs(p); }
__device__ __forceinline__ void st_stream(uint4* p, uint4 v) { __stcs(p, v); }

// ---- RMSNorm -------------------------------------------------------------------
// One row of `hidden` = 8 * nvec elements is owned by a group of G threads
// (G a power of two, 1..1024); thread r of the group holds vectors
// r, r + G, ..., r + (VPT-1) G (VPT <= 4) in registers between the sum of
// squares and the scaling pass, so every input byte is read from HBM once.
// All of a row's loads (x, and the residual) are issued before its first
// store.  Blocks hold max(G, 256) / G row groups and stride over the rows.
struct RmsNormParams {
    const uint4* x;        // [rows, nvec] input
    const uint4* w;        // [nvec] weight
    uint4* out;            // [rows, nvec] output (may equal x)
    uint4* res;            // [rows, nvec] residual, updated in place (RES only)
    long long rows;
    int nvec;
    int G;                 // threads per row
    float inv_hidden;
    float eps;
};

template <bool BF16, int VPT, bool RES>
__global__ void __launch_bounds__(1024) rmsnorm_kernel(const RmsNormParams p) {
    __shared__ float red[32];
    const int G = p.G;
    const int r = threadIdx.x & (G - 1);
    const int gi = threadIdx.x / G;
    const int rpb = blockDim.x / G;                      // rows per block pass
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    for (long long base = static_cast<long long>(blockIdx.x) * rpb; base < p.rows;
         base += static_cast<long long>(gridDim.x) * rpb) {
        const long long row = base + gi;
        const bool valid = row < p.rows;
        const long long off = row * p.nvec;
        uint4 v[VPT], rv[VPT];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = r + k * G;
            const bool in = valid && c < p.nvec;
            v[k] = in ? ld_stream(p.x + off + c) : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (RES) rv[k] = in ? ld_stream(p.res + off + c) : make_uint4(0u, 0u, 0u, 0u);
        }
        if constexpr (RES) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = r + k * G;
                float a[8], b[8];
                unpack8<BF16>(v[k], a);
                unpack8<BF16>(rv[k], b);
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] += b[e];
                v[k] = pack8<BF16>(a);                   // rnd(x + res): exact sum, one rounding
                if (valid && c < p.nvec) st_stream(p.res + off + c, v[k]);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float a[8];
            unpack8<BF16>(v[k], a);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], ss);
        }
        // Sum over the row's G threads: shuffles inside a warp, then shared
        // memory across the row's warps (G > 32 only).
        const int wspan = G < 32 ? G : 32;
        for (int o = wspan >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (G > 32) {
            if (lane == 0) red[warp] = ss;
            __syncthreads();
            const int nw = G >> 5;
            const int w0 = (warp / nw) * nw;
            ss = 0.f;
            for (int j = 0; j < nw; ++j) ss += red[w0 + j];
            __syncthreads();
        }
        const float rinv = rsqrtf(fmaf(ss, p.inv_hidden, p.eps));
        if (valid) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = r + k * G;
                if (c < p.nvec) {
                    float a[8], wt[8];
                    unpack8<BF16>(v[k], a);
                    unpack8<BF16>(__ldg(p.w + c), wt);
#pragma unroll
                    for (int e = 0; e < 8; ++e) a[e] *= rinv;
                    round8<BF16>(a);                     // rnd(x * r)
#pragma unroll
                    for (int e = 0; e < 8; ++e) a[e] *= wt[e];   // exact in fp32; rounded once by pack8
                    st_stream(p.out + off + c, pack8<BF16>(a));
                }
            }
        }
    }
}

// ---- RoPE ----------------------------------------------------------------------
// In place on Q and K given by element strides (head_dim contiguous), so both
// [B, H, S, D] (the attention layout) and [B, S, H, D] work.  A "unit" is what
// one thread rotates per head row: NeoX, 8 pairs = the 16-byte vector at
// dims 8u.. and its partner at rot_dim/2 + 8u..; GPT-J, 4 pairs in one 16-byte
// vector at dims 8u...  Thread (u, hg, tk) of a block owns unit u of the HB
// heads hg, hg + HG, ... (HG * HB >= H_q + H_kv) of one token per pass: it
// issues all of that token's loads first, then computes the 4 or 8 angles
// once for all those heads, then rotates and stores.  The inverse
// frequencies sit in shared memory (fp64, computed once per block).
struct RopeParams {
    uint4* q;
    uint4* k;                     // nullptr when H_kv == 0
    const int* pos;               // [B, S] positions, nullptr: position = s
    const float* inv_freq;        // [rot_dim / 2], nullptr: theta^(-2i/rot_dim)
    long long q_sb, q_sh, q_ss;   // strides in 16-byte vectors
    long long k_sb, k_sh, k_ss;
    long long n_tokens;           // B * S
    int S, H_q, H_kv;
    int rot_dim;
    int U, HG, TPB;               // units per row, head groups, tokens per block pass
    double log2_theta;
};

// a mod 2*pi into [-pi, pi]: Cody-Waite reduction with 2*pi split into a
// 53-bit head and its remainder, exact for the |a| < 2^31 that int positions
// times inverse frequencies <= 1 produce.
__device__ __forceinline__ float reduce_2pi(double a) {
    const double k = rint(a * 0.15915494309189535);        // 1 / (2 pi)
    double r = fma(-k, 6.283185307179586, a);               // 2 pi, rounded to double
    r = fma(-k, 2.4492935982947064e-16, r);                 // 2 pi - its double rounding
    return static_cast<float>(r);
}

template <bool BF16, bool NEOX, int HB>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
    constexpr int NP = NEOX ? 8 : 4;                       // pairs per unit
    __shared__ double s_f[512];                            // inverse frequencies, rot_dim / 2 <= 512
    for (int i = threadIdx.x; i < p.rot_dim / 2; i += blockDim.x)
        s_f[i] = p.inv_freq ? static_cast<double>(p.inv_freq[i]) : exp2(-(2.0 * i / p.rot_dim) * p.log2_theta);
    __syncthreads();
    const int u = threadIdx.x % p.U;
    const int rest = threadIdx.x / p.U;
    const int hg = rest % p.HG;
    const int tk = rest / p.HG;
    if (tk >= p.TPB) return;
    const double* f = s_f + NP * u;
    const int H = p.H_q + p.H_kv;
    const long long half_vec = p.rot_dim / 16;             // NeoX partner offset, in vectors
    for (long long t = static_cast<long long>(blockIdx.x) * p.TPB + tk; t < p.n_tokens;
         t += static_cast<long long>(gridDim.x) * p.TPB) {
        const long long b = t / p.S;
        const long long s = t - b * p.S;
        const int pos_i = p.pos ? __ldg(p.pos + t) : static_cast<int>(s);
        for (int h0 = hg; h0 < H; h0 += HB * p.HG) {
            uint4* rowp[HB];
            uint4 a[HB], c[HB];
#pragma unroll
            for (int m = 0; m < HB; ++m) {
                const int h = h0 + m * p.HG;
                rowp[m] = nullptr;
                if (h < H) {
                    rowp[m] = h < p.H_q ? p.q + b * p.q_sb + h * p.q_sh + s * p.q_ss
                                        : p.k + b * p.k_sb + (h - p.H_q) * p.k_sh + s * p.k_ss;
                    a[m] = rowp[m][u];
                    if constexpr (NEOX) c[m] = rowp[m][half_vec + u];
                }
            }
            float cs[NP], sn[NP];
#pragma unroll
            for (int j = 0; j < NP; ++j) sincosf(reduce_2pi(static_cast<double>(pos_i) * f[j]), &sn[j], &cs[j]);
#pragma unroll
            for (int m = 0; m < HB; ++m) {
                if (!rowp[m]) continue;
                if constexpr (NEOX) {
                    float x0[8], x1[8], y0[8], y1[8];
                    unpack8<BF16>(a[m], x0);
                    unpack8<BF16>(c[m], x1);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        y0[e] = fmaf(x0[e], cs[e], -x1[e] * sn[e]);
                        y1[e] = fmaf(x1[e], cs[e], x0[e] * sn[e]);
                    }
                    rowp[m][u] = pack8<BF16>(y0);
                    rowp[m][half_vec + u] = pack8<BF16>(y1);
                } else {
                    float x[8], y[8];
                    unpack8<BF16>(a[m], x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[2 * e] = fmaf(x[2 * e], cs[e], -x[2 * e + 1] * sn[e]);
                        y[2 * e + 1] = fmaf(x[2 * e + 1], cs[e], x[2 * e] * sn[e]);
                    }
                    rowp[m][u] = pack8<BF16>(y);
                }
            }
        }
    }
}

// ---- Query/key norm with RoPE ---------------------------------------------------
// y = rnd(rot(x * rsqrt(mean(x^2) + eps) * w)) on every head row of Q and K.  Bound by HBM (each
// element read once, written once); the rotation's angles are the same for all heads, so a block
// takes groups of whole tokens: while a group's first rows are on their way it computes each pair's four
// coefficients (cos and sin times both weights, for queries and for keys; angles in half turns,
// reduced in fp64) into shared memory, and a row then costs one scaling and four packed FMAs a
// pair.  8192 tokens of 40 heads of 128 take 33.4 us (5.0 TB/s; 25.6 us are the bytes), at 14.5 instructions
// an element and 2.5 a clock.  (Weights in registers and cos / sin alone in the table took 23
// instructions, 46.5 us.)  A row belongs to
// GS = 2^k >= D / 16 threads with two 8-element vectors each, paired so that both halves of a NeoX
// rotation are in one thread: vectors (u, u + rot_dim / 16) rotate, the rest pass through as
// pairs with cos = 1; the sum of squares is reduced by shuffles.
struct QkNormRopeParams {
    const uint4* q;
    const uint4* k;
    uint4* qo;
    uint4* ko;
    const uint4* qw;              // [D / 8], nullptr: ones
    const uint4* kw;
    const int* pos;               // [B, S] positions, nullptr: position = s
    const float* inv_freq;        // [rot_dim / 2], nullptr: theta^(-2i/rot_dim)
    unsigned q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;         // strides in 16-byte vectors
    unsigned qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
    long long n_tokens;           // B * S
    int S, H_q, H_kv, D, rot_dim;
    int GS;                       // threads per row, a power of two
    int TPB;                      // tokens per group
    int splits, rows_per_split;   // parts of a group's rows, and their rows (a multiple of 256 / GS)
    int items;                    // groups * splits, strided over by the blocks
    float eps, rot_scale, inv_D;
    double log2_theta;
};

constexpr int kQkNormRopeTokens = 8;                       // the largest TPB
constexpr int kQkNormRopePairs = 1024;                     // TPB * D / 2 at most

template <bool BF16, bool NEOX>
__global__ void __launch_bounds__(256, 4) qk_norm_rope_kernel(const QkNormRopeParams p) {
    constexpr int UNR = 2;                                 // rows a thread has in flight (1: 37.2 us; 3, in three blocks an SM: 37.0)
    // Pairs 2e, 2e + 1 of thread u, token t, queries (0) or keys (1): (A, A', B, B') and (C, C', S, S')
    // at [kind][t][2e, 2e + 1][u]:  y0 = x0 A + x1 B,  y1 = x1 C + x0 S.
    __shared__ float4 s_c[2 * kQkNormRopePairs];
    // Pair j = eU + u of a row: half turns per position, and the weights (w0, w1) for queries and keys.
    __shared__ double s_f[256];
    __shared__ float4 s_w[256];
    // 16-byte indices of a token's first input and output vector, [token][queries or keys], and its
    // position, of this group and of the next
    __shared__ ulonglong2 s_at[2][2 * kQkNormRopeTokens];
    __shared__ int s_pos[2][kQkNormRopeTokens];
    const int tid = threadIdx.x, half = p.rot_dim >> 1, H = p.H_q + p.H_kv;
    auto tokens = [&](int item, int buf) {
        const unsigned t = (item / p.splits) * p.TPB + tid;
        if (tid >= p.TPB || t >= p.n_tokens) return;
        const unsigned b = t / p.S, s = t - b * p.S;
        auto at = [&](const uint4* x, unsigned sb, unsigned ss) {
            return (reinterpret_cast<unsigned long long>(x) >> 4) + static_cast<unsigned long long>(b) * sb +
                   static_cast<unsigned long long>(s) * ss;
        };
        s_at[buf][2 * tid] = make_ulonglong2(at(p.q, p.q_sb, p.q_ss), at(p.qo, p.qo_sb, p.qo_ss));
        s_at[buf][2 * tid + 1] = make_ulonglong2(at(p.k, p.k_sb, p.k_ss), at(p.ko, p.ko_sb, p.ko_ss));
        s_pos[buf][tid] = p.pos ? p.pos[t] : static_cast<int>(s);
    };
    tokens(blockIdx.x, 0);
    const int U = p.D >> 4, r = p.rot_dim >> 4;            // threads of a row that hold something; that rotate (NeoX)
    // The pair whose coefficients this thread makes, of tokens ct, ct + ct_step, ...
    const int ct = tid / (8 * U), ct_step = 256 / (8 * U), cj = tid - ct * 8 * U, ce = cj / U, cu = cj - ce * U;
    int i0, i1, pr;
    if (NEOX) {
        i0 = cu < r ? 8 * cu + ce : 16 * cu + ce;
        i1 = cu < r ? i0 + half : i0 + 8;
        pr = cu < r ? i0 : -1;
    } else {
        i0 = 8 * (ce < 4 ? cu : cu + U) + 2 * (ce & 3);
        i1 = i0 + 1;
        pr = i0 < p.rot_dim ? i0 >> 1 : -1;
    }
    const bool rotates = pr >= 0;
    if (ct == 0) {
        auto weight = [](const uint4* w, int i) { return w ? to_f32<BF16>(reinterpret_cast<const uint16_t*>(w)[i]) : 1.f; };
        s_w[cj] = make_float4(weight(p.qw, i0), weight(p.qw, i1), weight(p.kw, i0), weight(p.kw, i1));
        s_f[cj] = !rotates ? 0.0 : 0.3183098861837907 *
                  (p.inv_freq ? static_cast<double>(p.inv_freq[pr]) : exp2(-(2.0 * pr / p.rot_dim) * p.log2_theta));
    }
    __syncthreads();

    // row groups, this thread's, its place in the row; tokens and heads from one of its rows to the next
    const int RG = 256 / p.GS, rg = tid / p.GS, u = tid & (p.GS - 1), dt = RG / H, dh = RG - dt * H;
    const int c0 = !NEOX || u < r ? u : 2 * u, c1 = !NEOX ? u + U : u < r ? u + r : 2 * u + 1;   // its vectors
    const bool on = u < U;

    int buf = 0;
    for (int item = blockIdx.x; item < p.items; item += gridDim.x, buf ^= 1) {
        const int group = item / p.splits, split = item - group * p.splits;
        const int left = static_cast<int>(p.n_tokens) - group * p.TPB, n_tok = left < p.TPB ? left : p.TPB;
        const int end = min((split + 1) * p.rows_per_split, n_tok * H);
        int row = split * p.rows_per_split + rg;
        int tk = row / H, h = row - tk * H;
        bool first = true;
        for (; row - rg < end; row += UNR * RG) {                            // (the same trips for the whole block)
            uint4 v[UNR][2];
            uint4* out[UNR];
            int at[UNR];                                                     // the row's coefficients; -1: no row
#pragma unroll
            for (int i = 0; i < UNR; ++i) {
                at[i] = -1;
                v[i][0] = v[i][1] = make_uint4(0u, 0u, 0u, 0u);
                if (row + i * RG < end && on) {
                    const bool is_q = h < p.H_q;
                    const unsigned hh = is_q ? h : h - p.H_q;
                    const ulonglong2 base = s_at[buf][2 * tk + (is_q ? 0 : 1)];
                    const uint4* src = reinterpret_cast<const uint4*>(
                        (base.x + static_cast<unsigned long long>(hh) * (is_q ? p.q_sh : p.k_sh)) << 4);
                    out[i] = reinterpret_cast<uint4*>(
                        (base.y + static_cast<unsigned long long>(hh) * (is_q ? p.qo_sh : p.ko_sh)) << 4);
                    at[i] = ((is_q ? 0 : n_tok) + tk) * 8 * U + u;
                    v[i][0] = ld_stream(src + c0);
                    v[i][1] = ld_stream(src + c1);
                }
                h += dh;
                tk += dt;
                if (h >= H) {
                    h -= H;
                    ++tk;
                }
            }
            if (first) {                                                     // while the first rows are on their way
                first = false;
                const float4 wt = s_w[cj];
                const double f = s_f[cj];
                for (int t = ct < ct_step ? ct : n_tok; t < n_tok; t += ct_step) {
                    float sn = 0.f, cs = 1.f;
                    if (rotates) {
                        const double a = s_pos[buf][t] * f;
                        sincospif(static_cast<float>(a - 2.0 * rint(0.5 * a)), &sn, &cs);
                        sn *= p.rot_scale;
                        cs *= p.rot_scale;
                    }
#pragma unroll
                    for (int kind = 0; kind < 2; ++kind) {
                        const float w0 = kind ? wt.z : wt.x, w1 = kind ? wt.w : wt.y;
                        float* c = reinterpret_cast<float*>(s_c + ((kind * n_tok + t) * 8 + (ce & ~1)) * U + cu) + (ce & 1);
                        c[0] = w0 * cs;
                        c[2] = -w1 * sn;
                        c[4 * U] = w1 * cs;
                        c[4 * U + 2] = w0 * sn;
                    }
                }
                if (item + static_cast<int>(gridDim.x) < p.items) tokens(item + gridDim.x, buf ^ 1);
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < UNR; ++i) {
                float x[2][8];
                float2 ss = make_float2(0.f, 0.f);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    unpack8<BF16>(v[i][c], x[c]);
#pragma unroll
                    for (int e = 0; e < 8; e += 2) ss = ffma2(make_float2(x[c][e], x[c][e + 1]), make_float2(x[c][e], x[c][e + 1]), ss);
                }
                float sum = ss.x + ss.y;
                for (int o = p.GS >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (at[i] < 0) continue;
                const float rinv = rsqrtf(fmaf(sum, p.inv_D, p.eps));
                const float2 rr = make_float2(rinv, rinv);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float4 ab = s_c[at[i] + e * U], cd = s_c[at[i] + (e + 1) * U];
                    float* y[4];                                             // x0, x0', x1, x1' of the two pairs
                    y[0] = NEOX ? &x[0][e] : &x[e >> 2][2 * (e & 3)];
                    y[1] = NEOX ? &x[0][e + 1] : y[0] + 2;
                    y[2] = NEOX ? &x[1][e] : y[0] + 1;
                    y[3] = NEOX ? &x[1][e + 1] : y[0] + 3;
                    const float2 a = fmul2(make_float2(*y[0], *y[1]), rr), b = fmul2(make_float2(*y[2], *y[3]), rr);
                    const float2 o0 = ffma2(a, make_float2(ab.x, ab.y), fmul2(b, make_float2(ab.z, ab.w)));
                    const float2 o1 = ffma2(b, make_float2(cd.x, cd.y), fmul2(a, make_float2(cd.z, cd.w)));
                    *y[0] = o0.x; *y[1] = o0.y; *y[2] = o1.x; *y[3] = o1.y;
                }
                st_stream(out[i] + c0, pack8<BF16>(x[0]));
                st_stream(out[i] + c1, pack8<BF16>(x[1]));
            }
        }
        __syncthreads();                                                 // the coefficients are free
    }
}

// ---- SwiGLU --------------------------------------------------------------------
// gate_up [rows, 2 * inter] (gate columns first, then up) -> out [rows, inter].
// Blocks stride over rows; a block's threads stride over the row's vectors,
// UNR vectors per thread per pass with all 2 * UNR loads issued first.
// silu(g) = g / (1 + 2^(-g log2 e)) with the MUFU exponential and the fast
// (reciprocal-multiply) division, ~2^-21 relative error in fp32, far below
// the 16-bit rounding that follows.  The IEEE division made the kernel
// issue-bound (5.1 TB/s against 6.0).  For g < -87.3 the denominator leaves the
// fast division's range and the result is -0 (the true |silu| < 1e-36).
struct SwigluParams {
    const uint4* gu;
    uint4* out;
    long long rows;
    int ivec;                     // inter / 8
};

template <bool BF16>
__global__ void __launch_bounds__(256) swiglu_kernel(const SwigluParams p) {
    constexpr int UNR = 4;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const uint4* g = p.gu + row * 2 * p.ivec;
        const uint4* up = g + p.ivec;
        uint4* o = p.out + row * p.ivec;
        for (int c0 = threadIdx.x; c0 < p.ivec; c0 += UNR * blockDim.x) {
            uint4 gv[UNR], uv[UNR];
#pragma unroll
            for (int j = 0; j < UNR; ++j) {
                const int c = c0 + j * blockDim.x;
                if (c < p.ivec) {
                    gv[j] = ld_stream(g + c);
                    uv[j] = ld_stream(up + c);
                }
            }
#pragma unroll
            for (int j = 0; j < UNR; ++j) {
                const int c = c0 + j * blockDim.x;
                if (c >= p.ivec) break;
                float x[8], y[8];
                unpack8<BF16>(gv[j], x);
                unpack8<BF16>(uv[j], y);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __fdividef(x[e], 1.f + __expf(-x[e]));
                round8<BF16>(x);                           // rnd(silu(g))
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= y[e];  // exact in fp32; rounded once by pack8
                st_stream(o + c, pack8<BF16>(x));
            }
        }
    }
}

}  // namespace kf
