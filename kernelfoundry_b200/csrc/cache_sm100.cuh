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
// The zero point as a float: 2^23 + z is exact, so the subtraction leaves z.
__device__ __forceinline__ float q4_zero(uint32_t w) { return __uint_as_float(0x4B000000u | (w & 15u)) - 8388608.0f; }

// Parameter word of a row from its extremes (lo <= 0 <= hi) and the reciprocal scale.
__device__ __forceinline__ uint32_t q4_params(float lo, float hi, bool finite, float* inv, float* zp) {
    const float c = 1.0f / 15.0f;
    float s = __fsub_rn(__fmul_rn(hi, c), __fmul_rn(lo, c));
    s = __uint_as_float((__float_as_uint(s) + 0x80u) & 0xFFFFFF00u);
    if (!(s >= 7.888609052210118e-31f)) s = 0.0f;           // 2^-100: keeps 1/s finite
    *inv = s == 0.0f ? 0.0f : __frcp_rn(s);
    *zp = fminf(fmaxf(rintf(__fmul_rn(-lo, *inv)), 0.0f), 15.0f);
    if (!finite) {
        *inv = 0.0f;
        *zp = 0.0f;
        return kQ4BadRow;
    }
    return __float_as_uint(s) | static_cast<uint32_t>(*zp);
}

__device__ __forceinline__ uint32_t q4_code(float x, float inv, float zp) {
    return static_cast<uint32_t>(fminf(fmaxf(__fadd_rn(rintf(__fmul_rn(x, inv)), zp), 0.0f), 15.0f));
}

struct Q4IoParams {
    uint8_t* cache;
    const int* slots;             // [B, S]
    uint16_t* k;
    uint16_t* v;
    long long k_sb, k_sh, k_ss;   // element strides
    long long v_sb, v_sh, v_ss;
    int B, S, H;
    int bs_log2;                  // log2(block_size)
    long long n_slots;            // n_blocks * block_size
};

// Byte address of the group that holds `slot` of head h.
template <int D>
__device__ __forceinline__ uint8_t* q4_group(uint8_t* cache, long long slot, int h, int H, int bs_log2) {
    const long long block = slot >> bs_log2;
    const long long groups = 1ll << (bs_log2 - 4);
    return cache + ((block * H + h) * groups + ((slot >> 4) & (groups - 1))) * Q4<D>::GROUP;
}

// One warp per (token, head, K or V) row; a lane holds D / 32 neighbouring dims.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) q4_write_kernel(const Q4IoParams p) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const long long rows = 2ll * p.B * p.S * p.H;
    for (long long r = (blockIdx.x * 256ll + threadIdx.x) >> 5; r < rows; r += gridDim.x * 8ll) {
        const bool is_v = r & 1;
        const int h = static_cast<int>((r >> 1) % p.H);
        const long long tok = (r >> 1) / p.H;
        const long long slot = p.slots[tok];
        if (slot < 0 || slot >= p.n_slots) continue;
        const long long b = tok / p.S, s = tok % p.S;
        const uint16_t* src = is_v ? p.v + b * p.v_sb + h * p.v_sh + s * p.v_ss : p.k + b * p.k_sb + h * p.k_sh + s * p.k_ss;
        float x[N], lo = 0.f, hi = 0.f;
        bool fin = true;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = to_f32<BF16>(src[lane * N + i]);
            fin = fin && isfinite(x[i]);
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
        }
        for (int o = 16; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        fin = __all_sync(0xffffffffu, fin);
        float inv, zp;
        const uint32_t word = q4_params(lo, hi, fin, &inv, &zp);
        uint8_t* grp = q4_group<D>(p.cache, slot, h, p.H, p.bs_log2);
        uint8_t* dst = grp + (is_v ? Q4<D>::V_CODES : 0) + (slot & 15) * Q4<D>::ROW + lane * (N / 2);
#pragma unroll
        for (int i = 0; i < N; i += 2)
            dst[i / 2] = fin ? static_cast<uint8_t>(q4_code(x[i], inv, zp) | (q4_code(x[i + 1], inv, zp) << 4)) : 0;
        if (lane == 0)
            reinterpret_cast<uint32_t*>(grp + (is_v ? Q4<D>::V_WORDS : Q4<D>::K_WORDS))[slot & 15] = word;
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(256) q4_read_kernel(const Q4IoParams p) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const long long rows = 2ll * p.B * p.S * p.H;
    for (long long r = (blockIdx.x * 256ll + threadIdx.x) >> 5; r < rows; r += gridDim.x * 8ll) {
        const bool is_v = r & 1;
        const int h = static_cast<int>((r >> 1) % p.H);
        const long long tok = (r >> 1) / p.H;
        const long long slot = p.slots[tok];
        const long long b = tok / p.S, s = tok % p.S;
        uint16_t* dst = is_v ? p.v + b * p.v_sb + h * p.v_sh + s * p.v_ss : p.k + b * p.k_sb + h * p.k_sh + s * p.k_ss;
        float sc = 0.f, zp = 0.f;
        const uint8_t* src = nullptr;
        if (slot >= 0 && slot < p.n_slots) {
            const uint8_t* grp = q4_group<D>(p.cache, slot, h, p.H, p.bs_log2);
            const uint32_t w = reinterpret_cast<const uint32_t*>(grp + (is_v ? Q4<D>::V_WORDS : Q4<D>::K_WORDS))[slot & 15];
            sc = q4_scale(w);
            zp = q4_zero(w);
            src = grp + (is_v ? Q4<D>::V_CODES : 0) + (slot & 15) * Q4<D>::ROW + lane * (N / 2);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t n = src ? (src[i / 2] >> (4 * (i & 1))) & 15u : 0u;
            dst[lane * N + i] = from_f32<BF16>(sc * (static_cast<float>(n) - zp));
        }
    }
}

}  // namespace kf
