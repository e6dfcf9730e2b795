// Attention over the 4-bit paged KV cache (include/kf_cache.h) for B200 (sm_100a).
//
//   x_j = scale * s_j (q . n_j - z_j sum(q)),  O = sum_j e^(x_j - m) t_j (n'_j - z'_j) / sum_j e^(x_j - m)
// with (s, z, n) a key's scale, zero point and codes, (t, z', n') a value's.
//
// One CTA per query row; a pass takes 256 keys, one per thread, then the row's running
// maximum, sum and output are updated (online softmax, all in fp32).
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
    int B, H_q, H_kv, G, S_q;
    int n_blocks, bs_log2, max_blocks;
    int causal, q_bf16, out_type;
    float scale;
};

template <int D>
__global__ void __launch_bounds__(256) q4_attn_kernel(const Q4AttnParams p) {
    __shared__ float q[D], prob[256], red[8], tsc[256], tzp[256];
    __shared__ const uint8_t* vrow[256];
    const int tid = threadIdx.x;
    const long long row = blockIdx.x;                       // (b * H_q + h) * S_q + i
    const int i = static_cast<int>(row % p.S_q);
    const int h = static_cast<int>(row / p.S_q % p.H_q);
    const int b = static_cast<int>(row / p.S_q / p.H_q);
    for (int d = tid; d < D; d += 256)
        q[d] = p.q_bf16 ? to_f32<true>(p.Q[row * D + d]) : to_f32<false>(p.Q[row * D + d]);
    __syncthreads();
    float qsum = 0.f;
    for (int d = 0; d < D; ++d) qsum += q[d];
    const long long cap = static_cast<long long>(p.max_blocks) << p.bs_log2;
    long long n = p.lens[b];
    n = n < 0 ? 0 : n > cap ? cap : n;
    if (p.causal) n -= p.S_q - 1 - i;
    const int hk = h / p.G;
    float m = -INFINITY, l = 0.f, o = 0.f;                  // thread d < D owns output dim d
    for (long long j0 = 0; j0 < n; j0 += 256) {
        const long long j = j0 + tid;
        float x = -INFINITY;
        vrow[tid] = nullptr;
        tsc[tid] = tzp[tid] = 0.f;
        if (j < n) {
            x = 0.f;
            const int blk = p.table[b * static_cast<long long>(p.max_blocks) + (j >> p.bs_log2)];
            if (blk >= 0 && blk < p.n_blocks) {
                const long long slot = (static_cast<long long>(blk) << p.bs_log2) + (j & ((1 << p.bs_log2) - 1));
                const uint8_t* g = q4_group<D>(const_cast<uint8_t*>(p.cache), slot, hk, p.H_kv, p.bs_log2);
                const int r = slot & 15;
                const uint32_t kw = reinterpret_cast<const uint32_t*>(g + Q4<D>::K_WORDS)[r];
                const uint32_t vw = reinterpret_cast<const uint32_t*>(g + Q4<D>::V_WORDS)[r];
                float dot = 0.f;
                for (int c = 0; c < D / 8; ++c) {
                    const uint32_t w = reinterpret_cast<const uint32_t*>(g + r * Q4<D>::ROW)[c];
                    for (int e = 0; e < 8; ++e) dot = fmaf(static_cast<float>((w >> (4 * e)) & 15u), q[8 * c + e], dot);
                }
                x = fmaf(-q4_zero(kw), qsum, dot) * q4_scale(kw) * p.scale;
                vrow[tid] = g + Q4<D>::V_CODES + r * Q4<D>::ROW;
                tsc[tid] = q4_scale(vw);
                tzp[tid] = q4_zero(vw);
            }
        }
        float mx = x;
        for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
        if ((tid & 31) == 0) red[tid >> 5] = mx;
        __syncthreads();
        mx = m;
        for (int w = 0; w < 8; ++w) mx = fmaxf(mx, red[w]);
        __syncthreads();
        const float pr = j < n ? expf(x - mx) : 0.f;
        prob[tid] = pr;
        float sum = pr;
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if ((tid & 31) == 0) red[tid >> 5] = sum;
        __syncthreads();
        const float corr = m == -INFINITY ? 0.f : expf(m - mx);
        l *= corr;
        for (int w = 0; w < 8; ++w) l += red[w];
        if (tid < D) {
            o *= corr;
            const int cnt = n - j0 < 256 ? static_cast<int>(n - j0) : 256;
            for (int k = 0; k < cnt; ++k)
                if (vrow[k])
                    o = fmaf(prob[k] * tsc[k], static_cast<float>((vrow[k][tid >> 1] >> (4 * (tid & 1))) & 15u) - tzp[k], o);
        }
        m = mx;
        __syncthreads();
    }
    if (tid < D) {
        const float y = l == 0.f ? 0.f : o / l;
        const long long at = row * D + tid;
        if (p.out_type == KF_OUT_F32) static_cast<float*>(p.O)[at] = y;
        else static_cast<uint16_t*>(p.O)[at] = p.out_type == KF_OUT_BF16 ? from_f32<true>(y) : from_f32<false>(y);
    }
    if (tid == 0) {
        if (p.Mi) p.Mi[row] = m;
        if (p.Li) p.Li[row] = l;
    }
}

}  // namespace kf
