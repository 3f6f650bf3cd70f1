// attention_q4.cuh -- decode attention over the 4-bit paged pool (b2_paged_attention_q4).
//
// Plain form: one CTA per (sequence, kv head), a block of 16 tokens at a time
// dequantised into shared memory, online softmax in fp32.
#pragma once

#include "kv_q4.cuh"

namespace b2 {

struct Q4AttnParams {
    const void* q;
    long long q_row_stride;
    const uint8_t* pool;
    const int* block_tables;
    const int* seq_lens;
    const int* key_starts;
    const float* slopes;
    void* out;
    int batch, n_head, n_kv_head, group, mbps, layer_idx, n_layer, num_blocks, window;
    float scale, softcap;
};

// Visible keys of a sequence: [first, n).
__device__ __forceinline__ void q4_range(const Q4AttnParams& p, int b, int* first, int* n, unsigned* err) {
    int len = __ldg(p.seq_lens + b);
    if (len < 0 || len > p.mbps * kBlockTokens) {
        *err |= B2_DEVERR_SEQ_LEN;
        len = min(max(len, 0), p.mbps * kBlockTokens);
    }
    int lo = 0;
    if (p.key_starts != nullptr) lo = max(lo, __ldg(p.key_starts + b));
    if (p.window > 0) lo = max(lo, len - p.window);
    *first = min(lo, len);
    *n = len;
}

constexpr int kQ4Threads = 256;
constexpr int kQ4MaxGroup = 8;

template <typename T, typename OutT, int DH>
__global__ void __launch_bounds__(kQ4Threads) paged_decode_q4_kernel(const Q4AttnParams p) {
    using C = Q4Chunk<DH>;
    __shared__ float s_q[kQ4MaxGroup][DH], s_k[kBlockTokens][DH + 1], s_v[kBlockTokens][DH];
    __shared__ float s_x[kQ4MaxGroup][kBlockTokens];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, hk = blockIdx.y, tid = threadIdx.x;
    unsigned err = 0;
    int first, n;
    q4_range(p, b, &first, &n, &err);
    for (int e = tid; e < p.group * DH; e += kQ4Threads) {
        const int h = hk * p.group + e / DH;
        s_q[e / DH][e % DH] =
            Elem<T>::to_f(static_cast<const T*>(p.q)[b * p.q_row_stride + static_cast<long long>(h) * DH + e % DH]);
    }
    constexpr int kOwn = kQ4MaxGroup * DH / kQ4Threads;
    float m[kOwn], l[kOwn], acc[kOwn];
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        m[o] = -INFINITY;
        l[o] = acc[o] = 0.0f;
    }
    for (int blk = first / kBlockTokens; blk * kBlockTokens < n; ++blk) {
        int id = __ldg(p.block_tables + static_cast<size_t>(b) * p.mbps + blk);
        if (id < 0 || id >= p.num_blocks) {
            err |= B2_DEVERR_BLOCK_ID;
            id = min(max(id, 0), p.num_blocks - 1);
        }
        const uint8_t* chunk = p.pool + ((static_cast<size_t>(id) * p.n_layer + p.layer_idx) * p.n_kv_head + hk) *
                                            static_cast<size_t>(C::kBytes);
        __syncthreads();
        for (int e = tid; e < kBlockTokens * DH; e += kQ4Threads) {
            const int t = e / DH, d = e % DH, g = d / 32, in = d % 32;
            const uint32_t kw = *reinterpret_cast<const uint32_t*>(chunk + C::k_word(t, in / 8, g));
            const uint32_t vw = *reinterpret_cast<const uint16_t*>(chunk + C::v_unit(t, in / 4, g));
            const __half2 kp = *reinterpret_cast<const __half2*>(chunk + C::kKParams + C::param(t, g));
            const __half2 vp = *reinterpret_cast<const __half2*>(chunk + C::kVParams + C::param(t, g));
            const int j = blk * kBlockTokens + t;
            s_k[t][d] = fmaf(static_cast<float>(static_cast<int>(kw >> (4 * (in % 8)) & 15u) - 8), __high2float(kp), __low2float(kp));
            s_v[t][d] = j < first || j >= n ? 0.0f
                                            : fmaf(static_cast<float>(static_cast<int>(vw >> (4 * (in % 4)) & 15u) - 8),
                                                   __high2float(vp), __low2float(vp));
        }
        __syncthreads();
        if (tid < p.group * kBlockTokens) {
            const int h = tid / kBlockTokens, t = tid % kBlockTokens, j = blk * kBlockTokens + t;
            float x = 0.0f;
            for (int d = 0; d < DH; ++d) x = fmaf(s_q[h][d], s_k[t][d], x);
            x *= p.scale;
            if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
            if (p.slopes != nullptr) x = fmaf(__ldg(p.slopes + hk * p.group + h), static_cast<float>(j - (n - 1)), x);
            s_x[h][t] = j < first || j >= n ? -INFINITY : x;
        }
        __syncthreads();
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
            const int e = tid + o * kQ4Threads, h = e / DH, d = e % DH;
            if (h >= p.group) continue;
            float mn = m[o];
            for (int t = 0; t < kBlockTokens; ++t) mn = fmaxf(mn, s_x[h][t]);
            const float c = expf(m[o] - mn);
            l[o] *= c;
            acc[o] *= c;
            for (int t = 0; t < kBlockTokens; ++t) {
                const float w = expf(s_x[h][t] - mn);
                l[o] += w;
                acc[o] = fmaf(w, s_v[t][d], acc[o]);
            }
            m[o] = mn;
        }
    }
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        const int e = tid + o * kQ4Threads, h = e / DH, d = e % DH;
        if (h >= p.group) continue;
        static_cast<OutT*>(p.out)[(static_cast<size_t>(b) * p.n_head + hk * p.group + h) * DH + d] =
            Elem<OutT>::from_f(first < n ? acc[o] / l[o] : 0.0f);
    }
    if (err != 0 && tid == 0 && hk == 0) flag_error(err);
}

}  // namespace b2
