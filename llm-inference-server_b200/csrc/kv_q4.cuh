// kv_q4.cuh -- the 4-bit paged KV pool: its layout, quantising rows into it and
// reading rows back (b2_kv_append_q4, b2_kv_gather_q4).
//
// A group of 32 head dims of one token's row has a step s and a middle m in f16 and
// codes c in 0..15; an element is s (c - 8) + m.  Codes are taken against the
// rounded s and m, so an element inside the group's range is off by at most s / 2
// plus what the two roundings move the range's ends by.  Everything is computed in
// fp32: with 16-bit inputs x - m is a short sum and (x - m) / s is at least
// 2^-12 (in steps) away from a rounding border it does not hit, so the fp32
// quotient rounds to the code the exact quotient rounds to.
//
// The m half sits low and the s half high in a 32-bit word: s >= 0, so words
// compare as their steps do.
#pragma once

#include "b2_common.cuh"

namespace b2 {

// One (block, layer, kv head) chunk: 16 tokens.
template <int DH>
struct Q4Chunk {
    static constexpr int kGroups = DH / 32;
    static constexpr int kCodes = kBlockTokens * DH / 2;          // bytes of K (or V) codes
    static constexpr int kParams = kBlockTokens * kGroups * 4;    // bytes of K (or V) params
    static constexpr int kKParams = kCodes;
    static constexpr int kV = kCodes + kParams;
    static constexpr int kVParams = kV + kCodes;
    static constexpr int kBytes = 2 * (kCodes + kParams);
    static constexpr int kPerPlane = 16 / kGroups;  // V units of a group in a 32-byte plane row
    static_assert(kBytes == 20 * DH, "chunk size");
    // byte of the word with dims 8 i .. 8 i + 7 of group g
    __host__ __device__ static constexpr int k_word(int t, int i, int g) { return t * (DH / 2) + (i * kGroups + g) * 4; }
    // byte of the unit with dims 4 r .. 4 r + 3 of group g
    __host__ __device__ static constexpr int v_unit(int t, int r, int g) {
        return kV + ((r / kPerPlane) * kBlockTokens + t) * 32 + (r % kPerPlane * kGroups + g) * 2;
    }
    __host__ __device__ static constexpr int param(int t, int g) { return (t * kGroups + g) * 4; }
};

struct KvQ4Params {
    uint8_t* pool;
    void* k;
    void* v;
    long long row_stride;
    const int* slots;
    int rows, n_kv_head, layer_idx, n_layer, num_blocks;
};

// Four neighbouring lanes share a group, 8 elements (16 bytes) each; a thread
// handles its 8 elements of K or of V.  Bound: HBM, 2 bytes read and 0.625
// written an element.
template <typename T, int DH, bool kAppend>
__global__ void __launch_bounds__(256) kv_q4_kernel(const KvQ4Params p) {
    using C = Q4Chunk<DH>;
    constexpr int G = C::kGroups;
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = p.n_kv_head * G * 4;  // threads per K (or V) row
    const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    // a whole group of four is in or out of range together
    const long long row2 = idx / per_row;  // row * 2 + (K | V)
    if (row2 >= 2ll * p.rows) return;
    const int c = static_cast<int>(idx - row2 * per_row);
    const long long row = row2 >> 1;
    const bool is_v = row2 & 1;
    const int i = c & 3, g = (c >> 2) % G, h = (c >> 2) / G;
    const int slot = __ldg(p.slots + row);
    if (slot < 0) return;
    if (slot / kBlockTokens >= p.num_blocks) {
        if (c == 0) flag_error(B2_DEVERR_BLOCK_ID);
        return;
    }
    const int t = slot % kBlockTokens;
    uint8_t* chunk = p.pool + ((static_cast<size_t>(slot / kBlockTokens) * p.n_layer + p.layer_idx) * p.n_kv_head + h) *
                                  static_cast<size_t>(C::kBytes);
    uint32_t* param = reinterpret_cast<uint32_t*>(chunk + (is_v ? C::kVParams : C::kKParams) + C::param(t, g));
    T* x_at = static_cast<T*>(is_v ? p.v : p.k) + row * p.row_stride + (h * DH + g * 32 + i * 8);
    uint32_t codes;
    if (kAppend) {
        float x[8];
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(x_at)), x);
        bool finite = true;
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            finite = finite && isfinite(x[e]);
            x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
        }
        const unsigned mask = 0xfu << (threadIdx.x & 28);
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(mask, lo, d));
            hi = fmaxf(hi, __shfl_xor_sync(mask, hi, d));
        }
        finite = __all_sync(mask, finite);
        const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
        const float s = __half2float(sh);
        const __half mh = __float2half_rn(fmaf(8.0f, s, lo));
        const float m = __half2float(mh);
        codes = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float k = s > 0.0f ? rintf(__fdiv_rn(x[e] - m, s)) + 8.0f : 8.0f;
            codes |= static_cast<uint32_t>(fminf(fmaxf(k, 0.0f), 15.0f)) << (4 * e);
        }
        if (!finite) codes = 0x88888888u;
        if (i == 0)
            *param = finite ? (static_cast<uint32_t>(__half_as_ushort(sh)) << 16 | __half_as_ushort(mh)) : 0x7fff7fffu;
        if (!is_v) {
            *reinterpret_cast<uint32_t*>(chunk + C::k_word(t, i, g)) = codes;
        } else {
            *reinterpret_cast<uint16_t*>(chunk + C::v_unit(t, 2 * i, g)) = static_cast<uint16_t>(codes);
            *reinterpret_cast<uint16_t*>(chunk + C::v_unit(t, 2 * i + 1, g)) = static_cast<uint16_t>(codes >> 16);
        }
    } else {
        const uint32_t w = *param;
        const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
        const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xffffu)));
        if (!is_v) {
            codes = *reinterpret_cast<const uint32_t*>(chunk + C::k_word(t, i, g));
        } else {
            codes = *reinterpret_cast<const uint16_t*>(chunk + C::v_unit(t, 2 * i, g)) |
                    static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(chunk + C::v_unit(t, 2 * i + 1, g))) << 16;
        }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[e] = fmaf(static_cast<float>(static_cast<int>(codes >> (4 * e) & 15u) - 8), s, m);
        *reinterpret_cast<uint4*>(x_at) = pack16<T>(x);
    }
}

}  // namespace b2
