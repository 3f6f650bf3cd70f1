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

// The codes of 8 elements against (m, s), packed from the low nibble up.  With q the fp32
// product (x - m) * (1 / s), off by at most 2^-22 |q|, rounding q gives the code wherever q is not
// within 1e-4 of a rounding border; the few elements that are take the division.
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[8], float m, float s) {
    constexpr float kMagic = 12582912.0f;  // 1.5 2^23: adding it rounds to an integer, ties to even
    const float rs = __frcp_rn(s);
    uint32_t codes = 0;
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = (x[e] - m) * rs;
        const float k = q + kMagic;
        far = fmaxf(far, fabsf(q - (k - kMagic)));
        codes |= static_cast<uint32_t>(min(max(static_cast<int>(__float_as_uint(k) - __float_as_uint(kMagic)), -8), 7) + 8) << (4 * e);
    }
    if (far > 0.4999f) {
        codes = 0;
#pragma unroll 1
        for (int e = 7; e >= 0; --e) {
            float v = x[0];
#pragma unroll
            for (int f = 1; f < 8; ++f) v = f == e ? x[f] : v;
            codes = codes << 4 | static_cast<uint32_t>(fminf(fmaxf(rintf(__fdiv_rn(v - m, s)) + 8.0f, 0.0f), 15.0f));
        }
    }
    return s > 0.0f ? codes : 0x88888888u;
}

// A CTA takes kRows rows; a thread 8 neighbouring elements (16 bytes) of K or of V in each, four
// lanes a group of 32.  Bound: HBM, 2 bytes and 0.625 an element.  Several rows a thread keep that many
// 16-byte loads in flight: at 65536 rows of 8 heads x 128 the read-back took 127 us with one row a thread
// (and a 64-bit division to find it) and takes KROWS4_GATHER with four.
template <typename T, int DH, bool kAppend, int kRows>
__global__ void __launch_bounds__(256) kv_q4_kernel(const KvQ4Params p) {
    using C = Q4Chunk<DH>;
    constexpr int G = C::kGroups;
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = p.n_kv_head * G * 4;  // threads for a K (or V) row
    const long long row0 = static_cast<long long>(blockIdx.x) * kRows;
    int slot[kRows];
    unsigned err = 0;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        slot[k] = row0 + k < p.rows ? __ldg(p.slots + row0 + k) : -1;
        if (slot[k] >= 0 && slot[k] / kBlockTokens >= p.num_blocks) {
            err |= B2_DEVERR_BLOCK_ID;
            slot[k] = -1;
        }
    }
    if (err != 0 && threadIdx.x == 0) flag_error(err);
    const size_t block_bytes = static_cast<size_t>(p.n_layer) * p.n_kv_head * C::kBytes;
#pragma unroll 1
    for (int c0 = 0; c0 < 2 * per_row; c0 += blockDim.x) {  // whole warps: the shuffles need every lane
        const int c = c0 + threadIdx.x;
        const bool mine = c < 2 * per_row;
        const bool is_v = c >= per_row;
        const int u = is_v ? c - per_row : c;
        const int i = u & 3, g = (u >> 2) % G, h = (u >> 2) / G;
        uint8_t* chunk0 = p.pool + (static_cast<size_t>(p.layer_idx) * p.n_kv_head + h) * C::kBytes;
        T* x0 = static_cast<T*>(is_v ? p.v : p.k) + row0 * p.row_stride + (h * DH + g * 32 + i * 8);
        if (kAppend) {
            uint4 raw[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k)
                raw[k] = mine && slot[k] >= 0 ? __ldg(reinterpret_cast<const uint4*>(x0 + k * p.row_stride)) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                float x[8];
                unpack16<T>(raw[k], x);
                float lo = INFINITY, hi = -INFINITY, zero = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    zero = fmaf(x[e], 0.0f, zero);  // NaN if an element is NaN or infinite
                    x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
                    lo = fminf(lo, x[e]);
                    hi = fmaxf(hi, x[e]);
                }
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
                    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
                    zero += __shfl_xor_sync(0xffffffffu, zero, d);
                }
                const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
                const __half mh = __float2half_rn(fmaf(8.0f, __half2float(sh), lo));
                if (!mine || slot[k] < 0) continue;
                const uint32_t codes = q4_codes(x, __half2float(mh), __half2float(sh));
                const int t = slot[k] % kBlockTokens;
                uint8_t* chunk = chunk0 + static_cast<size_t>(slot[k] / kBlockTokens) * block_bytes;
                if (i == 0)
                    *reinterpret_cast<uint32_t*>(chunk + (is_v ? C::kVParams : C::kKParams) + C::param(t, g)) =
                        zero == 0.0f ? (static_cast<uint32_t>(__half_as_ushort(sh)) << 16 | __half_as_ushort(mh)) : 0x7fff7fffu;
                if (!is_v) {
                    *reinterpret_cast<uint32_t*>(chunk + C::k_word(t, i, g)) = codes;
                } else {
                    *reinterpret_cast<uint16_t*>(chunk + C::v_unit(t, 2 * i, g)) = static_cast<uint16_t>(codes);
                    *reinterpret_cast<uint16_t*>(chunk + C::v_unit(t, 2 * i + 1, g)) = static_cast<uint16_t>(codes >> 16);
                }
            }
        } else {
            if (!mine) continue;
            uint32_t w[kRows], codes[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                if (slot[k] < 0) continue;
                const int t = slot[k] % kBlockTokens;
                const uint8_t* chunk = chunk0 + static_cast<size_t>(slot[k] / kBlockTokens) * block_bytes;
                w[k] = __ldg(reinterpret_cast<const uint32_t*>(chunk + (is_v ? C::kVParams : C::kKParams) + C::param(t, g)));
                codes[k] = !is_v ? __ldg(reinterpret_cast<const uint32_t*>(chunk + C::k_word(t, i, g)))
                                 : __ldg(reinterpret_cast<const uint16_t*>(chunk + C::v_unit(t, 2 * i, g))) |
                                       static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(chunk + C::v_unit(t, 2 * i + 1, g)))) << 16;
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                if (slot[k] < 0) continue;
                const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(w[k] >> 16)));
                const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(w[k] & 0xffffu)));
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = fmaf(static_cast<float>(static_cast<int>(codes[k] >> (4 * e) & 15u) - 8), s, m);
                *reinterpret_cast<uint4*>(x0 + k * p.row_stride) = pack16<T>(x);
            }
        }
    }
}

}  // namespace b2
