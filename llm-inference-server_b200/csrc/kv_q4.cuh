// kv_q4.cuh -- the 4-bit paged KV pool: its layout, quantising rows into it and
// reading rows back (b2_kv_append_q4, b2_kv_gather_q4).
//
// A group of 32 head dims of one token's row has a step s and a middle m in f16 and
// codes c in 0..15; an element is s (c - 8) + m.  Codes are taken against the
// rounded s and m, so an element inside the group's range is off by at most s / 2
// plus what the two roundings move the range's ends by.  Everything is computed in
// fp32, which decides the code where (x - m) / s lies within fp32's rounding of a border
// (an element 2^24 times smaller than m that would tip a tie does not count).
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

// Codes of 8 elements straight from the definition, packed from the low nibble up; rs the correctly rounded 1 / s.
// d rs with one correction step is the correctly rounded quotient (Markstein).
__device__ __forceinline__ uint32_t q4_codes_exact(const float (&x)[8], float m, float s, float rs) {
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float d = fminf(fmaxf(x[e], -65504.0f), 65504.0f) - m;
        const float q0 = d * rs, q = fmaf(fmaf(-q0, s, d), rs, q0);
        codes |= static_cast<uint32_t>(static_cast<int>(rintf(fminf(fmaxf(q, -8.0f), 7.0f))) + 8) << (4 * e);
    }
    return codes;
}

// The codes of 8 elements; rs = 1 / s, ms = -m / s.  q = x rs + ms in one fused step is off by at most 2^-22 (2 |ms| +
// 16) from the quotient, so rounding it gives the code wherever it is further than that from a rounding
// border: within `limit` of an integer.  No code needs cutting off where s is a normal f16 (off by 2^-11 of itself at
// most, which puts the range's upper end at 7.01; a subnormal s may be off by half of itself and the end
// at 14.5) and m's own rounding (2^-11 |m|) is under 0.45 s; elsewhere limit is 0.  What is not within it -- 0.06 %
// of the elements of normal bf16 rows, mostly exact ties; groups far from zero for their width; steps
// below 2^-14; saturated groups -- takes the definition.  Four codes are added up as c0 + 16 c1 + 256 c2 +
// 4096 c3 in fp32 (exact): fp32 instructions issue at twice the integer ones' rate.
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[8], float m, float s, float rs, float ms, float limit) {
    constexpr float kMagic = 12582912.0f;  // 1.5 2^23: adding it rounds to an integer, ties to even
    float far = 0.0f, packed[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        packed[w] = kMagic + 34952.0f;  // 8 (1 + 16 + 256 + 4096)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = fmaf(x[4 * w + e], rs, ms);
            const float k = (q + kMagic) - kMagic;
            far = fmaxf(far, fabsf(q - k));
            packed[w] = fmaf(k, static_cast<float>(1 << (4 * e)), packed[w]);
        }
    }
    if (far < limit)
        return __byte_perm(__float_as_uint(packed[0]), __float_as_uint(packed[1]), 0x5410);
    return q4_codes_exact(x, m, s, rs);
}

template <typename T>
struct Pair16;
template <>
struct Pair16<__half> {
    using Type = __half2;
};
template <>
struct Pair16<__nv_bfloat16> {
    using Type = __nv_bfloat162;
};

// Two of a word's values: codes in the low bits of both halves of c (as f16: 1024 + code, see below), w = (m, s).
__device__ __forceinline__ void q4_values2(uint32_t c, uint32_t w, float m, float* x0, float* x1) {
    asm("{\n\t.reg .f16 c0, c1, lo, hi;\n\t"
        "mov.b32 {c0, c1}, %2;\n\tmov.b32 {lo, hi}, %3;\n\t"
        "fma.rn.f32.f16 %0, c0, hi, %4;\n\tfma.rn.f32.f16 %1, c1, hi, %4;\n\t}"
        : "=f"(*x0), "=f"(*x1)
        : "r"(c), "r"(w), "f"(m));
}

// The 8 values of a codes word.  0x6400 | c is the f16 1024 + c (and 0x6400 | 16 c is 1024 + 16 c); taking 1032
// off (or 1/16 of it less 72) leaves c - 8, all exact; s (c - 8) + m is one fused step with an fp32 result.
__device__ __forceinline__ void q4_values(uint32_t codes, uint32_t w, float (&x)[8]) {
    const float m = __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xffffu)));
    const __half2 minus1032 = __float2half2_rn(-1032.0f), sixteenth = __float2half2_rn(0.0625f), minus72 = __float2half2_rn(-72.0f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t u = codes >> (8 * k);
        const uint32_t even = (u & 0x000f000fu) | 0x64006400u, odd = (u & 0x00f000f0u) | 0x64006400u;
        const __half2 e = __hadd2(*reinterpret_cast<const __half2*>(&even), minus1032);
        const __half2 o = __hfma2(*reinterpret_cast<const __half2*>(&odd), sixteenth, minus72);
        q4_values2(*reinterpret_cast<const uint32_t*>(&e), w, m, &x[2 * k], &x[2 * k + 4]);
        q4_values2(*reinterpret_cast<const uint32_t*>(&o), w, m, &x[2 * k + 1], &x[2 * k + 5]);
    }
}

// Quantising: a thread takes a whole group of 32 (64 bytes), so that what is per group -- extremes, step,
// middle, their conversions -- is worked out once and no lanes have to agree.  2 bytes read and 0.625
// written an element.  16384 rows of 8 heads x 128: 43 us with four lanes to a group, 23 us so (3.8 TB/s;
// floor 13.6).  Two things share the time: 16.5 instructions an element fill 71 % of the issue slots,
// and a thread's four loads are waited for at once (the largest stall; 5 CTAs an SM hide part of it).  The loads,
// 64 bytes apart, and the 2- and 4-byte stores take 2 and 2.8 times the sectors, in L1 and L2; DRAM sees each byte once.
template <typename T, int DH>
__global__ void __launch_bounds__(256) kv_append_q4_kernel(const KvQ4Params p, int rows_per_cta) {
    using C = Q4Chunk<DH>;
    using P = typename Pair16<T>::Type;
    constexpr int G = C::kGroups;
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = 2 * p.n_kv_head * G;  // groups of a row's K and V
    const size_t block_bytes = static_cast<size_t>(p.n_layer) * p.n_kv_head * C::kBytes;
#pragma unroll 1
    for (int idx = threadIdx.x; idx < rows_per_cta * per_row; idx += blockDim.x) {
        const int local = idx / per_row, c = idx - local * per_row;
        const long long row = static_cast<long long>(blockIdx.x) * rows_per_cta + local;
        if (row >= p.rows) return;
        const bool is_v = c >= per_row / 2;
        const int u = is_v ? c - per_row / 2 : c;
        const int g = u % G, h = u / G;
        const int slot = *(p.slots + row);
        const T* from = static_cast<const T*>(is_v ? p.v : p.k) + row * p.row_stride + (h * DH + g * 32);
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = *(reinterpret_cast<const uint4*>(from) + i);
        if (slot < 0) continue;
        if (slot / kBlockTokens >= p.num_blocks) {
            if (c == 0) flag_error(B2_DEVERR_BLOCK_ID);
            continue;
        }
        // extremes in the 16-bit type itself; NaN if an element is
        P a = *reinterpret_cast<const P*>(&raw[0].x), b = a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                a = __hmin2_nan(a, *reinterpret_cast<const P*>(&w[k]));
                b = __hmax2_nan(b, *reinterpret_cast<const P*>(&w[k]));
            }
        }
        float lo = Elem<T>::to_f(__hmin_nan(a.x, a.y)), hi = Elem<T>::to_f(__hmax_nan(b.x, b.y));
        const bool finite = lo > -INFINITY && hi < INFINITY;  // false for NaN
        const bool saturated = lo < -65504.0f || hi > 65504.0f;
        lo = fminf(fmaxf(lo, -65504.0f), 65504.0f);
        hi = fminf(fmaxf(hi, -65504.0f), 65504.0f);
        const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
        const float s = __half2float(sh);
        const __half mh = __float2half_rn(fmaf(8.0f, s, lo));
        const float m = __half2float(mh), rs = __frcp_rn(s), ms = -m * rs;
        const bool plain = !saturated && s >= 0x1p-14f && fabsf(ms) * 0x1p-11f < 0.45f;
        const float limit = plain ? 0.49999f - fabsf(ms) * 0x1p-21f : 0.0f;
        const int t = slot % kBlockTokens;
        uint8_t* chunk = p.pool + static_cast<size_t>(slot / kBlockTokens) * block_bytes +
                         (static_cast<size_t>(p.layer_idx) * p.n_kv_head + h) * C::kBytes;
        *reinterpret_cast<uint32_t*>(chunk + (is_v ? C::kVParams : C::kKParams) + C::param(t, g)) =
            finite ? (static_cast<uint32_t>(__half_as_ushort(sh)) << 16 | __half_as_ushort(mh)) : 0x7fff7fffu;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[8];
            unpack16<T>(raw[i], x);
            const uint32_t codes = s > 0.0f ? q4_codes(x, m, s, rs, ms, limit) : 0x88888888u;
            if (!is_v) {
                *reinterpret_cast<uint32_t*>(chunk + C::k_word(t, i, g)) = codes;
            } else {
                *reinterpret_cast<uint16_t*>(chunk + C::v_unit(t, 2 * i, g)) = static_cast<uint16_t>(codes);
                *reinterpret_cast<uint16_t*>(chunk + C::v_unit(t, 2 * i + 1, g)) = static_cast<uint16_t>(codes >> 16);
            }
        }
    }
}

// Reading back: a CTA takes kRows rows, a thread 8 neighbouring elements (16 bytes) of K or of V in each.  What
// does not depend on the row is worked out once, and the arithmetic stays off the integer and conversion
// pipes: 65531 rows of 8 heads x 128 took 127 us with one row a thread, 70 us with four, and take 66 us in a graph
// (5.3 TB/s) without conversions.
template <typename T, int DH, int kRows>
__global__ void __launch_bounds__(256) kv_gather_q4_kernel(const KvQ4Params p) {
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
        slot[k] = row0 + k < p.rows ? *(p.slots + row0 + k) : -1;
        if (slot[k] >= 0 && slot[k] / kBlockTokens >= p.num_blocks) {
            err |= B2_DEVERR_BLOCK_ID;
            slot[k] = -1;
        }
    }
    if (err != 0 && threadIdx.x == 0) flag_error(err);
    const size_t block_bytes = static_cast<size_t>(p.n_layer) * p.n_kv_head * C::kBytes;
#pragma unroll 1
    for (int c = threadIdx.x; c < 2 * per_row; c += blockDim.x) {
        const bool is_v = c >= per_row;
        const int u = is_v ? c - per_row : c;
        const int i = u & 3, g = (u >> 2) % G, h = (u >> 2) / G;
        const uint8_t* chunk0 = p.pool + (static_cast<size_t>(p.layer_idx) * p.n_kv_head + h) * C::kBytes;
        const uint8_t* param0 = chunk0 + (is_v ? C::kVParams : C::kKParams) + C::param(0, g);
        const uint8_t* code0 = chunk0 + (is_v ? C::v_unit(0, 2 * i, g) : C::k_word(0, i, g));
        const int code_stride = is_v ? 32 : DH / 2;
        constexpr int kNextUnit = C::v_unit(0, 1, 0) - C::v_unit(0, 0, 0);  // dims 4 .. 7 of a V thread: the next unit
        T* x0 = static_cast<T*>(is_v ? p.v : p.k) + row0 * p.row_stride + (h * DH + g * 32 + i * 8);
        uint32_t w[kRows], codes[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            w[k] = codes[k] = 0;
            if (slot[k] < 0) continue;
            const int t = slot[k] % kBlockTokens;
            const size_t at = static_cast<size_t>(slot[k] / kBlockTokens) * block_bytes;
            w[k] = *(reinterpret_cast<const uint32_t*>(param0 + at + t * (4 * G)));
            const uint8_t* from = code0 + at + t * code_stride;
            codes[k] = !is_v ? *reinterpret_cast<const uint32_t*>(from)
                             : __byte_perm(*reinterpret_cast<const uint16_t*>(from),
                                           *reinterpret_cast<const uint16_t*>(from + kNextUnit), 0x5410);
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            if (slot[k] < 0) continue;
            float x[8];
            q4_values(codes[k], w[k], x);
            *reinterpret_cast<uint4*>(x0 + k * p.row_stride) = pack16<T>(x);
        }
    }
}

}  // namespace b2
