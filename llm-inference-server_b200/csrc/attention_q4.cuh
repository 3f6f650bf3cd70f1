// attention_q4.cuh -- decode attention over the 4-bit paged pool (b2_paged_attention_q4).
//
// out[h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - R_h),  x_j the score in log2
// units, k and v read as s (c - 8) + m per group of 32 dims.  One query token reads
// every byte of its keys and values once, so the bound is HBM (1.25 head_dim
// bytes per token and kv head) as long as turning codes into products stays
// under the instruction rate that HBM leaves: about 3.5 instructions per
// element and lane.  A multiply-add per element, query head and lane is over
// that from two query heads per kv head on, so the products run on the tensor
// cores (mma.sync: its operands come straight from the registers the codes are
// unpacked in; tcgen05 would need them written back to shared memory at 4 times
// their size first, more shared-memory traffic than the codes themselves).
//
//   * A 4-bit code masked into a 16-bit half IS an f16: bits 0-3 give c 2^-24,
//     bits 4-7 give 16 c 2^-24 (subnormals; products with them are exact).  One
//     AND makes two A-operand elements; no conversion, no bias.
//   * Scores: A = 16 tokens x 16 dims of K codes, B = the query heads of the kv
//     head (up to 8 columns).  S = sum_g s_g (A q)_g + sum_g (m_g - 8 s_g) Q_g, Q_g the
//     group's sum of q; the first sum is taken in fp32, the second is one more
//     product whose columns are m and s and whose B is Q in two f16 parts.
//     q is scaled by a power of two to at most 2^9 (and a sixteenth of it where the code
//     counts 16 times): its f16 form is exact down to 2^-19 of the row's largest element
//     (f16; bf16 2^-22), and off by 2^-29 of that element at most below.
//   * Values: A = V codes transposed (16 dims x 16 tokens), B = f16(p s 2^k), k per
//     group of 32 dims; C adds up sum p s c.  The f16 rounding of p s would count
//     with c up to 15; adding the same product with A = -8 makes it count with
//     c - 8 instead.  sum p m is a product with A = m and B = f16(p).  Relative to
//     an output of the values' spread that leaves 2 10^-4 rms, as much as rounding
//     an output to f16 does.  k follows the largest step S that the warp has met in the group:
//     2^8 <= S 2^k < 2^11 (above 2^-1 if S is subnormal).  So f16 rounds a p s above 2^-22 S to
//     its 11 bits, and a smaller one to a multiple of 2^-32 S: 2^-30 S of output a key at most.
//   * Softmax: R_h is a reference that moves only when a score passes it by 4
//     (p <= 16); then, or when an s 2^k grows past 2^11, the accumulators are
//     rescaled.  Sums are fp32.  Weights are held as 2^11 p (up to 2^15): f16(p) would
//     drop what lies 25 binary orders below the largest, which in long contexts adds
//     up (3 % of the middles' sum at 2^20 such keys); 2^11 p drops n 2^-36 at most.
//
// Work: a step is two chunks -- the 20 * head_dim contiguous bytes of a block and kv
// head -- one after the other of an item (sequence, kv head).  The call's steps form one
// list, split evenly over all warps in contiguous parts.  A warp streams its steps
// through its own ring of shared memory with cp.async.bulk, without any CTA barrier.
// Pieces of an item (sequence, kv head) that several warps hold meet in shared
// memory, those of several CTAs in the workspace; the CTA that arrives last
// merges them in CTA order, so results do not depend on timing.
//
// Measured on one B200 (copy rate 6453 GB/s), a launch among others in a graph of a few ms at 1965 MHz:
//   32 sequences of 512 to 32768 tokens, 32/8 heads x 128, bf16   90 us, 4.4 TB/s
//   61 sequences, window 4096, capped scores, same heads          58 us, 3.9 TB/s
//   128 sequences of 256 to 1011 tokens, 25 heads x 64            47 us, 3.0 TB/s
//   64 sequences of 128 to 1024 tokens, 12 heads x 64             16 us, 1.7 TB/s
// (Run for seconds, the first one takes 97 us: at the 1000 W limit the clock falls to 1840 MHz.)  Streaming the same
// chunks without the arithmetic takes 68, 42, 29 and 9 us.  The rest is the chain of dependent instructions in a
// step with three warps a scheduler to hide it: 308 warp instructions a chunk of head_dim 128 fill half
// of the issue slots; warps wait for results of fixed latency and for the tensor pipe (34 % active).  On the
// short calls it is the chain from the wait for the kernel before to the first chunk (4 us) and through the
// merges (4 us).
#pragma once

#include <cfloat>

#include "blocks.cuh"
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
    unsigned* ws_count;  // [kQ4MaxCtas]
    float2* ws_ml;       // [2 grid][group]
    float* ws_acc;       // [2 grid][group][head_dim]
    int batch, n_head, n_kv_head, group, mbps, layer_idx, n_layer, num_blocks, window;
    unsigned kv_mul, kv_shift;  // n / n_kv_head = n * kv_mul >> kv_shift for n < 2^31
    float scale, cap, cap_inv;  // the score cap in log2 units (0: none) and its reciprocal, both finite
};

constexpr int kQ4Warps = 4;
constexpr int kQ4Threads = 32 * kQ4Warps;
// 128 registers a thread at head_dim 64, 168 at 128, where the sums alone take 32.  (128: 4 CTAs 95 us on long
// GQA contexts, 3 CTAs 93; one 32768-token sequence 29 against 25.5.  64, 128 sequences of 25 heads: 5 CTAs 54 us,
// 4 CTAs 49, 3 CTAs 58.  CTAs of 8 warps, two an SM: 98 us and 52.)
constexpr int q4_ctas_per_sm(int dh) { return dh == 64 ? 4 : 3; }
// Ring slots of a warp, a step (two chunks) each: 61 or 82 KB in flight an SM.  A third one cost 1 to 2 %.
constexpr int kQ4Slots = 2;
constexpr int kQ4MaxCtas = 1024;  // the workspace's counters: as many whatever the call's shape, so that calls of different shapes may share one
constexpr int kQ4MaxGroup = 8;
constexpr int kQ4FewParts = 4;  // parts of an item that a CTA merges straight from L2
constexpr int kQ4Weight = 11;   // weights are 2^kQ4Weight p
constexpr float kLog2e = 1.4426950408889634f;

// Bytes of one piece's state in shared memory: [group][head_dim] sums, [group] (R, l).
__host__ __device__ constexpr int q4_piece_bytes(int group, int dh) { return (group * (dh + 2) * 4 + 15) / 16 * 16; }

// Visible keys of a sequence: [first, n).
__device__ __forceinline__ void q4_range(const Q4AttnParams& p, int b, int* first, int* n, unsigned* err) {
    int len = *(p.seq_lens + b);
    if (len < 0 || len > p.mbps * kBlockTokens) {
        *err |= B2_DEVERR_SEQ_LEN;
        len = min(max(len, 0), p.mbps * kBlockTokens);
    }
    int lo = 0;
    if (p.key_starts != nullptr) lo = max(lo, *(p.key_starts + b));
    if (p.window > 0) lo = max(lo, len - p.window);
    *first = min(lo, len);
    *n = len;
}

__device__ __forceinline__ int q4_sequence(const Q4AttnParams& p, int item) {
    return static_cast<int>(static_cast<unsigned long long>(static_cast<unsigned>(item)) * p.kv_mul >> p.kv_shift);
}

// Steps (two blocks, the last one maybe one) over the blocks that hold visible keys.
__device__ __forceinline__ int q4_steps(int first, int n) {
    return first < n ? ((n - 1) / kBlockTokens - first / kBlockTokens) / 2 + 1 : 0;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The product alone (C = 0).
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Two fp32 operations in one instruction (sm_100): a = a op b, elementwise, for what the two heads of a lane do
// alike (long GQA contexts 94.0 -> 90.1 us, 25 heads x 64 48.0 -> 46.8, the same in four layouts of the module).
#define B2_F32X2(NAME, OP)                                                                                     \
    __device__ __forceinline__ void NAME(float (&a)[2], float b0, float b1) {                                  \
        asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t" OP                      \
            ".rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"                                                 \
            : "+f"(a[0]), "+f"(a[1])                                                                           \
            : "f"(b0), "f"(b1));                                                                               \
    }
B2_F32X2(mul2, "mul")
B2_F32X2(add2, "add")
B2_F32X2(sub2, "sub")
#undef B2_F32X2
__device__ __forceinline__ void fma2(float (&a)[2], float b0, float b1, float c0, float c1) {  // a += b c
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %5};\n\t"
        "fma.rn.f32x2 x, y, z, x;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a[0]), "+f"(a[1])
        : "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ void mul2_add(float (&a)[2], float b0, float b1, float c) {  // a = a b + c
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %4};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a[0]), "+f"(a[1])
        : "f"(b0), "f"(b1), "f"(c));
}

// N words from shared memory (volatile: they stay between the waits for a stage and its refill).
template <int N>
__device__ __forceinline__ void ld_words(uint32_t at, uint32_t (&w)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
}
__device__ __forceinline__ uint32_t ld_word(uint32_t at) {
    uint32_t w[1];
    ld_words<1>(at, w);
    return w[0];
}

// One item's running state in a warp.  Lane = 4 r + i.
template <int DH>
struct Q4State {
    static constexpr int G = DH / 32;
    float acc[G][2][4];  // [group][dims 4r+0,1 | 4r+2,3][(dim, head 2i), (dim, 2i+1), (dim+1, 2i), (dim+1, 2i+1)]
    float tz[4];         // row g: sum p m of group g
    float ref[2], l[2];  // heads 2i, 2i+1: the reference less kQ4Weight, and this lane's share of the weights
    uint32_t scale[G];   // high half: steps from here on need a smaller k; low half: 2^(k - kQ4Weight) as f16
    uint32_t qf[G][4];   // B fragments of head r
    uint32_t qb[2];      // B fragment of head r: Q_i 2^-6 as (high, low) f16 parts, and -8 times them
    float sc[2];         // S -> score in log2 units
    float slope[2];      // log2 units
};

// The scale word of a k from -7 to 25: s 2^k < 2^11 below the limit (an f16's exponent bits, 26 - k), and the factor
// exactly (a subnormal f16 below k = -3).  A step of just 2^(11 - k) may count as below the limit (the words' low halves
// decide): with p <= 2^4 its product is still in f16's range.
__device__ __forceinline__ uint32_t q4_scale(int k) {
    const int e = k - kQ4Weight;
    return static_cast<uint32_t>(26 - k) << 26 | static_cast<uint32_t>(e >= -14 ? (e + 15) << 10 : 1 << (e + 24));
}
__device__ __forceinline__ int q4_scale_k(uint32_t w) { return 26 - static_cast<int>(w >> 26); }

// s 2^(k - kQ4Weight), exactly: s in the high half of w, the factor in the low half of scale.
__device__ __forceinline__ float q4_scaled_step(uint32_t w, uint32_t scale) {
    float x;
    asm("{\n\t.reg .f16 m, s, f, limit;\n\tmov.b32 {m, s}, %1;\n\tmov.b32 {f, limit}, %2;\n\t"
        "fma.rn.f32.f16 %0, s, f, %3;\n\t}"
        : "=f"(x)
        : "r"(w), "r"(scale), "f"(0.0f));
    return x;
}

// Loads the query heads of item (b, hk) and clears the sums.
template <typename T, int DH>
__device__ __forceinline__ void q4_start(const Q4AttnParams& p, int b, int hk, Q4State<DH>& st) {
    constexpr int G = DH / 32;
    const int lane = threadIdx.x & 31, r = lane >> 2, i = lane & 3;
    float x[G][8];
    float top = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (r < p.group)
            raw = *(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_row_stride +
                                                       static_cast<long long>(hk * p.group + r) * DH + g * 32 + i * 8));
        unpack16<T>(raw, x[g]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[g][e]));
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    // 2^(8 - floor(log2 top)): the largest |q| lands in [2^8, 2^9)
    const int e2 = static_cast<int>(__float_as_uint(top) >> 23);  // biased exponent, 255 for an infinity
    const int up = e2 == 255 ? 0 : min(135 - e2, 126);
    const float norm = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
    float sum_i = 0.0f;  // Q_i = sum of q over group i
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float f16th = norm * 0.0625f;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(x[g][e], norm, sum);
        st.qf[g][0] = half2_bits(x[g][0] * norm, x[g][4] * norm);
        st.qf[g][1] = half2_bits(x[g][1] * f16th, x[g][5] * f16th);
        st.qf[g][2] = half2_bits(x[g][2] * norm, x[g][6] * norm);
        st.qf[g][3] = half2_bits(x[g][3] * f16th, x[g][7] * f16th);
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if (g == i) sum_i = sum;
    }
    sum_i *= 0x1p-6f;
    const float high = __half2float(__float2half_rn(sum_i));
    st.qb[0] = half2_bits(high, sum_i - high);
    st.qb[1] = half2_bits(-8.0f * high, -8.0f * (sum_i - high));
    // score = S 2^24 / norm * scale (finite, so that S = 0 stays 0); 1 / norm first, whose size is the opposite of a scale's
    // that gives scores in range
    const float unit = kLog2e * p.scale * __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * 0x1p24f;
    const float sc = fminf(fmaxf(unit, -FLT_MAX), FLT_MAX);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int src = 4 * (2 * i + h);
        st.sc[h] = __shfl_sync(0xffffffffu, sc, src);
        st.slope[h] = p.slopes != nullptr && 2 * i + h < p.group ? *(p.slopes + hk * p.group + 2 * i + h) * kLog2e : 0.0f;
        st.ref[h] = -FLT_MAX;
        st.l[h] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) st.scale[g] = q4_scale(25);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        st.tz[c] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) st.acc[g][0][c] = st.acc[g][1][c] = 0.0f;
    }
}

// What a lane reads of a chunk, as byte offsets.
template <int DH>
struct Q4Lane {
    using C = Q4Chunk<DH>;
    // Token of product row r (and r + 8: 8 later), and of product columns 2i and 2i + 1 (and 8
    // later).  Chosen so that the rows' K words, the lanes' V words and all params are read
    // without bank conflicts.
    int tk;
    uint32_t k, kp, kpi, va, vb, ma, mb;
    __device__ __forceinline__ Q4Lane() {
        const int lane = threadIdx.x & 31, r = lane >> 2, i = lane & 3;
        tk = (r & 1) ? 4 + ((r >> 1) ^ 3) : r >> 1;
        const int ta = i, tb = 4 + (i ^ 3);
        k = C::k_word(tk, i, 0);
        kp = C::kKParams + C::param(tk, 0);
        kpi = C::kKParams + C::param(tk, i & (C::kGroups - 1));
        va = C::v_unit(ta, r, 0);
        vb = C::v_unit(tb, r, 0);
        ma = C::kVParams + C::param(ta, r & (C::kGroups - 1));
        mb = C::kVParams + C::param(tb, r & (C::kGroups - 1));
    }
};

// One step: two chunks of 16 tokens at shared addresses stage[0] and stage[1], positions blk * 16 on
// and 16 later, keys [first, n) visible.  Two at a time: their products are independent, and the
// bookkeeping is paid once.  Where the item ends with the first chunk, stage[1] is stage[0]: the second
// chunk's tokens are past n, so their weights are 0, and the steps and middles that those meet are the first one's.
template <int DH>
__device__ __forceinline__ void q4_step(const Q4AttnParams& p, const Q4Lane<DH>& at, const uint32_t (&stage)[2], int blk,
                                        int first, int n, Q4State<DH>& st) {
    using C = Q4Chunk<DH>;
    constexpr int G = DH / 32;
    constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    const int pos = blk * kBlockTokens;
    const bool edge = pos < first || pos + 2 * kBlockTokens > n;
    if (__builtin_expect(edge, 0)) {
        // What masked tokens hold may be anything, NaN included: 0 * NaN must not reach the sums.
        const int lane = threadIdx.x & 31;
        const int j = pos + lane;
        if ((j < first || j >= n) && (lane < kBlockTokens || stage[1] != stage[0])) {
            const uint32_t to = stage[lane >> 4] + C::kVParams + C::param(lane & 15, 0);
#pragma unroll
            for (int g = 0; g < G; ++g) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + 4 * g), "r"(0) : "memory");
        }
        // these generic writes come before the copy that refills the stage
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    }
    float x[4][2];  // [tokens tk, tk + 8 of chunk 0, of chunk 1][head 2i, 2i + 1]
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        uint32_t ka[G], kb[G], pa[G], pb[G];
        ld_words<G>(stage[u] + at.k, ka);
        ld_words<G>(stage[u] + at.k + 8 * (DH / 2), kb);
        ld_words<G>(stage[u] + at.kp, pa);
        ld_words<G>(stage[u] + at.kp + 8 * 4 * G, pb);
        // sum over the groups of (m - 8 s) Q_g: columns (m_i, m_i, s_i, s_i) against (Q_i, -8 Q_i)
        float z[4];
        {
            const uint32_t wa = ld_word(stage[u] + at.kpi), wb = ld_word(stage[u] + at.kpi + 8 * 4 * G);
            mma_f16_first(z, __byte_perm(wa, wa, 0x1010), __byte_perm(wb, wb, 0x1010), __byte_perm(wa, wa, 0x3232),
                    __byte_perm(wb, wb, 0x3232), st.qb[0], st.qb[1]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            x[2 * u + t][0] = z[2 * t], x[2 * u + t][1] = z[2 * t + 1];
            mul2(x[2 * u + t], 0x1p-18f, 0x1p-18f);
        }
        // A product that adds to another's sum waits for it (some 20 cycles): all first ones go before all second ones.
        float c[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g)
            mma_f16_first(c[g], ka[g] & kLow, kb[g] & kLow, ka[g] & kHigh, kb[g] & kHigh, st.qf[g][0], st.qf[g][1]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t ua = ka[g] >> 8, ub = kb[g] >> 8;
            mma_f16(c[g], ua & kLow, ub & kLow, ua & kHigh, ub & kHigh, st.qf[g][2], st.qf[g][3]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float sa = half2_floats(pa[g]).y, sb = half2_floats(pb[g]).y;
            fma2(x[2 * u], sa, sa, c[g][0], c[g][1]);
            fma2(x[2 * u + 1], sb, sb, c[g][2], c[g][3]);
        }
    }
    // Rounded before the reference is taken off: the largest score's weight is 1 however large it is.
#pragma unroll
    for (int t = 0; t < 4; ++t) mul2(x[t], st.sc[0], st.sc[1]);
    if (__builtin_expect(p.cap > 0.0f, 0)) {
        // cap tanh(y), y = x / cap.  Up to 1/2: x (tanh(y) / y), with tanh(y) / y - 1 = y^2 R(y^2), R the minimax cubic
        // (2^-26 relative); beyond: cap (1 - 2 / (1 + e^2y)), whose 2^-22 of the cap is 2^-21 of the score there and would
        // be any share of a smaller one.
        float capped[4][2], top = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float y[2] = {x[t][0], x[t][1]};
            mul2(y, p.cap_inv, p.cap_inv);
            top = fmaxf(top, fmaxf(fabsf(y[0]), fabsf(y[1])));
            mul2(y, y[0], y[1]);
            float r[2] = {0.01724149f, 0.01724149f};
            mul2_add(r, y[0], y[1], -0.05304549f);
            mul2_add(r, y[0], y[1], 0.13325879f);
            mul2_add(r, y[0], y[1], -0.33333144f);
            mul2(r, y[0], y[1]);
            capped[t][0] = x[t][0], capped[t][1] = x[t][1];
            fma2(capped[t], x[t][0], x[t][1], r[0], r[1]);
        }
        if (__any_sync(0xffffffffu, top > 0.5f)) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float y = x[t][h] * p.cap_inv;
                    const float w = __fdividef(2.0f, 1.0f + ex2_approx(2.0f * kLog2e * y));
                    if (fabsf(y) > 0.5f) capped[t][h] = fmaf(-p.cap, w, p.cap);
                }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t][0] = capped[t][0], x[t][1] = capped[t][1];
    }
    if (__builtin_expect(p.slopes != nullptr, 0)) {
        const float d = static_cast<float>(pos + at.tk - (n - 1));
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[t][h] = fmaf(st.slope[h], d + 8.0f * t, x[t][h]);
    }
    if (__builtin_expect(edge, 0)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int j = pos + at.tk + 8 * t;
            if (j < first || j >= n) x[t][0] = x[t][1] = -INFINITY;
        }
    }
    uint32_t vp[4][G];  // V params of the four tokens
#pragma unroll
    for (int t = 0; t < 4; ++t) ld_words<G>(stage[t >> 1] + at.kp + C::kV + (t & 1) * 8 * 4 * G, vp[t]);
    float top[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) top[h] = fmaxf(fmaxf(x[0][h], x[1][h]), fmaxf(x[2][h], x[3][h]));
    bool grows = false;
#pragma unroll
    for (int g = 0; g < G; ++g) grows |= max(__vimax3_u32(vp[0][g], vp[1][g], vp[2][g]), vp[3][g]) >= st.scale[g];
    // The difference, not top - c > ref: from 2^26 on that sum rounds, to ref itself for a score 8 above it.
    // (no short circuit: branches here cost long GQA contexts 98 against 93 us)
    constexpr float kMost = kQ4Weight + 4;
    const bool moves = (top[0] - st.ref[0] > kMost) | (top[1] - st.ref[1] > kMost) | grows;
    if (__builtin_expect(__any_sync(0xffffffffu, moves), 0)) {
        float by[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint32_t s_top = 0;
#pragma unroll
            for (int t = 0; t < 4; ++t)  // NaN and infinite steps do not count
                if (vp[t][g] < 0x7c000000u) s_top = max(s_top, vp[t][g]);
            s_top = __reduce_max_sync(0xffffffffu, s_top);
            const int old = q4_scale_k(st.scale[g]), k = min(old, 23 - static_cast<int>(s_top >> 26));  // s 2^k < 2^9
            by[g] = __uint_as_float(static_cast<uint32_t>(127 + k - old) << 23);
            st.scale[g] = q4_scale(k);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
            const float ref = fmaxf(st.ref[h], __fadd_ru(top[h], -kQ4Weight));  // up: the weights stay below 2^15
            const float f = ex2_approx(st.ref[h] - ref);
            st.ref[h] = ref;
            st.l[h] *= f;
            st.tz[h] *= f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    st.acc[g][t][h] *= f * by[g];
                    st.acc[g][t][2 + h] *= f * by[g];
                }
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        sub2(x[t], st.ref[0], st.ref[1]);
        x[t][0] = ex2_approx(x[t][0]);  // 2^kQ4Weight p from here on
        x[t][1] = ex2_approx(x[t][1]);
        add2(st.l, x[t][0], x[t][1]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // sum p m: A rows = groups (rows from G on repeat them, unused)
        const uint32_t m0 = ld_word(stage[u] + at.ma), m1 = ld_word(stage[u] + at.mb);
        const uint32_t m2 = ld_word(stage[u] + at.ma + 8 * 4 * G), m3 = ld_word(stage[u] + at.mb + 8 * 4 * G);
        const uint32_t b0 = transpose8x8(half2_bits(x[2 * u][0], x[2 * u][1]));
        const uint32_t b1 = transpose8x8(half2_bits(x[2 * u + 1][0], x[2 * u + 1][1]));
        mma_f16(st.tz, __byte_perm(m0, m1, 0x5410), 0, __byte_perm(m2, m3, 0x5410), 0, b0, b1);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        uint32_t v[4][G / 2];  // words of product columns 2i, 2i + 1 and 8 later: groups 2w (low) and 2w + 1 (high)
        ld_words<G / 2>(stage[u] + at.va, v[0]);
        ld_words<G / 2>(stage[u] + at.vb, v[1]);
        ld_words<G / 2>(stage[u] + at.va + 256, v[2]);
        ld_words<G / 2>(stage[u] + at.vb + 256, v[3]);
        uint32_t b0[G], b1[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float sa = q4_scaled_step(vp[2 * u][g], st.scale[g]), sb = q4_scaled_step(vp[2 * u + 1][g], st.scale[g]);
            float pa[2] = {x[2 * u][0], x[2 * u][1]}, pb[2] = {x[2 * u + 1][0], x[2 * u + 1][1]};
            mul2(pa, sa, sa);
            mul2(pb, sb, sb);
            b0[g] = transpose8x8(half2_bits(pa[0], pa[1]));
            b1[g] = transpose8x8(half2_bits(pb[0], pb[1]));
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t pick = g & 1 ? 0x7632 : 0x5410;
            const uint32_t u0 = __byte_perm(v[0][g / 2], v[1][g / 2], pick), u1 = __byte_perm(v[2][g / 2], v[3][g / 2], pick);
            mma_f16(st.acc[g][0], u0 & kLow, u0 & kHigh, u1 & kLow, u1 & kHigh, b0[g], b1[g]);
            const uint32_t w0 = u0 >> 8, w1 = u1 >> 8;
            mma_f16(st.acc[g][1], w0 & kLow, w0 & kHigh, w1 & kLow, w1 & kHigh, b0[g], b1[g]);
        }
        // -8 in the units of even and odd dims: -8 2^-24 and -8 16 2^-24
#pragma unroll
        for (int g = 0; g < G; ++g) {
            mma_f16(st.acc[g][0], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0[g], b1[g]);
            mma_f16(st.acc[g][1], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0[g], b1[g]);
        }
    }
}

// Ends an item: this lane's sums for heads 2i + h, dims 32 g + 4 r .. + 3, and l over all tokens.
template <int DH>
__device__ __forceinline__ void q4_finish(Q4State<DH>& st, float (&out)[2][DH / 32][4], float (&l)[2]) {
    constexpr int G = DH / 32;
    const int i = threadIdx.x & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] = st.l[h];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float c = __shfl_sync(0xffffffffu, st.tz[h], 4 * g + i);
            const float f = __uint_as_float(static_cast<uint32_t>(127 + 24 + kQ4Weight - q4_scale_k(st.scale[g])) << 23);
            out[h][g][0] = fmaf(st.acc[g][0][h], f, c);
            out[h][g][1] = fmaf(st.acc[g][0][2 + h], f * 0.0625f, c);
            out[h][g][2] = fmaf(st.acc[g][1][h], f, c);
            out[h][g][3] = fmaf(st.acc[g][1][2 + h], f * 0.0625f, c);
        }
    }
}

template <typename OutT>
__device__ __forceinline__ void q4_store4(OutT* at, float a, float b, float c, float d) {
    if constexpr (sizeof(OutT) == 4) {
        *reinterpret_cast<float4*>(at) = make_float4(a, b, c, d);
    } else {
        OutT t[4] = {Elem<OutT>::from_f(a), Elem<OutT>::from_f(b), Elem<OutT>::from_f(c), Elem<OutT>::from_f(d)};
        *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(t);
    }
}

struct Q4Entry {
    int item;        // -1: none
    unsigned start;  // the item's first step in the list
    unsigned count;  // its steps
};

// Dynamic shared memory: [warp][slot] steps of two chunks, [warp] first pieces.
template <typename T, typename OutT, int DH>
__global__ void __launch_bounds__(kQ4Threads, q4_ctas_per_sm(DH)) paged_decode_q4_kernel(const Q4AttnParams p) {
    using C = Q4Chunk<DH>;
    constexpr int G = DH / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ unsigned s_seg[kQ4Threads + 1], s_scan[33];
    __shared__ Q4Entry s_entry[2 * kQ4Warps];
    __shared__ Q4Entry s_open[2];  // items of this CTA that other CTAs hold parts of
    __shared__ int s_last[2];
    __shared__ int2 s_parts[2];  // their first CTA and number of CTAs
    __shared__ uint64_t s_bars[kQ4Warps][kQ4Slots];
    __shared__ int4 s_list[kQ4Warps][64];  // the warp's next steps: (chunk, chunk or -1, item, first block)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i = lane & 3, r = lane >> 2;
    const int piece_bytes = q4_piece_bytes(p.group, DH);
    constexpr int kRing = kQ4Slots * 2 * C::kBytes;
    uint8_t* ring = smem + warp * kRing;
    uint8_t* pieces = smem + kQ4Warps * kRing;
    uint64_t* bars = s_bars[warp];
    // A piece's state: slot 0 (the warp's first steps) has its own room, slot 1 (its last) takes the drained ring.
    auto piece_at = [&](int w, int slot) {
        return reinterpret_cast<float*>(slot == 0 ? pieces + w * piece_bytes : smem + w * kRing);
    };
    if (lane == 0) {
#pragma unroll 1
        for (int s = 0; s < kQ4Slots; ++s) mbar_init(bars + s, 1);
        fence_mbar_init();
    }
    if (tid < 2 * kQ4Warps) s_entry[tid].item = -1;
    if (tid < 2) s_open[tid].item = -1;
    pdl_launch_dependents();
    pdl_wait();

    // The list of steps, by sequence, kv head and block: how many come before each thread's share of the sequences.
    unsigned err = 0;
    const int per = (p.batch + kQ4Threads - 1) / kQ4Threads;
    unsigned mine = 0;
#pragma unroll 1
    for (int b = min(tid * per, p.batch); b < min((tid + 1) * per, p.batch); ++b) {
        int first, n;
        q4_range(p, b, &first, &n, &err);
        mine += static_cast<unsigned>(q4_steps(first, n)) * p.n_kv_head;
    }
    if (blockIdx.x != 0) err = 0;
    unsigned total;
    s_seg[tid] = block_scan(mine, 0x7fffffffu, s_scan, &total);
    __syncthreads();
    // Fewer CTAs than launched where a warp would get less than a step.
    const unsigned ctas = max(1u, min(gridDim.x, (total + kQ4Warps - 1) / kQ4Warps));
    // Part (warp) i of the list: `each` steps, one more for the first `more` parts.
    const unsigned parts = ctas * kQ4Warps, each = total / parts, more = total - each * parts;
    auto bound = [&](unsigned part) { return part * each + min(part, more); };
    const bool active = blockIdx.x < ctas;
    const unsigned c0 = active ? bound(blockIdx.x * kQ4Warps + warp) : 0;
    const unsigned c1 = active ? bound(blockIdx.x * kQ4Warps + warp + 1) : 0;

    // Puts the 32 steps from `at` on into the warp's list, a step to a lane.
    auto locate = [&](unsigned at) {
        const unsigned c = at + lane;
        if (c < c1) {
            const int seg = last_at_most(s_seg, kQ4Threads, c);
            unsigned base = s_seg[seg];
            int b = seg * per, first, n, steps;
            unsigned none = 0;
#pragma unroll 1
            for (;; ++b) {
                q4_range(p, b, &first, &n, &none);
                steps = q4_steps(first, n);
                if (c < base + static_cast<unsigned>(steps) * p.n_kv_head || b + 1 == p.batch) break;
                base += static_cast<unsigned>(steps) * p.n_kv_head;
            }
            const int h = static_cast<int>(c - base) / steps;
            const int blk = first / kBlockTokens + 2 * (static_cast<int>(c - base) - h * steps);
            const int* entry = p.block_tables + static_cast<size_t>(b) * p.mbps + blk;
            const bool two = (blk + 1) * kBlockTokens < n;
            int id[2] = {*entry, two ? *(entry + 1) : 0};
            int4 step = make_int4(0, -1, b * p.n_kv_head + h, blk);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (id[k] < 0 || id[k] >= p.num_blocks) {
                    err |= B2_DEVERR_BLOCK_ID;
                    id[k] = min(max(id[k], 0), p.num_blocks - 1);
                }
                id[k] = static_cast<int>((static_cast<long long>(id[k]) * p.n_layer + p.layer_idx) * p.n_kv_head + h);
            }
            step.x = id[0];
            if (two) step.y = id[1];
            s_list[warp][c & 63] = step;
        }
        __syncwarp();
    };
    unsigned located = c0, issued = c0;
    const uint32_t ring_at = smem_addr(ring);

    Q4State<DH> st;
    int item = -1, first = 0, n = 0, from_blk = 0;
    unsigned from = c0;
    // Writes the item's result, or this warp's part of it where it holds not all of its steps.
    auto end_item = [&](unsigned upto) {
        float o[2][G][4], l[2];
        q4_finish<DH>(st, o, l);
        const int b = q4_sequence(p, item), hk = item - b * p.n_kv_head;
        const int steps = q4_steps(first, n);
        if (upto - from == static_cast<unsigned>(steps)) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (2 * i + h < p.group) {
                    const float inv = __fdividef(1.0f, l[h]);
                    OutT* row = static_cast<OutT*>(p.out) +
                                (static_cast<size_t>(b) * p.n_head + hk * p.group + 2 * i + h) * DH + 4 * r;
#pragma unroll
                    for (int g = 0; g < G; ++g)
                        q4_store4<OutT>(row + 32 * g, o[h][g][0] * inv, o[h][g][1] * inv, o[h][g][2] * inv, o[h][g][3] * inv);
                }
            return;
        }
        const int slot = upto == c1 ? 1 : 0;
        float* at = piece_at(warp, slot);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (2 * i + h < p.group) {
#pragma unroll
                for (int g = 0; g < G; ++g)
                    *reinterpret_cast<float4*>(at + (2 * i + h) * DH + 32 * g + 4 * r) =
                        make_float4(o[h][g][0], o[h][g][1], o[h][g][2], o[h][g][3]);
                if (r == 0) *reinterpret_cast<float2*>(at + p.group * DH + 2 * (2 * i + h)) = make_float2(st.ref[h], l[h]);
            }
        if (lane == 0)
            s_entry[2 * warp + slot] = Q4Entry{item, from - static_cast<unsigned>((from_blk - first / kBlockTokens) / 2),
                                               static_cast<unsigned>(steps)};
    };
    const Q4Lane<DH> offs;
    bool alive = true;
    // What is rare in the loop below and in q4_step is marked, to lie apart from the instructions of every step.
    unsigned c = c0, item_end = c0;
    int blk = 0;
    while (c0 < c1) {
        // Refill the ring: a lane copies a step.
        const unsigned limit = min(c1, c + kQ4Slots);
        if (__builtin_expect(limit > located, 0)) {
            locate(located);
            located += 32;
        }
        if (issued + lane < limit) {
            const unsigned idx = issued + lane, slot = (idx - c0) % kQ4Slots;
            const int4 step = s_list[warp][idx & 63];
            mbar_arrive_expect_tx(bars + slot, step.y >= 0 ? 2 * C::kBytes : C::kBytes);
            uint8_t* to = ring + slot * 2 * C::kBytes;
            bulk_g2s(to, p.pool + static_cast<size_t>(step.x) * C::kBytes, C::kBytes, bars + slot);
            if (step.y >= 0)
                bulk_g2s(to + C::kBytes, p.pool + static_cast<size_t>(step.y) * C::kBytes, C::kBytes, bars + slot);
        }
        issued = limit;
        __syncwarp();
        if (__builtin_expect(c == item_end, 0)) {
            if (item >= 0) end_item(c);
            if (c == c1) break;
            const int4 step = s_list[warp][c & 63];
            item = step.z;
            from = c;
            from_blk = blk = step.w;
            const int b = q4_sequence(p, item);
            unsigned none = 0;
            q4_range(p, b, &first, &n, &none);
            item_end = min(c1, c + static_cast<unsigned>(((n - 1) / kBlockTokens - blk) / 2 + 1));
            q4_start<T, DH>(p, b, item - b * p.n_kv_head, st);
        }
        const unsigned slot = (c - c0) % kQ4Slots;
        alive = __all_sync(0xffffffffu, mbar_wait_bounded(bars + slot, (c - c0) / kQ4Slots & 1));
        if (__builtin_expect(!alive, 0)) break;
        const uint32_t first_at = ring_at + slot * 2 * C::kBytes;
        const uint32_t at[2] = {first_at, (blk + 1) * kBlockTokens < n ? first_at + C::kBytes : first_at};
        q4_step<DH>(p, offs, at, blk, first, n, st);
        __syncwarp();  // every lane is done with the slot
        ++c;
        blk += 2;
    }
    if (!alive) {  // the copies in flight end before this CTA's shared memory goes
        err |= B2_DEVERR_TIMEOUT;
#pragma unroll 1
        for (; c < issued; ++c) mbar_wait_bounded(bars + (c - c0) % kQ4Slots, (c - c0) / kQ4Slots & 1);
    }
    // Sequences without a visible key.
#pragma unroll 1
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int lo, len;
        unsigned none = 0;
        q4_range(p, b, &lo, &len, &none);
        if (lo < len) continue;
        OutT* row = static_cast<OutT*>(p.out) + static_cast<size_t>(b) * p.n_head * DH;
#pragma unroll 1
        for (int e = tid * 4; e < p.n_head * DH; e += kQ4Threads * 4) q4_store4<OutT>(row + e, 0.0f, 0.0f, 0.0f, 0.0f);
    }
    __syncthreads();

    // Pieces of one item lie in consecutive entries (a run).  Every warp sees all entries in its
    // lanes and takes every kQ4Warps-th (run, head).
    const unsigned cta0 = active ? bound(blockIdx.x * kQ4Warps) : 0, cta1 = active ? bound((blockIdx.x + 1) * kQ4Warps) : 0;
    {
        const int it = lane < 2 * kQ4Warps ? s_entry[lane].item : -1;
        const unsigned valid = __ballot_sync(0xffffffffu, it >= 0);
        const unsigned before = valid & ((1u << lane) - 1);
        const int prev = __shfl_sync(0xffffffffu, it, before != 0 ? 31 - __clz(before) : lane);
        const unsigned starts = __ballot_sync(0xffffffffu, it >= 0 && (before == 0 || prev != it));
        const int tasks = __popc(starts) * p.group;
#pragma unroll 1
        for (int task = warp; task < tasks; task += kQ4Warps) {
            const int run = task / p.group, h = task - run * p.group;
            unsigned from_run = starts;
#pragma unroll 1
            for (int skip = run; skip > 0; --skip) from_run &= from_run - 1;
            const int e0 = __ffs(from_run) - 1;
            const unsigned later = starts & ~((2u << e0) - 1);
            const unsigned run_bits = valid & ~((1u << e0) - 1) & (later != 0 ? (later & (0u - later)) - 1 : 0xffffffffu);
            const Q4Entry en = s_entry[e0];
            const float* ml = piece_at(min(lane, 2 * kQ4Warps - 1) >> 1, lane & 1) + p.group * DH + 2 * h;
            const bool in_run = run_bits >> lane & 1u;
            const float ref = in_run ? ml[0] : -FLT_MAX;
            float top = ref;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float f = in_run ? ex2_approx(ref - top) : 0.0f;
            float l = in_run ? f * ml[1] : 0.0f;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
            float sum[G];
#pragma unroll
            for (int g = 0; g < G; ++g) sum[g] = 0.0f;
#pragma unroll 1
            for (unsigned left = run_bits; left != 0; left &= left - 1) {
                const int e = __ffs(left) - 1;
                const float* pc = piece_at(e >> 1, e & 1) + h * DH + lane;
                const float fe = __shfl_sync(0xffffffffu, f, e);
#pragma unroll
                for (int g = 0; g < G; ++g) sum[g] = fmaf(pc[32 * g], fe, sum[g]);
            }
            if (en.start >= cta0 && en.start + en.count <= cta1) {
                const int b = q4_sequence(p, en.item), hk = en.item - b * p.n_kv_head;
                const float inv = __fdividef(1.0f, l);
                OutT* row = static_cast<OutT*>(p.out) + (static_cast<size_t>(b) * p.n_head + hk * p.group + h) * DH;
#pragma unroll
                for (int g = 0; g < G; ++g) row[32 * g + lane] = Elem<OutT>::from_f(sum[g] * inv);
            } else {
                const int open = en.start >= cta0 ? 1 : 0;
                const size_t at = (static_cast<size_t>(blockIdx.x) * 2 + open) * p.group + h;
#pragma unroll
                for (int g = 0; g < G; ++g) __stcg(p.ws_acc + at * DH + 32 * g + lane, sum[g]);
                if (lane == 0) {
                    __stcg(p.ws_ml + at, make_float2(top, l));
                    if (h == 0) s_open[open] = en;
                }
            }
        }
    }
    __syncthreads();

    // Items over several CTAs: the last CTA to arrive merges, in CTA order.
    auto cta_of = [&](unsigned chunk) {
        const unsigned split = more * (each + 1);
        return (chunk < split ? chunk / (each + 1) : more + (chunk - split) / each) / kQ4Warps;
    };
    if (tid < 2) {
        s_last[tid] = 0;
        if (s_open[tid].item >= 0) {
            const unsigned f = cta_of(s_open[tid].start), last = cta_of(s_open[tid].start + s_open[tid].count - 1);
            s_parts[tid] = make_int2(static_cast<int>(f), static_cast<int>(last - f + 1));
            // release: this CTA's parts (ordered before by the barrier); acquire: the others'
            unsigned before;
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.ws_count + f) : "memory");
            if (before == last - f) {
                s_last[tid] = 1;
                p.ws_count[f] = 0;
            }
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int open = 0; open < 2; ++open) {
        if (!s_last[open]) continue;
        const Q4Entry en = s_open[open];
        const int f = s_parts[open].x, parts_n = s_parts[open].y;
        const int b = q4_sequence(p, en.item), hk = en.item - b * p.n_kv_head;
        // workspace row of part j and head h: the item's first CTA wrote its slot 1, the others slot 0
        auto row_of = [&](int j, int h) { return (2 * (f + j) + (j == 0 ? 1 : 0)) * p.group + h; };
        if (parts_n <= kQ4FewParts) {  // the usual case, in one trip to L2: every thread reads all it needs at once
#pragma unroll 1
            for (int e = tid * 4; e < p.group * DH; e += kQ4Threads * 4) {
                const int h = e / DH, d = e % DH;
                float2 ml[kQ4FewParts];
                float4 v[kQ4FewParts];
#pragma unroll
                for (int j = 0; j < kQ4FewParts; ++j) {
                    ml[j] = make_float2(-FLT_MAX, 0.0f);
                    v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (j < parts_n) {
                        ml[j] = __ldcg(p.ws_ml + row_of(j, h));
                        v[j] = __ldcg(reinterpret_cast<const float4*>(p.ws_acc + static_cast<size_t>(row_of(j, h)) * DH + d));
                    }
                }
                float top = ml[0].x, l = 0.0f;
#pragma unroll
                for (int j = 1; j < kQ4FewParts; ++j) top = fmaxf(top, ml[j].x);
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < kQ4FewParts; ++j) {
                    const float w = ex2_approx(ml[j].x - top);
                    l = fmaf(ml[j].y, w, l);
                    sum.x = fmaf(v[j].x, w, sum.x);
                    sum.y = fmaf(v[j].y, w, sum.y);
                    sum.z = fmaf(v[j].z, w, sum.z);
                    sum.w = fmaf(v[j].w, w, sum.w);
                }
                const float inv = __fdividef(1.0f, l);
                q4_store4<OutT>(static_cast<OutT*>(p.out) + (static_cast<size_t>(b) * p.n_head + hk * p.group + h) * DH + d,
                                sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
            }
            continue;
        }
        // the parts' weights and l, per head, in the (drained) rings: [group][parts] and [group]
        float* weight = reinterpret_cast<float*>(smem);
        float* denom = weight + p.group * parts_n;
        float4* partial = reinterpret_cast<float4*>(weight + (p.group * (parts_n + 1) + 3) / 4 * 4);
#pragma unroll 1
        for (int h = warp; h < p.group; h += kQ4Warps) {
            // a lane keeps its first two parts; beyond 64 parts they are read twice
            float2 ml[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                ml[k] = lane + 32 * k < parts_n ? __ldcg(p.ws_ml + row_of(lane + 32 * k, h)) : make_float2(-FLT_MAX, 0.0f);
            float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll 1
            for (int j = lane + 64; j < parts_n; j += 32) top = fmaxf(top, __ldcg(p.ws_ml + row_of(j, h)).x);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            float l = 0.0f;
#pragma unroll 1
            for (int j = lane, k = 0; j < parts_n; j += 32, ++k) {
                const float2 v = k == 0 ? ml[0] : k == 1 ? ml[1] : __ldcg(p.ws_ml + row_of(j, h));
                const float w = ex2_approx(v.x - top);
                weight[h * parts_n + j] = w;
                l = fmaf(v.y, w, l);
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
            if (lane == 0) denom[h] = l;
        }
        __syncthreads();
        // (head, 4 dims) to a thread; spare threads take shares of the parts
        const int quads = p.group * DH / 4;
        const int shares = max(1, kQ4Threads / quads);
#pragma unroll 1
        for (int e = tid; e < quads * shares; e += kQ4Threads) {
            const int share = e / quads, q = e - share * quads;
            const int h = q / (DH / 4), d = q % (DH / 4) * 4;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
            for (int j = share; j < parts_n; j += shares) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(p.ws_acc + static_cast<size_t>(row_of(j, h)) * DH + d));
                const float w = weight[h * parts_n + j];
                sum.x = fmaf(v.x, w, sum.x);
                sum.y = fmaf(v.y, w, sum.y);
                sum.z = fmaf(v.z, w, sum.z);
                sum.w = fmaf(v.w, w, sum.w);
            }
            if (shares > 1) {
                partial[e] = sum;
            } else {
                const float inv = __fdividef(1.0f, denom[h]);
                q4_store4<OutT>(static_cast<OutT*>(p.out) + (static_cast<size_t>(b) * p.n_head + hk * p.group + h) * DH + d,
                                sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
            }
        }
        if (shares > 1) {
            __syncthreads();
            if (tid < quads) {
                const int h = tid / (DH / 4), d = tid % (DH / 4) * 4;
                float4 sum = partial[tid];
#pragma unroll 1
                for (int s = 1; s < shares; ++s) {
                    const float4 v = partial[s * quads + tid];
                    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                }
                const float inv = __fdividef(1.0f, denom[h]);
                q4_store4<OutT>(static_cast<OutT*>(p.out) + (static_cast<size_t>(b) * p.n_head + hk * p.group + h) * DH + d,
                                sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
            }
        }
        __syncthreads();  // the shared arrays serve the next item
    }
    if (err != 0) flag_error(err);
}

}  // namespace b2
