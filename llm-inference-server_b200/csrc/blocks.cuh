// blocks.cuh -- block tables, slots and the free list of a paged pool, kept on
// the device (b2_block_map, b2_block_release).
//
// Two prefix sums over the sequences carry both operators: rows (or blocks to
// give back) before sequence b, and blocks needed before sequence b.  What
// bounds them is latency -- a launch, a chain of dependent loads, two scans -- not
// the few hundred KB they move, so each is one launch.  Map: every CTA reads all lengths
// and scans them for itself (n <= 16384 values, a few L2 lines a thread) and then
// writes its share of the rows; small calls take one CTA, others clusters of
// eight.  Only free_count and the lengths may be updated in place; then there is
// one cluster, every CTA of which has read them before its barrier, and they are
// written after it.  Into separate outputs the map of many rows takes more clusters
// (512 prompts, 139 k rows, in a graph: 13.7 us in place, 6.2 to 6.8 with five).  Release:
// one cluster, whose CTAs take a share of the sequences each and meet their totals.
#pragma once

#include <cooperative_groups.h>

#include "b2_common.cuh"

namespace b2 {

constexpr int kMapThreads = 1024;
constexpr int kMapCluster = 8;  // the portable cluster size
constexpr int kMapMaxSeqs = B2_MAP_MAX_SEQS;
constexpr int kMapPer = kMapMaxSeqs / kMapThreads;  // sequences per thread at most
constexpr int kMapKept = 8;
constexpr unsigned kMapRefused = 0x80000000u;
// Sums are cut off here (far above any free_count): a + b of two cut sums fits
// 32 bits, and min(a + b, cap) is associative.
constexpr unsigned kMapCap = 1u << 30;

struct BlockMapParams {
    int n, mbps, num_blocks, max_rows;
    const int* pre;
    const int* added;
    const int* free_list;
    const int* free_count;
    int* tables;
    int* slots;
    int* q_start;
    int* post;
    int* free_count_out;
};

struct BlockReleaseParams {
    int n, mbps, num_blocks;
    const int* tables;
    const int* lens;
    const int* release;
    int* free_list;
    const int* free_count;
    int* free_count_out;
    int* lens_out;
};

__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b, unsigned cap) { return min(a + b, cap); }

// Exclusive prefix of v (v <= cap) over the CTA's threads, and the total; sums
// stop at cap.  scratch: 33 words.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned cap, unsigned* scratch, unsigned* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    unsigned inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc = sat_add(inc, o, cap);
    }
    unsigned exc = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) exc = 0;
    __syncthreads();  // scratch may still be read from the scan before
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const unsigned w = lane < warps ? scratch[lane] : 0;
        unsigned winc = w;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned o = __shfl_up_sync(0xffffffffu, winc, d);
            if (lane >= d) winc = sat_add(winc, o, cap);
        }
        unsigned wexc = __shfl_up_sync(0xffffffffu, winc, 1);
        if (lane == 0) wexc = 0;
        scratch[lane] = wexc;
        if (lane == 31) scratch[32] = winc;
    }
    __syncthreads();
    *total = scratch[32];
    return sat_add(scratch[warp], exc, cap);
}

// Largest i in [0, n) with start[i] <= x (start ascending, start[0] = 0).
__device__ __forceinline__ int last_at_most(const unsigned* start, int n, unsigned x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int blocks_of(int tokens) {
    return static_cast<int>((static_cast<unsigned>(tokens) + kBlockTokens - 1) / kBlockTokens);
}

// free_count, cut to [0, num_blocks].
__device__ __forceinline__ int read_free_count(const int* p, int num_blocks, unsigned* err) {
    const int c = *reinterpret_cast<const volatile int*>(p);
    if (c < 0 || c > num_blocks) *err |= B2_DEVERR_BLOCK_ID;
    return min(max(c, 0), num_blocks);
}

// Shared words: row[n + 1], blk[n], pre[n].  kPer: sequences to a thread, at most; small calls take the
// kernel for one (the loops over them are unrolled, and a launch that is all latency pays for
// every instruction it fetches: 64 sequences 6.4 -> 4.8 us).
template <int kPer, bool kCluster>
__device__ __forceinline__ void block_map(const BlockMapParams& p) {
    extern __shared__ __align__(16) unsigned smem_u[];
    __shared__ unsigned scratch[33];
    __shared__ unsigned s_used;
    unsigned* s_row = smem_u;             // first row of sequence b
    unsigned* s_blk = s_row + p.n + 1;    // blocks needed before b; kMapRefused: b is refused
    int* s_pre = reinterpret_cast<int*>(s_blk + p.n);
    const int tid = threadIdx.x;
    const int rank = static_cast<int>(blockIdx.x);
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) s_used = 0;
    unsigned err = 0;
    const int free_count = read_free_count(p.free_count, p.num_blocks, &err);
    const int per = (p.n + kMapThreads - 1) / kMapThreads;
    const int b0 = min(tid * per, p.n), b1 = min(b0 + per, p.n);
    const unsigned row_cap = static_cast<unsigned>(p.max_rows);
    const long long len_cap = static_cast<long long>(p.mbps) * kBlockTokens;

    // rows before each sequence
    int add[kPer];
    unsigned rows = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        add[i] = 0;
        if (b0 + i < b1) {
            const int a = p.added != nullptr ? *(p.added + b0 + i) : 1;
            s_pre[b0 + i] = p.pre[b0 + i];
            add[i] = a;
            rows = sat_add(rows, min(static_cast<unsigned>(max(a, 0)), row_cap), row_cap);
        }
    }
    unsigned total_rows;
    unsigned row = block_scan(rows, row_cap, scratch, &total_rows);
    // blocks needed; a sequence whose lengths do not fit needs none and is refused
    unsigned need_sum = 0;
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = b0 + i;
        if (b < b1) {
            const unsigned r = min(static_cast<unsigned>(max(add[i], 0)), row_cap);
            s_row[b] = row;
            const int pre = s_pre[b];
            const bool ok = pre >= 0 && add[i] >= 0 && static_cast<long long>(pre) + add[i] <= len_cap &&
                            static_cast<unsigned long long>(row) + static_cast<unsigned>(add[i]) <= row_cap;
            if (!ok) {
                bad |= 1u << i;
                err |= B2_DEVERR_SEQ_LEN;
            } else {
                need_sum = sat_add(need_sum, static_cast<unsigned>(blocks_of(pre + add[i]) - blocks_of(pre)), kMapCap);
            }
            row = sat_add(row, r, row_cap);
        }
    }
    if (tid == 0) s_row[p.n] = total_rows;
    unsigned total_need;
    unsigned before = block_scan(need_sum, kMapCap, scratch, &total_need);
    unsigned used = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = b0 + i;
        if (b < b1) {
            const int pre = s_pre[b];
            if (bad >> i & 1u) {
                s_blk[b] = kMapRefused;
                continue;
            }
            const unsigned need = static_cast<unsigned>(blocks_of(pre + add[i]) - blocks_of(pre));
            const unsigned upto = sat_add(before, need, kMapCap);
            const bool ok = need == 0 || upto <= static_cast<unsigned>(free_count);
            if (!ok) err |= B2_DEVERR_NO_BLOCKS;
            else if (need != 0) used = upto;
            s_blk[b] = ok ? before : kMapRefused;
            before = upto;
        }
    }
    if (used != 0) atomicMax(&s_used, used);  // the same value whatever the order
    // Also the CTA's barrier: s_* are complete.  Where lengths or count are updated in place there is one
    // cluster, and every CTA has read them now.
    if constexpr (kCluster) cooperative_groups::this_cluster().sync();
    else __syncthreads();

    // rows, four to a thread: one binary search, one 16-byte store
    const int quads = (p.max_rows + 3) / 4;
    const int total = static_cast<int>(total_rows);
    for (int q = rank * kMapThreads + tid; q < quads; q += static_cast<int>(gridDim.x) * kMapThreads) {
        int out[4];
        int b = -1, blk_at = -1, id = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = q * 4 + k;
            out[k] = -1;
            if (r >= total) continue;
            if (b < 0) b = last_at_most(s_row, p.n, static_cast<unsigned>(r));
            while (static_cast<unsigned>(r) >= s_row[b + 1]) {
                ++b;
                blk_at = -1;
            }
            const unsigned base = s_blk[b];
            if (base == kMapRefused) continue;
            const int pre = s_pre[b];
            const int pos = pre + (r - static_cast<int>(s_row[b]));
            const int at = pos / kBlockTokens, have = blocks_of(pre);
            int* entry = p.tables + static_cast<size_t>(b) * p.mbps + at;
            if (at != blk_at) {
                blk_at = at;
                id = at < have ? *entry : *(p.free_list + (free_count - 1 - static_cast<int>(base) - (at - have)));
                if (id < 0 || id >= p.num_blocks) err |= B2_DEVERR_BLOCK_ID;
            }
            // the first position of a new block is always one of the new rows
            if (at >= have && pos % kBlockTokens == 0) *entry = id;
            if (id >= 0 && id < p.num_blocks) out[k] = id * kBlockTokens + pos % kBlockTokens;
        }
        if (q * 4 + 4 <= p.max_rows) {
            *reinterpret_cast<int4*>(p.slots + q * 4) = make_int4(out[0], out[1], out[2], out[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (q * 4 + k < p.max_rows) p.slots[q * 4 + k] = out[k];
        }
    }
    if (rank == 0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = b0 + i;
            if (b < b1) {
                if (p.q_start != nullptr) p.q_start[b] = static_cast<int>(s_row[b]);
                if (p.post != nullptr) p.post[b] = s_pre[b] + (s_blk[b] == kMapRefused ? 0 : add[i]);
            }
        }
        if (tid == 0) *p.free_count_out = free_count - static_cast<int>(s_used);
        if (err & (B2_DEVERR_SEQ_LEN | B2_DEVERR_NO_BLOCKS)) flag_error(err);
    }
    if (err & B2_DEVERR_BLOCK_ID) flag_error(B2_DEVERR_BLOCK_ID);
}

template <int kPer>
__global__ void __cluster_dims__(kMapCluster, 1, 1) __launch_bounds__(kMapThreads)
block_map_kernel(const BlockMapParams p) {
    block_map<kPer, true>(p);
}

// Up to kMapThreads sequences and 4 kMapThreads rows: one CTA, no cluster (64 sequences, one row each: 4.7 us in a
// cluster, 4.1 to 4.4 so).
__global__ void __launch_bounds__(kMapThreads) block_map_small_kernel(const BlockMapParams p) { block_map<1, false>(p); }

// CTA `rank` takes a contiguous share of the sequences; the shares' totals meet
// through distributed shared memory.  Shared words: first[share + 1], bad[share].
__global__ void __cluster_dims__(kMapCluster, 1, 1) __launch_bounds__(kMapThreads)
block_release_kernel(const BlockReleaseParams p) {
    extern __shared__ __align__(16) unsigned smem_u[];
    __shared__ unsigned scratch[33];
    __shared__ unsigned s_totals[kMapCluster];
    __shared__ unsigned s_any_bad;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x;
    const int rank = static_cast<int>(cluster.block_rank());
    const int share = (p.n + kMapCluster - 1) / kMapCluster;
    const int lo = min(rank * share, p.n), n = min(lo + share, p.n) - lo;
    unsigned* s_first = smem_u;            // table entries before sequence i of the share
    unsigned* s_bad = s_first + share + 1; // its entries that are no block ids
    cluster.barrier_arrive();  // waited for below, before the first access to another CTA's shared memory
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) s_any_bad = 0;
    unsigned err = 0;
    const int free_count = read_free_count(p.free_count, p.num_blocks, &err);
    constexpr int kPer = kMapPer / kMapCluster;
    const int per = (n + kMapThreads - 1) / kMapThreads;  // <= kPer
    const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
    unsigned have[kPer];
    int keep[kPer];
    unsigned sum = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        have[k] = 0;
        keep[k] = 0;
        if (i0 + k < i1) {
            const int b = lo + i0 + k;
            const int len = p.lens[b];
            const int cut = min(max(len, 0), p.mbps * kBlockTokens);
            if (*(p.release + b) != 0) {
                have[k] = static_cast<unsigned>(blocks_of(cut));
                if (cut != len) err |= B2_DEVERR_SEQ_LEN;
            } else {
                keep[k] = len;
            }
            s_bad[i0 + k] = 0;
            sum = sat_add(sum, have[k], kMapCap);
        }
    }
    unsigned total;
    unsigned first = block_scan(sum, kMapCap, scratch, &total);
#pragma unroll
    for (int k = 0; k < kPer; ++k)
        if (i0 + k < i1) {
            s_first[i0 + k] = first;
            first = sat_add(first, have[k], kMapCap);
        }
    if (tid == 0) s_first[n] = total;
    __syncthreads();
    // The first kMapKept ids of a thread stay in registers until their places are known.
    auto id_of = [&](unsigned e) {
        const int i = last_at_most(s_first, n, e);
        const int id = *(p.tables + static_cast<size_t>(lo + i) * p.mbps + (e - s_first[i]));
        if (id < 0 || id >= p.num_blocks) {
            atomicAdd(&s_bad[i], 1u);
            s_any_bad = 1;
            err |= B2_DEVERR_BLOCK_ID;
        }
        return id;
    };
    int kept[kMapKept];
#pragma unroll
    for (int k = 0; k < kMapKept; ++k) {
        const unsigned e = tid + k * kMapThreads;
        kept[k] = e < total ? id_of(e) : -1;
    }
#pragma unroll 1
    for (unsigned e = tid + kMapKept * kMapThreads; e < total; e += kMapThreads) id_of(e);
    __syncthreads();
    const bool any_bad = s_any_bad != 0;
    unsigned good = total;
    if (any_bad) {
        sum = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (i0 + k < i1) sum += have[k] - s_bad[i0 + k];
        first = block_scan(sum, kMapCap, scratch, &good);
    }
    cluster.barrier_wait();  // every CTA of the cluster has started
    if (tid < kMapCluster) *cluster.map_shared_rank(&s_totals[rank], tid) = good;
    cluster.sync();  // totals are in place; every CTA has read free_count and its lengths
    unsigned base = static_cast<unsigned>(free_count), end = base;
#pragma unroll
    for (int r = 0; r < kMapCluster; ++r) {
        if (r == rank) base = end;
        end = sat_add(end, s_totals[r], kMapCap);
    }
    const unsigned room = static_cast<unsigned>(p.num_blocks);
    if (end > room) err |= B2_DEVERR_BLOCK_ID;
    if (!any_bad) {
#pragma unroll
        for (int k = 0; k < kMapKept; ++k) {
            const unsigned e = tid + k * kMapThreads;
            if (e < total && base + e < room) p.free_list[base + e] = kept[k];
        }
#pragma unroll 1
        for (unsigned e = tid + kMapKept * kMapThreads; e < total; e += kMapThreads)
            if (base + e < room) p.free_list[base + e] = id_of(e);
    } else {  // rare: a thread closes the gaps of its own sequences
        unsigned at = base + first;
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            for (unsigned c = 0; c < have[k]; ++c) {
                const int id = *(p.tables + static_cast<size_t>(lo + i0 + k) * p.mbps + c);
                if (id < 0 || id >= p.num_blocks) continue;
                if (at < room) p.free_list[at] = id;
                ++at;
            }
    }
    if (p.lens_out != nullptr) {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (i0 + k < i1) p.lens_out[lo + i0 + k] = keep[k];
    }
    if (rank == 0 && tid == 0) *p.free_count_out = static_cast<int>(min(end, room));
    if (err != 0) flag_error(err);
}

}  // namespace b2
