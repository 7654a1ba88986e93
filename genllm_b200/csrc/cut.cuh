// cut.cuh — the `target` largest of a row of integer keys, by one CTA or by a
// cluster of them.
//
// Each CTA holds a slice of the row. Per pass the range [lo, hi] of the keys
// that are still undecided is cut into equal buckets, counted in shared memory
// and summed over the cluster through distributed shared memory; the bucket
// the cut falls into becomes the next range. Starting from the keys' own
// smallest and largest values, a spread row is cut in one to three passes, any
// row in ceil(bits / BITS). A lone CTA takes 2048 buckets; in a cluster one a thread, as
// each CTA reads every rank's counts and 2048 of them took longer than the pass
// they save.
#pragma once
#include <cooperative_groups.h>

#include "batch.cuh"

namespace gkv {

// Taken: every key above hi, and the first `ties` (in row order) of those in [lo, hi].
template <typename K>
struct Cut {
    K lo, hi;
    int ties;
    bool partial;  // more keys in [lo, hi] than ties
};

constexpr int kMaxCluster = 8;

// A row's barrier, and rank r's copy of a shared variable.
template <bool LONE>
__device__ __forceinline__ void row_sync() {
    if (LONE) __syncthreads();
    else cooperative_groups::this_cluster().sync();
}
template <bool LONE, typename T>
__device__ __forceinline__ T* at_rank(T* p, int r) {
    return LONE ? p : cooperative_groups::this_cluster().map_shared_rank(p, r);
}

template <typename K, int THREADS, bool LONE>
struct CutShared {
    static constexpr int kBits = LONE ? 11 : THREADS > 512 ? 10 : 9, kBins = 1 << kBits;
    int hist[2][kBins];
    K range[2];       // this CTA's smallest and largest undecided key
    int2 counts;      // how many keys it takes first, and how many others it has
    K warp_lo[THREADS / 32], warp_hi[THREADS / 32];
    int warp_sum[THREADS / 32], warp_rest[THREADS / 32];
    int found[2][3];  // bucket, keys above it, keys in it
};

__device__ __forceinline__ int bit_length(uint32_t x) { return 32 - __clz((int)x); }
__device__ __forceinline__ int bit_length(uint64_t x) { return 64 - __clzll((long long)x); }

template <typename K>
__device__ __forceinline__ void range_reduce(K& lo, K& hi) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(~0u, lo, o));
        hi = max(hi, __shfl_xor_sync(~0u, hi, o));
    }
}
template <>
__device__ __forceinline__ void range_reduce<uint32_t>(uint32_t& lo, uint32_t& hi) {
    lo = __reduce_min_sync(~0u, lo);
    hi = __reduce_max_sync(~0u, hi);
}

// The largest `target` keys of the row. Keys of `skip` and above come before
// all others, and among themselves by row order; keys of 0 stand aside. The row
// holds at least `target` keys that are not 0 (with fewer, all are taken).
// Every thread of the row's CTAs calls it, after a __syncthreads behind the
// writes of keys[0, n). It reads other CTAs' shared memory until it returns:
// the caller passes a row barrier (row_before) before any CTA exits.
template <typename K, int THREADS, bool LONE>
__device__ Cut<K> row_cut(const K* keys, int n, int target, K skip, CutShared<K, THREADS, LONE>& sh) {
    constexpr int kBits = CutShared<K, THREADS, LONE>::kBits, kBins = 1 << kBits, kWarps = THREADS / 32;
    constexpr int kRanks = LONE ? 1 : kMaxCluster;
    static_assert(kBins % THREADS == 0, "whole buckets per thread");
    constexpr int kPer = kBins / THREADS;
    const int ranks = LONE ? 1 : cooperative_groups::this_cluster().num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    K lo = ~(K)0, hi = 0;
    int firsts = 0, rest = 0;
    for (int i = tid; i < n; i += THREADS) {
        const K k = keys[i];
        if (k >= skip) {
            ++firsts;
        } else if (k) {
            ++rest;
            lo = min(lo, k);
            hi = max(hi, k);
        }
    }
    firsts = __reduce_add_sync(~0u, firsts);
    rest = __reduce_add_sync(~0u, rest);
    range_reduce(lo, hi);
    if (lane == 0) sh.warp_lo[warp] = lo, sh.warp_hi[warp] = hi, sh.warp_sum[warp] = firsts, sh.warp_rest[warp] = rest;
    for (int i = tid; i < kBins; i += THREADS) sh.hist[0][i] = 0;
    __syncthreads();
    lo = lane < kWarps ? sh.warp_lo[lane] : ~(K)0;
    hi = lane < kWarps ? sh.warp_hi[lane] : 0;
    firsts = __reduce_add_sync(~0u, lane < kWarps ? sh.warp_sum[lane] : 0);
    rest = __reduce_add_sync(~0u, lane < kWarps ? sh.warp_rest[lane] : 0);
    range_reduce(lo, hi);
    if (!LONE) {
        if (tid == 0) sh.range[0] = lo, sh.range[1] = hi, sh.counts = make_int2(firsts, rest);
        row_sync<LONE>();
        lo = ~(K)0, hi = 0, firsts = rest = 0;
        if (lane < ranks) {
            const K* remote = at_rank<LONE>(sh.range, lane);
            lo = remote[0];
            hi = remote[1];
            const int2 c = *at_rank<LONE>(&sh.counts, lane);
            firsts = c.x;
            rest = c.y;
        }
        firsts = __reduce_add_sync(~0u, firsts);
        rest = __reduce_add_sync(~0u, rest);
        range_reduce(lo, hi);
    }

    if (firsts > target) return {skip, ~(K)0, target, true};
    int want = min(target - firsts, rest);
    if (want == 0) return {skip, (K)(skip - 1), 0, false};

    for (int pass = 0;; ++pass) {
        int* hist = sh.hist[pass & 1];
        int* found = sh.found[pass & 1];
        const int bits = bit_length((K)(hi - lo));
        const int shift = bits > kBits ? bits - kBits : 0;
        for (int i = tid; i < n; i += THREADS) {
            const K k = keys[i];
            if (k >= lo && k <= hi) atomicAdd(&hist[(int)((k - lo) >> shift)], 1);
        }
        row_sync<LONE>();
        // The other buffer is free again: all ranks have read it before this barrier.
        for (int i = tid; i < kBins; i += THREADS) sh.hist[(pass + 1) & 1][i] = 0;
        // Buckets from the top, kPer a thread.
        int part[kRanks][kPer], count[kPer], sum = 0;
#pragma unroll
        for (int r = 0; r < kRanks; ++r) {
            const int* remote = at_rank<LONE>(hist, r < ranks ? r : 0);
#pragma unroll
            for (int i = 0; i < kPer; ++i) part[r][i] = r < ranks ? remote[kBins - 1 - (tid * kPer + i)] : 0;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            count[i] = 0;
#pragma unroll
            for (int r = 0; r < kRanks; ++r) count[i] += part[r][i];
            sum += count[i];
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) sh.warp_sum[warp] = inc;
        __syncthreads();
        int above = inc - sum + __reduce_add_sync(~0u, lane < warp ? sh.warp_sum[lane] : 0);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (above < want && want <= above + count[i]) {
                found[0] = kBins - 1 - (tid * kPer + i);
                found[1] = above;
                found[2] = count[i];
            }
            above += count[i];
        }
        __syncthreads();
        const int in_it = found[2];
        want -= found[1];
        lo = lo + ((K)found[0] << shift);
        hi = lo + min((K)(hi - lo), (K)(((K)1 << shift) - 1));  // lo + 2^shift may not fit
        if (shift == 0 || in_it == want) return {lo, hi, want, in_it > want};
    }
}

// What the warps before this one hold of a value per warp, and the CTA's sum;
// slots: one int per warp of shared memory. Every thread calls it.
template <int THREADS>
__device__ __forceinline__ int warps_before(int mine, int* slots, int* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) slots[warp] = mine;
    __syncthreads();
    const int x = lane < THREADS / 32 ? slots[lane] : 0;
    *all = __reduce_add_sync(~0u, x);
    return __reduce_add_sync(~0u, lane < warp ? x : 0);
}

// What the row's CTAs before this one hold of two values per CTA. Each rank
// stores its own into the others' slots (kMaxCluster of them) ahead of the
// barrier, so nothing reads another CTA's memory behind it.
template <bool LONE>
__device__ __forceinline__ int2 row_before(int2 mine, int2* slots) {
    if (LONE) {
        __syncthreads();
        if (threadIdx.x == 0) slots[0] = mine;
        __syncthreads();
        return make_int2(0, 0);
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, ranks = cluster.num_blocks(), rank = cluster.block_rank();
    if ((int)threadIdx.x < ranks) cluster.map_shared_rank(slots, threadIdx.x)[rank] = mine;
    cluster.sync();
    const int2 x = lane < rank ? slots[lane] : make_int2(0, 0);
    return make_int2(__reduce_add_sync(~0u, x.x), __reduce_add_sync(~0u, x.y));
}

// CTAs per row: enough to spread few rows over the SMs while a slice stays
// worth a CTA (slice_min keys), and enough for a slice to fit (slice_max).
inline int cluster_for(int rows, int64_t keys, int sms, int slice_min, int slice_max) {
    int c = 1;
    while (c < kMaxCluster && ((int64_t)rows * c * 2 <= 2 * sms && keys / (2 * c) >= slice_min)) c *= 2;
    while (c < kMaxCluster && (keys + c - 1) / c > slice_max) c *= 2;
    return c;
}

}  // namespace gkv
