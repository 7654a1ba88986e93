// batch_evict.cu — cut sequences back to their heaviest and most recent tokens.
//
// Per (sequence, kv head): of n slots, left = min(n, n_keep) stay: the recent
// ones, then those of the largest weights. Kept slots below `left` stay where
// they are; the i-th slot that became free there takes the i-th kept slot at
// or behind `left`. Sources lie at or behind `left`, destinations before it,
// so the rows move in place, in any order, and the fewest rows move.
#include <algorithm>

#include "batch.cuh"

namespace gkv {
namespace {

struct EvictParams {
    BatchView v;
    EvictLaunch e;
    int32_t* counts;  // [batch * hkv] moves of each head
    int32_t* left;    // [batch] new length, -1: skipped
    int2* moves;      // [batch * hkv][16 * table_pages] {to, from}
};

constexpr int kPlanThreads = 1024;
constexpr uint32_t kRecent = ~0u, kNaN32 = ~0u - 1;

__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return kNaN32;
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes 0
    return u >> 31 ? ~u : u | 0x80000000u;
}

// The positions of the CTA's threads that hold `flag`, in thread order: how
// many before this one; *all how many in all. sums: one int per warp.
__device__ __forceinline__ int rank_of(bool flag, int* sums, int* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t mask = __ballot_sync(0xFFFFFFFFu, flag);
    __syncthreads();
    if (lane == 0) sums[warp] = __popc(mask);
    __syncthreads();
    int before = __popc(mask & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    *all = total;
    return before;
}

__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const EvictParams p) {
    __shared__ int hist[256];
    __shared__ int found[2];
    __shared__ int sums[kPlanThreads / 32];
    pdl_trigger();
    pdl_wait();
    const BatchView& v = p.v;
    const int tid = threadIdx.x, bh = blockIdx.x, b = bh / v.hkv;
    const int len = v.lens[b];
    const int cap = v.table_pages * kPageSlots;
    if (len > cap && tid == 0) atomicOr(v.err, kErrBadLength);
    const int n = min(len, cap), left = min(n, p.e.n_keep);
    if (tid == 0) {
        if (bh % v.hkv == 0) p.left[b] = len < 0 ? -1 : left;
        if (n <= left) p.counts[bh] = 0;
    }
    if (len < 0) return;
    const size_t row = (size_t)bh * p.e.stride;
    const float* weights = p.e.weights + row;
    const int seen = p.e.seen[b], tracked = p.e.tracked ? p.e.tracked[b] : 0;
    auto position = [&](int t) { return t < tracked ? p.e.positions[row + t] : seen - (n - t); };
    if (n <= left) {
        for (int t = tid; t < n; t += kPlanThreads) {
            p.e.weights_out[row + t] = weights[t];
            p.e.positions_out[row + t] = position(t);
        }
        return;
    }
    auto key = [&](int t) { return position(t) >= seen - p.e.n_recent ? kRecent : key_of(weights[t]); };
    // The smallest kept key, byte by byte from the top.
    uint32_t prefix = 0;
    int want = left;
    for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
        for (int i = tid; i < 256; i += kPlanThreads) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += kPlanThreads) {
            const uint32_t k = key(t);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int rest = want, d = 255;
            while (d > 0 && hist[d] < rest) rest -= hist[d--];
            found[0] = d;
            found[1] = rest;
        }
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        want = found[1];
        __syncthreads();
    }
    // In slot order: `want` of the slots with that key stay, and all above it.
    int2* moves = p.moves + (size_t)bh * v.table_pages * kPageSlots;
    int equal = 0, holes = 0, sources = 0;
    for (int t0 = 0; t0 < n; t0 += kPlanThreads) {
        const int t = t0 + tid;
        const uint32_t k = t < n ? key(t) : 0;
        int all;
        const int same_before = equal + rank_of(t < n && k == prefix, sums, &all);
        equal += all;
        const bool kept = t < n && left > 0 && (k > prefix || (k == prefix && same_before < want));
        const bool hole = t < left && !kept, source = kept && t >= left;
        const int hole_at = holes + rank_of(hole, sums, &all);
        holes += all;
        const int source_at = sources + rank_of(source, sums, &all);
        sources += all;
        if (hole) moves[hole_at].x = t;
        if (source) moves[source_at].y = t;
        if (t < left && kept) {
            const int pos = position(t);
            const float w = weights[t];
            p.e.weights_out[row + t] = w;
            p.e.positions_out[row + t] = pos;
        }
    }
    __syncthreads();
    for (int i = tid; i < holes; i += kPlanThreads) {
        const int2 m = moves[i];
        p.e.weights_out[row + m.x] = weights[m.y];
        p.e.positions_out[row + m.x] = position(m.y);
    }
    if (tid == 0) p.counts[bh] = holes;
}

constexpr int kMoveThreads = 256;

// Moves the rows: one warp per move, K and V.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    constexpr int kChunks = D / 8;
    pdl_wait();
    const BatchView& v = p.v;
    const int lane = threadIdx.x & 31;
    const int bh = blockIdx.y, b = bh / v.hkv, h = bh % v.hkv;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && p.left[b] >= 0) p.e.lens_out[b] = p.left[b];
    if (p.left[b] < 0) return;
    const int count = p.counts[bh];
    const int2* moves = p.moves + (size_t)bh * v.table_pages * kPageSlots;
    const int2* table = v.table + b * v.table_stride;
    for (int i = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); i < count; i += gridDim.x * (kMoveThreads / 32)) {
        const int2 m = moves[i];
        const int2 to = table[m.x / kPageSlots], from = table[m.y / kPageSlots];
        if (min(min(to.x, to.y), min(from.x, from.y)) < 0 || max(max(to.x, to.y), max(from.x, from.y)) >= v.pool_pages) {
            if (lane == 0) atomicOr(v.err, kErrBadPage);
            continue;
        }
        for (int c = lane; c < 2 * kChunks; c += 32) {
            const bool is_v = c >= kChunks;
            uint16_t* pool = is_v ? v.v_base : v.k_base;
            const size_t src = ((size_t)(is_v ? from.y : from.x) * kPageSlots + m.y % kPageSlots) * v.hkv + h;
            const size_t dst = ((size_t)(is_v ? to.y : to.x) * kPageSlots + m.x % kPageSlots) * v.hkv + h;
            reinterpret_cast<uint4*>(pool + dst * D)[c % kChunks] = reinterpret_cast<const uint4*>(pool + src * D)[c % kChunks];
        }
    }
}

size_t round16(size_t x) { return (x + 15) / 16 * 16; }

}  // namespace

size_t evict_bytes(const BatchView& v) {
    const size_t heads = (size_t)v.batch * v.hkv;
    return round16(heads * 4) + round16((size_t)v.batch * 4) + heads * v.table_pages * kPageSlots * sizeof(int2);
}

cudaError_t configure_evict() { return cudaSuccess; }

cudaError_t launch_evict(const BatchView& v, const EvictLaunch& e, cudaStream_t stream) {
    const size_t heads = (size_t)v.batch * v.hkv;
    char* w = static_cast<char*>(e.workspace);
    EvictParams p{v, e, reinterpret_cast<int32_t*>(w), reinterpret_cast<int32_t*>(w + round16(heads * 4)),
                  reinterpret_cast<int2*>(w + round16(heads * 4) + round16((size_t)v.batch * 4))};
    cudaError_t err = launch_dependent(evict_plan_kernel, dim3((unsigned)heads), dim3(kPlanThreads), 0, stream, p);
    if (err != cudaSuccess) return err;
    // About eight CTAs per SM over all heads.
    const int x = (int)std::max<size_t>(1, (size_t)v.sms * 8 / heads);
    const dim3 grid(x, (unsigned)heads), block(kMoveThreads);
    return v.dim == 64    ? launch_dependent(evict_move_kernel<64>, grid, block, 0, stream, p)
           : v.dim == 128 ? launch_dependent(evict_move_kernel<128>, grid, block, 0, stream, p)
                          : launch_dependent(evict_move_kernel<256>, grid, block, 0, stream, p);
}

}  // namespace gkv
