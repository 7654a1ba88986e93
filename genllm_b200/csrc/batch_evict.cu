// batch_evict.cu — cut sequences back to their heaviest and most recent tokens.
//
// Per (sequence, kv head): of n slots, left = min(n, n_keep) stay: the recent
// ones, then those of the largest weights. Kept slots below `left` stay where
// they are; the i-th slot that became free there takes the i-th kept slot at
// or behind `left`. Sources lie at or behind `left`, destinations before it,
// so the rows move in place, in any order, and the fewest rows move.
//
// The plan kernel reads each weight once into shared memory as an ordered
// integer and cuts the row there (cut.cuh), bound by its chain of barriers
// (13 us on 8 rows of 32768, 14 on 256 rows of 4352); the move kernel is a copy,
// bound by HBM: 4 row lengths per move (K and V, read and written; 68 thousand
// moves of 256-byte rows in 13.4 us alone, 5.2 TB/s).
#include <algorithm>

#include "batch.cuh"
#include "cut.cuh"

namespace gkv {
namespace {

// One kept row behind the new length and the slot it goes to.
struct __align__(16) Move {
    int to, from;
    float weight;
    int position;
};

struct EvictParams {
    BatchView v;
    EvictLaunch e;
    int32_t* counts;   // [batch * hkv] moves of each head
    int32_t* left;     // [batch] new length, below 0: skipped
    Move* moves;       // [batch * hkv][8 * table_pages]: a head moves at most half its slots
    uint32_t* keys;    // [batch * hkv][16 * table_pages] where a slice does not fit in shared memory; else null
};

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
// Slots of a thread loaded at once, kept in registers while a run is one batch.
// More of them is longer code for a kernel that runs each line once: 8 / 10 / 12
// took 27.7 / 28.5 / 29.6 us on 8 rows of 32768 by clusters, 30.3 / 28.4 / 28.7
// on 256 rows of 4352 by lone CTAs.
template <bool LONE>
constexpr int kSlotBatch = LONE ? 10 : 8;
constexpr int kMaxSlice = 40960;  // keys of a CTA in shared memory: 160 KB
constexpr uint32_t kRecent = ~0u, kNaN32 = ~0u - 1;

__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return kNaN32;
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes 0
    return u >> 31 ? ~u : u | 0x80000000u;
}

// One cluster per (sequence, head), one slice of its slots per CTA; a warp
// takes a run of its slice, so ranks in slot order are ballots and prefix sums.
template <bool LONE>
__global__ void __launch_bounds__(kPlanThreads, 2) evict_plan_kernel(const EvictParams p) {
    namespace cg = cooperative_groups;
    constexpr int kBatch = kSlotBatch<LONE>;
    extern __shared__ uint32_t slice_keys[];
    __shared__ CutShared<uint32_t, kPlanThreads, LONE> cut_shared;
    __shared__ int slots[kPlanWarps];
    __shared__ int2 rank_slots[2][kMaxCluster];
    pdl_trigger();
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const BatchView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = LONE ? 1 : cluster.num_blocks(), rank = LONE ? 0 : cluster.block_rank();
    const int bh = blockIdx.x / ranks, b = bh / v.hkv;
    const int len = v.lens[b];
    const int cap = v.table_pages * kPageSlots;
    const bool first = rank == 0 && tid == 0;
    if (len > cap && first) atomicOr(v.err, kErrBadLength);
    const int n = min(len, cap), left = min(n, p.e.n_keep);
    if (first) {
        if (bh % v.hkv == 0) p.left[b] = len < 0 ? len : left;
        if (n <= left || left == 0) p.counts[bh] = 0;
    }
    if (len < 0 || left == 0) return;  // the whole cluster
    const size_t row = (size_t)bh * p.e.stride;
    const float* weights = p.e.weights + row;
    const int seen = p.e.seen[b], tracked = p.e.tracked ? p.e.tracked[b] : 0;
    auto position = [&](int t) { return t < tracked ? p.e.positions[row + t] : seen - (len - t); };
    const bool same_weights = p.e.weights_out == p.e.weights;
    const bool same_positions = p.e.positions_out == p.e.positions;
    // What a slot below `left` holds before the moves; in place there is little to write.
    auto stay = [&](int t, float w, int pos) {
        if (!same_weights) p.e.weights_out[row + t] = w;
        if (!same_positions || t >= tracked) p.e.positions_out[row + t] = pos;
    };
    if (n <= left) {
        for (int t = rank * kPlanThreads + tid; t < n; t += ranks * kPlanThreads) stay(t, weights[t], position(t));
        return;  // the whole cluster
    }
    // This CTA's slots [s0, s0 + m).
    const int slice = ((n + ranks - 1) / ranks + 31) / 32 * 32;
    const int s0 = min(n, rank * slice), m = min(n - s0, slice);
    uint32_t* keys = p.keys ? p.keys + (size_t)bh * cap + s0 : slice_keys;
    // A warp's run of the slice; its lanes' weights and positions, all loads of a
    // batch first. A run of one batch keeps them until the end.
    const int run = ((m + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
    const int i0 = min(m, warp * run), i1 = min(m, i0 + run);
    const bool one_batch = run <= 32 * kBatch;
    float w[kBatch];
    int pos[kBatch];
    auto load = [&](int ib) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = ib + j * 32 + lane;
            w[j] = i < i1 ? weights[s0 + i] : 0.f;
            pos[j] = i < i1 ? position(s0 + i) : 0;
        }
    };
    for (int ib = i0; ib < i1; ib += 32 * kBatch) {
        load(ib);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = ib + j * 32 + lane;
            if (i < i1) keys[i] = pos[j] >= seen - p.e.n_recent ? kRecent : key_of(w[j]);
        }
    }
    __syncthreads();
    const Cut<uint32_t> cut = row_cut<uint32_t, kPlanThreads, LONE>(keys, m, left, kRecent, cut_shared);

    const uint32_t below = (1u << lane) - 1;
    int equal = 0;  // keys of the cut's range before this run, in slot order
    if (cut.partial) {
        int mine = 0;
        for (int i = i0 + lane; i < i1; i += 32) mine += keys[i] >= cut.lo && keys[i] <= cut.hi;
        mine = __reduce_add_sync(~0u, mine);
        int all;
        equal = warps_before<kPlanThreads>(mine, slots, &all);
        equal += row_before<LONE>(make_int2(all, 0), rank_slots[0]).x;
    }
    auto kept_of = [&](int i, int* seen_equal) {
        const uint32_t k = i < i1 ? keys[i] : 0;
        const bool in = i < i1 && k >= cut.lo && k <= cut.hi;
        bool kept = i < i1 && (k > cut.hi || in);
        if (cut.partial) {
            const uint32_t mask = __ballot_sync(~0u, in);
            if (in) kept = *seen_equal + __popc(mask & below) < cut.ties;
            *seen_equal += __popc(mask);
        }
        return kept;
    };
    int holes = 0, sources = 0, at = equal;
    for (int i = i0; i < i1; i += 32) {
        const bool kept = kept_of(i + lane, &at);
        const int t = s0 + i + lane;
        holes += __popc(__ballot_sync(~0u, i + lane < i1 && t < left && !kept));
        sources += __popc(__ballot_sync(~0u, kept && t >= left));
    }
    int hole_all, source_all;
    int hole_at = warps_before<kPlanThreads>(holes, slots, &hole_all);
    int source_at = warps_before<kPlanThreads>(sources, slots, &source_all);
    const int2 before = row_before<LONE>(make_int2(hole_all, source_all), rank_slots[1]);
    hole_at += before.x;
    source_at += before.y;
    if (rank == ranks - 1 && tid == kPlanThreads - 1) {
        // The last run's end: the count of the whole row.
        p.counts[bh] = hole_at + holes;
    }
    Move* moves = p.moves + (size_t)bh * (cap / 2);
    at = equal;
    for (int ib = i0; ib < i1; ib += 32 * kBatch) {
        if (!one_batch) load(ib);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = ib + j * 32;
            if (i >= i1) break;
            const bool kept = kept_of(i + lane, &at);
            const int t = s0 + i + lane;
            const bool hole = i + lane < i1 && t < left && !kept, source = kept && t >= left;
            const uint32_t hole_mask = __ballot_sync(~0u, hole), source_mask = __ballot_sync(~0u, source);
            if (hole) moves[hole_at + __popc(hole_mask & below)].to = t;
            if (source) {
                Move& mv = moves[source_at + __popc(source_mask & below)];
                mv.from = t;
                mv.weight = w[j];
                mv.position = pos[j];
            }
            // Holes too: a move over a page that is not in the pool is skipped.
            if (i + lane < i1 && t < left) stay(t, w[j], pos[j]);
            hole_at += __popc(hole_mask);
            source_at += __popc(source_mask);
        }
    }
}

constexpr int kMoveThreads = 256;

// Moves the rows, kGroup moves of a warp in flight: lane j holds the K rows of
// move j, lane kGroup + j its V rows; then all lanes copy, 16 bytes each.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    constexpr int kChunks = D / 8, kGroup = D == 256 ? 4 : 8;
    constexpr int kCopies = kGroup * 2 * kChunks / 32;  // of a lane
    pdl_wait();
    const BatchView& v = p.v;
    const int lane = threadIdx.x & 31;
    const int bh = blockIdx.y, b = bh / v.hkv, h = bh % v.hkv;
    const int left = p.left[b], count = p.counts[bh];
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) p.e.lens_out[b] = left;
    if (left < 0) return;
    const Move* moves = p.moves + (size_t)bh * v.table_pages * (kPageSlots / 2);
    const int2* table = v.table + b * v.table_stride;
    const int step = gridDim.x * (kMoveThreads / 32) * kGroup;
    for (int i0 = (blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5)) * kGroup; i0 < count; i0 += step) {
        const int mine = lane % kGroup;
        int to_row = -1, from_row = -1;
        if (lane < 2 * kGroup && i0 + mine < count) {
            const Move m = moves[i0 + mine];
            const int2 to = table[m.to / kPageSlots], from = table[m.from / kPageSlots];
            if (min(min(to.x, to.y), min(from.x, from.y)) < 0 ||
                max(max(to.x, to.y), max(from.x, from.y)) >= v.pool_pages) {
                atomicOr(v.err, kErrBadPage);
            } else {
                if (lane < kGroup) {
                    p.e.weights_out[(size_t)bh * p.e.stride + m.to] = m.weight;
                    p.e.positions_out[(size_t)bh * p.e.stride + m.to] = m.position;
                }
                to_row = (lane < kGroup ? to.x : to.y) * kPageSlots + m.to % kPageSlots;
                from_row = (lane < kGroup ? from.x : from.y) * kPageSlots + m.from % kPageSlots;
            }
        }
        uint4 x[kCopies];
        uint4* dst[kCopies];
#pragma unroll
        for (int k = 0; k < kCopies; ++k) {
            const int at = k * 32 + lane, c = at % (2 * kChunks);
            const bool is_v = c >= kChunks;
            const int holder = at / (2 * kChunks) + (is_v ? kGroup : 0);
            const int from = __shfl_sync(~0u, from_row, holder), to = __shfl_sync(~0u, to_row, holder);
            uint4* pool = reinterpret_cast<uint4*>(is_v ? v.v_base : v.k_base);
            dst[k] = to < 0 ? nullptr : pool + ((size_t)to * v.hkv + h) * kChunks + c % kChunks;
            if (to >= 0) x[k] = pool[((size_t)from * v.hkv + h) * kChunks + c % kChunks];
        }
#pragma unroll
        for (int k = 0; k < kCopies; ++k)
            if (dst[k]) *dst[k] = x[k];
    }
}

size_t round16(size_t x) { return (x + 15) / 16 * 16; }

struct EvictSpace {
    int cluster;
    bool spill;  // keys in the workspace
    size_t left, moves, keys, all;
};
EvictSpace evict_space(const BatchView& v) {
    const size_t heads = (size_t)v.batch * v.hkv, cap = (size_t)v.table_pages * kPageSlots;
    EvictSpace s;
    s.cluster = cluster_for((int)heads, (int64_t)cap, v.sms, 2048, kMaxSlice);
    s.spill = (cap + s.cluster - 1) / s.cluster > kMaxSlice;
    s.left = round16(heads * sizeof(int32_t));
    s.moves = s.left + round16((size_t)v.batch * sizeof(int32_t));
    s.keys = s.moves + heads * (cap / 2) * sizeof(Move);
    s.all = s.keys + (s.spill ? heads * cap * sizeof(uint32_t) : 0);
    return s;
}

}  // namespace

size_t evict_bytes(const BatchView& v) { return evict_space(v).all; }

cudaError_t configure_evict() {
    const cudaError_t e = configure_kernel(evict_plan_kernel<true>, kMaxSlice * sizeof(uint32_t));
    return e != cudaSuccess ? e : configure_kernel(evict_plan_kernel<false>, kMaxSlice * sizeof(uint32_t));
}

cudaError_t launch_evict(const BatchView& v, const EvictLaunch& e, cudaStream_t stream) {
    const size_t heads = (size_t)v.batch * v.hkv, cap = (size_t)v.table_pages * kPageSlots;
    const EvictSpace s = evict_space(v);
    char* w = static_cast<char*>(e.workspace);
    EvictParams p{v,
                  e,
                  reinterpret_cast<int32_t*>(w),
                  reinterpret_cast<int32_t*>(w + s.left),
                  reinterpret_cast<Move*>(w + s.moves),
                  s.spill ? reinterpret_cast<uint32_t*>(w + s.keys) : nullptr};
    const size_t slice = ((cap + s.cluster - 1) / s.cluster + 31) / 32 * 32;
    cudaError_t err = launch_cluster(s.cluster == 1 ? evict_plan_kernel<true> : evict_plan_kernel<false>, (unsigned)heads, s.cluster, kPlanThreads,
                                     s.spill ? 0 : slice * sizeof(uint32_t), stream, p);
    if (err != cudaSuccess) return err;
    // About eight CTAs per SM over all heads.
    const int x = (int)std::max<size_t>(1, (size_t)v.sms * 8 / heads);
    const dim3 grid(x, (unsigned)heads), block(kMoveThreads);
    return v.dim == 64    ? launch_dependent(evict_move_kernel<64>, grid, block, 0, stream, p)
           : v.dim == 128 ? launch_dependent(evict_move_kernel<128>, grid, block, 0, stream, p)
                          : launch_dependent(evict_move_kernel<256>, grid, block, 0, stream, p);
}

}  // namespace gkv
