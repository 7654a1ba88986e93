// batch_pages.cu — per-page key bounds, and the pages they rank highest.
//
// Bounds: for a page's keys k_t (t its valid rows), lo_d = min_t k_td and
// hi_d = max_t k_td, exact in the keys' own type. For any query q and key of
// the page, q.k <= u(q) = sum_d (q_d >= 0 ? q_d hi_d : q_d lo_d).
// Selection: per kv head the pages with the largest max_g u(q_g), in the order
// of their values in 64 bits. u = hi.max(q, 0) + lo.min(q, 0) is a product of
// 16-bit matrices, so the tensor cores give every score to within E; only
// pages within 2 E of the cut can be misplaced by that, and these alone are
// summed again in fp64 (in which products of 16-bit floats are exact). On 213
// thousand tokens of 8 sequences, 8 kv heads of 128 (54 MB of bounds, 8 us), the
// scores take 14 us and the cut 13.5, each alone with cold caches (in a step the
// scores start late on some SMs and take 19, the cut has its keys in L2 and takes
// 9.5); all pages in fp64 had taken 87.
#include <algorithm>

#include "batch.cuh"
#include "cut.cuh"

namespace gkv {
namespace {

template <bool F16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if (F16) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if (F16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool F16>
__device__ __forceinline__ float2 floats_of(uint32_t w) {
    if (F16) return __half22float2(*reinterpret_cast<__half2*>(&w));
    return make_float2(bf16_lo(w), bf16_hi(w));
}

// Tokens of sequence b with `extra` more, at most what its table row reaches.
__device__ __forceinline__ int tokens_of(const BatchView& v, int b, int extra, bool flag) {
    const int len = v.lens[b];
    if (len < 0) return 0;
    const int cap = v.table_pages * kPageSlots;
    if (len > cap - extra) {
        if (flag) atomicOr(v.err, kErrBadLength);
        return cap;
    }
    return len + extra;
}

struct BoundsParams {
    BatchView v;
    const int32_t* start;
    uint16_t* bounds;
    int32_t extra;
};

constexpr int kBoundsThreads = 256, kBoundsCtas = 4;

// A lane takes 16 bytes of a page's slot [Hkv][D] down 8 of its 16 rows, the
// lane 16 on the other 8: a warp reads 256 bytes of two rows at once, 4 KB in
// flight, and two lanes meet once at the end. Bound: HBM. (A warp per page and
// head, reduced across all its lanes: 17 us on 114 thousand tokens of 4 heads
// of 64, of which the bytes are 10.)
template <bool F16, int D>
__global__ void __launch_bounds__(kBoundsThreads, kBoundsCtas) page_bounds_kernel(const BoundsParams p) {
    constexpr int kRows = kPageSlots / 2;
    extern __shared__ int base[];
    __shared__ int warp_sums[32];
    pdl_wait();
    pdl_trigger();
    const BatchView& v = p.v;
    auto first_page = [&](int b) { return p.start ? max(0, p.start[b]) / kPageSlots : 0; };
    scan_counts(v.batch, base, warp_sums, [&](int b) {
        return max(0, pages_of(tokens_of(v, b, p.extra, blockIdx.x == 0)) - first_page(b));
    });
    const int lane = threadIdx.x & 31, half = lane >> 4;
    const int chunks = v.hkv * (D / 8);  // of a slot
    const int64_t total = (int64_t)base[v.batch] * chunks;
    const int64_t step = (int64_t)gridDim.x * (kBoundsThreads / 2);
    constexpr uint32_t kInf = F16 ? 0x7C007C00u : 0x7F807F80u;
    for (int64_t t0 = (blockIdx.x * (kBoundsThreads / 32) + (threadIdx.x >> 5)) * 16; t0 < total; t0 += step) {
        const int64_t t = min(t0 + (lane & 15), total - 1);  // behind the end: the last one once more
        const int u = (int)(t / chunks), chunk = (int)(t - (int64_t)u * chunks);
        const int b = owner(base, v.batch, 1, u);
        const int lp = first_page(b) + (u - base[b]);
        const int valid = min(kPageSlots, tokens_of(v, b, p.extra, false) - lp * kPageSlots);
        const int page = v.table[b * v.table_stride + lp].x;
        const bool bad = page < 0 || page >= v.pool_pages;
        if (bad && chunk == 0) atomicOr(v.err, kErrBadPage);
        const uint4* row = reinterpret_cast<const uint4*>(v.k_base) + (size_t)(bad ? 0 : page) * kPageSlots * chunks + chunk;
        uint4 x[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int at = half * kRows + r;
            x[r] = __ldcs(row + (at < valid ? at : 0) * chunks);  // rows behind the sequence: its first again
        }
        uint4 lo = make_uint4(kInf, kInf, kInf, kInf), hi;
        hi = make_uint4(lo.x | 0x80008000u, lo.y | 0x80008000u, lo.z | 0x80008000u, lo.w | 0x80008000u);
        auto join = [&](const uint4& a, const uint4& c) {
            lo.x = min2_nan<F16>(lo.x, a.x), hi.x = max2_nan<F16>(hi.x, c.x);
            lo.y = min2_nan<F16>(lo.y, a.y), hi.y = max2_nan<F16>(hi.y, c.y);
            lo.z = min2_nan<F16>(lo.z, a.z), hi.z = max2_nan<F16>(hi.z, c.z);
            lo.w = min2_nan<F16>(lo.w, a.w), hi.w = max2_nan<F16>(hi.w, c.w);
        };
#pragma unroll
        for (int r = 0; r < kRows; ++r) join(x[r], x[r]);
        const uint4 other_lo = make_uint4(__shfl_xor_sync(~0u, lo.x, 16), __shfl_xor_sync(~0u, lo.y, 16),
                                          __shfl_xor_sync(~0u, lo.z, 16), __shfl_xor_sync(~0u, lo.w, 16));
        const uint4 other_hi = make_uint4(__shfl_xor_sync(~0u, hi.x, 16), __shfl_xor_sync(~0u, hi.y, 16),
                                          __shfl_xor_sync(~0u, hi.z, 16), __shfl_xor_sync(~0u, hi.w, 16));
        join(other_lo, other_hi);
        if (bad) continue;
        uint4* to = reinterpret_cast<uint4*>(p.bounds) + ((size_t)page * v.hkv + chunk / (D / 8)) * 2 * (D / 8) + chunk % (D / 8);
        to[half * (D / 8)] = half ? hi : lo;
    }
}

struct SelectParams {
    BatchView v;
    SelectLaunch s;
    int32_t group;
    int32_t heads, groups, lanes, workers;  // of the score kernel, as in the decode kernel's split
    uint32_t* approx;  // [batch][hkv][table_pages]
    uint32_t* tops;    // [batch][hkv][tiles of 16 pages] largest |bound|, as bits
    uint64_t* exact;   // [batch][hkv][table_pages], where many pages lie at the cut
    bool spill;        // a slice of keys does not fit in shared memory
};

// Scores as integers of the same order, above 0; a page taken in any case
// comes before every score, a NaN before every number.
constexpr uint64_t kTaken = ~0ull, kNaN = ~0ull - 1;
__device__ __forceinline__ uint64_t key_of(double x) {
    if (x != x) return kNaN;
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 becomes 0
    return u >> 63 ? ~u : u | (1ull << 63);
}
constexpr uint32_t kTaken32 = ~0u;
__device__ __forceinline__ uint32_t key32_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key >> 31 ? key & 0x7FFFFFFFu : ~key);
}

constexpr int kScoreWarps = 8;
constexpr int kMaxSlice = 16384;  // keys of a CTA in shared memory: 64 KB
constexpr int kMaxClose = 64;     // pages at the cut that are ranked in shared memory

// E of the tensor cores' score, relative to max |bound| * sum |q|: each of the
// D / 8 products of 16 steps adds 17 numbers, aligned to 24 bits of the largest
// (2^-23 of it each), and rounds. (Measured: at most 0.6 % of it, on normal,
// widely spread and cancelling values of both types.) kTiny: what products
// below fp32's normal range may lose.
template <int D>
constexpr float kScoreError = (D / 8) * 18 * 0x1p-23f;
constexpr float kTiny = 0x1p-117f;
constexpr uint32_t kKeyInf = 0xFF800000u, kKeyMinusInf = 0x007FFFFFu;  // key32_of the infinities

// The score of one page in fp64, by a whole warp; queries: [group][D] in shared memory.
template <bool F16, int D>
__device__ uint64_t exact_key(const SelectParams& p, int h, int page, const float* queries) {
    constexpr int kPer = D / 32;
    const int lane = threadIdx.x & 31;
    const uint16_t* lo = p.s.bounds + ((size_t)page * p.v.hkv + h) * 2 * D + lane * kPer;
    float l[kPer], x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
        const float2 a = floats_of<F16>(*reinterpret_cast<const uint32_t*>(lo + i));
        const float2 c = floats_of<F16>(*reinterpret_cast<const uint32_t*>(lo + D + i));
        l[i] = a.x, l[i + 1] = a.y, x[i] = c.x, x[i + 1] = c.y;
    }
    double best = -INFINITY;
    bool nan = false;
#pragma unroll 4
    for (int g = 0; g < p.group; ++g) {
        const float* q = queries + g * D + lane * kPer;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += (double)q[i] * (double)(q[i] >= 0.f ? x[i] : l[i]);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        nan |= sum != sum;
        best = fmax(best, sum);
    }
    return nan ? kNaN : key_of(best);
}

// Scores on the tensor cores, sixteen pages a step of a warp: the tiles of all
// sequences form one line, cut equally between the workers (one warp per kv
// head of a group), so that ragged batches load every SM alike. Step k of the
// product takes two pairs of dims of the 16-byte chunk that a lane loads of a
// page's row, so rows go from memory to the A fragment as they are. Bound: HBM.
template <bool F16, int D, int NT>
__global__ void __launch_bounds__(kScoreWarps * 32, NT == 1 && D <= 128 ? 2 : 1) page_score_kernel(const SelectParams p) {
    constexpr int kLoads = D / 32;  // 16-byte chunks of a lane's row, of either bound
    extern __shared__ int base[];   // tiles before each sequence
    __shared__ int warp_sums[32];
    pdl_wait();
    pdl_trigger();
    const BatchView& v = p.v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto pages_in = [&](int b, bool flag) { return pages_of(tokens_of(v, b, p.s.extra, flag)); };
    scan_counts(v.batch, base, warp_sums, [&](int b) {
        const int pages = pages_in(b, blockIdx.x == 0);
        return pages <= p.s.n_pages ? 0 : (pages + 15) / 16;  // fewer pages than places: all are taken
    });
    if (warp >= p.lanes * p.heads) return;
    const int total = base[v.batch] * p.groups, per = max(1, (total + p.workers - 1) / p.workers);
    const int worker = blockIdx.x * p.lanes + warp / p.heads, head_in = warp % p.heads;
    const int u0 = (int)min((int64_t)total, (int64_t)worker * per), u1 = min(total, u0 + per);
    const int quarter = lane & 3;
    const int max_tiles = (v.table_pages + 15) / 16;

    for (int u = u0; u < u1;) {
        const int b = owner(base, v.batch, p.groups, u);
        const int tiles = base[b + 1] - base[b], grp = (u - base[b] * p.groups) / tiles;
        const int seg0 = base[b] * p.groups + grp * tiles, end = min(u1, seg0 + tiles);
        const int h = grp * p.heads + head_in;
        if (h >= v.hkv) {
            u = end;
            continue;
        }
        // max(q, 0) for hi, min(q, 0) for lo, as B fragments.
        uint2 f[2][kLoads][2][NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int g = nt * 8 + (lane >> 2);
            const uint16_t* row = p.s.q + b * p.s.q_stride_batch + (int64_t)(h * p.group + g) * p.s.q_stride_head + quarter * 8;
#pragma unroll
            for (int k = 0; k < kLoads; ++k) {
                const uint4 x = g < p.group ? *reinterpret_cast<const uint4*>(row + k * 32) : make_uint4(0, 0, 0, 0);
                auto split = [](uint32_t w, uint32_t& pos, uint32_t& neg) {
                    const uint32_t mask = ((w >> 15 & 1) * 0xFFFFu) | ((w >> 31) * 0xFFFF0000u);
                    pos = w & ~mask;
                    neg = w & mask;
                };
                split(x.x, f[0][k][0][nt].x, f[1][k][0][nt].x);
                split(x.y, f[0][k][0][nt].y, f[1][k][0][nt].y);
                split(x.z, f[0][k][1][nt].x, f[1][k][1][nt].x);
                split(x.w, f[0][k][1][nt].y, f[1][k][1][nt].y);
            }
        }
        const int pages = pages_in(b, false);
        const int2* table = v.table + b * v.table_stride;
        uint32_t* keys = p.approx + ((size_t)b * v.hkv + h) * v.table_pages;
        uint32_t* tops = p.tops + ((size_t)b * v.hkv + h) * max_tiles;
        // This lane's rows are pages lane / 4 and lane / 4 + 8 of a tile.
        int next[2];
        auto fetch = [&](int tile) {
#pragma unroll
            for (int r = 0; r < 2; ++r) next[r] = table[min(tile * 16 + r * 8 + (lane >> 2), pages - 1)].x;
        };
        fetch(u - seg0);
        for (; u < end; ++u) {
            const int tile = u - seg0;
            bool bad[2];
            const uint4* row[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                bad[r] = next[r] < 0 || next[r] >= v.pool_pages;
                row[r] = reinterpret_cast<const uint4*>(p.s.bounds + ((size_t)(bad[r] ? 0 : next[r]) * v.hkv + h) * 2 * D) + quarter;
            }
            uint32_t top[2] = {0, 0};  // of this lane's rows
            float c[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
            constexpr int kHalves = D == 256 ? 2 : 1;  // bounds in flight: both, or one after the other
#pragma unroll
            for (int part = 0; part < kHalves; ++part) {
                constexpr int kTogether = 2 / kHalves;
                uint4 x[kTogether][2][kLoads];
#pragma unroll
                for (int w = 0; w < kTogether; ++w)
#pragma unroll
                    for (int k = 0; k < kLoads; ++k)
#pragma unroll
                        for (int r = 0; r < 2; ++r) x[w][r][k] = __ldcs(row[r] + k * 4 + (part + w == 0 ? D / 8 : 0));
                if (part == 0) fetch(min(tile + 1, tiles - 1));
#pragma unroll
                for (int w = 0; w < kTogether; ++w) {
                    const int low = part + w;
#pragma unroll
                    for (int k = 0; k < kLoads; ++k) {
                        const uint32_t a[2][4] = {{x[w][0][k].x, x[w][1][k].x, x[w][0][k].y, x[w][1][k].y},
                                                  {x[w][0][k].z, x[w][1][k].z, x[w][0][k].w, x[w][1][k].w}};
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            top[0] = __vmaxu2(top[0], __vmaxu2(a[half][0] & 0x7FFF7FFFu, a[half][2] & 0x7FFF7FFFu));
                            top[1] = __vmaxu2(top[1], __vmaxu2(a[half][1] & 0x7FFF7FFFu, a[half][3] & 0x7FFF7FFFu));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma16816<F16>(c[nt], a[half], f[low][k][half][nt].x, f[low][k][half][nt].y);
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float best = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (nt * 8 + quarter * 2 + j < p.group) best = fmaxf(best, c[nt][r * 2 + j]);
                best = fmaxf(best, __shfl_xor_sync(~0u, best, 1));
                best = fmaxf(best, __shfl_xor_sync(~0u, best, 2));
                const int lp = tile * 16 + r * 8 + (lane >> 2);
                const bool taken = lp < p.s.n_first || lp >= pages - p.s.n_last;
                if (taken || bad[r]) top[r] = 0;  // nobody looks at these bounds, whatever they are
                if (quarter == 0 && lp < pages) {
                    if (bad[r] && !taken) atomicOr(v.err, kErrBadPage);
                    keys[lp] = taken ? kTaken32 : bad[r] ? 1u : key32_of(best);
                }
            }
            const uint32_t both = __vmaxu2(top[0], top[1]);
            const uint32_t most = __reduce_max_sync(~0u, max(both & 0xFFFFu, both >> 16));
            if (lane == 0) tops[tile] = most;
        }
    }
}

// The taken pages of each (sequence, head) in rising order, one CTA or cluster
// a row. Bound: latency (a chain of barriers over a few kilobytes).
template <bool F16, int D, bool LONE, int THREADS>
__global__ void __launch_bounds__(THREADS) page_pick_kernel(const SelectParams p) {
    constexpr int kWarps = THREADS / 32;
    struct Close {
        uint64_t key;
        int page;
    };
    extern __shared__ __align__(16) float queries[];  // [group][D], and behind them the slice's keys
    uint32_t* slice_keys = reinterpret_cast<uint32_t*>(queries + p.group * D);
    __shared__ union {
        CutShared<uint32_t, THREADS, LONE> approx;
        CutShared<uint64_t, THREADS, LONE> exact;
    } cut_shared;
    __shared__ Close close[kMaxClose];
    __shared__ int close_page[kMaxClose];
    __shared__ int slots[kWarps];
    __shared__ int2 rank_slots[3][kMaxCluster];
    __shared__ uint32_t warp_top[kWarps];
    __shared__ float head_sum[kMaxBatchGroup];
    const BatchView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = LONE ? 1 : cooperative_groups::this_cluster().num_blocks();
    const int rank = LONE ? 0 : cooperative_groups::this_cluster().block_rank();
    const int bh = blockIdx.x / ranks, b = bh / v.hkv, h = bh % v.hkv;
    // Ahead of the wait: what the score kernel's own predecessors wrote (it lets
    // this one start once they are done), past L1.
    const int len = __ldcg(v.lens + b), cap = v.table_pages * kPageSlots;
    const int pages = len < 0 ? 0 : pages_of(min(len, cap - p.s.extra) + p.s.extra);
    for (int g = warp; g < p.group; g += kWarps) {
        float sum = 0.f;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(p.s.q + b * p.s.q_stride_batch +
                                                                (int64_t)(h * p.group + g) * p.s.q_stride_head);
        for (int d = lane; d < D / 2; d += 32) {
            const float2 x = floats_of<F16>(__ldcg(row + d));
            *reinterpret_cast<float2*>(queries + g * D + 2 * d) = x;
            sum += fabsf(x.x) + fabsf(x.y);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) head_sum[g] = sum;
    }
    pdl_wait();
    pdl_trigger();
    if (len < 0) return;  // the whole row
    int32_t* to = p.s.pages + (size_t)bh * p.s.n_pages;
    const int take = min(p.s.n_pages, pages);
    for (int i = take + rank * THREADS + tid; i < p.s.n_pages; i += ranks * THREADS) to[i] = -1;
    if (pages <= p.s.n_pages) {
        for (int i = rank * THREADS + tid; i < pages; i += ranks * THREADS) to[i] = i;
        return;  // the whole row
    }
    const int slice = ((pages + ranks - 1) / ranks + 31) / 32 * 32;
    const int p0 = min(pages, rank * slice), m = min(pages - p0, slice);
    const int2* table = v.table + b * v.table_stride;
    uint32_t* keys = p.approx + (size_t)bh * v.table_pages + p0;
    // Every CTA looks at all tiles' largest bounds.
    const int max_tiles = (v.table_pages + 15) / 16;
    uint32_t top = tid < (pages + 15) / 16 ? p.tops[(size_t)bh * max_tiles + tid] : 0;
    if (!p.spill) {
        for (int i = tid; i < m; i += 8 * THREADS) {
            uint32_t x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = keys[min(i + j * THREADS, m - 1)];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j * THREADS < m) slice_keys[i + j * THREADS] = x[j];
        }
        keys = slice_keys;
    }
    for (int i = tid + THREADS; i < (pages + 15) / 16; i += THREADS) top = max(top, p.tops[(size_t)bh * max_tiles + i]);
    top = __reduce_max_sync(~0u, top);
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(~0u, lane < kWarps ? warp_top[lane] : 0u);
    const Cut<uint32_t> cut = row_cut<uint32_t, THREADS, LONE>(keys, m, take, kTaken32, cut_shared.approx);

    // Pages above `in` are taken and pages below `out` are not, whatever the
    // error; without a finite one (infinities, NaN) every page is in question.
    float sum = lane < p.group ? head_sum[lane] : 0.f;
    const bool odd = __any_sync(~0u, !isfinite(sum));
#pragma unroll
    for (int o = 16; o; o >>= 1) sum = fmaxf(sum, __shfl_xor_sync(~0u, sum, o));
    const float most = floats_of<F16>(top).x * sum;
    uint32_t in = kTaken32 - 1, out = 1;
    if (cut.lo == kTaken32) {
        out = kTaken32;  // the forced pages are all
    } else if (!odd && isfinite(most)) {
        const float error = kScoreError<D> * most + kTiny;
        const float high = value_of(cut.hi), low = value_of(cut.lo);
        // Keys up to that of -infinity are no numbers: pages that are not in the pool.
        if (cut.hi <= kKeyMinusInf) in = cut.hi;
        else if (cut.hi < kKeyInf) in = key32_of(high + 2.f * error + fabsf(high) * 0x1p-22f);
        if (cut.lo > kKeyMinusInf) out = key32_of(low - 2.f * error - fabsf(low) * 0x1p-22f);
    }
    // A warp's run of the slice, in page order.
    const int run = ((m + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int i0 = min(m, warp * run), i1 = min(m, i0 + run);
    const uint32_t below = (1u << lane) - 1;
    int above = 0, at_cut = 0, above_all, cut_all;
    for (int i = i0; i < i1; i += 32) {
        const uint32_t k = i + lane < i1 ? keys[i + lane] : 0;
        above += __popc(__ballot_sync(~0u, k > in));
        at_cut += __popc(__ballot_sync(~0u, k >= out && k <= in));
    }
    int above_at = warps_before<THREADS>(above, slots, &above_all);
    int cut_at = warps_before<THREADS>(at_cut, slots, &cut_all);
    const int2 before = row_before<LONE>(make_int2(above_all, cut_all), rank_slots[0]);
    above_at += before.x;
    cut_at += before.y;
    // The row's totals: every rank's pair is in the slots.
    const int2 each = lane < ranks ? rank_slots[0][lane] : make_int2(0, 0);
    const int row_above = __reduce_add_sync(~0u, each.x), row_close = __reduce_add_sync(~0u, each.y);
    const int want = take - row_above;

    if (want == row_close || want <= 0) {
        // Nothing at the cut is left out (or, with forced pages alone, taken).
        int place = above_at + (want > 0 ? cut_at : 0);
        const uint32_t least = want > 0 ? out : in + 1;
        for (int i = i0; i < i1; i += 32) {
            const uint32_t mask = __ballot_sync(~0u, i + lane < i1 && keys[i + lane] >= least);
            if (mask >> lane & 1) to[place + __popc(mask & below)] = p0 + i + lane;
            place += __popc(mask);
        }
        return;
    }
    if (row_close <= kMaxClose) {
        // Every rank gets the exact scores of the few pages at the cut and ranks them itself.
        int at = cut_at;
        for (int i = i0; i < i1; i += 32) {
            const uint32_t k = i + lane < i1 ? keys[i + lane] : 0;
            const uint32_t mask = __ballot_sync(~0u, k >= out && k <= in);
            if (mask >> lane & 1) close_page[at + __popc(mask & below)] = p0 + i + lane;
            at += __popc(mask);
        }
        __syncthreads();
        for (int i = before.y + warp; i < before.y + cut_all; i += kWarps) {
            const int lp = close_page[i], page = table[lp].x;
            const uint64_t key = page < 0 || page >= v.pool_pages ? 1 : exact_key<F16, D>(p, h, page, queries);
            if (lane < ranks) {
                Close* remote = at_rank<LONE>(close, lane);
                remote[i].key = key;
                remote[i].page = lp;
            }
        }
        row_sync<LONE>();
        // keys at the cut become 0 (left out) or kTaken32.
        for (int i = tid; i < row_close; i += THREADS) {
            const Close mine = close[i];
            int better = 0;
            for (int j = 0; j < row_close; ++j)
                better += close[j].key > mine.key || (close[j].key == mine.key && close[j].page < mine.page);
            close_page[i] = better < want;
            if (mine.page >= p0 && mine.page < p0 + m) keys[mine.page - p0] = better < want ? kTaken32 : 0;
        }
        __syncthreads();
        int place = above_at;
        for (int i = 0; i < cut_at; ++i) place += close_page[i];
        for (int i = i0; i < i1; i += 32) {
            const uint32_t mask = __ballot_sync(~0u, i + lane < i1 && keys[i + lane] > in);
            if (mask >> lane & 1) to[place + __popc(mask & below)] = p0 + i + lane;
            place += __popc(mask);
        }
        return;
    }
    // Many pages at the cut: the cut again, over their exact scores.
    uint64_t* exact = p.exact + (size_t)bh * v.table_pages + p0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t k = keys[i];
        uint64_t key = k > in ? kTaken : 0;
        if (k >= out && k <= in) {
            const int page = table[p0 + i].x;
            key = page < 0 || page >= v.pool_pages ? 1 : exact_key<F16, D>(p, h, page, queries);
        }
        if (lane == 0) exact[i] = key;
    }
    __syncthreads();
    const Cut<uint64_t> fine = row_cut<uint64_t, THREADS, LONE>(exact, m, take, kTaken, cut_shared.exact);
    int equal = 0;  // keys of the cut's range before this run
    if (fine.partial) {
        int mine = 0, all;
        for (int i = i0 + lane; i < i1; i += 32) mine += exact[i] >= fine.lo && exact[i] <= fine.hi;
        equal = warps_before<THREADS>(__reduce_add_sync(~0u, mine), slots, &all);
        equal += row_before<LONE>(make_int2(all, 0), rank_slots[1]).x;
    }
    auto kept_mask = [&](int i, int* seen_equal) {
        const uint64_t k = i < i1 ? exact[i] : 0;
        const bool tied = i < i1 && k >= fine.lo && k <= fine.hi;
        bool kept = i < i1 && (k > fine.hi || tied);
        if (fine.partial) {
            const uint32_t mask = __ballot_sync(~0u, tied);
            if (tied) kept = *seen_equal + __popc(mask & below) < fine.ties;
            *seen_equal += __popc(mask);
        }
        return __ballot_sync(~0u, kept);
    };
    int count = 0, at = equal, all;
    for (int i = i0; i < i1; i += 32) count += __popc(kept_mask(i + lane, &at));
    int place = warps_before<THREADS>(count, slots, &all);
    place += row_before<LONE>(make_int2(all, 0), rank_slots[2]).x;
    at = equal;
    for (int i = i0; i < i1; i += 32) {
        const uint32_t mask = kept_mask(i + lane, &at);
        if (mask >> lane & 1) to[place + __popc(mask & below)] = p0 + i + lane;
        place += __popc(mask);
    }
}

template <typename F>
cudaError_t by_type(const BatchView& v, F f) {
    if (v.f16) return v.dim == 64 ? f.template operator()<true, 64>() : v.dim == 128 ? f.template operator()<true, 128>()
                                                                                  : f.template operator()<true, 256>();
    return v.dim == 64 ? f.template operator()<false, 64>() : v.dim == 128 ? f.template operator()<false, 128>()
                                                                          : f.template operator()<false, 256>();
}

struct LaunchBounds {
    BoundsParams p;
    cudaStream_t stream;
    template <bool F16, int D>
    cudaError_t operator()() const {
        // From a start on, the pages of a step or a chunk: a CTA per SM, so that the
        // kernel behind finds room beside them (a sparse step of 32k tokens waited
        // 1.5 us for four). From 0 on, all the SMs hold.
        const int64_t per_page = (int64_t)p.v.hkv * (D / 8) * 2, pages = p.start ? 4 : p.v.table_pages;
        const int64_t most = (p.v.batch * pages * per_page + kBoundsThreads - 1) / kBoundsThreads;
        const int64_t ctas = std::min<int64_t>(p.start ? std::max<int64_t>(most, p.v.sms) : most, p.v.sms * kBoundsCtas);
        return launch_dependent(page_bounds_kernel<F16, D>, dim3((unsigned)ctas), dim3(kBoundsThreads),
                                sizeof(int) * (size_t)(p.v.batch + 1), stream, p);
    }
};
struct SelectSpace {
    int cluster, threads;
    bool spill;
    size_t slice, tops, all;
};
SelectSpace select_space(const BatchView& v) {
    const size_t rows = (size_t)v.batch * v.hkv, pages = (size_t)v.table_pages;
    SelectSpace s;
    // A lone CTA while its slice fits: barriers of a cluster cost more than the keys it saves.
    s.cluster = 1;
    while (s.cluster < kMaxCluster && (pages + s.cluster - 1) / s.cluster > kMaxSlice) s.cluster *= 2;
    s.slice = ((pages + s.cluster - 1) / s.cluster + 31) / 32 * 32;
    s.spill = s.slice > kMaxSlice;
    // Barriers of 32 warps against passes over more keys a thread. Selecting for
    // one sequence (8 kv heads of 128) with 512 and with 1024 threads: 1024 pages
    // 10.5 and 11.1 us, 2049 12.4 and 12.9, 3000 14.4 and 13.3, 4000 15.3 and 13.8,
    // 8000 21.7 and 17.8. (With four sequences or more 1024 threads lead from 1024
    // pages on, by 3 to 6 % up to 3000.)
    s.threads = s.slice > 2560 ? 1024 : 512;
    const size_t approx = rows * pages * sizeof(uint64_t);
    s.tops = approx + rows * pages * sizeof(uint32_t);
    s.all = s.tops + rows * ((pages + 15) / 16) * sizeof(uint32_t);
    return s;
}

struct LaunchSelect {
    SelectParams p;
    SelectSpace s;
    cudaStream_t stream;
    template <bool F16, int D>
    cudaError_t operator()() const {
        const int ctas = D <= 128 && p.group <= 8 ? 2 : 1;  // of an SM
        SelectParams q = p;
        q.workers = p.v.sms * ctas * p.lanes;
        const size_t base = sizeof(int) * (size_t)(p.v.batch + 1);
        const dim3 grid(p.v.sms * ctas), block(kScoreWarps * 32);
        cudaError_t e = p.group > 8 ? launch_dependent(page_score_kernel<F16, D, 2>, grid, block, base, stream, q)
                                    : launch_dependent(page_score_kernel<F16, D, 1>, grid, block, base, stream, q);
        if (e != cudaSuccess) return e;
        auto* pick = s.cluster > 1 ? page_pick_kernel<F16, D, false, 1024>
                     : s.threads == 1024 ? page_pick_kernel<F16, D, true, 1024>
                                         : page_pick_kernel<F16, D, true, 512>;
        return launch_cluster(pick, (unsigned)(p.v.batch * p.v.hkv), s.cluster, s.threads,
                              sizeof(float) * p.group * D + (s.spill ? 0 : s.slice * sizeof(uint32_t)), stream, q);
    }
};
struct ConfigureSelect {
    template <bool F16, int D>
    cudaError_t operator()() const {
        constexpr size_t kMost = kMaxSlice * sizeof(uint32_t) + sizeof(float) * kMaxBatchGroup * D;
        cudaError_t e = configure_kernel(page_pick_kernel<F16, D, true, 512>, kMost);
        if (e == cudaSuccess) e = configure_kernel(page_pick_kernel<F16, D, true, 1024>, kMost);
        return e != cudaSuccess ? e : configure_kernel(page_pick_kernel<F16, D, false, 1024>, kMost);
    }
};

}  // namespace

cudaError_t launch_page_bounds(const BatchView& v, const int32_t* start, int32_t extra, uint16_t* bounds,
                               cudaStream_t stream) {
    return by_type(v, LaunchBounds{BoundsParams{v, start, bounds, extra}, stream});
}

size_t select_bytes(const BatchView& v) { return select_space(v).all; }

cudaError_t configure_select() {
    for (int f16 = 0; f16 < 2; ++f16)
        for (int dim = 64; dim <= 256; dim *= 2) {
            BatchView v{};
            v.f16 = f16;
            v.dim = dim;
            const cudaError_t e = by_type(v, ConfigureSelect{});
            if (e != cudaSuccess) return e;
        }
    return cudaSuccess;
}

cudaError_t launch_select_pages(const BatchView& v, const SelectLaunch& s, cudaStream_t stream) {
    const SelectSpace space = select_space(v);
    char* w = static_cast<char*>(s.workspace);
    SelectParams p;
    p.v = v;
    p.s = s;
    p.group = s.n_q_heads / v.hkv;
    p.groups = (v.hkv + kScoreWarps - 1) / kScoreWarps;
    p.heads = (v.hkv + p.groups - 1) / p.groups;
    p.lanes = kScoreWarps / p.heads;
    p.workers = 0;
    p.exact = reinterpret_cast<uint64_t*>(w);
    p.approx = reinterpret_cast<uint32_t*>(w + (size_t)v.batch * v.hkv * v.table_pages * sizeof(uint64_t));
    p.tops = reinterpret_cast<uint32_t*>(w + space.tops);
    p.spill = space.spill;
    return by_type(v, LaunchSelect{p, space, stream});
}

}  // namespace gkv
