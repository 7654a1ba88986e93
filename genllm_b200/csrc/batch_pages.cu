// batch_pages.cu — per-page key bounds, and the pages they rank highest.
//
// Bounds: for a page's keys k_t (t its valid rows), lo_d = min_t k_td and
// hi_d = max_t k_td, exact in the keys' own type. For any query q and key of
// the page, q.k <= u(q) = sum_d (q_d >= 0 ? q_d hi_d : q_d lo_d).
// Selection: per kv head the pages with the largest max_g u(q_g), in the order
// of their values in 64 bits. u = hi.max(q, 0) + lo.min(q, 0) is a product of
// 16-bit matrices, so the tensor cores give every score to within E; only
// pages within 2 E of the cut can be misplaced by that, and these alone are
// summed again in fp64 (in which products of 16-bit floats are exact). All
// pages in fp64 took 87 us on 213 thousand tokens of 8 sequences, of which the
// bounds' bytes are 8.
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

constexpr int kBoundsThreads = 256;

// One warp per (page, head): the page's rows of one head, 16 bytes a lane.
template <bool F16, int D>
__global__ void __launch_bounds__(kBoundsThreads) page_bounds_kernel(const BoundsParams p) {
    constexpr int kChunks = D / 8, kRows = 32 / kChunks;
    extern __shared__ int base[];
    __shared__ int warp_sums[32];
    pdl_wait();
    pdl_trigger();
    const BatchView& v = p.v;
    auto first_page = [&](int b) { return p.start ? max(0, p.start[b]) / kPageSlots : 0; };
    scan_counts(v.batch, base, warp_sums, [&](int b) {
        return max(0, pages_of(tokens_of(v, b, p.extra, blockIdx.x == 0)) - first_page(b));
    });
    const int lane = threadIdx.x & 31;
    const int c16 = lane % kChunks, r0 = lane / kChunks;
    const int64_t total = (int64_t)base[v.batch] * v.hkv;
    const int warps = gridDim.x * (kBoundsThreads / 32);
    constexpr uint32_t kInf = F16 ? 0x7C007C00u : 0x7F807F80u;
    for (int64_t w = blockIdx.x * (kBoundsThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
        const int u = (int)(w / v.hkv), h = (int)(w % v.hkv);
        const int b = owner(base, v.batch, 1, u);
        const int lp = first_page(b) + (u - base[b]);
        const int valid = min(kPageSlots, tokens_of(v, b, p.extra, false) - lp * kPageSlots);
        const int page = v.table[b * v.table_stride + lp].x;
        if (page < 0 || page >= v.pool_pages) {
            if (lane == 0) atomicOr(v.err, kErrBadPage);
            continue;
        }
        const uint16_t* row = v.k_base + ((size_t)page * kPageSlots * v.hkv + h) * D + c16 * 8;
        uint4 x[kPageSlots / kRows];
#pragma unroll
        for (int i = 0; i < kPageSlots / kRows; ++i) {
            const int r = i * kRows + r0;
            // Rows behind the sequence stand for its first row, which is valid.
            x[i] = *reinterpret_cast<const uint4*>(row + (size_t)(r < valid ? r : 0) * v.hkv * D);
        }
        uint4 lo = make_uint4(kInf, kInf, kInf, kInf), hi;
        hi = make_uint4(lo.x | 0x80008000u, lo.y | 0x80008000u, lo.z | 0x80008000u, lo.w | 0x80008000u);
#pragma unroll
        for (int i = 0; i < kPageSlots / kRows; ++i) {
            lo.x = min2_nan<F16>(lo.x, x[i].x), hi.x = max2_nan<F16>(hi.x, x[i].x);
            lo.y = min2_nan<F16>(lo.y, x[i].y), hi.y = max2_nan<F16>(hi.y, x[i].y);
            lo.z = min2_nan<F16>(lo.z, x[i].z), hi.z = max2_nan<F16>(hi.z, x[i].z);
            lo.w = min2_nan<F16>(lo.w, x[i].w), hi.w = max2_nan<F16>(hi.w, x[i].w);
        }
#pragma unroll
        for (int o = kChunks; o < 32; o <<= 1) {
            lo.x = min2_nan<F16>(lo.x, __shfl_xor_sync(~0u, lo.x, o)), hi.x = max2_nan<F16>(hi.x, __shfl_xor_sync(~0u, hi.x, o));
            lo.y = min2_nan<F16>(lo.y, __shfl_xor_sync(~0u, lo.y, o)), hi.y = max2_nan<F16>(hi.y, __shfl_xor_sync(~0u, hi.y, o));
            lo.z = min2_nan<F16>(lo.z, __shfl_xor_sync(~0u, lo.z, o)), hi.z = max2_nan<F16>(hi.z, __shfl_xor_sync(~0u, hi.z, o));
            lo.w = min2_nan<F16>(lo.w, __shfl_xor_sync(~0u, lo.w, o)), hi.w = max2_nan<F16>(hi.w, __shfl_xor_sync(~0u, hi.w, o));
        }
        uint4* to = reinterpret_cast<uint4*>(p.bounds + ((size_t)page * v.hkv + h) * 2 * D) + c16;
        if (r0 == 0) to[0] = lo;
        if (r0 == kRows - 1) to[kChunks] = hi;
    }
}

struct SelectParams {
    BatchView v;
    SelectLaunch s;
    int32_t group;
    uint64_t* exact;   // [batch][hkv][table_pages], where many pages lie at the cut
    uint32_t* approx;  // [batch][hkv][table_pages] where a slice does not fit in shared memory; else null
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

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMaxSlice = 32768;  // keys of a CTA in shared memory: 128 KB
constexpr int kMaxClose = 64;     // pages at the cut that are ranked in shared memory

// E of the tensor cores' score, relative to max |bound| * sum |q|: each of the
// D / 8 products of 16 steps adds 17 numbers, aligned to 24 bits of the largest
// (2^-23 of it each) and rounded; twice that is taken. kTiny: what products
// below fp32's normal range may lose.
template <int D>
constexpr float kScoreError = 2 * (D / 8) * 18 * 0x1p-23f;
constexpr float kTiny = 0x1p-117f;
constexpr uint32_t kKeyInf = 0xFF800000u, kKeyMinusInf = 0x007FFFFFu;  // key32_of the infinities

// The score of one page in fp64, by a whole warp.
template <bool F16, int D>
__device__ uint64_t exact_key(const SelectParams& p, int b, int h, int page) {
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
    for (int g = 0; g < p.group; ++g) {
        const uint16_t* q = p.s.q + b * p.s.q_stride_batch + (int64_t)(h * p.group + g) * p.s.q_stride_head + lane * kPer;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
            const float2 a = floats_of<F16>(*reinterpret_cast<const uint32_t*>(q + i));
            sum += (double)a.x * (double)(a.x >= 0.f ? x[i] : l[i]);
            sum += (double)a.y * (double)(a.y >= 0.f ? x[i + 1] : l[i + 1]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        nan |= sum != sum;
        best = fmax(best, sum);
    }
    return nan ? kNaN : key_of(best);
}

// One cluster per (sequence, head), a slice of its pages per CTA.
template <bool F16, int D, int NT>
__global__ void __launch_bounds__(kSelectThreads, 2) page_select_kernel(const SelectParams p) {
    namespace cg = cooperative_groups;
    constexpr int kLoads = D / 32;  // 16-byte chunks of a lane's row, of either bound
    struct Close {
        uint64_t key;
        int page;
    };
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ CutShared<uint32_t, kSelectThreads> cut_shared;
    __shared__ CutShared<uint64_t, kSelectThreads> exact_shared;
    __shared__ Close close[kMaxClose];
    __shared__ int close_page[kMaxClose];
    __shared__ int slots[kSelectWarps];
    __shared__ int2 rank_slots[3][kMaxCluster];
    __shared__ uint32_t warp_top[kSelectWarps];
    __shared__ float head_sum[kMaxBatchGroup];
    pdl_wait();
    pdl_trigger();
    cg::cluster_group cluster = cg::this_cluster();
    const BatchView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int bh = blockIdx.x / ranks, b = bh / v.hkv, h = bh % v.hkv;
    if (v.lens[b] < 0) return;  // the whole cluster
    const int pages = pages_of(tokens_of(v, b, p.s.extra, rank == 0 && tid == 0));
    int32_t* to = p.s.pages + (size_t)bh * p.s.n_pages;
    const int take = min(p.s.n_pages, pages);
    for (int i = take + rank * kSelectThreads + tid; i < p.s.n_pages; i += ranks * kSelectThreads) to[i] = -1;
    if (pages <= p.s.n_pages) {
        for (int i = rank * kSelectThreads + tid; i < pages; i += ranks * kSelectThreads) to[i] = i;
        return;  // the whole cluster
    }
    const int slice = ((pages + ranks - 1) / ranks + 31) / 32 * 32;
    const int p0 = min(pages, rank * slice), m = min(pages - p0, slice);
    const int2* table = v.table + b * v.table_stride;

    // Queries as B fragments: step k of the product takes two pairs of dims of
    // the 16-byte chunk that a lane loads of a page's row, so rows go from
    // memory to the A fragment as they are. First max(q, 0) (for hi), then min.
    uint2* frag = reinterpret_cast<uint2*>(smem);  // [2][kLoads][2][NT][32]
    constexpr int kFrags = 2 * kLoads * 2 * NT * 32;
    for (int i = tid; i < kFrags; i += kSelectThreads) {
        const int l = i & 31, nt = i / 32 % NT, half = i / (32 * NT) % 2, k = i / (64 * NT) % kLoads, low = i / (64 * NT * kLoads);
        const int g = nt * 8 + (l >> 2);
        uint2 x = make_uint2(0, 0);
        if (g < p.group) {
            const uint16_t* row = p.s.q + b * p.s.q_stride_batch + (int64_t)(h * p.group + g) * p.s.q_stride_head;
            x = *reinterpret_cast<const uint2*>(row + (k * 4 + (l & 3)) * 8 + half * 4);
            auto part = [&](uint32_t w) {
                const uint32_t neg = ((w >> 15 & 1) * 0xFFFFu) | ((w >> 31) * 0xFFFF0000u);
                return w & (low ? neg : ~neg);
            };
            x.x = part(x.x);
            x.y = part(x.y);
        }
        frag[i] = x;
    }
    for (int g = warp; g < p.group; g += kSelectWarps) {
        float sum = 0.f;
        const uint16_t* row = p.s.q + b * p.s.q_stride_batch + (int64_t)(h * p.group + g) * p.s.q_stride_head;
        for (int d = lane; d < D; d += 32) sum += fabsf(floats_of<F16>(row[d]).x);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) head_sum[g] = sum;
    }
    uint32_t* keys = p.approx ? p.approx + (size_t)bh * v.table_pages + p0
                              : reinterpret_cast<uint32_t*>(smem + kFrags * sizeof(uint2));
    __syncthreads();

    // Sixteen pages a warp: this lane's rows are pages lane / 4 and lane / 4 + 8.
    const int quarter = lane & 3;
    uint32_t top = 0;  // largest |bound|, as bits
    for (int i0 = warp * 16; i0 < m; i0 += kSelectWarps * 16) {
        int page[2];
        bool bad[2];
        const uint4* row[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            page[r] = table[p0 + min(i0 + r * 8 + (lane >> 2), m - 1)].x;
            bad[r] = page[r] < 0 || page[r] >= v.pool_pages;
            row[r] = reinterpret_cast<const uint4*>(p.s.bounds + ((size_t)(bad[r] ? 0 : page[r]) * v.hkv + h) * 2 * D) + quarter;
        }
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
        for (int low = 0; low < 2; ++low) {
            uint4 x[2][kLoads];
#pragma unroll
            for (int k = 0; k < kLoads; ++k)
#pragma unroll
                for (int r = 0; r < 2; ++r) x[r][k] = row[r][k * 4 + (low ? 0 : D / 8)];
#pragma unroll
            for (int k = 0; k < kLoads; ++k) {
                const uint32_t a[2][4] = {{x[0][k].x, x[1][k].x, x[0][k].y, x[1][k].y},
                                          {x[0][k].z, x[1][k].z, x[0][k].w, x[1][k].w}};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    top = __vmaxu2(top, __vmaxu2(a[half][0] & 0x7FFF7FFFu, a[half][1] & 0x7FFF7FFFu));
                    top = __vmaxu2(top, __vmaxu2(a[half][2] & 0x7FFF7FFFu, a[half][3] & 0x7FFF7FFFu));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint2 f = frag[(((low * kLoads + k) * 2 + half) * NT + nt) * 32 + lane];
                        mma16816<F16>(c[nt], a[half], f.x, f.y);
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
            const int i = i0 + r * 8 + (lane >> 2), lp = p0 + i;
            if (quarter == 0 && i < m) {
                const bool taken = lp < p.s.n_first || lp >= pages - p.s.n_last;
                if (bad[r] && !taken) atomicOr(v.err, kErrBadPage);
                keys[i] = taken ? kTaken32 : bad[r] ? 1u : key32_of(best);
            }
        }
    }
    top = __reduce_max_sync(~0u, max(top & 0xFFFFu, top >> 16));
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(~0u, lane < kSelectWarps ? warp_top[lane] : 0u);
    const Cut<uint32_t> cut = cluster_cut<uint32_t, kSelectThreads>(keys, m, take, kTaken32, &top, cut_shared);

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
        if (cut.hi < kKeyInf) in = key32_of(high + 2.f * error + fabsf(high) * 0x1p-22f);
        if (cut.lo > kKeyMinusInf) out = key32_of(low - 2.f * error - fabsf(low) * 0x1p-22f);
    }
    // A warp's run of the slice, in page order.
    const int run = ((m + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32;
    const int i0 = min(m, warp * run), i1 = min(m, i0 + run);
    const uint32_t below = (1u << lane) - 1;
    int above = 0, at_cut = 0, above_all, cut_all;
    for (int i = i0; i < i1; i += 32) {
        const uint32_t k = i + lane < i1 ? keys[i + lane] : 0;
        above += __popc(__ballot_sync(~0u, k > in));
        at_cut += __popc(__ballot_sync(~0u, k >= out && k <= in));
    }
    int above_at = warps_before<kSelectThreads>(above, slots, &above_all);
    int cut_at = warps_before<kSelectThreads>(at_cut, slots, &cut_all);
    const int2 before = cluster_before(make_int2(above_all, cut_all), rank_slots[0]);
    above_at += before.x;
    cut_at += before.y;
    // The row's totals: every rank's pair is in the slots.
    const int2 each = lane < ranks ? rank_slots[0][lane] : make_int2(0, 0);
    const int row_above = __reduce_add_sync(~0u, each.x), row_cut = __reduce_add_sync(~0u, each.y);
    const int want = take - row_above;

    if (want == row_cut || want <= 0) {
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
    if (row_cut <= kMaxClose) {
        // Every rank gets the exact scores of the few pages at the cut and ranks them itself.
        int at = cut_at;
        for (int i = i0; i < i1; i += 32) {
            const uint32_t k = i + lane < i1 ? keys[i + lane] : 0;
            const uint32_t mask = __ballot_sync(~0u, k >= out && k <= in);
            if (mask >> lane & 1) close_page[at + __popc(mask & below)] = p0 + i + lane;
            at += __popc(mask);
        }
        __syncthreads();
        for (int i = before.y + warp; i < before.y + cut_all; i += kSelectWarps) {
            const int lp = close_page[i], page = table[lp].x;
            const uint64_t key = page < 0 || page >= v.pool_pages ? 1 : exact_key<F16, D>(p, b, h, page);
            if (lane < ranks) {
                Close* remote = cluster.map_shared_rank(close, lane);
                remote[i].key = key;
                remote[i].page = lp;
            }
        }
        cluster.sync();
        // keys at the cut become 0 (left out) or kTaken32.
        for (int i = tid; i < row_cut; i += kSelectThreads) {
            const Close mine = close[i];
            int better = 0;
            for (int j = 0; j < row_cut; ++j)
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
            key = page < 0 || page >= v.pool_pages ? 1 : exact_key<F16, D>(p, b, h, page);
        }
        if (lane == 0) exact[i] = key;
    }
    __syncthreads();
    uint32_t unused = 0;
    const Cut<uint64_t> fine = cluster_cut<uint64_t, kSelectThreads>(exact, m, take, kTaken, &unused, exact_shared);
    int equal = 0;  // keys of the cut's range before this run
    if (fine.partial) {
        int mine = 0, all;
        for (int i = i0 + lane; i < i1; i += 32) mine += exact[i] >= fine.lo && exact[i] <= fine.hi;
        equal = warps_before<kSelectThreads>(__reduce_add_sync(~0u, mine), slots, &all);
        equal += cluster_before(make_int2(all, 0), rank_slots[1]).x;
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
    int place = warps_before<kSelectThreads>(count, slots, &all);
    place += cluster_before(make_int2(all, 0), rank_slots[2]).x;
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
        return launch_dependent(page_bounds_kernel<F16, D>, dim3(p.v.sms * 4), dim3(kBoundsThreads),
                                sizeof(int) * (size_t)(p.v.batch + 1), stream, p);
    }
};
struct SelectSpace {
    int cluster;
    bool spill;  // approximate keys in the workspace
    size_t slice, approx, all;
};
SelectSpace select_space(const BatchView& v) {
    const size_t rows = (size_t)v.batch * v.hkv;
    SelectSpace s;
    s.cluster = cluster_for((int)rows, v.table_pages, v.sms, 128, kMaxSlice);
    s.slice = (((size_t)v.table_pages + s.cluster - 1) / s.cluster + 31) / 32 * 32;
    s.spill = s.slice > kMaxSlice;
    s.approx = rows * v.table_pages * sizeof(uint64_t);
    s.all = s.approx + (s.spill ? rows * v.table_pages * sizeof(uint32_t) : 0);
    return s;
}

size_t frag_bytes(int dim, int tiles) { return (size_t)2 * (dim / 32) * 2 * tiles * 32 * sizeof(uint2); }

struct LaunchSelect {
    SelectParams p;
    SelectSpace s;
    cudaStream_t stream;
    template <bool F16, int D>
    cudaError_t operator()() const {
        const int tiles = p.group > 8 ? 2 : 1;
        const size_t smem = frag_bytes(D, tiles) + (s.spill ? 0 : s.slice * sizeof(uint32_t));
        return launch_cluster(tiles == 2 ? page_select_kernel<F16, D, 2> : page_select_kernel<F16, D, 1>,
                              (unsigned)(p.v.batch * p.v.hkv), s.cluster, kSelectThreads, smem, stream, p);
    }
};
struct ConfigureSelect {
    template <bool F16, int D>
    cudaError_t operator()() const {
        const int most = (int)(frag_bytes(D, 2) + kMaxSlice * sizeof(uint32_t));
        cudaError_t e = cudaFuncSetAttribute(page_select_kernel<F16, D, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(page_select_kernel<F16, D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        return e;
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
    const SelectParams p{v, s, s.n_q_heads / v.hkv, reinterpret_cast<uint64_t*>(w),
                         space.spill ? reinterpret_cast<uint32_t*>(w + space.approx) : nullptr};
    return by_type(v, LaunchSelect{p, space, stream});
}

}  // namespace gkv
