// batch_pages.cu — per-page key bounds, and the pages they rank highest.
//
// Bounds: for a page's keys k_t (t its valid rows), lo_d = min_t k_td and
// hi_d = max_t k_td, exact in the keys' own type. For any query q and key of
// the page, q.k <= u(q) = sum_d (q_d >= 0 ? q_d hi_d : q_d lo_d).
// Selection: per kv head the pages with the largest max_g u(q_g). The order
// of two pages hangs on the last bits of their sums, so these are formed in
// fp64 (a product of two 16-bit floats is exact in it); the result is then the
// same for any order of summation, up to 2^-52.
#include "batch.cuh"

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
    uint64_t* keys;  // [batch][hkv][table_pages]
};

// Scores as integers of the same order; a page taken in any case comes before
// every score, a NaN before every number.
constexpr uint64_t kTaken = ~0ull, kNaN = ~0ull - 1;
__device__ __forceinline__ uint64_t key_of(double x) {
    if (x != x) return kNaN;
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 becomes 0
    return u >> 63 ? ~u : u | (1ull << 63);
}

constexpr int kScoreThreads = 256;

template <bool F16, int D>
__global__ void __launch_bounds__(kScoreThreads) page_score_kernel(const SelectParams p) {
    constexpr int kPer = D / 32;  // dims of a lane
    extern __shared__ int base[];
    __shared__ int warp_sums[32];
    pdl_trigger();
    pdl_wait();
    const BatchView& v = p.v;
    scan_counts(v.batch, base, warp_sums, [&](int b) { return pages_of(tokens_of(v, b, p.s.extra, blockIdx.x == 0)); });
    const int lane = threadIdx.x & 31;
    const int64_t total = (int64_t)base[v.batch] * v.hkv;
    const int warps = gridDim.x * (kScoreThreads / 32);
    for (int64_t w = blockIdx.x * (kScoreThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
        const int u = (int)(w / v.hkv), h = (int)(w % v.hkv);
        const int b = owner(base, v.batch, 1, u);
        const int lp = u - base[b], pages = base[b + 1] - base[b];
        uint64_t key;
        const int page = v.table[b * v.table_stride + lp].x;
        if (lp < p.s.n_first || lp >= pages - p.s.n_last) {
            key = kTaken;
        } else if (page < 0 || page >= v.pool_pages) {
            if (lane == 0) atomicOr(v.err, kErrBadPage);
            key = 0;
        } else {
            const uint16_t* lo = p.s.bounds + ((size_t)page * v.hkv + h) * 2 * D + lane * kPer;
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
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                nan |= sum != sum;
                best = fmax(best, sum);
            }
            key = nan ? kNaN : key_of(best);
        }
        if (lane == 0) p.keys[((size_t)b * v.hkv + h) * v.table_pages + lp] = key;
    }
}

constexpr int kPickThreads = 512;

// The n_pages largest keys of one (sequence, head), equal ones by the lower
// index: the smallest taken key byte by byte from the top (a histogram of the
// keys that agree so far), then the indices in rising order.
__global__ void __launch_bounds__(kPickThreads) page_pick_kernel(const SelectParams p) {
    __shared__ int hist[256];
    __shared__ int found[2];
    __shared__ int warp_sums[2][kPickThreads / 32];
    pdl_wait();
    pdl_trigger();
    const BatchView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bh = blockIdx.x, b = bh / v.hkv;
    if (v.lens[b] < 0) return;
    const int pages = pages_of(tokens_of(v, b, p.s.extra, false));
    int32_t* to = p.s.pages + (size_t)bh * p.s.n_pages;
    const int take = min(p.s.n_pages, pages);
    for (int i = take + tid; i < p.s.n_pages; i += kPickThreads) to[i] = -1;
    if (pages <= p.s.n_pages) {
        for (int i = tid; i < pages; i += kPickThreads) to[i] = i;
        return;
    }
    const uint64_t* keys = p.keys + (size_t)bh * v.table_pages;
    uint64_t prefix = 0;
    int want = take;  // of the keys that agree with the prefix so far
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kPickThreads) hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < pages; i += kPickThreads) {
            const uint64_t k = keys[i];
            if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int left = want, d = 255;
            while (d > 0 && hist[d] < left) left -= hist[d--];
            found[0] = d;
            found[1] = left;
        }
        __syncthreads();
        prefix |= (uint64_t)found[0] << shift;
        want = found[1];
        __syncthreads();
    }
    // `want` keys equal to the prefix are taken, and all above it.
    int written = 0, equal = 0;
    for (int i0 = 0; i0 < pages; i0 += kPickThreads) {
        const int i = i0 + tid;
        const uint64_t k = i < pages ? keys[i] : 0;
        const bool above = i < pages && k > prefix, same = i < pages && k == prefix;
        const uint32_t same_mask = __ballot_sync(0xFFFFFFFFu, same), above_mask = __ballot_sync(0xFFFFFFFFu, above);
        if (lane == 0) warp_sums[0][warp] = __popc(same_mask), warp_sums[1][warp] = __popc(above_mask);
        __syncthreads();
        int same_before = equal, above_before = 0, same_all = 0, above_all = 0;
        for (int w = 0; w < kPickThreads / 32; ++w) {
            if (w < warp) same_before += warp_sums[0][w], above_before += warp_sums[1][w];
            same_all += warp_sums[0][w], above_all += warp_sums[1][w];
        }
        same_before += __popc(same_mask & ((1u << lane) - 1));
        above_before += __popc(above_mask & ((1u << lane) - 1));
        // Taken before this one: the ones above, and the equal ones while they last.
        const int at = written + above_before + min(same_before, want) - min(equal, want);
        if (above || (same && same_before < want)) to[at] = i;
        written += above_all + min(equal + same_all, want) - min(equal, want);
        equal += same_all;
        __syncthreads();
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
struct LaunchScores {
    SelectParams p;
    cudaStream_t stream;
    template <bool F16, int D>
    cudaError_t operator()() const {
        return launch_dependent(page_score_kernel<F16, D>, dim3(p.v.sms * 4), dim3(kScoreThreads),
                                sizeof(int) * (size_t)(p.v.batch + 1), stream, p);
    }
};

}  // namespace

cudaError_t launch_page_bounds(const BatchView& v, const int32_t* start, int32_t extra, uint16_t* bounds,
                               cudaStream_t stream) {
    return by_type(v, LaunchBounds{BoundsParams{v, start, bounds, extra}, stream});
}

size_t select_bytes(const BatchView& v) { return (size_t)v.batch * v.hkv * v.table_pages * sizeof(uint64_t); }

cudaError_t configure_select() { return cudaSuccess; }

cudaError_t launch_select_pages(const BatchView& v, const SelectLaunch& s, cudaStream_t stream) {
    const SelectParams p{v, s, s.n_q_heads / v.hkv, static_cast<uint64_t*>(s.workspace)};
    cudaError_t e = by_type(v, LaunchScores{p, stream});
    if (e != cudaSuccess) return e;
    return launch_dependent(page_pick_kernel, dim3(v.batch * v.hkv), dim3(kPickThreads), 0, stream, p);
}

}  // namespace gkv
