// batch_decode.cu — attention of one new token for each of many sequences over
// a paged cache, split over the pages and joined.
//
// For sequence b and query head q of kv head h, over the attended tokens t:
//   s_t = scale * q.k_t,  out = sum_t exp(s_t - lse) v_t,  lse = ln sum_t exp(s_t),
// in one pass over K and V with the running maximum and sum (fp32, in log2
// units); a sequence cut into several parts leaves (maximum, sum, un-normalised
// output) of each part in the workspace, joined in order by the second kernel.
//
// Work: the pages of all sequences form one line of units (x head groups); a
// worker takes an equal, contiguous part of it, whatever the lengths are, so
// ragged batches load every SM alike. It has at most two parts that other
// workers continue (its first and its last); what lies between it finishes
// itself. Bound: HBM (K and V once); a worker is one warp per kv head of a
// group, so that a page's [16][Hkv][D] bytes are read together.
//
// One unit is 16 keys of one head: S^T = K Q^T (M 16 keys, N 8 query heads)
// and O^T += V^T P^T (M 16 dims) on mma.sync, the keys' rows coming through a
// per-warp cp.async ring, 16-byte chunks XOR-permuted by row for ldmatrix.
// mma.sync and not tcgen05: at 16 query heads or fewer the products are far
// below the stream of K and V in cost, and each warp works without barriers.
//
// Measured (8 kv heads of 128, 32 query heads, bf16), a step with its join: 328 MB
// of 64 ragged sequences in 57.9 to 61.5 us (by GPU), 134 MB of one of 32768 tokens
// in 27.1, of which 2.5 pass before the first page is there; 1024 tokens with 16
// query heads in 8.6.
#include <algorithm>

#include "batch.cuh"

namespace gkv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr int kMaxGrid = 160;  // bounds the parts of a sequence: kMaxGrid workers times 8 to a CTA
constexpr int kRingBytes = 192 * 1024;
constexpr int kRingAlign = 512;  // the longest row: chunk offsets in a row are XORs of its address

struct DecodeParams {
    BatchView v;
    BatchDecodeLaunch d;
    BatchSplit s;
    int32_t group;       // query heads per kv head
    float scale_log2;
    float* part_acc;     // [2 workers][heads * group][D]
    float2* part_ml;     // [2 workers][heads * group] (maximum in log2 units, sum)
    float* lse2;         // [batch][Hq] log2 of the sum, for the totals: -inf without a key, NaN if all scores were -inf
    float* scores;       // [unit][16][group] scores in log2 units, for the totals; or null
};

__device__ __forceinline__ float exp2_of(float x) { return exp2_approx(x); }

// Tokens sequence b attends (with the new one), 0 for a skipped sequence;
// flags a length its table row cannot hold and leaves out what lies behind.
__device__ __forceinline__ int attended(const BatchView& v, const BatchDecodeLaunch& d, int b, bool flag) {
    const int len = v.lens[b];
    if (len < 0) return 0;
    const int cap = v.table_pages * kPageSlots;
    const int new_token = d.k_new ? 1 : 0;
    if (len > cap - new_token) {
        if (flag) atomicOr(v.err, kErrBadLength);
        return cap;
    }
    return len + new_token;
}

// Whether sequence b gains a token this step, and where.
__device__ __forceinline__ bool gains(const BatchView& v, const BatchDecodeLaunch& d, int b, int* pos) {
    const int len = v.lens[b];
    *pos = len;
    return d.k_new && len >= 0 && len < v.table_pages * kPageSlots;
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (F16) return __half22float2(*reinterpret_cast<__half2*>(&w));
    return make_float2(bf16_lo(w), bf16_hi(w));
}

// The leading 16-bit terms of two numbers, packed; x keeps what they leave.
// bf16 terms are cut off, not rounded: no conversion, and three of 8 bits are the
// 24 of an fp32 number.
template <bool F16>
__device__ __forceinline__ uint32_t take_term(float2& x) {
    float2 t;
    uint32_t r;
    if (F16) {
        r = pack2<F16>(x.x, x.y);
        t = unpack2<F16>(r);
    } else {
        r = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
        t = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xFFFF0000u), __uint_as_float(__float_as_uint(x.y) & 0xFFFF0000u));
    }
    x.x -= t.x;
    x.y -= t.y;
    return r;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// What a lane holds of one unit ahead of its loads. The ids stay unchecked
// until they are used, so that a load of 32 of them is not waited for.
struct Unit {
    int2 ids;
    int info;  // valid rows | kNewRow: the last of them is the new token | kv head << 16; 0: no page
};
constexpr int kNewRow = 1 << 8;

template <bool F16, int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) batch_decode_kernel(const DecodeParams p) {
    constexpr int kRow = D * 2;              // bytes of one head's row
    constexpr int kTile = kPageSlots * kRow;  // one unit's K (or V)
    constexpr int kStages = kRingBytes / (WARPS * 2 * kTile);
    constexpr int kChunks = kRow / 16;       // 16-byte chunks of a row
    constexpr int kRowsPerCopy = 32 / kChunks;
    constexpr int kCopies = kPageSlots / kRowsPerCopy;
    constexpr int kSteps = D / 16;
    constexpr int kTerms = F16 ? 2 : 3;  // of an attention weight
    // f16 steps by 2^-24 at its bottom: weights (at most 1) are taken times 2^15, so
    // that what two terms lose is 2^-40 of the part's largest, and not 2^-25. The
    // sums (l) hold the weights as they are. bf16 reaches as far down as fp32.
    constexpr float kLift = F16 ? 0x1p15f : 1.f;
    static_assert(kStages >= 2, "the ring holds one unit ahead");
    extern __shared__ uint8_t raw_smem[];
    uint8_t* smem = raw_smem + (kRingAlign - smem_addr(raw_smem) % kRingAlign) % kRingAlign;
    __shared__ int warp_sums[32];
    __shared__ int stage_info[WARPS][kStages];
    int* base = reinterpret_cast<int*>(smem + kRingBytes);

    const BatchView& v = p.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    // From here on the kernels behind may start: they read lengths and inputs
    // before this one is done, the workspace only after.
    pdl_trigger();

    const int n_list = p.d.pages ? p.d.n_pages : 0x7FFFFFFF;
    scan_counts(v.batch, base, warp_sums,
                [&](int b) { return min(n_list, pages_of(attended(v, p.d, b, blockIdx.x == 0))); });
    const int total = base[v.batch] * p.s.groups;
    const int per = max(1, (total + p.s.workers - 1) / p.s.workers);

    const int hq = p.d.n_q_heads;
    const int worker = blockIdx.x * p.s.lanes + warp / p.s.heads;
    const int head_in = warp % p.s.heads;
    // A worker without units still helps with the appends.
    const int64_t first = warp < p.s.lanes * p.s.heads ? min((int64_t)total, (int64_t)worker * per) : total;
    const int u0 = (int)first, u1 = (int)min((int64_t)total, first + per);

    const uint64_t policy = l2_policy_evict_first();
    uint8_t* ring = smem + warp * (kStages * 2 * kTile);
    const uint32_t ring_addr = smem_addr(ring);
    const size_t slot_stride = (size_t)v.hkv * D;

    // This lane's unit of the 32 from `from` on.
    auto fetch = [&](int from) {
        Unit n{make_int2(0, 0), 0};
        const int u = from + lane;
        if (u >= u1) return n;
        const int b = owner(base, v.batch, p.s.groups, u);
        const int count = base[b + 1] - base[b];
        const int r = u - base[b] * p.s.groups;
        const int grp = r / count, j = r - grp * count;
        const int h = grp * p.s.heads + head_in;
        if (h >= v.hkv) return n;
        const int tokens = attended(v, p.d, b, false);
        const int lp = p.d.pages ? p.d.pages[((size_t)b * v.hkv + h) * p.d.n_pages + j] : j;
        if (lp < 0 || lp >= pages_of(tokens)) return n;
        n.ids = v.table[b * v.table_stride + lp];
        n.info = min(kPageSlots, tokens - lp * kPageSlots) | h << 16;
        int pos;
        if (gains(v, p.d, b, &pos) && pos / kPageSlots == lp) n.info |= kNewRow;
        return n;
    };

    auto checked = [&](Unit n) {
        if (n.info && (min(n.ids.x, n.ids.y) < 0 || max(n.ids.x, n.ids.y) >= v.pool_pages)) {
            atomicOr(v.err, kErrBadPage);
            n.info = 0;
        }
        if (!n.info) n.ids = make_int2(0, 0);
        return n;
    };

    Unit cur = checked(fetch(u0)), next;
    int cur_from = u0;
    const int c16 = lane % kChunks, r0 = lane / kChunks;
    // This lane's 16 bytes of the first rows of a unit: in the page, and in the
    // ring, where row r holds chunk c at c ^ (r & 7).
    const uint32_t lane_src = (uint32_t)(r0 * v.hkv * kRow + c16 * 16);
    const uint32_t lane_dst = (uint32_t)(r0 * kRow + ((c16 ^ r0) << 4));
    const uint32_t row_step = (uint32_t)(kRowsPerCopy * v.hkv * kRow);
    int issue_at = 0, issue_stage = 0;  // units issued, and the stage of the next

    auto issue = [&]() {
        const int u = u0 + issue_at;
        if (u < u1) {
            if (u - cur_from >= 32) {
                cur = checked(next);
                cur_from += 32;
                next = fetch(cur_from + 32);
            }
            const int from = u - cur_from;
            const int k_id = __shfl_sync(0xFFFFFFFFu, cur.ids.x, from), v_id = __shfl_sync(0xFFFFFFFFu, cur.ids.y, from);
            const int info = __shfl_sync(0xFFFFFFFFu, cur.info, from);
            const int h = info >> 16, valid = info & 0xFF;
            if (lane == 0) stage_info[warp][issue_stage] = valid;
            const uint32_t dst = ring_addr + issue_stage * (2 * kTile) + lane_dst;
            const char* k = reinterpret_cast<const char*>(v.k_base) + ((size_t)k_id * (kPageSlots * v.hkv) + h) * kRow + lane_src;
            const char* vv = reinterpret_cast<const char*>(v.v_base) + ((size_t)v_id * (kPageSlots * v.hkv) + h) * kRow + lane_src;
            if ((info & 0xFFFF) == kPageSlots) {
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const uint32_t to = (dst ^ (((i * kRowsPerCopy) & 7) << 4)) + i * (kRowsPerCopy * kRow);
                    cp_async16(to, k + (size_t)i * row_step, 16u, policy);
                    cp_async16(to + kTile, vv + (size_t)i * row_step, 16u, policy);
                }
            } else {
                const int b = owner(base, v.batch, p.s.groups, u);
#pragma unroll 1
                for (int i = 0; i < kCopies; ++i) {
                    const int row = i * kRowsPerCopy + r0;
                    const uint32_t to = (dst ^ (((i * kRowsPerCopy) & 7) << 4)) + i * (kRowsPerCopy * kRow);
                    const void* ks = k + (size_t)i * row_step;
                    const void* vs = vv + (size_t)i * row_step;
                    if ((info & kNewRow) && row == valid - 1) {
                        ks = p.d.k_new + b * p.d.k_stride_batch + h * p.d.k_stride_head + c16 * 8;
                        vs = p.d.v_new + b * p.d.v_stride_batch + h * p.d.v_stride_head + c16 * 8;
                    }
                    // Rows behind the sequence become zeros: what the slots hold may be anything.
                    const uint32_t bytes = row < valid ? 16u : 0u;
                    cp_async16(to, ks, bytes, policy);
                    cp_async16(to + kTile, vs, bytes, policy);
                }
            }
            ++issue_at;
            if (++issue_stage == kStages) issue_stage = 0;
        }
        cp_async_commit();
    };

#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) issue();
    next = fetch(u0 + 32);

    for (int b = blockIdx.x; b < v.batch; b += gridDim.x) {
        // The new token's rows go to their page slot; its readers below take
        // them from the step's inputs, so neither waits for the other.
        int pos;
        if (gains(v, p.d, b, &pos)) {
            const int2 e = v.table[b * v.table_stride + pos / kPageSlots];
            const bool ok = e.x >= 0 && e.x < v.pool_pages && e.y >= 0 && e.y < v.pool_pages;
            if (!ok && tid == 0) atomicOr(v.err, kErrBadPage);
            for (int i = tid; ok && i < 2 * v.hkv * kChunks; i += blockDim.x) {
                const bool is_v = i >= v.hkv * kChunks;
                const int j = is_v ? i - v.hkv * kChunks : i, h = j / kChunks, c = j % kChunks;
                const uint16_t* src = is_v ? p.d.v_new + b * p.d.v_stride_batch + h * p.d.v_stride_head
                                           : p.d.k_new + b * p.d.k_stride_batch + h * p.d.k_stride_head;
                uint16_t* dst = (is_v ? v.v_base : v.k_base) +
                                (((size_t)(is_v ? e.y : e.x) * kPageSlots + pos % kPageSlots) * v.hkv + h) * D;
                reinterpret_cast<uint4*>(dst)[c] = reinterpret_cast<const uint4*>(src)[c];
            }
        }
        // Nothing to attend: zeros (a skipped sequence is left alone).
        if (v.lens[b] >= 0 && base[b + 1] == base[b]) {
            for (int i = tid; i < hq * D; i += blockDim.x) store_out(p.d.out, (size_t)b * hq * D + i, 0.f, p.d.out_dtype);
            for (int i = tid; i < hq; i += blockDim.x) {
                if (p.d.lse) p.d.lse[(size_t)b * hq + i] = -INFINITY;
                p.lse2[(size_t)b * hq + i] = -INFINITY;
            }
        }
    }

    const int g4 = lane >> 2, c2 = (lane & 3) * 2;  // fragment row, first column
    // This lane's row and first chunk for ldmatrix; step i is 2 i chunks on, which
    // under the permutation is an XOR (tiles start on multiples of their row).
    const int k_row = lane & 15, v_row = (lane & 7) + ((lane >> 4) << 3);
    const uint32_t k_at = k_row * kRow + (((lane >> 4) ^ (k_row & 7)) << 4);
    const uint32_t v_at = v_row * kRow + ((((lane >> 3) & 1) ^ (v_row & 7)) << 4);
    const int G = p.group;

    // A segment is what a worker has of one (sequence, head group): units
    // [begin, end) of the group's [seg0, seg1).
    struct Segment {
        int b, h, base, count, seg0, begin, end;
        bool mine;  // the last group may have fewer heads than warps
    };
    auto segment_at = [&](int u) {
        Segment g;
        g.b = owner(base, v.batch, p.s.groups, u);
        g.base = base[g.b];
        g.count = base[g.b + 1] - g.base;
        const int grp = (u - g.base * p.s.groups) / g.count;
        g.seg0 = g.base * p.s.groups + grp * g.count;
        g.begin = u;
        g.end = min(u1, g.seg0 + g.count);
        g.h = grp * p.s.heads + head_in;
        g.mine = g.h < v.hkv;
        return g;
    };
    // Q of a segment as B fragments (16 dims x 8 heads). With few query heads the
    // next segment's come in while this one's pages do.
    auto load_q = [&](const Segment& sg, uint32_t (&qf)[NT][kSteps][2]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int g = nt * 8 + g4;
            const bool there = sg.mine && g < G;
            const uint16_t* row = p.d.q + sg.b * p.d.q_stride_batch + (int64_t)(sg.h * G + g) * p.d.q_stride_head + c2;
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
                qf[nt][ks][0] = there ? *reinterpret_cast<const uint32_t*>(row + ks * 16) : 0u;
                qf[nt][ks][1] = there ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8) : 0u;
            }
        }
    };
    constexpr bool kAhead = NT == 1 && D <= 128;

    int u = u0, read_stage = 0;
    Segment sg{}, sg_next{};
    uint32_t qf[NT][kSteps][2], q_next[NT][kSteps][2];
    if (u0 < u1) {
        sg_next = segment_at(u0);
        load_q(sg_next, q_next);
    }
    while (u < u1) {
        sg = sg_next;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) qf[nt][ks][0] = q_next[nt][ks][0], qf[nt][ks][1] = q_next[nt][ks][1];
        if (sg.end < u1) {
            sg_next = segment_at(sg.end);
            if (kAhead) load_q(sg_next, q_next);
        }
        const int b = sg.b, h = sg.h, seg0 = sg.seg0, seg1 = sg.seg0 + sg.count, begin = sg.begin, end = sg.end;
        const bool mine = sg.mine;
        float* score_row = p.scores && mine
                               ? p.scores + ((size_t)sg.base * v.hkv + (size_t)h * sg.count) * (kPageSlots * G)
                               : nullptr;
        float acc[NT][kSteps][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }
        bool any_key = false;

        for (; u < end; ++u) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            issue();
            const int stage = read_stage;
            if (++read_stage == kStages) read_stage = 0;
            const int valid = stage_info[warp][stage];
            if (valid == 0) {
                // A skipped page gets no weight.
                for (int i = lane; score_row && i < kPageSlots * G; i += 32)
                    score_row[(size_t)(u - seg0) * (kPageSlots * G) + i] = -INFINITY;
                continue;
            }
            any_key = true;
            const uint32_t tile = ring_addr + stage * (2 * kTile);

            float s[NT][4], odd[NT][4];  // two chains of products
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][i] = odd[nt][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
                uint32_t a[4];
                ldmatrix4(a, (tile + k_at) ^ (ks * 32));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<F16>(ks & 1 ? odd[nt] : s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][i] += odd[nt][i];
            float2 rest[NT][2];  // the weights, less the terms taken so far
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][i] *= p.scale_log2;
                if (score_row) {
                    float* at = score_row + (size_t)(u - seg0) * (kPageSlots * G) + g4 * G + nt * 8 + c2;
                    const int left = G - nt * 8 - c2;
                    if (left > 0) at[0] = s[nt][0], at[8 * G] = s[nt][2];
                    if (left > 1) at[1] = s[nt][1], at[8 * G + 1] = s[nt][3];
                }
                if (valid < kPageSlots) {
                    if (g4 >= valid) s[nt][0] = s[nt][1] = -INFINITY;
                    if (g4 + 8 >= valid) s[nt][2] = s[nt][3] = -INFINITY;
                }
                float x0 = fmaxf(s[nt][0], s[nt][2]), x1 = fmaxf(s[nt][1], s[nt][3]);
                // The maximum moves seldom once some pages are in.
                if (__any_sync(0xFFFFFFFFu, x0 > m[nt][0] || x1 > m[nt][1])) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, o));
                        x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, o));
                    }
                    const float n0 = fmaxf(m[nt][0], x0), n1 = fmaxf(m[nt][1], x1);
                    const float a0 = n0 == m[nt][0] ? 1.f : exp2_of(m[nt][0] - n0);
                    const float a1 = n1 == m[nt][1] ? 1.f : exp2_of(m[nt][1] - n1);
                    m[nt][0] = n0;
                    m[nt][1] = n1;
                    l[nt][0] *= a0;
                    l[nt][1] *= a1;
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        acc[nt][i][0] *= a0;
                        acc[nt][i][1] *= a1;
                        acc[nt][i][2] *= a0;
                        acc[nt][i][3] *= a1;
                    }
                }
                // Scores of -inf alone leave the maximum there: their weights are 0.
                const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
                const float p0 = exp2_of(s[nt][0] - m0), p1 = exp2_of(s[nt][1] - m1);
                const float p2 = exp2_of(s[nt][2] - m0), p3 = exp2_of(s[nt][3] - m1);
                l[nt][0] += p0 + p2;
                l[nt][1] += p1 + p3;
                rest[nt][0] = make_float2(p0 * kLift, p1 * kLift);
                rest[nt][1] = make_float2(p2 * kLift, p3 * kLift);
            }
            // The product with V takes P as a sum of 16-bit terms: three of bf16 hold all
            // 24 bits of a weight, two of f16 22. A third term is 0.5 % of a ragged step
            // (57.6 -> 57.9 us), 2.5 % of one over page lists (51.0 -> 52.3).
            uint32_t a[kSteps][4];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) ldmatrix4_trans(a[i], (tile + kTile + v_at) ^ (i * 32));
#pragma unroll
            for (int t = 0; t < kTerms; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t b0 = transpose8x8(take_term<F16>(rest[nt][0])), b1 = transpose8x8(take_term<F16>(rest[nt][1]));
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) mma16816<F16>(acc[nt][i], a[i], b0, b1);
                }
        }
        if (!kAhead && sg.end < u1) load_q(sg_next, q_next);
        if (!mine) continue;

        const bool whole = begin == seg0 && end == seg1;
        const int rows = p.s.heads * G;
        const size_t slot = (size_t)(2 * worker + (begin == u0 ? 0 : 1)) * rows + head_in * G;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float inv[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][i] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][i], o);
                inv[i] = any_key ? 1.f / l[nt][i] / kLift : 0.f;
                const int g = nt * 8 + c2 + i;
                if (g4 != 0 || g >= G) continue;
                if (whole) {
                    const float e = any_key ? m[nt][i] + log2f(l[nt][i]) : -INFINITY;
                    const size_t q_row = (size_t)b * hq + h * G + g;
                    p.lse2[q_row] = any_key && l[nt][i] == 0.f ? NAN : e;
                    if (p.d.lse) p.d.lse[q_row] = e * kLn2;
                } else {
                    // A part whose scores were all -inf is told from one without keys by its maximum.
                    p.part_ml[slot + g] = make_float2(any_key && m[nt][i] == -INFINITY ? kLowest : m[nt][i], l[nt][i]);
                }
            }
            if (whole && p.d.out_dtype != 0) {
                // Transposed, so that a lane holds two neighbouring dims of one head.
                uint16_t* to = static_cast<uint16_t*>(p.d.out) + ((size_t)b * hq + h * G + nt * 8 + g4) * D + c2;
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float x = acc[nt][k][half * 2] * inv[0], y = acc[nt][k][half * 2 + 1] * inv[1];
                        const uint32_t w = transpose8x8(p.d.out_dtype == 30 ? pack2<false>(x, y) : pack2<true>(x, y));
                        if (nt * 8 + g4 < G) *reinterpret_cast<uint32_t*>(to + k * 16 + half * 8) = w;
                    }
                continue;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int g = nt * 8 + c2 + i;
                if (g >= G) continue;
                const float factor = whole ? inv[i] : 1.f / kLift;
                float* to = (whole ? static_cast<float*>(p.d.out) + ((size_t)b * hq + h * G) * D : p.part_acc + slot * D) +
                            (size_t)g * D + g4;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    to[k * 16] = acc[nt][k][i] * factor;
                    to[k * 16 + 8] = acc[nt][k][i + 2] * factor;
                }
            }
        }
    }
}

// Units of sequence b, as the decode kernel counted them. The join and the
// totals call it before their wait: the decode kernel lets them start when its
// own predecessors are done, and nothing of this call writes the lengths (they
// are read past L1, which may hold older ones).
__device__ __forceinline__ int units_of(const DecodeParams& p, int b) {
    const int len = __ldcg(p.v.lens + b);
    if (len < 0) return 0;
    const int tokens = min(len, p.v.table_pages * kPageSlots - (p.d.k_new ? 1 : 0)) + (p.d.k_new ? 1 : 0);
    return min(p.d.pages ? p.d.n_pages : 0x7FFFFFFF, pages_of(tokens));
}

__device__ __forceinline__ void store_lse(const DecodeParams& p, size_t q_row, float m, float l) {
    const float e = m == -INFINITY ? -INFINITY : m + log2f(l);
    p.lse2[q_row] = m != -INFINITY && l == 0.f ? NAN : e;
    if (p.d.lse) p.d.lse[q_row] = e * kLn2;
}

// Joins the parts of each cut sequence, in order. A segment of at most 32
// parts is joined one row (query head) a warp, or by four if there is room, a
// longer one by two to eight warps a row; when these are few (one long sequence), a quarter of a row's dims
// a CTA, so that its parts (2.4 MB at 32 heads and 147 parts) are fetched by
// many SMs. Bound: latency (2 us behind the wait at one long sequence, 3.3 at 64
// ragged ones). Everything but the loads
// comes before the wait for the decode kernel, no load depends on another, and
// a CTA of one row loads each maximum and sum once: once a warp took 4000 cycles
// at 147 parts, all of them asking the same few lines of L2. 72 registers, so
// that a CTA fits beside one of the decode kernel.
constexpr int kJoinWarps = 8, kJoinThreads = kJoinWarps * 32, kJoinCuts = 4, kFewParts = 32, kFetchParts = 8;
constexpr int kMaxParts = kMaxGrid * 8;

struct JoinShared {
    int warp_sums[32];
    int slots[kJoinWarps];
    int cut_segs[kMaxParts];  // segments: those of few parts from the front, the others from the back
    float2 ml[kMaxParts];     // of one row's parts
    float4 acc[kJoinWarps][64];
};

// One row's dims [cut * D / CUTS, + D / CUTS) from its `parts` parts, by the CTA.
template <int D, int CUTS, typename Slot>
__device__ __forceinline__ void join_row(const DecodeParams& p, JoinShared& sh, int parts, Slot slot, size_t q_row, int cut) {
    constexpr int kSpan = D / CUTS, kLanes = kSpan / 4 < 32 ? kSpan / 4 : 32;  // lanes of a part's span
    constexpr int kVecs = kSpan / 4 / kLanes;          // 16-byte loads of a lane and part
    constexpr int kStep = kJoinWarps * (32 / kLanes);  // parts of the CTA's one load
    constexpr int kBatch = 5;                          // parts of a lane in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part0 = warp * (32 / kLanes) + lane / kLanes;
    const size_t dims = cut * kSpan + (lane % kLanes) * 4;
    float4 x[kBatch][kVecs], acc[kVecs];
    auto load = [&](int from) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
                const int i = from + k * kStep;
                x[k][j] = i < parts ? __ldcg(reinterpret_cast<const float4*>(p.part_acc + slot(i) * D + dims + j * kLanes * 4))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
            }
    };
    load(part0);
    for (int i = threadIdx.x; i < parts; i += kJoinThreads) sh.ml[i] = __ldcg(&p.part_ml[slot(i)]);
    __syncthreads();
    float m = -INFINITY;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, sh.ml[i].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    auto factor_of = [&](float part_m) { return part_m == m ? 1.f : exp2_of(part_m - m); };
    float l = 0.f;
    for (int i = lane; i < parts; i += 32) l += sh.ml[i].y * factor_of(sh.ml[i].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = part0;;) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float f = i + k * kStep < parts ? factor_of(sh.ml[i + k * kStep].x) : 0.f;
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
                acc[j].x += x[k][j].x * f;
                acc[j].y += x[k][j].y * f;
                acc[j].z += x[k][j].z * f;
                acc[j].w += x[k][j].w * f;
            }
        }
        i += kBatch * kStep;
        if (i - part0 >= parts) break;
        load(i);
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
#pragma unroll
        for (int o = kLanes; o < 32; o <<= 1) {
            acc[j].x += __shfl_xor_sync(~0u, acc[j].x, o);
            acc[j].y += __shfl_xor_sync(~0u, acc[j].y, o);
            acc[j].z += __shfl_xor_sync(~0u, acc[j].z, o);
            acc[j].w += __shfl_xor_sync(~0u, acc[j].w, o);
        }
        if (lane < kLanes) sh.acc[warp][j * kLanes + lane] = acc[j];
    }
    __syncthreads();
    const float inv = m == -INFINITY ? 0.f : 1.f / l;  // no key at all: zeros
    if (threadIdx.x < kSpan) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) o += reinterpret_cast<const float*>(sh.acc[w])[threadIdx.x];
        store_out(p.d.out, q_row * D + cut * kSpan + threadIdx.x, o * inv, p.d.out_dtype);
    }
    if (cut == 0 && threadIdx.x == 0) store_lse(p, q_row, m, l);
    __syncthreads();
}

// One row by WARPS of the CTA's warps, each finding the row's maximum and sum
// for itself: several rows of a CTA, few warps asking the same lines. Every
// thread of the CTA calls it (there: whether its row is one).
template <int D, int WARPS, typename Slot>
__device__ __forceinline__ void join_rows(const DecodeParams& p, JoinShared& sh, bool there, int parts, Slot slot,
                                          size_t q_row) {
    constexpr int kLanes = D / 4 < 32 ? D / 4 : 32;  // lanes of a part
    constexpr int kVecs = D / 4 / kLanes;         // 16-byte loads of a lane and part
    constexpr int kStep = WARPS * (32 / kLanes);  // parts of one load of the row's warps
    constexpr int kBatch = 5;                     // parts of a lane in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part0 = (warp % WARPS) * (32 / kLanes) + lane / kLanes;
    const int dims = (lane % kLanes) * 4;
    float m = -INFINITY, l = 0.f;
    if (there) {
        float4 x[kBatch][kVecs], acc[kVecs];
        float top[kBatch];
        auto load = [&](int from) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = from + k * kStep;
                top[k] = i < parts ? __ldcg(&p.part_ml[slot(i)].x) : -INFINITY;
#pragma unroll
                for (int j = 0; j < kVecs; ++j)
                    x[k][j] = i < parts ? __ldcg(reinterpret_cast<const float4*>(p.part_acc + slot(i) * D + dims + j * kLanes * 4))
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        };
        load(part0);
        // A lane's running maximum and sum of parts lane, lane + 32, .., then the row's.
        for (int i0 = 0; i0 < parts; i0 += 32 * kBatch) {
            float2 ml[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = i0 + k * 32 + lane;
                ml[k] = i < parts ? __ldcg(&p.part_ml[slot(i)]) : make_float2(-INFINITY, 0.f);
            }
            float n = m;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) n = fmaxf(n, ml[k].x);
            l *= m == n ? 1.f : exp2_of(m - n);
            m = n;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) l += ml[k].x == m ? ml[k].y : ml[k].y * exp2_of(ml[k].x - m);
        }
        const float mine = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        l *= mine == m ? 1.f : exp2_of(mine - m);
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
        for (int j = 0; j < kVecs; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = part0;;) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const float f = i + k * kStep >= parts ? 0.f : top[k] == m ? 1.f : exp2_of(top[k] - m);
#pragma unroll
                for (int j = 0; j < kVecs; ++j) {
                    acc[j].x += x[k][j].x * f;
                    acc[j].y += x[k][j].y * f;
                    acc[j].z += x[k][j].z * f;
                    acc[j].w += x[k][j].w * f;
                }
            }
            i += kBatch * kStep;
            if (i - part0 >= parts) break;
            load(i);
        }
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) {
                acc[j].x += __shfl_xor_sync(~0u, acc[j].x, o);
                acc[j].y += __shfl_xor_sync(~0u, acc[j].y, o);
                acc[j].z += __shfl_xor_sync(~0u, acc[j].z, o);
                acc[j].w += __shfl_xor_sync(~0u, acc[j].w, o);
            }
            if (lane < kLanes) sh.acc[warp][j * kLanes + lane] = acc[j];
        }
    }
    __syncthreads();
    if (there) {
        const float inv = m == -INFINITY ? 0.f : 1.f / l;  // no key at all: zeros
        const int first = warp / WARPS * WARPS;
        for (int d = (warp - first) * 32 + lane; d < D; d += WARPS * 32) {
            float o = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) o += reinterpret_cast<const float*>(sh.acc[first + w])[d];
            store_out(p.d.out, q_row * D + d, o * inv, p.d.out_dtype);
        }
        if (warp == first && lane == 0) store_lse(p, q_row, m, l);
    }
    __syncthreads();
}

// One row by a warp: lane i holds part i's factor.
template <int D, typename Slot>
__device__ __forceinline__ void join_few(const DecodeParams& p, int parts, Slot slot, size_t q_row) {
    constexpr int kPer = D / 32, kBatch = D == 256 ? 4 : 8;
    const int lane = threadIdx.x & 31;
    const float2 ml = lane < parts ? __ldcg(&p.part_ml[slot(lane)]) : make_float2(-INFINITY, 0.f);
    float2 x[kBatch][kPer / 2], acc[kPer / 2];
    auto load = [&](int from) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
            for (int j = 0; j < kPer / 2; ++j)
                x[k][j] = from + k < parts
                              ? __ldcg(reinterpret_cast<const float2*>(p.part_acc + slot(from + k) * D + lane * kPer) + j)
                              : make_float2(0.f, 0.f);
    };
    load(0);
    float m = ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float c = ml.x == m ? 1.f : exp2_of(ml.x - m);
    float l = lane < parts ? ml.y * c : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
    for (int j = 0; j < kPer / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    for (int i = 0;;) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float f = __shfl_sync(~0u, c, i + k);
#pragma unroll
            for (int j = 0; j < kPer / 2; ++j) {
                acc[j].x += i + k < parts ? x[k][j].x * f : 0.f;
                acc[j].y += i + k < parts ? x[k][j].y * f : 0.f;
            }
        }
        i += kBatch;
        if (i >= parts) break;
        load(i);
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < kPer / 2; ++j) {
        store_out(p.d.out, q_row * D + lane * kPer + 2 * j, acc[j].x * inv, p.d.out_dtype);
        store_out(p.d.out, q_row * D + lane * kPer + 2 * j + 1, acc[j].y * inv, p.d.out_dtype);
    }
    if (lane == 0) store_lse(p, q_row, m, l);
}

template <int D>
__global__ void __maxnreg__(72) batch_join_kernel(const DecodeParams p) {
    extern __shared__ int base[];
    __shared__ JoinShared sh;
    scan_counts(p.v.batch, base, sh.warp_sums, [&](int b) { return units_of(p, b); });
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rows = p.s.heads * p.group;
    const int total = base[p.v.batch] * p.s.groups;
    const int per = max(1, (total + p.s.workers - 1) / p.s.workers);
    // A cut segment belongs to the first boundary between workers inside it.
    int n_few = 0, n_many = 0, n_some = 0;  // some: of the few, those that a warp does not fetch at once
    for (int w = 0; (int64_t)(w + 1) * per < total; w += kJoinThreads) {
        const int64_t u = (int64_t)(w + (int)threadIdx.x + 1) * per;  // the boundary's unit
        int seg = 0, parts = 0;
        if (u < total) {
            const int b = owner(base, p.v.batch, p.s.groups, (int)u);
            const int count = base[b + 1] - base[b], grp = ((int)u - base[b] * p.s.groups) / count;
            const int s0 = base[b] * p.s.groups + grp * count;
            seg = b * p.s.groups + grp;
            if (s0 < u && s0 >= u - per) parts = (s0 + count - 1) / per - (w + (int)threadIdx.x) + 1;
        }
        const bool few = parts && parts <= kFewParts, many = parts > kFewParts;
        const uint32_t few_mask = __ballot_sync(~0u, few), many_mask = __ballot_sync(~0u, many);
        const uint32_t some_mask = __ballot_sync(~0u, few && parts > kFetchParts);
        __syncthreads();
        if (lane == 0) sh.slots[warp] = __popc(few_mask) | __popc(some_mask) << 10 | __popc(many_mask) << 20;
        __syncthreads();
        const int x = lane < kJoinWarps ? sh.slots[lane] : 0;
        const int before = __reduce_add_sync(~0u, lane < warp ? x : 0), all = __reduce_add_sync(~0u, x);
        const uint32_t below = (1u << lane) - 1;
        if (few) sh.cut_segs[n_few + (before & 0x3FF) + __popc(few_mask & below)] = seg;
        if (many) sh.cut_segs[kMaxParts - 1 - (n_many + (before >> 20) + __popc(many_mask & below))] = seg;
        n_few += all & 0x3FF;
        n_some += all >> 10 & 0x3FF;
        n_many += all >> 20;
    }
    __syncthreads();
    // Of the longer segments' rows, as much to a CTA as leaves one item a CTA:
    // a quarter of one, one, two or four.
    const int many_rows = n_many * rows, few_rows = n_few * rows, ctas = gridDim.x;
    const int cuts = many_rows * kJoinCuts <= ctas ? kJoinCuts : 1;
    const int together = many_rows <= ctas ? 1 : many_rows <= 2 * ctas ? 2 : 4;
    const int many_items = (many_rows * cuts + together - 1) / together;
    // The others' rows have a warp each, or, if that would fetch again and again
    // and CTAs are left, four (8 sequences of 18 parts, 32 heads: 54.2 -> 51.1 us a
    // sparse step; 5 of 24 to 340 pages, 40 heads: 15.6 -> 15.0).
    const bool pairs = 2 * n_some > n_few && (few_rows + 1) / 2 + many_items <= ctas;
    const int few_blocks = (rows + kJoinWarps - 1) / kJoinWarps;
    const int few_items = pairs ? (few_rows + 1) / 2 : n_few * few_blocks, items = few_items + many_items;
    bool waited = false;
    for (int item = blockIdx.x; item < items; item += ctas) {
        const bool few = item < few_items, alone = few && !pairs;
        // A row of the CTA's warps: of its segment's, or of all the list's.
        const int line = alone ? item / few_blocks
                         : few ? item * 2 + warp * 2 / kJoinWarps
                               : (item - few_items) / cuts * together + warp * together / kJoinWarps;
        const bool listed = alone || line < (few ? few_rows : many_rows);
        const int at = !listed ? 0 : alone ? line : line / rows;
        const int row = alone ? (item - at * few_blocks) * kJoinWarps + warp : line - at * rows;
        const int seg = sh.cut_segs[few ? at : kMaxParts - 1 - at];
        const int b = seg / p.s.groups, grp = seg - b * p.s.groups;
        const int count = base[b + 1] - base[b];
        const int s0 = base[b] * p.s.groups + grp * count, w0 = s0 / per, parts = (s0 + count - 1) / per - w0 + 1;
        const bool there = listed && row < rows && grp * p.s.heads + row / p.group < p.v.hkv;
        // Part i lies in its worker's first slot, the segment's first part in the second unless it starts the worker's.
        const size_t slot0 = (size_t)2 * w0 * rows + row;
        const int shift0 = s0 != w0 * per ? rows : 0;
        auto slot = [&](int i) { return slot0 + (size_t)(2 * i) * rows + (i == 0 ? shift0 : 0); };
        const size_t q_row = (size_t)b * p.d.n_q_heads + grp * rows + row;
        if (!waited) {
            pdl_wait();
            pdl_trigger();
            waited = true;
        }
        if (alone) {
            if (there) join_few<D>(p, parts, slot, q_row);
        } else if (!few && together == 1) {
            // The CTA's warps have one row.
            if (there && cuts > 1) join_row<D, kJoinCuts>(p, sh, parts, slot, q_row, (item - few_items) % cuts);
            else if (there) join_row<D, 1>(p, sh, parts, slot, q_row, 0);
        } else if (few || together == 2) {
            join_rows<D, kJoinWarps / 2>(p, sh, there, parts, slot, q_row);
        } else {
            join_rows<D, kJoinWarps / 4>(p, sh, there, parts, slot, q_row);
        }
    }
    // Every CTA waits, so that this kernel ends behind the decode kernel.
    if (!waited) {
        pdl_wait();
        pdl_trigger();
    }
}

template <int V>
struct __align__(V * 4) Vec {
    float x[V];
};

// weights_out[t] = decay * weights_in[t] + sum over the head's queries of
// exp2(s_t - lse): a CTA per chunk of 1024 tokens of one (sequence, head), four
// tokens a thread in flight. Bound: HBM and L2, 4 G + 8 bytes a token and head
// (25 MB at 32768 tokens, 8 heads, G 4: 4.5 us of the step).
constexpr int kTotalsThreads = 256, kTotalsTokens = 4, kTotalsChunk = kTotalsThreads * kTotalsTokens;
template <int V>  // scores of one load: the group is a multiple of it
__global__ void __launch_bounds__(kTotalsThreads) batch_totals_kernel(const DecodeParams p) {
    extern __shared__ int chunks[];
    __shared__ int warp_sums[32];
    const int G = p.group, hkv = p.v.hkv;
    constexpr int kPages = kTotalsChunk / kPageSlots;
    // Chunks before each sequence, and units.
    int* base = chunks + p.v.batch + 1;
    scan_counts(p.v.batch, base, warp_sums, [&](int b) { return units_of(p, b); });
    __syncthreads();
    scan_counts(p.v.batch, chunks, warp_sums, [&](int b) { return (base[b + 1] - base[b] + kPages - 1) / kPages; });
    pdl_wait();
    pdl_trigger();
    const int64_t all = (int64_t)chunks[p.v.batch] * hkv;
    for (int64_t c = blockIdx.x; c < all; c += gridDim.x) {
        const int at = (int)(c / hkv), h = (int)(c - (int64_t)at * hkv);
        const int b = owner(chunks, p.v.batch, 1, at);
        const int t0 = (at - chunks[b]) * kTotalsChunk + threadIdx.x;
        const int units = base[b + 1] - base[b];
        const int len = p.v.lens[b], n = attended(p.v, p.d, b, false);
        const size_t row = ((size_t)b * hkv + h) * p.d.weights_stride;
        const float* s = p.scores + ((size_t)base[b] * hkv + (size_t)h * units) * kPageSlots * G;
        const float* e = p.lse2 + (size_t)b * p.d.n_q_heads + h * G;
        float sum[kTotalsTokens];
#pragma unroll
        for (int i = 0; i < kTotalsTokens; ++i) {
            const int t = t0 + i * kTotalsThreads;
            sum[i] = p.d.weights_in && t < min(n, len) ? p.d.decay * p.d.weights_in[row + t] : 0.f;
        }
        for (int g = 0; g < G; g += V) {
            Vec<V> x[kTotalsTokens];
#pragma unroll
            for (int i = 0; i < kTotalsTokens; ++i)
                x[i] = *reinterpret_cast<const Vec<V>*>(s + (size_t)min(t0 + i * kTotalsThreads, units * kPageSlots - 1) * G + g);
#pragma unroll
            for (int i = 0; i < kTotalsTokens; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) sum[i] += e[g + k] == -INFINITY ? 0.f : exp2_of(x[i].x[k] - e[g + k]);
        }
#pragma unroll
        for (int i = 0; i < kTotalsTokens; ++i) {
            const int t = t0 + i * kTotalsThreads;
            if (t < n) p.d.weights_out[row + t] = sum[i];
        }
    }
}

template <int D>
constexpr int warps_of() { return D == 256 ? 4 : 8; }

size_t smem_bytes(int batch) { return kRingAlign + kRingBytes + sizeof(int) * (size_t)(batch + 1); }

template <typename F>
cudaError_t for_kernel(bool f16, int dim, bool two, F f) {
#define GKV_CASE(F16, D, NT) \
    if (f16 == F16 && dim == D && two == (NT == 2)) return f(batch_decode_kernel<F16, D, NT, warps_of<D>()>);
    GKV_CASE(false, 64, 1)
    GKV_CASE(false, 64, 2)
    GKV_CASE(false, 128, 1)
    GKV_CASE(false, 128, 2)
    GKV_CASE(false, 256, 1)
    GKV_CASE(false, 256, 2)
    GKV_CASE(true, 64, 1)
    GKV_CASE(true, 64, 2)
    GKV_CASE(true, 128, 1)
    GKV_CASE(true, 128, 2)
    GKV_CASE(true, 256, 1)
    GKV_CASE(true, 256, 2)
#undef GKV_CASE
    return cudaErrorInvalidValue;
}

size_t round16(size_t x) { return (x + 15) / 16 * 16; }

struct DecodeSpace {
    size_t acc, ml, lse2, scores, all;
};
DecodeSpace decode_space(const BatchView& v, const BatchSplit& s, int n_q_heads, bool totals) {
    const size_t rows = (size_t)2 * s.workers * s.heads * (n_q_heads / v.hkv);
    DecodeSpace o;
    o.acc = 0;
    o.ml = o.acc + round16(rows * v.dim * sizeof(float));
    o.lse2 = o.ml + round16(rows * sizeof(float2));
    o.scores = o.lse2 + round16((size_t)v.batch * n_q_heads * sizeof(float));
    o.all = o.scores + (totals ? (size_t)v.batch * v.table_pages * kPageSlots * n_q_heads * sizeof(float) : 0);
    return o;
}

}  // namespace

BatchSplit batch_split(const BatchView& v) {
    BatchSplit s;
    s.warps = v.dim == 256 ? 4 : 8;
    // Groups of like size, so that a unit costs the same in each.
    s.groups = (v.hkv + s.warps - 1) / s.warps;
    s.heads = (v.hkv + s.groups - 1) / s.groups;
    s.lanes = s.warps / s.heads;
    s.grid = v.sms < kMaxGrid ? v.sms : kMaxGrid;
    s.workers = s.grid * s.lanes;
    return s;
}

size_t batch_decode_bytes(const BatchView& v, int32_t n_q_heads, bool totals) {
    return decode_space(v, batch_split(v), n_q_heads, totals).all;
}

cudaError_t configure_batch_decode() {
    for (int f16 = 0; f16 < 2; ++f16)
        for (int dim = 64; dim <= 256; dim *= 2)
            for (int two = 0; two < 2; ++two) {
                const cudaError_t e =
                    for_kernel(f16, dim, two, [](auto* k) { return configure_kernel(k, smem_bytes(kMaxBatch), true); });
                if (e != cudaSuccess) return e;
            }
    cudaError_t e = configure_kernel(batch_join_kernel<64>, 0, true);
    if (e == cudaSuccess) e = configure_kernel(batch_join_kernel<128>, 0, true);
    if (e == cudaSuccess) e = configure_kernel(batch_join_kernel<256>, 0, true);
    return e;
}

cudaError_t launch_batch_decode(const BatchView& v, const BatchDecodeLaunch& d, cudaStream_t stream) {
    DecodeParams p;
    p.v = v;
    p.d = d;
    p.s = batch_split(v);
    p.group = d.n_q_heads / v.hkv;
    p.scale_log2 = d.scale * kLog2e;
    const DecodeSpace o = decode_space(v, p.s, d.n_q_heads, d.weights_out != nullptr);
    char* w = static_cast<char*>(d.workspace);
    p.part_acc = reinterpret_cast<float*>(w + o.acc);
    p.part_ml = reinterpret_cast<float2*>(w + o.ml);
    p.lse2 = reinterpret_cast<float*>(w + o.lse2);
    p.scores = d.weights_out ? reinterpret_cast<float*>(w + o.scores) : nullptr;
    cudaError_t e = for_kernel(v.f16, v.dim, p.group > 8, [&](auto* k) {
        return launch_dependent(k, dim3(p.s.grid), dim3(p.s.warps * 32), smem_bytes(v.batch), stream, p);
    });
    if (e != cudaSuccess) return e;
    // The join is always launched: it also keeps the launches behind it from
    // starting before the appended rows are in their pages.
    // At most what runs at once: a second wave would start behind the first.
    const int items = v.batch * p.s.groups * p.s.heads * p.group * kJoinCuts;
    const dim3 grid((unsigned)std::min(items, v.sms));
    const size_t base_bytes = sizeof(int) * (size_t)(v.batch + 1);
    e = v.dim == 64    ? launch_dependent(batch_join_kernel<64>, grid, dim3(kJoinThreads), base_bytes, stream, p)
        : v.dim == 128 ? launch_dependent(batch_join_kernel<128>, grid, dim3(kJoinThreads), base_bytes, stream, p)
                       : launch_dependent(batch_join_kernel<256>, grid, dim3(kJoinThreads), base_bytes, stream, p);
    if (e != cudaSuccess || !d.weights_out) return e;
    auto* totals = p.group % 4 == 0   ? batch_totals_kernel<4>
                   : p.group % 2 == 0 ? batch_totals_kernel<2>
                                      : batch_totals_kernel<1>;
    return launch_dependent(totals, dim3(v.sms * 4), dim3(kTotalsThreads), sizeof(int) * (size_t)(2 * v.batch + 2), stream, p);
}

}  // namespace gkv
