// batch.cpp — C ABI of the batch tier (include/genllm_kv.h): argument checks
// and dispatch for decode, page bounds, page selection and eviction over many
// sequences of one paged pool. Every check comes before the first CUDA call.
#include <nvtx3/nvToolsExt.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/genllm_kv.h"
#include "batch.h"

namespace {

using gkv::BatchView;

constexpr int kMaxDevices = 64;
constexpr int kMaxKvHeads = 256;

int fail(int status, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    gkv::set_last_error(buf);
    return status;
}

int cuda_fail(cudaError_t e, const char* what) { return fail(GKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

struct NvtxRange {
    explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
    ~NvtxRange() { nvtxRangePop(); }
};

// Runs the body with `device` current and restores the caller's device.
class DeviceGuard {
   public:
    explicit DeviceGuard(int device) {
        ok_ = cudaGetDevice(&prev_) == cudaSuccess;
        if (ok_ && prev_ != device) ok_ = moved_ = cudaSetDevice(device) == cudaSuccess;
    }
    ~DeviceGuard() {
        if (moved_) cudaSetDevice(prev_);
    }
    bool ok() const { return ok_; }

   private:
    int prev_ = 0;
    bool ok_ = false, moved_ = false;
};

struct DeviceState {
    uint32_t* err = nullptr;
    int sms = 0;
};
std::mutex g_mu;
DeviceState g_state[kMaxDevices];

// The current device's error word and SM count, its kernels configured.
int device_state(int device, DeviceState* out) {
    std::lock_guard<std::mutex> lock(g_mu);
    DeviceState& s = g_state[device];
    if (!s.err) {
        DeviceState n;
        cudaError_t e = cudaDeviceGetAttribute(&n.sms, cudaDevAttrMultiProcessorCount, device);
        if (e == cudaSuccess) e = gkv::configure_batch_decode();
        if (e == cudaSuccess) e = gkv::configure_select();
        if (e == cudaSuccess) e = gkv::configure_evict();
        if (e == cudaSuccess) e = gkv::batch_error_word(&n.err);
        if (e != cudaSuccess) return cuda_fail(e, "batch tier setup");
        s = n;
    }
    *out = s;
    return GKV_OK;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The checks every entry point makes of its gkv_batch; no CUDA call.
int check_batch(const gkv_batch* b) {
    if (!b) return fail(GKV_ERR_INVALID, "null batch");
    const gkv_pool_desc& p = b->pool;
    if (p.dtype != GKV_BF16 && p.dtype != GKV_F16)
        return fail(GKV_ERR_UNSUPPORTED, "KV dtype %d: bf16 (30) and f16 (1) are built", p.dtype);
    if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
        return fail(GKV_ERR_UNSUPPORTED, "head_dim %d: 64, 128 and 256 are built", p.head_dim);
    if (p.n_kv_heads < 1 || p.n_kv_heads > kMaxKvHeads) return fail(GKV_ERR_INVALID, "n_kv_heads %d", p.n_kv_heads);
    if (p.pool_pages < 1 || p.pool_pages > INT32_MAX / GKV_PAGE_SLOTS) return fail(GKV_ERR_INVALID, "pool_pages %d", p.pool_pages);
    if (!p.k_base || !p.v_base || !aligned(p.k_base, 16) || !aligned(p.v_base, 16))
        return fail(GKV_ERR_INVALID, "pool bases must be non-null and 16-byte aligned");
    if (b->batch < 1 || b->batch > gkv::kMaxBatch)
        return fail(GKV_ERR_UNSUPPORTED, "batch %d: 1 to %d sequences", b->batch, gkv::kMaxBatch);
    if (b->table_pages < 1 || b->table_pages > INT32_MAX / GKV_PAGE_SLOTS || b->table_stride < b->table_pages)
        return fail(GKV_ERR_INVALID, "table_pages %d, table_stride %lld", b->table_pages, (long long)b->table_stride);
    // Pages are numbered along one line of 32-bit units.
    const int group = p.head_dim == 256 ? 4 : 8;
    if ((int64_t)b->batch * b->table_pages * ((p.n_kv_heads + group - 1) / group) > INT32_MAX / 2)
        return fail(GKV_ERR_UNSUPPORTED, "%d sequences of %d pages: too many in one call", b->batch, b->table_pages);
    if (!b->table || !b->lens || !aligned(b->table, 8) || !aligned(b->lens, 4))
        return fail(GKV_ERR_INVALID, "table and lens must be non-null and aligned");
    if (b->device < 0 || b->device >= kMaxDevices) return fail(GKV_ERR_INVALID, "device %d", b->device);
    return GKV_OK;
}

// Query heads: a whole number per kv head, at most kMaxBatchGroup.
int check_heads(const gkv_batch* b, int32_t n_q_heads) {
    const int hkv = b->pool.n_kv_heads;
    if (n_q_heads < 1 || n_q_heads % hkv)
        return fail(GKV_ERR_INVALID, "n_q_heads %d is not a multiple of n_kv_heads %d", n_q_heads, hkv);
    if (n_q_heads / hkv > gkv::kMaxBatchGroup)
        return fail(GKV_ERR_UNSUPPORTED, "%d query heads per kv head: at most %d", n_q_heads / hkv, gkv::kMaxBatchGroup);
    return GKV_OK;
}

// Rows of a strided [batch][heads][D] tensor start on 16 bytes; the stride of an
// extent of 1 is never used.
int check_rows(const void* p, int64_t batch, int64_t heads, int64_t stride_batch, int64_t stride_head, const char* what) {
    if (!p || !aligned(p, 16) || (batch > 1 && stride_batch % 8) || (heads > 1 && stride_head % 8))
        return fail(GKV_ERR_INVALID, "%s must be non-null with 16-byte aligned rows", what);
    return GKV_OK;
}

// Whether byte ranges [a, a + a_bytes) and [b, b + b_bytes) share a byte.
bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x < a_bytes : x - y < b_bytes;
}

// Bytes from the first to the last element of a strided [batch][heads][D]
// tensor of 16-bit elements; 0 for strides that run backwards.
size_t span_bytes(int64_t batch, int64_t heads, int64_t dim, int64_t stride_batch, int64_t stride_head) {
    if (batch == 1) stride_batch = 0;
    if (heads == 1) stride_head = 0;
    if (stride_batch < 0 || stride_head < 0) return 0;
    return 2 * (size_t)((batch - 1) * stride_batch + (heads - 1) * stride_head + dim);
}

// An array and its successor: the same memory or apart.
int check_successor(const void* in, const void* out, size_t bytes, const char* what) {
    if (in && in != out && overlap(in, bytes, out, bytes))
        return fail(GKV_ERR_INVALID, "%s overlaps its successor without being the same array", what);
    return GKV_OK;
}

BatchView view_of(const gkv_batch* b, const DeviceState& s) {
    BatchView v;
    v.k_base = static_cast<uint16_t*>(b->pool.k_base);
    v.v_base = static_cast<uint16_t*>(b->pool.v_base);
    v.table = reinterpret_cast<const int2*>(b->table);
    v.lens = b->lens;
    v.err = s.err;
    v.table_stride = b->table_stride;
    v.batch = b->batch;
    v.table_pages = b->table_pages;
    v.pool_pages = b->pool.pool_pages;
    v.hkv = b->pool.n_kv_heads;
    v.dim = b->pool.head_dim;
    v.f16 = b->pool.dtype == GKV_F16;
    v.sms = s.sms;
    return v;
}

int check_space(const void* workspace, size_t have, size_t need) {
    if (!workspace || !aligned(workspace, 16)) return fail(GKV_ERR_INVALID, "workspace must be non-null and 16-byte aligned");
    if (have < need) return fail(GKV_ERR_INVALID, "workspace of %zu bytes: %zu are needed", have, need);
    return GKV_OK;
}

// Selects the batch's device and looks its state up.
#define GKV_ENTER(b)                                                                         \
    DeviceGuard guard((b)->device);                                                          \
    if (!guard.ok()) return fail(GKV_ERR_CUDA, "cannot select device %d", (b)->device);      \
    DeviceState state;                                                                       \
    if (int st = device_state((b)->device, &state)) return st;

}  // namespace

extern "C" {

int gkv_batch_prepare(int device) {
    if (device < 0 || device >= kMaxDevices) return fail(GKV_ERR_INVALID, "device %d", device);
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(GKV_ERR_CUDA, "cannot select device %d", device);
    DeviceState state;
    return device_state(device, &state);
}

int gkv_batch_check_errors(int device, uint32_t* flags) {
    if (device < 0 || device >= kMaxDevices) return fail(GKV_ERR_INVALID, "device %d", device);
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(GKV_ERR_CUDA, "cannot select device %d", device);
    DeviceState state;
    if (int st = device_state(device, &state)) return st;
    uint32_t v = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&v, state.err, sizeof v, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && v) e = cudaMemset(state.err, 0, sizeof v);
    if (e != cudaSuccess) return cuda_fail(e, "batch error word");
    if (flags) *flags = v;
    return v ? fail(GKV_ERR_DEVICE, "batch error word 0x%x", v) : GKV_OK;
}

int gkv_batch_decode_workspace(const gkv_batch* b, int32_t n_q_heads, int32_t totals, size_t* bytes) {
    if (int st = check_batch(b)) return st;
    if (int st = check_heads(b, n_q_heads)) return st;
    if (!bytes) return fail(GKV_ERR_INVALID, "null bytes");
    GKV_ENTER(b)
    *bytes = gkv::batch_decode_bytes(view_of(b, state), n_q_heads, totals != 0);
    return GKV_OK;
}

int gkv_batch_decode(const gkv_batch* b, const gkv_batch_decode_args* a, gkv_stream_t stream) {
    NvtxRange range("gkv batch decode");
    if (int st = check_batch(b)) return st;
    if (!a) return fail(GKV_ERR_INVALID, "null arguments");
    if (int st = check_heads(b, a->n_q_heads)) return st;
    if (int st = check_rows(a->q, b->batch, a->n_q_heads, a->q_stride_batch, a->q_stride_head, "q")) return st;
    if (!a->k_new != !a->v_new) return fail(GKV_ERR_INVALID, "k_new and v_new come together");
    if (a->k_new) {
        if (int st = check_rows(a->k_new, b->batch, b->pool.n_kv_heads, a->k_stride_batch, a->k_stride_head, "k_new")) return st;
        if (int st = check_rows(a->v_new, b->batch, b->pool.n_kv_heads, a->v_stride_batch, a->v_stride_head, "v_new")) return st;
    }
    if (a->out_dtype != GKV_F32 && a->out_dtype != GKV_F16 && a->out_dtype != GKV_BF16)
        return fail(GKV_ERR_UNSUPPORTED, "output dtype %d", a->out_dtype);
    if (!a->out || !aligned(a->out, 16)) return fail(GKV_ERR_INVALID, "out must be non-null and 16-byte aligned");
    if (a->lse && !aligned(a->lse, 4)) return fail(GKV_ERR_INVALID, "lse must be 4-byte aligned");
    if (!std::isfinite(a->scale)) return fail(GKV_ERR_INVALID, "scale %g", (double)a->scale);
    if (a->pages && (a->n_pages < 1 || !aligned(a->pages, 4)))
        return fail(GKV_ERR_INVALID, "n_pages %d", a->n_pages);
    if (a->weights_out) {
        if (a->pages) return fail(GKV_ERR_UNSUPPORTED, "attention totals over a page list");
        if (!aligned(a->weights_out, 4) || !aligned(a->weights_in, 4) ||
            a->weights_stride < (int64_t)GKV_PAGE_SLOTS * b->table_pages)
            return fail(GKV_ERR_INVALID, "weights_stride %lld below 16 * table_pages", (long long)a->weights_stride);
        if (!std::isfinite(a->decay)) return fail(GKV_ERR_INVALID, "decay %g", (double)a->decay);
        if (int st = check_successor(a->weights_in, a->weights_out,
                                     sizeof(float) * (size_t)b->batch * b->pool.n_kv_heads * a->weights_stride, "weights_in"))
            return st;
    } else if (a->weights_in) {
        return fail(GKV_ERR_INVALID, "weights_in without weights_out");
    }
    // Rows of out are written while others' inputs are still read.
    const int64_t n = b->batch, hkv = b->pool.n_kv_heads, dim = b->pool.head_dim;
    const size_t out_bytes = (a->out_dtype == GKV_F32 ? 4 : 2) * (size_t)n * a->n_q_heads * dim;
    if (overlap(a->out, out_bytes, a->q, span_bytes(n, a->n_q_heads, dim, a->q_stride_batch, a->q_stride_head)) ||
        (a->k_new && (overlap(a->out, out_bytes, a->k_new, span_bytes(n, hkv, dim, a->k_stride_batch, a->k_stride_head)) ||
                      overlap(a->out, out_bytes, a->v_new, span_bytes(n, hkv, dim, a->v_stride_batch, a->v_stride_head)))))
        return fail(GKV_ERR_INVALID, "out overlaps an input");
    if (int st = check_space(a->workspace, a->workspace_bytes, 0)) return st;
    GKV_ENTER(b)
    const BatchView v = view_of(b, state);
    if (int st = check_space(a->workspace, a->workspace_bytes,
                             gkv::batch_decode_bytes(v, a->n_q_heads, a->weights_out != nullptr)))
        return st;
    gkv::BatchDecodeLaunch d;
    d.q = static_cast<const uint16_t*>(a->q);
    d.q_stride_batch = a->q_stride_batch;
    d.q_stride_head = a->q_stride_head;
    d.k_new = static_cast<const uint16_t*>(a->k_new);
    d.v_new = static_cast<const uint16_t*>(a->v_new);
    d.k_stride_batch = a->k_stride_batch;
    d.k_stride_head = a->k_stride_head;
    d.v_stride_batch = a->v_stride_batch;
    d.v_stride_head = a->v_stride_head;
    d.out = a->out;
    d.lse = a->lse;
    d.pages = a->pages;
    d.weights_in = a->weights_in;
    d.weights_out = a->weights_out;
    d.weights_stride = a->weights_stride;
    d.n_pages = a->n_pages;
    d.n_q_heads = a->n_q_heads;
    d.out_dtype = a->out_dtype;
    d.scale = a->scale;
    d.decay = a->decay;
    d.workspace = a->workspace;
    const cudaError_t e = gkv::launch_batch_decode(v, d, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? GKV_OK : cuda_fail(e, "batch decode launch");
}

int gkv_batch_page_bounds(const gkv_batch* b, const int32_t* start, int32_t extra, void* bounds,
                          gkv_stream_t stream) {
    NvtxRange range("gkv page bounds");
    if (int st = check_batch(b)) return st;
    if (!bounds || !aligned(bounds, 16) || !aligned(start, 4))
        return fail(GKV_ERR_INVALID, "bounds must be non-null and 16-byte aligned");
    if (extra < 0 || extra > GKV_PAGE_SLOTS * b->table_pages) return fail(GKV_ERR_INVALID, "extra %d", extra);
    GKV_ENTER(b)
    const cudaError_t e = gkv::launch_page_bounds(view_of(b, state), start, extra, static_cast<uint16_t*>(bounds),
                                                  reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? GKV_OK : cuda_fail(e, "page bounds launch");
}

int gkv_batch_select_workspace(const gkv_batch* b, size_t* bytes) {
    if (int st = check_batch(b)) return st;
    if (!bytes) return fail(GKV_ERR_INVALID, "null bytes");
    GKV_ENTER(b)
    *bytes = gkv::select_bytes(view_of(b, state));
    return GKV_OK;
}

int gkv_batch_select_pages(const gkv_batch* b, const gkv_batch_select_args* a, gkv_stream_t stream) {
    NvtxRange range("gkv select pages");
    if (int st = check_batch(b)) return st;
    if (!a) return fail(GKV_ERR_INVALID, "null arguments");
    if (int st = check_heads(b, a->n_q_heads)) return st;
    if (int st = check_rows(a->q, b->batch, a->n_q_heads, a->q_stride_batch, a->q_stride_head, "q")) return st;
    if (!a->bounds || !aligned(a->bounds, 16)) return fail(GKV_ERR_INVALID, "bounds must be non-null and 16-byte aligned");
    if (!a->pages || !aligned(a->pages, 4)) return fail(GKV_ERR_INVALID, "pages must be non-null");
    if (a->n_pages < 1 || a->n_first < 0 || a->n_last < 0 || (int64_t)a->n_first + a->n_last > a->n_pages)
        return fail(GKV_ERR_INVALID, "n_pages %d, n_first %d, n_last %d", a->n_pages, a->n_first, a->n_last);
    if (a->extra < 0 || a->extra > GKV_PAGE_SLOTS * b->table_pages) return fail(GKV_ERR_INVALID, "extra %d", a->extra);
    if (int st = check_space(a->workspace, a->workspace_bytes, 0)) return st;
    GKV_ENTER(b)
    const BatchView v = view_of(b, state);
    if (int st = check_space(a->workspace, a->workspace_bytes, gkv::select_bytes(v))) return st;
    const gkv::SelectLaunch s{static_cast<const uint16_t*>(a->q), a->q_stride_batch, a->q_stride_head,
                              static_cast<const uint16_t*>(a->bounds), a->pages, a->n_pages, a->n_first, a->n_last,
                              a->extra, a->n_q_heads, a->workspace};
    const cudaError_t e = gkv::launch_select_pages(v, s, reinterpret_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? GKV_OK : cuda_fail(e, "select pages launch");
}

int gkv_batch_evict_workspace(const gkv_batch* b, size_t* bytes) {
    if (int st = check_batch(b)) return st;
    if (!bytes) return fail(GKV_ERR_INVALID, "null bytes");
    GKV_ENTER(b)
    *bytes = gkv::evict_bytes(view_of(b, state));
    return GKV_OK;
}

int gkv_batch_evict(const gkv_batch* b, const gkv_batch_evict_args* a, gkv_stream_t stream) {
    NvtxRange range("gkv evict");
    if (int st = check_batch(b)) return st;
    if (!a) return fail(GKV_ERR_INVALID, "null arguments");
    if (!a->weights || !a->weights_out || !a->positions_out || !a->seen || !a->lens_out)
        return fail(GKV_ERR_INVALID, "weights, weights_out, positions_out, seen and lens_out must be non-null");
    if (a->tracked && !a->positions) return fail(GKV_ERR_INVALID, "tracked without positions");
    for (const void* p : {(const void*)a->weights, (const void*)a->weights_out, (const void*)a->positions,
                          (const void*)a->positions_out, (const void*)a->seen, (const void*)a->tracked,
                          (const void*)a->lens_out})
        if (!aligned(p, 4)) return fail(GKV_ERR_INVALID, "arrays must be 4-byte aligned");
    if (a->stride < (int64_t)GKV_PAGE_SLOTS * b->table_pages)
        return fail(GKV_ERR_INVALID, "stride %lld below 16 * table_pages", (long long)a->stride);
    const size_t bytes = sizeof(float) * (size_t)b->batch * b->pool.n_kv_heads * a->stride;
    if (int st = check_successor(a->weights, a->weights_out, bytes, "weights")) return st;
    if (int st = check_successor(a->positions, a->positions_out, bytes, "positions")) return st;
    if (a->n_keep < 0 || a->n_recent < 0 || a->n_recent > a->n_keep)
        return fail(GKV_ERR_INVALID, "n_keep %d, n_recent %d", a->n_keep, a->n_recent);
    if ((int64_t)b->batch * b->pool.n_kv_heads > 65535)
        return fail(GKV_ERR_UNSUPPORTED, "batch x kv heads above 65535");
    if (int st = check_space(a->workspace, a->workspace_bytes, 0)) return st;
    GKV_ENTER(b)
    const BatchView v = view_of(b, state);
    if (int st = check_space(a->workspace, a->workspace_bytes, gkv::evict_bytes(v))) return st;
    const gkv::EvictLaunch e{a->weights, a->weights_out, a->positions, a->positions_out, a->seen, a->tracked,
                             a->lens_out, a->stride, a->n_keep, a->n_recent, a->workspace};
    const cudaError_t err = gkv::launch_evict(v, e, reinterpret_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? GKV_OK : cuda_fail(err, "evict launch");
}

}  // extern "C"
