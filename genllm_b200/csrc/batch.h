// batch.h — internal launch interface of the batch tier (batch.cpp checks the
// arguments, batch_*.cu hold the kernels). Not part of the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.h"

namespace gkv {

constexpr int kMaxBatch = 4096;        // sequences: their page prefix sums sit in shared memory
constexpr int kMaxBatchGroup = 16;     // query heads per kv head: two 8-column tensor-core tiles
constexpr uint32_t kErrBadLength = 4;  // device error word: a length beyond its table row (bits 0, 1: device.cuh)

// A gkv_batch after its checks.
struct BatchView {
    uint16_t* k_base;
    uint16_t* v_base;
    const int2* table;
    const int32_t* lens;
    uint32_t* err;
    int64_t table_stride;
    int32_t batch;
    int32_t table_pages;
    int32_t pool_pages;
    int32_t hkv;
    int32_t dim;
    int32_t f16;  // 0: bf16
    int32_t sms;
};

// How the decode kernel divides its work: the same numbers size the workspace.
struct BatchSplit {
    int32_t warps;      // of a CTA
    int32_t heads;      // kv heads a worker takes together, one warp each
    int32_t groups;     // ceil(hkv / heads)
    int32_t lanes;      // workers of a CTA
    int32_t workers;    // of the grid
    int32_t grid;
};

struct BatchDecodeLaunch {
    const uint16_t* q;
    int64_t q_stride_batch, q_stride_head;
    const uint16_t* k_new;
    const uint16_t* v_new;
    int64_t k_stride_batch, k_stride_head, v_stride_batch, v_stride_head;
    void* out;
    float* lse;
    const int32_t* pages;
    const float* weights_in;
    float* weights_out;
    int64_t weights_stride;
    int32_t n_pages;
    int32_t n_q_heads;
    int32_t out_dtype;
    float scale;
    float decay;
    void* workspace;
};

cudaError_t batch_error_word(uint32_t** err);  // the current device's

BatchSplit batch_split(const BatchView& v);
size_t batch_decode_bytes(const BatchView& v, int32_t n_q_heads, bool totals);
cudaError_t configure_batch_decode();
cudaError_t launch_batch_decode(const BatchView& v, const BatchDecodeLaunch& d, cudaStream_t stream);

cudaError_t launch_page_bounds(const BatchView& v, const int32_t* start, int32_t extra, uint16_t* bounds,
                               cudaStream_t stream);

struct SelectLaunch {
    const uint16_t* q;
    int64_t q_stride_batch, q_stride_head;
    const uint16_t* bounds;
    int32_t* pages;
    int32_t n_pages, n_first, n_last, extra, n_q_heads;
    void* workspace;
};
size_t select_bytes(const BatchView& v);
cudaError_t configure_select();
cudaError_t launch_select_pages(const BatchView& v, const SelectLaunch& s, cudaStream_t stream);

struct EvictLaunch {
    const float* weights;
    float* weights_out;
    const int32_t* positions;
    int32_t* positions_out;
    const int32_t* seen;
    const int32_t* tracked;
    int32_t* lens_out;
    int64_t stride;
    int32_t n_keep, n_recent;
    void* workspace;
};
size_t evict_bytes(const BatchView& v);
cudaError_t configure_evict();
cudaError_t launch_evict(const BatchView& v, const EvictLaunch& e, cudaStream_t stream);

}  // namespace gkv
