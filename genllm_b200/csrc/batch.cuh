// batch.cuh — device helpers shared by the batch tier's kernels.
#pragma once
#include "batch.h"
#include "device.cuh"

namespace gkv {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Pages that hold n tokens, at most the table row's.
__device__ __forceinline__ int pages_of(int n) { return (n + kPageSlots - 1) / kPageSlots; }

// base[b] = sum of count(b') over b' < b, for b = 0 .. batch: every thread of
// the CTA calls it; base and warp_sums (32 ints) are shared memory. A thread
// sums a run of consecutive sequences, so one pass serves any batch.
template <typename Count>
__device__ __forceinline__ void scan_counts(int batch, int* base, int* warp_sums, Count count) {
    const int tid = threadIdx.x, n = blockDim.x, lane = tid & 31;
    if (batch <= 32) {
        // Every warp for itself: the same values, no barrier.
        int inc = lane < batch ? count(lane) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xFFFFFFFFu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane < batch) base[lane + 1] = inc;
        if (lane == 0) base[0] = 0;
        __syncwarp();
        return;
    }
    const int run = (batch + n - 1) / n;
    const int b0 = min(batch, tid * run), b1 = min(batch, b0 + run);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = count(b);
        base[b] = c;
        sum += c;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) warp_sums[tid >> 5] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < (tid >> 5); ++w) before += warp_sums[w];
    for (int b = b0; b < b1; ++b) {
        const int c = base[b];
        base[b] = before;
        before += c;
    }
    if (tid == n - 1) base[batch] = before;
    __syncthreads();
}

// The sequence that owns unit u: the last b with base[b] * per <= u.
__device__ __forceinline__ int owner(const int* base, int batch, int per, int u) {
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (base[mid] * per <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
                 "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// c += a b: 16 x 8 (fp32) = 16 x 16 by 16 x 8, both f16 or both bf16.
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Dynamic shared memory up to `bytes`; with `all` the SM's whole carveout, so
// that a CTA of the kernel behind fits beside this one's. (Kernels that load
// through L1 keep the driver's choice: page bounds took 17 us so, 22 with the
// whole carveout.)
template <typename Kernel>
inline cudaError_t configure_kernel(Kernel kernel, size_t bytes, bool all = false) {
    cudaError_t e = cudaSuccess;
    if (bytes) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && all)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e;
}

// Launch as a programmatic dependent: the kernel waits (pdl_wait) before it
// touches anything the kernels ahead of it on the stream write.
template <typename... Args, typename... Given>
inline cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                    Given... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args>(args)...);
}

// The same with one cluster of `cluster` CTAs per row.
template <typename Params>
inline cudaError_t launch_cluster(void (*kernel)(Params), unsigned rows, int cluster, int threads, size_t smem,
                                  cudaStream_t stream, const Params& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * cluster);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace gkv
