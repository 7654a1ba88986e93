// batch_error.cu — the batch tier's device error word, one per device.
#include "batch.h"

namespace gkv {
static __device__ uint32_t g_batch_err;

cudaError_t batch_error_word(uint32_t** err) {
    void* p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, g_batch_err);
    *err = static_cast<uint32_t*>(p);
    return e;
}
}  // namespace gkv
