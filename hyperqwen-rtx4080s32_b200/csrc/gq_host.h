// Host bookkeeping that the library's translation units share: the last CUDA error's text, the count of launches, and the device status
// word of the unit that holds the operators beside the quantized layers (gq_device_status answers for both units).
#pragma once
#include <cuda_runtime.h>
#include "../../include/gq_b200.h"

#define GQ_HIDDEN __attribute__((visibility("hidden")))

namespace gq {
GQ_HIDDEN int cuda_fail(cudaError_t e, const char *what);            // gq_b200.cu: keeps the text, returns GQ_ERR_CUDA
GQ_HIDDEN void count_launch();
GQ_HIDDEN cudaError_t block_status_read(int *code, cudaStream_t s);  // gq_block.cu: its word, queued on the stream
GQ_HIDDEN cudaError_t block_status_clear(cudaStream_t s);
}  // namespace gq

#define GQ_CUDA(call)                                              \
    do {                                                           \
        cudaError_t e_ = (call);                                   \
        if (e_ != cudaSuccess) return gq::cuda_fail(e_, #call);    \
    } while (0)
#define GQ_LAUNCHED()                                                        \
    do {                                                                     \
        cudaError_t e_ = cudaGetLastError();                                 \
        if (e_ != cudaSuccess) return gq::cuda_fail(e_, "kernel launch");    \
        gq::count_launch();                                                  \
    } while (0)
