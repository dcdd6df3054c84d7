// Host helpers shared by the library's source files.
#pragma once

#include <cuda_runtime.h>

namespace ms {

constexpr int kMaxDevices = 64;

// Records a failed CUDA call for ms_last_cuda_error and returns MS_E_CUDA.
__attribute__((visibility("hidden"))) int cuda_fail(cudaError_t e);

}  // namespace ms
