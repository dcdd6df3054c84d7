// Host helpers shared by the library's source files.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

namespace ms {

constexpr int kMaxDevices = 64;

// Records a failed CUDA call for ms_last_cuda_error and returns MS_E_CUDA.
__attribute__((visibility("hidden"))) int cuda_fail(cudaError_t e);

// A launch that may be set up while the kernel before it in the stream still
// runs (a programmatic dependent launch).  A call's first kernel waits
// (griddepcontrol.wait) before it touches memory and only then releases the
// next one, so the call's later kernels find the caller's tensors complete and
// their workspace free; they wait before they read what the call's own earlier
// kernels write.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, int shared, cudaStream_t s, const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = shared;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled through the runtime, so that the library needs no
// link to the driver.
inline cudaError_t encode_tiled(EncodeTiled *fn) {
  static std::atomic<EncodeTiled> known{nullptr};
  *fn = known.load(std::memory_order_acquire);
  if (*fn) return cudaSuccess;
  void *p = nullptr;
  cudaDriverEntryPointQueryResult found;
  cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
  if (e != cudaSuccess) return e;
  if (found != cudaDriverEntryPointSuccess || !p) return cudaErrorNotSupported;
  *fn = reinterpret_cast<EncodeTiled>(p);
  known.store(*fn, std::memory_order_release);
  return cudaSuccess;
}

}  // namespace ms
