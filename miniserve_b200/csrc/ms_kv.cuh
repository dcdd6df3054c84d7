// Helpers of the kernels that write and read paged caches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ms {

template <typename T>
__device__ __forceinline__ float2 kv_widen(uint32_t u);
template <>
__device__ __forceinline__ float2 kv_widen<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 kv_widen<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t kv_narrow(float x, float y);
template <>
__device__ __forceinline__ uint32_t kv_narrow<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t kv_narrow<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float kv_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float kv_to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void kv_from_float(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void kv_from_float(float x, __half &y) { y = __float2half_rn(x); }

// log2 of a page size, or -1.
inline int kv_page_shift(int64_t page_size) {
  for (int i = 0; i < 31; ++i)
    if (page_size == 1ll << i) return i;
  return -1;
}

// Page and offset of a slot, which is not negative.
__device__ __forceinline__ void kv_place(int64_t slot, int64_t page_size, int page_shift, int64_t &page, int64_t &offset) {
  if (page_shift >= 0) {
    page = slot >> page_shift;
    offset = slot & (page_size - 1);
  } else if (slot < (1ll << 32)) {
    page = (uint32_t)slot / (uint32_t)page_size;
    offset = (uint32_t)slot - (uint32_t)page * (uint32_t)page_size;
  } else {
    page = slot / page_size;
    offset = slot - page * page_size;
  }
}

}  // namespace ms
