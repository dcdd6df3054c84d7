// Layout of a cache held in 4 bits (ms_kv4_cache of include/mssample.h).
#pragma once

#include <stdint.h>

#include "../../include/mssample.h"

namespace ms {

constexpr int kK4Group = 32;  // entries that share a scale and a middle

// A token's head: row_bytes bytes of codes (a multiple of 16) and `groups`
// pairs of fp16 parameters (a power of two), of which head_dim uses `used`.
struct K4Layout {
  int row_bytes, groups, used;
};

inline K4Layout k4_layout(int head_dim) {
  const int used = (head_dim + kK4Group - 1) / kK4Group;
  const int stored = used < 2 ? 2 : used;
  return K4Layout{stored * kK4Group / 2, stored == 3 ? 4 : stored, used};
}

inline int k4_check(const ms_kv4_cache &c) {
  if (c.kv_heads < 1 || c.kv_heads > 65536 || c.head_dim < 1 || c.pages < 1 || c.pages > 0x7FFFFFFFll ||
      c.page_size < 1 || c.page_size > 0x7FFFFFFFll || !c.k_codes || !c.k_params || !c.v_codes || !c.v_params)
    return MS_E_INVALID;
  // the last byte's address is a 64-bit offset
  if (c.pages > 0x7FFFFFFFFFFFll / c.page_size / c.kv_heads) return MS_E_INVALID;
  // a slot's parameters are copied at once, its codes by 16 bytes: a range of a cache's pages lies so too
  if (c.head_dim % 16 || c.head_dim > 128 ||
      ((reinterpret_cast<uintptr_t>(c.k_codes) | reinterpret_cast<uintptr_t>(c.v_codes)) & 15) ||
      ((reinterpret_cast<uintptr_t>(c.k_params) | reinterpret_cast<uintptr_t>(c.v_params)) & (k4_layout(c.head_dim).groups * 4 - 1)))
    return MS_E_UNSUPPORTED;
  return MS_OK;
}

}  // namespace ms
