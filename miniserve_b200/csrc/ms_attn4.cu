// ms_kv4_attention -- attention of one or several tokens a row over a paged
// cache held in 4 bits (declared in include/mssample.h):
//
//   x_j = scale q . k_j,  o = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),
//   lse = m + log sum_j exp(x_j - m),  m = max_j x_j
//
// over the keys j that a token sees, k_j and v_j being what the cache stands
// for, not rounded.  Partial results over disjoint sets of keys combine
// exactly: (m, l = sum exp(x - m), O = sum exp(x - m) v) in fp32, weighed by
// exp(m - max m).
#include <algorithm>
#include <atomic>

#include "../../include/mssample.h"
#include "ms_attn4.cuh"
#include "ms_host.h"

namespace ms {

static int64_t a4_round(int64_t n) { return (n + 255) / 256 * 256; }

struct A4Plan {
  int group, queries, chunks, chunk_rows, sixteens;  // sixteens of the wide kernel, or 0
  int64_t split_warps;
  int64_t base, own_o, own_ml, bytes;  // workspace: a header, the rows' first units, the records
};

static A4Plan a4_plan(int64_t rows, int tokens, int heads, int kv_heads, int head_dim, bool fine, int sms) {
  A4Plan p{};
  const int groups = k4_layout(head_dim).used;
  p.group = heads / kv_heads;
  p.queries = tokens * p.group;
  // as few items as hold all query rows, and those of equal sizes
  p.chunks = (p.queries + a4_most(groups, fine) - 1) / a4_most(groups, fine);
  p.chunk_rows = (p.queries + p.chunks - 1) / p.chunks;
  const int sixteen = fine ? 8 : 16;
  p.sixteens = p.chunk_rows <= a4_narrow(fine) ? 0 : (p.chunk_rows + sixteen - 1) / sixteen;
  p.split_warps = (int64_t)sms * (p.sixteens ? a4_wide_ctas(groups, p.sixteens) : a4_narrow_ctas(groups)) * kA4Warps;
  const int64_t pieces = rows * kv_heads * p.chunks + p.split_warps;
  int64_t at = 256;  // A4Header
  p.base = at, at = a4_round(at + rows * 8);
  p.own_o = at, at = a4_round(at + pieces * p.chunk_rows * head_dim * 4);
  p.own_ml = at, at = a4_round(at + pieces * p.chunk_rows * 8);
  p.bytes = at;
  return p;
}

static int a4_sms(int dev) {
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

static bool a4_sizes(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim) {
  return rows >= 0 && rows <= kA4MaxRows && tokens >= 1 && tokens <= kA4MaxTokens && kv_heads >= 1 && heads >= 1 &&
         heads <= 65536 && heads % kv_heads == 0 && head_dim >= 1 && head_dim <= 128 &&
         rows * tokens * heads <= 0x7FFFFFFFll;
}

template <typename K>
static cudaError_t a4_launch(K *kernel, int shared, std::atomic<int> (&ready)[kMaxDevices], const A4Args &a, int dev, cudaStream_t s) {
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
    if (e != cudaSuccess) return e;
    ready[dev].store(1, std::memory_order_release);
  }
  return launch_dependent(kernel, (unsigned)(a.split_warps / kA4Warps), kA4Warps * 32, shared, s, a);
}
template <int NG, bool kFine, bool kWhole>
static cudaError_t a4_split_narrow(const A4Args &a, int dev, cudaStream_t s) {
  static std::atomic<int> ready[kMaxDevices];
  return a4_launch(ms_attn4_narrow_kernel<NG, kFine, kWhole>, kA4NarrowShared<NG>, ready, a, dev, s);
}
template <int NG, int NP, bool kFine, bool kWhole>
static cudaError_t a4_split_wide(const A4Args &a, int dev, cudaStream_t s) {
  static std::atomic<int> ready[kMaxDevices];
  return a4_launch(ms_attn4_wide_kernel<NG, NP, kFine, kWhole>, kA4WideShared<NG, NP>, ready, a, dev, s);
}
template <int NG, bool kFine, bool kWhole>
static cudaError_t a4_split(const A4Args &a, int sixteens, int dev, cudaStream_t s) {
  if (sixteens == 0) return a4_split_narrow<NG, kFine, kWhole>(a, dev, s);
  if (sixteens == 1) return a4_split_wide<NG, 1, kFine, kWhole>(a, dev, s);
  if constexpr (NG <= 2) {
    if (sixteens == 2) return a4_split_wide<NG, 2, kFine, kWhole>(a, dev, s);
    if (sixteens == 3) return a4_split_wide<NG, 3, kFine, kWhole>(a, dev, s);
  }
  return cudaErrorInvalidValue;
}
template <int NG>
static cudaError_t a4_split_as(const A4Args &a, int sixteens, int dev, cudaStream_t s) {
  const bool whole = a.x.cache.page_size % kA4Half == 0;
  if (a.x.dtype == MS_DTYPE_F16)
    return whole ? a4_split<NG, true, true>(a, sixteens, dev, s) : a4_split<NG, true, false>(a, sixteens, dev, s);
  return whole ? a4_split<NG, false, true>(a, sixteens, dev, s) : a4_split<NG, false, false>(a, sixteens, dev, s);
}
template <typename T, int DP>
static cudaError_t a4_merge(const A4Args &a, cudaStream_t s) {
  const int64_t outputs = a.x.rows * a.x.tokens * a.x.heads;
  if (a.merge_wide) return launch_dependent(ms_attn4_merge_kernel<T, DP, kMgWide>, (unsigned)outputs, kMgWide * 32, 0, s, a);
  return launch_dependent(ms_attn4_merge_kernel<T, DP, 1>, (unsigned)((outputs + kMgNarrow - 1) / kMgNarrow),
                          kMgNarrow * 32, 0, s, a);
}

}  // namespace ms

extern "C" {

int64_t ms_kv4_attention_workspace(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (!ms::a4_sizes(rows, tokens, heads, kv_heads, head_dim)) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const int sms = ms::a4_sms(dev);  // of either type
  return std::max(ms::a4_plan(rows, tokens, heads, kv_heads, head_dim, false, sms).bytes,
                  ms::a4_plan(rows, tokens, heads, kv_heads, head_dim, true, sms).bytes);
}

int ms_kv4_attention(const ms_kv4_attention_args *args, ms_stream_t stream) {
  if (!args) return MS_E_INVALID;
  const ms_kv4_attention_args &x = *args;
  if (x.dtype != MS_DTYPE_BF16 && x.dtype != MS_DTYPE_F16) return MS_E_DTYPE;
  int rc = ms::k4_check(x.cache);
  if (rc != MS_OK) return rc;
  if (!ms::a4_sizes(x.rows, x.tokens, x.heads, x.cache.kv_heads, x.cache.head_dim) || x.table_width < 0 ||
      x.table_width > 0x7FFFFFFFll || x.table_row < 0 || x.length_row < 0 || !(x.scale > 0.f) || x.scale > 2.0e38f)
    return MS_E_INVALID;
  if (x.rows == 0) return MS_OK;
  if (!x.q || !x.lengths || !x.out || !x.lse || !x.status || !x.workspace ||
      (reinterpret_cast<uintptr_t>(x.workspace) & 255) || (x.table_width > 0 && !x.table))
    return MS_E_INVALID;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return ms::cuda_fail(e);
  const ms::A4Plan p = ms::a4_plan(x.rows, x.tokens, x.heads, x.cache.kv_heads, x.cache.head_dim, x.dtype == MS_DTYPE_F16, ms::a4_sms(dev));
  if (x.workspace_bytes < p.bytes) return MS_E_INVALID;
  ms::A4Args a{};
  a.x = x;
  a.layout = ms::k4_layout(x.cache.head_dim);
  a.group = p.group, a.queries = p.queries, a.chunks = p.chunks, a.chunk_rows = p.chunk_rows;
  a.split_warps = p.split_warps;
  a.code_head = x.cache.page_size * a.layout.row_bytes;
  a.code_page = a.code_head * x.cache.kv_heads;
  char *w = static_cast<char *>(x.workspace);
  a.header = reinterpret_cast<ms::A4Header *>(w);
  a.base = reinterpret_cast<int64_t *>(w + p.base);
  a.own_o = reinterpret_cast<float *>(w + p.own_o);
  a.own_ml = reinterpret_cast<float2 *>(w + p.own_ml);
  a.scale_log2 = x.scale * 1.4426950408889634f;
  a.q_wide = ((x.q_row | x.q_token | x.q_head) & 7) == 0 && (reinterpret_cast<uintptr_t>(x.q) & 15) == 0;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (x.cache.page_size == 1ll << i) a.page_shift = i;
  {  // records that an output may have: the warps spread over the items, but no more than the longest has room for
      const int64_t items = x.rows * x.cache.kv_heads * p.chunks;
      const int64_t tiles = (x.table_width * x.cache.page_size + ms::kA4Tile - 1) / ms::kA4Tile;
    // (two rows of 131072 keys: 86 us with a CTA an output, 111 with a warp; 128 rows of five tokens 146 and 66)
    a.merge_wide = std::min(p.split_warps / items + 1, (tiles + ms::kA4Item) / (ms::kA4Item + 1) + 1) > 24;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (a.layout.used) {
    case 1: e = ms::a4_split_as<1>(a, p.sixteens, dev, s); break;
    case 2: e = ms::a4_split_as<2>(a, p.sixteens, dev, s); break;
    case 3: e = ms::a4_split_as<3>(a, p.sixteens, dev, s); break;
    default: e = ms::a4_split_as<4>(a, p.sixteens, dev, s); break;
  }
  if (e == cudaSuccess) {
    const bool narrow = x.cache.head_dim <= 64;
    if (x.dtype == MS_DTYPE_BF16)
      e = narrow ? ms::a4_merge<__nv_bfloat16, 64>(a, s) : ms::a4_merge<__nv_bfloat16, 128>(a, s);
    else
      e = narrow ? ms::a4_merge<__half, 64>(a, s) : ms::a4_merge<__half, 128>(a, s);
  }
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
