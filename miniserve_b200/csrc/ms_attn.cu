// ms_prefix_attention -- single-token attention of a batch over a paged cache
// (declared in include/mssample.h): every row sees the keys of a prefix that
// the batch shares, then its own.
//
//   x_j = scale q . k_j,  o = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),
//   lse = m + log sum_j exp(x_j - m),  m = max_j x_j
//
// Partial results over disjoint sets of keys combine exactly: each is kept as
// (m, l = sum exp(x - m), O = sum exp(x - m) v) in fp32 for a reference m near
// its maximum, and the merge weighs them by exp(m - max m).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/mssample.h"
#include "ms_attn.cuh"
#include "ms_host.h"

namespace ms {

static int64_t at_round(int64_t n) { return (n + 255) / 256 * 256; }

static int at_sms(int dev) {
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Parts of the prefix for the prefix kernel: the fewest waves of CTAs (two an
// SM) times tiles of one CTA, each CTA costing about four tiles besides (its
// queries, first copies and record), and the records' way through L2, written
// and read (about 3 MB a tile's time).
static int at_parts(int64_t ctas, int64_t tiles, int64_t record_bytes, int sms) {
  int best = 1;
  double least = 0;
  for (int n = 1; n <= 2 * sms && n <= tiles; ++n) {
    const double waves = (double)((ctas * n + 2 * sms - 1) / (2 * sms));
    const double cost = waves * ((double)((tiles + n - 1) / n) + 4.0) + (double)n * record_bytes * 2 / 3e6;
    if (n == 1 || cost < least) best = n, least = cost;
    if (ctas * n >= 4 * sms) break;
  }
  return best;
}

struct AtPlan {
  AtShape shape;
  int packed, split_prefix, pre_splits, pre_tiles;
  // workspace: a header, the rows' first tiles, the split kernel's records, the prefix kernel's
  int64_t base, own_o, own_ml, pre_o, pre_ml, bytes;
};

static AtPlan at_plan(int64_t rows, int heads, int kv_heads, int head_dim, int64_t prefix, int sms) {
  AtPlan p{};
  AtShape &s = p.shape;
  s.rows = rows, s.heads = heads, s.kv_heads = kv_heads, s.head_dim = head_dim;
  s.group = heads / kv_heads;
  s.chunks = (s.group + kAtRows - 1) / kAtRows;
  s.chunk_rows = s.group < kAtRows ? s.group : kAtRows;
  s.split_warps = (int64_t)sms * sp_ctas(head_dim) * kSpWarps;
  p.packed = (int)(rows * s.group);
  if (prefix > 0 && p.packed <= kAtRows) {
    // one chunk of query rows: the split kernel reads the prefix once as well, with more warps at it
    p.split_prefix = (int)prefix;
    if (p.packed > s.chunk_rows) s.chunk_rows = p.packed;
  } else if (prefix > 0) {
    p.pre_tiles = (p.packed + kPrRows - 1) / kPrRows;
    p.pre_splits = at_parts((int64_t)p.pre_tiles * kv_heads, (prefix + kPrKeys - 1) / kPrKeys,
                            (int64_t)p.packed * kv_heads * head_dim * 4, sms);
  }
  const int64_t pieces = rows * kv_heads * s.chunks + (p.split_prefix ? kv_heads : 0) + s.split_warps;
  const int64_t pre = (int64_t)p.pre_splits * kv_heads * p.packed;
  int64_t at = 256;  // AtHeader
  p.base = at, at = at_round(at + rows * 8);
  p.own_o = at, at = at_round(at + pieces * s.chunk_rows * head_dim * 4);
  p.own_ml = at, at = at_round(at + pieces * s.chunk_rows * 8);
  p.pre_o = at, at = at_round(at + pre * head_dim * 4);
  p.pre_ml = at, at = at_round(at + pre * 8);
  p.bytes = at;
  return p;
}

// About how many records an output may have: the split kernel's warps spread
// over its items, but no more than the longest item has room for.
static int64_t at_records(const AtArgs &a) {
  const AtShape &s = a.shape;
  auto pieces = [&](int64_t keys, int64_t items) {
    return std::min(s.split_warps / items + 1, (sp_tiles(keys) + kSpItem) / (kSpItem + 1) + 1);
  };
  int64_t n = a.pre_splits;
  if (a.split_prefix) n += pieces(a.split_prefix, s.kv_heads);
  const int64_t room = a.x.table_width * a.x.page_size;
  if (room > 0) n += pieces(room, s.rows * s.kv_heads * s.chunks);
  return n;
}
// records above which a CTA of sixteen warps takes an output (4 rows behind 131072 keys, 150 records: 96 us, 138
// us with a warp each; 64 rows with about 5: 90 us with a warp each, 97 with sixteen)
constexpr int64_t kMgMany = 24;

template <typename F>
static cudaError_t at_allow_shared(F *kernel, int bytes, std::atomic<int> (&ready)[kMaxDevices], int dev) {
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) ready[dev].store(1, std::memory_order_release);
  return e;
}

template <typename T, int DP, int NQ, bool kWhole, int kCtas>
static cudaError_t at_split(const AtArgs &a, int dev, cudaStream_t s) {
  static std::atomic<int> ready[kMaxDevices];
  auto *kernel = ms_attn_split_kernel<T, DP, NQ, kWhole, kCtas>;
  cudaError_t e = at_allow_shared(kernel, kSpShared<DP>, ready, dev);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, (unsigned)(a.shape.split_warps / kSpWarps), kSpWarps * 32, kSpShared<DP>, s, a);
}

template <typename T, int DP, int kCtas>
static cudaError_t at_split_as(const AtArgs &a, int dev, cudaStream_t s) {
  if (a.narrow) return a.whole ? at_split<T, DP, 1, true, kCtas>(a, dev, s) : at_split<T, DP, 1, false, kCtas>(a, dev, s);
  return a.whole ? at_split<T, DP, 2, true, kCtas>(a, dev, s) : at_split<T, DP, 2, false, kCtas>(a, dev, s);
}

// One of the caches as [pages, kv_heads, page_size, head_dim], read in boxes of
// one page's or a tile's tokens and 64 entries (128 bytes, swizzled).
// False where the layout cannot be described so.
static bool at_map(CUtensorMap *map, const ms_prefix_attention_args &x, const void *base, int64_t page, int64_t token,
                   int64_t head) {
  const bool inner = x.page_size % 8 == 0 && (x.page_size % kPrKeys == 0 || kPrKeys % x.page_size == 0);
  EncodeTiled fn;
  if (!inner || encode_tiled(&fn) != cudaSuccess) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)x.head_dim, (cuuint64_t)x.page_size, (cuuint64_t)x.kv_heads,
                              (cuuint64_t)x.pages};
  // a dimension of one entry may have any stride: one that a map accepts
  const int64_t row = (int64_t)x.head_dim;
  const cuuint64_t strides[3] = {(cuuint64_t)(x.page_size > 1 ? token : row) * 2,
                                 (cuuint64_t)(x.kv_heads > 1 ? head : row) * 2,
                                 (cuuint64_t)(x.pages > 1 ? page : row) * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)(x.page_size < kPrKeys ? x.page_size : kPrKeys), 1, 1};
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  return fn(map, x.dtype == MS_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void *>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
static cudaError_t at_run(AtArgs &a, int dev, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (a.pre_splits) {
    static std::atomic<int> ready[kMaxDevices];
    e = at_allow_shared(ms_attn_prefix_kernel<T, DP>, kPrSharedBytes<DP>, ready, dev);
    CUtensorMap kmap{}, vmap{};
    a.tma = at_map(&kmap, a.x, a.x.cache_k, a.x.ck_page, a.x.ck_token, a.x.ck_head) &&
            at_map(&vmap, a.x, a.x.cache_v, a.x.cv_page, a.x.cv_token, a.x.cv_head);
    if (e == cudaSuccess)
      e = launch_dependent(ms_attn_prefix_kernel<T, DP>, (unsigned)((int64_t)a.pre_tiles * a.shape.kv_heads * a.pre_splits),
                           kPrThreads, kPrSharedBytes<DP>, s, a, kmap, vmap);
  }
  if (e != cudaSuccess) return e;
  if constexpr (DP == 64)
    e = at_split_as<T, DP, sp_ctas(64)>(a, dev, s);
  else
    e = a.x.head_dim <= 96 ? at_split_as<T, DP, sp_ctas(96)>(a, dev, s) : at_split_as<T, DP, sp_ctas(128)>(a, dev, s);
  if (e != cudaSuccess) return e;
  const int64_t outputs = a.shape.rows * a.shape.heads;
  if (a.merge_wide)
    return launch_dependent(ms_attn_merge_kernel<T, DP, kMgWide>, (unsigned)outputs, kMgWide * 32, 0, s, a);
  return launch_dependent(ms_attn_merge_kernel<T, DP, 1>, (unsigned)((outputs + kMgNarrow - 1) / kMgNarrow),
                          kMgNarrow * 32, 0, s, a);
}

}  // namespace ms

extern "C" {

int64_t ms_prefix_attention_workspace(int64_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                      int64_t prefix_length) {
  if (prefix_length < 0 || prefix_length > ms::kAtMaxKeys || rows < 0 || rows > ms::kAtMaxRows || heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65536 ||
      head_dim < 1 || head_dim > 128 || rows * heads > 0x7FFFFFFFll)
    return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  return ms::at_plan(rows, heads, kv_heads, head_dim, prefix_length, ms::at_sms(dev)).bytes;
}

int ms_prefix_attention(const ms_prefix_attention_args *args, ms_stream_t stream) {
  if (!args) return MS_E_INVALID;
  const ms_prefix_attention_args &x = *args;
  if (x.dtype != MS_DTYPE_BF16 && x.dtype != MS_DTYPE_F16) return MS_E_DTYPE;
  if (x.rows < 0 || x.rows > ms::kAtMaxRows || x.heads < 1 || x.heads > 65536 || x.kv_heads < 1 ||
      x.heads % x.kv_heads || x.head_dim < 1 || x.pages < 1 || x.pages > 0x7FFFFFFFll || x.page_size < 1 ||
      x.page_size > 0x7FFFFFFFll || x.table_width < 0 || x.table_width > 0x7FFFFFFFll || x.table_row < 0 ||
      x.prefix_length < 0 || x.prefix_length > ms::kAtMaxKeys || !(x.scale > 0.f) || x.scale > 2.0e38f)  // in units of log2 it is finite too
    return MS_E_INVALID;
  if (x.rows * x.heads > 0x7FFFFFFFll) return MS_E_INVALID;
  // 16-byte rows: what the copies of the cache read
  const int64_t strides = x.ck_page | x.ck_token | x.ck_head | x.cv_page | x.cv_token | x.cv_head;
  if (x.head_dim > 128 || x.head_dim % 8 || (strides & 7) || (reinterpret_cast<uintptr_t>(x.cache_k) & 15) ||
      (reinterpret_cast<uintptr_t>(x.cache_v) & 15))
    return MS_E_UNSUPPORTED;
  if (x.rows == 0) return MS_OK;
  if (!x.q || !x.cache_k || !x.cache_v || !x.lengths || !x.out || !x.lse || !x.status || !x.workspace ||
      (reinterpret_cast<uintptr_t>(x.workspace) & 255) || (x.table_width > 0 && !x.table) ||
      (x.prefix_length > 0 && !x.prefix_pages))
    return MS_E_INVALID;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return ms::cuda_fail(e);
  ms::AtArgs a{};
  a.x = x;
  const ms::AtPlan p = ms::at_plan(x.rows, x.heads, x.kv_heads, x.head_dim, x.prefix_length, ms::at_sms(dev));
  if (x.workspace_bytes < p.bytes) return MS_E_INVALID;
  a.shape = p.shape;
  a.packed = p.packed, a.split_prefix = p.split_prefix, a.pre_splits = p.pre_splits, a.pre_tiles = p.pre_tiles;
  char *w = static_cast<char *>(x.workspace);
  a.header = reinterpret_cast<ms::AtHeader *>(w);
  a.base = reinterpret_cast<int64_t *>(w + p.base);
  a.own_o = reinterpret_cast<float *>(w + p.own_o);
  a.own_ml = reinterpret_cast<float2 *>(w + p.own_ml);
  a.pre_o = reinterpret_cast<float *>(w + p.pre_o);
  a.pre_ml = reinterpret_cast<float2 *>(w + p.pre_ml);
  a.scale_log2 = x.scale * 1.4426950408889634f;
  a.q_wide = ((x.q_row | x.q_head) & 7) == 0 && (reinterpret_cast<uintptr_t>(x.q) & 15) == 0;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (x.page_size == 1ll << i) a.page_shift = i;
  a.merge_wide = ms::at_records(a) > ms::kMgMany;
  a.narrow = p.shape.chunk_rows <= 8;
  a.whole = x.page_size % ms::kSpTile == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool narrow = x.head_dim <= 64;
  if (x.dtype == MS_DTYPE_BF16)
    e = narrow ? ms::at_run<__nv_bfloat16, 64>(a, dev, s) : ms::at_run<__nv_bfloat16, 128>(a, dev, s);
  else
    e = narrow ? ms::at_run<__half, 64>(a, dev, s) : ms::at_run<__half, 128>(a, dev, s);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
