// Attention over a paged cache: arguments, the split kernel (rows' own keys,
// and the prefix's where few rows share it), the prefix kernel (where more
// do) and the merge.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mssample.h"
#include "ms_tc.cuh"

namespace ms {

constexpr int kAtRows = 16;              // query heads of one chunk: up to two Ns of the warp products
constexpr int64_t kAtMaxRows = 1 << 20;  // rows of a call
constexpr int kAtMaxKeys = 0x3FFFFFFF;   // of the prefix, and of a row: their sum is an int
constexpr int kSpWarps = 4;              // warps of a split CTA
// Split CTAs of an SM: what heads of fewer entries leave of the latencies is
// hidden by more warps (64 rows of 4 key heads of 80: 76 us with two, 66 with
// three; of 128: 90 with two, 96 with three).
__host__ __device__ constexpr int sp_ctas(int head_dim) { return head_dim <= 64 ? 4 : head_dim <= 96 ? 3 : 2; }
constexpr int kSpTile = 16;              // keys of a split tile: the M of the warp products
constexpr int kSpItem = 2;               // cost of an item's queries and record, in tiles
constexpr int kSpStages = 2;             // tiles of a warp's ring: one is copied while the other is used
template <int DP>
constexpr int kSpStage = 2 * kSpTile * DP * 2;  // K, then V
template <int DP>
constexpr int kSpShared = kSpStages * kSpStage<DP> * kSpWarps;

struct AtHeader {
  int64_t share;  // units of one split warp
};

// l of a record that met a page outside the cache (its keys count as zeros
// there), and of one whose CTA gave up a wait: the merge flags the rows that
// read the record.
constexpr float kAtBadPage = -1.f;
constexpr float kAtLate = -2.f;

struct AtShape {
  int64_t rows;
  int heads, kv_heads, head_dim;
  int group;       // query heads of a key head
  int chunks;      // chunks of kAtRows query heads of a key head
  int chunk_rows;  // query rows of a record
  int64_t split_warps;
};

struct AtArgs {
  ms_prefix_attention_args x;
  AtShape shape;
  AtHeader *header;
  int64_t *base;    // [rows] where each row starts in the split kernel's sequence
  float *own_o;     // [pieces][chunk_rows][head_dim]
  float2 *own_ml;   // [pieces][chunk_rows] (reference in units of log2, l)
  float *pre_o;     // [splits][kv_heads][packed rows][head_dim], of the prefix kernel
  float2 *pre_ml;   // [splits][kv_heads][packed rows]
  float scale_log2;
  int packed;        // rows * group: the prefix's query rows of one key head, row b's heads at b * group
  int split_prefix;  // keys of the prefix that the split kernel takes: all or none
  int pre_splits;    // parts of the prefix that the prefix kernel takes; 0 where it does not run
  int pre_tiles;     // its query tiles of one key head
  int q_wide;        // q's heads start 16-byte aligned
  int tma;           // the cache can be read in boxes of a tile, or of pages that divide it
  int page_shift;    // log2 of the page size, or -1
  int merge_wide;    // the merge gives each output a CTA
  int narrow;        // at most 8 query rows an item
  int whole;         // page_size is a multiple of kSpTile: a tile lies in one page
};

template <typename T>
struct AtType;
template <>
struct AtType<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct AtType<__half> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

constexpr float kAtFar = 1048576.f;  // references (units of log2) above this are not used in a fused exponent

// What weights refer to for a running maximum m, both in units of log2.  The
// weights are rounded to the cache's type for their product with V, which
// then runs on the tensor cores with both operands of one type; the sum and
// O stay in fp32.  fp16 loses bits below 2^-14, so its weights are scaled up
// by 2^kUp, which records carry along exactly; bf16 has fp32's range.
template <typename T, int kUp>
__device__ __forceinline__ float at_reference(float m) {
  return m;
}
template <>
__device__ __forceinline__ float at_reference<__half, 15>(float m) {
  return fabsf(m) <= kAtFar / 2 ? m - 15.f : m;  // further off, m - 15 would be rounded past fp16's largest weight
}
template <>
__device__ __forceinline__ float at_reference<__half, 7>(float m) {
  return fabsf(m) <= kAtFar / 2 ? m - 7.f : m;
}
constexpr int kSpUp = 15;  // the split kernel's weights are at most 2^0 of the running maximum,
constexpr int kPrUp = 7;   // the prefix kernel's 2^8

__device__ __forceinline__ float at_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes, or zeros where there is no source.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// A row's own keys: its length, or 0 where the length does not fit its pages
// or is past kAtMaxKeys (the merge flags the row).
__device__ __forceinline__ int at_length(const ms_prefix_attention_args &x, int64_t b) {
  const int n = load_in(x.lengths + b);
  return n >= 0 && n <= kAtMaxKeys && (int64_t)n <= x.table_width * x.page_size ? n : 0;
}

// Transposed 8 x 8 matrix of 16-bit entries.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The split kernel's sequence: items (row, key head and chunk) in order, each
// of kSpItem units and one unit a tile; items without keys are not in it.
// Row -1 is the prefix, all rows' query heads of a key head being its one
// chunk.
__host__ __device__ __forceinline__ int64_t sp_tiles(int64_t keys) { return (keys + kSpTile - 1) / kSpTile; }
__device__ __forceinline__ int64_t sp_units(int64_t keys) { return keys > 0 ? sp_tiles(keys) + kSpItem : 0; }
// Index of an item among the items.
__device__ __forceinline__ int64_t sp_item(const AtArgs &a, int64_t b, int hc) {
  return b < 0 ? hc : (a.split_prefix ? a.shape.kv_heads : 0) + b * a.shape.kv_heads * a.shape.chunks + hc;
}

// Walks over a warp's tiles.
struct SpWalk {
  int64_t b, left;  // left: units of the share past this item
  int hc, tile, end, tiles, keys;
};

__device__ __forceinline__ void sp_row(const AtArgs &a, SpWalk &w) {
  w.keys = w.b < 0 ? a.split_prefix : at_length(a.x, w.b);
  w.tiles = (int)sp_tiles(w.keys);
}
__device__ __forceinline__ int sp_head(const AtArgs &a, const SpWalk &w) {  // key head
  return w.b < 0 ? w.hc : w.hc / a.shape.chunks;
}
// The next item's tiles within the share; tile == end where none are left.
__device__ __forceinline__ void sp_item_next(const AtArgs &a, SpWalk &w) {
  w.tile = w.end = 0;
  if (w.left <= kSpItem) return;
  if (++w.hc >= (w.b < 0 ? a.shape.kv_heads : a.shape.kv_heads * a.shape.chunks)) {
    w.hc = 0;
    do {  // a later row has keys: units are left
      ++w.b;
      sp_row(a, w);
    } while (w.tiles == 0);
  }
  const int64_t take = min(w.left, (int64_t)w.tiles + kSpItem);
  w.left -= take;
  w.end = (int)take - kSpItem;
}
__device__ __forceinline__ void sp_next(const AtArgs &a, SpWalk &w) {
  if (++w.tile >= w.end) sp_item_next(a, w);
}

// Split kernel.  All rows' items (and the prefix's, where its query rows fit
// one chunk) form one sequence; every warp takes an equal, contiguous share of
// it, whatever the rows' lengths, and works alone: a ring of tiles of 16 keys
// filled with 16-byte asynchronous copies, a page lookup one tile ahead of its
// copies, and products of m16n8k16 with the keys as M and the queries as N
// (S^T = K Q^T, O^T += V^T P^T; P^T changes fragments with movmatrix), so that
// 8 query heads leave no half of a product empty.  Where its share meets an
// item's tiles, it leaves one record at index item + warp, which is unique
// because both only grow along the sequence.
//
// Bound by the bytes of the cache.
template <typename T, int DP, int NQ, bool kWhole, int kCtas>
__global__ void __launch_bounds__(kSpWarps * 32, kCtas)
    ms_attn_split_kernel(const __grid_constant__ AtArgs a) {
  constexpr int kRow = DP * 2;                 // bytes of a key's row in the ring
  constexpr int kChunks = DP / 8;              // 16-byte chunks of a row
  constexpr int kStage = kSpStage<DP>, kStages = kSpStages;
  constexpr int kRowsStep = 32 / kChunks;      // rows of one copy instruction
  constexpr int kThreads = kSpWarps * 32;
  const float kNone = __uint_as_float(0xFF800000u);
  extern __shared__ __align__(128) unsigned char sp_ring[];
  __shared__ int64_t sums[kThreads + 1];  // units of the rows before each thread's run of rows, of one key head and chunk
  __shared__ int64_t warp_sums[kSpWarps];
  if (!a.pre_splits) grid_wait();  // the call's first kernel
  grid_release();
  const ms_prefix_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t rows = a.shape.rows;
  const int hcs = a.shape.kv_heads * a.shape.chunks;
  const int64_t run = (rows + kThreads - 1) / kThreads;
  const int64_t r0 = min(rows, tid * run), r1 = min(rows, r0 + run);
  {
    int64_t n = 0;
#pragma unroll 8
    for (int64_t b = r0; b < r1; ++b) n += sp_units(at_length(x, b));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xFFFFFFFFu, n, o);
      if (lane >= o) n += v;
    }
    if (lane == 31) warp_sums[warp] = n;
    if (tid == 0) sums[0] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSpWarps; ++i)
      if (i < warp) n += warp_sums[i];
    sums[tid + 1] = n;
    __syncthreads();
  }
  const int64_t before = sp_units(a.split_prefix) * a.shape.kv_heads;
  const int64_t total = before + sums[kThreads] * hcs;
  const int64_t share = max((int64_t)kSpItem + 1, (total + a.shape.split_warps - 1) / a.shape.split_warps);
  if (blockIdx.x == gridDim.x - 1) {  // for the merge: where each row starts (this CTA's own share is the last, often short)
    int64_t n = sums[tid];
    for (int64_t b = r0; b < r1; ++b) {
      a.base[b] = before + n * hcs;
      x.status[b] = at_length(x, b) != load_in(x.lengths + b) ? MS_ROW_BAD_LENGTH : MS_ROW_OK;
      n += sp_units(at_length(x, b));
    }
    if (tid == 0) a.header->share = share;
  }
  const int64_t wid = (int64_t)blockIdx.x * kSpWarps + warp;
  const int64_t u0 = wid * share, u1 = min(total, u0 + share);
  if (u0 >= u1) {
    grid_wait();
    return;
  }
  SpWalk load;
  {
    int64_t first = 0;  // the row that unit u0 lies in: its thread's run, then the row
    if (u0 < before) {
      load.b = -1;
      sp_row(a, load);
    } else {
      int lo = 0, hi = kThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (before + sums[mid + 1] * hcs > u0) hi = mid;
        else lo = mid + 1;
      }
      load.b = min(rows, lo * run);
      first = before + sums[lo] * hcs;
      sp_row(a, load);
      while (first + sp_units(load.keys) * hcs <= u0) {
        first += sp_units(load.keys) * hcs;
        ++load.b;
        sp_row(a, load);
      }
    }
    const int64_t units = load.tiles + kSpItem;
    load.hc = (int)((u0 - first) / units);
    const int64_t at = u0 - first - load.hc * units, take = min(u1 - u0, units - at);
    load.left = u1 - u0 - take;
    load.tile = (int)max((int64_t)0, at - kSpItem);
    load.end = (int)(at + take) - kSpItem;
    if (load.end <= load.tile) sp_item_next(a, load);
  }
  SpWalk now = load;
  const uint32_t ring = smem_addr(sp_ring) + warp * kStages * kStage;
  const int page_size = (int)x.page_size;
  const int chunk = lane % kChunks;
  const bool inside = chunk * 8 < x.head_dim;

  // One page for all lanes where tiles lie in one; else lanes 0-15 look up
  // the tile's keys for K, lanes 16-31 for V.
  int page = -1, offset = 0, head = 0, live_keys = 0;
  uint32_t met = 0;  // bit i: the tile issued i tiles ago met a bad page
  auto look = [&]() {
    page = -1;
    live_keys = 0;
    if (load.tile < load.end) {
      const int j = load.tile * kSpTile + (kWhole ? 0 : lane & 15);
      live_keys = load.keys - load.tile * kSpTile;
      if (j < load.keys) {
        const int p = a.page_shift >= 0 ? j >> a.page_shift : j / page_size;
        offset = j - p * page_size;
        page = load_in(load.b < 0 ? x.prefix_pages + p : x.table + load.b * x.table_row + p);
      }
      head = sp_head(a, load);
      sp_next(a, load);
    }
  };
  const int64_t kstep = (int64_t)(lane / kChunks) * x.ck_token + chunk * 8;
  const int64_t vstep = (int64_t)(lane / kChunks) * x.cv_token + chunk * 8;
  auto issue = [&](int stage) {
    const uint32_t dst = ring + stage * kStage + (lane / kChunks) * kRow;
    const bool good = page >= 0 && page < x.pages;
    const bool wrong = !good && (kWhole ? 0 : lane & 15) < live_keys;
    met = (met << 1) | (kWhole ? wrong : __any_sync(0xFFFFFFFFu, wrong));
    if (kWhole) {
      const T *ks = static_cast<const T *>(x.cache_k), *vs = static_cast<const T *>(x.cache_v);
      if (good) {
        ks += page * x.ck_page + offset * x.ck_token + head * x.ck_head + kstep;
        vs += page * x.cv_page + offset * x.cv_token + head * x.cv_head + vstep;
      }
#pragma unroll
      for (int i = 0; i < kSpTile / kRowsStep; ++i) {
        const int r = i * kRowsStep + lane / kChunks;
        const bool live = good && inside && r < live_keys;
        copy16(dst + i * kRowsStep * kRow + ((chunk ^ (r & 7)) << 4), live ? ks : x.cache_k, live);
        ks += kRowsStep * x.ck_token;
      }
#pragma unroll
      for (int i = 0; i < kSpTile / kRowsStep; ++i) {
        const int r = i * kRowsStep + lane / kChunks;
        const bool live = good && inside && r < live_keys;
        copy16(dst + (kSpTile + i * kRowsStep) * kRow + ((chunk ^ (r & 7)) << 4), live ? vs : x.cache_v, live);
        vs += kRowsStep * x.cv_token;
      }
    } else {
      int64_t at = -1;
      if (good)
        at = lane < 16 ? page * x.ck_page + offset * x.ck_token + head * x.ck_head
                       : page * x.cv_page + offset * x.cv_token + head * x.cv_head;
#pragma unroll
      for (int i = 0; i < 2 * kSpTile / kRowsStep; ++i) {
        const int r = i * kRowsStep + lane / kChunks;  // 0-15: K, 16-31: V
        const int64_t from = __shfl_sync(0xFFFFFFFFu, at, r);
        const bool live = from >= 0 && inside;
        const T *src = static_cast<const T *>(r < kSpTile ? x.cache_k : x.cache_v) + (live ? from + chunk * 8 : 0);
        copy16(dst + i * kRowsStep * kRow + ((chunk ^ (r & 7)) << 4), src, live);
      }
    }
  };

  look();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    issue(s);
    look();
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  uint32_t qf[NQ][DP / 16][2];
  float o[NQ][DP / 16][4];
  float m[NQ][2], l[NQ][2];
  bool fresh = true, broken = false;
  int stage = 0;
  while (now.tile < now.end) {
    issue(stage == 0 ? kStages - 1 : stage - 1);
    look();
    asm volatile("cp.async.commit_group;" ::: "memory");
    // query rows of the item: a chunk of one row's heads, or all rows' heads for the prefix
    const int h = sp_head(a, now), c = now.b < 0 ? 0 : now.hc - h * a.shape.chunks;
    const int n = now.b < 0 ? a.packed : min(kAtRows, a.shape.group - c * kAtRows);
    if (fresh) {
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        const int g = t * 8 + (lane >> 2);
        const int64_t b = now.b < 0 ? g / a.shape.group : now.b;
        const int head_q = h * a.shape.group + (now.b < 0 ? g % a.shape.group : c * kAtRows + g);
        const T *q = static_cast<const T *>(x.q) + (g < n ? b * x.q_row + head_q * x.q_head : 0) + (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < DP / 8; ++k) {
          uint32_t u = 0;
          if (g < n && k * 8 < x.head_dim) {
            if (a.q_wide) {
              u = load_in(reinterpret_cast<const unsigned int *>(q + k * 8));
            } else {
              const unsigned short *p = reinterpret_cast<const unsigned short *>(q + k * 8);
              u = (uint32_t)load_in(p) | ((uint32_t)load_in(p + 1) << 16);
            }
          }
          qf[t][k >> 1][k & 1] = u;
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
        m[t][0] = m[t][1] = kNone;
        l[t][0] = l[t][1] = 0.f;
      }
      fresh = broken = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint32_t kst = ring + stage * kStage, vst = kst + kSpTile * kRow;
    float sc[NQ][2][4] = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const int r = lane & 15, ch = 2 * k + (lane >> 4);
      uint32_t f[4];
      ldmatrix4(f, kst + r * kRow + ((ch ^ (r & 7)) << 4));
#pragma unroll
      for (int t = 0; t < NQ; ++t) AtType<T>::mma(sc[t][k & 1], f, qf[t][k][0], qf[t][k][1]);
    }
    // scores in units of log2: entries 0, 1 of key lane / 4, queries 2 (lane % 4) and the next; 2, 3 of key + 8
    broken |= (met >> (kStages - 1)) & 1;
    const int left = now.keys - now.tile * kSpTile;
    uint32_t p[NQ][2];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (sc[t][0][i] + sc[t][1][i]) * a.scale_log2;
      if (left < kSpTile) {  // keys past the end leave nothing
        if ((lane >> 2) >= left) w[0] = w[1] = kNone;
        if ((lane >> 2) + 8 >= left) w[2] = w[3] = kNone;
      }
      float top[2] = {fmaxf(w[0], w[2]), fmaxf(w[1], w[3])};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], s));
        top[i] = fmaxf(top[i], m[t][i]);
      }
      if (__any_sync(0xFFFFFFFFu, top[0] != m[t][0] || top[1] != m[t][1])) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // both -inf (no score yet above it): nothing to rescale
          const float f =
              m[t][i] == top[i] ? 1.f : at_exp2(at_reference<T, kSpUp>(m[t][i]) - at_reference<T, kSpUp>(top[i]));
          m[t][i] = top[i];
          l[t][i] *= f;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) o[t][k][i] *= f, o[t][k][2 + i] *= f;
        }
      }
      // a score of -inf has weight 0 whatever the maximum
      const float base[2] = {m[t][0] == kNone ? 0.f : at_reference<T, kSpUp>(m[t][0]),
                             m[t][1] == kNone ? 0.f : at_reference<T, kSpUp>(m[t][1])};
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = at_exp2(w[i] - base[i & 1]);
      l[t][0] += w[0] + w[2];
      l[t][1] += w[1] + w[3];
      p[t][0] = movmatrix(AtType<T>::pack(w[0], w[1]));
      p[t][1] = movmatrix(AtType<T>::pack(w[2], w[3]));
    }
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const int r = (lane & 7) + ((lane >> 4) << 3), ch = 2 * k + ((lane >> 3) & 1);
      uint32_t f[4];
      ldmatrix4t(f, vst + r * kRow + ((ch ^ (r & 7)) << 4));
#pragma unroll
      for (int t = 0; t < NQ; ++t) AtType<T>::mma(o[t][k], f, p[t][0], p[t][1]);
    }
    __syncwarp();  // the stage is read: the next round's copies may overwrite it
    if (now.tile + 1 == now.end) {
      const int64_t piece = sp_item(a, now.b, now.hc) + wid;
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], s);
          const int g = t * 8 + (lane & 3) * 2 + i;
          if (g < n) {
            const int64_t rec = piece * a.shape.chunk_rows + g;
            if (lane < 4) a.own_ml[rec] = make_float2(at_reference<T, kSpUp>(m[t][i]), broken ? kAtBadPage : l[t][i]);
            float *dst = a.own_o + rec * x.head_dim + (lane >> 2);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              if (k * 16 < x.head_dim) dst[k * 16] = o[t][k][i];
              if (k * 16 + 8 < x.head_dim) dst[k * 16 + 8] = o[t][k][2 + i];
            }
          }
        }
      }
      fresh = true;
    }
    if (++stage == kStages) stage = 0;
    sp_next(a, now);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  grid_wait();  // the merge that follows this grid reads the prefix kernel's records too
}

// Prefix kernel, where the prefix has more query rows than one chunk.  The
// rows' query heads of one key head are packed into tiles of 128 rows (M of
// the tcgen05 products), and a CTA takes one such tile over one part of the
// prefix, so that a key is read once for 128 query rows:
//
//   warps 0-3   softmax: a thread owns a row; 64 scores from tensor memory,
//               the weights (rounded to the cache's type) back over them
//   warps 4-5   copies of tiles of 64 keys (warp 4) and of their values (warp
//               5) into a ring of swizzled stages each: TMA boxes where a tile is
//               whole pages or within one, 16-byte asynchronous copies for other
//               page sizes and for the part-full last tile (what lies past the
//               prefix has to be zero)
//   warp 6      products: S = Q K^T into two buffers in turn, so that a tile's
//               scores are there when the last tile's weights are done; O += P V
//
// Two CTAs share an SM, so that one's latencies pass under the other's
// exponentials.  The maximum that the weights refer to moves only when a score
// passes it by 2^8 (the weights then stay below 2^8, or 2^15 in fp16, see
// at_reference): O is rescaled rarely.
//
// Bound by the latencies between a tile's steps (scores, maximum, exponentials,
// weights stored, products), which two CTAs hide in part; the exponentials (16
// a clock and SM) are the busiest pipe, 53 %: 128 x 64 scores are 512 clocks of exponentials and
// take about 700 (two CTAs on an SM: 1400 each), their products of 64-entry
// heads 64 each way.  512 rows of 14 / 2 heads of 64 behind 8192 keys: 29 us
// (15.3 GFLOP; the exponentials alone 14 us, the products 9), 46 us with the
// split kernel and the merge.  A quarter of the
// exponentials as polynomials on the FMA pipe gained 1 % and is not done.
constexpr int kPrThreads = 224;
constexpr int kPrRows = 128;
constexpr int kPrKeys = 64;    // keys of a tile
constexpr int kPrCols = 256;   // tensor memory: two buffers of S (P over it, two keys a column), then O
constexpr uint32_t kPrO = 2 * kPrKeys;
template <int DP>
constexpr int kPrStage = kPrKeys * DP * 2;
template <int DP>
constexpr int kPrStages = DP == 64 ? 4 : 2;  // of keys, and of values
template <int DP>
constexpr int kPrSharedBytes = 1024 + kPrRows * DP * 2 + 2 * kPrStages<DP> * kPrStage<DP>;

struct PrShared {
  uint64_t full[2][4], empty[2][4];  // of keys, of values
  uint64_t q_full, s_full[2], p_ready[2], pv_done, drained;
  uint32_t tmem;
  volatile int dead;  // a wait ran out: the records are kAtLate
  volatile int bad;   // a page of this part is outside the cache
};

// The largest of three values, and of 64.
__device__ __forceinline__ float at_max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float at_max64(const float (&s)[64]) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = s[i];
#pragma unroll
    for (int j = 4; j + 4 < 60; j += 8) t[i] = at_max3(t[i], s[i + j], s[i + j + 4]);
  }
  return at_max3(at_max3(t[0], t[1], at_max3(s[60], s[61], s[62])), t[2], fmaxf(t[3], s[63]));
}
// Two fp32 operations an instruction.
__device__ __forceinline__ float2 at_fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)),
        "l"(*reinterpret_cast<uint64_t *>(&c)));
  return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 at_add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
  return *reinterpret_cast<float2 *>(&d);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kPrThreads, 2)
    ms_attn_prefix_kernel(const __grid_constant__ AtArgs a, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap) {
  constexpr int KT = kPrKeys, kStages = kPrStages<DP>, kStage = kPrStage<DP>;
  extern __shared__ __align__(1024) unsigned char pr_raw[];
  __shared__ PrShared sh;
  unsigned char *qs = pr_raw + ((1024u - (smem_addr(pr_raw) & 1023u)) & 1023u);
  unsigned char *ring = qs + kPrRows * DP * 2;
  const ms_prefix_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // query tiles fastest: CTAs that run together read the same keys
  const int qt = blockIdx.x % a.pre_tiles;
  const int hs = blockIdx.x / a.pre_tiles;
  const int h = hs % a.shape.kv_heads, part = hs / a.shape.kv_heads;
  const int keys = (int)x.prefix_length;
  const int all = (keys + KT - 1) / KT;
  const int t0 = (int)((int64_t)all * part / a.pre_splits), t1 = (int)((int64_t)all * (part + 1) / a.pre_splits);
  const int tiles = t1 - t0;
  const int r0 = qt * kPrRows;
  const int live_rows = min(kPrRows, a.packed - r0);
  const int live_warps = (live_rows + 31) / 32;
  if (tid == 0) {
    for (int i = 0; i < 2 * kStages; ++i) {
      bar_init(&sh.full[i / kStages][i % kStages], 1);
      bar_init(&sh.empty[i / kStages][i % kStages], 1);
    }
    bar_init(&sh.q_full, 4);
    bar_init(&sh.s_full[0], 1);
    bar_init(&sh.s_full[1], 1);
    // one for each buffer: softmax may be two tiles ahead of the products' wait
    bar_init(&sh.p_ready[0], live_warps);
    bar_init(&sh.p_ready[1], live_warps);
    bar_init(&sh.pv_done, 1);
    bar_init(&sh.drained, 1);
    sh.dead = 0;
    sh.bad = 0;
    bar_init_fence();
  }
  if (warp == 6) tmem_alloc(&sh.tmem, kPrCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  grid_wait();  // the call's first kernel
  grid_release();

  if (warp < 4) {
    // the warp's 32 query rows, in 128-byte swizzled panels of 64 entries: a row is read by neighbouring lanes
    const int r = tid;
    {
      constexpr int kChunks = DP / 8, kRowsStep = 32 / kChunks;
      const int pr = r0 + r;
      int64_t at = -1;
      if (pr < a.packed) {
        const int64_t b = pr / a.shape.group;
        at = b * x.q_row + (int64_t)(h * a.shape.group + (pr - (int)b * a.shape.group)) * x.q_head;
      }
      const int chunk = lane % kChunks;
      uint4 v[32 / kRowsStep];
#pragma unroll
      for (int i = 0; i < 32 / kRowsStep; ++i) {
        const int64_t from = __shfl_sync(0xFFFFFFFFu, at, i * kRowsStep + lane / kChunks);
        v[i] = make_uint4(0, 0, 0, 0);
        if (from >= 0 && chunk * 8 < x.head_dim) {
          const T *src = static_cast<const T *>(x.q) + from + chunk * 8;
          if (a.q_wide) {
            v[i] = load_in(reinterpret_cast<const uint4 *>(src));
          } else {
            const unsigned short *p = reinterpret_cast<const unsigned short *>(src);
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = (uint32_t)load_in(p + 2 * k) | ((uint32_t)load_in(p + 2 * k + 1) << 16);
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 32 / kRowsStep; ++i) {
        const int row = warp * 32 + i * kRowsStep + lane / kChunks;
        *reinterpret_cast<uint4 *>(qs + (chunk >> 3) * kPrRows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) =
            v[i];
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) bar_arrive(&sh.q_full);
    }
    if (warp < live_warps) {
      const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
      const float kNone = __uint_as_float(0xFF800000u);
      const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
      float m = kNone;    // a score, raw
      float ref = kNone;  // what the weights refer to, in units of log2
      float2 l[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        const uint32_t buffer = lanes + (i & 1) * KT;
        ok = bar_wait_warp(&sh.s_full[i & 1], (i >> 1) & 1, sh.dead);
        if (!ok) break;
        tc_fence_after();
        float s[64];
        tmem_ld64(buffer, s);
        const int left = keys - (t0 + i) * KT;
        if (left < KT) {  // keys past the end leave nothing
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (j >= left) s[j] = kNone;
        }
        const float top = at_max64(s);
        const bool moved = (top - m) * a.scale_log2 > 8.f;  // not where both are -inf (a NaN)
        if (__any_sync(0xFFFFFFFFu, moved)) {
          const float next = moved ? at_reference<T, kPrUp>(top * a.scale_log2) : ref;
          const float f = ref == next ? 1.f : at_exp2(ref - next);
          ref = next;
          m = moved ? top : m;
#pragma unroll
          for (int j = 0; j < 2; ++j) l[j].x *= f, l[j].y *= f;
          if (i > 0) {  // O is at rest once the last tile's product is done (the one before is: S was waited for)
            ok = bar_wait_warp(&sh.pv_done, (i - 1) & 1, sh.dead);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < DP; c += 16) {
              uint32_t u[16];
              tmem_ld16(lanes + kPrO + c, u);
              tmem_wait_ld(u);
#pragma unroll
              for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(__uint_as_float(u[j]) * f);
              tmem_st16(lanes + kPrO + c, u);
            }
          }
        }
        // Past 2^20 the fused exponent s scale - ref would keep what rounding took from ref (whole units and more:
        // weights of 0 or infinity); there the difference of the raw scores, which is exact at the top, is scaled.
        float base = ref == kNone ? 0.f : ref;
        const bool far = fabsf(base) > kAtFar;
        if (__any_sync(0xFFFFFFFFu, far)) {
          const float from = far ? m : 0.f;
#pragma unroll
          for (int j = 0; j < 64; ++j) s[j] -= from;
          base = far ? 0.f : base;
        }
        const float2 base2 = make_float2(-base, -base);
        uint32_t u[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float2 e = at_fma2(make_float2(s[2 * j], s[2 * j + 1]), scale2, base2);
          const float2 w = make_float2(at_exp2(e.x), at_exp2(e.y));
          l[j & 1] = at_add2(l[j & 1], w);
          u[j] = AtType<T>::pack(w.x, w.y);
        }
        tmem_st32(buffer, u);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.p_ready[i & 1]);
      }
      // not pv_done: its phase may be two behind here, which its parity cannot tell from done
      if (ok) ok = bar_wait_warp(&sh.drained, 0, sh.dead) && !sh.dead;
      if (!ok) sh.dead = 1;
      tc_fence_after();
      const int pr = r0 + r;
      const int64_t rec = ((int64_t)part * a.shape.kv_heads + h) * a.packed + pr;
      // 32 columns at a time through the queries' memory (they have been used), so that a record's row is
      // written by neighbouring lanes
      unsigned char *turn = qs + warp * 4096;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        uint32_t u[32];
        tmem_ld32(lanes + kPrO + c, u);
        tmem_wait_ld32(u);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4 *>(turn + lane * 128 + ((j ^ (lane & 7)) << 4)) =
              make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
        __syncwarp();
        const int j = lane & 7;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * 4 + (lane >> 3);
          const uint4 v = *reinterpret_cast<const uint4 *>(turn + row * 128 + ((j ^ (row & 7)) << 4));
          if (r0 + warp * 32 + row < a.packed && c + j * 4 < x.head_dim)
            *reinterpret_cast<uint4 *>(a.pre_o + (rec - lane + row) * x.head_dim + c + j * 4) = v;
        }
        __syncwarp();
      }
      if (pr < a.packed) {
        // the copies' warps set `bad` before the last products could start
        const float sum = sh.bad ? kAtBadPage : (l[0].x + l[0].y) + (l[1].x + l[1].y);
        a.pre_ml[rec] = ok ? make_float2(ref, sum) : make_float2(0.f, kAtLate);
      }
    }
  } else if (warp < 6) {
    constexpr int kChunks = DP / 8;            // 16-byte chunks of a row
    constexpr int kRowsStep = 32 / kChunks;    // rows of one copy instruction
    constexpr int kPanels = DP / 64;
    const bool value = warp == 5;
    const int page_size = (int)x.page_size;
    uint64_t *full = sh.full[value], *empty = sh.empty[value];
    unsigned char *mine = ring + value * kStages * kStage;
    auto find = [&](int j, int &page, int &offset) {
      const int p = a.page_shift >= 0 ? j >> a.page_shift : j / page_size;
      offset = j - p * page_size;
      page = load_in(x.prefix_pages + p);
    };
    int stage = 0, phase = 1, i = 0;
    bool ok = true;
    if (a.tma) {  // tiles that lie in the prefix as a whole
      const int box = min(KT, page_size);  // rows of a TMA box: a lane's panel of one
      const int row = lane / kPanels * box, panel = lane % kPanels;
      const CUtensorMap *map = value ? &vmap : &kmap;
      const int last = min(tiles, keys / KT - t0);
      int page = 0, offset = 0;
      if (row < KT && last > 0) find(t0 * KT + row, page, offset);
      for (; i < last; ++i) {
        const int page_now = page, offset_now = offset;
        if (row < KT && i + 1 < last) find((t0 + i + 1) * KT + row, page, offset);
        ok = bar_wait_warp(&empty[stage], phase, sh.dead);
        if (!ok) break;
        if (lane == 0) bar_expect(&full[stage], kStage);
        __syncwarp();
        if (row < KT) {  // a page outside the cache is outside the map: zeros
          const bool good = page_now >= 0 && page_now < x.pages;
          if (!good) sh.bad = 1;
          tma_load_4d(mine + stage * kStage + panel * KT * 128 + row * 128, map, &full[stage], panel * 64, offset_now, h,
                      good ? page_now : -1);
        }
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    }
    // the rest: a copy's tile is announced once the next one's has been issued
    const T *cache = static_cast<const T *>(value ? x.cache_v : x.cache_k);
    const int64_t step_page = value ? x.cv_page : x.ck_page, step_token = value ? x.cv_token : x.ck_token,
                  step_head = value ? x.cv_head : x.ck_head;
    const int chunk = lane % kChunks;
    const bool inside = chunk * 8 < x.head_dim;
    int waiting = -1;  // stage of the tile issued last
    for (; i < tiles && ok; ++i) {
      int64_t at[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // a lane looks up two keys
        const int j = (t0 + i) * KT + k * 32 + lane;
        at[k] = -1;
        if (j < keys) {
          int page, offset;
          find(j, page, offset);
          if (page >= 0 && page < x.pages) at[k] = page * step_page + offset * step_token + h * step_head;
          else sh.bad = 1;
        }
      }
      ok = bar_wait_warp(&empty[stage], phase, sh.dead);
      if (!ok) break;
      const uint32_t dst = smem_addr(mine) + stage * kStage + (chunk >> 3) * KT * 128;
#pragma unroll
      for (int k = 0; k < KT / kRowsStep; ++k) {
        const int row = k * kRowsStep + lane / kChunks;
        const int64_t from = __shfl_sync(0xFFFFFFFFu, at[k * kRowsStep / 32], row & 31);
        const bool live = from >= 0 && inside;
        copy16(dst + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), cache + (live ? from + chunk * 8 : 0), live);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (waiting >= 0) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) bar_arrive(&full[waiting]);
      }
      waiting = stage;
      if (++stage == kStages) stage = 0, phase ^= 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (waiting >= 0) {
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) bar_arrive(&full[waiting]);
    }
    if (!ok) {  // boxes in flight: every stage's last phase, again bounded
      sh.dead = 1;
      for (int k = 0; k < kStages; ++k)
        if (k < stage || i >= kStages) bar_wait(&full[k], k < stage ? phase ^ 1 : phase);
    }
  } else {
    const uint32_t leader = tc_leader();
    constexpr uint32_t kQk = tc_idesc_f16<T>(KT, false), kPv = tc_idesc_f16<T>(DP, true);
    // descriptors of the first stage: later ones, and steps of a product, are added in units of 16 bytes
    const uint64_t qd = tc_desc(smem_addr(qs), 1024, 16), kd = tc_desc(smem_addr(ring), 1024, 16),
                   vd = tc_desc(smem_addr(ring + kStages * kStage), 1024, KT * 128);
    bool ok = bar_wait_warp(&sh.q_full, 0, sh.dead);
    auto scores = [&](int i) {
      const int stage = i % kStages;
      ok = ok && bar_wait_warp(&sh.full[0][stage], (i / kStages) & 1, sh.dead);
      if (!ok) return;
      tc_fence_after();
      const uint64_t k = kd + stage * (kStage >> 4);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        tc_mma_f16(leader, tmem + (i & 1) * KT, qd + (d >> 2) * (kPrRows * 8) + (d & 3) * 2, k + (d >> 2) * (KT * 8) + (d & 3) * 2,
                   kQk, d > 0);
      tc_commit(leader, &sh.s_full[i & 1]);
      tc_commit(leader, &sh.empty[0][stage]);
    };
    scores(0);
    if (tiles > 1) scores(1);
    for (int i = 0; i < tiles && ok; ++i) {
      const int stage = i % kStages;
      ok = bar_wait_warp(&sh.full[1][stage], (i / kStages) & 1, sh.dead) &&
           bar_wait_warp(&sh.p_ready[i & 1], (i >> 1) & 1, sh.dead);
      if (!ok) break;
      tc_fence_after();
      const uint64_t v = vd + stage * (kStage >> 4);
#pragma unroll
      for (int d = 0; d < KT / 16; ++d)
        tc_mma_f16_tmem(leader, tmem + kPrO, tmem + (i & 1) * KT + d * 8, v + d * 128, kPv, i > 0 || d > 0);
      tc_commit(leader, &sh.pv_done);
      tc_commit(leader, &sh.empty[1][stage]);
      if (i + 2 < tiles) {  // into the buffer whose weights have just been used
        ok = bar_wait_warp(&sh.pv_done, i & 1, sh.dead);
        if (ok) scores(i + 2);
      }
    }
    if (!ok) sh.dead = 1;
    tc_commit(leader, &sh.drained);
    bar_wait(&sh.drained, 0);  // products in flight end before tensor memory is freed
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 6) tmem_free(tmem, kPrCols);
}

// Merge: the records of a (row, query head) weighed by one warp of eight in a
// CTA, or by all sixteen of a CTA where there may be many records (kWarps); a
// record's entries are loaded before its weight is known.  What records stand
// for no result is added to the rows' statuses here.
constexpr int kMgNarrow = 8;  // warps of a CTA that each have an output of their own
constexpr int kMgWide = 16;   // warps of a CTA that share one

template <typename T, int DP, int kWarps>
__global__ void __launch_bounds__((kWarps > 1 ? kWarps : kMgNarrow) * 32)
    ms_attn_merge_kernel(const __grid_constant__ AtArgs a) {
  constexpr int kLanes = DP / 4;        // lanes of a record: four entries each
  constexpr int kSide = 32 / kLanes;    // records side by side
  constexpr int kBatch = 4;             // records in flight of a lane
  constexpr int kStep = kWarps * kSide;
  const float kNone = __uint_as_float(0xFF800000u);
  __shared__ float4 part[kWarps][kLanes];
  __shared__ float2 part_ml[kWarps];
  __shared__ int part_flags[kWarps];
  const ms_prefix_attention_args &x = a.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t out_row = kWarps > 1 ? blockIdx.x : (int64_t)blockIdx.x * kMgNarrow + warp;
  if (out_row >= a.shape.rows * a.shape.heads) return;  // warps alone
  const int64_t b = out_row / a.shape.heads;
  const int hq = (int)(out_row - b * a.shape.heads);
  const int h = hq / a.shape.group, g = hq - h * a.shape.group;
  const int c = g / kAtRows, hc = h * a.shape.chunks + c;
  const int raw = load_in(x.lengths + b), len = at_length(x, b);
  grid_wait();
  // the records: the row's own pieces, then the prefix's (the split kernel's or the prefix kernel's)
  const int64_t share = a.header->share, start = a.base[b];
  int64_t own = 0, pre = 0;
  int owns = 0, pres = 0;
  if (len > 0) {  // the warps whose shares meet the item's tiles
    const int64_t units = sp_units(len), u = start + hc * units, w = (u + kSpItem) / share;
    own = (sp_item(a, b, hc) + w) * a.shape.chunk_rows + g - c * kAtRows;
    owns = (int)((u + units - 1) / share - w) + 1;
  }
  const int packed_row = (int)b * a.shape.group + g;
  if (a.split_prefix) {
    const int64_t units = sp_units(a.split_prefix), u = h * units, w = (u + kSpItem) / share;
    pre = (sp_item(a, -1, h) + w) * a.shape.chunk_rows + packed_row;
    pres = (int)((u + units - 1) / share - w) + 1;
  } else if (a.pre_splits) {
    pre = (int64_t)h * a.packed + packed_row;
    pres = a.pre_splits;
  }
  const int64_t pre_step = a.split_prefix ? a.shape.chunk_rows : (int64_t)a.shape.kv_heads * a.packed;
  const float2 *pre_ml = a.split_prefix ? a.own_ml : a.pre_ml;
  const float *pre_o = a.split_prefix ? a.own_o : a.pre_o;
  const int pieces = owns + pres;
  const int side = lane / kLanes, d = (lane % kLanes) * 4;
  float top = kNone, sum = 0.f;
  int flags = 0;  // MS_ROW_* bits that the records stand for
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = (kWarps > 1 ? warp * kSide : 0) + side; __any_sync(0xFFFFFFFFu, p0 < pieces); p0 += kStep * kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int p = p0 + i * kStep;
      ml[i] = make_float2(kNone, 0.f);
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p < pieces) {
        const int64_t rec = p < owns ? own + (int64_t)p * a.shape.chunk_rows : pre + (p - owns) * pre_step;
        ml[i] = (p < owns ? a.own_ml : pre_ml)[rec];
        if (d < x.head_dim)
          v[i] = *reinterpret_cast<const float4 *>((p < owns ? a.own_o : pre_o) + rec * x.head_dim + d);
      }
    }
    float next = top;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) next = fmaxf(next, ml[i].x);
    const float f = top == next ? 1.f : at_exp2(top - next);
    top = next;
    sum *= f, y.x *= f, y.y *= f, y.z *= f, y.w *= f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float w = at_exp2(ml[i].x - (top == kNone ? 0.f : top));
      if (ml[i].y < 0.f) flags |= ml[i].y == kAtBadPage ? MS_ROW_BAD_PAGE : MS_ROW_WAIT_TIMEOUT;
      sum += w * ml[i].y;
      y.x += w * v[i].x, y.y += w * v[i].y, y.z += w * v[i].z, y.w += w * v[i].w;
    }
  }
  auto join = [&](float other, float other_sum, float4 other_y) {
    const float next = fmaxf(top, other), base = next == kNone ? 0.f : next;
    const float f = at_exp2(top - base), e = at_exp2(other - base);
    top = next;
    sum = sum * f + other_sum * e;
    y.x = y.x * f + other_y.x * e, y.y = y.y * f + other_y.y * e;
    y.z = y.z * f + other_y.z * e, y.w = y.w * f + other_y.w * e;
  };
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {
    const float other = __shfl_xor_sync(0xFFFFFFFFu, top, o), other_sum = __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    float4 v;
    v.x = __shfl_xor_sync(0xFFFFFFFFu, y.x, o), v.y = __shfl_xor_sync(0xFFFFFFFFu, y.y, o);
    v.z = __shfl_xor_sync(0xFFFFFFFFu, y.z, o), v.w = __shfl_xor_sync(0xFFFFFFFFu, y.w, o);
    join(other, other_sum, v);
  }
  flags = __reduce_or_sync(0xFFFFFFFFu, flags);
  if (kWarps > 1) {
    if (lane < kLanes) part[warp][lane] = y;
    if (lane == 0) part_ml[warp] = make_float2(top, sum), part_flags[warp] = flags;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll 5
    for (int i = 1; i < kWarps; ++i) join(part_ml[i].x, part_ml[i].y, part[i][lane % kLanes]);
    flags = __reduce_or_sync(0xFFFFFFFFu, part_flags[lane % kWarps]);
  }
  const bool empty = raw != len || flags != 0 || sum == 0.f;
  if (lane < kLanes && d < x.head_dim) {
    T *dst = static_cast<T *>(x.out) + b * x.out_row + hq * x.out_head + d;
    const float inv = 1.f / sum;
    const float e[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = AtType<T>::narrow(empty ? 0.f : e[i]);
  }
  if (lane == 0) {
    x.lse[out_row] = empty ? kNone : (top + log2f(sum)) * 0.6931471805599453f;
    if (flags) atomicOr(x.status + b, flags);  // one head's record may be late and another's not
  }
}

}  // namespace ms
