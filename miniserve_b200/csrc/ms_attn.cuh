// Attention over a paged cache: arguments, the split kernel (rows' own keys,
// and the prefix's where few rows share it) and the merge.
#pragma once

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
constexpr int kSpCtas = 2;               // split CTAs of an SM
constexpr int kSpTile = 16;              // keys of a split tile: the M of the warp products
constexpr int kSpItem = 2;               // cost of an item's queries and record, in tiles
constexpr int kSpRing = 24 * 1024;       // bytes of one warp's ring of tiles
constexpr int kSpShared = kSpRing * kSpWarps;

struct AtHeader {
  int64_t share;       // tiles of one split warp
  int32_t prefix_bad;  // a page of the prefix is outside the cache
};

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
  float2 *own_ml;   // [pieces][chunk_rows] (m in units of log2, l)
  float *pre_o;     // [splits][kv_heads][packed rows][head_dim], of the prefix kernel
  float2 *pre_ml;   // [splits][kv_heads][packed rows]
  float scale_log2;
  int packed;        // rows * group: the prefix's query rows of one key head, row b's heads at b * group
  int split_prefix;  // keys of the prefix that the split kernel takes: all or none
  int pre_splits;    // parts of the prefix that the prefix kernel takes; 0 where it does not run
  int pre_tiles;     // its query tiles of one key head
  int q_wide;        // q's heads start 16-byte aligned
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
  const int n = __ldg(x.lengths + b);
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
__device__ __forceinline__ int64_t sp_tiles(int64_t keys) { return (keys + kSpTile - 1) / kSpTile; }
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
template <typename T, int DP, int NQ, bool kWhole>
__global__ void __launch_bounds__(kSpWarps * 32, kSpCtas)
    ms_attn_split_kernel(const __grid_constant__ AtArgs a) {
  constexpr int kRow = DP * 2;                 // bytes of a key's row in the ring
  constexpr int kChunks = DP / 8;              // 16-byte chunks of a row
  constexpr int kStage = 2 * kSpTile * kRow;   // K, then V
  constexpr int kStages = kSpRing / kStage;
  constexpr int kRowsStep = 32 / kChunks;      // rows of one copy instruction
  constexpr int kThreads = kSpWarps * 32;
  const float kNone = __uint_as_float(0xFF800000u);
  extern __shared__ __align__(128) unsigned char sp_ring[];
  __shared__ int64_t sums[kThreads + 1];  // units of the rows before each thread's run of rows, of one key head and chunk
  __shared__ int64_t warp_sums[kSpWarps];
  __shared__ int bad;
  grid_release();
  const ms_prefix_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t rows = a.shape.rows;
  const int hcs = a.shape.kv_heads * a.shape.chunks;
  const int64_t run = (rows + kThreads - 1) / kThreads;
  const int64_t r0 = min(rows, tid * run), r1 = min(rows, r0 + run);
  {
    int64_t n = 0;
    for (int64_t b = r0; b < r1; ++b) n += sp_units(at_length(x, b));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xFFFFFFFFu, n, o);
      if (lane >= o) n += v;
    }
    if (lane == 31) warp_sums[warp] = n;
    if (tid == 0) sums[0] = 0, bad = 0;
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
  if (blockIdx.x == 0) {  // for the merge: where each row starts, and whether the prefix's pages are good
    int64_t n = sums[tid];
    for (int64_t b = r0; b < r1; ++b) {
      a.base[b] = before + n * hcs;
      n += sp_units(at_length(x, b));
    }
    const int64_t pages = (x.prefix_length + x.page_size - 1) / x.page_size;
    int seen = 0;
    for (int64_t p = tid; p < pages; p += kThreads) {
      const int32_t id = __ldg(x.prefix_pages + p);
      seen |= id < 0 || id >= x.pages;
    }
    if (seen) bad = 1;
    __syncthreads();
    if (tid == 0) a.header->share = share, a.header->prefix_bad = bad;
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
  const uint32_t ring = smem_addr(sp_ring) + warp * kSpRing;
  const int page_size = (int)x.page_size;
  const int chunk = lane % kChunks;
  const bool inside = chunk * 8 < x.head_dim;

  // One page for all lanes where tiles lie in one; else lanes 0-15 look up
  // the tile's keys for K, lanes 16-31 for V.
  int page = -1, offset = 0, head = 0, live_keys = 0;
  auto look = [&]() {
    page = -1;
    if (load.tile < load.end) {
      const int j = load.tile * kSpTile + (kWhole ? 0 : lane & 15);
      live_keys = load.keys - load.tile * kSpTile;
      if (j < load.keys) {
        const int p = j / page_size;
        offset = j - p * page_size;
        page = __ldg(load.b < 0 ? x.prefix_pages + p : x.table + load.b * x.table_row + p);
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
  bool fresh = true;
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
              u = __ldg(reinterpret_cast<const unsigned int *>(q + k * 8));
            } else {
              const unsigned short *p = reinterpret_cast<const unsigned short *>(q + k * 8);
              u = (uint32_t)__ldg(p) | ((uint32_t)__ldg(p + 1) << 16);
            }
          }
          qf[t][k >> 1][k & 1] = u;
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
        m[t][0] = m[t][1] = kNone;
        l[t][0] = l[t][1] = 0.f;
      }
      fresh = false;
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
          const float f = m[t][i] == top[i] ? 1.f : at_exp2(m[t][i] - top[i]);
          m[t][i] = top[i];
          l[t][i] *= f;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) o[t][k][i] *= f, o[t][k][2 + i] *= f;
        }
      }
      // a score of -inf has weight 0 whatever the maximum
      const float base[2] = {m[t][0] == kNone ? 0.f : m[t][0], m[t][1] == kNone ? 0.f : m[t][1]};
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
            if (lane < 4) a.own_ml[rec] = make_float2(m[t][i], l[t][i]);
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
//   warps 0-3   softmax: a thread owns a row; scores from tensor memory, the
//               weights (rounded to the cache's type) back to tensor memory
//   warps 4-5   copies: 16-byte asynchronous copies of key and value tiles
//               into a ring of swizzled 16 KB stages, pages looked up on the way
//   warp 6      products: S = Q K^T of the next tile ahead of O += P V of this
//
// Two CTAs share an SM, so that one's products run under the other's softmax.
// The maximum that the weights refer to moves only when a score passes it by
// 2^8 (the weights then stay below 2^8, within fp16): O is rescaled rarely.
//
// Bound by the exponentials (16 a clock and SM): 128 x 128 scores are 1024
// clocks, their products of 64-entry heads about 256.
constexpr int kPrThreads = 224;
constexpr int kPrRows = 128;
constexpr int kPrStage = 16 * 1024;
constexpr int kPrCols = 256;  // tensor memory: S, then P (two keys a column), then O
template <int DP>
constexpr int kPrKeys = kPrStage / (DP * 2);  // keys of a tile: 128, or 64 of 128-entry heads
template <int DP>
constexpr int kPrStages = DP == 64 ? 5 : 4;
template <int DP>
constexpr int kPrSharedBytes = 1024 + kPrRows * DP * 2 + kPrStages<DP> * kPrStage;

struct PrShared {
  uint64_t full[5], empty[5];
  uint64_t q_full, s_full, p_ready, pv_done, drained;
  uint32_t tmem;
  volatile int dead;  // a wait ran out: the records are NaN
};

__device__ __forceinline__ void tmem_ld64(uint32_t addr, float (&r)[64]) {
  uint32_t u[64];
#pragma unroll
  for (int i = 0; i < 2; ++i) tmem_ld32(addr + 32 * i, u + 32 * i);
  tmem_wait_ld64(u);
#pragma unroll
  for (int i = 0; i < 64; ++i) r[i] = __uint_as_float(u[i]);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kPrThreads, 2) ms_attn_prefix_kernel(const __grid_constant__ AtArgs a) {
  constexpr int KT = kPrKeys<DP>, kStages = kPrStages<DP>;
  constexpr uint32_t kP = KT, kO = KT + KT / 2;  // columns of P and O
  extern __shared__ __align__(1024) unsigned char pr_raw[];
  __shared__ PrShared sh;
  grid_release();
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
    for (int i = 0; i < kStages; ++i) {
      bar_init(&sh.full[i], 2);
      bar_init(&sh.empty[i], 1);
    }
    bar_init(&sh.q_full, 4);
    bar_init(&sh.s_full, 1);
    bar_init(&sh.p_ready, live_warps);
    bar_init(&sh.pv_done, 1);
    bar_init(&sh.drained, 1);
    sh.dead = 0;
    bar_init_fence();
  }
  if (warp == 6) tmem_alloc(&sh.tmem, kPrCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp < 4) {
    // this thread's query row, in 128-byte swizzled panels of 64 entries
    const int r = tid;
    {
      const int pr = r0 + r;
      const bool live = pr < a.packed;
      const int64_t b = live ? pr / a.shape.group : 0;
      const int head = h * a.shape.group + (live ? pr - (int)b * a.shape.group : 0);
      const T *src = static_cast<const T *>(x.q) + b * x.q_row + head * x.q_head;
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live && c * 8 < x.head_dim) {
          if (a.q_wide) {
            v = __ldg(reinterpret_cast<const uint4 *>(src + c * 8));
          } else {
            const unsigned short *p = reinterpret_cast<const unsigned short *>(src + c * 8);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(p + 2 * i) | ((uint32_t)__ldg(p + 2 * i + 1) << 16);
            v = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        *reinterpret_cast<uint4 *>(qs + (c >> 3) * kPrRows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) bar_arrive(&sh.q_full);
    }
    if (warp < live_warps) {
      const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
      const float kNone = __uint_as_float(0xFF800000u);
      float m = kNone, l = 0.f;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        ok = !sh.dead && bar_wait(&sh.s_full, i & 1);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
        const int key0 = (t0 + i) * KT;
        const bool cut = key0 + KT > keys;
        float s[64];
        float top = kNone;
#pragma unroll
        for (int half = 0; half < KT / 64; ++half) {  // the last half stays in registers
          tmem_ld64(lanes + half * 64, s);
          if (cut) {
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (key0 + half * 64 + j >= keys) s[j] = kNone;
          }
#pragma unroll
          for (int j = 0; j < 64; ++j) top = fmaxf(top, s[j]);
        }
        top *= a.scale_log2;
        const bool moved = top > m + 8.f || (m == kNone && top != kNone);
        bool waited = i == 0;
        if (__any_sync(0xFFFFFFFFu, moved)) {
          const float next = moved ? top : m;
          const float f = m == next ? 1.f : at_exp2(m - next);
          m = next;
          l *= f;
          if (i > 0) {
            ok = __all_sync(0xFFFFFFFFu, bar_wait(&sh.pv_done, (i - 1) & 1));
            if (!ok) break;
            waited = true;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
              uint32_t u[32];
              tmem_ld32(lanes + kO + c, u);
              tmem_wait_ld32(u);
#pragma unroll
              for (int j = 0; j < 32; ++j) u[j] = __float_as_uint(__uint_as_float(u[j]) * f);
              tmem_st32(lanes + kO + c, u);
            }
          }
        }
        const float base = m == kNone ? 0.f : m;
#pragma unroll
        for (int half = KT / 64 - 1; half >= 0; --half) {
          if (half != KT / 64 - 1) {
            tmem_ld64(lanes + half * 64, s);
                    if (cut) {
#pragma unroll
              for (int j = 0; j < 64; ++j)
                if (key0 + half * 64 + j >= keys) s[j] = kNone;
            }
          }
          uint32_t u[32];
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float e0 = at_exp2(fmaf(s[2 * j], a.scale_log2, -base));
            const float e1 = at_exp2(fmaf(s[2 * j + 1], a.scale_log2, -base));
            sum0 += e0;
            sum1 += e1;
            u[j] = AtType<T>::pack(e0, e1);
          }
          l += sum0 + sum1;
          if (!waited) {  // the previous tile's weights are still being read
            ok = __all_sync(0xFFFFFFFFu, bar_wait(&sh.pv_done, (i - 1) & 1));
            waited = true;
            tc_fence_after();
          }
          tmem_st32(lanes + kP + half * 32, u);
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.p_ready);
      }
      if (ok) ok = __all_sync(0xFFFFFFFFu, bar_wait(&sh.pv_done, (tiles - 1) & 1));
      if (!ok) sh.dead = 1;
      tc_fence_after();
      const int pr = r0 + r;
      const int64_t rec = ((int64_t)part * a.shape.kv_heads + h) * a.packed + pr;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t u[32];
        tmem_ld32(lanes + kO + c, u);
        tmem_wait_ld32(u);
        if (pr < a.packed) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (c + j < x.head_dim)
              *reinterpret_cast<uint4 *>(a.pre_o + rec * x.head_dim + c + j) =
                  make_uint4(u[j], u[j + 1], u[j + 2], u[j + 3]);
        }
      }
      if (pr < a.packed) a.pre_ml[rec] = ok ? make_float2(m, l) : make_float2(0.f, __uint_as_float(0x7FC00000u));
    }
  } else if (warp < 6) {
    constexpr int kRowsWarp = KT / 2;          // rows of a tile that one warp copies
    constexpr int kChunks = DP / 8;            // 16-byte chunks of a row
    constexpr int kRowsStep = 32 / kChunks;    // rows of one copy instruction
    constexpr int kLook = kRowsWarp / 32;      // rows that a lane looks up
    const int w = warp - 4, page_size = (int)x.page_size;
    const int count = 2 * tiles;  // loads: K0, then K(i + 1) and V(i) in turn, V of the last tile
    auto tile_of = [&](int n, bool &value) {
      // n = 0: K(0); 2i + 1: K(i + 1), 2i + 2: V(i); the last one is the last tile's V
      value = n == count - 1 || (n > 0 && (n & 1) == 0);
      return n == count - 1 ? tiles - 1 : value ? (n >> 1) - 1 : (n + 1) >> 1;
    };
    int page[kLook], offset[kLook];
    auto look = [&](int n) {
      bool value;
      const int tile = n < count ? tile_of(n, value) : 0;
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        const int j = (t0 + tile) * KT + w * kRowsWarp + i * 32 + lane;
        page[i] = -1;
        if (n < count && j < keys) {
          const int p = j / page_size;
          offset[i] = j - p * page_size;
          page[i] = __ldg(x.prefix_pages + p);
        }
      }
    };
    look(0);
    int stage = 0, phase = 1, sent = 0;
    bool ok = true;
    for (int n = 0; n < count; ++n) {
      bool value;
      tile_of(n, value);
      int64_t at[kLook];
#pragma unroll
      for (int i = 0; i < kLook; ++i)
        at[i] = page[i] < 0 || page[i] >= x.pages ? -1
                : value ? page[i] * x.cv_page + offset[i] * x.cv_token + h * x.cv_head
                        : page[i] * x.ck_page + offset[i] * x.ck_token + h * x.ck_head;
      look(n + 1);
      ok = !sh.dead && bar_wait(&sh.empty[stage], phase);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      const T *src = static_cast<const T *>(value ? x.cache_v : x.cache_k);
      const uint32_t dst = smem_addr(ring) + stage * kPrStage;
      const int chunk = lane % kChunks;
#pragma unroll
      for (int i = 0; i < kRowsWarp / kRowsStep; ++i) {
        const int rr = i * kRowsStep + lane / kChunks;
        const int64_t from = __shfl_sync(0xFFFFFFFFu, at[i * kRowsStep / 32], rr & 31);
        const bool live = from >= 0 && chunk * 8 < x.head_dim;
        const int row = w * kRowsWarp + rr;
        copy16(dst + (chunk >> 3) * KT * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4),
               src + (live ? from + chunk * 8 : 0), live);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (n >= 2) {  // two loads in flight: the one before them has landed
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.full[sent]);
        if (++sent == kStages) sent = 0;
      }
      if (++stage == kStages) stage = 0, phase ^= 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_async_proxy();
    __syncwarp();
    if (ok) {
      for (int n = count < 2 ? 0 : count - 2; n < count; ++n) {
        if (lane == 0) bar_arrive(&sh.full[sent]);
        if (++sent == kStages) sent = 0;
      }
    } else {
      sh.dead = 1;
    }
  } else if (lane == 0) {
    constexpr uint32_t kQk = tc_idesc_f16<T>(KT, false), kPv = tc_idesc_f16<T>(DP, true);
    const uint32_t q0 = smem_addr(qs), k0 = smem_addr(ring);
    int stage = 0, phase = 0;
    bool ok = bar_wait(&sh.q_full, 0);
    auto next = [&]() {
      if (++stage == kStages) stage = 0, phase ^= 1;
    };
    auto scores = [&]() {  // S of the tile in the present stage
      ok = ok && !sh.dead && bar_wait(&sh.full[stage], phase);
      if (!ok) return;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t panel = k >> 2, step = (k & 3) * 32;
        tc_mma_f16(tmem, tc_desc(q0 + panel * kPrRows * 128 + step, 1024, 16),
                   tc_desc(k0 + stage * kPrStage + panel * KT * 128 + step, 1024, 16), kQk, k > 0);
      }
      tc_commit(&sh.empty[stage]);
      tc_commit(&sh.s_full);
      next();
    };
    scores();
    for (int i = 0; i < tiles && ok; ++i) {
      ok = !sh.dead && bar_wait(&sh.p_ready, i & 1);
      if (!ok) break;
      tc_fence_after();
      if (i + 1 < tiles) scores();
      ok = ok && bar_wait(&sh.full[stage], phase);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < KT / 16; ++k)
        tc_mma_f16_tmem(tmem + kO, tmem + kP + k * 8, tc_desc(k0 + stage * kPrStage + k * 2048, 1024, KT * 128), kPv,
                        i > 0 || k > 0);
      tc_commit(&sh.empty[stage]);
      tc_commit(&sh.pv_done);
      next();
    }
    if (!ok) sh.dead = 1;
    tc_commit(&sh.drained);
    bar_wait(&sh.drained, 0);  // products in flight end before tensor memory is freed
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 6) tmem_free(tmem, kPrCols);
}

// Merge: one CTA per (row, query head) weighs the records of its pieces; the
// rows' statuses are found here.
constexpr int kMgThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kMgThreads) ms_attn_merge_kernel(const __grid_constant__ AtArgs a) {
  __shared__ float red[2 * kMgThreads / 32];
  __shared__ int flag;
  __shared__ float acc[kMgThreads / 32][128];
  const ms_prefix_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.x / a.shape.heads;
  const int hq = (int)(blockIdx.x - b * a.shape.heads);
  const int h = hq / a.shape.group, g = hq - h * a.shape.group;
  const int c = g / kAtRows, hc = h * a.shape.chunks + c;
  const int raw = __ldg(x.lengths + b);
  const int len = at_length(x, b);
  if (tid == 0) flag = raw != len ? MS_ROW_BAD_LENGTH : MS_ROW_OK;
  __syncthreads();
  {
    const int64_t pages = ((int64_t)len + x.page_size - 1) / x.page_size;
    bool bad = false;
    for (int64_t p = tid; p < pages; p += kMgThreads) {
      const int32_t id = __ldg(x.table + b * x.table_row + p);
      bad |= id < 0 || id >= x.pages;
    }
    if (bad) atomicOr(&flag, MS_ROW_BAD_PAGE);
  }
  grid_wait();
  if (tid == 0 && a.header->prefix_bad) atomicOr(&flag, MS_ROW_BAD_PAGE);
  // the records: the row's own pieces, then the prefix's (the split kernel's or the prefix kernel's)
  const int64_t share = a.header->share;
  int64_t own = 0, pre = 0;
  int owns = 0, pres = 0;
  {
    const int64_t units = sp_units(len);
    if (units > 0) {  // the warps whose shares meet the item's tiles
      const int64_t u = a.base[b] + hc * units, w = (u + kSpItem) / share;
      own = (sp_item(a, b, hc) + w) * a.shape.chunk_rows + g - c * kAtRows;
      owns = (int)((u + units - 1) / share - w) + 1;
    }
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
  auto ml_of = [&](int p) {
    return p < owns ? a.own_ml[own + (int64_t)p * a.shape.chunk_rows] : pre_ml[pre + (p - owns) * pre_step];
  };
  float top = __uint_as_float(0xFF800000u);
  for (int p = tid; p < pieces; p += kMgThreads) top = fmaxf(top, ml_of(p).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMgThreads / 32; ++i) top = fmaxf(top, red[i]);
  const float base = top == __uint_as_float(0xFF800000u) ? 0.f : top;
  float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p = warp; p < pieces; p += kMgThreads / 32) {
    const float2 ml = ml_of(p);
    const float w = at_exp2(ml.x - base);
    sum += w * ml.y;
    const float *src = p < owns ? a.own_o + (own + (int64_t)p * a.shape.chunk_rows) * x.head_dim
                                : pre_o + (pre + (p - owns) * pre_step) * x.head_dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d < x.head_dim) y[i] += w * src[d];
    }
  }
  if (lane == 0) red[kMgThreads / 32 + warp] = sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[warp][lane + 32 * i] = y[i];
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMgThreads / 32; ++i) sum += red[kMgThreads / 32 + i];
  const int st = flag;
  const bool empty = st != MS_ROW_OK || sum == 0.f;
  if (tid < x.head_dim) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kMgThreads / 32; ++i) v += acc[i][tid];
    T *dst = static_cast<T *>(x.out) + b * x.out_row + hq * x.out_head;
    dst[tid] = AtType<T>::narrow(empty ? 0.f : v / sum);
  }
  if (tid == 0) {
    x.lse[b * a.shape.heads + hq] =
        empty ? __uint_as_float(0xFF800000u) : (base + log2f(sum)) * 0.6931471805599453f;
    if (hq == 0) x.status[b] = st;
  }
}

}  // namespace ms
