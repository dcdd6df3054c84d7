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

constexpr int kAtRows = 16;              // query heads of one chunk: the M of the warp products
constexpr int64_t kAtMaxRows = 1 << 20;  // rows of a call
constexpr int kAtMaxKeys = 0x3FFFFFFF;   // of the prefix, and of a row: their sum is an int
constexpr int kSpWarps = 4;              // warps of a split CTA
constexpr int kSpCtas = 2;               // split CTAs of an SM
constexpr int kSpTile = 16;              // keys of a split tile
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
  int chunk_rows;  // query heads of a record
  int64_t split_warps;
};

struct AtArgs {
  ms_prefix_attention_args x;
  AtShape shape;
  AtHeader *header;
  int64_t *base;    // [rows] tiles of the rows before
  float *own_o;     // [pieces][chunk_rows][head_dim]
  float2 *own_ml;   // [pieces][chunk_rows] (m in units of log2, l)
  float scale_log2;
  int split_prefix;  // keys of the prefix that every row's split tiles start with
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

// Walks over (row, key head and chunk, tile) in order.
struct SpWalk {
  int64_t b;
  int hc, tile, tiles, keys;
  int64_t left;  // tiles of this warp still to visit, the present one among them
};

__device__ __forceinline__ void sp_row(const AtArgs &a, SpWalk &w) {
  w.keys = a.split_prefix + at_length(a.x, w.b);
  w.tiles = (w.keys + kSpTile - 1) / kSpTile;
}
__device__ __forceinline__ void sp_next(const AtArgs &a, SpWalk &w) {
  if (--w.left <= 0) return;
  if (++w.tile < w.tiles) return;
  w.tile = 0;
  if (++w.hc < a.shape.kv_heads * a.shape.chunks) return;
  w.hc = 0;
  do {  // a later row has tiles: some are left
    ++w.b;
    sp_row(a, w);
  } while (w.tiles == 0);
}

// Split kernel.  The tiles of 16 keys of all rows and key heads form one
// sequence; every warp takes an equal, contiguous share of it, whatever the
// rows' lengths, and works alone: a ring of tiles filled with 16-byte
// asynchronous copies, a page lookup one tile ahead of its copies, and
// products of m16n8k16 (the chunk's query heads are the M).  Where its share
// meets an item (row, key head, chunk), it leaves one record at index item +
// warp, which is unique because both only grow along the sequence.
//
// Bound by the bytes of the cache: a tile of 64-entry heads is 4 KB and costs
// the products of 16 rows whatever the group, far below their rate.
template <typename T, int DP>
__global__ void __launch_bounds__(kSpWarps * 32, kSpCtas)
    ms_attn_split_kernel(const __grid_constant__ AtArgs a) {
  constexpr int kRow = DP * 2;                 // bytes of a key's row in the ring
  constexpr int kChunks = DP / 8;              // 16-byte chunks of a row
  constexpr int kStage = 2 * kSpTile * kRow;   // K, then V
  constexpr int kStages = kSpRing / kStage;
  constexpr int kRowsStep = 32 / kChunks;      // rows of one copy instruction
  extern __shared__ __align__(128) unsigned char sp_ring[];
  __shared__ int64_t sums[kSpWarps * 32 + 1];
  __shared__ int bad;
  grid_release();
  const ms_prefix_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t rows = a.shape.rows;
  const int hcs = a.shape.kv_heads * a.shape.chunks;
  // the rows' tiles before each thread's run of rows
  const int64_t run = (rows + kSpWarps * 32 - 1) / (kSpWarps * 32);
  const int64_t r0 = min(rows, tid * run), r1 = min(rows, r0 + run);
  {
    int64_t n = 0;
    for (int64_t b = r0; b < r1; ++b) n += (a.split_prefix + at_length(x, b) + kSpTile - 1) / kSpTile;
    sums[tid + 1] = n;
    if (tid == 0) sums[0] = 0, bad = 0;
    __syncthreads();
    for (int o = 1; o < kSpWarps * 32; o <<= 1) {
      const int64_t v = tid >= o ? sums[tid + 1 - o] : 0;
      __syncthreads();
      sums[tid + 1] += v;
      __syncthreads();
    }
  }
  const int64_t total = sums[kSpWarps * 32] * hcs;
  const int64_t share = max((int64_t)1, (total + a.shape.split_warps - 1) / a.shape.split_warps);
  if (blockIdx.x == 0) {  // for the merge: where each row's tiles start, and whether the prefix's pages are good
    int64_t n = sums[tid];
    for (int64_t b = r0; b < r1; ++b) {
      a.base[b] = n;
      n += (a.split_prefix + at_length(x, b) + kSpTile - 1) / kSpTile;
    }
    const int64_t pages = (x.prefix_length + x.page_size - 1) / x.page_size;
    int seen = 0;
    for (int64_t p = tid; p < pages; p += kSpWarps * 32) {
      const int32_t id = __ldg(x.prefix_pages + p);
      seen |= id < 0 || id >= x.pages;
    }
    if (seen) bad = 1;
    __syncthreads();
    if (tid == 0) a.header->share = share, a.header->prefix_bad = bad;
  }
  const int64_t wid = (int64_t)blockIdx.x * kSpWarps + warp;
  const int64_t u0 = wid * share, u1 = min(total, u0 + share);
  if (u0 >= u1) return;
  SpWalk load;
  {  // the row that tile u0 of the sequence lies in: its thread's run, then the row
    int lo = 0, hi = kSpWarps * 32 - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid + 1] * hcs > u0) hi = mid;
      else lo = mid + 1;
    }
    load.b = min(rows, lo * run);
    int64_t first = sums[lo] * hcs;
    sp_row(a, load);
    while (first + (int64_t)load.tiles * hcs <= u0) {
      first += (int64_t)load.tiles * hcs;
      ++load.b;
      sp_row(a, load);
    }
    load.hc = (int)((u0 - first) / load.tiles);
    load.tile = (int)((u0 - first) - (int64_t)load.hc * load.tiles);
    load.left = u1 - u0;
  }
  SpWalk now = load;
  const uint32_t ring = smem_addr(sp_ring) + warp * kSpRing;
  const T *ck = static_cast<const T *>(x.cache_k), *cv = static_cast<const T *>(x.cache_v);
  const int page_size = (int)x.page_size;

  // lanes 0-15 look up the tile's keys for K, lanes 16-31 for V
  int page = -1, offset = 0, head = 0;
  auto look = [&]() {
    page = -1;
    if (load.left > 0) {
      const int j = load.tile * kSpTile + (lane & 15);
      if (j < load.keys) {
        const bool shared = j < a.split_prefix;
        const int i = shared ? j : j - a.split_prefix;
        const int p = i / page_size;
        offset = i - p * page_size;
        page = __ldg(shared ? x.prefix_pages + p : x.table + load.b * x.table_row + p);
      }
      head = load.hc / a.shape.chunks;
      sp_next(a, load);
    }
  };
  auto issue = [&](int stage) {
    int64_t at = -1;
    if (page >= 0 && page < x.pages)
      at = lane < 16 ? page * x.ck_page + offset * x.ck_token + head * x.ck_head
                     : page * x.cv_page + offset * x.cv_token + head * x.cv_head;
    const uint32_t dst = ring + stage * kStage;
    const int chunk = lane % kChunks;
#pragma unroll
    for (int i = 0; i < 2 * kSpTile / kRowsStep; ++i) {
      const int r = i * kRowsStep + lane / kChunks;  // 0-15: K, 16-31: V
      const int64_t from = __shfl_sync(0xFFFFFFFFu, at, r);
      const bool live = from >= 0 && chunk * 8 < x.head_dim;
      const T *src = (r < kSpTile ? ck : cv) + (live ? from + chunk * 8 : 0);
      copy16(dst + r * kRow + ((chunk ^ (r & 7)) << 4), src, live);
    }
  };

  look();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    issue(s);
    look();
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  bool fresh = true;
  int stage = 0;
  while (now.left > 0) {
    {
      const int ahead = stage == 0 ? kStages - 1 : stage - 1;
      issue(ahead);
      look();
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const int h = now.hc / a.shape.chunks, c = now.hc - h * a.shape.chunks;
    if (fresh) {
      const T *q = static_cast<const T *>(x.q) + now.b * x.q_row;
      const int n = min(kAtRows, a.shape.group - c * kAtRows);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int g = (lane >> 2) + (i & 1) * 8, d = k * 16 + (lane & 3) * 2 + (i >> 1) * 8;
          uint32_t u = 0;
          if (g < n && d < x.head_dim) {
            const unsigned short *p = reinterpret_cast<const unsigned short *>(
                q + (int64_t)(h * a.shape.group + c * kAtRows + g) * x.q_head + d);
            u = (uint32_t)__ldg(p) | ((uint32_t)__ldg(p + 1) << 16);
          }
          qf[k][i] = u;
        }
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      m[0] = m[1] = __uint_as_float(0xFF800000u);
      l[0] = l[1] = 0.f;
      fresh = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint32_t kst = ring + stage * kStage, vst = kst + kSpTile * kRow;
    float sc[2][4] = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const int r = (lane & 7) + ((lane >> 4) << 3), chunk = 2 * k + ((lane >> 3) & 1);
      uint32_t b[4];
      ldmatrix4(b, kst + r * kRow + ((chunk ^ (r & 7)) << 4));
      AtType<T>::mma(sc[0], qf[k], b[0], b[1]);
      AtType<T>::mma(sc[1], qf[k], b[2], b[3]);
    }
    // scores in units of log2; keys past the end leave nothing
    const int j0 = now.tile * kSpTile + (lane & 3) * 2;
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool seen = j0 + t * 8 + (i & 1) < now.keys;
        sc[t][i] = seen ? sc[t][i] * a.scale_log2 : __uint_as_float(0xFF800000u);
        top[i >> 1] = fmaxf(top[i >> 1], sc[t][i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
    }
    if (__any_sync(0xFFFFFFFFu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // both -inf (no score yet above it): nothing to rescale
        const float f = m[i] == top[i] ? 1.f : at_exp2(m[i] - top[i]);
        m[i] = top[i];
        l[i] *= f;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) o[n][2 * i] *= f, o[n][2 * i + 1] *= f;
      }
    }
    uint32_t p[4];
    {
      float w[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float base = m[i >> 1];
          w[t][i] = sc[t][i] == __uint_as_float(0xFF800000u) ? 0.f : at_exp2(sc[t][i] - base);
        }
      l[0] += (w[0][0] + w[0][1]) + (w[1][0] + w[1][1]);
      l[1] += (w[0][2] + w[0][3]) + (w[1][2] + w[1][3]);
      p[0] = AtType<T>::pack(w[0][0], w[0][1]);
      p[1] = AtType<T>::pack(w[0][2], w[0][3]);
      p[2] = AtType<T>::pack(w[1][0], w[1][1]);
      p[3] = AtType<T>::pack(w[1][2], w[1][3]);
    }
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      const int r = (lane & 7) + (((lane >> 3) & 1) << 3), chunk = 2 * n + (lane >> 4);
      uint32_t b[4];
      ldmatrix4t(b, vst + r * kRow + ((chunk ^ (r & 7)) << 4));
      AtType<T>::mma(o[2 * n], p, b[0], b[1]);
      AtType<T>::mma(o[2 * n + 1], p, b[2], b[3]);
    }
    __syncwarp();  // the stage is read: the next round's copies may overwrite it
    if (now.left == 1 || now.tile + 1 == now.tiles) {
      const int64_t piece = now.b * hcs + now.hc + wid;
      const int n = min(kAtRows, a.shape.group - c * kAtRows);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
        l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
        const int g = (lane >> 2) + i * 8;
        if (g < n) {
          const int64_t rec = piece * a.shape.chunk_rows + g;
          if ((lane & 3) == 0) a.own_ml[rec] = make_float2(m[i], l[i]);
          float *dst = a.own_o + rec * x.head_dim;
#pragma unroll
          for (int t = 0; t < DP / 8; ++t) {
            const int d = t * 8 + (lane & 3) * 2;
            if (d < x.head_dim) *reinterpret_cast<float2 *>(dst + d) = make_float2(o[t][2 * i], o[t][2 * i + 1]);
          }
        }
      }
      fresh = true;
    }
    if (++stage == kStages) stage = 0;
    sp_next(a, now);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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
  const int c = g / kAtRows, hcs = a.shape.kv_heads * a.shape.chunks, hc = h * a.shape.chunks + c;
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
  const int64_t tiles = ((int64_t)a.split_prefix + len + kSpTile - 1) / kSpTile;
  int64_t first = 0;
  int pieces = 0;
  if (tiles > 0) {
    const int64_t share = a.header->share, u = a.base[b] * hcs + hc * tiles;
    first = b * hcs + hc + u / share;
    pieces = (int)((u + tiles - 1) / share - u / share) + 1;
  }
  const int rr = g - c * kAtRows;
  float top = __uint_as_float(0xFF800000u);
  for (int p = tid; p < pieces; p += kMgThreads) top = fmaxf(top, a.own_ml[(first + p) * a.shape.chunk_rows + rr].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMgThreads / 32; ++i) top = fmaxf(top, red[i]);
  const float base = top == __uint_as_float(0xFF800000u) ? 0.f : top;
  float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p = warp; p < pieces; p += kMgThreads / 32) {
    const int64_t rec = (first + p) * a.shape.chunk_rows + rr;
    const float2 ml = a.own_ml[rec];
    const float w = at_exp2(ml.x - base);
    sum += w * ml.y;
    const float *src = a.own_o + rec * x.head_dim;
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
