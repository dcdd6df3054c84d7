// Attention over a paged cache held in 4 bits: arguments, the split kernels and
// the merge.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mssample.h"
#include "ms_attn.cuh"
#include "ms_kv4.cuh"
#include "ms_tc.cuh"

namespace ms {

constexpr int kA4Warps = 4;                // warps of a split CTA
constexpr int kA4Half = 16;                // keys of a product
constexpr int kA4Halves = 2, kA4Tile = kA4Halves * kA4Half;  // keys of a tile: they share copies, pages and checks
constexpr int kA4Item = 2;                 // cost of an item's queries and record, in tiles
constexpr int kA4Stages = 3;               // tiles of a warp's ring
constexpr float kA4Least = -3e38f;         // refers to nothing yet: every score is far above it
constexpr int64_t kA4MaxRows = 1 << 20;
constexpr int kA4MaxTokens = 1024;         // of a row
// Query rows of an item: up to eight in the narrow kernel, in the wide one as many
// sixteens as registers have room for; half of them where a query takes two rows
// (`fine`, below).  Two rows of 131072 keys, four queries a key head: 86 us narrow,
// 127 us wide.  128 rows of five tokens and seven heads a key head: 66 us as one
// item of three sixteens, 80 us as two of two, 69 us as three of one.
__host__ __device__ constexpr int a4_narrow(bool fine) { return fine ? 4 : 8; }
__host__ __device__ constexpr int a4_most(int groups, bool fine) { return (groups <= 2 ? 48 : 16) >> (fine ? 1 : 0); }
// Split CTAs of an SM, by what their registers allow.
__host__ __device__ constexpr int a4_narrow_ctas(int groups) { return groups <= 2 ? 4 : 3; }
__host__ __device__ constexpr int a4_wide_ctas(int groups, int sixteens) { return groups <= 2 && sixteens <= 1 ? 3 : 2; }

// A tile in a warp's ring: the keys' codes, the values', the
// keys' parameters, the values'.  A token's codes are an odd multiple of 16
// bytes apart, so that eight rows of 16 bytes lie in different banks.
template <int NG>
struct A4Ring {
  static constexpr int kRow = NG <= 2 ? 32 : NG * 16;  // bytes of a token's codes in the cache
  static constexpr int kPieces = kRow / 16;            // 16-byte pieces of them
  static constexpr int kPairs = NG <= 2 ? 2 : 4;       // pairs of parameters in the cache; 16 bytes here
  static constexpr int kPitch = NG <= 3 ? 48 : 80;
  static constexpr int kV = kA4Tile * kPitch, kKp = 2 * kV, kVp = kKp + kA4Tile * 16;
  static constexpr int kStage = kVp + kA4Tile * 16;
};
template <int NG>
constexpr int kA4NarrowShared = kA4Warps * kA4Stages * A4Ring<NG>::kStage;
template <int NG, int NP>
constexpr int kA4Queries = NP * (NG * 1024 + 512 + 256);  // bytes of a warp's queries in the wide kernel, their sums and m
template <int NG, int NP>
constexpr int kA4WideShared = kA4Warps * (kA4Stages * A4Ring<NG>::kStage + kA4Queries<NG, NP>);

struct A4Header {
  int64_t share;  // units of one split warp
};

struct A4Args {
  ms_kv4_attention_args x;
  K4Layout layout;
  int group;       // query heads of a key head
  int queries;     // tokens * group: query rows of a row's key head, token t's heads at t * group
  int chunks;      // items that they are split into
  int chunk_rows;  // query rows of an item, and of a record
  int64_t split_warps;
  A4Header *header;
  int64_t *base;   // [rows] where each row starts in the split kernel's sequence
  float *own_o;    // [pieces][chunk_rows][head_dim]
  float2 *own_ml;  // [pieces][chunk_rows] (reference in units of log2, l)
  float scale_log2;
  int q_wide;      // q's heads start 16-byte aligned
  int page_shift;  // log2 of the page size, or -1
  int merge_wide;  // the merge gives each output a CTA
  int64_t code_page, code_head;  // bytes of a page's codes of the keys, and of one head of it
};

// Keys of a row: its tokens' largest length; 0 where one of them does not fit
// the row's pages (the row is flagged).  `bad` says so.
__device__ __forceinline__ int a4_keys(const ms_kv4_attention_args &x, int64_t b, bool &bad) {
  int most = 0;
  bad = false;
  for (int t = 0; t < x.tokens; ++t) {
    const int n = load_in(x.lengths + b * x.length_row + t);
    bad = bad || n < 0 || n > kAtMaxKeys || (int64_t)n > x.table_width * x.cache.page_size;
    most = max(most, n);
  }
  return bad ? 0 : most;
}
__device__ __forceinline__ int64_t a4_units(int keys) { return keys > 0 ? (keys + kA4Tile - 1) / kA4Tile + kA4Item : 0; }

// Walks over a warp's tiles: the split kernel's sequence is rows' items (key
// head and chunk) in order, each of kA4Item units and one unit a tile.  A warp's
// share is far below 2^31 units (the kernel would run for days).
struct A4Walk {
  int b, left;  // left: units of the share past this item
  int hc, tile, end, keys;
};
// The next item's tiles within the share; tile == end where none are left.
__device__ __forceinline__ void a4_item_next(const A4Args &a, A4Walk &w) {
  w.tile = w.end = 0;
  if (w.left <= kA4Item) return;
  if (++w.hc >= a.x.cache.kv_heads * a.chunks) {
    w.hc = 0;
    do {  // a later row has keys: units are left
      bool bad;
      w.keys = a4_keys(a.x, ++w.b, bad);
    } while (w.keys == 0);
  }
  const int take = min(w.left, (w.keys + kA4Tile - 1) / kA4Tile + kA4Item);
  w.left -= take;
  w.end = take - kA4Item;
}

__device__ __forceinline__ void copy8(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(live ? 8 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix2(uint32_t (&r)[2], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix2t(uint32_t (&r)[2], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(addr)
               : "memory");
}
// d = a b + c, and d += a b.
__device__ __forceinline__ void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1, float c0, float c1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The upper eight rows of the product, of an A whose lower ones are zero.
__device__ __forceinline__ void a4_mma_top(float (&d)[2], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  [[maybe_unused]] float none0, none1;
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};"
      : "+f"(d[0]), "+f"(d[1]), "=f"(none0), "=f"(none1)
      : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
}
// movmatrix for values alone: the compiler may move it, as it may the products.
__device__ __forceinline__ uint32_t a4_turn(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t a4_pack(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// Of halves, subnormal ones too.
__device__ __forceinline__ uint32_t a4_add(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}
// Two weights as fp16, less what `rest` has of them as such: where it is all ones,
// what their rounding left.
template <bool kFine>
__device__ __forceinline__ uint32_t a4_weights(float x, float y, uint32_t rest) {
  const uint32_t whole = a4_pack(x, y);
  if (!kFine) return whole;
  const uint32_t less = whole & rest;
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&less));
  return a4_pack(x - f.x, y - f.y);
}
__device__ __forceinline__ float a4_low(uint32_t u) { return __low2float(*reinterpret_cast<const __half2 *>(&u)); }

__device__ __forceinline__ float2 a4_mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
  return *reinterpret_cast<float2 *>(&d);
}
// The groups' scales, times `by`, of a key (its parameters are at `params`) and of the next.
template <int NG>
__device__ __forceinline__ void a4_pair_scales(const unsigned char *params, float by, float2 (&s)[NG]) {
  uint32_t u[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (NG > 2) *reinterpret_cast<uint4 *>(u[i]) = *reinterpret_cast<const uint4 *>(params + i * 16);
    else *reinterpret_cast<uint2 *>(u[i]) = *reinterpret_cast<const uint2 *>(params + i * 16);
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) s[g] = a4_mul2(make_float2(a4_low(u[0][g]), a4_low(u[1][g])), make_float2(by, by));
}

// A CTA's start: where the shares of its warps begin.  False where this warp has
// none.  The last CTA (its own share is the last, often short) writes down for
// the merge where each row starts, and the rows' statuses.
__device__ __forceinline__ bool a4_begin(const A4Args &a, A4Walk &load) {
  constexpr int kThreads = kA4Warps * 32;
  __shared__ int64_t sums[kThreads + 1];  // units of the rows before each thread's run of rows, of one key head and chunk
  __shared__ int64_t warp_sums[kA4Warps];
  const ms_kv4_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t rows = x.rows;
  const int hcs = x.cache.kv_heads * a.chunks;
  const int64_t run = (rows + kThreads - 1) / kThreads;
  const int64_t r0 = min(rows, tid * run), r1 = min(rows, r0 + run);
  bool bad;
  {
    int64_t n = 0;
    for (int64_t b = r0; b < r1; ++b) n += a4_units(a4_keys(x, b, bad));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xFFFFFFFFu, n, o);
      if (lane >= o) n += v;
    }
    if (lane == 31) warp_sums[warp] = n;
    if (tid == 0) sums[0] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kA4Warps; ++i)
      if (i < warp) n += warp_sums[i];
    sums[tid + 1] = n;
    __syncthreads();
  }
  const int64_t total = sums[kThreads] * hcs;
  const int64_t share = max((int64_t)kA4Item + 1, (total + a.split_warps - 1) / a.split_warps);
  if (blockIdx.x == gridDim.x - 1) {
    int64_t n = sums[tid];
    for (int64_t b = r0; b < r1; ++b) {
      a.base[b] = n * hcs;
      const int keys = a4_keys(x, b, bad);
      x.status[b] = bad ? MS_ROW_BAD_LENGTH : MS_ROW_OK;
      n += a4_units(keys);
    }
    if (tid == 0) a.header->share = share;
  }
  const int64_t wid = (int64_t)blockIdx.x * kA4Warps + warp;
  const int64_t u0 = wid * share, u1 = min(total, u0 + share);
  if (u0 >= u1) return false;
  int lo = 0, hi = kThreads - 1;  // the row that unit u0 lies in: its thread's run, then the row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid + 1] * hcs > u0) hi = mid;
    else lo = mid + 1;
  }
  load.b = (int)min(rows, lo * run);
  int64_t first = sums[lo] * hcs;
  load.keys = a4_keys(x, load.b, bad);
  while (first + a4_units(load.keys) * hcs <= u0) {
    first += a4_units(load.keys) * hcs;
    load.keys = a4_keys(x, ++load.b, bad);
  }
  const int64_t units = a4_units(load.keys);
  load.hc = (int)((u0 - first) / units);
  const int64_t at = u0 - first - load.hc * units, take = min(u1 - u0, units - at);
  load.left = (int)(u1 - u0 - take);
  load.tile = (int)max((int64_t)0, at - kA4Item);
  load.end = (int)(at + take) - kA4Item;
  if (load.end <= load.tile) a4_item_next(a, load);
  return true;
}

// A warp's copies into its ring.  Where a half's keys lie in one page (kWhole),
// it is looked up once for all lanes; else lanes 0-15 (and 16-31 again) look up
// the half's keys.  Page ids are loaded a tile ahead of their use, and a tile's
// addresses are a page's, a head's and a lane's parts: this is work for every
// tile.
template <int NG, bool kWhole>
struct A4Copies {
  using R = A4Ring<NG>;
  static constexpr int kRow = R::kRow, kPieces = R::kPieces, kPairs = R::kPairs, kPitch = R::kPitch;
  static constexpr int kCopies = kA4Tile * kPieces / 32;  // of a tile's codes of the keys, and of the values

  const A4Args &a;
  A4Walk load;                  // at the tile that is copied next
  unsigned char *ring;
  int lane;
  int page[kA4Halves], offset[kA4Halves];
  const int *table = nullptr;   // of that tile's row
  int64_t head_at = 0;          // its head's codes in a page
  int live_keys = 0;            // of it; 0 where none is left
  uint32_t met = 0;             // bit i: the tile issued i tiles ago met a bad page

  __device__ __forceinline__ A4Copies(const A4Args &args, const A4Walk &walk, unsigned char *to)
      : a(args), load(walk), ring(to), lane(threadIdx.x & 31) {
    if (kPairs == 2) {  // the parameters' rows are 16 bytes here too: what lies behind the two pairs stays zero
      for (int s = 0; s < kA4Stages; ++s)
#pragma unroll
        for (int i = 0; i < kA4Halves; ++i)
          *reinterpret_cast<uint4 *>(ring + s * R::kStage + R::kKp + (i * 32 + lane) * 16) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    look(true);
#pragma unroll
    for (int s = 0; s < kA4Stages - 1; ++s) next(s);
  }
  // The next tile's copies, into a stage of the ring.
  __device__ __forceinline__ void next(int stage) {
    issue(stage);
    if (load.tile < load.end) {
      const bool item = ++load.tile >= load.end;
      if (item) a4_item_next(a, load);
      look(item);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Whether the tile whose turn it is, kA4Stages - 1 copies after its own, met a bad page.
  __device__ __forceinline__ bool broken() const { return (met >> (kA4Stages - 1)) & 1; }

 private:
  static __device__ __forceinline__ int64_t params_of(int64_t code) {
    return kPairs * 4 * 4 == kRow ? code >> 2 : code / kRow * (kPairs * 4);
  }
  __device__ __forceinline__ bool live(int i) const { return i * kA4Half + (kWhole ? 0 : lane & 15) < live_keys; }
  __device__ __forceinline__ bool in_cache(int i) const { return (unsigned)page[i] < (unsigned)a.x.cache.pages; }

  __device__ __forceinline__ void look(bool item) {  // at tile load.tile, the first of an item's or not
    live_keys = 0;
#pragma unroll
    for (int i = 0; i < kA4Halves; ++i) page[i] = offset[i] = 0;
    if (load.tile >= load.end) return;
    if (item) {
      head_at = load.hc / a.chunks * a.code_head;
      table = a.x.table + load.b * a.x.table_row;
    }
    const int page_size = (int)a.x.cache.page_size;
    live_keys = load.keys - load.tile * kA4Tile;
#pragma unroll
    for (int i = 0; i < kA4Halves; ++i) {
      const int j = load.tile * kA4Tile + i * kA4Half + (kWhole ? 0 : lane & 15);
      if (j < load.keys) {
        const int p = a.page_shift >= 0 ? j >> a.page_shift : j / page_size;
        offset[i] = a.page_shift >= 0 ? j & (page_size - 1) : j - p * page_size;
        page[i] = load_in(table + p);
      }
    }
  }
  __device__ __forceinline__ void issue(int stage) {
    const ms_kv4_cache &cache = a.x.cache;
    int64_t code[kA4Halves];  // the codes' place of a half's first key, or of the lane's
    bool wrong = false;
#pragma unroll
    for (int i = 0; i < kA4Halves; ++i) {
      wrong = wrong || (live(i) && !in_cache(i));
      code[i] = page[i] * a.code_page + head_at + (uint32_t)offset[i] * (int64_t)kRow;
    }
    met = (met << 1) | (kWhole ? wrong : __any_sync(0xFFFFFFFFu, wrong));
    const uint32_t dst = smem_addr(ring) + stage * R::kStage;
    if (kWhole && live_keys >= kA4Tile && !wrong) {  // all of the tile
      const unsigned char *ks = cache.k_codes + lane * 16, *vs = cache.v_codes + lane * 16;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        if (kPieces == 3) {
          const int at = i * 32 + lane, r = at / kPieces;
          const int64_t off = (r >= kA4Half ? code[1] - kA4Half * kRow : code[0]) + i * 512;
          const uint32_t to = dst + r * kPitch + (at - r * kPieces) * 16;
          copy16(to, ks + off, true);
          copy16(to + R::kV, vs + off, true);
        } else {
          constexpr int kEach = kCopies / kA4Halves;  // of a half
          const int64_t off = code[i / kEach] + i % kEach * 512;
          const uint32_t to = dst + lane / kPieces * kPitch + lane % kPieces * 16 + i * (32 / kPieces) * kPitch;
          copy16(to, ks + off, true);
          copy16(to + R::kV, vs + off, true);
        }
      }
      const int64_t off = params_of(lane >= 16 ? code[1] : code[0]) + (lane & 15) * (kPairs * 4);
      const char *kp = static_cast<const char *>(cache.k_params) + off, *vp = static_cast<const char *>(cache.v_params) + off;
      const uint32_t to = dst + R::kKp + lane * 16;
      copy_params(to, kp, true);
      copy_params(to + kA4Tile * 16, vp, true);
      return;
    }
    // the codes' place of key r of the tile, or -1
    auto code_of = [&](int r) {
      int64_t at = -1;
#pragma unroll
      for (int i = 0; i < kA4Halves; ++i) {
        const int64_t own = live(i) && in_cache(i) ? code[i] : -1;
        const int64_t from = kWhole ? (own >= 0 ? own + (r & 15) * kRow : -1) : __shfl_sync(0xFFFFFFFFu, own, r & 15);
        if (r >> 4 == i) at = from;
      }
      return r < live_keys ? at : -1;
    };
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = i * 32 + lane, r = at / kPieces, piece = at - r * kPieces;
      const int64_t from = code_of(r), off = from >= 0 ? from + piece * 16 : 0;
      copy16(dst + r * kPitch + piece * 16, cache.k_codes + off, from >= 0);
      copy16(dst + R::kV + r * kPitch + piece * 16, cache.v_codes + off, from >= 0);
    }
    const int64_t from = code_of(lane), off = from >= 0 ? params_of(from) : 0;
    const uint32_t to = dst + R::kKp + lane * 16;
    copy_params(to, static_cast<const char *>(cache.k_params) + off, from >= 0);
    copy_params(to + kA4Tile * 16, static_cast<const char *>(cache.v_params) + off, from >= 0);
  }
  static __device__ __forceinline__ void copy_params(uint32_t dst, const void *src, bool live) {
    if (kPairs == 4) copy16(dst, src, live);
    else copy8(dst, src, live);
  }
};

// A lane's eight entries 32 g + 8 c .. + 7 of every group of a query as they are
// stored, zeros where there is none.
template <int NG>
__device__ __forceinline__ void a4_query_load(const A4Args &a, bool live, int64_t at, uint32_t (&u)[NG][4]) {
  const int c = threadIdx.x & 3;
#pragma unroll
  for (int k = 0; k < NG; ++k) {
    u[k][0] = u[k][1] = u[k][2] = u[k][3] = 0;
    if (live && k * 32 + c * 8 < a.x.cache.head_dim) {
      const unsigned short *p = static_cast<const unsigned short *>(a.x.q) + at + c * 8 + k * 32;
      if (a.q_wide) {
        *reinterpret_cast<uint4 *>(u[k]) = load_in(reinterpret_cast<const uint4 *>(p));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[k][i] = (uint32_t)load_in(p + 2 * i) | ((uint32_t)load_in(p + 2 * i + 1) << 16);
      }
    }
  }
}
// They as fp16 scaled by a power of two that puts the row's largest in [2^5,
// 2^6): `down` undoes it.  As operands: the pairs of entries (0, 4), (1, 5) 2^-4,
// (2, 6) and (3, 7) 2^-4; and the groups' sums.
template <int NG>
__device__ __forceinline__ void a4_query(const A4Args &a, const uint32_t (&u)[NG][4], uint32_t (&f)[NG][4], float (&sum)[NG], float &down) {
  float most = 0.f;
  float e[NG][8];
#pragma unroll
  for (int k = 0; k < NG; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v;
      if (a.x.dtype == MS_DTYPE_BF16) v = make_float2(__uint_as_float(u[k][i] << 16), __uint_as_float(u[k][i] & 0xFFFF0000u));
      else v = __half22float2(*reinterpret_cast<const __half2 *>(&u[k][i]));
      e[k][2 * i] = v.x, e[k][2 * i + 1] = v.y;
      most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
    }
  }
  most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
  most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
  // 2^(5 - floor(log2 most)), as long as it and 1 over it are normal numbers
  const int power = most > 0.f ? min(126, 5 + 127 - (int)(__float_as_uint(most) >> 23)) : 0;
  const float up = __uint_as_float((uint32_t)(power + 127) << 23);
  down = __uint_as_float((uint32_t)(127 - power) << 23);
#pragma unroll
  for (int k = 0; k < NG; ++k) {
    sum[k] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[k][i] = __half2float(__float2half_rn(e[k][i] * up));
      sum[k] += e[k][i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float scale = i & 1 ? 0.0625f : 1.f;
      f[k][i] = a4_pack(e[k][i] * scale, e[k][i + 4] * scale);
    }
    sum[k] += __shfl_xor_sync(0xFFFFFFFFu, sum[k], 1);
    sum[k] += __shfl_xor_sync(0xFFFFFFFFu, sum[k], 2);
  }
}
// (-8 times, once) the sum of the lane's group c, in two halves.
template <int NG>
__device__ __forceinline__ void a4_sums(const float (&sum)[NG], uint32_t &high, uint32_t &low) {
  float own = 0.f;
#pragma unroll
  for (int k = 0; k < NG; ++k)
    if ((threadIdx.x & 3) == k) own = sum[k];
  const float h = __half2float(__float2half_rn(own));
  high = a4_pack(-8.f * h, h);
  low = a4_pack(-8.f * (own - h), own - h);
}
// A score's unit in units of log2: neither 0 nor infinite, for 0 times -inf is no number.  (Scores whose unit is held to
// 1e38 differ by 2^50 and more where they differ: their weights stay 0 and 1.)
__device__ __forceinline__ float a4_unit(float unit) { return fminf(fmaxf(unit, 1e-38f), 1e38f); }
// What weights that refer to score m are to be multiplied by when they come to
// refer to score `top`: where scores are far (past 2^20 units of log2) weights
// refer to m itself, else to the whole number nearest to it, `old` and `whole`.
__device__ __forceinline__ float a4_moved(float m, float old, bool far, float top, float whole, bool next_far, float unit) {
  return at_exp2(far ? (next_far ? (m - top) * unit : fmaf(m, unit, -whole)) : (next_far ? fmaf(-top, unit, old) : old - whole));
}
// A record's reference in units of log2, of a score m in units of 1 / `by`.
__device__ __forceinline__ float a4_record_reference(float m, float base, bool far, float by, float unit) {
  return m == kA4Least ? __uint_as_float(0xFF800000u) : far ? fminf(fmaxf(m * by * unit, -3e38f), 3e38f) : 7.f - base;
}
// The largest value scale of a tile, of either sign, from its values' parameters as
// products take them (rows of even parameters); an infinite one spoils its own group
// alone.
template <int kHalves>  // of the tile
__device__ __forceinline__ float a4_largest(const uint32_t (&vp)[kHalves][2], bool scale_lane) {
  float largest = 0.f;
#pragma unroll
  for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = __half22float2(__habs2(*reinterpret_cast<const __half2 *>(&vp[hf][i])));
      if (scale_lane) largest = fmaxf(largest, fmaxf(f.x <= 65504.f ? f.x : 0.f, f.y <= 65504.f ? f.y : 0.f));
    }
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, s));
  return largest;
}
// What weights are multiplied by beside the value scales, and the largest scale
// that fits it; returns the factor that it changed by.
struct A4Scale {
  float unit = 1.f, most = 0.f;
  __device__ __forceinline__ float fit(float largest) {
    if (!(largest > most)) return 1.f;
    const int e = (int)(__float_as_uint(largest) >> 23) - 126;  // 2^-(floor(log2 largest) + 1)
    const float next = __uint_as_float((uint32_t)(127 - e) << 23), factor = next / unit;
    unit = next;
    most = __uint_as_float((uint32_t)(127 + e) << 23);
    return factor;
  }
};
// Whether a pair of parameters is no number, or infinite.
__device__ __forceinline__ bool a4_none(uint32_t u) {
  return (u & 0x7C00u) == 0x7C00u || (u & 0x7C000000u) == 0x7C000000u;
}

// Split kernels: bound by what a code costs to become an operand and a weight.
// 64 ragged rows (up to 8192 keys of 4 heads of 128, four queries each, fp16) take
// 67 us, 202 MB at 3.0 TB/s; 2 rows of 131072 keys of 8 such heads (bf16) 86 us,
// 325 MB at 3.8 TB/s; 128 rows of five tokens (4096 keys of 2 heads of 64, seven
// queries each) 66 us; 8 rows of up to 700 keys 11.3 us, latency.  16 keys cost a
// warp some 400 operations (four groups in bf16, 26 of them products), 440 in fp16,
// 500 in the wide kernel; in the narrow one issue slots are half busy, three warps a
// scheduler (registers), the tensor pipe a quarter.
//
// All rows' items form one sequence; every warp takes an equal,
// contiguous share of it, whatever the rows' lengths, and works alone: a ring of
// tiles of 32 keys filled with asynchronous copies of the codes and
// parameters as they lie in the cache.  Where its share meets an item's tiles, it
// leaves one record at index item + warp, which is unique because both only grow
// along the sequence.
//
// Codes enter the products as they are: a code c in the lowest four bits of a
// 16-bit word is the fp16 number c 2^-24, and in the next four c 2^-20, both
// exact (subnormal), so that one AND makes two operands.  What a word's other
// nibbles need is one shift.  With scale s_g and middle z_g of group g:
//
//   q . k = sum_g s_g (q_g . c_g) + sum_g (z_g - 8 s_g) sum q_g
//   o     = sum_j (p_j s_jg) (c_j - 8) + sum_j p_j z_jg
//
// K: words are shifted so that codes are c 2^-22 and c 2^-18: a product's terms are
// aligned as if a subnormal factor had the smallest normal exponent, and cut off,
// so that two bits more leave a fifth of the scores' error (lse of one key 1.1e-6
// off as c 2^-24, 2e-7 so).  s_g weighs a group's sums in fp32; the rest is one more product, of the
// parameters as they lie with the queries' sums in two fp16 halves.  V: p s_g is
// rounded to fp16 once, and its rounding meets c - 8 and not c: the narrow kernel
// adds -8 times the same rounded weights, one more product with constants, the
// wide one subtracts 8 from the codes, which are many products' operands there.
// Either keeps the sums small: what a product's sum loses at its end would else
// grow with the keys.  The middles are one product with p.
//
// Queries' entries are off by 2^-26 of a row's largest at most.  Weights are at
// most 2^8 of what they refer to (it moves only when a score passes it by 2^8),
// scaled up by 2^7 (and up to 2^0.5: references are whole numbers), and by the
// power of two below 1 over the largest value scale met, so that fp16 holds them
// with 2^-21 and less of the largest at full precision; a smaller one is off by up to
// 2^-31 of the largest, so that a group whose scale is 2^-20 of the largest met loses
// bits of its codes' part.  p s_g and p are off by 2^-12 of themselves.  Beside a bf16
// answer's own 2^-9 that adds 1 to 2 % to its error (0.00172 for 0.00169); taking what
// rounding leaves there too would cost 93 us for 87 (2 rows of 131072 keys) and 91 for
// 66 (five tokens).  Beside an fp16 answer's 2^-12 it is as much again: for fp16 (kFine) a query takes two rows
// of a product, one of its weights and one of what rounding left of them (2^-23),
// and their sums are added at the end (64 ragged rows, four queries a key head: 62
// -> 67 us; the answers' error from 1.5 of what rounding them costs to 1.0).
//
// Narrow: up to eight query rows, S^T = K Q^T and O^T += V^T P^T, keys and values
// as A, so that no half of a product is empty; P^T changes fragments with
// movmatrix.  kFine: four, columns 4 to 7 being what rounding left of 0 to 3.
template <int NG, bool kFine, bool kWhole>
__global__ void __launch_bounds__(kA4Warps * 32, a4_narrow_ctas(NG))
    ms_attn4_narrow_kernel(const __grid_constant__ A4Args a) {
  using R = A4Ring<NG>;
  constexpr int kPitch = R::kPitch, kStage = R::kStage, kPairs = R::kPairs;
  const float kNone = __uint_as_float(0xFF800000u);
  extern __shared__ __align__(128) unsigned char a4_ring[];
  // Of the warps' queries, what a score of 1 is in units of log2: a score's own unit here is 2^22 times that, past fp32
  // where scale times q passes 1e31, and a record's reference is not.
  __shared__ float plain_units[kA4Warps][8];
  grid_wait();  // the call's first kernel
  grid_release();
  A4Walk now;
  if (!a4_begin(a, now)) return;
  const ms_kv4_attention_args &x = a.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  unsigned char *mine = a4_ring + warp * kA4Stages * kStage;
  A4Copies<NG, kWhole> copies(a, now, mine);
  const int hcs = x.cache.kv_heads * a.chunks;
  const bool scale_lane = (r & 1) == 0 && r < 2 * NG;  // its rows of the values' parameters are scales
  uint32_t qf[NG][4], qs[2];  // query r's operands
  const uint32_t rest = kFine && c >= 2 ? 0xFFFFFFFFu : 0u;
  float o[2 * NG][4];         // entries 32 g + 4 r + 2 i (0, 1) and the next (2, 3), of queries 2c and 2c + 1
  float z[2];                 // the middles' part: row r is parameter r of a key
  // of queries 2c and 2c + 1: what a score of 2^-22 is in units of log2, the score that weights refer to, the one past
  // which they do no longer, 7 less the whole number nearest to it in units of log2, the sum of weights, keys seen
  float unit[2], m[2], lim[2], base[2], l[2];
  int len[2];
  int least = 0;              // keys that every query of the item sees
  int n = 0;                  // queries of the item
  A4Scale v_scale;
  bool far = false;           // m is so large that base's rounding matters
  bool fresh = true, broken = false;
  int stage = 0;
  while (now.tile < now.end) {
    copies.next(stage == 0 ? kA4Stages - 1 : stage - 1);
    if (fresh) {
      const int h = now.hc / a.chunks, first = (now.hc - h * a.chunks) * a.chunk_rows;
      n = min(a.chunk_rows, a.queries - first);
      const int own = r & (a4_narrow(kFine) - 1), q = first + (own < n ? own : 0), token = q / a.group;
      float sum[NG], down;
      uint32_t u[NG][4];
      a4_query_load<NG>(a, own < n, now.b * x.q_row + token * x.q_token + (h * a.group + q - token * a.group) * x.q_head, u);
      a4_query<NG>(a, u, qf, sum, down);
      a4_sums<NG>(sum, qs[0], qs[1]);
      __syncwarp();  // the last item's have been read
      if (c == 0) plain_units[warp][r] = a4_unit(a.scale_log2 * down);
      least = 0x7FFFFFFF;
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // of the queries that this lane's columns of a product are
        const int g = (2 * c + i) & (a4_narrow(kFine) - 1);
        unit[i] = a4_unit(a.scale_log2 * 0x1p22f * __shfl_sync(0xFFFFFFFFu, down, g * 4));
        len[i] = g < n ? load_in(x.lengths + now.b * x.length_row + (first + g) / a.group) : 0x7FFFFFFF;
        least = min(least, len[i]);
        len[i] = min(len[i], now.keys);
        m[i] = lim[i] = kA4Least;
        base[i] = l[i] = z[i] = 0.f;
      }
      least = __reduce_min_sync(0xFFFFFFFFu, least);
#pragma unroll
      for (int i = 0; i < 2 * NG; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      v_scale = A4Scale();
      far = true;  // nothing is referred to yet
      fresh = broken = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kA4Stages - 1) : "memory");
    __syncwarp();
    broken |= copies.broken();
    unsigned char *here = mine + stage * kStage;
    const uint32_t kst = smem_addr(here);
    // rows of the matrices that ldmatrix takes: keys 0-7 and 8-15 of a half and group, then of the next group
    const uint32_t mat = (uint32_t)((lane & 15) * kPitch + (lane >> 4) * 16);
    float sc[kA4Halves][4];  // in units of 2^22: the scales stay as they are
#pragma unroll
    for (int hf = 0; hf < kA4Halves; ++hf) {
      const unsigned char *params = here + R::kKp + hf * kA4Half * 16;
      uint32_t p[2];
      ldmatrix2(p, kst + R::kKp + (hf * kA4Half + (lane & 15)) * 16);
      if (NG == 1 || NG == 3)
        if (c >= NG) p[0] = p[1] = 0;
      uint32_t pr[2][4];  // (scale, middle) of the groups of keys r and r + 8
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (kPairs == 4) *reinterpret_cast<uint4 *>(pr[i]) = *reinterpret_cast<const uint4 *>(params + (r + 8 * i) * 16);
        else *reinterpret_cast<uint2 *>(pr[i]) = *reinterpret_cast<const uint2 *>(params + (r + 8 * i) * 16);
      }
      a4_mma(sc[hf], p[0], p[1], p[0], p[1], qs[0], qs[1], 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[hf][i] *= 0x1p-22f;
      // the groups' first products, then their second ones, which wait for them
      uint32_t f[(NG + 1) / 2][4];
      float d[NG][4];
#pragma unroll
      for (int g = 0; g < NG; g += 2) ldmatrix4(f[g / 2], kst + hf * kA4Half * kPitch + mat + g * 16);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t w0 = f[g / 2][2 * (g & 1)] << 2, w1 = f[g / 2][2 * (g & 1) + 1] << 2;
        a4_mma(d[g], w0 & 0x003C003Cu, w1 & 0x003C003Cu, w0 & 0x03C003C0u, w1 & 0x03C003C0u, qf[g][0], qf[g][1], 0.f, 0.f);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t w0 = f[g / 2][2 * (g & 1)] >> 6, w1 = f[g / 2][2 * (g & 1) + 1] >> 6;
        a4_mma(d[g], w0 & 0x003C003Cu, w1 & 0x003C003Cu, w0 & 0x03C003C0u, w1 & 0x03C003C0u, qf[g][2], qf[g][3]);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float s0 = a4_low(pr[0][g]), s1 = a4_low(pr[1][g]);
        sc[hf][0] = fmaf(s0, d[g][0], sc[hf][0]);
        sc[hf][1] = fmaf(s0, d[g][1], sc[hf][1]);
        sc[hf][2] = fmaf(s1, d[g][2], sc[hf][2]);
        sc[hf][3] = fmaf(s1, d[g][3], sc[hf][3]);
      }
    }
    const int j0 = now.tile * kA4Tile;
    const bool partial = j0 + kA4Tile > least;  // some query does not see some key
    // A masked key's weight of 0 must not meet a middle that is no number: it is taken out of the products, and put
    // back for the queries that see the key.
    uint32_t lost = 0;  // bits g, 8 + g: queries 2c and 2c + 1 see a key whose group g is no number
    if (partial) {
#pragma unroll
      for (int hf = 0; hf < kA4Halves; ++hf) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (j0 + hf * kA4Half + r >= len[i]) sc[hf][i] = kNone;
          if (j0 + hf * kA4Half + r + 8 >= len[i]) sc[hf][2 + i] = kNone;
        }
        uint32_t *params = reinterpret_cast<uint32_t *>(here + R::kVp + (hf * kA4Half + r) * 16);
        uint32_t none[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if (a4_none(params[i * 32 + g])) none[i] |= 1u << g;
        if (!__any_sync(0xFFFFFFFFu, none[0] | none[1])) continue;
        if (sc[hf][0] != kNone) lost |= none[0];
        if (sc[hf][1] != kNone) lost |= none[0] << 8;
        if (sc[hf][2] != kNone) lost |= none[1];
        if (sc[hf][3] != kNone) lost |= none[1] << 8;
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) lost |= __shfl_xor_sync(0xFFFFFFFFu, lost, s);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if (none[i] & (1u << g)) params[i * 32 + g] = 0;
        __syncwarp();
      }
    }
    // the values' parameters as A: row r is parameter r (an even one is a scale), of keys 2c and 2c + 1, and 8 on
    uint32_t vp[kA4Halves][2];
    __half2 most = __float2half2_rn(0.f);
#pragma unroll
    for (int hf = 0; hf < kA4Halves; ++hf) {
      ldmatrix2t(vp[hf], kst + R::kVp + (hf * kA4Half + (lane & 15)) * 16);
      most = __hmax2(most, __hmax2(__habs2(*reinterpret_cast<__half2 *>(&vp[hf][0])), __habs2(*reinterpret_cast<__half2 *>(&vp[hf][1]))));
    }
    bool moves = scale_lane && (__low2float(most) > v_scale.most || __high2float(most) > v_scale.most);
    float high[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      high[i] = fmaxf(sc[0][i], sc[0][2 + i]);
      high[i] = fmaxf(high[i], fmaxf(sc[1][i], sc[1][2 + i]));
      moves = moves || high[i] > lim[i];
    }
    if (__any_sync(0xFFFFFFFFu, moves)) {
      const float factor = v_scale.fit(a4_largest(vp, scale_lane));
      float top[2], whole[2];
      bool next_far = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = high[i];
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], s));
        top[i] = fmaxf(top[i], m[i]);
        whole[i] = rintf(top[i] * unit[i]);
        next_far = next_far || !(fabsf(whole[i]) < kAtFar);
      }
      next_far = __any_sync(0xFFFFFFFFu, next_far);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = a4_moved(m[i], 7.f - base[i], far, top[i], whole[i], next_far, unit[i]);
        m[i] = top[i];
        lim[i] = top[i] == kA4Least ? kA4Least : top[i] + 8.f / unit[i];
        base[i] = 7.f - whole[i];
        l[i] *= f;
        z[i] *= f;
        const float fo = f * factor;
#pragma unroll
        for (int k = 0; k < 2 * NG; ++k) o[k][i] *= fo, o[k][2 + i] *= fo;
      }
      far = next_far;
    }
#pragma unroll
    for (int hf = 0; hf < kA4Halves; ++hf) {
      if (far) {  // the difference from m, which is exact near it; the base's rounding would be whole units
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[hf][i] = at_exp2(fmaf(sc[hf][i] - m[i & 1], unit[i & 1], 7.f));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[hf][i] = at_exp2(fmaf(sc[hf][i], unit[i & 1], base[i & 1]));
      }
    }
#pragma unroll
    for (int hf = 0; hf < kA4Halves; ++hf) {
      const unsigned char *params = here + R::kVp + hf * kA4Half * 16;
      uint32_t vr[2][4];  // (scale, middle) of the groups of keys r and r + 8
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (kPairs == 4) *reinterpret_cast<uint4 *>(vr[i]) = *reinterpret_cast<const uint4 *>(params + (r + 8 * i) * 16);
        else *reinterpret_cast<uint2 *>(vr[i]) = *reinterpret_cast<const uint2 *>(params + (r + 8 * i) * 16);
      }
      float w[4] = {sc[hf][0], sc[hf][1], sc[hf][2], sc[hf][3]};
      l[0] += w[0] + w[2];
      l[1] += w[1] + w[3];
      a4_mma_top(z, vp[hf][0], vp[hf][1], a4_turn(a4_weights<kFine>(w[0], w[1], rest)),
                 a4_turn(a4_weights<kFine>(w[2], w[3], rest)));
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] *= v_scale.unit;
      uint32_t pw[NG][2];  // weights times the groups' scales as B: keys 2c and 2c + 1 of query r, then keys + 8
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float s0 = a4_low(vr[0][g]), s1 = a4_low(vr[1][g]);
        pw[g][0] = a4_turn(a4_weights<kFine>(w[0] * s0, w[1] * s0, rest));
        pw[g][1] = a4_turn(a4_weights<kFine>(w[2] * s1, w[3] * s1, rest));
      }
      // -8 2^-24 and -8 2^-20, of the rows whose codes are in the lower and the upper nibble; then the codes
#pragma unroll
      for (int k = 0; k < 2 * NG; ++k)
        a4_mma(o[k], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pw[k / 2][0], pw[k / 2][1]);
      uint32_t f[4];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if ((g & 1) == 0) ldmatrix4t(f, kst + R::kV + hf * kA4Half * kPitch + mat + g * 16);
        const uint32_t w0 = f[2 * (g & 1)], w1 = f[2 * (g & 1) + 1], w2 = w0 >> 8, w3 = w1 >> 8;
        a4_mma(o[2 * g], w0 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x000F000Fu, w1 & 0x00F000F0u, pw[g][0], pw[g][1]);
        a4_mma(o[2 * g + 1], w2 & 0x000F000Fu, w2 & 0x00F000F0u, w3 & 0x000F000Fu, w3 & 0x00F000F0u, pw[g][0], pw[g][1]);
      }
    }
    if (lost && (r & 1)) {
      if ((lost >> (r >> 1)) & 1) z[0] = __uint_as_float(0x7FFFFFFFu);
      if ((lost >> (8 + (r >> 1))) & 1) z[1] = __uint_as_float(0x7FFFFFFFu);
    }
    __syncwarp();  // the stage is read: the next round's copies may overwrite it
    if (++stage == kA4Stages) stage = 0;
    if (++now.tile < now.end) continue;
    const int64_t piece = (int64_t)now.b * hcs + now.hc + (int64_t)blockIdx.x * kA4Warps + warp;
    if (kFine) {  // lanes c and c + 2 have the same queries
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        z[i] += __shfl_xor_sync(0xFFFFFFFFu, z[i], 2);
#pragma unroll
        for (int k = 0; k < 2 * NG; ++k) {
          o[k][i] += __shfl_xor_sync(0xFFFFFFFFu, o[k][i], 2);
          o[k][2 + i] += __shfl_xor_sync(0xFFFFFFFFu, o[k][2 + i], 2);
        }
      }
    }
    const float low = 0x1p17f / v_scale.unit, up = 0x1p13f / v_scale.unit;  // 2^24 and 2^20 without the weights' 2^7
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], s);
      const int g = c * 2 + i;
      const int64_t rec = piece * a.chunk_rows + g;
      if (g < n && r == 0)
        a.own_ml[rec] = make_float2(a4_record_reference(m[i], base[i], far, 0x1p22f, plain_units[warp][g]),
                                    broken ? kAtBadPage : l[i] * 0x1p-7f);
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float middle = __shfl_sync(0xFFFFFFFFu, z[i], (2 * k + 1) * 4 + c) * 0x1p-7f;
        const int d = k * 32 + r * 4;
        if (g < n && d < x.cache.head_dim)
          *reinterpret_cast<float4 *>(a.own_o + rec * x.cache.head_dim + d) =
              make_float4(fmaf(o[2 * k][i], low, middle), fmaf(o[2 * k][2 + i], up, middle),
                          fmaf(o[2 * k + 1][i], low, middle), fmaf(o[2 * k + 1][2 + i], up, middle));
      }
    }
    fresh = true;
    a4_item_next(a, now);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Wide: sixteen query rows a product, S = Q K^T and O += P V, the queries as A
// (from shared memory: registers are for the output's).  A lane has rows r and r
// + 8 of every sixteen and the keys and entries 2c and 2c + 1 of every eight, so
// that weights are operands where they are and a row's statistics are one
// lane's.  A code is made an operand once for all sixteens: with operands of
// eight queries each (movmatrix for every weight) 128 rows of five tokens took 82
// us.  All queries of an item are loaded before the first is used (one after
// another: 73 us, now 66).  kFine: eight queries a sixteen, row r + 8 being what
// rounding left of row r.
template <int NG, int NP, bool kFine, bool kWhole>
__global__ void __launch_bounds__(kA4Warps * 32, a4_wide_ctas(NG, NP))
    ms_attn4_wide_kernel(const __grid_constant__ A4Args a) {
  using R = A4Ring<NG>;
  constexpr int kOwn = kFine ? 1 : 2;  // a lane's queries of a sixteen
  constexpr int kPitch = R::kPitch, kStage = R::kStage;
  const float kNone = __uint_as_float(0xFF800000u);
  extern __shared__ __align__(128) unsigned char a4_ring[];
  grid_wait();  // the call's first kernel
  grid_release();
  A4Walk now;
  if (!a4_begin(a, now)) return;
  const ms_kv4_attention_args &x = a.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  unsigned char *mine = a4_ring + warp * kA4Stages * kStage;
  uint4 *queries = reinterpret_cast<uint4 *>(a4_ring + kA4Warps * kA4Stages * kStage + warp * kA4Queries<NG, NP>) + lane;
  uint4 *qs = queries + NP * NG * 64;  // the sums: row r, row r + 8, then their lower halves
  float2 *m = reinterpret_cast<float2 *>(qs - lane + NP * 32) + lane;  // of rows r and r + 8, as in the narrow kernel
  A4Copies<NG, kWhole> copies(a, now, mine);
  const int hcs = x.cache.kv_heads * a.chunks;
  const bool scale_lane = (r & 1) == 0 && r < 2 * NG;
  float o[NP][NG][4][4];      // entries 32 g + 8 c + i (0) and + 4 + i (1) of row r, then of row r + 8
  float z[NP][4];             // the scales' and the middles' parts of group c, of row r, then of row r + 8
  float unit[NP][kOwn], lim[NP][kOwn], base[NP][kOwn], l[NP][kOwn];  // as m
  int least = 0, n = 0;
  A4Scale v_scale;
  bool far = false, fresh = true, broken = false;
  int stage = 0;
  while (now.tile < now.end) {
    copies.next(stage == 0 ? kA4Stages - 1 : stage - 1);
    if (fresh) {
      const int h = now.hc / a.chunks, first = (now.hc - h * a.chunks) * a.chunk_rows;
      n = min(a.chunk_rows, a.queries - first);
      least = 0x7FFFFFFF;
      uint32_t u[NP][kOwn][NG][4];  // all loads before the first is waited for
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int g = (t * kOwn + i) * 8 + r, q = first + (g < n ? g : 0), token = q / a.group;
          a4_query_load<NG>(a, g < n, now.b * x.q_row + token * x.q_token + (h * a.group + q - token * a.group) * x.q_head, u[t][i]);
          if (g < n) least = min(least, load_in(x.lengths + now.b * x.length_row + token));
        }
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        uint32_t f[2][NG][4] = {}, parts[4] = {};
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          float sum[NG], down;
          a4_query<NG>(a, u[t][i], f[i], sum, down);
          a4_sums<NG>(sum, parts[i], parts[2 + i]);
          unit[t][i] = a4_unit(a.scale_log2 * down);
          lim[t][i] = kA4Least;
          base[t][i] = l[t][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) z[t][i] = 0.f;
        qs[t * 32] = make_uint4(parts[0], parts[1], parts[2], parts[3]);
        m[t * 32] = make_float2(kA4Least, kA4Least);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            queries[((t * NG + g) * 2 + k) * 32] = make_uint4(f[0][g][2 * k], f[1][g][2 * k], f[0][g][2 * k + 1], f[1][g][2 * k + 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][g][i][0] = o[t][g][i][1] = o[t][g][i][2] = o[t][g][i][3] = 0.f;
        }
      }
      least = __reduce_min_sync(0xFFFFFFFFu, least);
      v_scale = A4Scale();
      far = true;
      fresh = broken = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kA4Stages - 1) : "memory");
    __syncwarp();
    broken |= copies.broken();
    unsigned char *here = mine + stage * kStage;
    const uint32_t kst = smem_addr(here);
    const uint32_t mat = (uint32_t)((lane & 15) * kPitch + (lane >> 4) * 16);
#pragma unroll 1
    for (int hf = 0; hf < kA4Halves; ++hf) {
      const int j0 = now.tile * kA4Tile + hf * kA4Half;
      if (j0 >= now.keys) break;
      unsigned char *kps = here + R::kKp + hf * kA4Half * 16, *vps = here + R::kVp + hf * kA4Half * 16;
      float sc[NP][2][2 * kOwn];  // keys 8 j + 2c and the next, of row r, then of row r + 8
      {
        uint32_t p[2];
        ldmatrix2(p, smem_addr(kps) + (lane & 15) * 16);
        if (NG == 1 || NG == 3)
          if (c >= NG) p[0] = p[1] = 0;
#pragma unroll
        for (int t = 0; t < NP; ++t) {
          const uint4 q = qs[t * 32];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float d[4];
            a4_mma(d, q.x, q.y, q.z, q.w, p[j], p[j], 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 2 * kOwn; ++i) sc[t][j][i] = d[i];
          }
        }
        float2 s[2][NG];  // scales of keys 8 j + 2c and the next
#pragma unroll
        for (int j = 0; j < 2; ++j) a4_pair_scales<NG>(kps + (8 * j + 2 * c) * 16, 0x1p22f, s[j]);
        uint32_t f[4];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if ((g & 1) == 0) ldmatrix4(f, kst + hf * kA4Half * kPitch + mat + g * 16);
          const uint32_t w[2] = {f[2 * (g & 1)], f[2 * (g & 1) + 1]};
#pragma unroll
          for (int t = 0; t < NP; ++t) {
            const uint4 q0 = queries[((t * NG + g) * 2) * 32], q1 = queries[((t * NG + g) * 2 + 1) * 32];
            float d[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
              a4_mma(d[j], q0.x, q0.y, q0.z, q0.w, (w[j] << 2) & 0x003C003Cu, (w[j] << 2) & 0x03C003C0u, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 2; ++j)
              a4_mma(d[j], q1.x, q1.y, q1.z, q1.w, (w[j] >> 6) & 0x003C003Cu, (w[j] >> 6) & 0x03C003C0u);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 2 * kOwn; i += 2) {
                const float2 y = at_fma2(s[j][g], make_float2(d[j][i], d[j][i + 1]), make_float2(sc[t][j][i], sc[t][j][i + 1]));
                sc[t][j][i] = y.x, sc[t][j][i + 1] = y.y;
              }
          }
        }
      }
      uint32_t lost[NP] = {};  // bits g, 8 + g: rows r and r + 8 see a key whose group g is no number
      if (j0 + kA4Half > least) {  // some query does not see some key
        uint32_t none[4];        // of keys 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          none[k] = 0;
          const uint32_t *params = reinterpret_cast<const uint32_t *>(vps + (2 * c + (k & 1) + (k & 2) * 4) * 16);
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if (a4_none(params[g])) none[k] |= 1u << g;
        }
        const int h = now.hc / a.chunks, first = (now.hc - h * a.chunks) * a.chunk_rows;
#pragma unroll
        for (int t = 0; t < NP; ++t) {
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            const int g = (t * kOwn + i) * 8 + r;
            const int len = min(now.keys, g < n ? load_in(x.lengths + now.b * x.length_row + (first + g) / a.group) : 0x7FFFFFFF);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float &score = sc[t][k >> 1][2 * i + (k & 1)];
              if (j0 + 2 * c + (k & 1) + (k & 2) * 4 >= len) score = kNone;
              if (score != kNone) lost[t] |= none[k] << (8 * i);
            }
          }
          lost[t] |= __shfl_xor_sync(0xFFFFFFFFu, lost[t], 1);
          lost[t] |= __shfl_xor_sync(0xFFFFFFFFu, lost[t], 2);
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t *params = reinterpret_cast<uint32_t *>(vps + (2 * c + (k & 1) + (k & 2) * 4) * 16);
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if (none[k] & (1u << g)) params[g] = 0;
        }
        __syncwarp();
      }
      // the values' parameters as B: column r is parameter r, of keys 2c and 2c + 1, and 8 on
      uint32_t vp[1][2];
      ldmatrix2t(vp[0], smem_addr(vps) + (lane & 15) * 16);
      const __half2 most = __hmax2(__habs2(*reinterpret_cast<__half2 *>(&vp[0][0])), __habs2(*reinterpret_cast<__half2 *>(&vp[0][1])));
      bool moves = scale_lane && (__low2float(most) > v_scale.most || __high2float(most) > v_scale.most);
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          moves = moves || fmaxf(fmaxf(sc[t][0][2 * i], sc[t][0][2 * i + 1]), fmaxf(sc[t][1][2 * i], sc[t][1][2 * i + 1])) > lim[t][i];
      if (__any_sync(0xFFFFFFFFu, moves)) {
        const float factor = v_scale.fit(a4_largest(vp, scale_lane));
        float top[NP][2], old[NP][2];
        bool next_far = false;
#pragma unroll
        for (int t = 0; t < NP; ++t)
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            float y = fmaxf(fmaxf(sc[t][0][2 * i], sc[t][0][2 * i + 1]), fmaxf(sc[t][1][2 * i], sc[t][1][2 * i + 1]));
            y = fmaxf(y, __shfl_xor_sync(0xFFFFFFFFu, y, 1));
            y = fmaxf(y, __shfl_xor_sync(0xFFFFFFFFu, y, 2));
            old[t][i] = i ? m[t * 32].y : m[t * 32].x;
            top[t][i] = fmaxf(y, old[t][i]);
            next_far = next_far || !(fabsf(rintf(top[t][i] * unit[t][i])) < kAtFar);
          }
        next_far = __any_sync(0xFFFFFFFFu, next_far);
#pragma unroll
        for (int t = 0; t < NP; ++t)
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            const float whole = rintf(top[t][i] * unit[t][i]);
            const float f = a4_moved(old[t][i], 7.f - base[t][i], far, top[t][i], whole, next_far, unit[t][i]);
            lim[t][i] = top[t][i] == kA4Least ? kA4Least : top[t][i] + 8.f / unit[t][i];
            base[t][i] = next_far ? 7.f : 7.f - whole;
            l[t][i] *= f;
            const float fo = f * factor;
#pragma unroll
            for (int e = 2 * i; e < (kFine ? 4 : 2 * i + 2); ++e) {
              z[t][e] *= f;
#pragma unroll
              for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[t][g][k][e] *= fo;
            }
          }
        far = next_far;
#pragma unroll
        for (int t = 0; t < NP; ++t) m[t * 32] = make_float2(top[t][0], top[t][kOwn - 1]);
      }
      if (far) {  // the difference from m, which is exact near it; the base's rounding would be whole units
#pragma unroll
        for (int t = 0; t < NP; ++t) {
          const float2 by = m[t * 32];
#pragma unroll
          for (int k = 0; k < 4 * kOwn; ++k) sc[t][k / (2 * kOwn)][k % (2 * kOwn)] -= (k & 2) && !kFine ? by.y : by.x;
        }
      }
      float2 s[2][NG];  // scales of values 8 j + 2c and the next
#pragma unroll
      for (int j = 0; j < 2; ++j) a4_pair_scales<NG>(vps + (8 * j + 2 * c) * 16, v_scale.unit, s[j]);
      uint32_t v[NG][4][2], f[4];  // codes less 8
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if ((g & 1) == 0) ldmatrix4t(f, kst + R::kV + hf * kA4Half * kPitch + mat + g * 16);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t even = f[2 * (g & 1) + j], odd = even >> 8;
          v[g][0][j] = a4_add(even & 0x000F000Fu, 0x80088008u);
          v[g][1][j] = a4_add(even & 0x00F000F0u, 0x80808080u);
          v[g][2][j] = a4_add(odd & 0x000F000Fu, 0x80088008u);
          v[g][3][j] = a4_add(odd & 0x00F000F0u, 0x80808080u);
        }
      }
#pragma unroll
      for (int t = 0; t < NP; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int k = 2 * i; k < 2 * i + 2; ++k) sc[t][j][k] = at_exp2(fmaf(sc[t][j][k], unit[t][i], base[t][i]));
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          l[t][i] += (sc[t][0][2 * i] + sc[t][0][2 * i + 1]) + (sc[t][1][2 * i] + sc[t][1][2 * i + 1]);
        // weights as A: keys 2c and 2c + 1 of rows r and r + 8, then keys + 8
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          p[2 * j] = a4_pack(sc[t][j][0], sc[t][j][1]);
          p[2 * j + 1] = kFine ? a4_weights<true>(sc[t][j][0], sc[t][j][1], 0xFFFFFFFFu)
                               : a4_pack(sc[t][j][2 * kOwn - 2], sc[t][j][2 * kOwn - 1]);
        }
        a4_mma(z[t], p[0], p[1], p[2], p[3], vp[0][0], vp[0][1]);
        if (lost[t]) {
          if ((lost[t] >> c) & 1) z[t][1] = __uint_as_float(0x7FFFFFFFu);
          if ((lost[t] >> (8 + c)) & 1) z[t][3] = __uint_as_float(0x7FFFFFFFu);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
              const float2 y = a4_mul2(make_float2(sc[t][j][2 * i], sc[t][j][2 * i + 1]), s[j][g]);
              p[2 * j + i] = a4_pack(y.x, y.y);
              if (kFine) p[2 * j + 1] = a4_weights<true>(y.x, y.y, 0xFFFFFFFFu);
            }
#pragma unroll
          for (int i = 0; i < 4; ++i) a4_mma(o[t][g][i], p[0], p[1], p[2], p[3], v[g][i][0], v[g][i][1]);
        }
      }
    }
    __syncwarp();  // the stage is read: the next round's copies may overwrite it
    if (++stage == kA4Stages) stage = 0;
    if (++now.tile < now.end) continue;
    const int64_t piece = (int64_t)now.b * hcs + now.hc + (int64_t)blockIdx.x * kA4Warps + warp;
    const float low = 0x1p17f / v_scale.unit, up = 0x1p13f / v_scale.unit;  // 2^24 and 2^20 without the weights' 2^7
#pragma unroll
    for (int t = 0; t < NP; ++t) {
      if (kFine) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          z[t][e] += z[t][2 + e];
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[t][k][j][e] += o[t][k][j][2 + e];
        }
      }
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 1);
        l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 2);
        const int g = (t * kOwn + i) * 8 + r;
        const int64_t rec = piece * a.chunk_rows + g;
        if (g < n && c == 0)
          a.own_ml[rec] = make_float2(a4_record_reference(i ? m[t * 32].y : m[t * 32].x, base[t][i], far, 1.f, unit[t][i]),
                                      broken ? kAtBadPage : l[t][i] * 0x1p-7f);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const float middle = __shfl_sync(0xFFFFFFFFu, z[t][2 * i + 1], (lane & 28) + k) * 0x1p-7f;
          const int d = k * 32 + c * 8;
          if (g < n && d < x.cache.head_dim) {
            float4 *to = reinterpret_cast<float4 *>(a.own_o + rec * x.cache.head_dim + d);
            float y[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                y[e][j] = fmaf(o[t][k][j][2 * i + e], j & 1 ? up : low, middle);
            to[0] = make_float4(y[0][0], y[0][1], y[0][2], y[0][3]);
            to[1] = make_float4(y[1][0], y[1][1], y[1][2], y[1][3]);
          }
        }
      }
    }
    fresh = true;
    a4_item_next(a, now);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Merge: the records of an output (row, token, query head) weighed by one warp
// of eight in a CTA, or by all sixteen of a CTA where there may be many records.
template <typename T, int DP, int kWarps>
__global__ void __launch_bounds__((kWarps > 1 ? kWarps : kMgNarrow) * 32) ms_attn4_merge_kernel(const __grid_constant__ A4Args a) {
  constexpr int kLanes = DP / 4;      // lanes of a record: four entries each
  constexpr int kSide = 32 / kLanes;  // records side by side
  constexpr int kBatch = 4;           // records in flight of a lane
  constexpr int kStep = kWarps * kSide;
  const float kNone = __uint_as_float(0xFF800000u);
  __shared__ float4 part[kWarps][kLanes];
  __shared__ float2 part_ml[kWarps];
  __shared__ int part_bad[kWarps];
  const ms_kv4_attention_args &x = a.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t at = kWarps > 1 ? blockIdx.x : (int64_t)blockIdx.x * kMgNarrow + warp;
  const int64_t each = (int64_t)x.tokens * x.heads;
  if (at >= x.rows * each) return;  // warps alone
  const int64_t b = at / each;
  const int th = (int)(at - b * each), token = th / x.heads, hq = th - token * x.heads;
  const int h = hq / a.group, q = token * a.group + (hq - h * a.group), chunk = q / a.chunk_rows;
  const int hc = h * a.chunks + chunk, hcs = x.cache.kv_heads * a.chunks;
  grid_wait();
  bool bad_length;
  const int keys = a4_keys(x, b, bad_length);
  const int64_t share = a.header->share, start = a.base[b];
  int64_t own = 0;
  int pieces = 0;
  if (keys > 0) {  // the warps whose shares meet the item's tiles
    const int64_t units = a4_units(keys), u = start + hc * units, w = (u + kA4Item) / share;
    own = (b * hcs + hc + w) * a.chunk_rows + q - chunk * a.chunk_rows;
    pieces = (int)((u + units - 1) / share - w) + 1;
  }
  const int side = lane / kLanes, d = (lane % kLanes) * 4;
  const int dim = x.cache.head_dim;
  float top = kNone, sum = 0.f;
  bool bad = false;
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
        const int64_t rec = own + (int64_t)p * a.chunk_rows;
        ml[i] = a.own_ml[rec];
        if (d < dim) v[i] = *reinterpret_cast<const float4 *>(a.own_o + rec * dim + d);
      }
    }
    float next = top;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) next = fmaxf(next, ml[i].x);
    const float base = next == kNone ? 0.f : next;
    const float f = at_exp2(top - base);
    top = next;
    sum *= f, y.x *= f, y.y *= f, y.z *= f, y.w *= f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float w = at_exp2(ml[i].x - base);
      bad = bad || ml[i].y < 0.f;
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
  bad = __any_sync(0xFFFFFFFFu, bad);
  if (kWarps > 1) {
    if (lane < kLanes) part[warp][lane] = y;
    if (lane == 0) part_ml[warp] = make_float2(top, sum), part_bad[warp] = bad;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll 5
    for (int i = 1; i < kWarps; ++i) join(part_ml[i].x, part_ml[i].y, part[i][lane % kLanes]);
    bad = __any_sync(0xFFFFFFFFu, part_bad[lane % kWarps]);
  }
  const bool empty = bad_length || bad || sum == 0.f;
  if (lane < kLanes && d < dim) {
    T *dst = static_cast<T *>(x.out) + b * x.out_row + token * x.out_token + hq * x.out_head + d;
    const float inv = 1.f / sum;
    const float e[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = AtType<T>::narrow(empty ? 0.f : e[i]);
  }
  if (lane == 0) {
    x.lse[at] = empty ? kNone : (top + log2f(sum)) * 0.6931471805599453f;
    if (bad) atomicOr(x.status + b, MS_ROW_BAD_PAGE);
  }
}

}  // namespace ms
