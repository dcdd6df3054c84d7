// Attention over a paged cache held in 4 bits: arguments, the split kernel and
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
constexpr int kA4Half = 16;                // keys of a product: the M of the scores', the K of the output's
constexpr int kA4Item = 2;                 // cost of an item's queries and record, in tiles
constexpr int kA4Stages = 3;               // tiles of a warp's ring
constexpr float kA4Least = -3e38f;         // refers to nothing yet: every score is far above it
constexpr int64_t kA4MaxRows = 1 << 20;
constexpr int kA4MaxTokens = 1024;         // of a row
// Bytes of a token's codes in the ring: an odd multiple of 16, so that eight
// rows of 16 bytes lie in different banks.
template <int NG>
constexpr int kA4Pitch = NG <= 3 ? 48 : 80;
// Products of a tile: a tile of 32 keys pays for its copies, page and checks
// once, where registers have room for its scores.
template <int NQ>
constexpr int kA4Halves = NQ <= 1 ? 2 : 1;
template <int NG, int NQ>
constexpr int kA4Stage = kA4Halves<NQ> * kA4Half * 2 * (kA4Pitch<NG> + 16);  // K and V codes, K and V parameters
// Queries of more than four fragments a lane stay in shared memory: registers
// are for the output's.
template <int NG, int NQ>
constexpr bool kA4QShared = NG * NQ > 4;
template <int NG, int NQ>
constexpr int kA4Queries = kA4QShared<NG, NQ> ? NG * NQ * 512 : 0;  // bytes of a warp's
template <int NG, int NQ>
constexpr int kA4Shared = kA4Warps * (kA4Stages * kA4Stage<NG, NQ> + kA4Queries<NG, NQ>);
// Split CTAs of an SM, by what their registers allow.
template <int NG, int NQ>
constexpr int kA4Ctas = NG <= 2 ? (NQ <= 1 ? 4 : NQ <= 3 ? 3 : 2) : (NQ <= 1 ? 3 : 2);
// Query rows of an item, at most: eights that registers have room for.
__host__ __device__ constexpr int a4_most(int groups) { return groups <= 2 ? 40 : 16; }

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
  int tile;        // keys of the split kernel's tiles
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
__device__ __forceinline__ int64_t a4_units(int keys, int tile) { return keys > 0 ? (keys + tile - 1) / tile + kA4Item : 0; }

// Walks over a warp's tiles: the split kernel's sequence is rows' items (key
// head and chunk) in order, each of kA4Item units and one unit a tile.  A warp's
// share is far below 2^31 units (the kernel would run for days).
struct A4Walk {
  int b, left;  // left: units of the share past this item
  int hc, tile, end, keys;
};
// The next item's tiles within the share; tile == end where none are left.
template <int kTile>
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
  const int take = min(w.left, (w.keys + kTile - 1) / kTile + kA4Item);
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
__device__ __forceinline__ float a4_low(uint32_t u) { return __low2float(*reinterpret_cast<const __half2 *>(&u)); }

// Split kernel.  All rows' items form one sequence; every warp takes an equal,
// contiguous share of it, whatever the rows' lengths, and works alone: a ring
// of tiles of 32 or 16 keys filled with asynchronous copies of the codes and
// parameters as they lie in the cache, a page lookup a tile ahead of its
// copies, and products of m16n8k16 with the keys (S^T = K Q^T) and the values
// (O^T += V^T P^T) as A.  Where its share meets an item's tiles, it leaves one
// record at index item + warp, which is unique because both only grow along
// the sequence.
//
// Codes enter the products as they are: a code c in the lowest four bits of a
// 16-bit word is the fp16 number c 2^-24, and in the next four c 2^-20, both
// exact (subnormal), so that one AND makes two operands.  What a word's other
// nibbles need is one shift.  With scale s_g and middle z_g of group g:
//
//   q . k = sum_g s_g (q_g . c_g) + sum_g (z_g - 8 s_g) sum q_g
//   o     = sum_j (p_j s_jg) (c_j - 8) + sum_j p_j z_jg
//
// K: s_g weighs a group's sums in fp32; the rest is one more product, of the
// parameters as they lie with the queries' sums in two fp16 halves.  V: p s_g is rounded to fp16 once,
// -8 times the same rounded weights is one more product with constants, so
// that a weight's rounding meets c - 8 and not c; the middles are one product
// with p.
//
// Queries enter as fp16, scaled by a power of two that puts a row's largest in
// [2^5, 2^6): entries are off by 2^-26 of it at most.  Weights are at most 2^8
// of what they refer to (it moves only when a score passes it by 2^8), scaled up
// by 2^7 (and up to 2^0.5: references are whole numbers), and by the power of two
// below 1 over the largest value scale met, so that fp16 holds them with 2^-21
// and less of the largest at full precision.
template <int NG, int NQ, bool kWhole>
__global__ void __launch_bounds__(kA4Warps * 32, kA4Ctas<NG, NQ>)
    ms_attn4_split_kernel(const __grid_constant__ A4Args a) {
  constexpr int kThreads = kA4Warps * 32;
  constexpr int kPitch = kA4Pitch<NG>, kStage = kA4Stage<NG, NQ>, kStages = kA4Stages;
  constexpr int kHalves = kA4Halves<NQ>, kTile = kHalves * kA4Half;
  constexpr int kRow = NG <= 2 ? 32 : NG * 16;  // bytes of a token's codes in the cache
  constexpr int kPieces = kRow / 16;            // 16-byte pieces of them
  constexpr int kPairs = NG <= 2 ? 2 : 4;       // pairs of parameters in the cache
  const float kNone = __uint_as_float(0xFF800000u);
  extern __shared__ __align__(128) unsigned char a4_ring[];
  __shared__ int64_t sums[kThreads + 1];  // units of the rows before each thread's run of rows, of one key head and chunk
  __shared__ int64_t warp_sums[kA4Warps];
  grid_wait();  // the call's first kernel
  grid_release();
  const ms_kv4_attention_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t rows = x.rows;
  const int hcs = x.cache.kv_heads * a.chunks;
  const int64_t run = (rows + kThreads - 1) / kThreads;
  const int64_t r0 = min(rows, tid * run), r1 = min(rows, r0 + run);
  bool bad;
  {
    int64_t n = 0;
    for (int64_t b = r0; b < r1; ++b) n += a4_units(a4_keys(x, b, bad), kTile);
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
  if (blockIdx.x == gridDim.x - 1) {  // for the merge: where each row starts (this CTA's own share is the last, often short)
    int64_t n = sums[tid];
    for (int64_t b = r0; b < r1; ++b) {
      a.base[b] = n * hcs;
      const int keys = a4_keys(x, b, bad);
      x.status[b] = bad ? MS_ROW_BAD_LENGTH : MS_ROW_OK;
      n += a4_units(keys, kTile);
    }
    if (tid == 0) a.header->share = share;
  }
  const int64_t wid = (int64_t)blockIdx.x * kA4Warps + warp;
  const int64_t u0 = wid * share, u1 = min(total, u0 + share);
  if (u0 >= u1) return;
  A4Walk load;
  {
    int lo = 0, hi = kThreads - 1;  // the row that unit u0 lies in: its thread's run, then the row
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid + 1] * hcs > u0) hi = mid;
      else lo = mid + 1;
    }
    load.b = (int)min(rows, lo * run);
    int64_t first = sums[lo] * hcs;
    load.keys = a4_keys(x, load.b, bad);
    while (first + a4_units(load.keys, kTile) * hcs <= u0) {
      first += a4_units(load.keys, kTile) * hcs;
      load.keys = a4_keys(x, ++load.b, bad);
    }
    const int64_t units = a4_units(load.keys, kTile);
    load.hc = (int)((u0 - first) / units);
    const int64_t at = u0 - first - load.hc * units, take = min(u1 - u0, units - at);
    load.left = (int)(u1 - u0 - take);
    load.tile = (int)max((int64_t)0, at - kA4Item);
    load.end = (int)(at + take) - kA4Item;
    if (load.end <= load.tile) a4_item_next<kTile>(a, load);
  }
  A4Walk now = load;
  unsigned char *mine = a4_ring + warp * kStages * kStage;
  const uint32_t ring = smem_addr(mine);
  constexpr int kV = kTile * kPitch, kKp = 2 * kV, kVp = kKp + kTile * 16;  // of a stage
  if (kPairs == 2) {  // the parameters' rows are 16 bytes there too: what lies behind the two pairs stays zero
    for (int s = 0; s < kStages; ++s)
#pragma unroll
      for (int i = 0; i < kHalves; ++i)
        *reinterpret_cast<uint4 *>(mine + s * kStage + kKp + (i * 32 + lane) * 16) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  const int page_size = (int)x.cache.page_size;

  // Copies.  Where a half's keys lie in one page, it is looked up once for all lanes; else lanes 0-15 (and 16-31 again)
  // look up the half's keys.  Page ids are loaded a tile ahead of their use, and a tile's addresses are a page's, a
  // head's and a lane's parts: this is work for every 32 keys.
  int page[kHalves], offset[kHalves];
  const int *table = nullptr;  // of the next tile's row
  int64_t head_at = 0;         // its head's codes in a page
  int live_keys = 0;           // of the next tile; 0 where none is left
  uint32_t met = 0;            // bit i: the tile issued i tiles ago met a bad page
  auto look = [&](bool item) {  // at tile load.tile, the first of an item's or not
    live_keys = 0;
    if (load.tile >= load.end) return;
    if (item) {
      head_at = load.hc / a.chunks * a.code_head;
      table = x.table + load.b * x.table_row;
    }
    live_keys = load.keys - load.tile * kTile;
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      const int j = load.tile * kTile + i * kA4Half + (kWhole ? 0 : lane & 15);
      page[i] = offset[i] = 0;
      if (j < load.keys) {
        const int p = a.page_shift >= 0 ? j >> a.page_shift : j / page_size;
        offset[i] = a.page_shift >= 0 ? j & (page_size - 1) : j - p * page_size;
        page[i] = load_in(table + p);
      }
    }
  };
  auto step = [&]() {
    if (load.tile >= load.end) return;  // none is left
    const bool item = ++load.tile >= load.end;
    if (item) a4_item_next<kTile>(a, load);
    look(item);
  };
  constexpr int kCopies = (kTile * kPieces + 31) / 32;  // of a tile's codes of the keys, and of the values
  const unsigned char *k_lane = x.cache.k_codes + lane * 16, *v_lane = x.cache.v_codes + lane * 16;
  const uint32_t d_lane = ring + lane / kPieces * kPitch + lane % kPieces * 16;  // of copy 0
  auto params_of = [](int64_t code) { return kPairs * 4 * 4 == kRow ? code >> 2 : code / kRow * (kPairs * 4); };
  auto issue = [&](int stage) {
    int64_t code[kHalves];  // the codes' place of a half's first key, or of the lane's
    bool wrong = false;
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      const bool live = i * kA4Half + (kWhole ? 0 : lane & 15) < live_keys;
      wrong = wrong || (live && (unsigned)page[i] >= (unsigned)x.cache.pages);
      code[i] = page[i] * a.code_page + head_at + (uint32_t)offset[i] * (int64_t)kRow;
    }
    met = (met << 1) | (kWhole ? wrong : __any_sync(0xFFFFFFFFu, wrong));
    if (kWhole && live_keys >= kTile && !wrong) {  // all of the tile
      const uint32_t dst = d_lane + stage * kStage;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        if (kPieces == 3) {
          const int at = i * 32 + lane, r = at / kPieces;
          const int64_t off = (kHalves > 1 && r >= kA4Half ? code[kHalves - 1] - kA4Half * kRow : code[0]) + i * 512;
          const uint32_t to = ring + stage * kStage + r * kPitch + (at - r * kPieces) * 16;
          if (kTile * kPieces % 32 == 0 || r < kTile) {
            copy16(to, k_lane + off, true);
            copy16(to + kV, v_lane + off, true);
          }
        } else {
          constexpr int kEach = kCopies / kHalves;  // of a half
          const int64_t off = code[i / kEach] + i % kEach * 512;
          copy16(dst + i * (32 / kPieces) * kPitch, k_lane + off, true);
          copy16(dst + kV + i * (32 / kPieces) * kPitch, v_lane + off, true);
        }
      }
      const int64_t off = params_of(kHalves > 1 && lane >= 16 ? code[kHalves - 1] : code[0]) + (lane & 15) * (kPairs * 4);
      const char *ks = static_cast<const char *>(x.cache.k_params) + off, *vs = static_cast<const char *>(x.cache.v_params) + off;
      const uint32_t to = ring + stage * kStage + kKp + lane * 16;
      if (kHalves == 1) {
        if (kPairs == 4) copy16(to, lane < 16 ? ks : vs, true);
        else copy8(to, lane < 16 ? ks : vs, true);
      } else if (kPairs == 4) {
        copy16(to, ks, true);
        copy16(to + kTile * 16, vs, true);
      } else {
        copy8(to, ks, true);
        copy8(to + kTile * 16, vs, true);
      }
      return;
    }
    // the codes' place of key r of the tile, or -1
    const uint32_t dst = ring + stage * kStage;
    auto code_of = [&](int r) {
      int64_t at = -1;
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        const bool fine = i * kA4Half + (kWhole ? 0 : lane & 15) < live_keys && (unsigned)page[i] < (unsigned)x.cache.pages;
        const int64_t own = fine ? code[i] : -1;
        const int64_t from = kWhole ? (own >= 0 ? own + (r & 15) * kRow : -1) : __shfl_sync(0xFFFFFFFFu, own, r & 15);
        if (r >> 4 == i) at = from;
      }
      return r < live_keys ? at : -1;
    };
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = i * 32 + lane, r = at / kPieces, piece = at - r * kPieces;
      const int64_t from = code_of(r), off = from >= 0 ? from + piece * 16 : 0;
      if (kTile * kPieces % 32 == 0 || r < kTile) {
        copy16(dst + r * kPitch + piece * 16, x.cache.k_codes + off, from >= 0);
        copy16(dst + kV + r * kPitch + piece * 16, x.cache.v_codes + off, from >= 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      const int64_t from = code_of(kHalves == 1 ? lane & 15 : lane), off = from >= 0 ? params_of(from) : 0;
      const bool key = kHalves == 1 ? lane < 16 : i == 0;
      const char *src = static_cast<const char *>(key ? x.cache.k_params : x.cache.v_params) + off;
      if (kPairs == 4) copy16(dst + kKp + (i * 32 + lane) * 16, src, from >= 0);
      else copy8(dst + kKp + (i * 32 + lane) * 16, src, from >= 0);
    }
  };

  look(true);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    issue(s);
    step();
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Queries as B: pairs of entries (8c, 8c + 4), (8c + 1, 8c + 5) 2^-4, ... of a group.
  constexpr bool kQShared = kA4QShared<NG, NQ>;
  uint32_t qf[kQShared ? 1 : NQ][NG][4];
  unsigned char *q_shared = a4_ring + kA4Warps * kStages * kStage + warp * kA4Queries<NG, NQ> + lane * 16;
  uint32_t qs[NQ][2];          // (-8 times, once) the sum of group c, in two halves
  float o[NQ][2 * NG][4];      // entries 32 g + 4 r + 2 i (0, 1) and the next (2, 3), of queries 2c and 2c + 1
  float z[NQ][2];              // the middles' part: row r is parameter r of a key
  // of queries 2c and 2c + 1: what a score of 1 is in units of log2, the score that weights refer to, the one past which
  // they do no longer, the sum of weights, and the keys that they see
  float unit[NQ][2], m[NQ][2], lim[NQ][2], l[NQ][2];
  float base[NQ][2];           // 7 less the whole number nearest to m in units of log2
  int len[NQ][2];
  int least = 0;               // keys that every query of the item sees
  int n = 0;                   // queries of the item
  float v_unit = 1.f;          // weights are multiplied by it and the value's scale
  float v_most = 0.f;          // largest value scale that fits it
  bool far = false;            // m unit is so large that its rounding matters
  bool fresh = true, broken = false;
  int stage = 0;
  const int r = lane >> 2, c = lane & 3;
  const bool scale_lane = (r & 1) == 0 && r < 2 * NG;  // its rows of the parameters are scales
  while (now.tile < now.end) {
    issue(stage == 0 ? kStages - 1 : stage - 1);
    step();
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (fresh) {
      const int h = now.hc / a.chunks, first = (now.hc - h * a.chunks) * a.chunk_rows;
      n = min(a.chunk_rows, a.queries - first);
      least = 0x7FFFFFFF;
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        const int g = t * 8 + r;
        const int token = (first + (g < n ? g : 0)) / a.group, q_head = h * a.group + (first + (g < n ? g : 0)) - token * a.group;
        const int64_t at = now.b * x.q_row + token * x.q_token + q_head * x.q_head + c * 8;
        float most = 0.f;
        float e[NG][8];
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          uint32_t u[4] = {0, 0, 0, 0};
          if (g < n && k * 32 + c * 8 < x.cache.head_dim) {
            const unsigned short *p = static_cast<const unsigned short *>(x.q) + at + k * 32;
            if (a.q_wide) {
              *reinterpret_cast<uint4 *>(u) = load_in(reinterpret_cast<const uint4 *>(p));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) u[i] = (uint32_t)load_in(p + 2 * i) | ((uint32_t)load_in(p + 2 * i + 1) << 16);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 f;
            if (x.dtype == MS_DTYPE_BF16) f = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
            else f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            e[k][2 * i] = f.x, e[k][2 * i + 1] = f.y;
            most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
        // 2^(5 - floor(log2 most)), as long as it and 1 over it are normal numbers
        const int power = most > 0.f ? min(126, 5 + 127 - (int)(__float_as_uint(most) >> 23)) : 0;
        const float up = __uint_as_float((uint32_t)(power + 127) << 23), down = __uint_as_float((uint32_t)(127 - power) << 23);
        float sum[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          sum[k] = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            e[k][i] = __half2float(__float2half_rn(e[k][i] * up));
            sum[k] += e[k][i];
          }
          uint32_t f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float down4 = i & 1 ? 0.0625f : 1.f;
            f[i] = a4_pack(e[k][i] * down4, e[k][i + 4] * down4);
          }
          sum[k] += __shfl_xor_sync(0xFFFFFFFFu, sum[k], 1);
          sum[k] += __shfl_xor_sync(0xFFFFFFFFu, sum[k], 2);
          if constexpr (kQShared) {
            *reinterpret_cast<uint4 *>(q_shared + (t * NG + k) * 512) = make_uint4(f[0], f[1], f[2], f[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[t][k][i] = f[i];
          }
        }
        float own = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k)
          if (c == k) own = sum[k];
        const float high = __half2float(__float2half_rn(own));
        qs[t][0] = a4_pack(-8.f * high, high);
        qs[t][1] = a4_pack(-8.f * (own - high), own - high);
        // of the queries that this lane's columns of a product are
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // neither 0 nor infinite: 0 times -inf is no number
          unit[t][i] = a.scale_log2 * (NQ == 1 ? 0x1p24f : 1.f) * __shfl_sync(0xFFFFFFFFu, down, 8 * c + 4 * i);
          unit[t][i] = fminf(fmaxf(unit[t][i], 1e-38f), 1e38f);
          const int g2 = t * 8 + 2 * c + i;
          len[t][i] = g2 < n ? load_in(x.lengths + now.b * x.length_row + (first + g2) / a.group) : 0x7FFFFFFF;
          least = min(least, len[t][i]);
          len[t][i] = min(len[t][i], now.keys);
          m[t][i] = kA4Least;
          lim[t][i] = kA4Least;
          base[t][i] = 0.f;
          l[t][i] = z[t][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
      }
      least = __reduce_min_sync(0xFFFFFFFFu, least);
      v_unit = 1.f, v_most = 0.f;
      far = true;  // nothing is referred to yet
      fresh = broken = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    broken |= (met >> (kStages - 1)) & 1;
    const uint32_t kst = ring + stage * kStage;
    unsigned char *here = mine + stage * kStage;
    // rows of the matrices that ldmatrix takes: keys 0-7 and 8-15 of a half and group, then of the next group
    const uint32_t mat = (uint32_t)((lane & 15) * kPitch + (lane >> 4) * 16);
    float sc[kHalves][NQ][4];
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      const uint32_t kcodes = kst + hf * kA4Half * kPitch + mat;
      const unsigned char *params = here + kKp + hf * kA4Half * 16;
      uint32_t p[2];
      ldmatrix2(p, kst + kKp + (hf * kA4Half + (lane & 15)) * 16);
      if (NG == 1 || NG == 3)
        if (c >= NG) p[0] = p[1] = 0;
      uint32_t pr[2][4];  // (scale, middle) of the groups of keys r and r + 8
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (kPairs == 4) *reinterpret_cast<uint4 *>(pr[i]) = *reinterpret_cast<const uint4 *>(params + (r + 8 * i) * 16);
        else *reinterpret_cast<uint2 *>(pr[i]) = *reinterpret_cast<const uint2 *>(params + (r + 8 * i) * 16);
      }
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        a4_mma(sc[hf][t], p[0], p[1], p[0], p[1], qs[t][0], qs[t][1], 0.f, 0.f);
        if (NQ == 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[hf][t][i] *= 0x1p-24f;  // or the scales by 2^24: fewer of these
        }
      }
      // the groups' first products, then their second ones, which wait for them
      uint32_t f[(NG + 1) / 2][4];
#pragma unroll
      for (int g = 0; g < NG; g += 2) ldmatrix4(f[g / 2], kcodes + g * 16);
      constexpr int kAt = kQShared ? 1 : NG;  // groups at a time: registers
#pragma unroll
      for (int g0 = 0; g0 < NG; g0 += kAt) {
        float d[kAt][NQ][4];
        uint4 b[kAt][NQ];
#pragma unroll
        for (int k = 0; k < kAt; ++k) {
          const int g = g0 + k;
          const uint32_t w0 = f[g / 2][2 * (g & 1)], w1 = f[g / 2][2 * (g & 1) + 1];
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            if constexpr (kQShared) b[k][t] = *reinterpret_cast<const uint4 *>(q_shared + (t * NG + g) * 512);
            else b[k][t] = make_uint4(qf[t][g][0], qf[t][g][1], qf[t][g][2], qf[t][g][3]);
            a4_mma(d[k][t], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, b[k][t].x, b[k][t].y, 0.f, 0.f);
          }
        }
#pragma unroll
        for (int k = 0; k < kAt; ++k) {
          const int g = g0 + k;
          const uint32_t w2 = f[g / 2][2 * (g & 1)] >> 8, w3 = f[g / 2][2 * (g & 1) + 1] >> 8;
#pragma unroll
          for (int t = 0; t < NQ; ++t)
            a4_mma(d[k][t], w2 & 0x000F000Fu, w3 & 0x000F000Fu, w2 & 0x00F000F0u, w3 & 0x00F000F0u, b[k][t].z, b[k][t].w);
        }
#pragma unroll
        for (int k = 0; k < kAt; ++k) {
          const int g = g0 + k;
          const float s0 = a4_low(pr[0][g]) * (NQ == 1 ? 1.f : 0x1p24f), s1 = a4_low(pr[1][g]) * (NQ == 1 ? 1.f : 0x1p24f);
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            sc[hf][t][0] = fmaf(s0, d[k][t][0], sc[hf][t][0]);
            sc[hf][t][1] = fmaf(s0, d[k][t][1], sc[hf][t][1]);
            sc[hf][t][2] = fmaf(s1, d[k][t][2], sc[hf][t][2]);
            sc[hf][t][3] = fmaf(s1, d[k][t][3], sc[hf][t][3]);
          }
        }
      }
    }
    const int j0 = now.tile * kTile;
    const bool partial = j0 + kTile > least;  // some query does not see some key
    if (partial) {
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (j0 + hf * kA4Half + r >= len[t][i]) sc[hf][t][i] = kNone;
            if (j0 + hf * kA4Half + r + 8 >= len[t][i]) sc[hf][t][2 + i] = kNone;
          }
    }
    // A masked key's weight of 0 must not meet a middle that is no number: it is taken out of the products, and put
    // back for the queries that see the key.
    uint32_t lost[NQ] = {};  // bits g, 8 + g: queries 2c and 2c + 1 see a key whose group g is no number
    if (partial) {
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        uint32_t none[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(here + kVp + (hf * kA4Half + r + 8 * i) * 16 + g * 4);
            if ((u & 0x7C00u) == 0x7C00u || (u & 0x7C000000u) == 0x7C000000u) none[i] |= 1u << g;
          }
        if (!__any_sync(0xFFFFFFFFu, none[0] | none[1])) continue;
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          if (sc[hf][t][0] != kNone) lost[t] |= none[0];
          if (sc[hf][t][1] != kNone) lost[t] |= none[0] << 8;
          if (sc[hf][t][2] != kNone) lost[t] |= none[1];
          if (sc[hf][t][3] != kNone) lost[t] |= none[1] << 8;
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) lost[t] |= __shfl_xor_sync(0xFFFFFFFFu, lost[t], s);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if (none[i] & (1u << g)) *reinterpret_cast<uint32_t *>(here + kVp + (hf * kA4Half + r + 8 * i) * 16 + g * 4) = 0;
        __syncwarp();
      }
    }
    // the values' parameters as A: row r is parameter r (an even one is a scale), of keys 2c and 2c + 1, and 8 on
    uint32_t vp[kHalves][2];
    __half2 most = __float2half2_rn(0.f);
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      ldmatrix2t(vp[hf], kst + kVp + (hf * kA4Half + (lane & 15)) * 16);
      most = __hmax2(most, __hmax2(*reinterpret_cast<__half2 *>(&vp[hf][0]), *reinterpret_cast<__half2 *>(&vp[hf][1])));
    }
    bool moves = scale_lane && (__low2float(most) > v_most || __high2float(most) > v_most);
#pragma unroll
    for (int t = 0; t < NQ; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float high = fmaxf(sc[0][t][i], sc[0][t][2 + i]);
        if (kHalves > 1) high = fmaxf(high, fmaxf(sc[kHalves - 1][t][i], sc[kHalves - 1][t][2 + i]));
        moves = moves || high > lim[t][i];
      }
    if (__any_sync(0xFFFFFFFFu, moves)) {
      float largest = 0.f;  // value scale; an infinite one spoils its own group alone
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&vp[hf][i]));
          if (scale_lane) largest = fmaxf(largest, fmaxf(f.x <= 65504.f ? f.x : 0.f, f.y <= 65504.f ? f.y : 0.f));
        }
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, s));
      float v_factor = 1.f;
      if (largest > v_most) {  // 2^-(floor(log2 largest) + 1)
        const int e = (int)(__float_as_uint(largest) >> 23) - 126;
        const float next = __uint_as_float((uint32_t)(127 - e) << 23);
        v_factor = next / v_unit;
        v_unit = next;
        v_most = __uint_as_float((uint32_t)(127 + e) << 23);
      }
      float top[NQ][2], whole[NQ][2];
      bool next_far = false;
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[t][i] = fmaxf(sc[0][t][i], sc[0][t][2 + i]);
          if (kHalves > 1) top[t][i] = fmaxf(top[t][i], fmaxf(sc[kHalves - 1][t][i], sc[kHalves - 1][t][2 + i]));
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) top[t][i] = fmaxf(top[t][i], __shfl_xor_sync(0xFFFFFFFFu, top[t][i], s));
          top[t][i] = fmaxf(top[t][i], m[t][i]);
          whole[t][i] = rintf(top[t][i] * unit[t][i]);
          next_far = next_far || !(fabsf(whole[t][i]) < kAtFar);
        }
      }
      next_far = __any_sync(0xFFFFFFFFu, next_far);
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // from what the weights referred to: m unit itself where far, else the whole number nearest to it
          const float old = 7.f - base[t][i];
          const float f = at_exp2(far ? (next_far ? (m[t][i] - top[t][i]) * unit[t][i] : fmaf(m[t][i], unit[t][i], -whole[t][i]))
                                      : (next_far ? fmaf(-top[t][i], unit[t][i], old) : old - whole[t][i]));
          m[t][i] = top[t][i];
          lim[t][i] = top[t][i] == kA4Least ? kA4Least : top[t][i] + 8.f / unit[t][i];
          base[t][i] = 7.f - whole[t][i];
          l[t][i] *= f;
          z[t][i] *= f;
          const float fo = f * v_factor;
#pragma unroll
          for (int k = 0; k < 2 * NG; ++k) o[t][k][i] *= fo, o[t][k][2 + i] *= fo;
        }
      }
      far = next_far;
    }
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      if (far) {  // the difference from m, which is exact near it; the base's rounding would be whole units
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[hf][t][i] = at_exp2(fmaf(sc[hf][t][i] - m[t][i & 1], unit[t][i & 1], 7.f));
      } else {
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[hf][t][i] = at_exp2(fmaf(sc[hf][t][i], unit[t][i & 1], base[t][i & 1]));
      }
    }
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      const unsigned char *params = here + kVp + hf * kA4Half * 16;
      uint32_t vr[2][4];  // (scale, middle) of the groups of keys r and r + 8
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (kPairs == 4) *reinterpret_cast<uint4 *>(vr[i]) = *reinterpret_cast<const uint4 *>(params + (r + 8 * i) * 16);
        else *reinterpret_cast<uint2 *>(vr[i]) = *reinterpret_cast<const uint2 *>(params + (r + 8 * i) * 16);
      }
      float vs[2][NG];
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) vs[i][g] = a4_low(vr[i][g]) * (NQ == 1 ? 1.f : v_unit);
      uint32_t pw[NQ][NG][2];  // weights times the groups' scales as B: keys 2c and 2c + 1 of query r, then keys + 8
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        float w[4] = {sc[hf][t][0], sc[hf][t][1], sc[hf][t][2], sc[hf][t][3]};
        l[t][0] += w[0] + w[2];
        l[t][1] += w[1] + w[3];
        a4_mma_top(z[t], vp[hf][0], vp[hf][1], a4_turn(a4_pack(w[0], w[1])), a4_turn(a4_pack(w[2], w[3])));
        if (NQ == 1) w[0] *= v_unit, w[1] *= v_unit, w[2] *= v_unit, w[3] *= v_unit;  // or the scales: fewer of these
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          pw[t][g][0] = a4_turn(a4_pack(w[0] * vs[0][g], w[1] * vs[0][g]));
          pw[t][g][1] = a4_turn(a4_pack(w[2] * vs[1][g], w[3] * vs[1][g]));
        }
      }
      // -8 2^-24 and -8 2^-20, of the rows whose codes are in the lower and the upper nibble; then the codes
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            a4_mma(o[t][2 * g + i], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pw[t][g][0], pw[t][g][1]);
      uint32_t f[4];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if ((g & 1) == 0) ldmatrix4t(f, kst + kV + hf * kA4Half * kPitch + mat + g * 16);
        const uint32_t w0 = f[2 * (g & 1)], w1 = f[2 * (g & 1) + 1], w2 = w0 >> 8, w3 = w1 >> 8;
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          a4_mma(o[t][2 * g], w0 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x000F000Fu, w1 & 0x00F000F0u, pw[t][g][0], pw[t][g][1]);
          a4_mma(o[t][2 * g + 1], w2 & 0x000F000Fu, w2 & 0x00F000F0u, w3 & 0x000F000Fu, w3 & 0x00F000F0u, pw[t][g][0], pw[t][g][1]);
        }
      }
    }
    if (partial) {
#pragma unroll
      for (int t = 0; t < NQ; ++t)
        if (lost[t]) {
          const float nan = __uint_as_float(0x7FFFFFFFu);
          if ((r & 1) && (lost[t] >> (r >> 1)) & 1) z[t][0] = nan;
          if ((r & 1) && (lost[t] >> (8 + (r >> 1))) & 1) z[t][1] = nan;
        }
    }
    __syncwarp();  // the stage is read: the next round's copies may overwrite it
    if (++stage == kStages) stage = 0;
    if (++now.tile < now.end) continue;
    const int64_t piece = (int64_t)now.b * hcs + now.hc + wid;
    const float low = 0x1p17f / v_unit, high = 0x1p13f / v_unit;  // 2^24 and 2^20 without the weights' 2^7
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], s);
        const int g = t * 8 + c * 2 + i;
        const int64_t rec = piece * a.chunk_rows + g;
        // what the weights refer to, to the last bit: a query that saw no score refers to nothing
        const float ref = m[t][i] == kA4Least ? kNone : far ? fminf(fmaxf(m[t][i] * unit[t][i], -3e38f), 3e38f) : 7.f - base[t][i];
        if (g < n && r == 0) a.own_ml[rec] = make_float2(ref, broken ? kAtBadPage : l[t][i] * 0x1p-7f);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const float middle = __shfl_sync(0xFFFFFFFFu, z[t][i], (2 * k + 1) * 4 + c) * 0x1p-7f;
          const int d = k * 32 + r * 4;
          if (g < n && d < x.cache.head_dim)
            *reinterpret_cast<float4 *>(a.own_o + rec * x.cache.head_dim + d) =
                make_float4(fmaf(o[t][2 * k][i], low, middle), fmaf(o[t][2 * k][2 + i], high, middle),
                            fmaf(o[t][2 * k + 1][i], low, middle), fmaf(o[t][2 * k + 1][2 + i], high, middle));
        }
      }
    }
    fresh = true;
    a4_item_next<kTile>(a, now);
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
    const int64_t units = a4_units(keys, a.tile), u = start + hc * units, w = (u + kA4Item) / share;
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
