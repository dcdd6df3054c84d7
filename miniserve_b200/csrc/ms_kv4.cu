// ms_kv4_append and ms_kv4_read -- a paged cache held in 4 bits, written with
// the position rotation applied on the way, and read back (declared in
// include/mssample.h).
//
// Every 32 entries y of a head (the last ones of a head may be fewer) share a
// scale s and a middle m, both fp16:
//
//   s = (max y - min y) / 15,  m = min y + 8 s,
//   code = clamp(rint((y - m) / s) + 8, 0, 15),  y ~ m + s (code - 8)
//
// m is computed from the rounded s and the codes from the rounded m, so that
// these two roundings (2^-12 of 15 s and of m, beside the codes' s / 2) move
// the range by less than a hundredth of a step where m is within its size.
// The divisions are products with the rounded reciprocals of 15 and s.  The
// rotated entries are not rounded to the model's type in between.
//
// Both are bound by bytes: an append reads each entry in 2 bytes and writes
// 5 bits of it, a read back the reverse.  Measured: 20011 tokens of 32 query and
// 8 + 8 key and value heads of 128 in 94 us, 436 MB at 4.6 TB/s (70 % of a plain
// copy's rate: every entry costs some ten operations, issue slots are 60 % busy and
// 44 % of the warps resident; a thread loads both sides of a key's pairs and turns
// one, and every key head loads the table again); 8 tokens in 2.2 us, a launch.
// 65536 tokens of 8 heads of 128 read back in 62 us, 352 MB at 5.7 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mssample.h"
#include "ms_host.h"
#include "ms_kv.cuh"
#include "ms_kv4.cuh"
#include "ms_tc.cuh"

namespace ms {

constexpr int kK4Threads = 256;

// Quotients of numbers below 2^16 (or, by divisors up to 64, below 2^26) from a
// product: u / d is the high word of u ceil(2^32 / d), as long as u times what
// the ceiling adds (less than d) is below 2^32.
struct K4Divisor {
  uint32_t d, inverse;
};
static K4Divisor k4_divisor(int64_t d) { return K4Divisor{(uint32_t)d, (uint32_t)((0x100000000ull + d - 1) / d)}; }
__device__ __forceinline__ int k4_over(int u, const K4Divisor &d) { return d.d == 1 ? u : (int)__umulhi((uint32_t)u, d.inverse); }

__device__ __forceinline__ float k4_min(float x, float y) {  // a NaN stays
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float k4_min3(float x, float y, float z) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float k4_max3(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float k4_max(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// kV entries as floats.
template <typename T, int kV>
__device__ __forceinline__ void k4_load(const T *p, float (&x)[kV]) {
  if constexpr (kV == 1) {
    x[0] = kv_to_float(load_in(p));
  } else {
    uint32_t u[kV / 2];
    if constexpr (kV == 8) *reinterpret_cast<uint4 *>(u) = load_in(reinterpret_cast<const uint4 *>(p));
    else *reinterpret_cast<uint2 *>(u) = load_in(reinterpret_cast<const uint2 *>(p));
#pragma unroll
    for (int i = 0; i < kV / 2; ++i) {
      const float2 f = kv_widen<T>(u[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
// kN floats of a table row.
template <int kN>
__device__ __forceinline__ void k4_table(const float *p, float (&x)[kN]) {
  if constexpr (kN == 1) x[0] = load_in(p);
  else if constexpr (kN == 2) *reinterpret_cast<float2 *>(x) = load_in(reinterpret_cast<const float2 *>(p));
  else {
#pragma unroll
    for (int i = 0; i < kN; i += 4) *reinterpret_cast<float4 *>(x + i) = load_in(reinterpret_cast<const float4 *>(p + i));
  }
}

// Entries e0 .. e0 + 7 of a head, rotated where they lie below `rotary` and the
// head turns.  Pieces of kV entries lie on one side of a rotation (the host
// chooses kV so).  Products and sums are rounded apart: what is quantised then
// does not depend on how a compiler contracts them.
template <typename T, bool kInterleaved, int kV>
__device__ __forceinline__ void k4_entries(const T *src, int e0, bool turns, int rotary, const float *row, float (&y)[8]) {
  const int half = rotary >> 1;
#pragma unroll
  for (int p = 0; p < 8; p += kV) {
    const int e = e0 + p;
    float x[kV];
    k4_load<T, kV>(src + e, x);
    if (!turns || e >= rotary) {
#pragma unroll
      for (int i = 0; i < kV; ++i) y[p + i] = x[i];
    } else if constexpr (kInterleaved && kV > 1) {
      float c[kV / 2], s[kV / 2];
      k4_table<kV / 2>(row + (e >> 1), c);
      k4_table<kV / 2>(row + half + (e >> 1), s);
#pragma unroll
      for (int i = 0; i < kV / 2; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        y[p + 2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
        y[p + 2 * i + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
      }
    } else {
      const bool first = kInterleaved ? (e & 1) == 0 : e < half;
      const int at = kInterleaved ? e >> 1 : first ? e : e - half;  // pair of the piece's first entry
      float other[kV], c[kV], s[kV];
      k4_load<T, kV>(src + (kInterleaved ? e ^ 1 : first ? e + half : e - half), other);
      k4_table<kV>(row + at, c);
      k4_table<kV>(row + half + at, s);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float own = __fmul_rn(x[i], c[i]), cross = __fmul_rn(other[i], s[i]);
        y[p + i] = first ? __fsub_rn(own, cross) : __fadd_rn(own, cross);
      }
    }
  }
}

struct K4AppendArgs {
  ms_kv4_append_args a;
  K4Layout layout;
  int page_shift;
  int q_blocks;             // the first blocks: queries
  int q_tokens, kv_tokens;  // tokens of a block
  int q_slots;              // threads' heads of a token: h, and h + q_slots
  int piece, q_piece;       // entries loaded at once (8, 4 or 1) of the keys and values, and of the queries
  K4Divisor units, q_token;     // of a head's pieces of the queries, and of a token's
  K4Divisor chunks, kv_token;   // of a stored head's 8-entry chunks, and of a token's
};

constexpr int kK4Tokens = 64;  // tokens of a block, at most

__device__ __forceinline__ int64_t k4_position(const ms_kv4_append_args &a, int64_t t, bool &good) {
  int64_t at = 0;
  good = true;
  if (a.rotary > 0) {
    at = load_in(a.positions + t);
    good = at >= 0 && at < a.table_rows;
  }
  return good ? at : 0;
}

// kV entries as they are, and one of them (two of them, where kV > 1).
template <typename T, int kV>
struct K4Raw {
  uint32_t u[kV / 2];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kV == 8) *reinterpret_cast<uint4 *>(u) = load_in(reinterpret_cast<const uint4 *>(p));
    else *reinterpret_cast<uint2 *>(u) = load_in(reinterpret_cast<const uint2 *>(p));
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (kV == 8) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(u);
    else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(u);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kV / 2; ++i) u[i] = 0;
  }
};
template <typename T>
struct K4Raw<T, 1> {
  T x;
  __device__ __forceinline__ void load(const T *p) { x = load_in(p); }
  __device__ __forceinline__ void store(T *p) const { *p = x; }
  __device__ __forceinline__ void clear() { kv_from_float(0.f, x); }
};
// Pairs of x and y turned by cosines c and sines s.
template <typename T, bool kInterleaved, int kV>
__device__ __forceinline__ void k4_turn(K4Raw<T, kV> &x, K4Raw<T, kV> &y, const float (&c)[kV], const float (&s)[kV]) {
  if constexpr (kV == 1) {
    const float f = kv_to_float(x.x), g = kv_to_float(y.x);
    kv_from_float(f * c[0] - g * s[0], x.x);
    kv_from_float(g * c[0] + f * s[0], y.x);
  } else {
#pragma unroll
    for (int k = 0; k < kV / 2; ++k) {
      const float2 f = kv_widen<T>(x.u[k]), g = kv_widen<T>(y.u[k]);
      if (kInterleaved) {  // word k of x is pair k, word k of y is pair kV / 2 + k
        const int i = kV / 2 + k;
        x.u[k] = kv_narrow<T>(f.x * c[k] - f.y * s[k], f.y * c[k] + f.x * s[k]);
        y.u[k] = kv_narrow<T>(g.x * c[i] - g.y * s[i], g.y * c[i] + g.x * s[i]);
      } else {  // word k holds the first (x) and second (y) entries of pairs 2k and 2k + 1
        x.u[k] = kv_narrow<T>(f.x * c[2 * k] - g.x * s[2 * k], f.y * c[2 * k + 1] - g.y * s[2 * k + 1]);
        y.u[k] = kv_narrow<T>(g.x * c[2 * k] + f.x * s[2 * k], g.y * c[2 * k + 1] + f.y * s[2 * k + 1]);
      }
    }
  }
}

// Queries: a thread owns both sides of kV pairs (or 2 kV copied entries) of up
// to two heads, which share its cosines and sines; q_out may be q itself.  Its
// loads are issued before anything that depends on the token's position.
template <typename T, bool kInterleaved, int kV>
__device__ __forceinline__ void k4_queries(const K4AppendArgs &p) {
  const ms_kv4_append_args &a = p.a;
  const int half = a.rotary >> 1;
  const int64_t t0 = (int64_t)blockIdx.x * p.q_tokens;
  const int tokens = (int)min((int64_t)p.q_tokens, a.tokens - t0), items = tokens * (int)p.q_token.d;
  for (int u = threadIdx.x; u < items; u += kK4Threads) {
    const int tl = tokens == 1 ? 0 : k4_over(u, p.q_token), w = u - tl * (int)p.q_token.d;
    const int h = k4_over(w, p.units), j = w - h * (int)p.units.d;
    const int64_t t = t0 + tl;
    const bool rotates = j * 2 * kV < a.rotary, both = h + p.q_slots < a.heads;
    const int lo = rotates && !kInterleaved ? j * kV : j * 2 * kV, hi = rotates && !kInterleaved ? lo + half : lo + kV;
    const T *src = static_cast<const T *>(a.q) + t * a.q_token + h * a.q_head;
    K4Raw<T, kV> x[2], y[2];
    x[0].load(src + lo), y[0].load(src + hi);
    if (both) {
      const T *next = src + p.q_slots * a.q_head;
      x[1].load(next + lo), y[1].load(next + hi);
    }
    bool good;
    const int64_t at = k4_position(a, t, good);
    float c[kV], s[kV];
    if (rotates) {
      k4_table<kV>(a.table + at * a.rotary + j * kV, c);
      k4_table<kV>(a.table + at * a.rotary + half + j * kV, s);
    }
    T *dst = static_cast<T *>(a.q_out) + t * a.q_out_token + h * a.q_out_head;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !both) break;
      if (!good) x[i].clear(), y[i].clear();
      else if (rotates) k4_turn<T, kInterleaved, kV>(x[i], y[i], c, s);
      x[i].store(dst + lo), y[i].store(dst + hi);
      dst += p.q_slots * a.q_out_head;
    }
  }
}

// Eight entries (none where `inside` is not set) of a group that four
// neighbouring threads share: its codes, its parameters, and whether fp16 does
// not hold it.
__device__ __forceinline__ uint32_t k4_encode(const float (&y)[8], bool inside, __half2 &param, bool &lost) {
  float lo = __uint_as_float(0x7F800000u), hi = -lo;
  if (inside) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) lo = k4_min3(lo, y[i], y[i + 1]), hi = k4_max3(hi, y[i], y[i + 1]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = k4_min(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
    hi = k4_max(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
  }
  param = __halves2half2(__float2half_rn(0.f), __float2half_rn(0.f));
  lost = false;
  if (hi < lo) return 0;  // the padding behind a head
  const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)),
               middle = __float2half_rn(__fadd_rn(lo, 8.f * __half2float(scale)));
  const float s = __half2float(scale), m = __half2float(middle);
  if (!(s <= 65504.f && fabsf(m) <= 65504.f)) {  // what fp16 does not hold, and what is not a number, reads back as NaN
    param = __halves2half2(__float2half_rn(0.f), __ushort_as_half(0x7FFF));
    lost = true;
    return 0x88888888u;
  }
  param = __halves2half2(scale, middle);
  const float inverse = s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t word = 0;
  if (inside) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // the nearest whole number from the low bits of its sum with 1.5 * 2^23 (+ 8)
      const float step = fminf(fmaxf(__fmul_rn(__fsub_rn(y[i], m), inverse), -8.f), 7.f);
      word |= (__float_as_uint(__fadd_rn(step, 12582920.f)) & 15u) << (4 * i);
    }
  }
  return word;
}

// Keys and values: a thread takes 8 entries of a key head and the same 8 of its
// value head, and four neighbouring threads a group of each.  A token's keys
// and values are all one block's, so that its status is written once, whatever
// its groups hold.  (A thread for keys or values alone finds slot, position and
// addresses twice: 20011 tokens appended and read back 169 us, so 121.)
template <typename T, bool kInterleaved, int kV>
__device__ __forceinline__ void k4_quantise(const K4AppendArgs &p, int *flags) {
  const ms_kv4_append_args &a = p.a;
  const int64_t t0 = (int64_t)((int)blockIdx.x - p.q_blocks) * p.kv_tokens;
  const int tokens = (int)min((int64_t)p.kv_tokens, a.tokens - t0);
  for (int i = threadIdx.x; i < tokens; i += kK4Threads) flags[i] = 0;
  __syncthreads();
  const int items = tokens * (int)p.kv_token.d;
  for (int u0 = threadIdx.x & ~31; u0 < items; u0 += kK4Threads) {  // whole warps: the shuffles
    const int u = u0 + (threadIdx.x & 31);
    const bool live = u < items;
    const int tl = live && tokens > 1 ? k4_over(u, p.kv_token) : 0, w = live ? u - tl * (int)p.kv_token.d : 0;
    const int h = k4_over(w, p.chunks), chunk = w - h * (int)p.chunks.d;
    const int64_t t = t0 + tl;
    const int64_t slot = load_in(a.slots + t);
    bool good;
    const int64_t at = k4_position(a, t, good);
    int status = good ? 0 : MS_ROW_BAD_POSITION;
    if (slot >= a.cache.pages * a.cache.page_size) status |= MS_ROW_BAD_SLOT;
    const bool write = live && slot >= 0 && status == 0, inside = write && chunk * 8 < a.cache.head_dim;
    float y[2][8];
    if (inside) {
      k4_entries<T, kInterleaved, kV>(static_cast<const T *>(a.v) + t * a.v_token + h * a.v_head, chunk * 8, false, a.rotary,
                                      nullptr, y[1]);
      k4_entries<T, kInterleaved, kV>(static_cast<const T *>(a.k) + t * a.k_token + h * a.k_head, chunk * 8, true, a.rotary,
                                      a.table + at * a.rotary, y[0]);
    }
    uint32_t word[2];
    __half2 param[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      bool lost;
      word[side] = k4_encode(y[side], inside, param[side], lost);
      if (lost) status |= MS_ROW_NONFINITE;
    }
    if (write) {
      int64_t page, offset;
      kv_place(slot, a.cache.page_size, p.page_shift, page, offset);
      const int64_t row = (page * a.cache.kv_heads + h) * a.cache.page_size + offset;
      const int64_t code_at = row * p.layout.row_bytes + chunk * 4, param_at = row * p.layout.groups + (chunk >> 2);
      *reinterpret_cast<uint32_t *>(a.cache.k_codes + code_at) = word[0];
      *reinterpret_cast<uint32_t *>(a.cache.v_codes + code_at) = word[1];
      if ((chunk & 3) == 0) {
        static_cast<__half2 *>(a.cache.k_params)[param_at] = param[0];
        static_cast<__half2 *>(a.cache.v_params)[param_at] = param[1];
      }
    }
    if (live && (chunk & 3) == 0 && status) atomicOr(&flags[tl], status);
  }
  __syncthreads();
  if (a.status)
    for (int i = threadIdx.x; i < tokens; i += kK4Threads) a.status[t0 + i] = flags[i];
}

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kK4Threads, 4) ms_kv4_append_kernel(const __grid_constant__ K4AppendArgs p) {
  __shared__ int flags[kK4Tokens];
  grid_wait();
  if ((int)blockIdx.x < p.q_blocks) {
    if (p.q_piece == 8) k4_queries<T, kInterleaved, 8>(p);
    else if (p.q_piece == 4) k4_queries<T, kInterleaved, 4>(p);
    else k4_queries<T, kInterleaved, 1>(p);
  } else {
    if (p.piece == 8) k4_quantise<T, kInterleaved, 8>(p, flags);
    else if (p.piece == 4) k4_quantise<T, kInterleaved, 4>(p, flags);
    else k4_quantise<T, kInterleaved, 1>(p, flags);
  }
}

struct K4ReadArgs {
  ms_kv4_read_args a;
  K4Layout layout;
  int page_shift;
  int tokens;  // tokens of a block
  int wide;    // outputs are stored in 16 bytes
  int slots, heads;         // threads' heads of a token: h, and h + slots where heads is 2
  K4Divisor chunks, token;  // of a head's 8-entry chunks, and of a token's
};

// Eight entries of codes and (scale, middle), as pairs of T.  A code in a half's
// low bits over the bits of 1024 is 1024 + code: less 1032, exact, it is code - 8.
template <typename T>
__device__ __forceinline__ void k4_decode(uint32_t word, __half2 param, uint32_t (&out)[4]) {
  const __half2 less = __floats2half2_rn(-1032.f, -1032.f);
  __half2 step[4];  // entries i and i + 4
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = ((word >> (4 * i)) & 0x000F000Fu) | 0x64006400u;
    step[i] = __hadd2(*reinterpret_cast<const __half2 *>(&u), less);
  }
  const float s = __low2float(param), m = __high2float(param);
  if constexpr (__is_same(T, __half)) {
    const __half2 s2 = __low2half2(param), m2 = __high2half2(param);
    __half2 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __hfma2(step[i], s2, m2);  // rounded once
    if (!(fmaf(8.f, fabsf(s), fabsf(m)) <= 65000.f)) {  // finite entries stay finite, NaN stays
      const __half2 most = __floats2half2_rn(65504.f, 65504.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = __hmax2_nan(__hmin2_nan(y[i], most), __hneg2(most));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2 low = __lows2half2(y[2 * i], y[2 * i + 1]), high = __highs2half2(y[2 * i], y[2 * i + 1]);
      out[i] = *reinterpret_cast<const uint32_t *>(&low), out[2 + i] = *reinterpret_cast<const uint32_t *>(&high);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = __half22float2(step[2 * i]), g = __half22float2(step[2 * i + 1]);
      out[i] = kv_narrow<T>(fmaf(s, f.x, m), fmaf(s, g.x, m));
      out[2 + i] = kv_narrow<T>(fmaf(s, f.y, m), fmaf(s, g.y, m));
    }
  }
}

// A thread takes 8 entries of a key head and the same 8 of its value head, of one
// or, where that leaves threads enough for the GPU four times over, two heads
// (65536 tokens: 71 us with one, 62 with two).
template <typename T>
__global__ void __launch_bounds__(kK4Threads) ms_kv4_read_kernel(const __grid_constant__ K4ReadArgs p) {
  grid_wait();
  const ms_kv4_read_args &a = p.a;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int tokens = (int)min((int64_t)p.tokens, a.tokens - t0), items = tokens * (int)p.token.d;
  for (int u = threadIdx.x; u < items; u += kK4Threads) {
    const int tl = tokens == 1 ? 0 : k4_over(u, p.token), w = u - tl * (int)p.token.d;
    const int h = k4_over(w, p.chunks), chunk = w - h * (int)p.chunks.d;
    const int64_t t = t0 + tl, slot = load_in(a.slots + t);
    const bool bad = slot >= a.cache.pages * a.cache.page_size, live = slot >= 0 && !bad;
    if (w == 0 && a.status) a.status[t] = bad ? MS_ROW_BAD_SLOT : MS_ROW_OK;
    int64_t page = 0, offset = 0;
    if (live) kv_place(slot, a.cache.page_size, p.page_shift, page, offset);
    const int64_t row = (page * a.cache.kv_heads + h) * a.cache.page_size + offset;
    const int64_t code_at = row * p.layout.row_bytes + chunk * 4, param_at = row * p.layout.groups + (chunk >> 2);
    uint32_t word[2][2];
    __half2 param[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // all loads first
      word[i][0] = word[i][1] = 0;
      param[i][0] = param[i][1] = __halves2half2(__float2half_rn(0.f), __float2half_rn(0.f));
      if (live && (i == 0 || (p.heads > 1 && h + p.slots < a.cache.kv_heads))) {
        const int64_t rows = i * p.slots * a.cache.page_size;
        word[i][0] = load_in(reinterpret_cast<const uint32_t *>(a.cache.k_codes + code_at + rows * p.layout.row_bytes));
        word[i][1] = load_in(reinterpret_cast<const uint32_t *>(a.cache.v_codes + code_at + rows * p.layout.row_bytes));
        param[i][0] = load_in(static_cast<const __half2 *>(a.cache.k_params) + param_at + rows * p.layout.groups);
        param[i][1] = load_in(static_cast<const __half2 *>(a.cache.v_params) + param_at + rows * p.layout.groups);
      }
    }
    T *k = static_cast<T *>(a.k_out) + t * a.k_token + h * a.k_head + chunk * 8;
    T *v = static_cast<T *>(a.v_out) + t * a.v_token + h * a.v_head + chunk * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !(p.heads > 1 && h + p.slots < a.cache.kv_heads)) break;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        T *dst = side ? v : k;
        uint32_t out[4];
        k4_decode<T>(word[i][side], param[i][side], out);
        if (p.wide) {
          *reinterpret_cast<uint4 *>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const T *pair = reinterpret_cast<const T *>(&out[j]);
            dst[2 * j] = pair[0], dst[2 * j + 1] = pair[1];
          }
        }
      }
      k += p.slots * a.k_head, v += p.slots * a.v_head;
    }
  }
}

// Tokens of a block: each thread up to `items` items, so that a block's start and
// end are paid for, but no fewer blocks than fill the GPU.  20011 tokens appended
// and read back, four items of keys and values and two of queries: 119 us; one
// and two 126, eight and two 122, four and one 123.
static int k4_tokens(int64_t tokens, int64_t per_token, int items) {
  const int64_t fill = tokens * per_token / (148 * 8 * kK4Threads);
  const int64_t each = fill < 1 ? 1 : fill < items ? fill : items;
  const int64_t n = each * kK4Threads / per_token;
  return (int)(n < 1 ? 1 : n > kK4Tokens ? kK4Tokens : n);
}

template <typename T>
static cudaError_t k4_append(const K4AppendArgs &p, int64_t blocks, cudaStream_t s) {
  auto *kernel = p.a.interleaved ? ms_kv4_append_kernel<T, true> : ms_kv4_append_kernel<T, false>;
  return launch_dependent(kernel, (unsigned)blocks, kK4Threads, 0, s, p);
}

}  // namespace ms

extern "C" {

int ms_kv4_append(const ms_kv4_append_args *args, ms_stream_t stream) {
  if (!args) return MS_E_INVALID;
  ms::K4AppendArgs p{};
  p.a = *args;
  const ms_kv4_append_args &a = p.a;
  if (a.dtype != MS_DTYPE_BF16 && a.dtype != MS_DTYPE_F16) return MS_E_DTYPE;
  if (a.tokens < 0 || a.tokens > 0x7FFFFFFFll || a.heads < 0 || a.heads > 65536 || a.rotary < 0 ||
      a.rotary > a.cache.head_dim || (a.rotary & 1))
    return MS_E_INVALID;
  int rc = ms::k4_check(a.cache);
  if (rc != MS_OK) return rc;
  if (a.tokens == 0) return MS_OK;
  if (!a.k || !a.v || !a.slots || (a.heads > 0 && (!a.q || !a.q_out)) ||
      (a.rotary > 0 && (!a.positions || !a.table || a.table_rows < 1)))
    return MS_E_INVALID;
  p.layout = ms::k4_layout(a.cache.head_dim);
  p.page_shift = ms::kv_page_shift(a.cache.page_size);
  p.chunks = ms::k4_divisor(p.layout.row_bytes / 4);
  // the largest pieces that strides and bases allow: of the keys and values those that lie on one side of a rotation,
  // of the queries those that come in pairs
  const bool table = a.rotary == 0 || (reinterpret_cast<uintptr_t>(a.table) & 15) == 0;
  const int64_t strides = a.k_token | a.k_head | a.v_token | a.v_head, q_strides = a.q_token | a.q_head | a.q_out_token | a.q_out_head;
  const uint64_t bases = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v),
                 q_bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out);
  const int side = a.interleaved ? a.rotary : a.rotary / 2;
  auto largest = [&](auto fits) { return table && fits(8) ? 8 : table && fits(4) ? 4 : 1; };
  p.piece = largest([&](int v) {
    return side % v == 0 && (strides & (v - 1)) == 0 && (bases & (2 * v - 1)) == 0;
  });
  p.q_piece = largest([&](int v) {
    return a.rotary % (2 * v) == 0 && (q_strides & (v - 1)) == 0 && (q_bases & (2 * v - 1)) == 0;
  });
  p.units = ms::k4_divisor(a.cache.head_dim / (2 * p.q_piece));
  p.q_slots = (a.heads + 1) / 2;
  const int64_t kv_items = (int64_t)a.cache.kv_heads * p.chunks.d, q_items = (int64_t)p.q_slots * p.units.d;
  p.kv_token = ms::k4_divisor(kv_items);
  p.q_token = ms::k4_divisor(q_items ? q_items : 1);
  p.kv_tokens = ms::k4_tokens(a.tokens, kv_items, 4);
  p.q_tokens = q_items ? ms::k4_tokens(a.tokens, q_items, 2) : 1;
  p.q_blocks = q_items ? (int)((a.tokens + p.q_tokens - 1) / p.q_tokens) : 0;
  const int64_t blocks = p.q_blocks + (a.tokens + p.kv_tokens - 1) / p.kv_tokens;
  if (blocks > 0x7FFFFFFFll) return MS_E_INVALID;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = a.dtype == MS_DTYPE_BF16 ? ms::k4_append<__nv_bfloat16>(p, blocks, s)
                                           : ms::k4_append<__half>(p, blocks, s);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

int ms_kv4_read(const ms_kv4_read_args *args, ms_stream_t stream) {
  if (!args) return MS_E_INVALID;
  ms::K4ReadArgs p{};
  p.a = *args;
  const ms_kv4_read_args &a = p.a;
  if (a.dtype != MS_DTYPE_BF16 && a.dtype != MS_DTYPE_F16) return MS_E_DTYPE;
  if (a.tokens < 0 || a.tokens > 0x7FFFFFFFll) return MS_E_INVALID;
  int rc = ms::k4_check(a.cache);
  if (rc != MS_OK) return rc;
  if (a.tokens == 0) return MS_OK;
  if (!a.slots || !a.k_out || !a.v_out) return MS_E_INVALID;
  p.layout = ms::k4_layout(a.cache.head_dim);
  p.page_shift = ms::kv_page_shift(a.cache.page_size);
  p.chunks = ms::k4_divisor(a.cache.head_dim / 8);
  p.heads = a.tokens * a.cache.kv_heads * p.chunks.d > 4ll * 148 * 2048 ? 2 : 1;
  p.slots = (a.cache.kv_heads + p.heads - 1) / p.heads;
  p.token = ms::k4_divisor((int64_t)p.slots * p.chunks.d);
  p.tokens = ms::k4_tokens(a.tokens, p.token.d, 4);
  p.wide = ((a.k_token | a.k_head | a.v_token | a.v_head) & 7) == 0 &&
           ((reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) & 15) == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto *kernel = a.dtype == MS_DTYPE_BF16 ? ms::ms_kv4_read_kernel<__nv_bfloat16> : ms::ms_kv4_read_kernel<__half>;
  cudaError_t e = ms::launch_dependent(kernel, (unsigned)((a.tokens + p.tokens - 1) / p.tokens), ms::kK4Threads, 0, s, p);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
