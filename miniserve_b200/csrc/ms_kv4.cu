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
// 5 bits of it, a read back the reverse.
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
  int q_blocks;           // the first blocks: queries
  int q_tokens, kv_tokens;  // tokens of a block
  int chunks;             // 8-entry chunks of a stored head
  int piece, q_piece;     // entries loaded at once (8, 4 or 1) of the keys and values, and of the queries
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

template <typename T, int kV>
__device__ __forceinline__ void k4_store(T *p, const float (&x)[kV]) {
  if constexpr (kV == 1) {
    kv_from_float(x[0], *p);
  } else {
    uint32_t u[kV / 2];
#pragma unroll
    for (int i = 0; i < kV / 2; ++i) u[i] = kv_narrow<T>(x[2 * i], x[2 * i + 1]);
    if constexpr (kV == 8) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(u);
    else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(u);
  }
}

// Queries: a thread owns both sides of kV pairs (or 2 kV copied entries) of a
// head, so that q_out may be q itself.
template <typename T, bool kInterleaved, int kV>
__device__ __forceinline__ void k4_queries(const K4AppendArgs &p) {
  const ms_kv4_append_args &a = p.a;
  const int units = a.cache.head_dim / (2 * kV), half = a.rotary >> 1;
  const int64_t t0 = (int64_t)blockIdx.x * p.q_tokens;
  const int per_token = a.heads * units;
  const int items = (int)min((int64_t)p.q_tokens, a.tokens - t0) * per_token;
  for (int u = threadIdx.x; u < items; u += kK4Threads) {
    const int tl = u / per_token, w = u - tl * per_token;
    const int h = w / units, j = w - h * units;
    const int64_t t = t0 + tl;
    const bool rotates = j * 2 * kV < a.rotary;
    const int lo = rotates && !kInterleaved ? j * kV : j * 2 * kV, hi = rotates && !kInterleaved ? lo + half : lo + kV;
    const T *src = static_cast<const T *>(a.q) + t * a.q_token + h * a.q_head;
    float x[kV], y[kV];
    k4_load<T, kV>(src + lo, x);
    k4_load<T, kV>(src + hi, y);
    bool good;
    const int64_t at = k4_position(a, t, good);
    if (!good) {
#pragma unroll
      for (int i = 0; i < kV; ++i) x[i] = y[i] = 0.f;
    } else if (rotates) {
      float c[kV], s[kV];
      k4_table<kV>(a.table + at * a.rotary + j * kV, c);
      k4_table<kV>(a.table + at * a.rotary + half + j * kV, s);
      auto turn = [](float &f, float &g, float cosine, float sine) {
        const float first = f * cosine - g * sine;
        g = g * cosine + f * sine;
        f = first;
      };
      if constexpr (kInterleaved && kV > 1) {
#pragma unroll
        for (int i = 0; i < kV / 2; ++i) {
          turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
          turn(y[2 * i], y[2 * i + 1], c[kV / 2 + i], s[kV / 2 + i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) turn(x[i], y[i], c[i], s[i]);
      }
    }
    T *dst = static_cast<T *>(a.q_out) + t * a.q_out_token + h * a.q_out_head;
    k4_store<T, kV>(dst + lo, x);
    k4_store<T, kV>(dst + hi, y);
  }
}

// Keys and values: a thread takes 8 entries of one head, and four neighbouring
// threads a group, whose extremes two shuffles find.  A token's keys and
// values are all one block's, so that its status is written once, whatever its
// groups hold.
template <typename T, bool kInterleaved, int kV>
__device__ __forceinline__ void k4_quantise(const K4AppendArgs &p, int *flags) {
  const ms_kv4_append_args &a = p.a;
  const int64_t t0 = (int64_t)((int)blockIdx.x - p.q_blocks) * p.kv_tokens;
  const int tokens = (int)min((int64_t)p.kv_tokens, a.tokens - t0);
  for (int i = threadIdx.x; i < tokens; i += kK4Threads) flags[i] = 0;
  __syncthreads();
  const int per_token = 2 * a.cache.kv_heads * p.chunks;
  const int items = tokens * per_token;
  for (int u0 = threadIdx.x & ~31; u0 < items; u0 += kK4Threads) {  // whole warps: the shuffles
    const int u = u0 + (threadIdx.x & 31);
    const bool live = u < items;
    const int tl = live ? u / per_token : 0, w = live ? u - tl * per_token : 0;
    const int side = w / p.chunks, chunk = w - side * p.chunks;
    const bool key = side < a.cache.kv_heads;
    const int h = key ? side : side - a.cache.kv_heads;
    const int64_t t = t0 + tl;
    const int64_t slot = load_in(a.slots + t);
    bool good;
    const int64_t at = k4_position(a, t, good);
    int status = good ? 0 : MS_ROW_BAD_POSITION;
    if (slot >= a.cache.pages * a.cache.page_size) status |= MS_ROW_BAD_SLOT;
    const bool write = live && slot >= 0 && status == 0;
    const bool inside = write && chunk * 8 < a.cache.head_dim;
    float y[8];
    float lo = __uint_as_float(0x7F800000u), hi = -lo;
    bool finite = true;
    if (inside) {
      const T *src = key ? static_cast<const T *>(a.k) + t * a.k_token + h * a.k_head
                         : static_cast<const T *>(a.v) + t * a.v_token + h * a.v_head;
      k4_entries<T, kInterleaved, kV>(src, chunk * 8, key, a.rotary, a.table + at * a.rotary, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, y[i]);
        hi = fmaxf(hi, y[i]);
        finite = finite && fabsf(y[i]) <= 3.402823466e38f;
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    const uint32_t all = __ballot_sync(0xFFFFFFFFu, finite);
    finite = ((all >> (threadIdx.x & 28)) & 15u) == 15u;  // the group's four threads
    uint32_t word = 0;
    __half scale = __float2half_rn(0.f), middle = scale;
    if (hi >= lo || !finite) {  // not the padding behind a head
      scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
      middle = __float2half_rn(__fadd_rn(lo, 8.f * __half2float(scale)));
      const float s = __half2float(scale), m = __half2float(middle);
      finite = finite && fabsf(s) <= 65504.f && fabsf(m) <= 65504.f;
      if (!finite) {  // what fp16 does not hold, and what is not a number, reads back as NaN
        scale = __float2half_rn(0.f);
        middle = __ushort_as_half(0x7FFF);
        word = 0x88888888u;
        status |= MS_ROW_NONFINITE;
      } else if (inside) {
        const float inverse = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float code = rintf(__fmul_rn(__fsub_rn(y[i], m), inverse)) + 8.f;
          word |= (uint32_t)__float2int_rn(fminf(fmaxf(code, 0.f), 15.f)) << (4 * i);
        }
      }
    }
    if (write) {
      int64_t page, offset;
      kv_place(slot, a.cache.page_size, p.page_shift, page, offset);
      const int64_t row = (page * a.cache.kv_heads + h) * a.cache.page_size + offset;
      uint8_t *codes = key ? a.cache.k_codes : a.cache.v_codes;
      void *params = key ? a.cache.k_params : a.cache.v_params;
      *reinterpret_cast<uint32_t *>(codes + row * p.layout.row_bytes + chunk * 4) = word;
      if ((chunk & 3) == 0)
        static_cast<__half2 *>(params)[row * p.layout.groups + (chunk >> 2)] = __halves2half2(scale, middle);
    }
    if (live && (chunk & 3) == 0 && status) atomicOr(&flags[tl], status);
  }
  __syncthreads();
  if (a.status)
    for (int i = threadIdx.x; i < tokens; i += kK4Threads) a.status[t0 + i] = flags[i];
}

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kK4Threads) ms_kv4_append_kernel(const __grid_constant__ K4AppendArgs p) {
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
  int chunks;  // 8-entry chunks of a head
  int tokens;  // tokens of a block
  int wide;    // outputs are stored in 16 bytes
};

template <typename T>
__device__ __forceinline__ uint32_t k4_narrow(float x, float y) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half)) {  // finite entries stay finite
    x = fabsf(x) <= 3.402823466e38f ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
    y = fabsf(y) <= 3.402823466e38f ? fminf(fmaxf(y, -65504.f), 65504.f) : y;
  }
  return kv_narrow<T>(x, y);
}

// A thread takes 8 entries of a key head and the same 8 of its value head.
template <typename T>
__global__ void __launch_bounds__(kK4Threads) ms_kv4_read_kernel(const __grid_constant__ K4ReadArgs p) {
  grid_wait();
  const ms_kv4_read_args &a = p.a;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int per_token = a.cache.kv_heads * p.chunks;
  const int items = (int)min((int64_t)p.tokens, a.tokens - t0) * per_token;
  for (int u = threadIdx.x; u < items; u += kK4Threads) {
    const int tl = u / per_token, w = u - tl * per_token;
    const int h = w / p.chunks, chunk = w - h * p.chunks;
    const int64_t t = t0 + tl, slot = load_in(a.slots + t);
    const bool bad = slot >= a.cache.pages * a.cache.page_size, live = slot >= 0 && !bad;
    if (w == 0 && a.status) a.status[t] = bad ? MS_ROW_BAD_SLOT : MS_ROW_OK;
    uint32_t word[2] = {0, 0};
    __half2 param[2];
    param[0] = param[1] = __halves2half2(__float2half_rn(0.f), __float2half_rn(0.f));
    if (live) {
      int64_t page, offset;
      kv_place(slot, a.cache.page_size, p.page_shift, page, offset);
      const int64_t row = (page * a.cache.kv_heads + h) * a.cache.page_size + offset;
      const int64_t code_at = row * p.layout.row_bytes + chunk * 4, param_at = row * p.layout.groups + (chunk >> 2);
      word[0] = load_in(reinterpret_cast<const uint32_t *>(a.cache.k_codes + code_at));
      word[1] = load_in(reinterpret_cast<const uint32_t *>(a.cache.v_codes + code_at));
      param[0] = load_in(static_cast<const __half2 *>(a.cache.k_params) + param_at);
      param[1] = load_in(static_cast<const __half2 *>(a.cache.v_params) + param_at);
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      T *dst = side ? static_cast<T *>(a.v_out) + t * a.v_token + h * a.v_head
                    : static_cast<T *>(a.k_out) + t * a.k_token + h * a.k_head;
      dst += chunk * 8;
      const float s = __low2float(param[side]), m = __high2float(param[side]);
      uint32_t out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = (float)((int)((word[side] >> (8 * i)) & 15) - 8), y = (float)((int)((word[side] >> (8 * i + 4)) & 15) - 8);
        out[i] = k4_narrow<T>(fmaf(s, x, m), fmaf(s, y, m));
      }
      if (p.wide) {
        *reinterpret_cast<uint4 *>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T *pair = reinterpret_cast<const T *>(&out[i]);
          dst[2 * i] = pair[0], dst[2 * i + 1] = pair[1];
        }
      }
    }
  }
}

// Tokens of a block: each thread a few items, so that a block's start and end
// are paid for, but no fewer blocks than fill the GPU.
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
  p.chunks = p.layout.row_bytes / 4;
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
  const int64_t kv_items = 2ll * a.cache.kv_heads * p.chunks;
  const int64_t q_items = (int64_t)a.heads * (a.cache.head_dim / (2 * p.q_piece));
  p.kv_tokens = ms::k4_tokens(a.tokens, kv_items, 4);
  p.q_tokens = q_items ? ms::k4_tokens(a.tokens, q_items, 4) : 1;
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
  p.chunks = a.cache.head_dim / 8;
  p.tokens = ms::k4_tokens(a.tokens, (int64_t)a.cache.kv_heads * p.chunks, 4);
  p.wide = ((a.k_token | a.k_head | a.v_token | a.v_head) & 7) == 0 &&
           ((reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) & 15) == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto *kernel = a.dtype == MS_DTYPE_BF16 ? ms::ms_kv4_read_kernel<__nv_bfloat16> : ms::ms_kv4_read_kernel<__half>;
  cudaError_t e = ms::launch_dependent(kernel, (unsigned)((a.tokens + p.tokens - 1) / p.tokens), ms::kK4Threads, 0, s, p);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
