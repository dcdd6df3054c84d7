// ms_kv_append -- new keys and values into a paged cache, the position
// rotation applied on the way (declared in include/mssample.h).
//
// Each rotated pair (a, b) of a head becomes (a c - b s, b c + a s) with the
// cosine c and sine s of the token's position, from an fp32 table; the other
// entries and the values are copied.  The arithmetic is fp32, rounded once to
// the cache's type.
//
// Bound by bytes: every element is read once and written once, and one
// table row of rotary fp32 pairs per token serves all its heads.  A thread
// owns 16 entries of a head (two 16-byte loads and stores: eight pairs, or 16
// copied entries), keeps its eight cosines and sines in registers and turns
// one to kKvHeads heads with them.  30011 tokens of 14 + 2 + 2 heads of 64
// (139 MB): 28.5 us, 4.9 TB/s, 75 % of the measured copy rate; issue slots are
// 60 % busy (address arithmetic and conversions) with four CTAs an SM.  512
// tokens of 32 + 8 + 8 heads of 128 (12.7 MB): 4.1 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mssample.h"
#include "ms_host.h"
#include "ms_tc.cuh"

namespace ms {

template <typename T>
__device__ __forceinline__ float2 kv_widen(uint32_t u);
template <>
__device__ __forceinline__ float2 kv_widen<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 kv_widen<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t kv_narrow(float x, float y);
template <>
__device__ __forceinline__ uint32_t kv_narrow<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t kv_narrow<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float kv_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float kv_to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void kv_from_float(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void kv_from_float(float x, __half &y) { y = __float2half_rn(x); }

struct KvArgs {
  ms_kv_append_args a;
  int page_shift;         // log2 of the page size, or -1
  int slots;              // head slots of one token
  int q_slots, kv_slots;  // of them, of the queries, and of the keys and the values each
  int per_token;          // threads of one token, where a token's threads are not a block's dimensions
  int tokens_cta;         // tokens of one CTA
};

// The token's cache row and status: bit set and no row for a bad slot or
// position, no row and MS_ROW_OK for a negative slot.
struct KvRow {
  int64_t page;
  int64_t offset;
  int64_t position;
  int32_t status;
  bool write;
};

__device__ __forceinline__ KvRow kv_row(const KvArgs &p, int64_t t) {
  const ms_kv_append_args &a = p.a;
  KvRow r{0, 0, 0, MS_ROW_OK, false};
  const int64_t slot = load_in(a.slots + t);
  if (slot >= a.pages * a.page_size) {
    r.status |= MS_ROW_BAD_SLOT;
  } else if (slot >= 0) {
    if (p.page_shift >= 0) {
      r.page = slot >> p.page_shift;
      r.offset = slot & (a.page_size - 1);
    } else if (slot < (1ll << 32)) {
      r.page = (uint32_t)slot / (uint32_t)a.page_size;
      r.offset = (uint32_t)slot - (uint32_t)r.page * (uint32_t)a.page_size;
    } else {
      r.page = slot / a.page_size;
      r.offset = slot - r.page * a.page_size;
    }
    r.write = true;
  }
  if (a.rotary > 0) {
    r.position = load_in(a.positions + t);
    if (r.position < 0 || r.position >= a.table_rows) {
      r.status |= MS_ROW_BAD_POSITION;
      r.position = 0;
    }
  }
  if (r.status != MS_ROW_OK) r.write = false;
  return r;
}

// Source of head h of token t.
template <typename T>
__device__ __forceinline__ const T *kv_source(const ms_kv_append_args &a, int64_t t, int h) {
  if (h < a.heads) return static_cast<const T *>(a.q) + t * a.q_token + h * a.q_head;
  h -= a.heads;
  if (h < a.kv_heads) return static_cast<const T *>(a.k) + t * a.k_token + h * a.k_head;
  return static_cast<const T *>(a.v) + t * a.v_token + (h - a.kv_heads) * a.v_head;
}
// Its destination (null where nothing is written).
template <typename T>
__device__ __forceinline__ T *kv_target(const ms_kv_append_args &a, const KvRow &r, int64_t t, int h) {
  if (h < a.heads) return static_cast<T *>(a.q_out) + t * a.q_out_token + h * a.q_out_head;
  if (!r.write) return nullptr;
  h -= a.heads;
  if (h < a.kv_heads) return static_cast<T *>(a.cache_k) + r.page * a.ck_page + r.offset * a.ck_token + h * a.ck_head;
  return static_cast<T *>(a.cache_v) + r.page * a.cv_page + r.offset * a.cv_token + (h - a.kv_heads) * a.cv_head;
}

constexpr int kKvThreads = 256;
// heads of a thread: 30011 tokens take 34.8 us with one, 29.0 with two, 31.5 with three (registers)
constexpr int kKvHeads = 2;

// kV entries (8: 16 bytes, 4: 8 bytes) at once: the halves that a thread owns.
template <int kV>
struct KvVec;
template <>
struct KvVec<8> {
  uint4 v;
};
template <>
struct KvVec<4> {
  uint2 v;
};

// Wide path: head_dim and rotary multiples of 2 kV, every stride a multiple of
// kV entries and every base aligned to them (checked on the host).  Threads
// are (chunk of 2 kV entries, head slot, token); a slot is up to kHeads heads
// of one of q, k and v, so that a thread finds its addresses once and steps
// along them.  Its loads are issued before anything that depends on the
// token's slot, position and table row.  8-byte pieces cost twice the threads,
// each with its slot, position and addresses: 20000 tokens of 14 + 2 + 2 heads
// of 80, 40 of them rotated (115 MB), take 30.7 us.
template <typename T, bool kInterleaved, int kHeads, int kV>
__global__ void __launch_bounds__(kKvThreads, 4) ms_kv_append_kernel(const __grid_constant__ KvArgs p) {
  grid_wait();
  const ms_kv_append_args &a = p.a;
  const int j = threadIdx.x;
  const int64_t t = (int64_t)blockIdx.x * blockDim.z + threadIdx.z;
  if (t >= a.tokens) return;
  const bool rotates = j * 2 * kV < a.rotary;
  // entries of the two halves a rotating thread owns
  const int lo = (!rotates || kInterleaved) ? j * 2 * kV : j * kV;
  const int hi = (!rotates || kInterleaved) ? lo + kV : lo + (a.rotary >> 1);
  for (int slot = threadIdx.y; slot < p.slots; slot += blockDim.y) {
    // the slot's heads: h, h + step, ... of q, k or v
    const bool query = slot < p.q_slots, key = !query && slot < p.q_slots + p.kv_slots;
    const int h = slot - (query ? 0 : key ? p.q_slots : p.q_slots + p.kv_slots);
    const int step = query ? p.q_slots : p.kv_slots, heads = query ? a.heads : a.kv_heads;
    const int64_t src_head = query ? a.q_head : key ? a.k_head : a.v_head;
    const T *src = static_cast<const T *>(query ? a.q : key ? a.k : a.v) +
                   t * (query ? a.q_token : key ? a.k_token : a.v_token) + h * src_head;
    KvVec<kV> x[kHeads], y[kHeads];
    {
      const T *from = src;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (h + i * step < heads) {
          x[i] = *reinterpret_cast<const KvVec<kV> *>(from + lo);
          y[i] = *reinterpret_cast<const KvVec<kV> *>(from + hi);
        }
        from += step * src_head;
      }
    }
    const KvRow r = kv_row(p, t);
    if (slot == 0 && j == 0 && a.status) a.status[t] = r.status;
    if (!query && !r.write) continue;
    float c[kV], s[kV];
    const bool turns = rotates && (query || key);
    if (turns) {
      const float *row = a.table + r.position * a.rotary + j * kV;
#pragma unroll
      for (int i = 0; i < kV; i += 4) {
        *reinterpret_cast<float4 *>(c + i) = load_in(reinterpret_cast<const float4 *>(row + i));
        *reinterpret_cast<float4 *>(s + i) = load_in(reinterpret_cast<const float4 *>(row + (a.rotary >> 1) + i));
      }
    }
    const int64_t dst_head = query ? a.q_out_head : key ? a.ck_head : a.cv_head;
    T *dst = static_cast<T *>(query ? a.q_out : key ? a.cache_k : a.cache_v) + h * dst_head;
    if (query) dst += t * a.q_out_token;
    else if (key) dst += r.page * a.ck_page + r.offset * a.ck_token;
    else dst += r.page * a.cv_page + r.offset * a.cv_token;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (h + i * step >= heads) break;
      uint32_t *xs = reinterpret_cast<uint32_t *>(&x[i]), *ys = reinterpret_cast<uint32_t *>(&y[i]);
      if (r.status & MS_ROW_BAD_POSITION) {
        x[i] = y[i] = KvVec<kV>{};
      } else if (turns) {
#pragma unroll
        for (int k = 0; k < kV / 2; ++k) {
          const float2 f = kv_widen<T>(xs[k]), g = kv_widen<T>(ys[k]);
          if (kInterleaved) {  // word k of x is pair k, word k of y is pair kV / 2 + k
            xs[k] = kv_narrow<T>(f.x * c[k] - f.y * s[k], f.y * c[k] + f.x * s[k]);
            ys[k] = kv_narrow<T>(g.x * c[kV / 2 + k] - g.y * s[kV / 2 + k], g.y * c[kV / 2 + k] + g.x * s[kV / 2 + k]);
          } else {  // word k holds the first (x) and second (y) entries of pairs 2k and 2k + 1
            const float c0 = c[2 * k], c1 = c[2 * k + 1], s0 = s[2 * k], s1 = s[2 * k + 1];
            xs[k] = kv_narrow<T>(f.x * c0 - g.x * s0, f.y * c1 - g.y * s1);
            ys[k] = kv_narrow<T>(g.x * c0 + f.x * s0, g.y * c1 + f.y * s1);
          }
        }
      }
      *reinterpret_cast<KvVec<kV> *>(dst + lo) = x[i];
      *reinterpret_cast<KvVec<kV> *>(dst + hi) = y[i];
      dst += step * dst_head;
    }
  }
}

// Any head_dim, rotary and stride: a thread owns one pair, or two copied
// entries, of a head.  Bound by instructions, a load and a store for every two
// bytes: 30000 tokens of 13 + 3 + 3 heads of 35 (80 MB) take 79 us.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kKvThreads) ms_kv_append_any_kernel(const __grid_constant__ KvArgs p) {
  grid_wait();
  const ms_kv_append_args &a = p.a;
  const int half = a.rotary >> 1;
  const int units = half + (a.head_dim - a.rotary + 1) / 2;
  const int heads = a.heads + 2 * a.kv_heads;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_cta;
  for (int u = threadIdx.x; u < p.tokens_cta * p.per_token; u += kKvThreads) {
    const int tl = u / p.per_token, w = u - tl * p.per_token;
    const int64_t t = t0 + tl;
    if (t >= a.tokens) return;
    const int slot = w / units, j = w - slot * units;
    const KvRow r = kv_row(p, t);
    if (w == 0 && a.status) a.status[t] = r.status;
    const bool rotates = j < half;
    int lo, hi;
    float c = 1.f, s = 0.f;
    if (rotates) {
      lo = kInterleaved ? 2 * j : j;
      hi = kInterleaved ? 2 * j + 1 : j + half;
      c = load_in(a.table + r.position * a.rotary + j);
      s = load_in(a.table + r.position * a.rotary + half + j);
    } else {
      lo = a.rotary + 2 * (j - half);
      hi = lo + 1;
    }
    for (int h = slot; h < heads; h += p.slots) {
      const T *src = kv_source<T>(a, t, h);
      T *dst = kv_target<T>(a, r, t, h);
      if (!dst) continue;
      if (r.status & MS_ROW_BAD_POSITION) {
        kv_from_float(0.f, dst[lo]);
        if (hi < a.head_dim) kv_from_float(0.f, dst[hi]);
      } else if (rotates && h < a.heads + a.kv_heads) {
        const float x = kv_to_float(src[lo]), y = kv_to_float(src[hi]);
        kv_from_float(x * c - y * s, dst[lo]);
        kv_from_float(y * c + x * s, dst[hi]);
      } else {
        const T x = src[lo];
        if (hi < a.head_dim) {
          const T y = src[hi];
          dst[hi] = y;
        }
        dst[lo] = x;
      }
    }
  }
}

template <typename T, int kV>
cudaError_t launch_kv_wide(KvArgs &p, int each, cudaStream_t s) {
  const ms_kv_append_args &a = p.a;
  const int units = a.head_dim / (2 * kV);
  p.q_slots = (a.heads + each - 1) / each;
  p.kv_slots = (a.kv_heads + each - 1) / each;
  p.slots = p.q_slots + 2 * p.kv_slots;
  const int y = p.slots < kKvThreads / units ? p.slots : kKvThreads / units;
  const int z = kKvThreads / (units * y) < 64 ? kKvThreads / (units * y) : 64;
  auto *kernel = a.interleaved ? ms_kv_append_kernel<T, true, 1, kV> : ms_kv_append_kernel<T, false, 1, kV>;
  if (each > 1)
    kernel = a.interleaved ? ms_kv_append_kernel<T, true, kKvHeads, kV> : ms_kv_append_kernel<T, false, kKvHeads, kV>;
  return launch_dependent(kernel, (unsigned)((a.tokens + z - 1) / z), dim3(units, y, z), 0, s, p);
}

// `wide`: entries that can be moved at once (8, 4 or 1).
template <typename T>
cudaError_t launch_kv_append(KvArgs &p, int wide, cudaStream_t s) {
  const ms_kv_append_args &a = p.a;
  const int heads = a.heads + 2 * a.kv_heads;
  // one head a thread until the call fills the GPU's threads a few times
  // over; then up to kKvHeads, which share the thread's table row
  const int each = a.tokens * heads * a.head_dim > 16 * 4ll * 148 * 2048 ? kKvHeads : 1;
  if (wide == 8) return launch_kv_wide<T, 8>(p, each, s);
  if (wide == 4) return launch_kv_wide<T, 4>(p, each, s);
  const int units = a.rotary / 2 + (a.head_dim - a.rotary + 1) / 2;
  p.slots = (heads + each - 1) / each;
  p.per_token = units * p.slots;
  p.tokens_cta = p.per_token < kKvThreads ? kKvThreads / p.per_token : 1;
  const unsigned grid = (unsigned)((a.tokens + p.tokens_cta - 1) / p.tokens_cta);
  auto *kernel = a.interleaved ? ms_kv_append_any_kernel<T, true> : ms_kv_append_any_kernel<T, false>;
  return launch_dependent(kernel, grid, kKvThreads, 0, s, p);
}

}  // namespace ms

extern "C" int ms_kv_append(const ms_kv_append_args *args, ms_stream_t stream) {
  if (!args) return MS_E_INVALID;
  ms::KvArgs p{};
  p.a = *args;
  const ms_kv_append_args &a = p.a;
  if (a.dtype != MS_DTYPE_BF16 && a.dtype != MS_DTYPE_F16) return MS_E_DTYPE;
  if (a.tokens < 0 || a.tokens > 0x7FFFFFFFll || a.heads < 0 || a.heads > 65536 || a.kv_heads < 1 ||
      a.kv_heads > 65536 || a.head_dim < 1 || a.head_dim > 4096 || a.rotary < 0 || a.rotary > a.head_dim ||
      (a.rotary & 1) || a.pages < 1 || a.page_size < 1 || a.page_size > 0x7FFFFFFFll ||
      a.pages > (int64_t)(0x7FFFFFFFFFFFFFFFull / (uint64_t)a.page_size))
    return MS_E_INVALID;
  if (a.tokens == 0) return MS_OK;
  if (!a.k || !a.v || !a.slots || !a.cache_k || !a.cache_v) return MS_E_INVALID;
  if (a.heads > 0 && (!a.q || !a.q_out)) return MS_E_INVALID;
  if (a.rotary > 0 && (!a.positions || !a.table || a.table_rows < 1)) return MS_E_INVALID;
  // the widest pieces that sizes, strides and bases allow (the table is read in 16 bytes either way)
  uint64_t bases = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                   reinterpret_cast<uintptr_t>(a.cache_k) | reinterpret_cast<uintptr_t>(a.cache_v);
  if (a.heads > 0) bases |= reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out);
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a.page_size == 1ll << i) p.page_shift = i;
  int64_t strides = a.k_token | a.k_head | a.v_token | a.v_head | a.ck_page | a.ck_token | a.ck_head | a.cv_page |
                    a.cv_token | a.cv_head;
  if (a.heads > 0) strides |= a.q_token | a.q_head | a.q_out_token | a.q_out_head;
  const bool table = a.rotary == 0 || (reinterpret_cast<uintptr_t>(a.table) & 15) == 0;
  auto fits = [&](int v) {
    return a.head_dim % (2 * v) == 0 && a.head_dim / (2 * v) <= ms::kKvThreads && a.rotary % (2 * v) == 0 && table &&
           (strides & (v - 1)) == 0 && (bases & (2 * v - 1)) == 0;
  };
  const int wide = fits(8) ? 8 : fits(4) ? 4 : 1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = a.dtype == MS_DTYPE_BF16 ? ms::launch_kv_append<__nv_bfloat16>(p, wide, s)
                                           : ms::launch_kv_append<__half>(p, wide, s);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}
