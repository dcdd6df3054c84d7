// 8-bit integer product with a scale for each token and each output channel
// (declared in include/mssample.h): ms_quantize_rows, ms_int8_matmul and the
// two in one call, ms_int8_linear.
//
//   s_t = max_k |x[t, k]| / 127,  q[t, k] = rint(x[t, k] / s_t)
//   out[t, n] = s_t w_n sum_k q[t, k] wq[n, k] + bias_n
//
// The sum is exact in int32: with |q| <= 127 and K <= 131072 its magnitude is
// at most 127 * 128 K < 2^31.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/mssample.h"
#include "ms_host.h"
#include "ms_int8_tiling.h"
#include "ms_tc.cuh"

namespace ms {

// ------------------------------------------------------------ quantisation
constexpr int kQuThreads = 256;

template <typename T>
__device__ __forceinline__ void qu_load8(const T *p, float (&v)[8]);
template <>
__device__ __forceinline__ void qu_load8<float>(const float *p, float (&v)[8]) {
  *reinterpret_cast<float4 *>(v) = load_in(reinterpret_cast<const float4 *>(p));
  *reinterpret_cast<float4 *>(v + 4) = load_in(reinterpret_cast<const float4 *>(p) + 1);
}
template <>
__device__ __forceinline__ void qu_load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&v)[8]) {
  const uint4 u = load_in(reinterpret_cast<const uint4 *>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void qu_load8<__half>(const __half *p, float (&v)[8]) {
  const uint4 u = load_in(reinterpret_cast<const uint4 *>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float qu_float(float x) { return x; }
__device__ __forceinline__ float qu_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float qu_float(__half x) { return __half2float(x); }

__device__ __forceinline__ int qu_round(float x, float scale) {
  return max(-127, min(127, __float2int_rn(__fdiv_rn(x, scale))));
}

// One CTA per token, the row in registers between its two uses: groups of
// eight entries where rows are 16-byte aligned (`wide`), else single ones.
// What exceeds kQuKeep groups or entries a thread is read again.
constexpr int kQuKeep = 4;

template <typename T, bool kWide>
__global__ void __launch_bounds__(kQuThreads) ms_quantize_kernel(const T *x, int64_t ldx, int K, int8_t *q, int64_t ldq,
                                                               float *scale) {
  grid_wait();     // the call's first kernel: what it reads, and the weights, are in memory
  grid_release();  // before the product may load weights
  __shared__ uint32_t red[kQuThreads / 32];
  constexpr int kEach = kWide ? 8 : 1;  // entries of a unit
  constexpr int kKeep = kWide ? kQuKeep : 4 * kQuKeep;
  const T *row = x + (int64_t)blockIdx.x * ldx;
  int8_t *out = q + (int64_t)blockIdx.x * ldq;
  const int tid = threadIdx.x;
  const int units = K / kEach;
  auto read = [&](int i, float (&v)[kEach]) {
    if constexpr (kWide) qu_load8<T>(row + (int64_t)i * 8, v);
    else v[0] = qu_float(row[i]);
  };
  uint32_t top = 0;  // the largest magnitude's bits: NaN above infinity above finite
  auto raise = [&](const float (&v)[kEach]) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  };
  float keep[kKeep][kEach];
#pragma unroll
  for (int u = 0; u < kKeep; ++u) {
    const int i = tid + u * kQuThreads;
    if (i < units) read(i, keep[u]);
  }
#pragma unroll
  for (int u = 0; u < kKeep; ++u)
    if (tid + u * kQuThreads < units) raise(keep[u]);
  for (int i = tid + kKeep * kQuThreads; i < units; i += kQuThreads) {
    float v[kEach];
    read(i, v);
    raise(v);
  }
  const int rest = units * kEach + tid;  // at most seven entries past the groups
  if (rest < K) top = max(top, __float_as_uint(qu_float(row[rest])) & 0x7FFFFFFFu);
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuThreads / 32; ++i) top = max(top, red[i]);
  const bool finite = top < 0x7F800000u;
  const float s = finite ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7FC00000u);
  const bool live = s > 0.f;  // false for an all-zero row and for a NaN scale: its integers are zero
  if (tid == 0) scale[blockIdx.x] = s;
  auto write = [&](int i, const float (&v)[kEach]) {
    if constexpr (kWide) {
      uint32_t w[2] = {0, 0};
      if (live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)(uint8_t)qu_round(v[j], s) << (8 * (j & 3));
      }
      *reinterpret_cast<uint2 *>(out + (int64_t)i * 8) = make_uint2(w[0], w[1]);
    } else {
      out[i] = live ? (int8_t)qu_round(v[0], s) : (int8_t)0;
    }
  };
#pragma unroll
  for (int u = 0; u < kKeep; ++u)
    if (tid + u * kQuThreads < units) write(tid + u * kQuThreads, keep[u]);
  for (int i = tid + kKeep * kQuThreads; i < units; i += kQuThreads) {
    float v[kEach];
    read(i, v);
    write(i, v);
  }
  if (rest < K) out[rest] = live ? (int8_t)qu_round(qu_float(row[rest]), s) : (int8_t)0;
}

template <typename T>
static cudaError_t run_quantize(const void *x, int64_t M, int64_t K, int64_t ldx, int8_t *q, int64_t ldq, float *scale,
                         bool wide, cudaStream_t s) {
  auto *kernel = wide ? ms_quantize_kernel<T, true> : ms_quantize_kernel<T, false>;
  return launch_dependent(kernel, (unsigned)M, kQuThreads, 0, s, static_cast<const T *>(x), ldx, (int)K, q, ldq, scale);
}

static cudaError_t launch_quantize(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, int8_t *q, int64_t ldq,
                                   float *scale, cudaStream_t s) {
  const int esz = dtype == MS_DTYPE_F32 ? 4 : 2;
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * esz) % 16 == 0 &&
                    (reinterpret_cast<uintptr_t>(q) & 7) == 0 && ldq % 8 == 0;
  if (dtype == MS_DTYPE_F32) return run_quantize<float>(x, M, K, ldx, q, ldq, scale, wide, s);
  if (dtype == MS_DTYPE_BF16) return run_quantize<__nv_bfloat16>(x, M, K, ldx, q, ldq, scale, wide, s);
  return run_quantize<__half>(x, M, K, ldx, q, ldq, scale, wide, s);
}

// ----------------------------------------------------------------- product
// D[channel, token] = W[128 channels, K] X[tokens, K]^T on tcgen05 (kind::i8),
// the channels on the 128 lanes of tensor memory and the tokens on its
// columns: a small batch is a narrow N and the weights stream through once,
// and in the epilogue a warp's 32 lanes are 32 consecutive channels of one
// token, so its stores are whole lines.
//
// A persistent CTA per SM walks over (channel tile, token tile) pairs, token
// tiles fastest, so that the weights of a channel tile come from HBM once.
// Warps 0 and 10 load K steps of 128 bytes of the channels and of the tokens
// with TMA (128-byte swizzle, zero beyond K, channels or tokens), warp 1
// issues the products into one of two accumulators of 256 columns, warps 2-9
// scale and store the other one.
//
// Large batches are bound by what an SM can read (64 bytes a clock): a tile of
// 128 channels x 256 tokens reads 96 bytes a clock at the products' full rate.
// There two SMs take a tile of 256 channels together (kPair: a cluster of two,
// products of cta_group::2): each loads its 128 channels and half of the
// tokens, 64 bytes a clock, the first CTA issues the products for both, and
// each stores its own channels.
//
// With their quantisation, a few dozen calls on end: 1 x 896 x 151936 to fp32
// 27.8 us (137 MB of weights, 4.9 TB/s; 25.5 us in a graph); 512 x 896 x 151936
// 87.7 us (449 MB, 5.1 TB/s, 79 % of the measured copy rate); 2048 x 4096 x 8192
// to bf16 56.7 us (2.4 POP/s, tensor pipe 79 % busy; 256 tiles over 74 pairs
// leave 13 % of the rounds idle).  Calls that last a second or more meet the
// GPU's power limit: the last two then take 102 us (1305 MHz) and 65 us (1590
// MHz), in a graph as well.
constexpr int kI8Epilogue = 8;  // warps: two for each 32 lanes of tensor memory, on alternate 16 columns
constexpr int kI8Threads = 64 + 32 * kI8Epilogue + 32;

struct I8Shared {
  uint64_t full[kI8MaxStages], empty[kI8MaxStages];
  uint64_t acc_full[2], acc_empty[2], drained;
  uint32_t tmem;
  volatile int dead;  // a wait ran out: the rest of the outputs are NaN
  alignas(16) float xs[2][kI8Cols];
};

struct I8Args {
  const float *x_scale, *w_scale, *bias;
  void *out;
  int64_t ldo;
  int M, N, K;
  int bn;      // tokens of a tile: a multiple of 16, at most 256
  int rows;    // channels of a tile, at most kI8Rows
  int stages;
  int after_quantize;  // launched with the quantisation as its programmatic dependency
};

__device__ __forceinline__ void i8_store(float *p, float y) { *p = y; }
__device__ __forceinline__ void i8_store(__nv_bfloat16 *p, float y) { *p = __float2bfloat16_rn(y); }
__device__ __forceinline__ void i8_store(__half *p, float y) { *p = __float2half_rn(y); }

// 16 columns (tokens) of a lane's channel, scaled and stored ldo apart.
template <typename T, bool kAll>
__device__ __forceinline__ void i8_columns(const uint32_t (&r)[16], const float *xs, float ws, float bias, T *out,
                                           int64_t ldo, int count) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 s = *reinterpret_cast<const float4 *>(xs + i);
    const float e[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kAll || i + j < count) i8_store(out, fmaf((float)(int)r[i + j], e[j] * ws, bias));
      out += ldo;
    }
  }
}

template <typename T, bool kPair>
__global__ void __launch_bounds__(kI8Threads, 1)
    ms_int8_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                   const __grid_constant__ I8Args a) {
  extern __shared__ __align__(1024) unsigned char i8_raw[];
  __shared__ I8Shared sh;
  unsigned char *ring = i8_raw + ((1024u - (smem_addr(i8_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this CTA's or pair's tiles, and this CTA's channels and tokens of one
  constexpr int kCtas = kPair ? 2 : 1;
  const uint32_t rank = kPair ? cluster_rank() : 0;
  const int64_t worker = blockIdx.x / kCtas, workers = gridDim.x / kCtas;
  const int tok_tiles = (a.M + a.bn - 1) / a.bn;
  const int span = a.rows * kCtas;
  const int64_t tiles = (int64_t)((a.N + span - 1) / span) * tok_tiles;
  const int steps = (a.K + kI8Step - 1) / kI8Step;
  constexpr uint32_t wbytes = kI8Rows * kI8Step;
  const uint32_t xbytes = (uint32_t)(a.bn / kCtas) * kI8Step, both = (uint32_t)a.rows * kI8Step + xbytes;
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      bar_init(&sh.full[i], 1);
      bar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh.acc_full[i], 1);
      bar_init(&sh.acc_empty[i], kI8Epilogue * kCtas);
    }
    bar_init(&sh.drained, 1);
    sh.dead = 0;
    bar_init_fence();
  }
  if (warp == 1) {
    if (kPair) tmem_alloc_pair(&sh.tmem, 2 * kI8Cols);
    else tmem_alloc(&sh.tmem, 2 * kI8Cols);
  }
  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync();  // the other CTA's barriers are ready
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == 0 || warp == kI8Threads / 32 - 1) {
    // weights (announced with the tokens' bytes; they need not wait for the quantisation), and tokens
    const bool tokens = warp != 0;
    const uint32_t leader = tc_leader();
    const uint32_t dst0 = smem_addr(ring) + (tokens ? wbytes : 0), bytes = wbytes + xbytes;
    const uint32_t full0 = kPair ? leader_addr(&sh.full[0]) : smem_addr(&sh.full[0]);
    const CUtensorMap *map = tokens ? &xmap : &wmap;
    if (tokens && a.after_quantize) grid_wait();
    int stage = 0, phase = 1, issued = 0;
    bool ok = true;
    for (int64_t tile = worker; tile < tiles && ok; tile += workers) {
      const int row = tokens ? (int)(tile % tok_tiles) * a.bn + (int)rank * (a.bn / kCtas)
                             : (int)(tile / tok_tiles) * span + (int)rank * a.rows;
      for (int k = 0; k < steps; ++k) {
        ok = bar_wait_warp(&sh.empty[stage], phase, sh.dead);
        if (!ok) break;
        // the first CTA's barrier counts both CTAs' bytes
        if (!tokens && rank == 0) bar_expect(leader, &sh.full[stage], both * kCtas);
        if (kPair) tma_load_2d_pair(leader, dst0 + stage * bytes, map, full0 + stage * 8, k * kI8Step, row);
        else tma_load_2d(leader, dst0 + stage * bytes, map, full0 + stage * 8, k * kI8Step, row);
        issued = min(issued + 1, a.stages);
        if (++stage == a.stages) stage = 0, phase ^= 1;
      }
    }
    if (!ok) {  // copies in flight: their last phase of each stage, again bounded
      sh.dead = 1;
      for (int i = 0; i < a.stages && rank == 0; ++i)
        if (i < stage || issued == a.stages) bar_wait(&sh.full[i], i < stage ? phase ^ 1 : phase);
    }
  } else if (warp == 1) {
    const uint32_t leader = tc_leader();
    const uint32_t idesc = tc_idesc_i8(kI8Rows * kCtas, a.bn);
    int stage = 0, phase = 0, n = 0;
    bool ok = true;
    auto commit = [&](uint64_t *bar) {
      if (kPair) tc_commit_pair(leader, bar);
      else tc_commit(leader, bar);
    };
    for (int64_t tile = worker; tile < tiles && ok && rank == 0; tile += workers, ++n) {
      const int acc = n & 1;
      ok = bar_wait_warp(&sh.acc_empty[acc], ((n >> 1) & 1) ^ 1, sh.dead);
      tc_fence_after();
      for (int k = 0; k < steps && ok; ++k) {
        ok = bar_wait_warp(&sh.full[stage], phase, sh.dead);
        if (!ok) break;
        tc_fence_after();
        const uint32_t st = smem_addr(ring + stage * (wbytes + xbytes));
        const uint64_t wd = tc_desc(st, 1024, 16), xd = tc_desc(st + wbytes, 1024, 16);
#pragma unroll
        for (int j = 0; j < kI8Step / 32; ++j) {
          if (kPair) tc_mma_i8_pair(leader, tmem + acc * kI8Cols, wd + 2 * j, xd + 2 * j, idesc, k > 0 || j > 0);
          else tc_mma_i8(leader, tmem + acc * kI8Cols, wd + 2 * j, xd + 2 * j, idesc, k > 0 || j > 0);
        }
        commit(&sh.empty[stage]);
        if (++stage == a.stages) stage = 0, phase ^= 1;
      }
      if (ok) commit(&sh.acc_full[acc]);
    }
    if (!ok) sh.dead = 1;
    if (rank == 0) commit(&sh.drained);
    bar_wait(&sh.drained, 0);  // products in flight end before tensor memory is freed
  } else {
    const int quad = warp & 3;
    const int et = threadIdx.x - 64;
    if (a.after_quantize) grid_wait();
    // a tile's scales are loaded under the tile before: a token's by each thread, this lane's channel's
    static_assert(32 * kI8Epilogue == kI8Cols, "a thread for each token of a tile");
    float xs = 0.f, ws = 0.f, bias = 0.f;
    auto scales = [&](int64_t tile) {
      if (tile >= tiles) return;
      const int ch = (int)(tile / tok_tiles) * span + (int)rank * a.rows + quad * 32 + lane;
      const int t = (int)(tile % tok_tiles) * a.bn + et;
      if (et < a.bn && t < a.M) xs = load_in(a.x_scale + t);
      const bool live = quad * 32 + lane < a.rows && ch < a.N;
      ws = live ? load_in(a.w_scale + ch) : 0.f;
      bias = live && a.bias ? load_in(a.bias + ch) : 0.f;
    };
    scales(worker);
    int n = 0;
    for (int64_t tile = worker; tile < tiles; tile += workers, ++n) {
      const int acc = n & 1;
      const int n0 = (int)(tile / tok_tiles) * span + (int)rank * a.rows, t0 = (int)(tile % tok_tiles) * a.bn;
      const int count = min(a.bn, a.M - t0);
      const int ch = quad * 32 + lane < a.rows ? n0 + quad * 32 + lane : a.N;  // a.N: not a channel of this tile
      const float scale = ws, add = bias;
      sh.xs[acc][et] = xs;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kI8Epilogue) : "memory");
      scales(tile + workers);
      if (!sh.dead && !bar_wait(&sh.acc_full[acc], (n >> 1) & 1)) sh.dead = 1;
      __syncwarp();
      tc_fence_after();
      const float factor = sh.dead ? __uint_as_float(0x7FC00000u) : scale;
      const int first = (warp - 2) / 4 * 16;
      T *out = static_cast<T *>(a.out) + (int64_t)(t0 + first) * a.ldo + ch;
      const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + acc * kI8Cols;
      constexpr int kNext = kI8Epilogue * 4;  // columns to this warp's next 16
      uint32_t r[2][16];  // the next 16 columns are read under the stores of these
      if (first < count) tmem_ld16(from + first, r[0]);
#pragma unroll 1
      for (int c = first; c < count; c += 2 * kNext) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = c + kNext * k;
          if (at >= count) break;
          tmem_wait_ld(r[k]);
          if (at + kNext < count) tmem_ld16(from + at + kNext, r[k ^ 1]);
          if (ch < a.N) {
            if (at + 16 <= count)
              i8_columns<T, true>(r[k], sh.xs[acc] + at, factor, add, out, a.ldo, 16);
            else
              i8_columns<T, false>(r[k], sh.xs[acc] + at, factor, add, out, a.ldo, count - at);
          }
          __syncwarp();
          out += kNext * a.ldo;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kPair) bar_arrive_leader(&sh.acc_empty[acc]);
        else bar_arrive(&sh.acc_empty[acc]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync();  // neither CTA's memory or barriers are used by the other any more
  tc_fence_after();
  if (warp == 1) {
    if (kPair) tmem_free_pair(tmem, 2 * kI8Cols);
    else tmem_free(tmem, 2 * kI8Cols);
  }
}

// A [rows, K] int8 matrix read in tiles of `box` rows and 128 bytes.
static cudaError_t i8_map(CUtensorMap *map, const void *p, int64_t rows, int64_t K, int64_t ld, int box) {
  EncodeTiled fn;
  cudaError_t e = encode_tiled(&fn);
  if (e != cudaSuccess) return e;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t boxes[2] = {(cuuint32_t)kI8Step, (cuuint32_t)box};
  const cuuint32_t unit[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(p), dims, strides, boxes, unit,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, bool kPair>
static cudaError_t launch_int8_as(I8Args &a, const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, int sms,
                                  int dev, cudaStream_t s) {
  static std::atomic<int> ready[kMaxDevices];
  constexpr int kCtas = kPair ? 2 : 1;
  cudaError_t e = cudaSuccess;
  if (!ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(ms_int8_kernel<T, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, kI8Ring + 1024);
    if (e != cudaSuccess) return e;
    ready[dev].store(1, std::memory_order_release);
  }
  const int64_t tok_tiles = (a.M + (int64_t)a.bn - 1) / a.bn;
  const int stage = i8_stage_bytes(a.bn, kPair);
  a.stages = i8_stages(a.M, a.K, a.bn, kPair);
  const int64_t span = (int64_t)a.rows * kCtas;
  const int64_t tiles = (a.N + span - 1) / span * tok_tiles;
  CUtensorMap wmap, xmap;
  e = i8_map(&wmap, wq, a.N, a.K, ldw, a.rows);
  if (e == cudaSuccess) e = i8_map(&xmap, xq, a.M, a.K, ldx, a.bn / kCtas);
  if (e != cudaSuccess) return e;
  const int64_t workers = tiles < sms / kCtas ? tiles : sms / kCtas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(workers * kCtas));
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = a.stages * stage + 1024;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (kPair) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 2;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (a.after_quantize) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  e = cudaLaunchKernelEx(&cfg, ms_int8_kernel<T, kPair>, wmap, xmap, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
static cudaError_t launch_int8_out(I8Args &a, const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, int dev,
                                   cudaStream_t s) {
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const I8Tiling t = i8_tiling(a.M, a.N, a.K, sizeof(T), sms);
  a.bn = t.bn, a.rows = t.rows;
  return t.pair ? launch_int8_as<T, true>(a, xq, ldx, wq, ldw, sms, dev, s)
                : launch_int8_as<T, false>(a, xq, ldx, wq, ldw, sms, dev, s);
}

static cudaError_t launch_int8(const int8_t *xq, int64_t ldx, const float *x_scale, int64_t M, const int8_t *wq,
                               int64_t ldw, const float *w_scale, int64_t N, int64_t K, const float *bias, void *out,
                               int out_dtype, int64_t ldo, bool after_quantize, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  I8Args a{};
  a.x_scale = x_scale, a.w_scale = w_scale, a.bias = bias, a.out = out, a.ldo = ldo;
  a.M = (int)M, a.N = (int)N, a.K = (int)K, a.after_quantize = after_quantize;
  if (out_dtype == MS_DTYPE_F32) return launch_int8_out<float>(a, xq, ldx, wq, ldw, dev, s);
  if (out_dtype == MS_DTYPE_BF16) return launch_int8_out<__nv_bfloat16>(a, xq, ldx, wq, ldw, dev, s);
  return launch_int8_out<__half>(a, xq, ldx, wq, ldw, dev, s);
}

static bool i8_dtype(int d) { return d == MS_DTYPE_F32 || d == MS_DTYPE_BF16 || d == MS_DTYPE_F16; }
static bool i8_rows(const void *p, int64_t ld, int64_t K) {  // what a tile load needs
  return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld >= K && ld % 16 == 0 && ld < (1ll << 40);
}
constexpr int64_t kI8MaxK = 131072;
constexpr int64_t kI8MaxRows = 0x7FFFFFFFll - 256;

}  // namespace ms

extern "C" {

int ms_quantize_rows(const void *x, int dtype, int64_t M, int64_t K, int64_t ldx, int8_t *q, int64_t ldq, float *scale,
                     ms_stream_t stream) {
  if (!ms::i8_dtype(dtype)) return MS_E_DTYPE;
  if (M < 0 || M > ms::kI8MaxRows || K < 1 || ldx < K || ldq < K) return MS_E_INVALID;
  if (K > ms::kI8MaxK) return MS_E_UNSUPPORTED;
  if (M == 0) return MS_OK;
  if (!x || !q || !scale) return MS_E_INVALID;
  cudaError_t e = ms::launch_quantize(x, dtype, M, K, ldx, q, ldq, scale, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

static int int8_check(int64_t M, int64_t K, const int8_t *wq, int64_t ldw, const float *w_scale, int64_t N, void *out,
                      int out_dtype, int64_t ldo) {
  if (!ms::i8_dtype(out_dtype)) return MS_E_DTYPE;
  if (M < 0 || M > ms::kI8MaxRows || N < 1 || N > ms::kI8MaxRows || K < 1 || ldo < N) return MS_E_INVALID;
  if (K > ms::kI8MaxK) return MS_E_UNSUPPORTED;
  if (M == 0) return MS_OK;
  if (!ms::i8_rows(wq, ldw, K) || !w_scale || !out) return MS_E_INVALID;
  return MS_OK;
}

int ms_int8_matmul(const int8_t *xq, int64_t ldx, const float *x_scale, int64_t M, const int8_t *wq, int64_t ldw,
                   const float *w_scale, int64_t N, int64_t K, const float *bias, void *out, int out_dtype,
                   int64_t ldo, ms_stream_t stream) {
  const int rc = int8_check(M, K, wq, ldw, w_scale, N, out, out_dtype, ldo);
  if (rc != MS_OK || M == 0) return rc;
  if (!ms::i8_rows(xq, ldx, K) || !x_scale) return MS_E_INVALID;
  cudaError_t e = ms::launch_int8(xq, ldx, x_scale, M, wq, ldw, w_scale, N, K, bias, out, out_dtype, ldo, false,
                                  reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

int64_t ms_int8_workspace(int64_t M, int64_t K) {
  if (M < 0 || K < 1 || M > ms::kI8MaxRows || K > ms::kI8MaxK) return 0;
  return (M * 4 + 15) / 16 * 16 + M * ((K + 15) / 16 * 16);
}

int ms_int8_linear(const void *x, int dtype, int64_t ldx, int64_t M, const int8_t *wq, int64_t ldw,
                   const float *w_scale, int64_t N, int64_t K, const float *bias, void *out, int out_dtype,
                   int64_t ldo, void *workspace, ms_stream_t stream) {
  if (!ms::i8_dtype(dtype)) return MS_E_DTYPE;
  const int rc = int8_check(M, K, wq, ldw, w_scale, N, out, out_dtype, ldo);
  if (rc != MS_OK || M == 0) return rc;
  if (!x || ldx < K || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)) return MS_E_INVALID;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  float *scale = static_cast<float *>(workspace);
  const int64_t ldq = (K + 15) / 16 * 16;
  int8_t *q = static_cast<int8_t *>(workspace) + (M * 4 + 15) / 16 * 16;
  cudaError_t e = ms::launch_quantize(x, dtype, M, K, ldx, q, ldq, scale, s);
  if (e == cudaSuccess)
    e = ms::launch_int8(q, ldq, scale, M, wq, ldw, w_scale, N, K, bias, out, out_dtype, ldo, true, s);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
