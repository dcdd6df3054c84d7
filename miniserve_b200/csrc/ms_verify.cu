// ms_verify_drafts -- drafted tokens against a target model's logits, from
// given uniforms (declared in include/mssample.h).
//
// With p_i = softmax(logits_i / T) and the draft's probabilities q_i, draft d_i
// is accepted when u_i q_i(d_i) < p_i(d_i).  At the first one refused the token
// is drawn from max(p_i - q_i, 0), and where all are accepted one more from p:
// the tokens are distributed as if each had been drawn from p_i.  Draws run in
// index order: the first token whose running mass passes u times the whole.
//
// Two kernels: the statistics of every position's logits (largest value, sum of
// weights; read once, bound by bytes), then one cluster of CTAs a row that
// decides and draws from one position.  Decisions compare numbers that are
// 1e-7 off at worst in 2^-24 of all cases; a draw compares with a running mass
// at every one of the vocabulary's borders, so that its weights and sums are in
// 64 bits: with 32 about one draw in a thousand would land beside its token.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/mssample.h"
#include "ms_host.h"
#include "ms_tc.cuh"

namespace ms {

constexpr int kVfThreads = 256;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfCluster = 8;     // CTAs of a row's draw
constexpr int kVfMaxDrafts = 255;
constexpr int64_t kVfMaxVocab = 0x7FFFFFFFll - 4096;

// Of a slice of one position's logits.
struct VfRecord {
  double sum;   // of exp2((x - top) c)
  float top;    // largest value
  int index;    // its first place
  int flags;    // MS_ROW_NONFINITE
};

struct VfArgs {
  ms_verify_args x;
  VfRecord *records;  // [rows][drafts + 1][slices]
  int slices;
  int64_t slice;      // entries of a slice
};

template <int DT>
struct VfType;
template <>
struct VfType<MS_DTYPE_F32> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ void wide(const uint4 &u, float *x) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float one(const T *p) { return load_in(p); }
};
template <>
struct VfType<MS_DTYPE_BF16> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ void wide(const uint4 &u, float *x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  static __device__ __forceinline__ float one(const T *p) { return __bfloat162float(load_in(p)); }
};
template <>
struct VfType<MS_DTYPE_F16> {
  using T = __half;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ void wide(const uint4 &u, float *x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float one(const T *p) { return __half2float(load_in(p)); }
};

__device__ __forceinline__ float vf_max_nan(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float vf_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Drafts of a row, at most `most`: those before the first negative one.  By a
// whole warp.
__device__ __forceinline__ int vf_drafts(const ms_verify_args &x, int64_t b, int most) {
  for (int i = 0; i < most; i += 32) {
    const int at = i + (threadIdx.x & 31);
    const bool end = at >= most || load_in(x.draft_tokens + b * x.draft_row + at) < 0;
    const uint32_t ends = __ballot_sync(0xFFFFFFFFu, end);
    if (ends) return i + __ffs(ends) - 1;
  }
  return most;
}
// A temperature that rows can be drawn at.
__device__ __forceinline__ bool vf_heat(double t) { return t >= 0.0 && t <= 1.7976931348623157e308; }

// Statistics: a CTA takes a slice of one position.  The maximum moves with the
// values; weights are fp32, their sums of one step go into fp64.
template <int DT>
__global__ void __launch_bounds__(kVfThreads) ms_verify_stats_kernel(const __grid_constant__ VfArgs a) {
  using V = VfType<DT>;
  constexpr int kVec = V::kVec, kSteps = 16 / kVec * 2;  // 16-byte loads in flight: 32 values
  const float kNone = __uint_as_float(0xFF800000u), kInf = __uint_as_float(0x7F800000u);
  grid_wait();
  grid_release();
  const ms_verify_args &x = a.x;
  const int slice = blockIdx.x % a.slices;
  const int64_t at = blockIdx.x / a.slices, b = at / (x.drafts + 1);
  const int i = (int)(at - b * (x.drafts + 1));
  if (vf_drafts(x, b, i) < i) return;
  const double heat = load_in(x.temperature + b);
  const bool greedy = heat == 0.0;
  // finite and not 0, so that it makes neither a number of 0 times infinity
  const float c = greedy ? 1.f : (float)fmin(fmax(1.4426950408889634 / heat, 1e-37), 3e38);
  const typename V::T *row = static_cast<const typename V::T *>(x.logits) + b * x.logits_row + i * x.logits_pos;
  // 16-byte pieces: the first one starts before the row where the row does not start on one
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename V::T));
  const int64_t pieces = (x.vocab + skew + kVec - 1) / kVec;
  const int64_t each = a.slice / kVec, first = slice * each, last = min(pieces, first + each);
  float top = kNone;
  double sum = 0.0;
  int index = 0x7FFFFFFF, flags = 0;
  for (int64_t p0 = first + threadIdx.x; p0 < last; p0 += kSteps * kVfThreads) {
    float v[kSteps][kVec];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t e = (p0 + s * kVfThreads) * kVec - skew;
      if (p0 + s * kVfThreads >= last) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) v[s][k] = kNone;
      } else if (e >= 0 && e + kVec <= x.vocab) {
        V::wide(load_in(reinterpret_cast<const uint4 *>(row + e)), v[s]);
      } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k) v[s][k] = e + k >= 0 && e + k < x.vocab ? V::one(row + e + k) : kNone;
      }
    }
    float most = kNone;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int k = 0; k < kVec; k += 2) most = vf_max_nan(most, v[s][k], v[s][k + 1]);
    if (!(most < kInf)) {  // NaN reads as -inf
      flags = MS_ROW_NONFINITE;
      most = kNone;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          if (v[s][k] != v[s][k]) v[s][k] = kNone;
          most = fmaxf(most, v[s][k]);
        }
    }
    if (most > top) {
      sum = sum == 0.0 ? 0.0 : sum * (double)vf_exp2((top - most) * c);
      top = most;
      if (greedy) {
        index = 0x7FFFFFFF;
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s)
#pragma unroll
          for (int k = kVec - 1; k >= 0; --k)
            if (v[s][k] == top) index = (int)((p0 + s * kVfThreads) * kVec - skew + k);
      }
    }
    if (!greedy && top > kNone) {
      float part = 0.f;
      if (top < kInf) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int k = 0; k < kVec; ++k) part += vf_exp2((v[s][k] - top) * c);
      } else {  // infinite values share the weight
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int k = 0; k < kVec; ++k) part += v[s][k] == kInf ? 1.f : 0.f;
      }
      sum += (double)part;
    }
  }
  __shared__ VfRecord part[kVfWarps];
  auto join = [&](float t, double s, int k, int f) {
    const float next = fmaxf(top, t);
    if (top < next) sum = sum == 0.0 ? 0.0 : sum * (double)vf_exp2((top - next) * c);
    if (t < next) s = s == 0.0 ? 0.0 : s * (double)vf_exp2((t - next) * c);
    index = t > top ? k : t < top ? index : min(index, k);
    top = next;
    sum += s;
    flags |= f;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xFFFFFFFFu, top, o);
    const double s = __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const int k = __shfl_xor_sync(0xFFFFFFFFu, index, o), f = __shfl_xor_sync(0xFFFFFFFFu, flags, o);
    join(t, s, k, f);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = VfRecord{sum, top, index, flags};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kVfWarps; ++w) join(part[w].top, part[w].sum, part[w].index, part[w].flags);
    a.records[at * a.slices + slice] = VfRecord{sum, top, index, flags};
  }
}

__device__ __forceinline__ uint32_t vf_remote(const void *p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void vf_send(uint32_t to, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(v) : "memory");
}

struct VfShared {
  double mass[2][kVfCluster * kVfWarps];  // of the cluster's warps, in index order
  double odd[kVfCluster];                 // CTAs that met a draft probability that is none
  double accepted[kVfMaxDrafts + 1];      // p_i(d_i)
  double scan[kVfWarps];
  double z;
  float top;
  int index, flags, stop, drafts, status;
  int owner, last;
};

// Decision and draw: a cluster of eight CTAs takes a row.  Every CTA joins the
// row's records and decides, alike; then each sums its eighth of the position
// that is drawn from, warp by warp, the warps' sums are sent to all CTAs, and
// the CTA that holds the drawn place looks for it.
template <int DT>
__global__ void __launch_bounds__(kVfThreads) ms_verify_draw_kernel(const __grid_constant__ VfArgs a) {
  using V = VfType<DT>;
  const float kNone = __uint_as_float(0xFF800000u);
  __shared__ VfShared sh;
  const ms_verify_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank();
  const int64_t b = blockIdx.x / kVfCluster;
  grid_wait();
  const double heat = load_in(x.temperature + b), inv = 1.0 / heat;
  const bool greedy = heat == 0.0;
  if (warp == 0) {
    const int n = vf_drafts(x, b, x.drafts);
    bool bad = false;
    for (int i = lane; i < n; i += 32) bad = bad || load_in(x.draft_tokens + b * x.draft_row + i) >= x.vocab;
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (lane == 0) {
      sh.drafts = n;
      sh.status = (vf_heat(heat) ? MS_ROW_OK : MS_ROW_BAD_TEMPERATURE) | (bad ? MS_ROW_BAD_DRAFT : MS_ROW_OK);
      sh.stop = n;
      sh.flags = 0;
    }
  }
  __syncthreads();
  const int n = sh.drafts;
  auto give_up = [&](int status) {  // by the first CTA
    for (int i = tid; i <= x.drafts; i += kVfThreads) {
      x.tokens[b * (x.drafts + 1) + i] = -1;
      x.probs[b * (x.drafts + 1) + i] = 0.f;
    }
    if (tid == 0) x.counts[b] = 0, x.status[b] = status;
  };
  if (sh.status != MS_ROW_OK) {
    if (rank == 0) give_up(sh.status);
    return;
  }
  // weight of a value relative to the position's largest
  auto weigh = [&](float v, float top) { return v == top ? 1.0 : v == v ? exp(((double)v - (double)top) * inv) : 0.0; };
  auto logits = [&](int i) { return static_cast<const typename V::T *>(x.logits) + b * x.logits_row + i * x.logits_pos; };

  struct Whole {
    float top;
    double z;
    int index, flags;
  };
  auto join = [&](int i) {  // by a warp: position i's records
    Whole w{kNone, 0.0, 0x7FFFFFFF, 0};
    const VfRecord *r = a.records + (b * (x.drafts + 1) + i) * a.slices;
    for (int s = lane; s < a.slices; s += 32) {
      const VfRecord &v = r[s];
      w.flags |= v.flags;
      if (v.top > w.top) w.top = v.top, w.index = v.index;
      else if (v.top == w.top) w.index = min(w.index, v.index);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t = __shfl_xor_sync(0xFFFFFFFFu, w.top, o);
      const int k = __shfl_xor_sync(0xFFFFFFFFu, w.index, o);
      if (t > w.top) w.top = t, w.index = k;
      else if (t == w.top) w.index = min(w.index, k);
    }
    w.flags = __reduce_or_sync(0xFFFFFFFFu, w.flags);
    for (int s = lane; s < a.slices; s += 32) w.z += r[s].sum * weigh(r[s].top, w.top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w.z += __shfl_xor_sync(0xFFFFFFFFu, w.z, o);
    return w;
  };
  for (int i = warp; i < n; i += kVfWarps) {
    const Whole w = join(i);
    if (lane == 0) {
      const int64_t d = load_in(x.draft_tokens + b * x.draft_row + i);
      const double u = load_in(x.uniforms + b * x.uniform_row + i);
      const float v = V::one(logits(i) + d);
      const double p = greedy ? (d == w.index ? 1.0 : 0.0) : w.top > kNone ? weigh(v, w.top) / w.z : 0.0;
      const double q = x.draft_probs && !greedy ? (double)load_in(x.draft_probs + b * x.probs_row + i * x.probs_pos + d) : 1.0;
      sh.accepted[i] = p;
      if (!(u * q < p)) atomicMin(&sh.stop, i);
    }
  }
  __syncthreads();
  const int f = sh.stop;
  for (int i = warp; i <= f; i += kVfWarps) {  // what the positions up to the one that is drawn from hold
    const Whole w = join(i);
    if (lane == 0) {
      if (w.flags) atomicOr(&sh.flags, w.flags);
      if (i == f) sh.top = w.top, sh.index = w.index;
    }
  }
  __syncthreads();
  const float top = sh.top;
  if (!greedy && top == kNone) {
    if (rank == 0) give_up(MS_ROW_ALL_MASKED | sh.flags);
    return;
  }
  auto finish = [&](int64_t token, double p, int flags) {  // by a warp
    for (int i = lane; i <= x.drafts; i += 32) {
      const int64_t o = b * (x.drafts + 1) + i;
      x.tokens[o] = i < f ? load_in(x.draft_tokens + b * x.draft_row + i) : i == f ? token : -1;
      x.probs[o] = i < f ? (float)sh.accepted[i] : i == f ? (float)p : 0.f;
    }
    if (lane == 0) x.counts[b] = f + 1, x.status[b] = flags;
  };
  if (greedy) {
    if (rank == 0 && warp == 0) finish(top == kNone ? 0 : sh.index, 1.0, sh.flags);
    return;
  }
  __syncwarp();
  cluster_sync();  // the others have started
  const typename V::T *row = logits(f);
  const bool refused = f < n;
  const float *q = refused && x.draft_probs ? x.draft_probs + b * x.probs_row + f * x.probs_pos : nullptr;
  const int64_t without = refused && !q ? load_in(x.draft_tokens + b * x.draft_row + f) : -1;
  // the warp's part of the vocabulary
  const int64_t per = ((x.vocab + kVfCluster * kVfWarps - 1) / (kVfCluster * kVfWarps) + 31) / 32 * 32;
  const int part = rank * kVfWarps + warp;
  const int64_t lo = min(x.vocab, part * per), hi = min(x.vocab, lo + per);
  int odd = 0;
  // mass of entry j: of p alone, or of what is left of it
  enum { kWhole, kRest };
  double z_inv = 0.0;
  auto mass = [&](int64_t j, int kind) {
    const double w = weigh(V::one(row + j), top);
    if (kind == kWhole) return w;
    if (!q) return j == without ? 0.0 : w;
    const float d = load_in(q + j);
    if (!(d >= 0.f && d <= 3.402823466e38f)) odd = 1;
    return fmax(w * z_inv - fmax((double)d, 0.0), 0.0);  // a NaN reads as 0
  };
  auto sums = [&](int kind, int buffer) {
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    int64_t j = lo + lane;
    for (; j + 96 < hi; j += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += mass(j + 32 * k, kind);
    }
    for (; j < hi; j += 32) s[0] += mass(j, kind);
    double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    if (lane < kVfCluster) vf_send(vf_remote(&sh.mass[buffer][part], lane), t);
    if (kind == kRest && q) {
      const int any = __syncthreads_or(odd);
      if (tid < kVfCluster) vf_send(vf_remote(&sh.odd[rank], tid), (double)any);
    }
    __syncwarp();
    cluster_sync();
  };
  auto total = [&](int buffer) {
    double t = 0.0;
    for (int i = 0; i < kVfCluster * kVfWarps; ++i) t += sh.mass[buffer][i];
    return t;
  };
  double z = 0.0;
  int kind = kWhole, buffer = 0;
  if (q) {
    sums(kWhole, 0);
    z = total(0);
    z_inv = 1.0 / z;
  }
  int flags = sh.flags;
  if (refused) {
    kind = kRest, buffer = 1;
    sums(kRest, 1);
    if (q)
      for (int i = 0; i < kVfCluster; ++i) flags |= sh.odd[i] != 0.0 ? MS_ROW_NONFINITE : 0;
  } else {
    sums(kWhole, 0);
    z = total(0);
  }
  double all = total(buffer);
  if (refused && !(all > 0.0)) {  // nothing left: from p as it is
    kind = kWhole, buffer = 0;
    if (!q) sums(kWhole, 0), z = total(0);
    all = z;
  } else if (refused && !q) {
    z = all + weigh(V::one(row + without), top);
  }
  // the warp's part that holds the drawn place
  const double r = load_in(x.uniforms + b * x.uniform_row + x.drafts) * all;
  double before = 0.0;
  int found = -1, nonzero = 0;
  {
    double run = 0.0;
    for (int i = 0; i < kVfCluster * kVfWarps; ++i) {
      const double s = sh.mass[buffer][i];
      if (found < 0 && s > 0.0) {
        nonzero = i;
        before = run;
        if (run + s > r) found = i;
      }
      run += s;
    }
    if (found < 0) found = nonzero;  // rounding: the last part with mass
  }
  if (found / kVfWarps != rank) return;
  // all threads of this CTA look through it, each a run of entries
  const int64_t from = min(x.vocab, found * per), to = min(x.vocab, from + per);
  const int run = (int)((to - from + kVfThreads - 1) / kVfThreads);
  const int64_t t0 = min(to, from + (int64_t)tid * run), t1 = min(to, t0 + run);
  if (tid == 0) sh.owner = 0x7FFFFFFF, sh.last = -1;
  double s = 0.0;
  for (int64_t j = t0; j < t1; ++j) s += mass(j, kind);
  double incl = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  double base = before;
  for (int i = 0; i < warp; ++i) base += sh.scan[i];
  if (s > 0.0) {
    if (base + incl > r) atomicMin(&sh.owner, tid);
    atomicMax(&sh.last, tid);
  }
  __syncthreads();
  const int owner = sh.owner != 0x7FFFFFFF ? sh.owner : sh.last;
  if (tid / 32 != owner / 32) return;
  int64_t token = 0;
  double p = 0.0;
  if (tid == owner) {
    double at = base + (incl - s);
    for (int64_t j = t0; j < t1; ++j) {
      const double v = mass(j, kind);
      if (v > 0.0) {
        token = j;
        at += v;
        if (at > r) break;
      }
    }
    p = weigh(V::one(row + token), top) / z;
  }
  token = __shfl_sync(0xFFFFFFFFu, token, owner & 31);
  p = __shfl_sync(0xFFFFFFFFu, p, owner & 31);
  finish(token, p, flags);
}

// Slices of a position: so many that the positions fill the GPU, of 2048
// entries at least.
static void vf_slices(int64_t positions, int64_t vocab, int *slices, int64_t *slice) {
  const int64_t want = std::max<int64_t>(1, (148 * 8 + positions - 1) / positions);
  int64_t each = (vocab + want - 1) / want;
  each = std::max<int64_t>(2048, (each + 2047) / 2048 * 2048);
  *slice = each;
  *slices = (int)((vocab + 8 + each - 1) / each);  // 8: a row may start inside a piece
}

static bool vf_sizes(int64_t rows, int32_t drafts, int64_t vocab) {
  return rows >= 0 && rows <= 0x7FFFFFFFll / kVfCluster && drafts >= 0 && drafts <= kVfMaxDrafts && vocab >= 1 &&
         vocab <= kVfMaxVocab;
}

template <int DT>
static cudaError_t vf_run(const VfArgs &a, cudaStream_t s) {
  const int64_t positions = a.x.rows * (a.x.drafts + 1);
  cudaError_t e = launch_dependent(ms_verify_stats_kernel<DT>, (unsigned)(positions * a.slices), kVfThreads, 0, s, a);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.x.rows * kVfCluster));
  cfg.blockDim = dim3(kVfThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kVfCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, ms_verify_draw_kernel<DT>, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace ms

extern "C" {

int64_t ms_verify_workspace(int64_t rows, int32_t drafts, int64_t vocab) {
  if (!ms::vf_sizes(rows, drafts, vocab) || rows == 0) return 0;
  int slices;
  int64_t slice;
  ms::vf_slices(rows * (drafts + 1), vocab, &slices, &slice);
  return rows * (drafts + 1) * slices * (int64_t)sizeof(ms::VfRecord);
}

int ms_verify_drafts(const ms_verify_args *args, ms_stream_t stream) {
  if (!args) return MS_E_INVALID;
  const ms_verify_args &x = *args;
  if (x.dtype != MS_DTYPE_F32 && x.dtype != MS_DTYPE_BF16 && x.dtype != MS_DTYPE_F16) return MS_E_DTYPE;
  if (!ms::vf_sizes(x.rows, x.drafts, x.vocab)) return MS_E_INVALID;
  if (x.rows == 0) return MS_OK;
  if (!x.logits || !x.uniforms || !x.temperature || !x.tokens || !x.probs || !x.counts || !x.status || !x.workspace ||
      (reinterpret_cast<uintptr_t>(x.workspace) & 15) || (x.drafts > 0 && !x.draft_tokens) ||
      x.workspace_bytes < ms_verify_workspace(x.rows, x.drafts, x.vocab))
    return MS_E_INVALID;
  ms::VfArgs a{};
  a.x = x;
  a.records = static_cast<ms::VfRecord *>(x.workspace);
  ms::vf_slices(x.rows * (x.drafts + 1), x.vocab, &a.slices, &a.slice);
  if (x.rows * (x.drafts + 1) > 0x7FFFFFFFll / a.slices) return MS_E_INVALID;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = x.dtype == MS_DTYPE_F32    ? ms::vf_run<MS_DTYPE_F32>(a, s)
                  : x.dtype == MS_DTYPE_BF16 ? ms::vf_run<MS_DTYPE_BF16>(a, s)
                                             : ms::vf_run<MS_DTYPE_F16>(a, s);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
