// ms_verify_drafts -- drafted tokens against a target model's logits, from
// given uniforms (declared in include/mssample.h).
//
// With p_i = softmax(logits_i / T) and the draft's probabilities q_i, draft d_i
// is accepted when u_i q_i(d_i) < p_i(d_i).  At the first one refused the token
// is drawn from max(p_i - q_i, 0), and where all are accepted one more from p:
// the tokens are distributed as if each had been drawn from p_i.  Draws run in
// index order: the first token whose running mass passes u times the whole.
//
// Two kernels.  The first reads every position's logits once, for their largest
// values and the sums of their weights in fp32 (bound by bytes): what the
// decisions compare with is off by up to 1e-6, which decides at most one case in a
// million otherwise.  The second, a cluster of CTAs a row, decides and draws from one
// position.  A draw compares with the running mass at every one of the
// vocabulary's borders, so that its weights and sums are in 64 bits: with 32
// about one draw in a thousand would land beside its token.
//
// Measured, four drafts a row over 151936 fp32 logits: 64 rows 64 us, of which
// the sums, 175 MB at 5.2 TB/s, are 34 and the draws 30 (latency: fp64 operations
// one after the other, and the sums' way through the cluster); one row 17 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/mssample.h"
#include "ms_host.h"
#include "ms_tc.cuh"

namespace ms {

constexpr int kVfThreads = 128;   // of a CTA that sums slices
constexpr int kVfSums = 6;        // such CTAs of an SM: what their rings leave room for
constexpr int kVfPieces = 4;      // 16-byte pieces of a lane's batch of values
constexpr int kVfStages = 4;      // batches of a warp's ring
constexpr int kVfCluster = 8;     // CTAs of a row's draw, at most
constexpr int kVfMaxDrafts = 255;
constexpr int64_t kVfMaxVocab = 0x7FFFFFFFll - 65536;

// Of a slice of one position's logits.
struct VfRecord {
  double sum;  // of the weights, relative to the largest value's
  float top;   // largest value
  int index;   // its first place
  int flags;   // MS_ROW_NONFINITE
};

struct VfArgs {
  ms_verify_args x;
  VfRecord *records;  // [rows][drafts + 1][slices]
  int slices;
  int slice;          // entries of a slice
  int ranks;          // CTAs of a row's draw
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
// Two fp32 operations an instruction.
__device__ __forceinline__ float2 vf_add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
  return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 vf_mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
  return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 vf_fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
  return *reinterpret_cast<float2 *>(&d);
}
// A difference of logits in units of log2 is its `part` times `by`: finite and
// not 0, so that neither makes a number of 0 times infinity.  The part is one
// half where logits past fp32's largest difference still weigh something.
struct VfUnit {
  float part, by;
};
__device__ __forceinline__ VfUnit vf_unit(double heat) {
  if (heat == 0.0) return VfUnit{1.f, 1.f};
  const double unit = 1.4426950408889634 / heat;
  // (float)1.4e-45, the least fp32 value, times the largest difference is 1e-6
  return unit < 1e-30 ? VfUnit{0.5f, (float)fmax(2.0 * unit, 1.4e-45)} : VfUnit{1.f, (float)fmin(unit, 3e38)};
}
// A sum of weights relative to `from`, as one relative to `to`, which is not below it.
__device__ __forceinline__ double vf_moved(double sum, float from, float to, VfUnit unit) {
  return from == to || sum == 0.0 ? sum : sum * (double)vf_exp2(fmaf(from, unit.part, -to * unit.part) * unit.by);
}

// A thread's values so far.
struct VfSum {
  float top;
  double sum;  // of the weights, relative to top's
  int index, flags;
};

// One more batch of values, piece s's at s * 32 pieces from place `first` on.
template <int kPieces, int kVec>
__device__ __forceinline__ void vf_add(VfSum &a, float (&v)[kPieces][kVec], int first, bool greedy, VfUnit unit) {
  const float kNone = __uint_as_float(0xFF800000u), kInf = __uint_as_float(0x7F800000u);
  float most = kNone;
#pragma unroll
  for (int s = 0; s < kPieces; ++s)
#pragma unroll
    for (int k = 0; k < kVec; k += 2) most = vf_max_nan(most, v[s][k], v[s][k + 1]);
  if (!(most < kInf)) {  // NaN reads as -inf
    a.flags = MS_ROW_NONFINITE;
    most = kNone;
#pragma unroll
    for (int s = 0; s < kPieces; ++s)
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        if (v[s][k] != v[s][k]) v[s][k] = kNone;
        most = fmaxf(most, v[s][k]);
      }
  }
  if (most > a.top) {
    a.sum = vf_moved(a.sum, a.top, most, unit);
    a.top = most;
    if (greedy) {
      a.index = 0x7FFFFFFF;
#pragma unroll
      for (int s = kPieces - 1; s >= 0; --s)
#pragma unroll
        for (int k = kVec - 1; k >= 0; --k)
          if (v[s][k] == most) a.index = first + s * 32 * kVec + k;
    }
  }
  if (greedy || a.top == kNone) return;
  float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  if (a.top < kInf) {
    const float2 from = make_float2(-a.top * unit.part, -a.top * unit.part), part_of = make_float2(unit.part, unit.part),
                 by = make_float2(unit.by, unit.by);
#pragma unroll
    for (int s = 0; s < kPieces; ++s)
#pragma unroll
      for (int k = 0; k < kVec; k += 2) {
        const float2 t = vf_mul2(vf_fma2(make_float2(v[s][k], v[s][k + 1]), part_of, from), by);
        part[(k >> 1) & 1] = vf_add2(part[(k >> 1) & 1], make_float2(vf_exp2(t.x), vf_exp2(t.y)));
      }
  } else {  // infinite values share the weight
#pragma unroll
    for (int s = 0; s < kPieces; ++s)
#pragma unroll
      for (int k = 0; k < kVec; ++k) part[0].x += v[s][k] == kInf ? 1.f : 0.f;
  }
  a.sum += (double)((part[0].x + part[0].y) + (part[1].x + part[1].y));
}

// Sums: a warp takes a slice of a position; a ring of asynchronous copies, each
// lane's pieces for itself, keeps three batches on their way while it weighs the
// fourth.  CTAs are small and many: positions behind a row's drafts have none,
// and what a slice costs varies.
template <int DT>
__global__ void __launch_bounds__(kVfThreads, kVfSums) ms_verify_sums_kernel(const __grid_constant__ VfArgs a) {
  using V = VfType<DT>;
  constexpr int kVec = V::kVec, kPieces = kVfPieces;
  const float kNone = __uint_as_float(0xFF800000u);
  __shared__ uint4 ring[kVfThreads / 32][kVfStages][kPieces][32];
  grid_wait();
  grid_release();
  const ms_verify_args &x = a.x;
  const int lane = threadIdx.x & 31;
  // fewer than 2^31 items (the host's check): divisions in 32 bits
  const uint32_t item = blockIdx.x * (kVfThreads / 32) + (threadIdx.x >> 5);
  const uint32_t at = item / (uint32_t)a.slices, row_at = at / (uint32_t)(x.drafts + 1);
  const int slice = (int)(item - at * a.slices), i = (int)(at - row_at * (x.drafts + 1));
  const int64_t b = row_at;
  if (b >= x.rows) return;
  const double heat = load_in(x.temperature + b);
  if (vf_drafts(x, b, i) < i || !vf_heat(heat)) return;
  const bool greedy = heat == 0.0;
  const VfUnit unit = vf_unit(heat);
  const typename V::T *row = static_cast<const typename V::T *>(x.logits) + b * x.logits_row + i * x.logits_pos;
  // 16-byte pieces: the first one starts before the row where the row does not start on one.  Pieces `inner` .. `outer`
  // - 1 lie in the row as a whole.
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename V::T));
  const int vocab = (int)x.vocab;
  const int first = slice * (a.slice / kVec), last = min((vocab + skew + kVec - 1) / kVec, first + a.slice / kVec);
  const int inner = skew ? 1 : 0, outer = min((vocab + skew) / kVec, last);
  const uint4 *base = reinterpret_cast<const uint4 *>(row - skew);
  VfSum mine{kNone, 0.0, 0x7FFFFFFF, 0};
  uint4 (*mine_ring)[kPieces][32] = ring[threadIdx.x >> 5];
  auto fetch = [&](int p0, int stage) {
#pragma unroll
    for (int s = 0; s < kPieces; ++s) {
      const int p = p0 + s * 32;
      const bool in = p >= inner && p < outer;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(&mine_ring[stage][s][lane])),
                   "l"(in ? base + p : reinterpret_cast<const uint4 *>(a.records)), "r"(in ? 16 : 0)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kStep = 32 * kPieces;
#pragma unroll
  for (int s = 0; s < kVfStages - 1; ++s) fetch(first + lane + s * kStep, s);
  int stage = 0;
  for (int p0 = first + lane; p0 - lane < last; p0 += kStep) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kVfStages - 2) : "memory");
    float v[kPieces][kVec];
#pragma unroll
    for (int s = 0; s < kPieces; ++s) V::wide(mine_ring[stage][s][lane], v[s]);
    fetch(p0 + (kVfStages - 1) * kStep, stage == 0 ? kVfStages - 1 : stage - 1);
    if (++stage == kVfStages) stage = 0;
    if (p0 - lane < inner || p0 - lane + kStep > outer) {  // the row's ends
#pragma unroll
      for (int s = 0; s < kPieces; ++s) {
        const int p = p0 + s * 32;
        if (p < inner || p >= outer) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            const int e = p * kVec - skew + k;
            v[s][k] = p < last && e >= 0 && e < vocab ? V::one(row + e) : kNone;
          }
        }
      }
    }
    vf_add<kPieces, kVec>(mine, v, p0 * kVec - skew, greedy, unit);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // the lanes' sums, relative to the slice's largest value
  float top = mine.top;
  int index = mine.index;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xFFFFFFFFu, top, o);
    const int k = __shfl_xor_sync(0xFFFFFFFFu, index, o);
    if (t > top) top = t, index = k;
    else if (t == top) index = min(index, k);
  }
  double sum = vf_moved(mine.sum, mine.top, top, unit);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  const int flags = __reduce_or_sync(0xFFFFFFFFu, mine.flags);
  if (lane == 0) a.records[item] = VfRecord{sum, top, index, flags};
}

// Weights in 64 bits.  2^(t / 128) for t = v c - R, c = 128 log2(e) /
// temperature: the nearest whole number k of t gives the power of two (k / 128
// rounded down) and a table's place; the rest r of at most a half is a power
// series of three terms, (r ln 2 / 128)^4 / 24 < 2^-38 off.  R is a multiple of
// 128 near the largest value's t.  The table is there sixteen times, a copy for
// each pair of lanes, so that no two copies share a bank; its high words have
// the place's bits taken off, so that k 2^13 added to one is the scaled power.
constexpr int kVfSteps = 128, kVfCopies = 16;
struct VfPowers {
  double of[kVfSteps];  // 2^(i / 128), by its power series
  constexpr VfPowers() : of() {
    for (int i = 0; i < kVfSteps; ++i) {
      const double x = 0.69314718055994530942 * i / kVfSteps;
      double sum = 1.0;
      for (int k = 24; k > 0; --k) sum = 1.0 + sum * x / k;
      of[i] = sum;
    }
  }
};
__device__ const VfPowers vf_powers{};

constexpr double kVfMagic = 6755399441055744.0;  // 1.5 * 2^52: the low word of a sum with it is a whole number
constexpr double kVfLeast = 1000.0;              // weights below 2^-1000 count as 0
constexpr double kVfMost = 3.4028234663852886e38;  // the largest fp32 value

struct VfScale {
  double c;     // steps of a unit of logit
  double base;  // kVfMagic - R
  float least;  // values below it weigh nothing
  // v c is far inside whole numbers' range.  Where it is not (temperatures so small that neighbouring values are 2^21
  // steps apart, or an infinite value), the largest value weighs 1 and all others nothing.
  bool plain;
};
// Of the steps c of a unit of logit at a temperature, for a largest value that is not -inf.
__device__ __forceinline__ VfScale vf_scale(double c, double heat, float top) {
  VfScale s;
  s.c = c;
  s.plain = fabs((double)top) * c < 35184372088832.0 && c < 1e290;  // 2^45
  s.base = kVfMagic - (s.plain ? kVfSteps * ceil((double)top * c * (1.0 / kVfSteps)) : 0.0);
  // rounded up, which passes no value of `top`: a value below 2^-1000 would wrap the power's exponent
  s.least = s.plain ? __double2float_ru(fmax((double)top - kVfLeast * 0.69314718055994530942 * heat, -kVfMost)) : top;
  return s;
}
// Relative to 2^(R / 128) or, of scales that are not plain, to the largest
// value's; for values from `least` on.
__device__ __forceinline__ double vf_power(const VfScale &s, float v, const double *power) {
  const double x = (double)v, shifted = fma(x, s.c, s.base), r = fma(x, s.c, s.base - shifted);
  const int k = __double2loint(shifted);
  const double g = power[(k & (kVfSteps - 1)) * kVfCopies + (threadIdx.x & (kVfCopies - 1))];
  const double f = __hiloint2double(__double2hiint(g) + (k << 13), __double2loint(g));
  constexpr double ln = 0.69314718055994530942 / kVfSteps;
  return s.plain ? fma(f, r * fma(r, fma(r, ln * ln * ln / 6.0, ln * ln / 2.0), ln), f) : 1.0;
}
__device__ __forceinline__ double vf_weight(const VfScale &s, float v, const double *power) {
  return v >= s.least ? vf_power(s, v, power) : 0.0;  // a NaN is not
}

__device__ __forceinline__ uint32_t vf_remote(const void *p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void vf_send(uint32_t to, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(v) : "memory");
}
__device__ __forceinline__ double vf_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// Running sums over a warp's lanes.
__device__ __forceinline__ double vf_warp_run(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double e = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += e;
  }
  return v;
}
// The first lane whose running mass, on top of `before`, passes r, or by rounding the last one with mass; `before`
// becomes the mass up to it.  False where no lane has mass, or, unless `end`, none passes r: `before` then has all lanes'.
__device__ __forceinline__ bool vf_find(double mass, double r, bool end, double &before, int &found) {
  const double run = vf_warp_run(mass);
  const uint32_t some = __ballot_sync(0xFFFFFFFFu, mass > 0.0);
  const uint32_t past = __ballot_sync(0xFFFFFFFFu, mass > 0.0 && before + run > r);
  const bool here = past || (end && some);
  found = past ? __ffs(past) - 1 : 31 - __clz(some | 1);
  before += __shfl_sync(0xFFFFFFFFu, here ? run - mass : run, here ? found : 31);
  return here;
}

// What a part's sums are of: the weights, of all entries or of all but a draft;
// what is left, by the first kernel's z, of the entries that have more weight
// than the draft gave them, and what it gave those; what is left by the exact z.
enum { kVfAll, kVfMore, kVfTaken, kVfRest, kVfKinds };

constexpr int kVfRun = 8;  // batches whose draft probabilities are summed in fp32

template <int kThreads>
struct VfShared {
  double given[kThreads];                    // the runs' sums of a thread
  double power[kVfSteps * kVfCopies];
  double sum[kVfKinds][kThreads / 32];       // of the CTA's warps
  double mass[kVfKinds][kVfCluster];         // of the cluster's CTAs, in index order
  double odd[kVfCluster];                    // CTAs that met a draft probability that is none
  double share[kVfMaxDrafts + 1];            // 1 over the sum of a position's weights
  VfScale scale[kVfMaxDrafts + 1];
  float accepted[kVfMaxDrafts + 1];          // p_i(d_i)
  int draft[kVfMaxDrafts + 1];
  int index[kVfMaxDrafts + 1], flags[kVfMaxDrafts + 1];
  bool none[kVfMaxDrafts + 1];               // all values are -inf
  double c, heat;
  VfUnit unit;
  int stop, drafts, status;
};

// Decision and draw: a cluster of CTAs takes a row.  Every CTA joins the row's
// records and decides, alike; then each sums its part of the position that is
// drawn from, the sums are sent to all CTAs, and the CTA that holds the drawn
// place looks for it: in its warps' sums, in the warps' parts of that warp's
// entries, and in those 32 at a time.
//
// What the draft's probabilities leave, max(w / z - q, 0), needs the whole z of
// the weights w first.  One pass is enough all the same: the first kernel's z is
// known to 1e-6, and the entries that it puts on the wrong side of w / z = q are
// those where next to nothing is left, so that the sum over its side, S = sum (w
// / z - q) and Q = sum q, is S + (S + Q) (z / z' - 1) for the exact z' to 2e-12,
// with Q to 2e-6 of itself (fp32 over a row of 2^24 tokens, a CTA's: borders were
// off by 1e-10).  Where all that is left is itself small (a draft model that is
// the target, nearly), a second pass takes the exact z.
//
// fp64 operations take some 40 cycles one after the other, and divisions several
// hundred: one thread makes a position's scale, and 32-wide scans stand where a
// loop over eight sums would do.
template <int DT, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) ms_verify_draw_kernel(const __grid_constant__ VfArgs a) {
  using V = VfType<DT>;
  constexpr int kWarps = kThreads / 32;
  const float kNone = __uint_as_float(0xFF800000u);
  __shared__ VfShared<kThreads> sh;
  const ms_verify_args &x = a.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), ranks = a.ranks;
  const int64_t b = blockIdx.x / ranks;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for before a CTA writes to another
  const double entry = vf_powers.of[(tid >> 1) % kVfSteps];
  grid_wait();
  const double u = load_in(x.uniforms + b * x.uniform_row + x.drafts);  // the draw's
  if (warp == 0) {
    const double heat = load_in(x.temperature + b);
    const int n = vf_drafts(x, b, x.drafts);
    bool bad = false;
    for (int i = lane; i < n; i += 32) {
      const int64_t d = load_in(x.draft_tokens + b * x.draft_row + i);
      bad = bad || d >= x.vocab;
      sh.draft[i] = (int)d;
    }
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (lane == 0) {
      sh.drafts = sh.stop = n;
      sh.status = (vf_heat(heat) ? MS_ROW_OK : MS_ROW_BAD_TEMPERATURE) | (bad ? MS_ROW_BAD_DRAFT : MS_ROW_OK);
      sh.heat = heat;
      sh.c = 1.4426950408889634 * kVfSteps / heat;
      sh.unit = vf_unit(heat);
    }
  }
  sh.given[tid] = 0.0;
  if (tid < 2 * kVfSteps) {
    const int step = tid >> 1;
    const double g = __hiloint2double(__double2hiint(entry) - (step << 13), __double2loint(entry));
#pragma unroll
    for (int i = 0; i < kVfCopies / 2; ++i) sh.power[step * kVfCopies + (tid & 1) * (kVfCopies / 2) + i] = g;
  }
  __syncthreads();
  const int n = sh.drafts;
  auto meet = [&]() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); };
  auto give_up = [&](int status) {  // by the first CTA
    for (int i = tid; i <= x.drafts; i += kThreads) {
      x.tokens[b * (x.drafts + 1) + i] = -1;
      x.probs[b * (x.drafts + 1) + i] = 0.f;
    }
    if (tid == 0) x.counts[b] = 0, x.status[b] = status;
  };
  if (sh.status != MS_ROW_OK) {
    if (rank == 0) give_up(sh.status);
    __syncwarp();
    meet();
    return;
  }
  const VfUnit unit = sh.unit;
  const bool greedy = sh.heat == 0.0;
  auto logits = [&](int i) { return static_cast<const typename V::T *>(x.logits) + b * x.logits_row + i * x.logits_pos; };
  for (int i = warp; i <= n; i += kWarps) {  // the positions' records
    const int d = i < n ? sh.draft[i] : 0;
    double chance = 0.0, q = 1.0;
    float v = kNone;
    if (i < n && lane == 0) {
      chance = load_in(x.uniforms + b * x.uniform_row + i);
      v = V::one(logits(i) + d);
      if (x.draft_probs && !greedy) q = load_in(x.draft_probs + b * x.probs_row + i * x.probs_pos + d);
    }
    const VfRecord *r = a.records + (b * (x.drafts + 1) + i) * a.slices;
    VfSum all{kNone, 0.0, 0x7FFFFFFF, 0};
    for (int s = lane; s < a.slices; s += 32) {
      const VfRecord e = r[s];
      const float next = fmaxf(all.top, e.top);
      all.sum = vf_moved(all.sum, all.top, next, unit) + vf_moved(e.sum, e.top, next, unit);
      all.index = e.top > all.top ? e.index : e.top < all.top ? all.index : min(all.index, e.index);
      all.top = next;
      all.flags |= e.flags;
    }
    float top = all.top;
    int index = all.index;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t = __shfl_xor_sync(0xFFFFFFFFu, top, o);
      const int k = __shfl_xor_sync(0xFFFFFFFFu, index, o);
      if (t > top) top = t, index = k;
      else if (t == top) index = min(index, k);
    }
    const int flags = __reduce_or_sync(0xFFFFFFFFu, all.flags);
    const double z = vf_warp_sum(vf_moved(all.sum, all.top, top, unit));
    if (lane == 0) {
      if (top == kNone) index = 0;  // all are as large
      sh.index[i] = index, sh.flags[i] = flags, sh.none[i] = top == kNone;
      double p = 0.0;
      if (greedy) {
        p = d == index ? 1.0 : 0.0;
      } else if (top > kNone) {
        const VfScale s = vf_scale(sh.c, sh.heat, top);
        const double share = 1.0 / (vf_power(s, top, sh.power) * z);
        p = vf_weight(s, v, sh.power) * share;
        sh.scale[i] = s, sh.share[i] = share;
      }
      if (i < n) {
        sh.accepted[i] = (float)p;
        if (!(chance * q < p)) atomicMin(&sh.stop, i);
      }
    }
  }
  __syncthreads();
  const int f = sh.stop;
  int flags = 0;
  for (int i = 0; i <= f; ++i) flags |= sh.flags[i];
  const bool none = sh.none[f];
  auto finish = [&](int64_t token, double p) {  // by a warp
    for (int i = lane; i <= x.drafts; i += 32) {
      const int64_t o = b * (x.drafts + 1) + i;
      x.tokens[o] = i < f ? sh.draft[i] : i == f ? token : -1;
      x.probs[o] = i < f ? sh.accepted[i] : i == f ? (float)p : 0.f;
    }
    if (lane == 0) x.counts[b] = f + 1, x.status[b] = flags;
  };
  if (greedy || none) {
    if (rank == 0 && !greedy) give_up(MS_ROW_ALL_MASKED | flags);
    if (rank == 0 && greedy && warp == 0) finish(sh.index[f], 1.0);
    __syncwarp();
    meet();
    return;
  }
  const typename V::T *row = logits(f);
  const bool refused = f < n;
  const float *q = refused && x.draft_probs ? x.draft_probs + b * x.probs_row + f * x.probs_pos : nullptr;
  int without = refused && !q ? sh.draft[f] : -1;
  const VfScale scale = sh.scale[f];
  const double first_share = sh.share[f];
  double share = first_share;  // 1 / z
  uint32_t odd = 0;  // the largest bit pattern of the draft's probabilities: those past the finite ones are none
  // a warp's part of the vocabulary, of one CTA after the other
  const int64_t per = ((x.vocab + ranks * kWarps - 1) / (ranks * kWarps) + 31) / 32 * 32;
  {  // the CTA's entries on their way to L2
    const int64_t from = min(x.vocab, rank * kWarps * per), to = min(x.vocab, from + kWarps * per);
    auto touch = [&](const char *p, const char *end) {
      for (p += tid * 128; p < end; p += kThreads * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    };
    touch(reinterpret_cast<const char *>(row + from), reinterpret_cast<const char *>(row + to));
    if (q) touch(reinterpret_cast<const char *>(q + from), reinterpret_cast<const char *>(q + to));
  }
  constexpr std::integral_constant<int, kVfAll> kAll{};
  constexpr std::integral_constant<int, kVfMore> kMore{};
  constexpr std::integral_constant<int, kVfRest> kRest{};
  // an entry's part in the sums s of a kind
  auto add = [&](double (&s)[2], float &given, float v, float d, bool in, auto kind) {
    const double w = vf_power(scale, v, sh.power);
    const bool some = in && v >= scale.least;  // a NaN is not
    if constexpr (kind.value == kVfAll) {
      if (some) s[0] += w;
    } else {
      d += 0.f;  // no -0
      odd = max(odd, __float_as_uint(d));
      const double taken = (double)fmaxf(d, 0.f);  // a NaN reads as 0
      const double rest = fma(w, share, -taken);
      const bool more = some && __double2hiint(rest) > 0;  // above 2^-1023, that is
      if constexpr (kind.value == kVfMore) {
        if (some) s[0] += w;
        if (more) s[1] += rest, given += fmaxf(d, 0.f);
      } else {
        if (more) s[0] += rest;
      }
    }
  };
  // entries lo .. hi - 1 by a warp
  auto part = [&](int64_t lo, int64_t hi, double (&s)[3], auto kind) {
    constexpr int kBatch = 8;
    constexpr bool kTakes = kind.value != kVfAll;
    double t[2][2] = {};
    float given[2] = {0.f, 0.f};
    const int end = (int)hi;
    for (int j0 = (int)lo; j0 < end; j0 += 32 * kBatch) {
      const int j = j0 + lane;
      const typename V::T *at = row + j;
      const float *taken = q + j;
      float v[kBatch], d[kBatch];
      if (j0 + 32 * kBatch <= end && (kTakes || (unsigned)(without - j0) >= 32 * kBatch)) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) v[k] = V::one(at + 32 * k), d[k] = kTakes ? load_in(taken + 32 * k) : 0.f;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) add(t[k & 1], given[k & 1], v[k], d[k], true, kind);
      } else {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const bool in = j + 32 * k < end;
          v[k] = in ? V::one(at + 32 * k) : kNone;
          d[k] = in && kTakes ? load_in(taken + 32 * k) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (j0 + 32 * k < end) add(t[k & 1], given[k & 1], v[k], d[k], j + 32 * k != without, kind);
      }
      if constexpr (kind.value == kVfMore) {
        constexpr int kRun = 32 * kBatch * kVfRun;
        if (((j0 - (int)lo) & (kRun - 1)) == kRun - 32 * kBatch) {
          sh.given[tid] += (double)(given[0] + given[1]);
          given[0] = given[1] = 0.f;
        }
      }
    }
    s[0] = vf_warp_sum(t[0][0] + t[1][0]);
    if constexpr (kind.value == kVfMore) {
      s[1] = vf_warp_sum(t[0][1] + t[1][1]);
      s[2] = vf_warp_sum(sh.given[tid] + (double)(given[0] + given[1]));
    }
  };
  // Every CTA's sums of its part to all of them, at places `slot` on.
  bool met = false;
  auto sums = [&](int slot, auto kind) {
    constexpr int kSums = kind.value == kVfMore ? 3 : 1;
    const int64_t lo = min(x.vocab, (rank * kWarps + warp) * per), hi = min(x.vocab, lo + per);
    double s[3];
    part(lo, hi, s, kind);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kSums; ++i) sh.sum[slot + i][warp] = s[i];
    }
    const int any = __syncthreads_or(odd > 0x7F7FFFFFu);
    if (!met) {
      __syncwarp();
      meet();
      met = true;
    }
    if (warp < kSums) {
      const double all = vf_warp_sum(lane < kWarps ? sh.sum[slot + warp][lane] : 0.0);
      if (lane < ranks) {
        vf_send(vf_remote(&sh.mass[slot + warp][rank], lane), all);
        if (warp == 0) vf_send(vf_remote(&sh.odd[rank], lane), (double)any);
      }
    }
    __syncwarp();
    cluster_sync();
  };
  // A lane's part of the row, of CTAs or of warps, as the draw sees it: nothing where what is left of a part is within
  // the rounding of its sums: of Q 33 roundings to fp32, 2e-6, in the part of it that the exact z moves, and per / 64
  // roundings of 2^-53.  What the sums find left is at most what is left by the exact z, but for that: a part that is
  // chosen holds an entry to draw.
  int slot = kVfAll;
  double moved = 0.0;  // by the exact z, over the first kernel's: its share less 1
  auto mass = [&](const double *of, int pitch, int count) {
    if (lane >= count) return 0.0;
    if (slot != kVfMore) return of[slot * pitch + lane];
    const double left = of[kVfMore * pitch + lane], all = left + of[kVfTaken * pitch + lane];
    const double rest = fma(all, moved, left);
    return rest > fma(fabs(moved), 2e-6, fma((double)per, 0x1p-57, 1e-13)) * all ? rest : 0.0;
  };
  auto whole = [&]() { return vf_warp_sum(mass(&sh.mass[0][0], kVfCluster, ranks)); };
  double all;
  if (!q) {
    sums(kVfAll, kAll);
    all = whole();
    const double z = all + (refused ? vf_weight(scale, V::one(row + without), sh.power) : 0.0);
    share = 1.0 / z;
    if (!(all > 0.0)) {  // nothing left: from p as it is
      without = -1;
      slot = kVfRest;  // not where others may still read
      sums(kVfRest, kAll);
      all = whole();
    }
  } else {
    sums(kVfAll, kMore);
    share = 1.0 / whole();
    moved = (share - first_share) / first_share;
    slot = kVfMore;
    all = whole();
    if (!(all > 1e-3)) {
      slot = kVfRest;
      sums(kVfRest, kRest);
      all = whole();
    }
    if (__any_sync(0xFFFFFFFFu, lane < ranks && sh.odd[lane] != 0.0)) flags |= MS_ROW_NONFINITE;
    if (!(all > 0.0)) {
      slot = kVfAll;
      all = whole();
    }
  }
  const bool rest = q && slot != kVfAll;
  const double r = u * all;
  double before = 0.0;
  int found;
  vf_find(mass(&sh.mass[0][0], kVfCluster, ranks), r, true, before, found);
  if (found != rank) return;
  vf_find(mass(&sh.sum[0][0], kWarps, kWarps), r, true, before, found);
  const int64_t begin = min(x.vocab, (rank * kWarps + found) * per), end = min(x.vocab, begin + per);
  // that warp's entries, a part for each warp
  const int64_t step = ((end - begin + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t lo = min(end, begin + warp * step), hi = min(end, lo + step);
  {
    double s[3];
    if (rest) part(lo, hi, s, kRest);
    else part(lo, hi, s, kAll);
    __syncthreads();  // the sums above have been read
    if (lane == 0) sh.sum[0][warp] = s[0];
    __syncthreads();
  }
  vf_find(lane < kWarps ? sh.sum[0][lane] : 0.0, r, true, before, found);
  if (found != warp) return;
  // the warp's entries, a run for each lane; then the entries of the lane that is found
  auto mass_at = [&](int64_t j) {
    double s[2] = {0.0, 0.0};
    float given = 0.f;
    if (rest) add(s, given, V::one(row + j), load_in(q + j), true, kRest);
    else add(s, given, V::one(row + j), 0.f, (int)j != without, kAll);
    return s[0];
  };
  const int64_t run = (hi - lo + 31) / 32;
  int64_t token = lo, from = min(hi, lo + lane * run);
  if (run > 1) {
    double s = 0.0;
    for (int64_t j = from; j < min(hi, from + run); ++j) s += mass_at(j);
    vf_find(s, r, true, before, found);
    token = lo + found * run;
  }
  for (int64_t end = run > 1 ? min(hi, token + run) : hi, j0 = token; j0 < end; j0 += 32) {
    const double m = j0 + lane < end ? mass_at(j0 + lane) : 0.0;
    const uint32_t some = __ballot_sync(0xFFFFFFFFu, m > 0.0);
    if (some) token = j0 + 31 - __clz(some);  // the last one so far, should none pass r by rounding
    if (vf_find(m, r, false, before, found)) {
      token = j0 + found;
      break;
    }
  }
  finish(token, vf_weight(scale, V::one(row + token), sh.power) * share);
}

// Entries of a slice: about four slices for each warp that an SM has room for,
// but 4096 entries (what a slice costs besides its entries is that of 1000), or
// what fills the GPU once, of 1024 entries at least.  64 rows: 66 us with one
// slice a warp, 65 with two to six.
static void vf_slices(int64_t positions, int64_t vocab, int *slices, int *slice) {
  const int64_t warps = 148ll * kVfSums * (kVfThreads / 32);
  auto each = [&](int64_t all) {
    const int64_t want = std::max<int64_t>(1, (all + positions - 1) / positions);
    return ((vocab + want - 1) / want + 1023) / 1024 * 1024;
  };
  *slice = (int)std::max(each(4 * warps), std::min<int64_t>(4096, each(warps)));
  *slices = (int)((vocab + 8 + *slice - 1) / *slice);  // 8: a row may start inside a piece
}

static bool vf_sizes(int64_t rows, int32_t drafts, int64_t vocab) {
  return rows >= 0 && rows <= 0x7FFFFFFFll / kVfCluster && drafts >= 0 && drafts <= kVfMaxDrafts && vocab >= 1 &&
         vocab <= kVfMaxVocab;
}

template <int DT, int kThreads>
static cudaError_t vf_draw(const VfArgs &a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.x.rows * a.ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, ms_verify_draw_kernel<DT, kThreads>, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Draws by CTAs of 1024 threads where every row's cluster has SMs of its own: one
// row takes 16.4 us so and 19.2 with 256 threads; 64 rows 85 us and 63.
template <int DT>
static cudaError_t vf_run(const VfArgs &a, cudaStream_t s) {
  const int64_t items = a.x.rows * (a.x.drafts + 1) * a.slices;
  const unsigned blocks = (unsigned)((items + kVfThreads / 32 - 1) / (kVfThreads / 32));
  cudaError_t e = launch_dependent(ms_verify_sums_kernel<DT>, blocks, kVfThreads, 0, s, a);
  if (e != cudaSuccess) return e;
  return a.x.rows * kVfCluster <= 148 ? vf_draw<DT, 1024>(a, s) : vf_draw<DT, 256>(a, s);
}

}  // namespace ms

extern "C" {

int64_t ms_verify_workspace(int64_t rows, int32_t drafts, int64_t vocab) {
  if (!ms::vf_sizes(rows, drafts, vocab) || rows == 0) return 0;
  int slices, slice;
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
  // CTAs of a row: as many as one wave has room for (four of 256 threads an SM), so that every row's draw runs at once.
  // 200 rows of 32003 logits in clusters of two 37.7 us, of four 37.9, of one 42.4; 64 of 151936 of eight 63, of four 75.
  a.ranks = ms::kVfCluster;
  while (a.ranks > 1 && x.rows * a.ranks > 148 * 4) a.ranks >>= 1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = x.dtype == MS_DTYPE_F32    ? ms::vf_run<MS_DTYPE_F32>(a, s)
                  : x.dtype == MS_DTYPE_BF16 ? ms::vf_run<MS_DTYPE_BF16>(a, s)
                                             : ms::vf_run<MS_DTYPE_F16>(a, s);
  return e == cudaSuccess ? MS_OK : ms::cuda_fail(e);
}

}  // extern "C"
