// Device helpers of the tensor-core kernels: mbarriers with bounded waits,
// TMA tile loads, and tcgen05 (allocation, descriptors, products, tensor
// memory reads and writes).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ms {

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ------------------------------------------------------------- mbarriers
__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// By the one lane of a converged warp that has `leader` set.
__device__ __forceinline__ void bar_expect(uint32_t leader, uint64_t *bar, uint32_t bytes) {
  asm volatile(
      "{ .reg .pred q; setp.ne.u32 q, %2, 0; @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1; }" ::"r"(
          smem_addr(bar)),
      "r"(bytes), "r"(leader)
      : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
static __device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, const volatile int *dead) {
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  for (uint32_t it = 1;; ++it) {
    if (bar_try(bar, parity)) return true;
    if ((it & 63u) == 0u) {
      if (dead && *dead) return false;
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
      if (t - t0 > 1000000000ull) return false;
    }
  }
}
// Waits for the phase of the given parity; false after about 1 s.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity) {
  const uint32_t b = smem_addr(bar);
  return bar_try(b, parity) || bar_wait_slow(b, parity, nullptr);
}
// For a whole warp: false, for all its lanes, where the wait ran out or another
// warp's had.
__device__ __forceinline__ bool bar_wait_warp(uint64_t *bar, uint32_t parity, const volatile int &dead) {
  const uint32_t b = smem_addr(bar);
  if (__all_sync(0xFFFFFFFFu, bar_try(b, parity))) return true;
  return __all_sync(0xFFFFFFFFu, bar_wait_slow(b, parity, &dead));
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Programmatic dependent launch: wait for the preceding grid's completion,
// let the following grid start.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A load of the caller's or of the grid before's data.  A grid launched so is
// resident while the one before it still writes; only a coherent load is
// certain to stay behind grid_wait.  (The read-only path, __ldg, is for memory
// that nothing writes during the kernel's whole life.)
template <typename T>
__device__ __forceinline__ T load_in(const T *p) {
  return *p;
}

// -------------------------------------------------------------------- TMA
// By the one lane of a converged warp that has `leader` set.
__device__ __forceinline__ void tma_load_2d(uint32_t leader, uint32_t dst, const void *map, uint32_t bar, int x, int y) {
  asm volatile(
      "{ .reg .pred q; setp.ne.u32 q, %5, 0; @q "
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2]; "
      "}" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void *dst, const void *map, uint64_t *bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_addr(dst)),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// ---------------------------------------------------------------- tcgen05
// Called by one whole warp; `cols` is a power of two, at least 32.
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The lane that issues a warp's products.  The whole warp walks through the
// code around them, so that descriptors and addresses stay in uniform
// registers; inside one lane's branch every product costs moves of them.
__device__ __forceinline__ uint32_t tc_leader() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one;
}
// The barrier is arrived at when every product the leader issued has finished.
__device__ __forceinline__ void tc_commit(uint32_t leader, uint64_t *bar) {
  asm volatile(
      "{ .reg .pred q; setp.ne.u32 q, %1, 0; @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 "
      "[%0]; }" ::"r"(smem_addr(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- pairs of CTAs (clusters of two) that issue one product over both
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of the pair's first CTA's copy of a shared variable.
__device__ __forceinline__ uint32_t leader_addr(const void *p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_addr(p)));
  return r;
}
// Relaxed: it orders nothing but tensor memory reads that have been waited for
// (tc_fence_before); a release at cluster scope would wait for the stores.
__device__ __forceinline__ void bar_arrive_leader(uint64_t *bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
}
// A tile into this CTA's memory, announced to the first CTA's barrier.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t leader, uint32_t dst, const void *map, uint32_t leader_bar,
                                                 int x, int y) {
  asm volatile(
      "{ .reg .pred q; setp.ne.u32 q, %5, 0; @q "
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2]; }" ::"r"(dst),
      "l"(map), "r"(leader_bar), "r"(x), "r"(y), "r"(leader)
      : "memory");
}
// By one warp of each CTA of the pair.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// Arrives at the barrier of both CTAs.
__device__ __forceinline__ void tc_commit_pair(uint32_t leader, uint64_t *bar) {
  asm volatile(
      "{ .reg .pred q; setp.ne.u32 q, %1, 0; @q "
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2; }" ::"r"(
          smem_addr(bar)),
      "r"(leader), "h"((uint16_t)3)
      : "memory");
}

// Shared-memory operand in 128-byte swizzled rows: groups of eight rows are
// `stride` bytes apart; `lead` is the distance of 64-element panels of a
// transposed operand (unused otherwise).
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t stride, uint32_t lead) {
  return ((uint64_t)((addr >> 4) & 0x3FFF)) | ((uint64_t)((lead >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((stride >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}

// int8 x int8 -> int32: A [m, 32], B [n, 32], both K-major; m is 128, or 256
// over a pair (each CTA has half of A's rows, B's rows and D's rows).
__device__ __forceinline__ uint32_t tc_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_i8_pair(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               bool accumulate) {
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 p, %4, 0; setp.ne.u32 q, %5, 0; @q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, "
      "%2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_mma_i8(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 p, %4, 0; setp.ne.u32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
      : "memory");
}

// 16 consecutive columns of this warp's 32 lanes.  The registers hold them
// after tmem_wait_ld, which names them so that no use moves ahead of it.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// 32 columns, read or written; 64 read.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
#define MS_TC_RW16(r, o)                                                                                     \
  "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), \
      "+r"(r[o + 7]), "+r"(r[o + 8]), "+r"(r[o + 9]), "+r"(r[o + 10]), "+r"(r[o + 11]), "+r"(r[o + 12]),      \
      "+r"(r[o + 13]), "+r"(r[o + 14]), "+r"(r[o + 15])
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MS_TC_RW16(r, 0), MS_TC_RW16(r, 16) : : "memory");
}
__device__ __forceinline__ void tmem_wait_ld64(uint32_t (&r)[64]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : MS_TC_RW16(r, 0), MS_TC_RW16(r, 16), MS_TC_RW16(r, 32), MS_TC_RW16(r, 48)
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float (&r)[64]) {
  uint32_t u[64];
  tmem_ld32(addr, u);
  tmem_ld32(addr + 32, u + 32);
  tmem_wait_ld64(u);
#pragma unroll
  for (int i = 0; i < 64; ++i) r[i] = __uint_as_float(u[i]);
}

// 16-bit floats x 16-bit floats -> fp32, M = 128: A [128, 16] K-major (shared
// or tensor memory), B [n, 16] K-major, or [16, n] when `transposed`.
template <typename T>
__device__ __forceinline__ constexpr uint32_t tc_idesc_f16(int n, bool transposed);
template <>
__device__ __forceinline__ constexpr uint32_t tc_idesc_f16<__nv_bfloat16>(int n, bool transposed) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((transposed ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((128u >> 4) << 24);
}
template <>
__device__ __forceinline__ constexpr uint32_t tc_idesc_f16<__half>(int n, bool transposed) {
  return (1u << 4) | ((transposed ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_f16(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 p, %4, 0; setp.ne.u32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_mma_f16_tmem(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 p, %4, 0; setp.ne.u32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
      : "memory");
}

}  // namespace ms
