// Tensor-core (tcgen05) building blocks of the kernels that use them:
// shared-memory descriptors, commits, fences, and the bounded waits of
// warp-specialised kernels.
#pragma once

#include "mi_device.cuh"

namespace mi {

// Shared-memory matrix descriptor, no swizzle, K-major: core matrices of 8
// rows x 16 B; lbo = byte distance between K-adjacent core matrices, sbo =
// between M/N-adjacent ones; bit 46 = descriptor version 1 (sm_100).
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) |
         ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void mbar_arrive_one(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// try_wait that lets the thread sleep until the phase completes (or about a
// microsecond passes), so that waiting warps leave their issue slots to the
// warps that compute.
__device__ __forceinline__ bool mbar_try_wait_sleep(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity), "r"(1000u)
      : "memory");
  return ok != 0;
}

// Bounded wait of one thread: gives up when another role has flagged an
// abort, or after kSpinLimit polls (then it flags one).
__device__ __forceinline__ bool tc_wait1(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
  for (uint32_t it = 0;; it++) {
    if (mbar_try_wait_sleep(bar, parity)) return true;
    if ((it & 31u) == 31u && *abort_flag) return false;
    if (it >= kSpinLimit) {
      *abort_flag = 1;
      if (err) atomicExch(err, 5 /* MI_CUDA_ERR_TIMEOUT */);
      return false;
    }
  }
}
// The same for a whole warp (every lane polls, the warp leaves together).
// Re-polling a completed phase is safe: none of the barriers a warp waits on
// can complete its next phase without that warp's own arrival.
__device__ __forceinline__ bool tc_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                             int32_t* err) {
  for (uint32_t it = 0;; it++) {
    if (__all_sync(0xffffffffu, mbar_try_wait_sleep(bar, parity))) return true;
    if ((it & 31u) == 31u && __any_sync(0xffffffffu, *abort_flag != 0)) return false;
    if (it >= kSpinLimit) {
      *abort_flag = 1;
      if (err && (threadIdx.x & 31) == 0) atomicExch(err, 5 /* MI_CUDA_ERR_TIMEOUT */);
      return false;
    }
  }
}

// The same where the phase has usually completed: looks once before it sleeps.
__device__ __forceinline__ bool tc_wait_ready(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
  return __all_sync(0xffffffffu, mbar_test(bar, parity)) || tc_wait_warp(bar, parity, abort_flag, err);
}

}  // namespace mi
