// What the tensor-core kernels share: mbarriers with bounded waits, tensor memory's
// fences and commits, descriptors of operands in shared memory.
#pragma once

#include "common.cuh"

namespace shlo {

constexpr uint64_t kWaitLimitNs = 2000000000ull;

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok) : "r"(smem_at(b)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_test(uint64_t *b, uint32_t parity) {  // without waiting
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok) : "r"(smem_at(b)), "r"(parity) : "memory");
  return ok != 0;
}
// A wait of two seconds at most; it ends early when another warp gave up.
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity, volatile int *gone) {
  if (bar_try(b, parity)) return true;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  for (uint32_t i = 1;; i++) {
    if (bar_try(b, parity)) return true;
    if ((i & 255) == 0) {
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
      if (*gone || t - t0 > kWaitLimitNs) {
        *gone = 1;
        return false;
      }
    }
  }
}
// The same for a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, volatile int *gone) {
  return __all_sync(~0u, bar_wait(b, parity, gone));
}
// What is still on the way when a block gives up is waited for, for two seconds at most.
__device__ __forceinline__ void bar_drain(uint64_t *b, uint32_t parity) {
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  do {
    if (bar_try(b, parity)) return;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  } while (t - t0 < kWaitLimitNs);
}
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint64_t *b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_at(b)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}
// Shared-memory operands in the 128-byte swizzle: rows of 128 bytes, eight rows
// a group of 1024; `lead` bytes between 64-value blocks (N-major operands).
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t lead) {
  return (uint64_t)((at >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

}  // namespace shlo
