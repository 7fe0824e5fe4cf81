// Asynchronous copies into shared memory and the barriers they complete on (sm_100a).
#pragma once

#include <stdint.h>

namespace gsb {

constexpr uint64_t kWaitNs = 4000000000ull;  // after which a wait gives up

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Bounded wait; false when it gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int* gave_up, uint64_t limit_ns = kWaitNs) {
  for (int i = 0; i < 256; ++i)
    if (bar_try(bar, parity)) return true;
  const uint64_t t0 = now_ns();
  while (now_ns() - t0 < limit_ns) {
    for (int i = 0; i < 64; ++i)
      if (bar_try(bar, parity)) return true;
  }
  atomicExch(gave_up, 1);
  return false;
}

// `bytes` (a multiple of 16) from a 16-byte aligned global address; completes on bar.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
      "r"(bytes), "r"(bar)
      : "memory");
}

// After a wait gave up: time for the copies in flight to land before the block ends.
__device__ __forceinline__ void let_copies_land() {
  for (int i = 0; i < 1000; ++i) __nanosleep(10000);
}

// Device word (of the current device) that is set when a bounded wait of a token-side kernel gave up;
// NULL on a CUDA error.
int* gave_up_flag();

}  // namespace gsb
