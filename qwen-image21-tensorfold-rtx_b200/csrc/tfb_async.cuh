// Asynchronous copies and their barriers, shared by the attention kernels. Every wait is bounded (kWaitLimitNs): a
// wait that runs out records its code in the device error word and tells its caller to stop.
#pragma once

#include "tfb_common.cuh"

namespace tfb {

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_arrive_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Returns at once where bar_try may suspend the thread (about 128 cycles even for a completed phase).
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
template <bool POLL>
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, int* err, int code, long long limit) {
  const unsigned long long t0 = globaltimer();
  for (uint32_t it = 1;; ++it) {
    if (POLL ? bar_test(bar, parity) : bar_try(bar, parity)) return true;
    if ((it & 255) == 0) {
      if (*reinterpret_cast<volatile int*>(err) != 0) return false;
      if (static_cast<long long>(globaltimer() - t0) > limit) {
        atomicCAS(err, 0, code);
        return false;
      }
    }
  }
}
template <bool POLL = false>
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int* err, int code,
                                         long long limit = kWaitLimitNs) {
  const uint32_t a = smem_u32(bar);
  return (POLL ? bar_test(a, parity) : bar_try(a, parity)) || bar_wait_slow<POLL>(a, parity, err, code, limit);
}
// A whole warp's wait, with one answer for all lanes: a lane may find the phase complete where another has run out of time or
// seen an error. (Every lane looks: one lane's answer handed round took longer.)
template <bool POLL = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code,
                                          long long limit = kWaitLimitNs) {
  return __all_sync(0xffffffffu, bar_wait<POLL>(bar, parity, err, code, limit));
}

// A wait (bounded as well) for what is in flight after an error: it does not stop at the error itself.
__device__ __forceinline__ void bar_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer();
  while (!bar_test(smem_u32(bar), parity) && static_cast<long long>(globaltimer() - t0) < kWaitLimitNs) {
  }
}

// Contiguous global -> shared copy (16-byte aligned, a multiple of 16 bytes) that completes on `bar`.
__device__ __forceinline__ void copy_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void copy_tensor_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

}  // namespace tfb
