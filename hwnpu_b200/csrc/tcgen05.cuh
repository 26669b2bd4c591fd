// tcgen05.cuh: mbarriers, bulk copies and the 5th-generation tensor cores (tcgen05) as the kernels of
// tcgemm.cu and paged_prompt.cu use them.
#ifndef HWNPU_TCGEN05_CUH
#define HWNPU_TCGEN05_CUH

#include "device.cuh"

namespace hc {

constexpr long long kTcSpin = 2000000000ll;  // clock cycles a wait may take

__device__ __forceinline__ uint32_t tc_saddr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void tc_bar_init(uint64_t *b, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc_saddr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void tc_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(tc_saddr(b)) : "memory");
}
__device__ __forceinline__ void tc_expect_tx(uint64_t *b, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(tc_saddr(b)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool tc_try(uint64_t *b, unsigned parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred P;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 P, [%1], %2, %3;\n"
      " selp.u32 %0, 1, 0, P;\n}\n"
      : "=r"(ok)
      : "r"(tc_saddr(b)), "r"(parity), "n"(1000)
      : "memory");
  return ok != 0;
}
// Waits for the phase of the given parity to complete, at most kTcSpin cycles; on running out it
// records code in *status (the first one) and returns.
__device__ __forceinline__ void tc_wait(uint64_t *b, unsigned parity, int *status, int code) {
  if (tc_try(b, parity)) return;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (tc_try(b, parity)) return;
    if (clock64() - t0 > kTcSpin) {
      atomicCAS(status, 0, code);
      return;
    }
  }
}
// True on one thread of a converged warp.
__device__ __forceinline__ bool tc_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tc_bulk(void *dst, const void *src, unsigned bytes, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc_saddr(dst)),
      "l"(src), "r"(bytes), "r"(tc_saddr(bar))
      : "memory");
}

// ---- tcgen05 --------------------------------------------------------------------------------
// Shared-memory matrix descriptor of a K-major operand without swizzle: core matrices of 8 rows x
// 16 bytes (128 contiguous bytes); lbo: bytes between the two core matrices of one MMA's 16
// columns, sbo: bytes between core matrices 8 rows apart; version 1 (bits 46-47).
__device__ __forceinline__ uint64_t tc_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) |
         (uint64_t((sbo >> 4) & 0x3FFFu) << 32) | (uint64_t(1) << 46);
}
__device__ __forceinline__ void tc_mma(uint32_t tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrives on b once every MMA this thread issued before has completed.
__device__ __forceinline__ void tc_commit(uint64_t *b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tc_saddr(b))
               : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// Makes this thread's shared-memory stores visible to the tensor core (the async proxy).
__device__ __forceinline__ void tc_fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 columns of the accumulator for this warp's 32 lanes (rows) into v.
__device__ __forceinline__ void tc_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

}  // namespace hc

#endif
