// tcgen05 pieces of the prefill attention kernels (e4m3 and 4-bit pages): f16 MMA, TMEM loads and
// stores by lane, and bounded waits that end a CTA's loops through a shared abort flag.
#pragma once

#include "common.cuh"
#include "sm100.cuh"

namespace ada {
namespace tca {

constexpr unsigned int ERR_TILE_WAIT = 0x70;

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 16 consecutive fp32 columns of this thread's TMEM lane; the values are valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Wait for this thread's tcgen05.ld, then pin the 16 registers after the wait (an empty volatile
// asm that redefines them), so no use of them is scheduled before it.
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]));
}
__device__ __forceinline__ void tmem_pin16(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// try_wait with a suspend-time hint: the thread sleeps until the phase completes (or the hint
// runs out) instead of spinning, so waiting roles leave the issue slots to the working ones.
__device__ __forceinline__ bool try_wait_sleep(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(sm100::smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

// Bounded wait (2 s): gives up when another role aborted, or sets the abort flag and the error
// code when the phase never completes.
__device__ __forceinline__ bool wait_b(uint64_t* bar, uint32_t parity, volatile int* abort_v, unsigned int* err) {
  if (try_wait_sleep(bar, parity)) return true;
  const uint64_t t0 = sm100::globaltimer();
  for (;;) {
    if (try_wait_sleep(bar, parity)) return true;
    if (*abort_v) return false;
    if (sm100::globaltimer() - t0 > 2000000000ull) {
      *abort_v = 1;
      if (err) atomicOr(err, ERR_TILE_WAIT);
      return false;
    }
  }
}

// The same for a whole warp, with one outcome for all lanes: what follows may be warp-collective.  (A lane that gave up
// alone would be missing there, and the others would wait for it for good.)
__device__ __forceinline__ bool wait_w(uint64_t* bar, uint32_t parity, volatile int* abort_v, unsigned int* err) {
  if (__all_sync(0xffffffffu, try_wait_sleep(bar, parity))) return true;
  const uint64_t t0 = sm100::globaltimer();
  for (;;) {
    if (__all_sync(0xffffffffu, try_wait_sleep(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_v)) return false;
    if (__any_sync(0xffffffffu, sm100::globaltimer() - t0 > 2000000000ull)) {
      *abort_v = 1;
      if (err) atomicOr(err, ERR_TILE_WAIT);
      return false;
    }
  }
}

}  // namespace tca
}  // namespace ada
