// tcgen05 products issued by a converged warp.
#pragma once
#include "tc_common.cuh"

namespace tpp {

// Matrix descriptors (128-byte swizzle, 8-row groups 1 KB apart) as a low word, which a
// step along the tile moves, and a high word that never changes.
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return (addr >> 4) | (lbo >> 4) << 16;
}
// The warp that issues runs converged, with operands the same in every lane, and only the
// instruction itself is the elected lane's (`on`): inside a one-lane branch each operand
// would go through a vector register first, which made an MMA cost 160 clocks, not 64.
__device__ __forceinline__ bool elect_lane() {
  uint32_t on;
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, e;\n\t}"
      : "=r"(on));
  return on != 0;
}
__device__ __forceinline__ void mma_ss(bool on, uint32_t d, uint32_t a_lo, uint32_t b_lo,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %6, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHi), "r"((uint32_t)on)
      : "memory");
}
__device__ __forceinline__ void mma_ts(bool on, uint32_t d, uint32_t a, uint32_t b_lo,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %6, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHi), "r"((uint32_t)on)
      : "memory");
}
__device__ __forceinline__ void commit(bool on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)), "r"((uint32_t)on)
      : "memory");
}
// 32 lanes x 32 bit, 8 consecutive columns per thread.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
// mbar_wait in little code: a kernel of many roles and waits outgrows the instruction cache
// (with the loops unrolled packed_attn_kernel had 210 KB, and every wait cost 250 clocks).
__device__ __forceinline__ bool wait_short(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kWaitLimit; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  if (err) atomicExch(err, code);
  return false;
}
// The same value from every lane, as the compiler can see.
__device__ __forceinline__ int same(int v) { return __shfl_sync(0xffffffffu, v, 0); }

}  // namespace tpp
