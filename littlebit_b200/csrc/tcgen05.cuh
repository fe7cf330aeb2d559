// Fifth-generation tensor cores: tcgen05.mma kind::i8, TMEM, shared-memory operand
// descriptors, and waits that give up.  Shared by the tensor-core executor of the
// LittleBit linear (wide.cu) and the 8-bit integer product (int8.cu).
#pragma once

#include "common.cuh"

namespace lbx {

// ---------------------------------------------------------------------------
// tcgen05 / TMEM
// ---------------------------------------------------------------------------
LBX_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
LBX_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// (one full warp)
LBX_DEV void tmem_alloc(uint32_t *dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
LBX_DEV void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D[128 x N] (+)= A[128 x 32] . B[N x 32]^T, s8 x s8 -> s32, both K-major
LBX_DEV void umma_i8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive on `bar` once every tcgen05.mma issued so far by this thread completed
LBX_DEV void umma_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
LBX_DEV void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 32 lanes x NC consecutive 32-bit columns: thread i gets lane (base lane + i)
template <int NC>
LBX_DEV void tmem_ld(uint32_t taddr, uint32_t *r);
template <>
LBX_DEV void tmem_ld<4>(uint32_t a, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
template <>
LBX_DEV void tmem_ld<8>(uint32_t a, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(a));
}
template <>
LBX_DEV void tmem_ld<16>(uint32_t a, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(a));
}
template <>
LBX_DEV void tmem_ld<32>(uint32_t a, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
// NC columns in loads of at most 32
template <int NC>
LBX_DEV void tmem_ld_cols(uint32_t a, uint32_t *r) {
  if constexpr (NC <= 32) {
    tmem_ld<NC>(a, r);
  } else {
    tmem_ld<32>(a, r);
    tmem_ld_cols<NC - 32>(a + 32, r + 32);
  }
}

// Shared-memory matrix descriptor of a K-major operand in 128-byte swizzle
// atoms (8 rows x 128 bytes, 1024-byte aligned, stacked every 1024 bytes):
// start address >> 4 in bits 0-13, leading byte offset 16 B (unused by this
// layout), stride byte offset 1024 B, descriptor version 1 (bit 46), swizzle
// mode 2 (128 B) in bits 61-63.  Advancing the start by 32 bytes selects the
// next K=32 slice inside the atom (the swizzle applies to the full address).
LBX_DEV uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// instruction descriptor: D s32 (bits 4-5 = 2), A and B s8 (bits 7-9, 10-12
// = 1), both K-major, N >> 3 in bits 17-22, M >> 4 = 8 (M = 128) in bits 24-28
__host__ __device__ constexpr uint32_t idesc_i8(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// byte offset of (row n, K byte c < 128) in a stack of swizzled atoms
LBX_DEV uint32_t sw128_off(int n, int c) {
  return (uint32_t)((n >> 3) * 1024 + (n & 7) * 128 + ((((c >> 4) ^ n) & 7) << 4) + (c & 15));
}
LBX_DEV uint8_t *align1024(uint8_t *p) {
  return p + ((1024u - (smem_u32(p) & 1023u)) & 1023u);
}

// (try_wait suspends the thread in hardware until the phase completes or a
// short time limit passes, so waiting warps leave the issue slots to the
// working ones)
LBX_DEV bool wd_wait(uint64_t *bar, uint32_t parity, int code, volatile int *abort) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 7u) == 7) {  // (a wait that is soon over reads no clock)
      if (*abort) return false;
      uint64_t t;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (it == 7) t0 = t;
      else if (t - t0 > 1000000000ull) {
        *abort = 1;
        atomicCAS(&g_lbx_device_error, 0, code);
        return false;
      }
    }
  }
}
LBX_DEV void mbar_arrive1(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

}  // namespace lbx
