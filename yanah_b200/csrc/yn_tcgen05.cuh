// Thin PTX wrappers shared by the tensor-core kernels: shared-memory operand
// descriptors, tcgen05 commits and fences, TMA tile copies, mbarrier arrivals.
#pragma once
#include <cuda.h>

#include "yn_common.cuh"

namespace ynb {

YN_DEV uint64_t tc_desc(uint32_t smem_addr) {
  // K-major, 128-byte swizzle: start address (>>4), leading offset 1 (unused
  // for swizzled K-major), stride offset 1024 bytes between 8-row atoms,
  // version 1, layout type 2 (SWIZZLE_128B)
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
  d |= (uint64_t)1u << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

YN_DEV void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

YN_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
YN_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

YN_DEV void tc_tma_rows(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

YN_DEV void mbar_arrive1(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

}  // namespace ynb
