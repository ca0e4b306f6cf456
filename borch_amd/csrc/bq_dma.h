// Loads straight into LDS, and the waits and barriers that they need.
#pragma once

#include "bq_common.h"

namespace bq {

// One 16-byte-per-lane load straight into LDS (no VGPR staging): lane l's 16 bytes land at
// LDS byte address m0v + 16 * l. Issued from inline assembly so that the compiler, which
// cannot tell these writes from the fragment reads of the other buffer, does not add a
// full vmcnt wait before every LDS read; the caller waits (vmcnt) before the barrier that
// publishes a stage. M0 is written here and used by nothing else in these kernels; the
// s_nop covers the M0-write -> LDS-DMA hazard.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t m0v) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "s"(m0v)
               : "m0");
#pragma clang diagnostic pop
}
__device__ __forceinline__ void wait_dma_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// A barrier orders LDS stores, not loads still in flight: before a barrier after which a
// buffer this wave read is refilled, its reads must have returned.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// The barrier alone: no memory access moves over it, and none is waited for. Every wave of the
// workgroup reaches as many, where the branches of whole waves differ.
__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_dma() {
  static_assert(N >= 0 && N <= 63, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace bq
