// LDS DMA and the waits of a ring of stages that it fills (fp8_gemm.hip, linear.hip).
#pragma once

#include "common.h"

namespace usaf {
namespace {

typedef __attribute__((address_space(3))) void* lds_void_ptr;

// Rows of 128 bytes: 16-byte chunk c of row r sits at c ^ g_swz(r), which spreads the reads of 16 rows' chunks over the banks.
__device__ __forceinline__ int g_swz(int r) { return (r >> 1) & 7; }

// LDS DMA: lane l's 16 (4) bytes at base + off land at lds + 16 l (4 l); base and lds are
// wave-uniform.  Inline asm, since beside the compiler's own LDS DMA every LDS read would
// wait for all of them.  M0 takes the LDS address; the wait states cover a base that comes
// out of readfirstlane.  They count in vmcnt only, which the ring waits for itself.
__device__ __forceinline__ void g_dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
__device__ __forceinline__ void g_dma4(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return reinterpret_cast<const uint8_t*>((uintptr_t)(((uint64_t)hi << 32) | (uint64_t)lo));
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace
}  // namespace usaf
