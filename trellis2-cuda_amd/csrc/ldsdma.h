// Loads straight from global memory into LDS, and the counted waits and barriers of the loops that run on them.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace {
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 rsrc4(const void* p, uint32_t bytes) {  // a raw buffer's descriptor, in SGPRs
  const uint64_t b = (uint64_t)(uintptr_t)p;
  return i32x4{(int32_t)__builtin_amdgcn_readfirstlane((uint32_t)b), (int32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)),
               (int32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// 16 bytes per lane, global -> LDS: lane l's land at dst + 16 l. Inline assembly, so that the compiler does not put a
// wait for it before every LDS read; the loops that use it count them. M0 (dst) needs one wait state between its scalar write
// and the load that reads it, which the compiler does not insert in here.
__device__ __forceinline__ void dma16(i32x4 r, uint32_t lds, uint32_t off, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               ::"s"(lds), "v"(off), "s"(r), "s"(soff) : "memory", "m0");
}
// The same to lds + AT
template <int AT>
__device__ __forceinline__ void dma16_at(i32x4 r, uint32_t lds, uint32_t off, int soff) {
  asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               ::"s"(lds), "v"(off), "s"(r), "s"(soff), "n"(AT) : "memory", "m0", "scc");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
}  // namespace
