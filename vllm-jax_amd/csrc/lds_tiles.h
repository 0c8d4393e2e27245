// LDS access of the latent-attention kernels: direct global->LDS loads
// (lds_dma.h: a wave waits for its own with wait_vm), reads of tile operands,
// waits and barriers.
#pragma once

#include "lds_dma.h"
#include "pa_common.h"

namespace pa {

typedef s16x4 __attribute__((address_space(3))) * lds_tr_ptr;
typedef void __attribute__((address_space(3))) * lds_void;
typedef const char __attribute__((address_space(3))) * lds_bytes;

__device__ __forceinline__ u32x4 lds_ld16(uint32_t a) {
  return *reinterpret_cast<const u32x4 __attribute__((address_space(3)))*>((lds_bytes)(uintptr_t)a);
}
__device__ __forceinline__ u32x2 lds_tr8(uint32_t a) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(uintptr_t)a));
}
// Loads into a block whose address is made scalar here.
__device__ __forceinline__ void lds_dma16(const void* g, uint32_t block) {
  lds_load16(g, __builtin_amdgcn_readfirstlane(block));
}
__device__ __forceinline__ void lds_dma16s(uint32_t voff, const void* base, uint32_t block) {
  lds_load16s(voff, base, __builtin_amdgcn_readfirstlane(block));
}
// (a base that a vector instruction makes)
__device__ __forceinline__ void lds_dma16v(uint32_t voff, const void* base, uint32_t block) {
  lds_load16v(voff, base, __builtin_amdgcn_readfirstlane(block));
}
__device__ __forceinline__ void lds_dma16v_once(uint32_t voff, const void* base, uint32_t block) {
  lds_load16v_once(voff, base, __builtin_amdgcn_readfirstlane(block));
}
// s_waitcnt vmcnt(N), other counters untouched
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N < 64);
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8)); }

// Workgroup barrier that LDS accesses do not cross, in the compiler either.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// 16-byte chunk swizzles (XOR on the chunk's low bits) of tiles by row length,
// so that 16 rows' reads of one chunk land on distinct banks; those of 256 bytes
// and more, and value_swz128 for 128, also keep the four rows of a transposing
// read apart.
__device__ __forceinline__ int swz256(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
__device__ __forceinline__ int swz128(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swz64(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int value_swz128(int r) { return (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }

}  // namespace pa
