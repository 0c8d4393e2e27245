// Direct global->LDS loads of gfx950, 16 bytes a lane: lane l's 16 bytes land at
// LDS byte address block + 16 * l (block wave-uniform).
//
// Inline asm, so that the compiler does not insert its conservative "wait for
// every LDS DMA" before unrelated LDS reads: a wave waits for its own loads
// (vmcnt), and a barrier behind the wait makes them visible to the others.  The
// compiler does not look for hazards inside asm either, so the wait states that
// the hardware asks software for stand here: one between the write of M0 and the
// load, and for a scalar base five between a vector instruction that writes it
// (v_readfirstlane, v_readlane) and the load, of which s_mov is one.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pa {

__device__ __forceinline__ void lds_load16(const void* g, uint32_t block) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(block)
               : "memory", "m0");
}

// The same from a scalar base: lane l loads the 16 bytes at base + voff.  The
// base comes from scalar instructions (tests/test_lds_load_waits.py looks for
// vector ones too near in the built library): with the waits of the form below
// the long prefills took 1.1 % longer.
__device__ __forceinline__ void lds_load16s(uint32_t voff, const void* base, uint32_t block) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(block)
               : "memory", "m0");
}

// The same from a base that a vector instruction may have made just before.
__device__ __forceinline__ void lds_load16v(uint32_t voff, const void* base, uint32_t block) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(block)
               : "memory", "m0");
}

// And for data that is read once: it does not displace other lines of L2.
__device__ __forceinline__ void lds_load16v_once(uint32_t voff, const void* base, uint32_t block) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voff), "s"(base), "s"(block)
               : "memory", "m0");
}

}  // namespace pa
