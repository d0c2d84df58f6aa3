// Loads from memory straight into LDS that the caller waits for.
//
// The compiler waits for all of a wavefront's loads into LDS before any read of LDS
// that may alias, also where the read is of another buffer: a tile on its way while
// the one before it is used would arrive first.  These are in assembly, so that it
// knows of none; dma_wait() and a barrier come before the data is read.  They have no
// register results, so none is in flight while it looks free.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace spyre_hip {

// A raw buffer of `bytes` at a wave-uniform address.
typedef uint32_t dma_rsrc __attribute__((ext_vector_type(4)));
__device__ __forceinline__ dma_rsrc dma_buffer(const void* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  return dma_rsrc{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at))),
                  static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32))) & 0xffffu, bytes, 0x00020000u};
}

// The byte address in LDS of an object there.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

// Lane l's 16 bytes at byte voff + soff of the buffer go to LDS byte dst + 16 l (dst,
// soff wave-uniform); where voff is not within the buffer they are zeros.
// A memory instruction that reads a scalar register needs 5 wait states after a vector
// instruction that wrote it, and one that uses m0 needs 1 after its write; the hardware
// checks neither, and for a load in assembly the compiler does not either (a spilled soff
// comes back by v_readlane right before it).  s_mov and s_nop 3 are 1 + 4.
__device__ __forceinline__ void dma16(dma_rsrc r, uint32_t dst, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(dst), "v"(voff), "s"(r), "s"(soff)
               : "memory", "m0");
}

__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

}  // namespace spyre_hip
