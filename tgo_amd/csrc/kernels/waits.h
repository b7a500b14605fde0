// waits.h -- a wave's waits for its own LDS accesses and DMA, without the fences that
// would wait for every load in flight.
#pragma once

#include "../common.h"

namespace tgohip {

// s_waitcnt vmcnt(0) lgkmcnt(0), and no memory access moves across it: the wave's DMA has
// landed, and its LDS reads have returned, before other data goes where they read.
__device__ __forceinline__ void pack_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
}
// A barrier without a memory fence, which would wait for every DMA in flight; no
// memory access moves across it.
__device__ __forceinline__ void pack_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Orders a wave's own LDS writes before its other lanes' reads (and back).
__device__ __forceinline__ void pack_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace tgohip
