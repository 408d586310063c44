// cx_dma.hpp -- loads from memory to LDS that kernels wait for by count.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cx {

// 16 bytes a lane from memory to LDS, lane after lane from `to` on, which wave_vm and a
// barrier wait for.  (The builtin would make every read of LDS wait for all of them.)
__device__ __forceinline__ void load_lds16(const char* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(to), "v"(from) : "memory", "m0");
}
// Waits until at most N of the wave's loads are under way, and its LDS writes are done.
template <int N>
__device__ __forceinline__ void wave_vm() {
  constexpr int n = N < 0 ? 0 : N > 63 ? 63 : N;
  __builtin_amdgcn_s_waitcnt((n & 15) | ((n >> 4) << 14) | (7 << 4));
}

}  // namespace cx
