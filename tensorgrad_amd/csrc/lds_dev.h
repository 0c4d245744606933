// Loads from memory straight into LDS: their addresses and their wait. Shared by the attention kernels and k_linear.hip.
#pragma once
#include "gemm_dev.h"   // the loads

namespace tgk {

__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }   // stores too
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

}  // namespace tgk
