// Loads, barriers and branches that the compiler is not to take for something else.
#pragma once

#include <hip/hip_runtime.h>

namespace ekv {

#if defined(__HIPCC__)

// A load of memory that is not LDS. The compiler cannot tell for an address that a select chose, and its load for either
// kind returns in no order, so that a wait for one would wait for all that are under way.
template <typename V>
__device__ __forceinline__ V load_global(const char* at) {
    return *(const __attribute__((address_space(1))) V*)(at);
}

// A barrier for what is in LDS. __syncthreads() also waits for every load from memory that is under way, and would end
// each prefetch at the next barrier.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Keeps what stands beside it under its branch: without it the compiler computes a rare branch's selects every time.
__device__ __forceinline__ void rarely() { asm volatile(""); }

#endif

}  // namespace ekv
