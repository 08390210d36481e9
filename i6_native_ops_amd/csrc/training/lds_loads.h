// Loads from memory to LDS that bypass the registers, and waiting for them.
#pragma once
#include "train_common.h"

namespace i6train {

// Waits for this wave's reads of LDS, and for its loads but the last `kLeft`; then for the other waves.
template <int kLeft> __device__ __forceinline__ void wait_and_meet() {
    static_assert(kLeft < 16, "one field of the instruction");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | kLeft);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }

// A description of `bytes` bytes from p on; reads behind them give 0.
using descriptor = uint32_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ descriptor describe(const void* p, int64_t bytes) {
    const uint64_t at = (uint64_t)p;
    const auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    return descriptor{uniform((uint32_t)at), uniform((uint32_t)(at >> 32) & 0xffffu), uniform(bytes > 0xffffffffll ? 0xffffffffu : (uint32_t)bytes), 0x00020000u};
}

// 64 lanes x 16 bytes from the described memory, at `from` + `offset`, to LDS from address `to` on, lane after lane.  Written out because the compiler
// takes every later read of LDS to depend on it and waits for all loads there; wait_and_meet() counts them instead.  No register receives
// anything; m0, which takes the address in LDS, is used by nothing else here.
__device__ __forceinline__ void load_to_lds(descriptor d, uint32_t to, uint32_t from, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(from), "s"(d), "s"(offset) : "memory");
}

}  // namespace i6train
