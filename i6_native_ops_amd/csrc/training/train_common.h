// Shared by the kernels of libi6train.so (include/i6train.h): element types, wave-wide reductions, host-side checks.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../../include/i6train.h"

namespace i6train {

using bf16 = __bf16;
using f16 = _Float16;

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// `add` of 64 lanes' values, in all of them: within rows of 16 lanes from 1, 2, 4 and 8 lanes below, then the last lane of rows 0 and 2 to rows 1 and 3,
// then that of row 1 to rows 2 and 3.  `none` is what lanes without a neighbour add.
template <typename F> __device__ __forceinline__ uint32_t wave_reduce(uint32_t x, uint32_t none, F add) {
#define I6_STEP(ctrl, rows) x = add(x, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, ctrl, rows, 0xf, false));
    I6_STEP(0x111, 0xf)
    I6_STEP(0x112, 0xf)
    I6_STEP(0x114, 0xf)
    I6_STEP(0x118, 0xf)
    I6_STEP(0x142, 0xa)
    I6_STEP(0x143, 0xc)
#undef I6_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// Of bit patterns of magnitudes, whose order as whole numbers is that of the magnitudes with NaN on top.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    return wave_reduce(x, 0, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ float wave_sum(float x) {
    return __uint_as_float(wave_reduce(__float_as_uint(x), 0, [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

inline size_t elem_size(int dtype) { return dtype == I6TRAIN_BF16 ? 2 : 4; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
template <typename A, typename B> __host__ __device__ inline A ceil_div(A a, B b) { return (a + (A)b - 1) / (A)b; }
inline bool valid_dtype(int dtype) { return dtype == I6TRAIN_F32 || dtype == I6TRAIN_BF16; }

// A launch has fewer than 2^32 threads in each dimension.
inline bool launchable(int64_t groups, int threads) { return groups < ((int64_t)1 << 32) / threads; }

// The status of the last launch, as a code of this library.
inline int launched() { return hipGetLastError() == hipSuccess ? I6TRAIN_OK : I6TRAIN_ERR_LAUNCH; }

// Where kernels report a problem: {code, sequence} in pinned host memory of the current device; null if there is none.
int* status_slot();

#define I6TRAIN_TRY(call)                                \
    do {                                                 \
        const int try_rc_ = (call);                      \
        if (try_rc_ != I6TRAIN_OK) return try_rc_;       \
    } while (0)

}  // namespace i6train
