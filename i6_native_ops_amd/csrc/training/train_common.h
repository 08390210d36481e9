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

template <int DTYPE> struct Elem;
template <> struct Elem<I6TRAIN_F32> { using type = float; };
template <> struct Elem<I6TRAIN_BF16> { using type = bf16; };

inline size_t elem_size(int dtype) { return dtype == I6TRAIN_BF16 ? 2 : 4; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
template <typename A, typename B> __host__ __device__ inline A ceil_div(A a, B b) { return (a + (A)b - 1) / (A)b; }
inline bool valid_dtype(int dtype) { return dtype == I6TRAIN_F32 || dtype == I6TRAIN_BF16; }

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
