// Orthogonal factors of matrices by Newton-Schulz products, and the optimiser's step on them (include/i6orth.h).
//
// X has n rows and m >= n columns.  An iteration is three products for all matrices of the call, a launch each:  A = X X^T,
// B = b A + c A A,  X = a X + B X.  A and B are symmetric: of the first two only the tiles on and below the diagonal are formed, and written to both
// places.  X is kept as it is and transposed, so that both operands of every product have consecutive k.
//
// Operands are two 16-bit floating-point halves, x = x1 + x2, of 22 bits, times a power of two that brings the largest value they can have (X: 1.21, A: 1.46,
// B: 2.9) below 2^16; of (x1 + x2)(y1 + y2) the last term is below the precision.  Half the bits would do for the products, but not for what becomes of them: an error in A is one of
// left singular vectors of all sizes, and the small ones grow 3.4 times in each iteration, 485 times in five.
#include <cmath>

#include "train_common.h"
#include "../../../include/i6orth.h"

namespace i6train {
namespace {

using f16x4 = f16 __attribute__((ext_vector_type(4)));
using f16x8 = f16 __attribute__((ext_vector_type(8)));
using acc_t = float __attribute__((ext_vector_type(4)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kLeastNorm = 1e-7;
constexpr float kScaleX = 0x1p15f, kScaleA = 0x1p15f, kScaleB = 0x1p14f;
constexpr int kMaxTensors = 40;          // x 96 bytes: the arguments of a kernel may have 4 KB
constexpr int kThreads = 256;
constexpr int kTile = 128, kStep = 32, kRowPad = 32;
constexpr int kParts = 256;              // partial sums of squares of a matrix

struct Matrix {
    const void* update;
    void* result;
    float* momentum;
    f16 *x, *xt, *xt_next, *a, *b;       // halves one after another
    double* parts;
    int rows, cols, n, m, np, mp;        // n, m: the smaller and the larger; np, mp: rounded up
    float keep, rate;
    int first;                           // workgroup
    int parts_n;
};
static_assert(sizeof(Matrix) <= 112, "kernel arguments");
struct Table {
    Matrix t[kMaxTensors - 6];
    int count;
    float mu;
    int nesterov;
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");

__device__ __forceinline__ const Matrix& find(const Table& tab, int wg) {
    int lo = 0, hi = tab.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.t[mid].first <= wg) lo = mid; else hi = mid;
    }
    return tab.t[lo];
}

__device__ __forceinline__ void halves(float v, f16& hi, f16& lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// ------------------------------------------------------------------------------------------------------ norms, operands

// Momentum, and sums of squares.
template <typename T> __global__ __launch_bounds__(kThreads) void orth_norms(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    const int part = blockIdx.x - t.first;
    const int64_t n = (int64_t)t.rows * t.cols;
    const T* g = static_cast<const T*>(t.update);
    double sum = 0.0;
    for (int64_t i = (int64_t)part * kThreads + threadIdx.x; i < n; i += (int64_t)t.parts_n * kThreads) {
        float u = (float)g[i];
        if (t.momentum) {
            const float m = fmaf(tab.mu, t.momentum[i], (1.f - tab.mu) * u);
            t.momentum[i] = m;
            u = tab.nesterov ? fmaf(tab.mu, m, (1.f - tab.mu) * u) : m;
        }
        sum += (double)u * (double)u;
    }
    __shared__ double waves[kThreads / kWave];
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) t.parts[part] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

// X and its transpose, tiles of 64 x 64 of the update.
template <typename T> __global__ __launch_bounds__(kThreads) void orth_operands(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    const int tiles_c = ceil_div(t.cols, 64), tile = blockIdx.x - t.first, r0 = tile / tiles_c * 64, c0 = tile % tiles_c * 64;
    __shared__ float values[64][65];
    __shared__ double total[kThreads / kWave];
    double sum = 0.0;
    for (int i = threadIdx.x; i < t.parts_n; i += kThreads) sum += t.parts[i];
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) total[threadIdx.x >> 6] = sum;
    __syncthreads();
    const double norm = sqrt((total[0] + total[1]) + (total[2] + total[3]));
    const float scale = (float)((double)kScaleX / (norm < kLeastNorm ? kLeastNorm : norm));
    const T* g = static_cast<const T*>(t.update);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r < 64; r += 4) {
        const int row = r0 + r, col = c0 + lane;
        float u = 0.f;
        if (row < t.rows && col < t.cols) {
            const int64_t i = (int64_t)row * t.cols + col;
            u = (float)g[i];
            if (t.momentum) u = tab.nesterov ? fmaf(tab.mu, t.momentum[i], (1.f - tab.mu) * u) : t.momentum[i];
        }
        values[r][lane] = u * scale;
    }
    __syncthreads();
    // the matrix as it lies is X, or its transpose
    const bool wide = t.rows <= t.cols;
    const auto store = [&](f16* to, int row, int col, int rows, int stride, int64_t half, float v) {
        if (row >= rows || col >= stride) return;
        f16 hi, lo;
        halves(v, hi, lo);
        to[(int64_t)row * stride + col] = hi;
        to[half + (int64_t)row * stride + col] = lo;
    };
    const int64_t half_x = (int64_t)t.n * t.mp, half_xt = (int64_t)t.m * t.np;
    for (int r = wave; r < 64; r += 4) {
        if (wide) {
            store(t.x, r0 + r, c0 + lane, t.n, t.mp, half_x, values[r][lane]);
            store(t.xt, c0 + r, r0 + lane, t.m, t.np, half_xt, values[lane][r]);
        } else {
            store(t.xt, r0 + r, c0 + lane, t.m, t.np, half_xt, values[r][lane]);
            store(t.x, c0 + r, r0 + lane, t.n, t.mp, half_x, values[lane][r]);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ products

enum Kind { kGram, kFactor, kUpdate, kLast };

// C[i][j] = sum_k P[i][k] Q[j][k]: P = Q = X, P = Q = A, and P = B, Q = X^T.
template <typename T, int KIND> __global__ __launch_bounds__(kThreads, 2) void orth_product(Table tab) {
    constexpr int kStride = kStep + 8;
    const Matrix& t = find(tab, blockIdx.x);
    constexpr bool kSymmetric = KIND == kGram || KIND == kFactor;
    const f16* p = KIND == kGram ? t.x : (KIND == kFactor ? t.a : t.b);
    const f16* q = KIND == kGram ? t.x : (KIND == kFactor ? t.a : t.xt);
    const int rows_p = t.n, rows_q = kSymmetric ? t.n : t.m, k_all = KIND == kGram ? t.mp : t.np;
    const int64_t half_p = (int64_t)rows_p * k_all, half_q = (int64_t)rows_q * k_all;
    int tile = blockIdx.x - t.first, ti = 0, tj = 0;
    if (kSymmetric) {
        while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        const int tiles_j = ceil_div(rows_q, kTile);
        ti = tile / tiles_j;
        tj = tile % tiles_j;
    }
    const int i0 = ti * kTile, j0 = tj * kTile;
    __shared__ __align__(16) f16 sp[2][kTile * kStride], sq[2][kTile * kStride];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave & 1, wj = wave >> 1;
    // a thread loads 16 halves of a row
    const int row = threadIdx.x >> 1, at = (threadIdx.x & 1) * 16;
    const f16* from_p = p + (int64_t)min(i0 + row, rows_p - 1) * k_all + at;
    const f16* from_q = q + (int64_t)min(j0 + row, rows_q - 1) * k_all + at;
    f16x8 in[8];
    const auto fetch = [&](int k) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                in[h * 4 + c] = *reinterpret_cast<const f16x8*>(from_p + h * half_p + k + c * 8);
                in[h * 4 + 2 + c] = *reinterpret_cast<const f16x8*>(from_q + h * half_q + k + c * 8);
            }
    };
    acc_t acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
    fetch(0);
    for (int k = 0; k < k_all; k += kStep) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                *reinterpret_cast<f16x8*>(&sp[h][row * kStride + at + c * 8]) = in[h * 4 + c];
                *reinterpret_cast<f16x8*>(&sq[h][row * kStride + at + c * 8]) = in[h * 4 + 2 + c];
            }
        __syncthreads();
        if (k + kStep < k_all) fetch(k + kStep);
        f16x8 fq[2][4];
        const int from = (lane & 15) * kStride + (lane >> 4) * 8;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 4; j++) fq[h][j] = *reinterpret_cast<const f16x8*>(&sq[h][(wj * 64 + j * 16) * kStride + from]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f16x8 hi = *reinterpret_cast<const f16x8*>(&sp[0][(wi * 64 + i * 16) * kStride + from]);
            const f16x8 lo = *reinterpret_cast<const f16x8*>(&sp[1][(wi * 64 + i * 16) * kStride + from]);
#if __HIP_DEVICE_COMPILE__
#pragma unroll
            for (int j = 0; j < 4; j++) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, fq[1][j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, fq[0][j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, fq[0][j], acc[i][j], 0, 0, 0);
            }
#endif
        }
    }
    // what becomes of a tile
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int ci = i0 + wi * 64 + i * 16 + 4 * (lane >> 4) + r, cj = j0 + wj * 64 + j * 16 + (lane & 15);
                const float c = acc[i][j][r];
                if (ci >= t.n) continue;
                f16 hi, lo;
                if (kSymmetric) {
                    if (cj > ci) continue;
                    const int64_t half = (int64_t)t.n * t.np, here = (int64_t)ci * t.np + cj, there = (int64_t)cj * t.np + ci;
                    f16* to = KIND == kGram ? t.a : t.b;
                    float v;
                    if (KIND == kGram) {
                        v = c * (kScaleA / (kScaleX * kScaleX));
                    } else {
                        const float a = (float)t.a[here] + (float)t.a[half + here];
                        v = fmaf(kC * (kScaleB / (kScaleA * kScaleA)), c, kB * (kScaleB / kScaleA) * a);
                    }
                    halves(v, hi, lo);
                    to[here] = hi;
                    to[half + here] = lo;
                    to[there] = hi;
                    to[half + there] = lo;
                } else {
                    if (cj >= t.m) continue;
                    const int64_t half_x = (int64_t)t.n * t.mp, here = (int64_t)ci * t.mp + cj;
                    const float x = (float)t.x[here] + (float)t.x[half_x + here];
                    const float v = fmaf(kA, x, c * (1.f / kScaleB));
                    if (KIND == kUpdate) {
                        const int64_t half_xt = (int64_t)t.m * t.np, there = (int64_t)cj * t.np + ci;
                        halves(v, hi, lo);
                        t.x[here] = hi;
                        t.x[half_x + here] = lo;
                        t.xt_next[there] = hi;
                        t.xt_next[half_xt + there] = lo;
                    } else {
                        const int64_t out = t.rows <= t.cols ? (int64_t)ci * t.cols + cj : (int64_t)cj * t.cols + ci;
                        T* to = static_cast<T*>(t.result) + out;
                        const float o = v * (1.f / kScaleX);
                        *to = t.momentum ? (T)fmaf(-t.rate, o, (float)*to * t.keep) : (T)o;
                    }
                }
            }
}

// No iterations: X itself.
template <typename T> __global__ __launch_bounds__(kThreads) void orth_copy(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    const int64_t n = (int64_t)t.rows * t.cols, i = (int64_t)(blockIdx.x - t.first) * kThreads + threadIdx.x;
    if (i >= n) return;
    const int r = (int)(i / t.cols), c = (int)(i % t.cols);
    const int64_t at = t.rows <= t.cols ? (int64_t)r * t.mp + c : (int64_t)c * t.mp + r;
    const float o = ((float)t.x[at] + (float)t.x[(int64_t)t.n * t.mp + at]) * (1.f / kScaleX);
    T* to = static_cast<T*>(t.result) + i;
    *to = t.momentum ? (T)fmaf(-t.rate, o, (float)*to * t.keep) : (T)o;
}

// Columns behind the last, which the products run over: zeros.
__global__ __launch_bounds__(kThreads) void orth_pads(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    const int row = (blockIdx.x - t.first) * kThreads + threadIdx.x;
    const auto clear = [&](f16* p, int rows, int cols, int stride) {
        if (row >= rows) return;
        for (int h = 0; h < 2; h++)
            for (int c = cols; c < stride; c++) p[(int64_t)h * rows * stride + (int64_t)row * stride + c] = (f16)0.f;
    };
    clear(t.x, t.n, t.m, t.mp);
    clear(t.xt, t.m, t.n, t.np);
    clear(t.xt_next, t.m, t.n, t.np);
    clear(t.a, t.n, t.n, t.np);
    clear(t.b, t.n, t.n, t.np);
}

// ---------------------------------------------------------------------------------------------------------------- host

template <typename N> N round_up(N n, int to) { return (n + to - 1) / to * to; }

struct Places {
    size_t x, xt, xt_next, a, b, parts, all;
    int n, m, np, mp, parts_n;
    explicit Places(const i6orth_tensor& t) {
        n = t.rows < t.cols ? t.rows : t.cols;
        m = t.rows < t.cols ? t.cols : t.rows;
        np = round_up(n, kRowPad);
        mp = round_up(m, kRowPad);
        const int64_t values = (int64_t)n * m, groups = ceil_div(values, (int64_t)kThreads * 16);
        parts_n = (int)(groups < kParts ? groups : kParts);
        const size_t sx = align256((size_t)2 * n * mp * sizeof(f16)), sxt = align256((size_t)2 * m * np * sizeof(f16)), sa = align256((size_t)2 * n * np * sizeof(f16));
        x = 0;
        xt = x + sx;
        xt_next = xt + sxt;
        a = xt_next + sxt;
        b = a + sa;
        parts = b + sa;
        all = parts + align256(kParts * sizeof(double));
    }
};

int checked(const i6orth_tensor* tensors, int n, int dtype) {
    if (n < 0 || (n > 0 && !tensors) || !valid_dtype(dtype)) return I6TRAIN_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < n; i++) {
        const i6orth_tensor& t = tensors[i];
        if (t.rows < 0 || t.cols < 0) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (t.rows == 0 || t.cols == 0) continue;
        if (!t.update || !t.result || (t.momentum == nullptr) != (tensors[0].momentum == nullptr)) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (t.rows > 32768 || t.cols > 32768) return I6TRAIN_ERR_TOO_LARGE;
    }
    return I6TRAIN_OK;
}

// A launch over all matrices of a table, `groups` workgroups for each.
template <typename Groups, typename Launch> int over(Table& tab, Groups groups, Launch launch) {
    int64_t all = 0;
    for (int i = 0; i < tab.count; i++) {
        tab.t[i].first = (int)all;
        all += groups(tab.t[i]);
    }
    if (!launchable(all, kThreads)) return I6TRAIN_ERR_TOO_LARGE;
    launch(dim3((unsigned)all));
    return launched();
}

template <typename T> int run(Table& tab, int iterations, hipStream_t s) {
    const dim3 threads(kThreads);
    const auto tiles = [](int n) { return ceil_div(n, kTile); };
    const auto triangle = [&](const Matrix& t) { return (int64_t)tiles(t.n) * (tiles(t.n) + 1) / 2; };
    const auto all_tiles = [&](const Matrix& t) { return (int64_t)tiles(t.n) * tiles(t.m); };
    I6TRAIN_TRY(over(tab, [](const Matrix& t) { return (int64_t)t.parts_n; }, [&](dim3 g) { orth_norms<T><<<g, threads, 0, s>>>(tab); }));
    I6TRAIN_TRY(over(tab, [](const Matrix& t) { return (int64_t)ceil_div(t.m, kThreads); }, [&](dim3 g) { orth_pads<<<g, threads, 0, s>>>(tab); }));
    I6TRAIN_TRY(over(tab, [](const Matrix& t) { return (int64_t)ceil_div(t.rows, 64) * ceil_div(t.cols, 64); }, [&](dim3 g) { orth_operands<T><<<g, threads, 0, s>>>(tab); }));
    if (iterations == 0)
        return over(tab, [](const Matrix& t) { return ceil_div((int64_t)t.rows * t.cols, (int64_t)kThreads); }, [&](dim3 g) { orth_copy<T><<<g, threads, 0, s>>>(tab); });
    for (int i = 0; i < iterations; i++) {
        I6TRAIN_TRY(over(tab, triangle, [&](dim3 g) { orth_product<T, kGram><<<g, threads, 0, s>>>(tab); }));
        I6TRAIN_TRY(over(tab, triangle, [&](dim3 g) { orth_product<T, kFactor><<<g, threads, 0, s>>>(tab); }));
        if (i + 1 < iterations) I6TRAIN_TRY(over(tab, all_tiles, [&](dim3 g) { orth_product<T, kUpdate><<<g, threads, 0, s>>>(tab); }));
        else I6TRAIN_TRY(over(tab, all_tiles, [&](dim3 g) { orth_product<T, kLast><<<g, threads, 0, s>>>(tab); }));
        for (int j = 0; j < tab.count; j++) {
            f16* xt = tab.t[j].xt;
            tab.t[j].xt = tab.t[j].xt_next;
            tab.t[j].xt_next = xt;
        }
    }
    return I6TRAIN_OK;
}

}  // namespace
}  // namespace i6train

using namespace i6train;

extern "C" {

int i6orth_workspace_size(const i6orth_tensor* tensors, int n_tensors, int dtype, size_t* bytes) {
    I6TRAIN_TRY(checked(tensors, n_tensors, dtype));
    if (!bytes) return I6TRAIN_ERR_INVALID_ARGUMENT;
    size_t all = 0;
    for (int i = 0; i < n_tensors; i++)
        if (tensors[i].rows > 0 && tensors[i].cols > 0) all += Places(tensors[i]).all;
    *bytes = all;
    return I6TRAIN_OK;
}

int i6orth_step(const i6orth_tensor* tensors, int n_tensors, int dtype, int iterations, double mu, int nesterov, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    I6TRAIN_TRY(i6orth_workspace_size(tensors, n_tensors, dtype, &need));
    if (iterations < 0 || !(mu >= 0 && mu < 1)) return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (need == 0) return I6TRAIN_OK;
    if (!workspace || workspace_bytes < need) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    char* at = static_cast<char*>(workspace);
    Table tab;
    tab.count = 0;
    tab.mu = (float)mu;
    tab.nesterov = nesterov;
    const auto flush = [&]() {
        if (tab.count == 0) return I6TRAIN_OK;
        const int rc = dtype == I6TRAIN_BF16 ? run<bf16>(tab, iterations, (hipStream_t)stream) : run<float>(tab, iterations, (hipStream_t)stream);
        tab.count = 0;
        return rc;
    };
    for (int i = 0; i < n_tensors; i++) {
        const i6orth_tensor& t = tensors[i];
        if (t.rows == 0 || t.cols == 0) continue;
        if (tab.count == (int)(sizeof(tab.t) / sizeof(tab.t[0]))) I6TRAIN_TRY(flush());
        const Places p(t);
        Matrix& m = tab.t[tab.count++];
        m.update = t.update; m.result = t.result; m.momentum = t.momentum;
        m.x = reinterpret_cast<f16*>(at + p.x); m.xt = reinterpret_cast<f16*>(at + p.xt); m.xt_next = reinterpret_cast<f16*>(at + p.xt_next);
        m.a = reinterpret_cast<f16*>(at + p.a); m.b = reinterpret_cast<f16*>(at + p.b);
        m.parts = reinterpret_cast<double*>(at + p.parts);
        m.rows = t.rows; m.cols = t.cols; m.n = p.n; m.m = p.m; m.np = p.np; m.mp = p.mp;
        m.keep = t.keep; m.rate = t.rate; m.parts_n = p.parts_n;
        at += p.all;
    }
    return flush();
}

}  // extern "C"
