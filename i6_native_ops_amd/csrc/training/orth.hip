// Orthogonal factors of matrices by Newton-Schulz products, and the optimiser's step on them (include/i6orth.h).
//
// X has n rows and m >= n columns.  An iteration is three products for all matrices of the call, a launch each:  A = X X^T,
// B = a + b A + c A A,  X = B X.  A and B are symmetric: of the first two only the tiles on and below the diagonal are formed, and written to both
// places.  X is kept as it is and transposed, so that both operands of every product have consecutive k.
//
// Operands are two 16-bit floating-point halves, x = x1 + x2, of 22 bits, times a power of two that brings the largest value they can have (X: 1.21, A: 1.46,
// B: 3.45) below 2^16; of (x1 + x2)(y1 + y2) the last term is below the precision.  Half the bits would do for the products, but not for what becomes of them: an error in A is one of
// left singular vectors of all sizes, and the small ones grow 3.4 times in each iteration, 485 times in five.
//
// 24 matrices of 4096 x 2048 in 16 bits: 19.1 - 19.4 ms, of which 0.46 norms and operands, 4 x 2.18 + 1.19 X = B X, 5 x 1.14 A, 5 x 0.69 B: 20 TFLOP of 16-bit products at 1040 TFLOP/s, where
// the library's product of 8192 x 8192 reaches 1135 on such values; both are bound by the matrix units and the clock that the card holds under them (1.96 - 2.15 GHz).  With the step
// on momenta and parameters 19.9 ms.
#include <algorithm>
#include <cmath>

#include "lds_loads.h"
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
constexpr int kMaxTensors = 34;          // x 112 bytes: the arguments of a kernel may have 4 KB
// Of a table's workspace, unless one matrix alone has more.  More at once is no faster: of 4096 x 2048 in 16 bits 24 matrices take 19.3 ms, 12 of them 9.7; of 4096 x 11008 24 take 185, 6 of them 46.
constexpr size_t kTableBytes = (size_t)4 << 30;
constexpr int kThreads = 256;
constexpr int kRowPad = 64;               // of columns: what the products run over
constexpr int kCus = 256;
constexpr double kSmallRound = 0.62;     // of tiles of 128 x 128, two a unit, to one of 256 x 256
constexpr int kPartSteps = 16;
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
    Matrix t[kMaxTensors];
    int count, groups;
    int quarters;                        // of the tiles of 256 x 256 from this one on; -1: tiles of the kernel's own size
    int parts;                           // of the columns that a product runs over, where tiles are few
    acc_t* partial;                      // [tiles][parts][a tile's accumulators]
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

// Where a value's first half is in a matrix of `stride` columns; the second one is 32 places behind.  32 first and 32 second halves in turn are 128 bytes, what a stage
// takes of a row.
__device__ __forceinline__ int64_t place(int row, int col, int stride) { return (int64_t)row * 2 * stride + (col >> 5) * 64 + (col & 31); }

__device__ __forceinline__ void halves(float v, f16& hi, f16& lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// ------------------------------------------------------------------------------------------------------ norms, operands

// The sum over a workgroup, in all its threads; `waves` is room in LDS.
template <int N> __device__ __forceinline__ double sum_of_all(double sum, double* waves) {
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < N / kWave; i++) sum += waves[i];
    return sum;
}

// N values of a row side by side, in one load if `whole`; zeros behind the last.
template <typename T, int N> __device__ __forceinline__ void load_some(float (&v)[N], const T* p, int64_t left, bool whole) {
    using P = T __attribute__((ext_vector_type(N)));
    if (whole && left >= N) {
        const P x = *reinterpret_cast<const P*>(p);
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = (float)x[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = e < left ? (float)p[e] : 0.f;
}

// Momentum, and the sum of the squares of a thread's share: pieces of 8 values from `first` on.
template <typename T> __device__ __forceinline__ double squares_of(const Matrix& t, float mu, bool nesterov, int64_t first, int64_t step) {
    const int64_t n = (int64_t)t.rows * t.cols;
    const T* g = static_cast<const T*>(t.update);
    const bool whole = (uintptr_t)g % 16 == 0, whole_m = (uintptr_t)t.momentum % 16 == 0;
    double sum = 0.0;
    for (int64_t i = first * 8; i < n; i += step * 8) {
        float u[8], m[8];
        load_some(u, g + i, n - i, whole);
        if (t.momentum) {
            load_some(m, t.momentum + i, n - i, whole_m);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                m[e] = fmaf(mu, m[e], (1.f - mu) * u[e]);
                u[e] = nesterov ? fmaf(mu, m[e], (1.f - mu) * u[e]) : m[e];
            }
            if (whole_m && n - i >= 8) {
                *reinterpret_cast<acc_t*>(t.momentum + i) = acc_t{m[0], m[1], m[2], m[3]};
                *reinterpret_cast<acc_t*>(t.momentum + i + 4) = acc_t{m[4], m[5], m[6], m[7]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (e < n - i) t.momentum[i + e] = m[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) sum += (double)u[e] * (double)u[e];
    }
    return sum;
}

template <typename T> __global__ __launch_bounds__(kThreads) void orth_norms(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    __shared__ double waves[kThreads / kWave];
    const int part = blockIdx.x - t.first;
    const double sum = sum_of_all<kThreads>(squares_of<T>(t, tab.mu, tab.nesterov, (int64_t)part * kThreads + threadIdx.x, (int64_t)t.parts_n * kThreads), waves);
    if (threadIdx.x == 0) t.parts[part] = sum;
}

// X and its transpose: a tile of 64 x 64 of the update, from row r0 and column c0 on.
using Turned = float[64][65];
template <typename T> __device__ __forceinline__ void operands_of(const Matrix& t, float mu, bool nesterov, double sum, int r0, int c0, Turned& values) {
    const double norm = sqrt(sum);
    const float scale = (float)((double)kScaleX / (norm < kLeastNorm ? kLeastNorm : norm));
    const T* g = static_cast<const T*>(t.update);
    const bool whole = (uintptr_t)g % 16 == 0 && t.cols % 8 == 0, whole_m = (uintptr_t)t.momentum % 16 == 0 && t.cols % 8 == 0;
    for (int i = threadIdx.x; i < 64 * 8; i += kThreads) {
        const int r = i >> 3, c = (i & 7) * 8, row = r0 + r, col = c0 + c;
        const int64_t at = (int64_t)row * t.cols + col, left = row < t.rows ? t.cols - col : 0;
        float u[8], m[8];
        load_some(u, g + (left > 0 ? at : 0), left, whole);
        if (t.momentum) {
            load_some(m, t.momentum + (left > 0 ? at : 0), left, whole_m);
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = nesterov ? fmaf(mu, m[e], (1.f - mu) * u[e]) : m[e];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) values[r][c + e] = u[e] * scale;
    }
    __syncthreads();
    // the matrix as it lies is X, or its transpose; behind the last column there are zeros
    const bool wide = t.rows <= t.cols;
    const auto store = [&](f16* to, int rows, int stride, int row0, int col0, bool turned) {
        for (int i = threadIdx.x; i < 64 * 8; i += kThreads) {
            const int r = i >> 3, c = (i & 7) * 8, row = row0 + r, col = col0 + c;
            if (row >= rows || col >= stride) continue;
            f16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f16 h, l;
                halves(turned ? values[c + e][r] : values[r][c + e], h, l);
                hi[e] = h;
                lo[e] = l;
            }
            f16* at = to + place(row, col, stride);
            *reinterpret_cast<f16x8*>(at) = hi;
            *reinterpret_cast<f16x8*>(at + 32) = lo;
        }
    };
    store(wide ? t.x : t.xt, t.rows, wide ? t.mp : t.np, r0, c0, false);
    store(wide ? t.xt : t.x, t.cols, wide ? t.np : t.mp, c0, r0, true);
}

template <typename T> __global__ __launch_bounds__(kThreads) void orth_operands(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    const int tiles_c = ceil_div(t.cols, 64), tile = blockIdx.x - t.first;
    __shared__ Turned values;
    __shared__ double waves[kThreads / kWave];
    double sum = 0.0;
    for (int i = threadIdx.x; i < t.parts_n; i += kThreads) sum += t.parts[i];
    operands_of<T>(t, tab.mu, tab.nesterov, sum_of_all<kThreads>(sum, waves), tile / tiles_c * 64, tile % tiles_c * 64, values);
}

// ------------------------------------------------------------------------------------------------------------ products

enum Kind { kGram, kFactor, kUpdate, kLast };

// Few tiles of long products: parts of the columns by workgroups of their own, kPart, whose sums kJoin adds up in their order.
enum Mode { kWhole, kPart, kJoin };
// Halves of the operands that a product takes: the first ones alone; both, without the product of the second ones; all four products.
constexpr int kOne = 1, kThree = 2, kFour = 3;

// The packed halves of a value, and four of them side by side.
__device__ __forceinline__ uint32_t packed(float v) {
    f16 hi, lo;
    halves(v, hi, lo);
    return (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
}

// C[i][j] = sum_k P[i][k] Q[j][k]: P = Q = X, P = Q = A, and P = B, Q = X^T.  Tiles of 32 S x 32 S, four waves with 16 S x 16 S each.  A stage has of every row 128 bytes:
// 32 k, first and second halves (kHalves = 2), or the first halves of 64 k.  In LDS a row's eight pieces of 16 bytes are turned by the row, so that eight lanes that read
// eight rows' pieces reach all banks; the loads, which write LDS in order, take them from the turned places.
template <typename T, int KIND, int S, int kHalves, Mode MODE> __device__ __forceinline__ void product_of(const Matrix& t, int ti, int tj, char* lds, int parts, int part, acc_t* partial) {
    constexpr int kTile = 32 * S, kSide = kTile * 128, kStage = 2 * kSide, kLoads = S;       // per wave, stage and operand
    constexpr bool kSymmetric = KIND == kGram || KIND == kFactor;
    constexpr int kStep = kHalves == kOne ? 64 : 32;
    const f16* p = KIND == kGram ? t.x : (KIND == kFactor ? t.a : t.b);
    const f16* q = KIND == kGram ? t.x : (KIND == kFactor ? t.a : t.xt);
    const int rows_q = kSymmetric ? t.n : t.m, k_all = KIND == kGram ? t.mp : t.np;
    const int i0 = ti * kTile, j0 = tj * kTile;
    const int lane = threadIdx.x & 63, wave = wave_index(), wi = wave & 1, wj = wave >> 1;

    const int64_t row_bytes = (int64_t)k_all * 4;
    const descriptor from_p = describe(reinterpret_cast<const char*>(p) + i0 * row_bytes, min(t.n - i0, kTile) * row_bytes);
    const descriptor from_q = describe(reinterpret_cast<const char*>(q) + j0 * row_bytes, min(rows_q - j0, kTile) * row_bytes);
    uint32_t from;                       // of the lane's piece: 8 rows a load
    {
        const int row = wave * kLoads * 8 + (lane >> 3), piece = (lane & 7) ^ (lane >> 3);
        from = (uint32_t)(row * row_bytes) + (kHalves == kOne ? (piece >> 2) * 128 + (piece & 3) * 16 : piece * 16);
    }
    const uint32_t lds0 = lds_address(lds) + wave * kLoads * 1024, eight_rows = (uint32_t)(8 * row_bytes);
    const auto fetch = [&](int i, int stage, uint32_t offset) {
        const uint32_t to = lds0 + stage * kStage + (i & 1) * kSide + (i >> 1) * 1024;
        load_to_lds(i & 1 ? from_q : from_p, to, from + (i >> 1) * eight_rows, offset);
    };
    constexpr uint32_t kStepBytes = kHalves == kOne ? 256 : 128;
    acc_t acc[S][S];
#pragma unroll
    for (int i = 0; i < S; i++)
#pragma unroll
        for (int j = 0; j < S; j++) acc[i][j] = 0.f;
    const int steps = k_all / kStep, per = MODE == kPart ? ceil_div(steps, parts) : steps, begin = MODE == kPart ? min(part * per, steps) : 0, end = min(begin + per, steps);
    if (MODE != kJoin && begin < end) {
#pragma unroll
        for (int i = 0; i < 2 * kLoads; i++) fetch(i, 0, (uint32_t)begin * kStepBytes);
    }
    // fragments: the lane's row, and pieces 0 .. 3 and 4 .. 7
    const uint32_t read0 = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16), read1 = read0 ^ 64;
    for (int k = 0; MODE != kJoin && k < end - begin; k++) {
        wait_and_meet<0>();
        const char* sp = lds + (k & 1) * kStage + wi * (16 * S * 128);
        const char* sq = lds + (k & 1) * kStage + kSide + wj * (16 * S * 128);
        f16x8 fq[2][S], fp[2][2];
#pragma unroll
        for (int j = 0; j < S; j++) {
            fq[0][j] = *reinterpret_cast<const f16x8*>(sq + read0 + j * 2048);
            fq[1][j] = *reinterpret_cast<const f16x8*>(sq + read1 + j * 2048);
        }
        fp[0][0] = *reinterpret_cast<const f16x8*>(sp + read0);
        fp[0][1] = *reinterpret_cast<const f16x8*>(sp + read1);
        const uint32_t offset = (uint32_t)(begin + k + 1) * kStepBytes;
        const bool more = k + 1 < end - begin;
#pragma unroll
        for (int i = 0; i < S; i++) {
            if (i + 1 < S) {
                fp[(i + 1) & 1][0] = *reinterpret_cast<const f16x8*>(sp + read0 + (i + 1) * 2048);
                fp[(i + 1) & 1][1] = *reinterpret_cast<const f16x8*>(sp + read1 + (i + 1) * 2048);
            }
            if (more) {
                fetch(2 * i, (k + 1) & 1, offset);
                fetch(2 * i + 1, (k + 1) & 1, offset);
            }
            const f16x8 p0 = fp[i & 1][0], p1 = fp[i & 1][1];
#if __HIP_DEVICE_COMPILE__
            if (kHalves != kOne) {
                if (kHalves == kFour) {
#pragma unroll
                    for (int j = 0; j < S; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p1, fq[1][j], acc[i][j], 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < S; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p0, fq[1][j], acc[i][j], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < S; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p1, fq[0][j], acc[i][j], 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < S; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p1, fq[1][j], acc[i][j], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < S; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p0, fq[0][j], acc[i][j], 0, 0, 0);
#endif
        }
    }
    if (MODE != kWhole) {
        constexpr int kTileSums = 4 * S * S * 64;
        acc_t* mine = partial + (MODE == kPart ? (int64_t)part * kTileSums : 0) + wave * S * S * 64 + lane;
#pragma unroll 2
        for (int x = 0; x < (MODE == kPart ? 1 : parts); x++)
#pragma unroll
            for (int i = 0; i < S; i++)
#pragma unroll
                for (int j = 0; j < S; j++) {
                    acc_t* at = mine + (int64_t)x * kTileSums + (i * S + j) * 64;
                    if (MODE == kPart) *at = acc[i][j];
                    else acc[i][j] += *at;
                }
        if (MODE == kPart) return;
    }
    // What becomes of a tile: 64 of a wave's rows at a time go through LDS, from where lanes take eight values side by side, of rows and of columns.  A row's words are turned by
    // its number, so that neither way two lanes meet in a bank.
    const int at = 4 * (lane >> 4), ci0 = i0 + wi * 16 * S, cj0 = j0 + wj * 16 * S;
    const bool wide = t.rows <= t.cols, whole = t.cols % 8 == 0 && (uintptr_t)t.result % 16 == 0;
    constexpr int kWidth = 16 * S;
    uint32_t* mine = reinterpret_cast<uint32_t*>(lds) + wave * 64 * kWidth;
    const auto turn = [](int r) { return ((r >> 3 & 7) << 3) ^ ((r >> 2 & 3) << 4); };
    // halves of eight packed words
    const auto store_halves = [&](f16* to, const uint32_t (&w)[8]) {
        const auto first = [&](int i) { return __builtin_amdgcn_perm(w[i + 1], w[i], 0x05040100); };
        const auto second = [&](int i) { return __builtin_amdgcn_perm(w[i + 1], w[i], 0x07060302); };
        *reinterpret_cast<uint4*>(to) = make_uint4(first(0), first(2), first(4), first(6));
        *reinterpret_cast<uint4*>(to + 32) = make_uint4(second(0), second(2), second(4), second(6));
    };
    const auto store_result = [&](int r, int c, const uint32_t (&w)[8]) {
        if (r >= t.rows || c >= t.cols) return;
        T* to = static_cast<T*>(t.result) + (int64_t)r * t.cols + c;
        const int left = t.cols - c;
        float was[8];
        if (t.momentum) {
            load_some(was, to, left, whole);
#pragma unroll
            for (int e = 0; e < 8; e++) was[e] = fmaf(-t.rate, __uint_as_float(w[e]), was[e] * t.keep);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) was[e] = __uint_as_float(w[e]);
        }
        if (whole) {
            using T8 = T __attribute__((ext_vector_type(8)));
            T8 v;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (T)was[e];
            *reinterpret_cast<T8*>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < left) to[e] = (T)was[e];
        }
    };
    wait_and_meet<0>();
#pragma unroll
    for (int strip = 0; strip < S / 4; strip++) {
#pragma unroll
        for (int i4 = 0; i4 < 4; i4++) {
            const int i = strip * 4 + i4, ci = ci0 + i * 16 + at;
#pragma unroll
            for (int j = 0; j < S; j++) {
                const int cj = cj0 + j * 16 + (lane & 15);
                const bool there = cj < rows_q && ci < t.np;
                acc_t v = acc[i][j];
                if (KIND == kGram) v *= kScaleA / (kScaleX * kScaleX);
                if (KIND == kFactor) {   // A is symmetric: a lane's four rows of a column are four columns of a row
                    const f16* own = t.a + place(there ? cj : 0, there ? ci : 0, t.np);
                    const acc_t x = __builtin_convertvector(*reinterpret_cast<const f16x4*>(own), acc_t) + __builtin_convertvector(*reinterpret_cast<const f16x4*>(own + 32), acc_t);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        v[e] = fmaf(kC * (kScaleB / (kScaleA * kScaleA)), v[e], kB * (kScaleB / kScaleA) * x[e]);
                        if (ci + e == cj) v[e] += kA * kScaleB;
                    }
                }
                if (KIND == kUpdate) v *= 1.f / kScaleB;
                if (KIND == kLast) v *= 1.f / (kScaleB * kScaleX);
                const int turned = (j * 16 + (lane & 15)) ^ turn(i4 * 16 + at);
#pragma unroll
                for (int e = 0; e < 4; e++) mine[(i4 * 16 + at + e) * kWidth + turned] = KIND == kLast ? __float_as_uint(v[e]) : (there && ci + e < t.n ? packed(v[e]) : 0);
            }
        }
        asm volatile("" ::: "memory");   // a wave's own part of LDS, which it reads in the order of its writes
        if (KIND != kLast || wide) {
            const int stride = kSymmetric ? t.np : t.mp;
            f16* out = KIND == kGram ? t.a : (KIND == kFactor ? t.b : t.x);
#pragma unroll 4
            for (int x = lane; x < 64 * (kWidth / 8); x += 64) {
                const int r = x / (kWidth / 8), c = x % (kWidth / 8) * 8, ci = ci0 + strip * 64 + r, cj = cj0 + c;
                const uint4* from = reinterpret_cast<const uint4*>(mine + r * kWidth + (c ^ turn(r)));
                const uint4 u = from[0], v = from[1];
                const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                if (KIND == kLast) store_result(ci, cj, w);
                else if (ci < t.n && cj < stride) store_halves(out + place(ci, cj, stride), w);
            }
        }
        if (KIND == kLast ? !wide : !kSymmetric || ti != tj) {
            f16* out = KIND == kGram ? t.a : (KIND == kFactor ? t.b : t.xt_next);
#pragma unroll 4
            for (int x = lane; x < 8 * kWidth; x += 64) {
                const int r = x >> 3, c = (x & 7) * 8, cj = cj0 + r, ci = ci0 + strip * 64 + c;
                const uint32_t *from0 = mine + c * kWidth + (r ^ turn(c)), *from1 = mine + (c + 4) * kWidth + (r ^ turn(c + 4));
                const uint32_t w[8] = {from0[0], from0[kWidth], from0[2 * kWidth], from0[3 * kWidth], from1[0], from1[kWidth], from1[2 * kWidth], from1[3 * kWidth]};
                if (KIND == kLast) store_result(cj, ci, w);
                else if (cj < rows_q && ci < t.np) store_halves(out + place(cj, ci, t.np), w);
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
}

constexpr int stages_bytes(int S) { return 2 * 2 * 32 * S * 128; }
template <typename T, int KIND, int S, int kHalves, Mode MODE> __global__ __launch_bounds__(kThreads, S == 8 ? 1 : 2) void orth_product(Table tab) {
    constexpr int kTile = 32 * S;
    __shared__ __align__(128) char lds[stages_bytes(S)];
    // neighbours in the order of the tiles go to the same eighth of the card, which has a cache of its own
    const int per = ceil_div(tab.groups, 8), wg = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (wg >= tab.groups) return;
    const bool quarter = S == 4 && MODE == kWhole && tab.quarters >= 0;
    const int number = quarter ? tab.quarters + wg / 4 : (MODE == kPart ? wg / tab.parts : wg), side = quarter ? 256 : kTile;
    const Matrix& t = find(tab, number);
    int tile = number - t.first, ti = 0, tj = 0;
    if (KIND == kGram || KIND == kFactor) {
        while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
        tj = tile - ti * (ti + 1) / 2;
    } else {                             // four rows of tiles side by side
        const int tiles_i = ceil_div(t.n, side), tiles_j = ceil_div(t.m, side), four_rows = tile / (4 * tiles_j), high = min(4, tiles_i - 4 * four_rows);
        tile -= four_rows * 4 * tiles_j;
        ti = 4 * four_rows + tile % high;
        tj = tile / high;
    }
    if (quarter) {
        ti = 2 * ti + (wg >> 1 & 1);
        tj = 2 * tj + (wg & 1);
        if (KIND == kGram || KIND == kFactor ? tj > ti || ti * kTile >= t.n : ti * kTile >= t.n || tj * kTile >= t.m) return;
    }
    product_of<T, KIND, S, kHalves, MODE>(t, ti, tj, lds, tab.parts, MODE == kPart ? wg % tab.parts : 0, tab.partial + (int64_t)number * tab.parts * (4 * S * S * 64));
}

// Small matrices: a workgroup does all of it for one, X and A (then B) in LDS.  A wave has sixteen rows of X, or a part of their columns, in 32 bits in its registers.
// All four products of the halves: short sums have little error of their own beside that of the last one, and matrix instructions are not what is waited for.
// What bounds it are the waits of a chain of products that has 15 links: two matrices of 128 x 64 take 40 us.
constexpr int kSmallThreads = 512, kSmallBytes = 140 * 1024, kSmallTiles = 8;
__host__ __device__ constexpr int small_parts(int n) { return n <= 16 ? 8 : (n <= 32 ? 4 : (n <= 64 ? 2 : 1)); }     // waves of sixteen rows
__host__ __device__ constexpr int up32(int n) { return (n + 31) / 32 * 32; }
constexpr bool is_small(int n, int m) {
    return n <= 128 && (m + 15) / 16 <= kSmallTiles * small_parts(n) && (int64_t)up32(n) * (up32(m) + 8 + up32(n) + 8) * 4 <= kSmallBytes;
}

// Operands of sixteen rows and 32 k, first or second halves: a lane has k = 4 (lane >> 4) .. + 3 and 16 more.
__device__ __forceinline__ f16x8 two(f16x4 a, f16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ f16x8 rows_of(const f16* p, int stride, int row0, int k0, int lane) {
    const f16* at = p + (row0 + (lane & 15)) * stride + k0 + 4 * (lane >> 4);
    return two(*reinterpret_cast<const f16x4*>(at), *reinterpret_cast<const f16x4*>(at + 16));
}
__device__ __forceinline__ f16x8 columns_of(const f16* p, int stride, int col0, int k0, int lane) {     // reads that turn 4 rows x 16 columns within 16 lanes
    f16x8 r = {};
#if __HIP_DEVICE_COMPILE__
    using s16x4 = short __attribute__((ext_vector_type(4)));
    using P = __attribute__((address_space(3))) s16x4*;
    const f16* at = p + (k0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * stride + col0 + 4 * (lane & 3);
    r = two(__builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)at)), __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 16 * stride))));
#endif
    return r;
}
// The lane, of which the compiler does not know that it is the same as before: addresses are formed where they are used, or those of all tiles fill the registers.
__device__ __forceinline__ int this_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}
__device__ __forceinline__ acc_t multiplied(f16x8 a, f16x8 b, acc_t c) {
#if __HIP_DEVICE_COMPILE__
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#endif
    return c;
}

template <typename T> __global__ __launch_bounds__(kSmallThreads) void orth_small(Table tab, int iterations) {
    __shared__ __align__(16) f16 room[kSmallBytes / 2];
    __shared__ double waves[kSmallThreads / kWave];
    const Matrix& t = tab.t[blockIdx.x];
    const int n32 = up32(t.n), m32 = up32(t.m), sx = m32 + 8, sa = n32 + 8, plane_x = n32 * sx, plane_a = n32 * sa;
    f16* x = room;
    f16* a = room + 2 * plane_x;
    for (int i = threadIdx.x; i < (plane_x + plane_a) / 4; i += kSmallThreads) reinterpret_cast<uint4*>(room)[i] = make_uint4(0, 0, 0, 0);
    const double norm = sqrt(sum_of_all<kSmallThreads>(squares_of<T>(t, tab.mu, tab.nesterov, threadIdx.x, kSmallThreads), waves));
    const float scale = (float)((double)kScaleX / (norm < kLeastNorm ? kLeastNorm : norm));
    const bool wide = t.rows <= t.cols;
    const T* g = static_cast<const T*>(t.update);
    for (int i = threadIdx.x; i < t.rows * t.cols; i += kSmallThreads) {
        const int r = i / t.cols, c = i - r * t.cols, at = wide ? r * sx + c : c * sx + r;
        float u = (float)g[i];
        if (t.momentum) u = tab.nesterov ? fmaf(tab.mu, t.momentum[i], (1.f - tab.mu) * u) : t.momentum[i];
        halves(u * scale, x[at], x[plane_x + at]);
    }
    __syncthreads();
    const int wave = wave_index();
    int lane = this_lane(), at = 4 * (lane >> 4), own = lane & 15;
    const int parts = small_parts(t.n), row0 = wave / parts * 16, part = wave % parts, tiles_n = ceil_div(t.n, 16), tiles_m = ceil_div(t.m, 16);
    const bool mine = row0 < t.n;
    constexpr int kA16 = 8;
    acc_t xr[kSmallTiles], ar[kA16];
    const acc_t none = 0.f;
#pragma unroll
    for (int i = 0; i < kSmallTiles; i++) {
        xr[i] = none;
        const int j = part + parts * i;
        if (mine && j < tiles_m) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f16* from = x + (row0 + at + e) * sx + 16 * j + own;
                xr[i][e] = (float)from[0] + (float)from[plane_x];
            }
        }
    }
    // X X^T or A A: rows by rows
    const auto square = [&](const f16* p, int stride, int plane, int k_all, auto take) {
        acc_t hi[kA16], lo[kA16];
#pragma unroll
        for (int i = 0; i < kA16; i++) hi[i] = lo[i] = none;
        if (mine)
            for (int k = 0; k < k_all; k += 32) {
                const int lane = this_lane();
                const f16x8 p0 = rows_of(p, stride, row0, k, lane), p1 = rows_of(p + plane, stride, row0, k, lane);
#pragma unroll
                for (int i = 0; i < kA16; i++) {
                    const int j = part + parts * i;
                    if (j >= tiles_n) continue;
                    const f16x8 q0 = rows_of(p, stride, 16 * j, k, lane), q1 = rows_of(p + plane, stride, 16 * j, k, lane);
                    hi[i] = multiplied(p0, q0, hi[i]);
                    lo[i] = multiplied(p1, q0, multiplied(p0, q1, multiplied(p1, q1, lo[i])));
                }
            }
#pragma unroll
        for (int i = 0; i < kA16; i++) ar[i] = take(hi[i] + lo[i], ar[i]);
    };
    const auto store_square = [&]() {    // both are symmetric: a lane's four rows of a column are four columns of a row
        if (!mine) return;
        const int lane = this_lane(), at = 4 * (lane >> 4), own = lane & 15;
#pragma unroll
        for (int i = 0; i < kA16; i++) {
            const int j = part + parts * i;
            if (j >= tiles_n) continue;
            f16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                f16 h, l;
                halves(ar[i][e], h, l);
                hi[e] = h;
                lo[e] = l;
            }
            f16* to = a + (16 * j + own) * sa + row0 + at;
            *reinterpret_cast<f16x4*>(to) = hi;
            *reinterpret_cast<f16x4*>(to + plane_a) = lo;
        }
    };
    for (int it = 0; it < iterations; it++) {
        square(x, sx, plane_x, m32, [&](acc_t v, acc_t) { return v * (kScaleA / (kScaleX * kScaleX)); });
        store_square();
        __syncthreads();
        square(a, sa, plane_a, n32, [&](acc_t v, acc_t was) { return v * (kC * (kScaleB / (kScaleA * kScaleA))) + was * (kB * (kScaleB / kScaleA)); });
        __syncthreads();
        store_square();
        __syncthreads();
        acc_t v[kSmallTiles];
#pragma unroll
        for (int i = 0; i < kSmallTiles; i++) v[i] = none;
        if (mine)
            for (int k = 0; k < n32; k += 32) {
                const int lane = this_lane();
                const f16x8 p0 = rows_of(a, sa, row0, k, lane), p1 = rows_of(a + plane_a, sa, row0, k, lane);
#pragma unroll
                for (int i = 0; i < kSmallTiles; i++) {
                    const int j = part + parts * i;
                    if (j >= tiles_m) continue;
                    const f16x8 q0 = columns_of(x, sx, 16 * j, k, lane), q1 = columns_of(x + plane_x, sx, 16 * j, k, lane);
                    v[i] = multiplied(p0, q0, multiplied(p1, q0, multiplied(p0, q1, multiplied(p1, q1, v[i]))));
                }
            }
        __syncthreads();
        const bool last = it + 1 == iterations;
        lane = this_lane();
        at = 4 * (lane >> 4);
        own = lane & 15;
#pragma unroll
        for (int i = 0; i < kSmallTiles; i++) {
            const int j = part + parts * i, cj = 16 * j + own;
            if (!mine || j >= tiles_m) continue;
            xr[i] = xr[i] * kA + v[i] * (1.f / kScaleB);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int ci = row0 + at + e;
                if (!last) {
                    f16* to = x + ci * sx + cj;
                    halves(xr[i][e], to[0], to[plane_x]);
                } else if (ci < t.n && cj < t.m) {
                    const float o = xr[i][e] * (1.f / kScaleX);
                    T* to = static_cast<T*>(t.result) + (wide ? ci * t.cols + cj : cj * t.cols + ci);
                    *to = t.momentum ? (T)fmaf(-t.rate, o, (float)*to * t.keep) : (T)o;
                }
            }
        }
        __syncthreads();
    }
}

// No iterations: X itself.
template <typename T> __global__ __launch_bounds__(kThreads) void orth_copy(Table tab) {
    const Matrix& t = find(tab, blockIdx.x);
    const int64_t n = (int64_t)t.rows * t.cols, i = (int64_t)(blockIdx.x - t.first) * kThreads + threadIdx.x;
    if (i >= n) return;
    const int r = (int)(i / t.cols), c = (int)(i % t.cols);
    const f16* x = t.rows <= t.cols ? t.x + place(r, c, t.mp) : t.x + place(c, r, t.mp);
    const float o = ((float)x[0] + (float)x[32]) * (1.f / kScaleX);
    T* to = static_cast<T*>(t.result) + i;
    *to = t.momentum ? (T)fmaf(-t.rate, o, (float)*to * t.keep) : (T)o;
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
    const i6orth_tensor* first = nullptr;        // of those that have values; the others' pointers mean nothing
    for (int i = 0; i < n; i++) {
        const i6orth_tensor& t = tensors[i];
        if (t.rows < 0 || t.cols < 0) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (t.rows == 0 || t.cols == 0) continue;
        if (!first) first = &t;
        if (!t.update || !t.result || (t.momentum == nullptr) != (first->momentum == nullptr)) return I6TRAIN_ERR_INVALID_ARGUMENT;
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

// Tiles that do not fill the card: how many parts of its columns a product is formed in.  A step takes 0.8 us, a part's sums are read in half of that, another launch takes 7: so no
// parts below 16 steps of 32 columns, four steps at least in each, and about the root of their number of them.  Without and with, in 32 bits: one matrix of 200 x 4096 656 -> 308 us,
// of 1024 x 1024 497 -> 404, 8 of 60 x 2000 332 -> 212.  Sums in parts are also nearer: with all four products 3.0e-6 -> 1.4e-6 off 64 bits in the last of these.
struct Parts {
    bool few;
    int parts;
    size_t bytes;
};
Parts parts_of(const Table& tab, bool gram, bool symmetric) {
    int64_t tiles = 0;
    int steps = 0;
    for (int i = 0; i < tab.count; i++) {
        const Matrix& t = tab.t[i];
        const int64_t r = ceil_div(t.n, 128);
        tiles += symmetric ? r * (r + 1) / 2 : r * ceil_div(t.m, 128);
        steps = std::max(steps, (gram ? t.mp : t.np) / 32);
    }
    Parts p{tiles > 0 && tiles <= kCus, 1, 0};
    if (p.few && steps >= kPartSteps) p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({2 * kCus / tiles, steps / 4, (int64_t)sqrt(1.6 * steps)}));
    if (p.parts > 1) p.bytes = (size_t)tiles * p.parts * 128 * 128 * sizeof(float);
    return p;
}

// A product over all matrices.  Tiles of 256 x 256 keep the matrix units busier, one workgroup a unit; tiles of 128 x 128, two a unit, waste less of small matrices and of the
// last round.  So there are whole rounds of large tiles, and the rest is large ones or their quarters; or all tiles are small.  A round of small tiles takes 0.62 of one of large
// ones (2048 columns: 89 us and 146).
template <typename T, int KIND, int kHalves> int multiply(Table& tab, hipStream_t s) {
    constexpr bool kSymmetric = KIND == kGram || KIND == kFactor;
    const auto tiles = [](const Matrix& t, int side) {
        const int64_t i = ceil_div(t.n, side);
        return kSymmetric ? i * (i + 1) / 2 : i * ceil_div(t.m, side);
    };
    const Parts split = parts_of(tab, KIND == kGram, kSymmetric);
    if (split.few) {                     // all four products: matrix instructions are not what is waited for, and short sums have little error beside that of the last one
        constexpr int kAll = kHalves == kOne ? kOne : kFour;
        tab.quarters = -1;
        tab.parts = split.parts;
        return over(tab, [&](const Matrix& t) { return tiles(t, 128); }, [&](dim3 g) {
            const auto grid = [](unsigned n) { return dim3(ceil_div(n, 8u) * 8); };
            if (split.parts > 1) {
                tab.groups = (int)g.x * split.parts;
                orth_product<T, KIND, 4, kAll, kPart><<<grid(tab.groups), dim3(kThreads), 0, s>>>(tab);
            }
            tab.groups = (int)g.x;
            if (split.parts > 1) orth_product<T, KIND, 4, kAll, kJoin><<<grid(g.x), dim3(kThreads), 0, s>>>(tab);
            else orth_product<T, KIND, 4, kAll, kWhole><<<grid(g.x), dim3(kThreads), 0, s>>>(tab);
        });
    }
    int64_t large = 0, small = 0;
    for (int i = 0; i < tab.count; i++) {
        large += tiles(tab.t[i], 256);
        small += tiles(tab.t[i], 128);
    }
    const auto small_rounds = [](int64_t n) { return kSmallRound * (double)ceil_div(n, (int64_t)(2 * kCus)); };
    const int64_t rounds = large / kCus, rest = large - rounds * kCus;
    const double with_quarters = (double)rounds + small_rounds(rest * 4), all_large = (double)ceil_div(large, (int64_t)kCus);
    const auto launch_large = [&](int64_t n) {
        tab.groups = (int)n;
        tab.quarters = -1;
        orth_product<T, KIND, 8, kHalves, kWhole><<<dim3((unsigned)(ceil_div(n, (int64_t)8) * 8)), dim3(kThreads), 0, s>>>(tab);
    };
    const auto launch_small = [&](int64_t n, int64_t quarters) {
        tab.groups = (int)n;
        tab.quarters = (int)quarters;
        orth_product<T, KIND, 4, kHalves, kWhole><<<dim3((unsigned)(ceil_div(n, (int64_t)8) * 8)), dim3(kThreads), 0, s>>>(tab);
    };
    if (small_rounds(small) < std::min(with_quarters, all_large)) return over(tab, [&](const Matrix& t) { return tiles(t, 128); }, [&](dim3 g) { launch_small(g.x, -1); });
    return over(tab, [&](const Matrix& t) { return tiles(t, 256); }, [&](dim3) {
        if (all_large <= with_quarters) return launch_large(large);
        if (rounds) launch_large(rounds * kCus);
        launch_small(rest * 4, rounds * kCus);
    });
}

template <typename T> int run(Table& tab, bool small, int iterations, hipStream_t s) {
    const dim3 threads(kThreads);
    if (small) {
        orth_small<T><<<dim3(tab.count), dim3(kSmallThreads), 0, s>>>(tab, iterations);
        return launched();
    }
    I6TRAIN_TRY(over(tab, [](const Matrix& t) { return (int64_t)t.parts_n; }, [&](dim3 g) { orth_norms<T><<<g, threads, 0, s>>>(tab); }));
    I6TRAIN_TRY(over(tab, [](const Matrix& t) { return (int64_t)ceil_div(t.rows, 64) * ceil_div(t.cols, 64); }, [&](dim3 g) { orth_operands<T><<<g, threads, 0, s>>>(tab); }));
    if (iterations == 0)
        return over(tab, [](const Matrix& t) { return ceil_div((int64_t)t.rows * t.cols, (int64_t)kThreads); }, [&](dim3 g) { orth_copy<T><<<g, threads, 0, s>>>(tab); });
    for (int i = 0; i < iterations; i++) {
        I6TRAIN_TRY((multiply<T, kGram, kThree>(tab, s)));
        I6TRAIN_TRY((multiply<T, kFactor, kThree>(tab, s)));
        // 16-bit results: nothing follows in which an error of the last product grows.  Half the bits of B's and X's values change what the result is off by from 1.66e-3 (its
        // rounding alone) to 1.69e-3, relative 2-norm, and the product takes 1.16 ms instead of 1.98 (24 matrices of 4096 x 2048).
        if (i + 1 < iterations) I6TRAIN_TRY((multiply<T, kUpdate, kThree>(tab, s)));
        else I6TRAIN_TRY((multiply<T, kLast, sizeof(T) == 2 ? kOne : kThree>(tab, s)));
        for (int j = 0; j < tab.count; j++) {
            f16* xt = tab.t[j].xt;
            tab.t[j].xt = tab.t[j].xt_next;
            tab.t[j].xt_next = xt;
        }
    }
    return I6TRAIN_OK;
}

// What all matrices of a table share.
size_t shared_bytes(const Table& tab) { return std::max(parts_of(tab, true, true).bytes, std::max(parts_of(tab, false, true).bytes, parts_of(tab, false, false).bytes)); }

// f(table, small, bytes) for the matrices of a call, as many at once as a table has room for and kTableBytes hold; bytes are those of the workspace that they have of their own, from its
// start on: one table follows the other on the stream, and small matrices need none.  Which way a matrix goes depends on it alone.
template <typename F> int in_tables(const i6orth_tensor* tensors, int n_tensors, int iterations, char* workspace, F f) {
    Table tab{};
    for (const bool small : {true, false}) {
        size_t own = 0;
        const auto flush = [&]() {
            if (tab.count == 0) return I6TRAIN_OK;
            const int rc = f(tab, small, own);
            tab.count = 0;
            own = 0;
            return rc;
        };
        for (int i = 0; i < n_tensors; i++) {
            const i6orth_tensor& t = tensors[i];
            if (t.rows == 0 || t.cols == 0) continue;
            const Places p(t);
            if (small != (iterations > 0 && is_small(p.n, p.m))) continue;
            const size_t more = small ? 0 : p.all;
            if (tab.count == kMaxTensors || (tab.count > 0 && own + more > kTableBytes)) I6TRAIN_TRY(flush());
            char* at = workspace + own;
            Matrix& m = tab.t[tab.count++];
            m.update = t.update; m.result = t.result; m.momentum = t.momentum;
            m.x = reinterpret_cast<f16*>(at + p.x); m.xt = reinterpret_cast<f16*>(at + p.xt); m.xt_next = reinterpret_cast<f16*>(at + p.xt_next);
            m.a = reinterpret_cast<f16*>(at + p.a); m.b = reinterpret_cast<f16*>(at + p.b);
            m.parts = reinterpret_cast<double*>(at + p.parts);
            m.rows = t.rows; m.cols = t.cols; m.n = p.n; m.m = p.m; m.np = p.np; m.mp = p.mp;
            m.keep = t.keep; m.rate = t.rate; m.parts_n = p.parts_n;
            own += more;
        }
        I6TRAIN_TRY(flush());
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
    size_t most = 0;
    for (const int iterations : {0, 1})          // without iterations small matrices go the others' way
        I6TRAIN_TRY(in_tables(tensors, n_tensors, iterations, nullptr, [&](Table& tab, bool small, size_t own) {
            most = std::max(most, own + (small || iterations == 0 ? 0 : align256(shared_bytes(tab))));
            return I6TRAIN_OK;
        }));
    *bytes = most;
    return I6TRAIN_OK;
}

int i6orth_step(const i6orth_tensor* tensors, int n_tensors, int dtype, int iterations, double mu, int nesterov, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    I6TRAIN_TRY(i6orth_workspace_size(tensors, n_tensors, dtype, &need));
    if (iterations < 0 || !(mu >= 0 && mu < 1)) return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (need == 0) return I6TRAIN_OK;
    if (!workspace || workspace_bytes < need) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    return in_tables(tensors, n_tensors, iterations, static_cast<char*>(workspace), [&](Table& tab, bool small, size_t own) {
        tab.mu = (float)mu;
        tab.nesterov = nesterov;
        tab.partial = reinterpret_cast<acc_t*>(static_cast<char*>(workspace) + own);
        return dtype == I6TRAIN_BF16 ? run<bf16>(tab, small, iterations, (hipStream_t)stream) : run<float>(tab, small, iterations, (hipStream_t)stream);
    });
}

}  // extern "C"
