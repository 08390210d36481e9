// Output layer and frame-wise cross entropy without the logits (include/i6train.h).
//
//   forward    z = W h + b in tiles, in registers; per tile and frame the maximum and the sum of exp(z - maximum), joined over
//              the tiles afterwards;  loss = log sum exp z - z_y
//   backward   for one piece of the vocabulary after another: z again, G = g (softmax(z) - [f = y]) rounded to the operands'
//              precision, then  dh += G W  and  dW = G^T h
//
// All three products run through one kernel, product(): C[m][n] = sum_k A[m][k] B[n][k] on the matrix units, both operands with
// consecutive k, which differs in what becomes of a finished tile.  So that k is consecutive, G is written in both layouts, and h
// and W are transposed once per backward call.
//
// The frames of a batch are packed first: only frames that belong to a sequence are rows of the products, and what the others
// hold is not read.  How many there are is known on the device alone: tiles behind the last row return at once.
//
// 32-bit operands.  The matrix units have 16-bit operands at sixteen times the rate of 32-bit ones.  A value x is split into x1 = f16(s x)
// and x2 = f16(2^11 (s x - x1)), s a power of two that brings the tensor's largest value to 2^14..2^15: 22 bits down to 2^-29 of the largest
// value.  Of (x1 + x2 2^-11)(y1 + y2 2^-11) the last term is below the precision and left out: the k-loop runs over x1 y2 and x2 y1,
// scales the accumulators by 2^-11, and goes on with x1 y1.
#include <cmath>

#include "train_common.h"

namespace i6train {
namespace {

constexpr int kTile = 128;           // rows and columns of a workgroup's tile
constexpr int kStep = 64;            // k of one turn: 128 bytes of a row
constexpr int kThreads = 256;
constexpr float kLow = 0x1p-11f;     // weight of the second half of a 32-bit value

template <typename T> struct Frag;
template <> struct Frag<bf16> { using type = bf16 __attribute__((ext_vector_type(8))); };
template <> struct Frag<f16> { using type = f16 __attribute__((ext_vector_type(8))); };
using acc_t = float __attribute__((ext_vector_type(16)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ acc_t mfma(Frag<bf16>::type a, Frag<bf16>::type b, acc_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ acc_t mfma(Frag<f16>::type a, Frag<f16>::type b, acc_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// What the kernels tell each other: at the start of the forward workspace.
struct Header {
    int rows;                 // frames that belong to a sequence
    uint32_t most_x, most_w;  // largest finite magnitudes, as bit patterns (32-bit operands)
};
struct BackHeader {
    uint32_t most_g;
};

// The power of two that brings `most` to 2^14 .. 2^15, and its inverse.
__device__ __forceinline__ int scale_exponent(uint32_t most) {
    if (most == 0) return 0;
    const int e = (int)(most >> 23) - 127;         // (subnormals: -127)
    const int k = 14 - e;
    return k > 100 ? 100 : k;
}

// ------------------------------------------------------------------------------------------------------------- rows

// offsets[b]: the first row of sequence b.  One workgroup.
__global__ __launch_bounds__(1024) void ce_begin(const int32_t* lens, int B, int T, int* offsets, Header* header) {
    __shared__ int sums[16];
    __shared__ int carry;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    for (int base = 0; base < B; base += 1024) {
        const int b = base + threadIdx.x;
        int n = b < B ? lens[b] : 0;
        n = n < 0 ? 0 : (n > T ? T : n);
        int sum = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        if (lane == 63) sums[wave] = sum;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < wave; w++) before += sums[w];
        if (b < B) offsets[b] = before + sum - n;
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + sum;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        header->rows = carry;
        header->most_x = 0;
        header->most_w = 0;
    }
}

__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ void most_of(uint32_t m, uint32_t* to) {
    for (int d = 32; d; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
        m = o > m ? o : m;
    }
    if ((threadIdx.x & 63) == 0 && m) atomicMax(to, m);       // a maximum: the order does not matter
}

__device__ __forceinline__ bool has_target(int y, int classes) { return y >= 0 && y < classes; }

// Largest magnitude of a matrix of floats; `lens`: its rows are frames (b, t), and those without a target do not count.
__global__ __launch_bounds__(256) void ce_most(const float* x, int64_t stride_b, int64_t stride_t, int64_t rows, int T, int D, const int32_t* lens, const int32_t* targets,
                                               int64_t tgt_b, int64_t tgt_t, int classes, uint32_t* most) {
    uint32_t m = 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        const int64_t b = r / T, t = r % T;
        if (lens && (t >= lens[b] || !has_target(targets[b * tgt_b + t * tgt_t], classes))) continue;
        const float* row = x + b * stride_b + t * stride_t;
        for (int d = threadIdx.x & 63; d < D; d += 64) {
            const uint32_t v = finite_bits(row[d]);
            m = v > m ? v : m;
        }
    }
    most_of(m, most);
}

// x as one 16-bit value or two.
__device__ __forceinline__ void split(float x, int exponent, f16& high, f16& low) {
    const float s = ldexpf(x, exponent);
    high = (f16)s;
    low = fabsf(s) < 65504.f ? (f16)((s - (float)high) * 0x1p11f) : (f16)0.f;       // infinities and NaN are in the first half alone
}

// Frames and weights as operands: [row][halves][Kp], zeros behind column D.
struct PackArgs {
    const void* x;  int64_t stride_b, stride_t;
    int64_t rows;  int T, D, Kp, classes;
    const int32_t *lens, *offsets, *targets;  int64_t tgt_b, tgt_t;      // null for weights
    const uint32_t* most;
    void* out;
    int *row_frame, *row_target;
    float* loss;
};

template <typename In, typename T>
__global__ __launch_bounds__(256) void ce_pack(PackArgs a) {
    constexpr int S = sizeof(In) == 4 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int exponent = S == 2 ? scale_exponent(*a.most) : 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * 4) {
        const int64_t b = r / a.T, t = r % a.T;
        int64_t row = r;
        bool used = true;
        if (a.lens) {
            if (t >= a.lens[b]) {
                if (lane == 0) a.loss[r] = 0.f;
                continue;
            }
            row = a.offsets[b] + t;
            const int target = a.targets[b * a.tgt_b + t * a.tgt_t];
            used = has_target(target, a.classes);      // a frame without a target: zeros, whatever it holds
            if (lane == 0) {
                a.row_frame[row] = (int)r;
                a.row_target[row] = target;
            }
        }
        const In* x = static_cast<const In*>(a.x) + b * a.stride_b + t * a.stride_t;
        T* out = static_cast<T*>(a.out) + row * (S * (int64_t)a.Kp);
        for (int d = lane; d < a.Kp; d += 64) {
            if constexpr (S == 2) {
                f16 high = (f16)0.f, low = (f16)0.f;
                if (used && d < a.D) split(x[d], exponent, high, low);
                out[d] = high;
                out[a.Kp + d] = low;
            } else {
                out[d] = used && d < a.D ? x[d] : (T)0.f;
            }
        }
    }
}

// out[h][c][r] = in[r][h][c] for 16-bit values, rows r < *n_rows (or `rows`); zeros up to Rp.  Tiles of 64 x 64.
struct TransposeArgs {
    const uint16_t* in;  int64_t row_stride, half_stride;
    int rows;  const int* n_rows;  int cols;
    uint16_t* out;  int64_t col_stride, out_half;       // of the transposed matrix
};
__global__ __launch_bounds__(256) void ce_transpose(TransposeArgs a) {
    __shared__ uint16_t tile[64][66];
    const int rows = a.n_rows ? *a.n_rows : a.rows;
    const int64_t r0 = (int64_t)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64, half = blockIdx.z;
    if (r0 >= ceil_div(rows, 64) * (int64_t)64) return;
    const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
    for (int i = y; i < 64; i += 4) {
        const int64_t r = r0 + i;
        const int c = c0 + x;
        tile[i][x] = r < rows && c < a.cols ? a.in[r * a.row_stride + half * a.half_stride + c] : (uint16_t)0;
    }
    __syncthreads();
    for (int i = y; i < 64; i += 4) {
        const int c = c0 + i;
        if (c < a.cols) a.out[c * a.col_stride + half * a.out_half + r0 + x] = tile[x][i];
    }
}

// ---------------------------------------------------------------------------------------------------------- product

struct Operand {
    const void* p;
    int64_t row_stride;       // elements
    int64_t half_stride;      // elements to the second halves
    int rows;                 // rows that may be read
    const int* n_rows;        // if they are known on the device alone
};
struct ProductArgs {
    Operand a, b;
    int K;                    // of one half; multiple of kStep
    const int* n_k;           // K = n_k rounded up to kStep, where it is known on the device alone
    int splits;               // blockIdx.z takes one of so many ranges of k
};

enum Kind { kStatistics, kGradient, kStore };

struct EpilogueArgs {
    // kStatistics, kGradient: m is the class, n the row (frame)
    const void* bias;  int bias_f32;
    const Header* header;  const BackHeader* back;
    int first_class, classes;              // of this piece; classes of the layer
    const int* row_target;
    float2* part;  float* target_logit;    // [tile of classes][rows_p], [rows_p]
    int64_t rows_p;
    const float *lse, *row_scale;
    void* g;  int64_t g_stride, g_half;    // [row][halves][piece]
    void* gt;  int64_t gt_stride, gt_half; // [class][halves][rows_p]
    // kStore: m, n as they are; float [split][m][n]
    float* out;  int64_t out_stride, out_split;
    int add;
};

template <typename T, int KIND>
__global__ __launch_bounds__(kThreads) void product(ProductArgs p, EpilogueArgs e) {
    constexpr int S = sizeof(T) == 2 && __is_same(T, f16) ? 2 : 1;
    using F = typename Frag<T>::type;
    __shared__ u32x4 lds[2][kTile * kStep / 8];              // A and B: rows of 8 chunks of 16 bytes, chunk c of row r at place c ^ (r & 7)
    __shared__ float join[2][2][kTile];

    const int rows_a = p.a.n_rows ? *p.a.n_rows : p.a.rows, rows_b = p.b.n_rows ? *p.b.n_rows : p.b.rows;
    const int m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
    if (m0 >= rows_a || n0 >= rows_b) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave & 1, wn = wave >> 1;
    int K = p.n_k ? ceil_div(*p.n_k, kStep) * kStep : p.K;
    int k0 = 0;
    if (p.splits > 1) {
        const int each = ceil_div(ceil_div(K, kStep), p.splits) * kStep;
        k0 = min(K, (int)blockIdx.z * each);
        K = min(K, k0 + each);
    }

    acc_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;

    // rows behind the last are the last one again: read, and never stored
    const T *pa[4], *pb[4];
    int place[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int at = i * kThreads + tid, r = at >> 3, c = at & 7;
        pa[i] = static_cast<const T*>(p.a.p) + (int64_t)min(m0 + r, rows_a - 1) * p.a.row_stride + c * 8;
        pb[i] = static_cast<const T*>(p.b.p) + (int64_t)min(n0 + r, rows_b - 1) * p.b.row_stride + c * 8;
        place[i] = r * 8 + (c ^ (r & 7));
    }
    const auto segment = [&](int64_t off_a, int64_t off_b) {
        for (int k = k0; k < K; k += kStep) {
            u32x4 ra[4], rb[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ra[i] = *reinterpret_cast<const u32x4*>(pa[i] + off_a + k);
                rb[i] = *reinterpret_cast<const u32x4*>(pb[i] + off_b + k);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                lds[0][place[i]] = ra[i];
                lds[1][place[i]] = rb[i];
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < kStep / 16; kk++) {
                F fa[2], fb[2];
                const int c = kk * 2 + (lane >> 5);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int rm = wm * 64 + i * 32 + (lane & 31), rn = wn * 64 + i * 32 + (lane & 31);
                    fa[i] = __builtin_bit_cast(F, lds[0][rm * 8 + (c ^ (rm & 7))]);
                    fb[i] = __builtin_bit_cast(F, lds[1][rn * 8 + (c ^ (rn & 7))]);
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) acc[i][j] = mfma(fa[i], fb[j], acc[i][j]);
            }
        }
    };
    if constexpr (S == 2) {
        segment(0, p.b.half_stride);
        segment(p.a.half_stride, 0);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] *= kLow;
    }
    segment(0, 0);

    // register r of a 32 x 32 block: row (r & 3) + 8 (r >> 2) + 4 (lane >> 5), column lane & 31
    const int row_in = 4 * (lane >> 5), col_in = lane & 31;

    if constexpr (KIND == kStore) {
        float* out = e.out + (int64_t)blockIdx.z * e.out_split;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int n = n0 + wn * 64 + j * 32 + col_in;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int m = m0 + wm * 64 + i * 32 + row_in + (r & 3) + 8 * (r >> 2);
                    if (m < rows_a && n < rows_b) {
                        float* at = out + (int64_t)m * e.out_stride + n;
                        *at = e.add ? *at + acc[i][j][r] : acc[i][j][r];
                    }
                }
            }
        return;
    }

    // logits: the scales of 32-bit operands go, the bias comes
    const int down = S == 2 ? -(scale_exponent(e.header->most_x)) : 0, down_w = S == 2 ? -(scale_exponent(e.header->most_w)) : 0;
    const int classes = min(e.classes - e.first_class, rows_a);
    float bias[2][16];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int m = m0 + wm * 64 + i * 32 + row_in + (r & 3) + 8 * (r >> 2);
            float v = 0.f;
            if (e.bias && m < classes)
                v = e.bias_f32 ? static_cast<const float*>(e.bias)[e.first_class + m] : (float)static_cast<const bf16*>(e.bias)[e.first_class + m];
            bias[i][r] = v;
        }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float z = acc[i][j][r];
                if (S == 2) z = ldexpf(ldexpf(z, down), down_w);
                acc[i][j][r] = z + bias[i][r];
            }

    if constexpr (KIND == kStatistics) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int col = wn * 64 + j * 32 + col_in, n = n0 + col;
            const int target = n < rows_b ? e.row_target[n] : -1;
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int m = m0 + wm * 64 + i * 32 + row_in + (r & 3) + 8 * (r >> 2);
                    if (m >= classes) acc[i][j][r] = -INFINITY;
                    else if (e.first_class + m == target) e.target_logit[n] = acc[i][j][r];
                    most = fmaxf(most, acc[i][j][r]);
                }
            most = fmaxf(most, __shfl_xor(most, 32));
            const float base = most == -INFINITY ? 0.f : most;        // a tile of classes that are all -inf: the sum is 0, not NaN
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) sum += exp2_fast((acc[i][j][r] - base) * kLog2e);
            sum += __shfl_xor(sum, 32);
            if (lane < 32) {
                join[wm][0][col] = most;
                join[wm][1][col] = sum;
            }
        }
        __syncthreads();
        if (tid < kTile && n0 + tid < rows_b) {
            const float ma = join[0][0][tid], mb = join[1][0][tid], most = fmaxf(ma, mb), base = most == -INFINITY ? 0.f : most;
            const float sum = join[0][1][tid] * exp2_fast((ma - base) * kLog2e) + join[1][1][tid] * exp2_fast((mb - base) * kLog2e);
            e.part[(int64_t)blockIdx.x * e.rows_p + n0 + tid] = make_float2(most, sum);
        }
        return;
    }

    if constexpr (KIND == kGradient) {
        const int g_exponent = S == 2 ? scale_exponent(e.back->most_g) : 0;
        T* g = static_cast<T*>(e.g);
        T* gt = static_cast<T*>(e.gt);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int n = n0 + wn * 64 + j * 32 + col_in;
            const bool there = n < rows_b;
            const int target = there ? e.row_target[n] : -1;
            const float lse = there ? e.lse[n] : 0.f, scale = there ? e.row_scale[n] : 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int m = m0 + wm * 64 + i * 32 + row_in + (r & 3) + 8 * (r >> 2);
                    float v = exp2_fast((acc[i][j][r] - lse) * kLog2e) * scale;
                    if (e.first_class + m == target) v -= scale;
                    if (m >= classes || !there) v = 0.f;
                    // columns up to the end of the tile are there in both, zero behind the last class or row
                    if constexpr (S == 2) {
                        f16 high, low;
                        split(v, g_exponent, high, low);
                        if (there) {
                            g[(int64_t)n * e.g_stride + m] = high;
                            g[(int64_t)n * e.g_stride + e.g_half + m] = low;
                        }
                        if (m < classes) {
                            gt[(int64_t)m * e.gt_stride + n] = high;
                            gt[(int64_t)m * e.gt_stride + e.gt_half + n] = low;
                        }
                    } else {
                        if (there) g[(int64_t)n * e.g_stride + m] = (T)v;
                        if (m < classes) gt[(int64_t)m * e.gt_stride + n] = (T)v;
                    }
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- the rest

// Statistics of the tiles joined: loss and log sum of a row.
__global__ __launch_bounds__(256) void ce_finish(const Header* header, const float2* part, int tiles, int64_t rows_p, const int* row_frame,
                                                 const int* row_target, const float* target_logit, int T, int F, float* lse, float* loss, int* report) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= header->rows) return;
    float most = -INFINITY, sum = 0.f;
    for (int i = 0; i < tiles; i++) {
        const float2 p = part[i * rows_p + row];
        const float m = fmaxf(most, p.x), base = m == -INFINITY ? 0.f : m;
        sum = sum * exp2_fast((most - base) * kLog2e) + p.y * exp2_fast((p.x - base) * kLog2e);
        most = m;
    }
    const float l = most + log2_fast(sum) * kLn2;
    lse[row] = l;
    const int y = row_target[row], frame = row_frame[row];
    float v = 0.f;
    if (y >= 0 && y < F) {
        v = l - target_logit[row];
    } else if (y >= F) {
        v = __builtin_nanf("");
        if (report) {
            __hip_atomic_store(report + 1, frame / T, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            __hip_atomic_store(report, I6TRAIN_ERR_BAD_TARGET, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
        }
    }
    loss[frame] = v;
}

__global__ void ce_clear(BackHeader* back) { back->most_g = 0; }

// The incoming gradient of each row; rows without a target, or with one that is out of range, have none.
__global__ __launch_bounds__(256) void ce_row_scale(const Header* header, const int* row_frame, const int* row_target, const float* grad_loss, int64_t stride_b,
                                                    int64_t stride_t, int T, int F, float* row_scale, uint32_t* most) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    float g = 0.f;
    if (row < header->rows) {
        const int frame = row_frame[row], y = row_target[row];
        if (y >= 0 && y < F) g = grad_loss[(int64_t)(frame / T) * stride_b + (int64_t)(frame % T) * stride_t];
        row_scale[row] = g;
    }
    most_of(finite_bits(g), most);
}

// grad_hidden: rows back to their frames.
template <typename Out>
__global__ __launch_bounds__(256) void ce_store_hidden(const Header* header, const BackHeader* back, const int* offsets, const int32_t* lens, const int32_t* targets,
                                                       int64_t tgt_b, int64_t tgt_t, const float* acc, int B, int T, int F, int D, Out* out) {
    const int lane = threadIdx.x & 63;
    const bool scaled = sizeof(Out) == 4;
    const int down = scaled ? -scale_exponent(back->most_g) : 0, down_w = scaled ? -scale_exponent(header->most_w) : 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < (int64_t)B * T; r += (int64_t)gridDim.x * 4) {
        const int64_t b = r / T, t = r % T;
        const bool live = t < lens[b];
        const float* row = acc + (live ? (int64_t)(offsets[b] + t) * D : 0);
        const bool bad = live && targets[b * tgt_b + t * tgt_t] >= F;
        for (int d = lane; d < D; d += 64) {
            float v = live ? row[d] : 0.f;
            if (scaled) v = ldexpf(ldexpf(v, down), down_w);
            out[r * D + d] = (Out)(bad ? __builtin_nanf("") : v);
        }
    }
}

// One piece of grad_weight: the ranges of k joined.
template <typename Out>
__global__ __launch_bounds__(256) void ce_store_weight(const Header* header, const BackHeader* back, const float* part, int splits, int64_t split_stride, int64_t n, Out* out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
    for (int s = 0; s < splits; s++) v += part[s * split_stride + i];
    if (sizeof(Out) == 4) v = ldexpf(ldexpf(v, -scale_exponent(back->most_g)), -scale_exponent(header->most_x));
    out[i] = (Out)v;
}

// grad_bias: sums over the rows.  One workgroup per class.
template <typename T, typename Out>
__global__ __launch_bounds__(256) void ce_store_bias(const Header* header, const BackHeader* back, const T* gt, int64_t stride, int64_t half, Out* out) {
    constexpr int S = sizeof(Out) == 4 ? 2 : 1;
    __shared__ float sums[4];
    const T* row = gt + blockIdx.x * stride;
    float v = 0.f;
    for (int i = threadIdx.x; i < header->rows; i += 256) {
        v += (float)row[i];
        if (S == 2) v += (float)row[half + i] * kLow;
    }
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        v = sums[0] + sums[1] + sums[2] + sums[3];
        if (S == 2) v = ldexpf(v, -scale_exponent(back->most_g));
        out[blockIdx.x] = (Out)v;
    }
}

// ------------------------------------------------------------------------------------------------------------- host

constexpr size_t kPieceBytes = (size_t)256 << 20;      // of G, both layouts: the caches in front of the memory hold 256 MB

template <typename N> N round_up(N n, N to) { return ceil_div(n, to) * to; }

// Where things are in the workspaces.
struct Layout {
    int S, Kp, row_tiles, class_tiles, piece, splits;
    int64_t rows_p;
    bool own_weight;                    // weights are copied as operands
    size_t header, offsets, row_frame, row_target, target_logit, lse, x, w, part, forward;
    size_t back, row_scale, xt, wt, g, gt, dx, dw, backward;
};

bool valid(const i6train_ce_problem* p) {
    return p && p->B > 0 && p->T > 0 && p->F > 0 && p->D > 0 && valid_dtype(p->dtype) && p->weight && p->targets && p->seq_lens;
}

int layout(const i6train_ce_problem& p, Layout& l) {
    const int64_t rows = (int64_t)p.B * p.T;
    if (rows > (1 << 22) || p.F > (1 << 22) || p.D > (1 << 16)) return I6TRAIN_ERR_TOO_LARGE;
    l.S = p.dtype == I6TRAIN_F32 ? 2 : 1;
    l.Kp = round_up(p.D, kStep);
    l.row_tiles = (int)ceil_div(rows, (int64_t)kTile);
    l.class_tiles = ceil_div(p.F, kTile);
    l.rows_p = (int64_t)l.row_tiles * kTile;
    l.own_weight = !(p.dtype == I6TRAIN_BF16 && p.D % kStep == 0 && (uintptr_t)p.weight % 16 == 0 && p.weight_stride_f % 8 == 0);
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
    l.header = take(sizeof(Header));
    l.offsets = take(4 * (size_t)p.B);
    l.row_frame = take(4 * l.rows_p);
    l.row_target = take(4 * l.rows_p);
    l.target_logit = take(4 * l.rows_p);
    l.lse = take(4 * l.rows_p);
    l.x = take((size_t)rows * l.S * l.Kp * 2);
    l.w = l.own_weight ? take((size_t)p.F * l.S * l.Kp * 2) : 0;
    l.part = take(sizeof(float2) * l.class_tiles * l.rows_p);
    l.forward = at;

    at = 0;
    int64_t piece = (int64_t)(kPieceBytes / (4 * (size_t)l.S * l.rows_p)) / kTile * kTile;
    const int64_t all = (int64_t)l.class_tiles * kTile;
    piece = piece < kTile ? kTile : (piece > all ? all : piece);
    l.piece = (int)piece;
    const int64_t tiles = piece / kTile * ceil_div(p.D, kTile);
    l.splits = (int)ceil_div((int64_t)512, tiles);
    const int most = (int)ceil_div(rows, (int64_t)512);
    if (l.splits > most) l.splits = most;
    l.back = take(sizeof(BackHeader));
    l.row_scale = take(4 * l.rows_p);
    l.xt = take((size_t)p.D * l.S * l.rows_p * 2);
    l.wt = take((size_t)p.D * l.S * all * 2);
    l.g = take((size_t)l.rows_p * l.S * piece * 2);
    l.gt = take((size_t)piece * l.S * l.rows_p * 2);
    l.dx = take(4 * (size_t)l.rows_p * p.D);
    l.dw = take(4 * (size_t)l.splits * piece * p.D);
    l.backward = at;
    return I6TRAIN_OK;
}

int groups_for(int64_t rows) { return (int)(rows < 16384 ? ceil_div(rows, (int64_t)4) : 4096); }

template <typename In, typename T>
int forward(const i6train_ce_problem& p, const Layout& l, float* loss, char* ws, hipStream_t s) {
    constexpr int S = sizeof(In) == 4 ? 2 : 1;
    const int64_t rows = (int64_t)p.B * p.T;
    Header* header = (Header*)(ws + l.header);
    int* offsets = (int*)(ws + l.offsets);
    ce_begin<<<dim3(1), dim3(1024), 0, s>>>(p.seq_lens, p.B, p.T, offsets, header);
    if (S == 2) {
        ce_most<<<dim3(groups_for(rows)), dim3(256), 0, s>>>((const float*)p.hidden, p.hidden_stride_b, p.hidden_stride_t, rows, p.T, p.D, p.seq_lens, p.targets, p.targets_stride_b,
                                                                p.targets_stride_t, p.F, &header->most_x);
        ce_most<<<dim3(groups_for(p.F)), dim3(256), 0, s>>>((const float*)p.weight, 0, p.weight_stride_f, p.F, p.F, p.D, nullptr, nullptr, 0, 0, 0, &header->most_w);
    }
    PackArgs a{};
    a.x = p.hidden; a.stride_b = p.hidden_stride_b; a.stride_t = p.hidden_stride_t;
    a.rows = rows; a.T = p.T; a.D = p.D; a.Kp = l.Kp; a.classes = p.F;
    a.lens = p.seq_lens; a.offsets = offsets; a.targets = p.targets; a.tgt_b = p.targets_stride_b; a.tgt_t = p.targets_stride_t;
    a.most = &header->most_x;
    a.out = ws + l.x; a.row_frame = (int*)(ws + l.row_frame); a.row_target = (int*)(ws + l.row_target); a.loss = loss;
    ce_pack<In, T><<<dim3(groups_for(rows)), dim3(256), 0, s>>>(a);
    if (l.own_weight) {
        PackArgs w{};
        w.x = p.weight; w.stride_t = p.weight_stride_f;
        w.rows = p.F; w.T = p.F; w.D = p.D; w.Kp = l.Kp;
        w.most = &header->most_w; w.out = ws + l.w;
        ce_pack<In, T><<<dim3(groups_for(p.F)), dim3(256), 0, s>>>(w);
    }
    const void* weight = l.own_weight ? ws + l.w : p.weight;
    const int64_t weight_stride = l.own_weight ? S * (int64_t)l.Kp : p.weight_stride_f;
    ProductArgs q{};
    q.a = {weight, weight_stride, l.Kp, p.F, nullptr};
    q.b = {ws + l.x, S * (int64_t)l.Kp, l.Kp, 0, &header->rows};
    q.K = l.Kp; q.splits = 1;
    EpilogueArgs e{};
    e.bias = p.bias; e.bias_f32 = p.dtype == I6TRAIN_F32; e.header = header; e.classes = p.F;
    e.row_target = (int*)(ws + l.row_target); e.part = (float2*)(ws + l.part); e.target_logit = (float*)(ws + l.target_logit); e.rows_p = l.rows_p;
    product<T, kStatistics><<<dim3(l.class_tiles, l.row_tiles), dim3(kThreads), 0, s>>>(q, e);
    ce_finish<<<dim3(ceil_div(rows, (int64_t)256)), dim3(256), 0, s>>>(header, e.part, l.class_tiles, l.rows_p, (int*)(ws + l.row_frame), e.row_target, e.target_logit, p.T, p.F,
                                                                       (float*)(ws + l.lse), loss, status_slot());
    return launched();
}

template <typename In, typename T>
int backward(const i6train_ce_problem& p, const Layout& l, const float* grad_loss, int64_t gs_b, int64_t gs_t, void* grad_hidden, void* grad_weight, void* grad_bias,
             const char* fw, char* ws, hipStream_t s) {
    constexpr int S = sizeof(In) == 4 ? 2 : 1;
    const int64_t rows = (int64_t)p.B * p.T;
    const Header* header = (const Header*)(fw + l.header);
    BackHeader* back = (BackHeader*)(ws + l.back);
    const int* row_target = (const int*)(fw + l.row_target);
    float* row_scale = (float*)(ws + l.row_scale);
    const int64_t all = (int64_t)l.class_tiles * kTile;
    ce_clear<<<dim3(1), dim3(1), 0, s>>>(back);
    ce_row_scale<<<dim3(ceil_div(rows, (int64_t)256)), dim3(256), 0, s>>>(header, (const int*)(fw + l.row_frame), row_target, grad_loss, gs_b, gs_t, p.T, p.F, row_scale, &back->most_g);
    const void* weight = l.own_weight ? fw + l.w : p.weight;
    const int64_t weight_stride = l.own_weight ? S * (int64_t)l.Kp : p.weight_stride_f;
    TransposeArgs x{(const uint16_t*)(fw + l.x), S * (int64_t)l.Kp, l.Kp, 0, &header->rows, p.D, (uint16_t*)(ws + l.xt), S * l.rows_p, l.rows_p};
    if (grad_weight) ce_transpose<<<dim3(l.rows_p / 64, ceil_div(p.D, 64), S), dim3(256), 0, s>>>(x);
    TransposeArgs w{(const uint16_t*)weight, weight_stride, l.Kp, p.F, nullptr, p.D, (uint16_t*)(ws + l.wt), S * all, all};
    if (grad_hidden) ce_transpose<<<dim3(ceil_div(p.F, 64), ceil_div(p.D, 64), S), dim3(256), 0, s>>>(w);

    for (int first = 0; first < p.F; first += l.piece) {
        const int classes = p.F - first < l.piece ? p.F - first : l.piece;
        const int Kc = round_up(classes, kStep);
        ProductArgs q{};
        q.a = {(const T*)weight + first * weight_stride, weight_stride, l.Kp, classes, nullptr};
        q.b = {fw + l.x, S * (int64_t)l.Kp, l.Kp, 0, &header->rows};
        q.K = l.Kp; q.splits = 1;
        EpilogueArgs e{};
        e.bias = p.bias; e.bias_f32 = p.dtype == I6TRAIN_F32; e.header = header; e.back = back; e.first_class = first; e.classes = p.F;
        e.row_target = row_target; e.rows_p = l.rows_p; e.lse = (const float*)(fw + l.lse); e.row_scale = row_scale;
        e.g = ws + l.g; e.g_stride = S * (int64_t)l.piece; e.g_half = l.piece;
        e.gt = ws + l.gt; e.gt_stride = S * l.rows_p; e.gt_half = l.rows_p;
        product<T, kGradient><<<dim3(ceil_div(classes, kTile), l.row_tiles), dim3(kThreads), 0, s>>>(q, e);
        if (grad_hidden) {
            ProductArgs d{};
            d.a = {ws + l.g, S * (int64_t)l.piece, l.piece, 0, &header->rows};
            d.b = {(const T*)(ws + l.wt) + first, S * all, all, p.D, nullptr};
            d.K = Kc; d.splits = 1;
            EpilogueArgs o{};
            o.out = (float*)(ws + l.dx); o.out_stride = p.D; o.add = first > 0;
            product<T, kStore><<<dim3(l.row_tiles, ceil_div(p.D, kTile)), dim3(kThreads), 0, s>>>(d, o);
        }
        if (grad_weight) {
            ProductArgs d{};
            d.a = {ws + l.gt, S * l.rows_p, l.rows_p, classes, nullptr};
            d.b = {ws + l.xt, S * l.rows_p, l.rows_p, p.D, nullptr};
            d.n_k = &header->rows; d.splits = l.splits;
            EpilogueArgs o{};
            o.out = (float*)(ws + l.dw); o.out_stride = p.D; o.out_split = (int64_t)l.piece * p.D;
            product<T, kStore><<<dim3(ceil_div(classes, kTile), ceil_div(p.D, kTile), l.splits), dim3(kThreads), 0, s>>>(d, o);
            const int64_t n = (int64_t)classes * p.D;
            ce_store_weight<In><<<dim3(ceil_div(n, (int64_t)256)), dim3(256), 0, s>>>(header, back, o.out, l.splits, o.out_split, n, (In*)grad_weight + (int64_t)first * p.D);
        }
        if (grad_bias)
            ce_store_bias<T, In><<<dim3(classes), dim3(256), 0, s>>>(header, back, (const T*)(ws + l.gt), S * l.rows_p, l.rows_p, (In*)grad_bias + first);
    }
    if (grad_hidden)
        ce_store_hidden<In><<<dim3(groups_for(rows)), dim3(256), 0, s>>>(header, back, (const int*)(fw + l.offsets), p.seq_lens, p.targets, p.targets_stride_b, p.targets_stride_t,
                                                                         (const float*)(ws + l.dx), p.B, p.T, p.F, p.D, (In*)grad_hidden);
    return launched();
}

}  // namespace
}  // namespace i6train

using namespace i6train;

extern "C" {

int i6train_ce_workspace_size(const i6train_ce_problem* p, size_t* forward_bytes, size_t* backward_bytes) {
    if (!valid(p) || !forward_bytes || !backward_bytes) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Layout l;
    I6TRAIN_TRY(layout(*p, l));
    *forward_bytes = l.forward;
    *backward_bytes = l.backward;
    return I6TRAIN_OK;
}

int i6train_ce_forward(const i6train_ce_problem* p, float* loss, void* workspace, size_t workspace_bytes, void* stream) {
    if (!valid(p) || !p->hidden || !loss || !workspace || (uintptr_t)workspace % 256) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Layout l;
    I6TRAIN_TRY(layout(*p, l));
    if (workspace_bytes < l.forward) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    if (p->dtype == I6TRAIN_F32) return forward<float, f16>(*p, l, loss, (char*)workspace, (hipStream_t)stream);
    return forward<bf16, bf16>(*p, l, loss, (char*)workspace, (hipStream_t)stream);
}

int i6train_ce_backward(const i6train_ce_problem* p, const float* grad_loss, int64_t grad_stride_b, int64_t grad_stride_t, void* grad_hidden, void* grad_weight, void* grad_bias,
                        const void* forward_workspace, size_t forward_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (!valid(p) || !grad_loss || !forward_workspace || !workspace || (uintptr_t)workspace % 256) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Layout l;
    I6TRAIN_TRY(layout(*p, l));
    if (forward_bytes < l.forward || workspace_bytes < l.backward) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    if (p->dtype == I6TRAIN_F32)
        return backward<float, f16>(*p, l, grad_loss, grad_stride_b, grad_stride_t, grad_hidden, grad_weight, grad_bias, (const char*)forward_workspace, (char*)workspace, (hipStream_t)stream);
    return backward<bf16, bf16>(*p, l, grad_loss, grad_stride_b, grad_stride_t, grad_hidden, grad_weight, grad_bias, (const char*)forward_workspace, (char*)workspace, (hipStream_t)stream);
}

}  // extern "C"
