// Output layer and frame-wise cross entropy without the logits (include/i6train.h).
//
//   forward    z = W h + b in tiles, in registers; per tile and frame the maximum and the sum of exp(z - maximum), joined over
//              the tiles afterwards;  loss = log sum exp z - z_y
//   backward   for one piece of the vocabulary after another: z again, G = g (softmax(z) - [f = y]) rounded to the operands'
//              precision, then  dh += G W  and  dW = G^T h
//
// All three products run through one function, product_of(): C[m][n] = sum_k A[m][k] B[n][k] on the matrix units.  An operand lies in memory
// with consecutive k (W and h for the logits, G for dh) or with consecutive m or n (W for dh, G and h for dW) and is turned
// as it is read from LDS, so nothing is transposed or written twice.
//
// The frames of a batch are packed first: only frames that belong to a sequence are rows of the products, and what the others
// hold is not read.  How many there are is known on the device alone: workgroups without a tile return at once.
//
// Operands.  The matrix units take 16 bits fast, so every tensor has a form in 16-bit values, and sums are held in 32 bits.
//
//   bfloat16   Logits are formed from the values as they are, in instructions for bfloat16: no product is rounded and no value is too large or too small.  The
//              gradients' products take 16-bit floating-point values with 11 bits, which hold G to 2^-12 of each value instead of the 2^-9 that bfloat16
//              would leave, and W and h, times a power of two that brings the tensor's largest value to 2^14 .. 2^15, exactly down to 2^-29 of the largest.
//   float      x is split into x1 = f16(s x) and x2 = f16(2^11 (s x - x1)), s such a power of two: 22 bits down to 2^-29 of the largest value, an error of 2^-51 of it
//              below.  Of (x1 + x2 2^-11)(y1 + y2 2^-11) the last term is below the precision and left out: the k-loop runs over x1 y2 and x2 y1, scales the
//              accumulators by 2^-11, and goes on with x1 y1: three times the work, on units whose rate for 16-bit operands is sixteen times that for 32-bit ones.
//
// One scale for a tensor is good where its values are not too different: in every row but those of zeros the values that are not 0 have a geometric mean (G: an incoming
// gradient) that the forms above hold well beside the tensor's largest value (kRows, kShares).  That is looked up on the device.  Where it is not so (frames,
// classes or features millions of times larger than others, incoming gradients over many powers of ten), the same kernels take another way, `wide`: for bfloat16 the gradients' products
// too are formed in bfloat16, with G rounded to it; for float the products are formed from the 32-bit values, in the matrix instructions that take
// them: a sixteenth of the rate, and as precise as a plain product (a training step of 44 800 frames, F = 5001, D = 500: 3.0 ms, 9.7 where the gradients' products alone are
// formed so, 15.6 where the logits are too).
//
// Logits are in units of log 2 from the accumulators on: exponentials and logarithms are single instructions.
//
// Large layers are bound by the matrix units and by the power they draw: the chip lowers its clock to 1.9 - 2.1 GHz under them.  28 800 frames, F = 12001, D = 512 in
// bfloat16 (0.353 TFLOP a product): on several cards statistics 357 - 367 us (960 - 990 TFLOP/s), G 2 x 232 - 238 us (740 - 760, writing 690 MB), dh and dW
// 2 x 354 - 360 us (980 - 1000), all that goes over the operands alone 80 us.  44 800 frames, F = 5001, D = 500 in 32 bits: the three parts of the statistics run at 1090 TFLOP/s, of dh and dW at 870.
#include <cmath>
#include <type_traits>

#include "lds_loads.h"
#include "train_common.h"

namespace i6train {
namespace {

constexpr int kM = 256;              // rows of a workgroup's tile of C, and, per two waves of 128 x 64 each, 64 columns
constexpr int kN = 128;              // its columns where the tile's logits are worked on
constexpr int kThreads = 256;
constexpr int kParts = 256;          // partial results of what looks over a tensor
constexpr int kShareParts = 64;      // those over the incoming gradients, one for a lane of every wave that joins them
constexpr int kPackGroups = 4096;    // at most, of ce_pack: in bfloat16 it looks over the tensors as well
constexpr int kLookThreads = 1024;   // every wave waits for lengths, targets and rows in turn: many waves, few rows each
constexpr int kPad = 64;             // rows and columns of operands are padded with zeros to multiples of this
constexpr float kLow = 0x1p-11f;     // weight of the second half of a 32-bit value
// By how many powers of two the mean of a row (and an incoming gradient) may be below the tensor's largest value in the fast forms; S: halves of a value.
// What is below a value's last bit, 2^-51 of the largest (16 bits: 2^-40), is then 2^-25 (2^-20) of the row's mean, 2^-29 (2^-24) of the frame's share.
template <int S> constexpr int kRows = S == 2 ? 26 : 20;
template <int S> constexpr int kShares = S == 2 ? 22 : 16;

using f16x2 = f16 __attribute__((ext_vector_type(2)));
using f16x4 = f16 __attribute__((ext_vector_type(4)));
using f16x8 = f16 __attribute__((ext_vector_type(8)));
using bf16x4 = bf16 __attribute__((ext_vector_type(4)));
using bf16x8 = bf16 __attribute__((ext_vector_type(8)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using acc_t = float __attribute__((ext_vector_type(4)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

template <typename N, typename M> __host__ __device__ constexpr N round_up(N n, M to) { return (n + (N)to - 1) / (N)to * (N)to; }

// At the start of the forward workspace.
struct Header {
    int rows;                        // frames that belong to a sequence
    int up_x, up_w;                  // in 32 bits: exponents of the scales of frames and weights,
    int wide;                        // and whether their rows are too different for one
};
// At the start of the backward workspace.
struct BackHeader {
    int rows, up_x, up_w, wide_rows; // the same, in bfloat16 too
    int up_g, wide;                  // of G; how the gradients' products are formed
    alignas(16) uint32_t most[kShareParts], least[kShareParts];      // incoming gradients: partial results
};
// Partial results over a tensor: the largest finite value, as its bit pattern, and the least mean exponent of a row that is not 0.
struct Parts {
    uint32_t *most_x, *least_x, *most_w, *least_w;
    int n;                           // of each
};
constexpr uint32_t kNone = 255;                            // no row

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t wave_min(uint32_t x) { return wave_reduce(x, 0xffffffffu, umin); }

// The exponent of the power of two that brings a tensor's largest value to 2^14 .. 2^15, and whether that is good for all its rows, from
// partial results: in every lane of a whole wave.
struct Scale {
    int up;
    bool wide;
};
__device__ __forceinline__ Scale scale_of(const uint32_t* most_parts, const uint32_t* least_parts, int n, int range) {
    uint32_t most = 0, least = kNone;
#pragma unroll 4
    for (int i = threadIdx.x & 63; i < n; i += 64) {
        most = umax(most, most_parts[i]);
        least = umin(least, least_parts[i]);
    }
    most = wave_max(most);
    least = wave_min(least);
    if (most == 0) return {0, false};
    const int top = (int)(most >> 23), up = 14 - (top - 127);
    if (up > 100) return {100, true};                      // scales and their products are normal numbers
    return {up, (int)least < top - range};
}

__device__ __forceinline__ bool has_target(int y, int classes) { return y >= 0 && y < classes; }

// ------------------------------------------------------------------------------------------------------ preparation

struct Frames {
    const void* hidden;  int64_t stride_b, stride_t;
    const int32_t* lens;
    const int32_t* targets;  int64_t tgt_b, tgt_t;
    int B, T, F, D, Kp;
};
struct Weights {
    const void* p;  int64_t stride;
    const void* bias;
};

// Eight values from column c on; zeros behind column D.
template <typename In> __device__ __forceinline__ void load8(const In* row, int c, int D, bool aligned, float (&v)[8]) {
    if (aligned && c + 8 <= D) {
        if constexpr (sizeof(In) == 2) {
            using V = In __attribute__((ext_vector_type(8)));
            const V x = *reinterpret_cast<const V*>(row + c);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = (float)x[i];
        } else {
            using V = In __attribute__((ext_vector_type(4)));
            const V x = *reinterpret_cast<const V*>(row + c), y = *reinterpret_cast<const V*>(row + c + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = x[i]; v[4 + i] = y[i]; }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = c + i < D ? (float)row[c + i] : 0.f;
}

// What a wave has seen of a tensor.
struct Seen {
    uint32_t most = 0, least = kNone;
    int exponents = 0, values_in = 0;          // of the row: what a lane has seen of it
    __device__ __forceinline__ void values(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t b = finite_bits(v[i]);
            most = umax(most, b);
            exponents += (int)(b >> 23);
            values_in += b != 0;
        }
    }
    __device__ __forceinline__ void end_row() {               // by the whole wave
        const float sum = wave_sum((float)exponents), n = wave_sum((float)values_in);
        if (n > 0.f) least = umin(least, (uint32_t)(sum * rcp_fast(n)));
        exponents = values_in = 0;
    }
};

// Workgroup 0: offsets[b], the first row of sequence b.  In 32 bits also: the next kParts look over the frames with a target, the
// last kParts over the weights.
template <typename In>
__global__ __launch_bounds__(kLookThreads) void ce_look(Frames f, Weights w, int* offsets, Header* header, Parts parts) {
    constexpr int kWaves = kLookThreads / kWave;
    __shared__ int sums[kWaves];
    __shared__ uint32_t most_of[kWaves], least_of[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (blockIdx.x == 0) {
        int carry = 0;
        for (int base = 0; base < f.B; base += kLookThreads) {
            const int b = base + threadIdx.x;
            int n = b < f.B ? f.lens[b] : 0;
            n = n < 0 ? 0 : (n > f.T ? f.T : n);
            int sum = n;
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(sum, d);
                if (lane >= d) sum += o;
            }
            if (lane == 63) sums[wave] = sum;
            __syncthreads();
            int before = carry;
            for (int i = 0; i < wave; i++) before += sums[i];
            if (b < f.B) offsets[b] = before + sum - n;
            for (int i = 0; i < kWaves; i++) carry += sums[i];
            __syncthreads();
        }
        if (threadIdx.x == 0) header->rows = carry;
        return;
    }
    const bool weights = blockIdx.x > kParts;
    const int part = (blockIdx.x - 1) % kParts;
    const In* base = static_cast<const In*>(weights ? w.p : f.hidden);
    const int64_t rows = weights ? f.F : (int64_t)f.B * f.T;
    Seen seen;
    for (int64_t r = (int64_t)part * kWaves + wave; r < rows; r += kParts * kWaves) {
        const In* row;
        if (weights) {
            row = base + r * w.stride;
        } else {
            const int b = (int)(r / f.T), t = (int)(r % f.T);
            if (t >= f.lens[b] || !has_target(f.targets[b * f.tgt_b + t * f.tgt_t], f.F)) continue;
            row = base + b * f.stride_b + t * f.stride_t;
        }
        const bool aligned = (uintptr_t)row % 16 == 0;
        for (int c = lane * 8; c < f.D; c += 512) {
            float v[8];
            load8(row, c, f.D, aligned, v);
            seen.values(v);
        }
        seen.end_row();
    }
    uint32_t most = wave_max(seen.most), least = seen.least;
    if (lane == 0) {
        most_of[wave] = most;
        least_of[wave] = least;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWaves; i++) {
            most = umax(most, most_of[i]);
            least = umin(least, least_of[i]);
        }
        (weights ? parts.most_w : parts.most_x)[part] = most;
        (weights ? parts.least_w : parts.least_x)[part] = least;
    }
}

// A 32-bit value as two halves.
__device__ __forceinline__ void split(float s, f16& high, f16& low) {
    high = (f16)s;
    low = fabsf(s) < 65504.f ? (f16)((s - (float)high) * 0x1p11f) : (f16)0.f;       // infinities and NaN are in the first half alone
}
template <typename In> __device__ __forceinline__ void store_operand(f16* out, int Kp, int c, const float (&v)[8], int up) {
    if constexpr (sizeof(In) == 2) {
        bf16x8 as_they_are;
#pragma unroll
        for (int i = 0; i < 8; i++) as_they_are[i] = (bf16)v[i];
        *reinterpret_cast<bf16x8*>(out + c) = as_they_are;
    } else {
        f16x8 high, low;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f16 h, l;
            split(ldexpf(v[i], up), h, l);
            high[i] = h;
            low[i] = l;
        }
        *reinterpret_cast<f16x8*>(out + c) = high;
        *reinterpret_cast<f16x8*>(out + Kp + c) = low;
    }
}

struct Packed {
    f16 *x, *w;                      // [row][halves][Kp] (bfloat16: its values), zeros behind column D and in rows up to a multiple of kPad; in 32 bits not where `wide`
    int *row_frame, *row_target;
    float* loss;
};

// A wave per row: frames as operands, then weights.  In bfloat16 it looks over them as well.
template <typename In>
__global__ __launch_bounds__(kThreads) void ce_pack(Frames f, Weights w, const int* offsets, Header* header, Parts parts, Packed o) {
    constexpr int S = sizeof(In) == 4 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    int up_x = 0, up_w = 0;
    bool store = true;
    if constexpr (S == 2) {
        const Scale x = scale_of(parts.most_x, parts.least_x, parts.n, kRows<S>), y = scale_of(parts.most_w, parts.least_w, parts.n, kRows<S>);
        up_x = x.up;
        up_w = y.up;
        store = !(x.wide || y.wide);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            header->up_x = up_x;
            header->up_w = up_w;
            header->wide = !store;
        }
    }
    Seen frames_seen, weights_seen;
    const int64_t frames = (int64_t)f.B * f.T, n_weights = round_up(f.F, kPad), all = frames + kPad + n_weights;
    const int64_t row_size = S * (int64_t)f.Kp;
    const float none[8] = {};
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < all; r += (int64_t)gridDim.x * 4) {
        if (r >= frames + kPad) {
            const int64_t row = r - frames - kPad;
            const In* x = static_cast<const In*>(w.p) + row * w.stride;
            const bool aligned = (uintptr_t)x % 16 == 0;
            for (int c = lane * 8; c < f.Kp && store; c += 512) {
                float v[8];
                if (row < f.F) {
                    load8(x, c, f.D, aligned, v);
                    if (S == 1) weights_seen.values(v);
                }
                store_operand<In>(o.w + row * row_size, f.Kp, c, row < f.F ? v : none, up_w);
            }
            if (S == 1 && row < f.F) weights_seen.end_row();
            continue;
        }
        if (r >= frames) {
            const int64_t row = header->rows + (r - frames);
            if (row < round_up((int64_t)header->rows, kPad))
                for (int c = lane * 8; c < f.Kp && store; c += 512) store_operand<In>(o.x + row * row_size, f.Kp, c, none, 0);
            continue;
        }
        const int b = (int)(r / f.T), t = (int)(r % f.T);
        if (t >= f.lens[b]) {
            if (lane == 0) o.loss[r] = 0.f;
            continue;
        }
        const int64_t row = offsets[b] + t;
        const int target = f.targets[b * f.tgt_b + t * f.tgt_t];
        const bool used = has_target(target, f.F);      // a frame without a target: zeros, whatever it holds
        const In* x = static_cast<const In*>(f.hidden) + b * f.stride_b + t * f.stride_t;
        const bool aligned = (uintptr_t)x % 16 == 0;
        for (int c = lane * 8; c < f.Kp && store; c += 512) {
            float v[8];
            if (used) {
                load8(x, c, f.D, aligned, v);
                if (S == 1) frames_seen.values(v);
            }
            store_operand<In>(o.x + row * row_size, f.Kp, c, used ? v : none, up_x);
        }
        if (S == 1 && used) frames_seen.end_row();
        if (lane == 0) {
            o.row_frame[row] = (int)r;
            o.row_target[row] = target;
        }
    }
    if constexpr (S == 1) {
        __shared__ uint32_t seen[4][4];
        const uint32_t mine[4] = {wave_max(frames_seen.most), frames_seen.least, wave_max(weights_seen.most), weights_seen.least};
        if (lane == 0)
            for (int i = 0; i < 4; i++) seen[threadIdx.x >> 6][i] = mine[i];
        __syncthreads();
        if (threadIdx.x == 0) {
            parts.most_x[blockIdx.x] = umax(umax(seen[0][0], seen[1][0]), umax(seen[2][0], seen[3][0]));
            parts.least_x[blockIdx.x] = umin(umin(seen[0][1], seen[1][1]), umin(seen[2][1], seen[3][1]));
            parts.most_w[blockIdx.x] = umax(umax(seen[0][2], seen[1][2]), umax(seen[2][2], seen[3][2]));
            parts.least_w[blockIdx.x] = umin(umin(seen[0][3], seen[1][3]), umin(seen[2][3], seen[3][3]));
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- product

struct Operand {
    const f16* p;
    const f16* wide;          // bfloat16: the values as they are, laid out alike
    int64_t row_stride;       // elements between rows; a row has consecutive k, or consecutive m (n)
    int64_t half_stride;      // elements to the second halves
    int64_t bytes;            // of the buffer, from p on
    int rows;                 // m (n) that there are, or kFrames
};
constexpr int kFrames = -1;   // as many as there are frames, which is known on the device alone
struct ProductArgs {
    Operand a, b;
    int K;                    // of one half; a multiple of kPad; or kFrames: rounded up to it
    int splits;               // ranges of k, one tile of C each
};

enum Kind { kStatistics, kGradient, kHidden, kWeight };

struct EpilogueArgs {
    // kStatistics, kGradient: m is the class, n the row
    const void* bias;
    const Header* header;  BackHeader* back;
    int first_class, piece_classes;        // of this piece
    const int* row_target;
    float2* part;                          // [tile of classes][rows_p]: maximum, sum
    int64_t rows_p;
    float* target_logit;                   // in units of log 2, from the accumulators: the same bits as in the sum over the classes
    const float *lse, *row_scale;
    f16* g;  int64_t g_stride, g_half;     // [row][halves][piece]
    // kHidden: m is the row, n the feature
    float* sum;  int64_t sum_stride;       // [range of k][m][n] over the pieces so far
    int add, last;                         // to what is there; to `out`: the last piece in one range
    const int* row_frame;
    int classes;
    void* out;
    Frames f;  Weights w;                  // the caller's tensors, for products of 32-bit values
    // kWeight: m is the class, n the feature; ranges of k one after another
    float* part_out;  int64_t part_stride;      // (the stride for kHidden as well)
    float* bias_out;  int64_t bias_stride; // [range][class], sums of G over the rows
};

// One operand's part of a stage: R rows of the tile by kK.  LDS is filled by loads that bypass the registers and write 64 lanes x 16 bytes in
// order; which 16 bytes a lane asks for is free, and places them so that reading has no bank conflicts.
//   consecutive k:   row r has kK / 8 chunks of 8 k; chunk c lies at place c ^ turn(r) of the row, other ones in 16 rows (256 bytes: 64 banks).  A fragment is one read of 16 bytes.
//   consecutive m:   k has R / 8 chunks of 8 m; chunk c lies at place c ^ turn(k): pairs of chunks (16 m) stay together, and 8 k lie in other 32 bytes.  A fragment is two
//                    reads that transpose 4 k x 16 m within 16 lanes.
// A fragment: 16 rows by 32 k, lane l has row l & 15 and 8 k from 8 (l >> 4) on.
template <int R, bool kConsecutiveK, int kWaves, int kK> struct Side {
    static constexpr int kLoads = R * kK * 2 / 1024 / kWaves;      // per wave and stage
    static constexpr int kBytes = R * kK * 2;
    descriptor source;
    uint32_t from[kLoads];       // byte offsets of this lane's chunks at k = 0
    uint32_t step, half;         // bytes from stage to stage, and to the second halves
    uint32_t to;                 // this wave's place in a stage
    int read[kK / 32];           // consecutive k: byte offsets of this lane's fragments of the first 16 rows
    int base, row, x;            // consecutive m: those of its k, the first row's, and what its places are turned by

    static __device__ __forceinline__ int turn(int i) {
        if (!kConsecutiveK) return ((i & 3) << 1) | (i & 8);
        return kK == 32 ? ((i >> 1) & 2) ^ ((i >> 3) & 1) * 3 : (i >> 1) & 7;
    }
    __device__ __forceinline__ void set(const Operand& o, bool wide, int rows, int first, int k0, int base_row) {
        const int lane = threadIdx.x & 63, wave = wave_index();
        const int64_t origin = kConsecutiveK ? first * o.row_stride + k0 : k0 * o.row_stride + first;
        source = describe((wide && o.wide ? o.wide : o.p) + origin, o.bytes - origin * 2);
        half = (uint32_t)(o.half_stride * 2);
        to = wave * 1024;
        step = kConsecutiveK ? kK * 2 : (uint32_t)(kK * o.row_stride * 2);
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int slot = (i * kWaves + wave) * 64 + lane;
            if (kConsecutiveK) {
                const int r = slot / (kK / 8), c = (slot % (kK / 8)) ^ turn(r);
                from[i] = (uint32_t)(min(r, rows - 1 - first) * o.row_stride * 2 + c * 16);      // rows behind the last are the last again
            } else {
                const int k = slot / (R / 8), c = (slot % (R / 8)) ^ turn(k);
                const int last = (int)((o.row_stride - first) / 8 - 1);                          // columns behind the row's end as well
                from[i] = (uint32_t)(k * o.row_stride * 2 + min(c, last) * 16);
            }
        }
        if (kConsecutiveK) {
            const int r = base_row + (lane & 15);
#pragma unroll
            for (int h = 0; h < kK / 32; h++) read[h] = r * kK * 2 + ((h * 4 + (lane >> 4)) ^ turn(r)) * 16;
        } else {
            const int k = (lane >> 4) * 8 + ((lane & 15) >> 2);
            base = k * (R * 2) + ((lane & 3) >> 1) * 16 + (lane & 1) * 8;
            row = base_row * 2;
            x = turn(k) * 16;
        }
    }
    __device__ __forceinline__ void fetch(int i, uint32_t lds, uint32_t offset) const {
        load_to_lds(source, lds + to + i * kWaves * 1024, from[i], offset);
    }
    // rows 16 b .. + 15, k of 32 h .. + 31
    __device__ __forceinline__ f16x8 fragment(const char* lds, int b, int h) const {
        if constexpr (kConsecutiveK) {
            return *reinterpret_cast<const f16x8*>(lds + read[h] + b * 16 * kK * 2);
        } else {
            const char* at = lds + base + ((row + b * 32) ^ x) + h * 32 * (R * 2);
            using P = __attribute__((address_space(3))) s16x4*;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 4 * (R * 2)));
            return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

constexpr int kGStride = kM * 2 + 16;      // bytes of a row of G in LDS

// A wave's block of 16 x 64 of C to memory, times two powers of two, through LDS of the wave's own: rows of 64 values in accesses of 16 bytes instead of one
// value a lane.  row(r) is where row r begins, or null; `cols` of the columns are there; `whole`: every 16 bytes of a row are aligned.
constexpr int kBlockBytes = 16 * (64 * 4 + 16);
template <typename Out, typename Row>
__device__ __forceinline__ void store_block(char* lds, const acc_t (&c)[4], float by, float by_too, int cols, bool whole, Row row) {
    constexpr int kStride = 64 * sizeof(Out) + 16, kPer = 16 / sizeof(Out), kLanes = 64 / kPer, kRows = 64 / kLanes;
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *reinterpret_cast<Out*>(lds + (4 * (lane >> 4) + r) * kStride + (j * 16 + (lane & 15)) * sizeof(Out)) = (Out)(c[j][r] * by * by_too);
    __builtin_amdgcn_wave_barrier();        // the wave's reads of LDS follow its writes
#pragma unroll
    for (int k = 0; k < 16 / kRows; k++) {
        const int r = k * kRows + lane / kLanes, n = lane % kLanes * kPer;
        const u32x4 v = *reinterpret_cast<const u32x4*>(lds + r * kStride + n * sizeof(Out));
        Out* to = row(r);
        if (!to || n >= cols) continue;
        if (whole && n + kPer <= cols) {
            *reinterpret_cast<u32x4*>(to + n) = v;
        } else {
            Out w[kPer];
            __builtin_memcpy(w, &v, 16);
            for (int i = 0; i < kPer && n + i < cols; i++) to[n + i] = w[i];
        }
    }
}

// A wave's 128 x 64 of a product of 32-bit values, straight from memory: h and W from the caller's tensors, G as floats.  A matrix instruction
// takes 4 k, one from each 16 lanes; lane l has k = 4 (l >> 4) + i of 16 in the i-th one.  Bound by the units for 32-bit operands.
template <int KIND>
__device__ __forceinline__ void product_of_floats(const ProductArgs& p, const EpilogueArgs& e, int rows, int rows_a, int rows_b, int m0, int n0, int k0, int end, bool with_bias,
                                                  acc_t (&acc)[8][4], float (&bias_sum)[8]) {
#if __HIP_DEVICE_COMPILE__
    constexpr bool kLogits = KIND == kStatistics || KIND == kGradient;
    const int lane = threadIdx.x & 63, k_in = (lane >> 4) * 4;
    const float* w = static_cast<const float*>(e.w.p) + e.first_class * e.w.stride;
    // a frame's features, and all bits of `there` off where it has no target: what such frames hold does not count
    const auto frame_of = [&](int row, uint32_t& there) -> const float* {
        there = has_target(e.row_target[row], e.f.F) ? there : 0u;
        const int frame = e.row_frame[row];
        return static_cast<const float*>(e.f.hidden) + frame / e.f.T * e.f.stride_b + frame % e.f.T * e.f.stride_t;
    };
    const float *a_row[8], *b_row[4];
    uint32_t b_there[4] = {~0u, ~0u, ~0u, ~0u};
    const auto masked = [](float v, uint32_t there) { return __uint_as_float(__float_as_uint(v) & there); };
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int m = min(m0 + i * 16 + (lane & 15), rows_a - 1);
        a_row[i] = kLogits ? w + m * e.w.stride : reinterpret_cast<const float*>(p.a.p) + (KIND == kHidden ? m * (p.a.row_stride / 2) : m);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = min(n0 + j * 16 + (lane & 15), rows_b - 1);
        b_row[j] = kLogits ? frame_of(n, b_there[j]) : w + n;
    }
    end = min(end, kLogits ? e.f.D : (KIND == kHidden ? e.piece_classes : rows));       // the k that there are
#pragma unroll 1
    for (int k = k0; k < end; k += 16) {
        float a[8][4], b[4][4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            // loads of the last k instead of those behind it, and then zeros
            const int at = min(k + k_in + c, end - 1);
            uint32_t there = k + k_in + c < end ? ~0u : 0u;
            const uint32_t a_there = there;
            const float* x = KIND == kWeight ? frame_of(at, there) : nullptr;
#pragma unroll
            for (int i = 0; i < 8; i++) a[i][c] = masked(a_row[i][KIND == kWeight ? at * (p.a.row_stride / 2) : at], a_there);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v = kLogits ? b_row[j][at] : (KIND == kHidden ? b_row[j][at * e.w.stride] : x[min(n0 + j * 16 + (lane & 15), rows_b - 1)]);
                b[j][c] = masked(v, there & b_there[j]);
            }
        }
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (KIND == kWeight && with_bias) bias_sum[i] += a[i][c];
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][c], b[j][c], acc[i][j], 0, 0, 0);
            }
    }
#endif
}

// In           type of the user's tensors: two halves where it has 32 bits
// KIND         what becomes of a tile
// NW           pairs of waves: a tile has 64 NW columns
// kWide        the product is formed the other way: from 32-bit values, or from bfloat16 ones where it would be 16-bit floating-point ones of 11 bits
// index        of the workgroup among those of this product
template <typename In, int KIND, int NW> struct Shape {
    static constexpr int kWaves = 2 * NW, kCols = 64 * NW, kStages = NW == 2 ? 3 : 2, kK = NW == 2 ? 32 : 64;
    static constexpr int kStageBytes = (kM + kCols) * kK * 2;
    static constexpr bool kLogits = KIND == kStatistics || KIND == kGradient;
    static constexpr int kBytes = kStages * kStageBytes + (kLogits ? kM * 4 : 0) + (KIND == kStatistics ? 5 * kCols * 4 : 0);
};

// kFloats      G leaves as floats
// frames       how many there are
// up, wide     kGradient: the exponent of its scale, and whether what takes it is formed the other way
template <typename In, int KIND, int NW, bool kWide, bool kFloats = false>
__device__ __forceinline__ void product_of(const ProductArgs& p, const EpilogueArgs& e, char* lds, int index, int frames, int up = 0, bool wide = false) {
#if __HIP_DEVICE_COMPILE__
    constexpr int S = sizeof(In) == 4 ? 2 : 1;
    constexpr bool kAk = KIND != kWeight, kBk = KIND == kStatistics || KIND == kGradient;      // consecutive k
    using Sh = Shape<In, KIND, NW>;
    constexpr int kWaves = Sh::kWaves, kCols = Sh::kCols, kStages = Sh::kStages, kStageBytes = Sh::kStageBytes, kK = Sh::kK;
    constexpr bool kLogits = Sh::kLogits;
    static_assert(KIND != kGradient || (kCols == kN && kN * kGStride <= kStages * kStageBytes), "G goes through the stages' LDS");
    float* bias = reinterpret_cast<float*>(lds + kStages * kStageBytes);
    float (*join)[kCols] = reinterpret_cast<float (*)[kCols]>(lds + kStages * kStageBytes + kM * 4);
    int* target_of = reinterpret_cast<int*>(join[4]);

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), wm = wave & 1, wn = wave >> 1;
    const int rows_a = p.a.rows == kFrames ? frames : p.a.rows, rows_b = p.b.rows == kFrames ? frames : p.b.rows;

    // Workgroups go round the eight dies; each die has an L2 of its own, so it gets a range of tiles of its own, in groups of eight tiles of A:
    // the 64 tiles that a die works on at a time have 8 + 8 operand tiles among them, not 64 + 1.
    const int tiles_m = ceil_div(rows_a, kM), tiles_n = ceil_div(rows_b, kCols), tiles = tiles_m * tiles_n * p.splits;
    const int each = ceil_div(tiles, 8);
    int tile = (index & 7) * each + (index >> 3);
    if ((index >> 3) >= each || tile >= tiles) return;
    const int part_of_k = tile / (tiles_m * tiles_n);
    tile -= part_of_k * tiles_m * tiles_n;
    const int group = tile / (8 * tiles_n), in_group = min(8, tiles_m - group * 8);
    tile -= group * 8 * tiles_n;
    const int tile_m = group * 8 + tile % in_group, tile_n = tile / in_group;
    const int m0 = tile_m * kM, n0 = tile_n * kCols;

    int K = p.K == kFrames ? round_up(frames, kPad) : p.K;
    int k0 = 0;
    if (p.splits > 1) {
        const int range = ceil_div(ceil_div(K, kK), p.splits) * kK;
        k0 = min(K, part_of_k * range);
        K = min(K, k0 + range);
    }
    const int steps = (K - k0) / kK, all = S == 2 ? 3 * steps : steps;

    Side<kM, kAk, kWaves, kK> A;
    Side<kCols, kBk, kWaves, kK> B;
    A.set(p.a, kWide, rows_a, m0, k0, wm * 128);
    B.set(p.b, kWide, rows_b, n0, k0, wn * 64);
    float bias_in = -INFINITY;        // classes behind the last: -inf, no probability
    if (kLogits && tid < kM && m0 + tid < rows_a) bias_in = e.bias ? (float)static_cast<const In*>(e.bias)[e.first_class + m0 + tid] : 0.f;
    int target_in = -1;
    if (KIND == kStatistics && tid < kCols && n0 + tid < rows_b) target_in = e.row_target[n0 + tid];

    // register r of a 16 x 16 block: row 4 (lane >> 4) + r, column lane & 15
    const int row_in = wm * 128 + 4 * (lane >> 4), col_in = wn * 64 + (lane & 15);
    acc_t acc[8][4];
    if (KIND == kHidden && e.add) {
        const float* sum = e.sum + part_of_k * e.part_stride + (int64_t)m0 * e.sum_stride + n0;
        const float scaled = S == 2 && all > 0 && !kWide ? 1.f / kLow : 1.f;       // taken back on the way, below
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int n = min(col_in + j * 16, rows_b - n0 - 1);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int m = min(row_in + i * 16 + r, rows_a - m0 - 1);
                    acc[i][j][r] = sum[(int64_t)m * e.sum_stride + n] * scaled;
                }
            }
        // here, or the compiler waits for all loads before the products of every stage
        __builtin_amdgcn_s_waitcnt(0x0f70);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
    }

    const uint32_t stages = lds_address(lds);
    constexpr int kLoadsA = Side<kM, kAk, kWaves, kK>::kLoads, kPerStage = kLoadsA + Side<kCols, kBk, kWaves, kK>::kLoads;
    uint32_t next_a = 0, next_b = 0;           // offsets of the stage that is fetched next
    const auto place_of = [&](int it) {
        if constexpr (S == 2) {
            const int part = it >= 2 * steps ? 2 : (it >= steps ? 1 : 0), k = it - part * steps;       // high x low, low x high, high x high
            next_a = __builtin_amdgcn_readfirstlane(k * A.step + (part == 1 ? A.half : 0));
            next_b = __builtin_amdgcn_readfirstlane(k * B.step + (part == 0 ? B.half : 0));
        } else {
            next_a = it * A.step;
            next_b = it * B.step;
        }
    };
    const auto fetch = [&](int i, int at) {    // load i of a stage
        if (i < kLoadsA) A.fetch(i, stages + at, next_a);
        else B.fetch(i - kLoadsA, stages + at + A.kBytes, next_b);
    };
    f16x8 fa[2][8], fb[2][4];
    const auto read = [&](auto set, int i, int at, int h) {      // fragment i of 32 k
        if (i < 4) fb[set.value][i] = B.fragment(lds + at + A.kBytes, i, h);
        else fa[set.value][i - 4] = A.fragment(lds + at, i - 4, h);
    };
    // kWeight: the fragments of A are G with the rows along k; the gradient of the bias is their sum
    const bool with_bias = KIND == kWeight && e.bias_out && tile_n == 0 && wn == 0;
    float bias_sum[8] = {};
    int it = 0, at = 0;                                          // stage, and where in LDS it is
    // 32 k of a stage: the products of one set of fragments, while the other set is read: the next 32 k of the stage, or the first of the next one.  Before
    // those are read the waves meet: this stage is in registers and its LDS free for another one, and the next stage has come in.
    // Reads and loads are spread over the products: issued all at once, the loads of eight waves fill the queue of the compute unit, and no product starts
    // until they have gone through.  A fragment of A is read when the one two before it has been used: registers for ten, not sixteen.
    const auto part_of_stage = [&](auto set, auto last, auto in_bf16) {
        constexpr int kSet = set.value;
        constexpr bool kLast = last.value;
        const std::integral_constant<int, 1 - kSet> other{};
        int free = 0;
        bool more = false;
        if (kLast) {
            if (it + kStages - 1 < all) wait_and_meet<(kStages - 2) * kPerStage>();
            else wait_and_meet<0>();
            free = at;
            more = it + kStages < all;
            if (more) place_of(it + kStages);
            at = at == (kStages - 1) * kStageBytes ? 0 : at + kStageBytes;
        }
        if (KIND == kWeight && with_bias && (S == 1 || it >= steps)) {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int r = 0; r < 8; r++) bias_sum[i] += in_bf16.value ? (float)__builtin_bit_cast(bf16x8, fa[kSet][i])[r] : (float)fa[kSet][i][r];
        }
        constexpr int kReadAt[12] = {0, 2, 4, 6, 8, 10, 12, 14, 16, 18, 20, 24};
#pragma unroll
        for (int n = 0; n < 32; n++) {
            if constexpr (in_bf16.value)
                acc[n >> 2][n & 3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fa[kSet][n >> 2]), __builtin_bit_cast(bf16x8, fb[kSet][n & 3]), acc[n >> 2][n & 3], 0, 0, 0);
            else
                acc[n >> 2][n & 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[kSet][n >> 2], fb[kSet][n & 3], acc[n >> 2][n & 3], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 12; i++)
                if (kReadAt[i] == n) read(other, i, at, kLast ? 0 : 1);         // behind the last stage: what is there, and not used
            if (kLast && more && n % 4 == 1 && n / 4 < kPerStage) fetch(n / 4, free);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const auto scale = [&] {                                     // between the second and the third part of 32-bit operands
        if (S == 2 && it == 2 * steps) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] *= kLow;
                bias_sum[i] *= kLow;
            }
        }
    };
    const auto run = [&](auto in_bf16) {
#pragma unroll
        for (int n = 0; n < kStages; n++) {
            if (n >= all) break;
            place_of(n);
#pragma unroll
            for (int i = 0; i < kPerStage; i++) fetch(i, n * kStageBytes);
        }
        if (all >= kStages) wait_and_meet<(kStages - 1) * kPerStage>();
        else wait_and_meet<0>();
        constexpr std::integral_constant<int, 0> first{};
        constexpr std::integral_constant<int, 1> second{};
#pragma unroll
        for (int i = 0; i < 12; i++) read(first, i, 0, 0);
        __builtin_amdgcn_s_setprio(1);
        for (; it < all; it++) {
            scale();
            part_of_stage(first, std::bool_constant<kK == 32>{}, in_bf16);
            if constexpr (kK == 32) {
                if (++it == all) break;
                scale();
            }
            part_of_stage(second, std::true_type{}, in_bf16);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    if (all > 0) {
        if constexpr (S == 2 && kWide) product_of_floats<KIND>(p, e, frames, rows_a, rows_b, m0 + wm * 128, n0 + wn * 64, k0, K, with_bias, acc, bias_sum);
        else run(std::bool_constant<S == 1 && (kLogits || kWide)>{});
    }

    if constexpr (KIND == kWeight) {
        __syncthreads();
        float* out = e.part_out + part_of_k * e.part_stride + n0 + wn * 64;
#pragma unroll
        for (int i = 0; i < 8; i++)
            store_block<float>(lds + wave * kBlockBytes, acc[i], 1.f, 1.f, rows_b - n0 - wn * 64, rows_b % 4 == 0, [&](int r) -> float* {
                const int m = m0 + wm * 128 + i * 16 + r;
                return m < rows_a ? out + (int64_t)m * rows_b : nullptr;
            });
        if (with_bias) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float v = bias_sum[i] + __shfl_xor(bias_sum[i], 16);
                v += __shfl_xor(v, 32);
                const int m = m0 + wm * 128 + i * 16 + lane;
                if (lane < 16 && m < rows_a) e.bias_out[part_of_k * e.bias_stride + m] = v;
            }
        }
        return;
    }

    if constexpr (KIND == kHidden) {
        if (!e.last) {
            __syncthreads();
            float* sum = e.sum + part_of_k * e.part_stride + n0 + wn * 64;
#pragma unroll
            for (int i = 0; i < 8; i++)
                store_block<float>(lds + wave * kBlockBytes, acc[i], 1.f, 1.f, rows_b - n0 - wn * 64, rows_b % 4 == 0, [&](int r) -> float* {
                    const int m = m0 + wm * 128 + i * 16 + r;
                    return m < rows_a ? sum + (int64_t)m * e.sum_stride : nullptr;
                });
            return;
        }
        // back to the frames, scales off; where the target is out of range, NaN
        int* frames = reinterpret_cast<int*>(lds + kWaves * kBlockBytes);
        __syncthreads();
        for (int i = tid; i < kM; i += 64 * kWaves) {
            const int m = m0 + i;
            frames[i] = m < rows_a ? (e.row_target[m] >= e.classes ? ~e.row_frame[m] : e.row_frame[m]) : 0;
        }
        const float unscale = ldexpf(1.f, -e.back->up_g), unscale_w = kWide ? 1.f : ldexpf(1.f, -e.back->up_w);
        __syncthreads();
        In* out = static_cast<In*>(e.out) + n0 + wn * 64;
        const bool whole = rows_b % (16 / (int)sizeof(In)) == 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (frames[row_in + i * 16 + r] < 0) acc[i][0][r] = acc[i][1][r] = acc[i][2][r] = acc[i][3][r] = __builtin_nanf("");
            store_block<In>(lds + wave * kBlockBytes, acc[i], unscale, unscale_w, rows_b - n0 - wn * 64, whole, [&](int r) -> In* {
                const int m = wm * 128 + i * 16 + r, frame = frames[m];
                return m0 + m < rows_a ? out + (int64_t)(frame < 0 ? ~frame : frame) * rows_b : nullptr;
            });
        }
        return;
    }

    if (tid < kM) bias[tid] = bias_in * kLog2e;
    if (KIND == kStatistics && tid < kCols) target_of[tid] = has_target(target_in, rows_a) ? target_in - m0 : -1;
    const float per = S == 1 || kWide ? kLog2e : fminf(ldexpf(kLog2e, -(e.header->up_x + e.header->up_w)), 0x1p127f);
    __syncthreads();
    // logits in units of log 2
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float4 b = *reinterpret_cast<const float4*>(&bias[row_in + i * 16]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            acc[i][j][0] = fmaf(acc[i][j][0], per, b.x);
            acc[i][j][1] = fmaf(acc[i][j][1], per, b.y);
            acc[i][j][2] = fmaf(acc[i][j][2], per, b.z);
            acc[i][j][3] = fmaf(acc[i][j][3], per, b.w);
        }
    }

    if constexpr (KIND == kStatistics) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // the wave that holds a target's logit leaves it to the loss, which then is not below 0, and to the gradient
            const int y = target_of[col_in + j * 16] - wm * 128;
            const bool here = y >= 0 && y < 128 && ((y >> 2) & 3) == (lane >> 4);
            if (__ballot(here)) {
                float logit = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) logit = (y & ~12) == i * 16 + r ? acc[i][j][r] : logit;
                if (here) e.target_logit[n0 + col_in + j * 16] = logit;
            }
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) most = fmaxf(most, acc[i][j][r]);
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float base = most == -INFINITY ? 0.f : most;        // classes that are all ruled out: the sum is 0, not NaN
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) sum += exp2_fast(acc[i][j][r] - base);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane < 16) {
                join[wm * 2][col_in + j * 16] = most;
                join[wm * 2 + 1][col_in + j * 16] = sum;
            }
        }
        __syncthreads();
        if (tid < kCols && n0 + tid < rows_b) {
            const float ma = join[0][tid], mb = join[2][tid], most = fmaxf(ma, mb), base = most == -INFINITY ? 0.f : most;
            const float sum = join[1][tid] * exp2_fast(ma - base) + join[3][tid] * exp2_fast(mb - base);
            e.part[(int64_t)tile_m * e.rows_p + n0 + tid] = make_float2(most, sum);
        }
    }

    if constexpr (KIND == kGradient) {
        const auto target_of_row = [&](int n) { return (exp2_fast(e.target_logit[n] - e.lse[n]) - 1.f) * ldexpf(e.row_scale[n], up); };
        if constexpr (kFloats) {
            // four classes from each lane, a column at a time
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int n = n0 + col_in + j * 16, at = min(n, rows_b - 1);
                const float lse = n < rows_b ? e.lse[at] : INFINITY, scale = n < rows_b ? e.row_scale[at] : 0.f;
                const int y = e.row_target[at] - e.first_class - m0 - row_in;
                const bool there = n < rows_b && y >= 0 && y < rows_a - m0 - row_in;
                const float value = there ? target_of_row(at) : 0.f;
                float* g = reinterpret_cast<float*>(e.g) + n * (e.g_stride / 2) + m0 + row_in;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    acc_t v;
#pragma unroll
                    for (int r = 0; r < 4; r++) v[r] = there && y == i * 16 + r ? value : exp2_fast(acc[i][j][r] - lse) * scale;
                    *reinterpret_cast<acc_t*>(g + i * 16) = v;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = n0 + col_in + j * 16;
            const float lse = n < rows_b ? e.lse[n] : INFINITY, scale = n < rows_b ? ldexpf(e.row_scale[n], up) : 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float v = exp2_fast(acc[i][j][r] - lse) * scale;
                    if constexpr (S == 2) {
                        f16x2 halves;      // both in the accumulator's register
                        f16 high, low;
                        split(v, high, low);
                        halves[0] = high;
                        halves[1] = low;
                        acc[i][j][r] = __builtin_bit_cast(float, halves);
                    } else {
                        acc[i][j][r] = v;
                    }
                }
        }
        // the target's value of each row, in the place it has in this tile
        int place = -1;
        float at_target = 0.f;
        if (tid < kN && n0 + tid < rows_b) {
            const int y = e.row_target[n0 + tid] - e.first_class - m0;
            if (y >= 0 && y < min(kM, rows_a - m0)) {
                place = y;
                at_target = target_of_row(n0 + tid);
            }
        }
#pragma unroll 1
        for (int h = 0; h < S; h++) {
            // through LDS, so that whole rows of the tile are written at once
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f16x4 v;
                    if constexpr (S == 2) {
                        const uint32_t which = h ? 0x07060302u : 0x05040100u;       // upper or lower 16 bits of two registers
                        uint32_t pair[2];
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            pair[r] = __builtin_amdgcn_perm(__float_as_uint(acc[i][j][2 * r + 1]), __float_as_uint(acc[i][j][2 * r]), which);
                        v = __builtin_bit_cast(f16x4, pair);
                    } else if (wide) {
                        bf16x4 u;
#pragma unroll
                        for (int r = 0; r < 4; r++) u[r] = (bf16)acc[i][j][r];
                        v = __builtin_bit_cast(f16x4, u);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++) v[r] = (f16)acc[i][j][r];
                    }
                    *reinterpret_cast<f16x4*>(lds + (col_in + j * 16) * kGStride + (row_in + i * 16) * 2) = v;
                }
            __syncthreads();
            if (place >= 0) {
                f16 high, low;
                split(at_target, high, low);
                if (S == 1 && wide) high = __builtin_bit_cast(f16, (bf16)at_target);
                *reinterpret_cast<f16*>(lds + tid * kGStride + place * 2) = h == 0 ? high : low;
            }
            __syncthreads();
            f16* g = e.g + n0 * e.g_stride + h * e.g_half + m0;
#pragma unroll 4
            for (int i = 0; i < kN / 8; i++) {
                const int r = i * 8 + (tid >> 5), c = tid & 31;
                *reinterpret_cast<u32x4*>(g + r * e.g_stride + c * 8) = *reinterpret_cast<const u32x4*>(lds + r * kGStride + c * 16);
            }
            if (h + 1 < S) __syncthreads();
        }
    }
#endif
}

template <typename In, int KIND, int NW>
__global__ __launch_bounds__(128 * NW, 2) void product(ProductArgs p, EpilogueArgs e) {
    __shared__ alignas(16) char lds[Shape<In, KIND, NW>::kBytes];
#if __HIP_DEVICE_COMPILE__
    constexpr bool kHalves = sizeof(In) == 4;
    const int index = blockIdx.x, frames = e.header->rows, wide_rows = e.header->wide;
    if constexpr (KIND == kGradient) {
        const Scale g = scale_of(e.back->most, e.back->least, kShareParts, kShares<kHalves ? 2 : 1>);
        const bool wide = g.wide || (kHalves ? wide_rows : e.back->wide_rows);
        const int up = wide ? 0 : g.up;
        if (index == 0 && threadIdx.x == 0) {
            e.back->up_g = up;
            e.back->wide = wide;
        }
        if constexpr (!kHalves) product_of<In, KIND, NW, false>(p, e, lds, index, frames, up, wide);
        else if (wide_rows) product_of<In, KIND, NW, true, true>(p, e, lds, index, frames, up);
        else if (wide) product_of<In, KIND, NW, false, true>(p, e, lds, index, frames, up);
        else product_of<In, KIND, NW, false>(p, e, lds, index, frames, up);
    } else {
        if (kHalves && wide_rows) product_of<In, KIND, NW, kHalves>(p, e, lds, index, frames);
        else product_of<In, KIND, NW, false>(p, e, lds, index, frames);
    }
#endif
}

// dh and dW of a piece in one launch, the first `hidden` workgroups (a multiple of eight) for dh: neither needs the other, and where dh leaves compute
// units idle, dW runs beside it (14 400 frames, F = 264, D = 512 in bfloat16: a training step 85 us, 98 us with one after the other).
struct BothArgs {
    ProductArgs p;
    EpilogueArgs e;
};
template <typename In, int NW>
__global__ __launch_bounds__(128 * NW, 2) void products_back(BothArgs h, BothArgs w, int hidden, const BackHeader* back) {
    static_assert(Shape<In, kHidden, NW>::kBytes == Shape<In, kWeight, NW>::kBytes);
    __shared__ alignas(16) char lds[Shape<In, kHidden, NW>::kBytes];
    const int index = blockIdx.x, frames = back->rows;
    if (back->wide) {
        if (index < hidden) product_of<In, kHidden, NW, true>(h.p, h.e, lds, index, frames);
        else product_of<In, kWeight, NW, true>(w.p, w.e, lds, index - hidden, frames);
    } else {
        if (index < hidden) product_of<In, kHidden, NW, false>(h.p, h.e, lds, index, frames);
        else product_of<In, kWeight, NW, false>(w.p, w.e, lds, index - hidden, frames);
    }
}
template <typename In> void launch_back(bool narrow, unsigned hidden, unsigned groups, const BothArgs& h, const BothArgs& w, const BackHeader* back, hipStream_t s) {
    if (groups == 0) return;
    if (narrow) products_back<In, 2><<<dim3(groups), dim3(256), 0, s>>>(h, w, (int)hidden, back);
    else products_back<In, 4><<<dim3(groups), dim3(512), 0, s>>>(h, w, (int)hidden, back);
}

// ---------------------------------------------------------------------------------------------------------- the rest

// Statistics of the tiles joined: loss and log sum of a row.  In bfloat16 the last workgroups join 256 each of what ce_pack's have seen, for the backward pass.
template <typename In>
__global__ __launch_bounds__(64) void ce_finish(const Header* header, Parts seen, Parts joined, const float2* part, int tiles, int64_t rows_p, const int* row_frame,
                                                 const int* row_target, const float* target_logit, const void* bias, int T, int F, float* lse, float* loss, int* report) {
    const int row = blockIdx.x * 64 + threadIdx.x;
    const int group = (int)blockIdx.x - (int)(gridDim.x - joined.n);
    if (group >= 0) {
        const int i = group * 256 + threadIdx.x * 4;
        const bool there = i < seen.n;
        const auto join = [&](const uint32_t* from, uint32_t* to, uint32_t none, auto better, auto of_wave) {
            u32x4 v = none;
            if (there) v = *reinterpret_cast<const u32x4*>(from + i);
            const uint32_t best = of_wave(better(better(v.x, v.y), better(v.z, v.w)));
            if (threadIdx.x == 0) to[group] = best;
        };
        join(seen.most_x, joined.most_x, 0u, umax, [](uint32_t v) { return wave_max(v); });
        join(seen.least_x, joined.least_x, kNone, umin, [](uint32_t v) { return wave_min(v); });
        join(seen.most_w, joined.most_w, 0u, umax, [](uint32_t v) { return wave_max(v); });
        join(seen.least_w, joined.least_w, kNone, umin, [](uint32_t v) { return wave_min(v); });
        return;
    }
    if (row >= header->rows) return;
    float most = -INFINITY, sum = 0.f;
    for (int i = 0; i < tiles; i += 8) {
        float2 p[8];
        float m = most;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            p[k] = i + k < tiles ? part[(i + k) * rows_p + row] : make_float2(-INFINITY, 0.f);
            m = fmaxf(m, p[k].x);
        }
        const float base = m == -INFINITY ? 0.f : m;
        sum *= exp2_fast(most - base);
#pragma unroll
        for (int k = 0; k < 8; k++) sum += p[k].y * exp2_fast(p[k].x - base);
        most = m;
    }
    const float l = most + log2_fast(sum);
    lse[row] = l;
    const int y = row_target[row], frame = row_frame[row];
    float v = 0.f;
    if (has_target(y, F)) {
        const float logit = target_logit[row];
        v = (l - logit) * kLn2;
        if (logit == -INFINITY && bias) {      // a bias beside which the rest is nothing, and which is too large in units of log 2
            const float b = static_cast<const In*>(bias)[y];
            if (b * kLog2e == -INFINITY) v = l * kLn2 - b;
        }
    } else if (y >= F) {
        v = __builtin_nanf("");
        if (report) {
            __hip_atomic_store(report + 1, frame / T, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            __hip_atomic_store(report, I6TRAIN_ERR_BAD_TARGET, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
        }
    }
    loss[frame] = v;
}

// Of bfloat16 values: as 16-bit floating-point values of 11 bits, scaled.  Null: not needed.
struct Copies {
    const bf16 *x, *w;
    f16 *x_out, *w_out;
    int64_t w_values;
};

// The first kShareParts workgroups: the incoming gradient of each row; rows without a target, or with one that is out of range, have none.  The
// next ones: zeros in the frames behind the ends.  The others, in bfloat16: copies of the operands.
template <typename Out>
__global__ __launch_bounds__(256) void ce_row_scale(const Header* header, const int* row_frame, const int* row_target, const float* grad_loss, int64_t stride_b,
                                                    int64_t stride_t, Frames f, Parts joined, Copies copies, int zeros, float* row_scale, BackHeader* back, Out* grad_hidden) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int helper = (int)blockIdx.x - kShareParts;
    if (helper >= 0 && helper < zeros) {
        const int64_t frames = (int64_t)f.B * f.T;
        for (int64_t r = (int64_t)helper * 4 + wave; r < frames; r += (int64_t)zeros * 4) {
            const int b = (int)(r / f.T), t = (int)(r % f.T);
            if (t < f.lens[b]) continue;
            for (int d = lane; d < f.D; d += 64) grad_hidden[r * f.D + d] = (Out)0.f;
        }
        return;
    }
    const bool first_group = blockIdx.x == 0, copier = helper >= 0;
    const int rows = header->rows;
    // copies: what a thread reads first is on its way while the scales are looked up
    const int64_t start = (int64_t)(helper - zeros) * 2048 + threadIdx.x * 8, stride = (int64_t)((int)gridDim.x - kShareParts - zeros) * 2048;
    const int64_t w_end = copies.w_out ? copies.w_values : 0, x_end = copies.x_out ? round_up((int64_t)rows, kPad) * f.Kp : 0;
    bf16x8 w_first, x_first;
    if (copier && start < w_end) w_first = *reinterpret_cast<const bf16x8*>(copies.w + start);
    if (copier && start < x_end) x_first = *reinterpret_cast<const bf16x8*>(copies.x + start);
    int up_x = header->up_x, up_w = header->up_w;
    bool wide = header->wide;
    if (sizeof(Out) == 2 && (copier || first_group)) {
        const Scale x = scale_of(joined.most_x, joined.least_x, joined.n, kRows<1>), w = scale_of(joined.most_w, joined.least_w, joined.n, kRows<1>);
        up_x = x.up;
        up_w = w.up;
        wide = x.wide || w.wide;
    }
    if (first_group && threadIdx.x == 0) {
        back->rows = rows;
        back->up_x = up_x;
        back->up_w = up_w;
        back->wide_rows = wide;
    }
    if (copier) {
        const auto copy = [&](const bf16* from, f16* to, int64_t end, bf16x8 v, int up) {
            for (int64_t i = start; i < end; i += stride) {
                if (i != start) v = *reinterpret_cast<const bf16x8*>(from + i);
                f16x8 u;
#pragma unroll
                for (int k = 0; k < 8; k++) u[k] = (f16)ldexpf((float)v[k], up);
                *reinterpret_cast<f16x8*>(to + i) = u;
            }
        };
        if (!wide) {
            copy(copies.w, copies.w_out, w_end, w_first, up_w);
            copy(copies.x, copies.x_out, x_end, x_first, up_x);
        }
        return;
    }
    __shared__ uint32_t most_of[4], least_of[4];
    uint32_t most = 0, least = kNone;
    for (int row = blockIdx.x * 256 + threadIdx.x; row < rows; row += kShareParts * 256) {
        float g = 0.f;
        const int frame = row_frame[row];
        if (has_target(row_target[row], f.F)) g = grad_loss[(int64_t)(frame / f.T) * stride_b + (int64_t)(frame % f.T) * stride_t];
        row_scale[row] = g;
        const uint32_t size = finite_bits(g);
        most = umax(most, size);
        if (size) least = umin(least, size >> 23);
    }
    most = wave_max(most);
    least = wave_min(least);
    if (lane == 0) {
        most_of[wave] = most;
        least_of[wave] = least;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        back->most[blockIdx.x] = umax(umax(most_of[0], most_of[1]), umax(most_of[2], most_of[3]));
        back->least[blockIdx.x] = umin(umin(least_of[0], least_of[1]), umin(least_of[2], least_of[3]));
    }
}

// One piece of grad_weight and grad_bias: the ranges of k joined, scales off.  A workgroup has 256 values, a quarter of the ranges for each wave.
template <typename Out>
__global__ __launch_bounds__(256) void ce_store_weight(const BackHeader* back, const float* part, int splits, int64_t split_stride, int64_t n, Out* out,
                                                       const float* bias_part, int64_t bias_stride, int classes, Out* bias) {
    using V = float __attribute__((ext_vector_type(4)));
    __shared__ V sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float down = ldexpf(1.f, -back->up_g), down_x = back->wide ? 1.f : ldexpf(1.f, -back->up_x);
    const int64_t groups = ceil_div(n, (int64_t)256);
    const bool of_bias = blockIdx.x >= groups;            // the last workgroups
    const int64_t i = (of_bias ? blockIdx.x - groups : blockIdx.x) * 256 + lane * 4, all = of_bias ? classes : n, stride = of_bias ? bias_stride : split_stride;
    const float* from = of_bias ? bias_part : part;
    Out* to = of_bias ? bias : out;
    if (!to) return;
    V v = 0.f;
    if (i + 4 <= all && stride % 4 == 0) {
#pragma unroll 8
        for (int s = wave; s < splits; s += 4) v += *reinterpret_cast<const V*>(from + s * stride + i);
    } else {
        for (int s = wave; s < splits; s += 4)
            for (int k = 0; k < 4 && i + k < all; k++) v[k] += from[s * stride + i + k];
    }
    sums[wave][lane] = v;
    __syncthreads();
    if (wave != 0) return;
    v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (i + k < all) to[i + k] = (Out)(v[k] * down * (of_bias ? 1.f : down_x));
}

// grad_hidden where its sums over the classes were formed in ranges: joined, scales off, back to the frames.  A workgroup has 256 values, a quarter of the
// ranges for each wave.
template <typename Out>
__global__ __launch_bounds__(256) void ce_store_hidden(const Header* header, const BackHeader* back, const float* part, int splits, int64_t split_stride, const int* row_frame,
                                                       const int* row_target, int F, int D, Out* out) {
    __shared__ float sums[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float down = ldexpf(1.f, -back->up_g), down_w = back->wide ? 1.f : ldexpf(1.f, -back->up_w);
    const int64_t first = (int64_t)blockIdx.x * 256, all = (int64_t)header->rows * D;
    if (first >= all) return;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int64_t i = first + k * 64 + lane;
        float v = 0.f;
        if (i < all) {
#pragma unroll 8
            for (int s = wave; s < splits; s += 4) v += part[s * split_stride + i];
        }
        sums[wave][k * 64 + lane] = v;
    }
    __syncthreads();
    const int64_t i = first + threadIdx.x;
    if (i >= all) return;
    const int row = (int)(i / D), d = (int)(i - (int64_t)row * D), t = threadIdx.x;
    const float v = ((sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t])) * down * down_w;
    out[(int64_t)row_frame[row] * D + d] = (Out)(row_target[row] >= F ? __builtin_nanf("") : v);
}

// ------------------------------------------------------------------------------------------------------------- host

// Of G.  Memory that a step needs against its time, which a join of dh and more workgroups' ends take (headline layer, 28 800 x 12001 x 512 in bfloat16: 1635 us with 256 MB,
// 1584 with 512, 1573 with 1 GB, which is all of it).
constexpr size_t kPieceBytes = (size_t)512 << 20;

// Where things are in the workspaces.
struct Layout {
    int S, Kp, row_tiles, class_tiles, piece, splits, hidden_splits;
    bool narrow;
    int64_t rows, rows_p, weights_p;
    size_t header, seen, joined, offsets, row_frame, row_target, target_logit, lse, x, w, part, x_bytes, w_bytes, forward;
    size_t back, row_scale, x_copy, w_copy, g, dx, dw, db, g_bytes, backward;
    int pack_groups, parts, joins;
};

bool valid(const i6train_ce_problem* p) {
    return p && p->B > 0 && p->T > 0 && p->F > 0 && p->D > 0 && valid_dtype(p->dtype) && p->weight && p->targets && p->seq_lens;
}

int groups_for(int64_t rows) { return (int)(rows < 4 * kPackGroups ? round_up(ceil_div(rows, (int64_t)4), 4) : kPackGroups); }

int layout(const i6train_ce_problem& p, Layout& l) {
    l.rows = (int64_t)p.B * p.T;
    if (l.rows > (1 << 22) || p.F > (1 << 22) || p.D > (1 << 14)) return I6TRAIN_ERR_TOO_LARGE;
    // (the launches with the most workgroups; those of large tiles have half as many of twice the threads)
    if (!launchable(round_up(ceil_div((int64_t)p.F, (int64_t)kM) * ceil_div(l.rows, (int64_t)kN), 8), kThreads)) return I6TRAIN_ERR_TOO_LARGE;
    l.S = p.dtype == I6TRAIN_F32 ? 2 : 1;
    l.Kp = round_up(p.D, kPad);
    l.row_tiles = (int)ceil_div(l.rows, (int64_t)kN);
    l.class_tiles = ceil_div(p.F, kM);
    l.rows_p = (int64_t)l.row_tiles * kN;
    l.weights_p = round_up(p.F, kPad);
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
    l.header = take(sizeof(Header));
    l.pack_groups = groups_for(l.rows + kPad + l.weights_p);
    l.parts = l.S == 2 ? kParts : round_up(l.pack_groups, 4);
    l.joins = l.S == 2 ? 0 : ceil_div(l.parts, 256);
    l.seen = take(4 * sizeof(uint32_t) * l.parts);
    l.joined = take(4 * sizeof(uint32_t) * kPackGroups / 256);
    l.offsets = take(4 * (size_t)p.B);
    l.row_frame = take(4 * l.rows_p);
    l.row_target = take(4 * l.rows_p);
    l.target_logit = take(4 * l.rows_p);
    l.lse = take(4 * l.rows_p);
    l.x_bytes = (size_t)l.rows_p * l.S * l.Kp * 2;
    l.w_bytes = (size_t)l.weights_p * l.S * l.Kp * 2;
    l.x = take(l.x_bytes);
    l.w = take(l.w_bytes);
    l.part = take(sizeof(float2) * l.class_tiles * l.rows_p);
    l.forward = at;

    at = 0;
    int64_t piece = (int64_t)(kPieceBytes / (2 * (size_t)l.S * l.rows_p)) / kM * kM;
    const int64_t classes = (int64_t)l.class_tiles * kM, most_piece = ((int64_t)1 << 31) / (2 * l.S * l.Kp) / kM * kM;      // (offsets within its weights have 32 bits)
    piece = piece > most_piece ? most_piece : piece;
    piece = piece < kM ? kM : (piece > classes ? classes : piece);
    l.piece = (int)round_up(ceil_div(classes, ceil_div(classes, piece)), kM);      // pieces of one size
    // Few tiles leave compute units idle, which tiles of 128 columns leave less (both gradients of 4000 frames, F = 1000, D = 384: 30 us with tiles of 256 columns, 25 with 128,
    // in 32 bits 70, 56; 8000 frames, F = 1000, D = 512: 32, 28 and 77, 66); more tiles are faster as large ones (8000 frames, F = 2000, D = 512: 49, 50 and 106, 110), and if
    // half of each is empty, as fast (28800 frames, F = 12001, D = 128: 602, 626 and 1653, 1554 with G; 8000 frames, F = 5001, D = 128: 55, 44 and 120, 103).
    const int64_t row_tiles = ceil_div(l.rows, (int64_t)kM), class_tiles = l.piece / kM;
    l.narrow = row_tiles * ceil_div(p.D, 256) <= 64 && (class_tiles * ceil_div(p.D, 256) <= 8 || p.D <= 128);
    const int columns = l.narrow ? 128 : 256, at_once = l.narrow ? 512 : 256;      // of a tile, and how many the compute units hold
    const int64_t tiles = class_tiles * ceil_div(p.D, columns);
    int64_t splits = at_once / tiles < 1 ? 1 : at_once / tiles;
    const int64_t most = ceil_div(l.rows, (int64_t)512), least = ceil_div((int64_t)l.rows_p * l.S * (l.piece > l.Kp ? l.piece : l.Kp) * 2, (int64_t)1 << 31);
    splits = splits > most ? most : splits;
    l.splits = (int)(splits < least ? least : splits);      // offsets within a range of k have 32 bits
    l.back = take(sizeof(BackHeader));
    l.row_scale = take(4 * l.rows_p);
    l.x_copy = take(l.S == 1 ? l.x_bytes : 0);
    l.w_copy = take(l.S == 1 ? l.w_bytes : 0);
    l.g_bytes = (size_t)l.rows_p * l.S * l.piece * 2;
    l.g = take(l.g_bytes);
    // Few rows: the sums over the classes are formed in ranges, or a handful of workgroups would go through the whole vocabulary (100 frames, F = 8346, D = 64, float: 69 us
    // a training step, 414 us in one range; 4000 frames, F = 5001, D = 512, float: 355 and 508).  Ranges are of 256 classes at least, of 512 where there are many tiles, whose
    // join costs more than shorter ranges win (4000 frames, F = 1000, D = 1024, bfloat16: 101 us in one range, 131 in three of 334).
    // Two ranges win nothing, as dW runs where dh leaves units idle (16000 frames, F = 5001, D = 512, bfloat16: 390 us in one range, 449 in two).
    const int64_t hidden_tiles = row_tiles * ceil_div(p.D, columns), room = (l.piece < p.F ? l.piece : p.F) / (hidden_tiles < 32 ? 256 : 512);
    const int64_t ranges = room < at_once / hidden_tiles ? room : at_once / hidden_tiles;
    l.hidden_splits = ranges > 2 ? (int)ranges : 1;
    l.dx = take(l.piece < p.F || l.hidden_splits > 1 ? 4 * (size_t)l.hidden_splits * l.rows_p * p.D : 0);
    l.dw = take(4 * (size_t)l.splits * l.piece * p.D);
    l.db = take(4 * (size_t)l.splits * l.piece);
    l.backward = at;
    return I6TRAIN_OK;
}

Frames frames_of(const i6train_ce_problem& p, const Layout& l) {
    return {p.hidden, p.hidden_stride_b, p.hidden_stride_t, p.seq_lens, p.targets, p.targets_stride_b, p.targets_stride_t, p.B, p.T, p.F, p.D, l.Kp};
}

template <int NW> int64_t tiles_of(int64_t rows_a, int64_t rows_b) { return ceil_div(rows_a, (int64_t)kM) * ceil_div(rows_b, (int64_t)(64 * NW)); }

// Workgroups for a product: a multiple of the dies.
template <int NW> unsigned groups_of(const ProductArgs& q, int64_t rows_a, int64_t rows_b) { return (unsigned)round_up(tiles_of<NW>(rows_a, rows_b) * q.splits, 8); }

template <typename In, int KIND, int NW> void launch_product(const ProductArgs& q, const EpilogueArgs& e, int64_t rows_a, int64_t rows_b, hipStream_t s) {
    product<In, KIND, NW><<<dim3(groups_of<NW>(q, rows_a, rows_b)), dim3(128 * NW), 0, s>>>(q, e);
}

Parts parts_at(const char* ws, int n, int room) {
    uint32_t* at = (uint32_t*)ws;
    return {at, at + room, at + 2 * room, at + 3 * room, n};
}

template <typename In>
int forward(const i6train_ce_problem& p, const Layout& l, float* loss, char* ws, hipStream_t s) {
    constexpr int S = sizeof(In) == 4 ? 2 : 1;
    const Frames f = frames_of(p, l);
    const Weights w{p.weight, p.weight_stride_f, p.bias};
    Header* header = (Header*)(ws + l.header);
    int* offsets = (int*)(ws + l.offsets);
    const Parts parts = parts_at(ws + l.seen, l.parts, l.parts), joined = parts_at(ws + l.joined, l.joins, kPackGroups / 256);
    ce_look<In><<<dim3(S == 2 ? 1 + 2 * kParts : 1), dim3(kLookThreads), 0, s>>>(f, w, offsets, header, parts);
    const Packed o{(f16*)(ws + l.x), (f16*)(ws + l.w), (int*)(ws + l.row_frame), (int*)(ws + l.row_target), loss};
    ce_pack<In><<<dim3(l.pack_groups), dim3(kThreads), 0, s>>>(f, w, offsets, header, parts, o);
    ProductArgs q{};
    q.a = {o.w, nullptr, l.S * (int64_t)l.Kp, l.Kp, (int64_t)l.w_bytes, p.F};
    q.b = {o.x, nullptr, l.S * (int64_t)l.Kp, l.Kp, (int64_t)l.x_bytes, kFrames};
    q.K = l.Kp; q.splits = 1;
    EpilogueArgs e{};
    e.bias = p.bias; e.header = header; e.part = (float2*)(ws + l.part); e.rows_p = l.rows_p;
    e.row_target = o.row_target; e.row_frame = o.row_frame; e.target_logit = (float*)(ws + l.target_logit);
    e.f = f; e.w = w;
    // Large tiles need fewer bytes for a product, but one workgroup has the compute unit and nothing runs beside its end.  They are for long loops (bfloat16, 28800 frames,
    // F = 12001: D = 512 366 us with small tiles, 344 with large ones, D = 128 175, 197) whose tiles go round the compute units more than twice, or once where small ones do
    // not (D = 512, F = 5001: 2400 frames 37, 34 us; 3200 frames, 260 large tiles, 38, 48 us; in 32 bits 8000 frames 143, 135).
    const int64_t small = tiles_of<2>(p.F, l.rows), large = tiles_of<4>(p.F, l.rows);
    if (l.Kp * (S == 2 ? 3 : 1) >= 512 && (large > 512 || (small > 256 && large <= 256))) launch_product<In, kStatistics, 4>(q, e, p.F, l.rows, s);
    else launch_product<In, kStatistics, 2>(q, e, p.F, l.rows, s);
    ce_finish<In><<<dim3(ceil_div(l.rows, (int64_t)64) + l.joins), dim3(64), 0, s>>>(header, parts, joined, e.part, l.class_tiles, l.rows_p, o.row_frame, o.row_target, e.target_logit, p.bias, p.T, p.F,
                                                                             (float*)(ws + l.lse), loss, status_slot());
    return launched();
}

template <typename In>
int backward(const i6train_ce_problem& p, const Layout& l, const float* grad_loss, int64_t gs_b, int64_t gs_t, void* grad_hidden, void* grad_weight, void* grad_bias,
             const char* fw, char* ws, hipStream_t s) {
    const Header* header = (const Header*)(fw + l.header);
    BackHeader* back = (BackHeader*)(ws + l.back);
    const int* row_target = (const int*)(fw + l.row_target);
    float* row_scale = (float*)(ws + l.row_scale);
    const f16 *x = (const f16*)(fw + l.x), *w = (const f16*)(fw + l.w);
    f16* g = (f16*)(ws + l.g);
    float *dx = (float*)(ws + l.dx), *dw = (float*)(ws + l.dw), *db = grad_bias ? (float*)(ws + l.db) : nullptr;
    const int64_t row_size = l.S * (int64_t)l.Kp, g_stride = l.S * (int64_t)l.piece;
    const int zeros = grad_hidden ? (int)(l.rows < 4096 ? ceil_div(l.rows, (int64_t)4) : 1024) : 0;
    int copiers = 0;
    if (l.S == 1) {
        const int64_t need = ceil_div((int64_t)(l.x_bytes > l.w_bytes ? l.x_bytes : l.w_bytes), (int64_t)4096);
        copiers = (int)(need < 4096 ? need : 4096);
    }
    const f16 *x16 = x, *w16 = w;             // of the gradients' products
    Copies copies{};
    if (l.S == 1) {
        x16 = (f16*)(ws + l.x_copy); w16 = (f16*)(ws + l.w_copy);
        copies = {(const bf16*)x, (const bf16*)w, grad_weight ? (f16*)x16 : nullptr, grad_hidden ? (f16*)w16 : nullptr, (int64_t)(l.w_bytes / 2)};
    }
    const Frames f = frames_of(p, l);
    const Parts joined = parts_at(fw + l.joined, l.joins, kPackGroups / 256);
    ce_row_scale<In><<<dim3(kShareParts + zeros + copiers), dim3(256), 0, s>>>(header, (const int*)(fw + l.row_frame), row_target, grad_loss, gs_b, gs_t, f, joined, copies, zeros, row_scale, back, (In*)grad_hidden);
    for (int first = 0; first < p.F; first += l.piece) {
        const int classes = p.F - first < l.piece ? p.F - first : l.piece;
        ProductArgs q{};
        q.a = {w + first * row_size, nullptr, row_size, l.Kp, (int64_t)l.w_bytes - first * row_size * 2, classes};
        q.b = {x, nullptr, row_size, l.Kp, (int64_t)l.x_bytes, kFrames};
        q.K = l.Kp; q.splits = 1;
        EpilogueArgs e{};
        e.bias = p.bias; e.header = header; e.back = back; e.first_class = first; e.piece_classes = classes;
        e.f = f; e.w = {p.weight, p.weight_stride_f, p.bias}; e.row_frame = (const int*)(fw + l.row_frame);
        e.row_target = row_target; e.target_logit = (float*)(fw + l.target_logit); e.lse = (const float*)(fw + l.lse); e.row_scale = row_scale;
        e.g = g; e.g_stride = g_stride; e.g_half = l.piece;
        launch_product<In, kGradient, 2>(q, e, classes, l.rows, s);
        BothArgs h{}, v{};
        unsigned of_hidden = 0, of_weight = 0;
        if (grad_hidden) {
            h.p.a = {g, nullptr, g_stride, l.piece, (int64_t)l.g_bytes, kFrames};
            h.p.b = {w16 + first * row_size, w + first * row_size, row_size, l.Kp, (int64_t)l.w_bytes - first * row_size * 2, p.D};
            h.p.K = round_up(classes, kPad); h.p.splits = l.hidden_splits;
            h.e = e;
            h.e.classes = p.F;
            h.e.sum = dx; h.e.sum_stride = p.D; h.e.part_stride = (int64_t)l.rows_p * p.D; h.e.add = first > 0; h.e.last = first + l.piece >= p.F && l.hidden_splits == 1;
            h.e.out = grad_hidden;
            of_hidden = l.narrow ? groups_of<2>(h.p, l.rows, p.D) : groups_of<4>(h.p, l.rows, p.D);
        }
        if (grad_weight || grad_bias) {
            v.p.a = {g, nullptr, g_stride, l.piece, (int64_t)l.g_bytes, classes};
            v.p.b = {x16, x, row_size, l.Kp, (int64_t)l.x_bytes, p.D};
            v.e = e;
            v.p.K = kFrames; v.p.splits = l.splits;
            v.e.part_out = dw; v.e.part_stride = (int64_t)l.piece * p.D; v.e.bias_out = db; v.e.bias_stride = l.piece;
            of_weight = l.narrow ? groups_of<2>(v.p, classes, p.D) : groups_of<4>(v.p, classes, p.D);
        }
        // dh that fills the compute units more than once leaves idle ones at its end alone, which long workgroups of dW do not fill (subword units, 44 800 x 5001 x 500
        // in 32 bits: a training step 3.00 ms apart, 3.03 together)
        const bool apart = of_hidden > (l.narrow ? 512 : 256) && of_weight;
        if (apart) launch_back<In>(l.narrow, of_hidden, of_hidden, h, v, back, s);
        const unsigned with = apart ? 0 : of_hidden;
        launch_back<In>(l.narrow, with, with + of_weight, h, v, back, s);
        if (of_hidden && l.hidden_splits > 1 && first + l.piece >= p.F)
            ce_store_hidden<In><<<dim3((unsigned)ceil_div(l.rows * p.D, (int64_t)256)), dim3(256), 0, s>>>(header, back, dx, l.hidden_splits, h.e.part_stride, h.e.row_frame, row_target, p.F,
                                                                                                          p.D, (In*)grad_hidden);
        if (of_weight) {
            const int64_t n = (int64_t)classes * p.D;
            ce_store_weight<In><<<dim3((unsigned)(ceil_div(n, (int64_t)256) + ceil_div(classes, 256))), dim3(256), 0, s>>>(
                back, dw, l.splits, v.e.part_stride, n, grad_weight ? (In*)grad_weight + (int64_t)first * p.D : nullptr, db, v.e.bias_stride, classes,
                grad_bias ? (In*)grad_bias + first : nullptr);
        }
    }
    return launched();
}

#include "cross_entropy_small.inc"

}  // namespace
}  // namespace i6train

using namespace i6train;

extern "C" {

int i6train_ce_workspace_size(const i6train_ce_problem* p, size_t* forward_bytes, size_t* backward_bytes) {
    if (!valid(p) || !forward_bytes || !backward_bytes) return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (is_small(*p)) {
        *forward_bytes = small_forward_bytes(*p);
        *backward_bytes = small_backward_bytes(*p);
        return I6TRAIN_OK;
    }
    Layout l;
    I6TRAIN_TRY(layout(*p, l));
    *forward_bytes = l.forward;
    *backward_bytes = l.backward;
    return I6TRAIN_OK;
}

int i6train_ce_forward(const i6train_ce_problem* p, float* loss, void* workspace, size_t workspace_bytes, void* stream) {
    if (!valid(p) || !p->hidden || !loss || !workspace || (uintptr_t)workspace % 256) return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (is_small(*p)) {
        if (workspace_bytes < small_forward_bytes(*p)) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
        const auto run = p->dtype == I6TRAIN_F32 ? small_forward<float> : small_forward<bf16>;
        return run(*p, loss, (char*)workspace, (hipStream_t)stream);
    }
    Layout l;
    I6TRAIN_TRY(layout(*p, l));
    if (workspace_bytes < l.forward) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    if (p->dtype == I6TRAIN_F32) return forward<float>(*p, l, loss, (char*)workspace, (hipStream_t)stream);
    return forward<bf16>(*p, l, loss, (char*)workspace, (hipStream_t)stream);
}

int i6train_ce_backward(const i6train_ce_problem* p, const float* grad_loss, int64_t grad_stride_b, int64_t grad_stride_t, void* grad_hidden, void* grad_weight, void* grad_bias,
                        const void* forward_workspace, size_t forward_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (!valid(p) || !grad_loss || !forward_workspace || !workspace || (uintptr_t)workspace % 256) return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (is_small(*p)) {
        if (!p->hidden) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (forward_bytes < small_forward_bytes(*p) || workspace_bytes < small_backward_bytes(*p)) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
        const auto run = p->dtype == I6TRAIN_F32 ? small_backward<float> : small_backward<bf16>;
        return run(*p, grad_loss, grad_stride_b, grad_stride_t, grad_hidden, grad_weight, grad_bias, (const char*)forward_workspace, (char*)workspace, (hipStream_t)stream);
    }
    Layout l;
    I6TRAIN_TRY(layout(*p, l));
    if (!p->hidden) return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (forward_bytes < l.forward || workspace_bytes < l.backward) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    const auto run = p->dtype == I6TRAIN_F32 ? backward<float> : backward<bf16>;
    return run(*p, l, grad_loss, grad_stride_b, grad_stride_t, grad_hidden, grad_weight, grad_bias, (const char*)forward_workspace, (char*)workspace, (hipStream_t)stream);
}

}  // extern "C"
