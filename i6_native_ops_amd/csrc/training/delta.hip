// Gated delta rule over the frames of a batch (include/i6delta.h):  S' = f S,  S = S' + k (w (v - S'^T k))^T,  o = S^T q.
//
// Chunks of C frames.  With c_i the sum of log f up to frame i of a chunk, D_ij = exp(c_i - c_j) and S0 the state in front of it, the rows
// u_i = w_i (v_i - S'_i^T k_i) that are written solve a triangular system, and all else are products:
//   (1 + A) U = R,  R = w (V - exp(c) K S0),  A_ij = w_i D_ij k_i.k_j (j < i)
//   O = exp(c) Q S0 + P U,  P_ij = D_ij q_i.k_j (j <= i);   S1 = exp(c_C) S0 + (exp(c_C - c) K)^T U
// Backward, with G1 the gradient of S1, from the last chunk to the first:
//   dU = P^T dO + exp(c_C - c) K G1,  (1 + A)^T dR = dU,  dV = w dR,  G0 = exp(c_C) G1 + (exp(c) Q)^T dO - (w exp(c) K)^T dR
// and from S0, G1, U and dR of a chunk all gradients of its q, k, gates, for all chunks at once (delta_gradients32, delta_gradients16).
//
// Every column of the state goes its own way: a wave has columns of its own, their states in registers as they come out of the matrix
// instructions, which is also how these take them for their second operand (with the order of k that both operands share), so states, R, U, O and their
// gradients never leave the wave; K, Q, A and P go through LDS.
//
// Single frames read and write the state, 134 KB of it for a head of 128 x 128: 64 streams of 8 heads 12.9 us, 5.3 TB/s.
#include <algorithm>
#include <cmath>

#include "train_common.h"
#include "../../../include/i6delta.h"

namespace i6train {
namespace {

using acc_t = float __attribute__((ext_vector_type(4)));
using bf16x8 = bf16 __attribute__((ext_vector_type(8)));

constexpr float kNormEps = 1e-6f;
constexpr int kThreads = 256;
constexpr int kC = 32;                   // frames of a chunk

struct Rows {                            // of the chunks' frames, [B][H][chunks C]
    float c, c_rest;                     // sum of log f within the chunk, as two floats
    float w, rk, rq;                     // share, 1 / length of key and query
    float start, end, pad;               // exp(c), exp(c_C - c)
};

struct Args {
    const void *q, *k, *v, *gate, *beta;
    int64_t q_b, q_t, q_g, k_b, k_t, k_g, v_b, v_t, v_h, gate_b, gate_t, gate_h, beta_b, beta_t, beta_h;
    const int32_t* lens;
    const float* initial;
    int B, T, H, G, K, V, chunks;
    void* o;
    float* last;
    Rows* rows;                          // of all chunks; null: frame by frame
    float *states, *u;                   // [B][H][chunks][K][V], [B][H][chunks C][V]; null: not for training
    // backward
    const void* d_o;
    int64_t do_b, do_t, do_h;
    const float* d_last;
    float *ends, *dr, *d_initial;        // gradients of the states behind the chunks, of R
    void *d_q, *d_k, *d_v, *d_gate, *d_beta;
    float *d_q_head, *d_k_head;          // [B][T][H][K], where heads share keys
};

__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * kLog2e); }
__device__ __forceinline__ int len_of(const Args& a, int b) {
    if (!a.lens) return a.T;
    const int n = a.lens[b];
    return n < 0 ? 0 : (n > a.T ? a.T : n);
}
__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }
// For sums over a chunk.  A gate of -inf: a factor that is 0, and sums that stay numbers; one that is no number stays that.
__device__ __forceinline__ float log_kept(float gate) {
    const float x = log_sigmoid(gate);
    return x < -1e6f ? -1e6f : x;
}
__device__ __forceinline__ float sigmoid(float x) {
    const float e = expf(-fabsf(x));
    return (x >= 0.f ? 1.f : e) / (1.f + e);
}

// Four values of a row of `n` from value `at` on; zeros behind them.
__device__ __forceinline__ acc_t load_piece(const float* row, int at, int n, bool whole) {
    if (whole && at + 4 <= n) return *reinterpret_cast<const acc_t*>(row + at);
    acc_t p;
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = at + i < n ? row[at + i] : 0.f;
    return p;
}

// -------------------------------------------------------------------------------------------------- products of 16 x 16 x 16
// An accumulator: lane l has column l & 15 and rows 4 (l >> 4) .. + 3.  Of the second operand a lane has k = 4 (l >> 4) .. + 3 of its column:
// an accumulator is one as it is.  Of the first operand it has the same k of row l & 15.
__device__ __forceinline__ acc_t product(acc_t a, acc_t b, acc_t c) {
#if __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
#endif
    return c;
}

// A matrix in LDS, rows of kStride floats.
template <int kStride> struct Tile {
    float* p;
    // first operand: rows 16 m .., k 16 n ..
    __device__ __forceinline__ acc_t rows(int m, int n) const {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const acc_t*>(p + (16 * m + (lane & 15)) * kStride + 16 * n + 4 * (lane >> 4));
    }
    // the transpose as first operand: its rows are columns 16 m .., its k are rows 16 n ..
    __device__ __forceinline__ acc_t columns(int m, int n) const {
        const int lane = threadIdx.x & 63;
        const float* at = p + (16 * n + 4 * (lane >> 4)) * kStride + 16 * m + (lane & 15);
        acc_t v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = at[i * kStride];
        return v;
    }
    __device__ __forceinline__ void put(int m, int n, acc_t v) const {
        const int lane = threadIdx.x & 63;
        float* at = p + (16 * m + 4 * (lane >> 4)) * kStride + 16 * n + (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; i++) at[i * kStride] = v[i];
    }
};

// What stands behind is not moved in front: loads and their addresses would otherwise fill the registers.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ acc_t four(const float* p) { return *reinterpret_cast<const acc_t*>(p); }

// ------------------------------------------------------------------------------------------------------ a chunk's matrices

// What a chunk's workgroup holds of keys, queries and decays in LDS.
template <int KP> struct Chunk {
    static constexpr int kStride = KP + 4, kSquare = kC + 4;
    float k[kC * kStride], q[kC * kStride];
    float a[kC * kSquare], p[kC * kSquare], inverse[kC * 20];
    float c[kC], c_rest[kC], w[kC], rk[kC], rq[kC];
    float from_start[kC], to_end[kC];    // exp(c), exp(c_C - c)
};

// Keys and queries of a chunk, loaded ahead: kPer pieces of each for a thread.
template <int KP> struct Ahead {
    static constexpr int kPieces = KP / 4, kThreadsPerRow = kThreads / kC, kPer = (kPieces + kThreadsPerRow - 1) / kThreadsPerRow;
    acc_t k[kPer], q[kPer];
    float gate, beta;
    __device__ __forceinline__ void fetch(const Args& a, int b, int h, int first, int len, bool whole) {
        const int row = threadIdx.x / kThreadsPerRow, j = threadIdx.x % kThreadsPerRow, t = first + row;
        const int g = h / (a.H / a.G);
        const float* kr = static_cast<const float*>(a.k) + b * a.k_b + t * a.k_t + g * a.k_g;
        const float* qr = static_cast<const float*>(a.q) + b * a.q_b + t * a.q_t + g * a.q_g;
        const acc_t none = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = (i * kThreadsPerRow + j) * 4;
            const bool there = t < len && at < a.K;
            k[i] = there ? load_piece(kr, at, a.K, whole) : none;
            q[i] = there ? load_piece(qr, at, a.K, whole) : none;
        }
        if (threadIdx.x < kC) {
            const int tt = first + threadIdx.x;
            const bool there = tt < len;
            gate = there ? static_cast<const float*>(a.gate)[b * a.gate_b + tt * a.gate_t + h * a.gate_h] : 0.f;
            beta = there ? static_cast<const float*>(a.beta)[b * a.beta_b + tt * a.beta_t + h * a.beta_h] : 0.f;
        }
    }
    // to LDS, with lengths, shares and decays.  The sum of log f is taken in 64 bits: differences of it are what counts, and it may be far larger.
    __device__ __forceinline__ void store(Chunk<KP>& s, int first, int len) {
        const int row = threadIdx.x / kThreadsPerRow, j = threadIdx.x % kThreadsPerRow;
        float kk = 0.f, qq = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = (i * kThreadsPerRow + j) * 4;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                kk = fmaf(k[i][e], k[i][e], kk);
                qq = fmaf(q[i][e], q[i][e], qq);
            }
            if (at < KP) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s.k[row * Chunk<KP>::kStride + at + e] = k[i][e];
                    s.q[row * Chunk<KP>::kStride + at + e] = q[i][e];
                }
            }
        }
#pragma unroll
        for (int m = 1; m < kThreadsPerRow; m *= 2) {
            kk += __shfl_xor(kk, m);
            qq += __shfl_xor(qq, m);
        }
        if (j == 0) {
            s.rk[row] = 1.f / sqrtf(kk + kNormEps);
            s.rq[row] = 1.f / sqrtf(qq + kNormEps);
        }
        if (threadIdx.x < kWave) {
            const int i = threadIdx.x;
            const bool there = i < kC && first + i < len;
            double c = there ? (double)log_kept(gate) : 0.0;
#pragma unroll
            for (int m = 1; m < kC; m *= 2) {
                const double before = __shfl_up(c, m);
                if (i >= m) c += before;
            }
            const double end = __shfl(c, kC - 1);
            if (i < kC) {
                const float hi = (float)c;
                s.c[i] = hi;
                s.c_rest[i] = (float)(c - (double)hi);
                s.w[i] = there ? sigmoid(beta) : 0.f;
                s.from_start[i] = exp_fast(hi);
                s.to_end[i] = exp_fast((float)(end - c));
            }
        }
    }
};

// Row of the n-th block of a lower triangle.
__device__ __forceinline__ int block_row(int n) {
    int i = 0;
    while ((i + 1) * (i + 2) / 2 <= n) i++;
    return i;
}

// A (strictly lower) and P (lower) of the chunk into LDS, without the blocks above the diagonal.
template <int KP> __device__ __forceinline__ void squares(Chunk<KP>& s) {
    constexpr int M = kC / 16;
    const Tile<Chunk<KP>::kStride> k{s.k};
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll 1
    for (int n = wave; n < M * (M + 1); n += 4) {       // lower blocks, of A and P in turn
        const int which = n & 1, i = block_row(n >> 1), j = (n >> 1) - i * (i + 1) / 2;
        const Tile<Chunk<KP>::kStride> left{which ? s.q : s.k};
        acc_t v = 0.f;
#pragma unroll
        for (int x = 0; x < KP / 16; x++) v = product(left.rows(i, x), k.rows(j, x), v);
        const int col = 16 * j + (lane & 15), row = 16 * i + 4 * (lane >> 4);
        const float c = s.c[col], c_rest = s.c_rest[col], r = s.rk[col];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int at = row + e;
            const float d = exp_fast((s.c[at] - c) + (s.c_rest[at] - c_rest));
            const float by = which ? s.rq[at] : s.rk[at] * s.w[at];
            v[e] = (which ? col <= at : col < at) ? v[e] * r * d * by : 0.f;
        }
        Tile<Chunk<KP>::kSquare>{which ? s.p : s.a}.put(i, j, v);
    }
}

// The inverses of 1 + A's blocks on the diagonal, a block for a wave, by substitution: sixteen lanes have four rows, which they solve among themselves, and what
// these rows take from those below is a product.  (The product of 1 + A's powers would need fewer steps, but with keys that are alike its terms are thousands of times
// larger than the result.)
template <int KP> __device__ __forceinline__ void invert(Chunk<KP>& s) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, group = lane >> 4, col = lane & 15;
    if (wave >= kC / 16) return;
    const acc_t row = -Tile<Chunk<KP>::kSquare>{s.a}.rows(wave, wave);
    const float* block = s.a + (16 * wave + 4 * group) * Chunk<KP>::kSquare + 16 * wave + 4 * group;
    const acc_t l1 = four(block + Chunk<KP>::kSquare), l2 = four(block + 2 * Chunk<KP>::kSquare), l3 = four(block + 3 * Chunk<KP>::kSquare);
    acc_t t = 0.f, left;
#pragma unroll
    for (int i = 0; i < 4; i++) left[i] = 4 * group + i == col ? 1.f : 0.f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        acc_t x = left;
        x[1] = fmaf(-l1[0], x[0], x[1]);
        x[2] = fmaf(-l2[1], x[1], fmaf(-l2[0], x[0], x[2]));
        x[3] = fmaf(-l3[2], x[2], fmaf(-l3[1], x[1], fmaf(-l3[0], x[0], x[3])));
        const acc_t none = 0.f;
        x = group == g ? x : none;
        t += x;
        if (g < 3) left = product(row, x, left);
    }
    Tile<20>{s.inverse}.put(wave, 0, t);
}

// Values at rows 16 m + 4 (lane >> 4) + r of a matrix, as accumulators.
template <int NT, int M>
__device__ __forceinline__ void load_columns(acc_t (&v)[M][NT], const float* p, int64_t stride, int rows, int col, int cols) {
    const int at = 4 * ((threadIdx.x & 63) >> 4);
    p += at * stride + col;
    asm volatile("" : "+v"(p));       // rows' addresses are formed here, or the compiler keeps them all from chunk to chunk
#pragma unroll
    for (int m = 0; m < M; m++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool there = 16 * m + at + e < rows;
#pragma unroll
            for (int j = 0; j < NT; j++) v[m][j][e] = there && col + j < cols ? p[j] : 0.f;
            p += stride;
        }
        p += 12 * stride;
    }
}
template <int NT, int M>
__device__ __forceinline__ void store_columns(const acc_t (&v)[M][NT], float* p, int64_t stride, int rows, int col, int cols) {
    const int at = 4 * ((threadIdx.x & 63) >> 4);
    p += at * stride + col;
    asm volatile("" : "+v"(p));       // rows' addresses are formed here, or the compiler keeps them all from chunk to chunk
#pragma unroll
    for (int m = 0; m < M; m++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool there = 16 * m + at + e < rows;
#pragma unroll
            for (int j = 0; j < NT; j++)
                if (there && col + j < cols) p[j] = v[m][j][e];
            p += stride;
        }
        p += 12 * stride;
    }
}

// A value that is no number belongs to its frame and those behind it, but products of whole blocks would take it to the frames of its block in front of it, too: there it is multiplied
// by 0, and that is NaN.  So from the first such row of R on, in its column, rows are 0 while the chunk's system is solved and read, and NaN behind that.  A sum with 0 times each
// value says whether there is one, which is all that a chunk pays for it.  Whether: the whole wave; `first`: the lane's column.
__device__ __forceinline__ void fill_from(acc_t& v, int m, int first, float by) {
    const int at = 16 * m + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (at + e >= first) v[e] = by;
}
template <int M> __device__ __forceinline__ bool take_out(acc_t (&r)[M], int& first) {
    float probe = 0.f;
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) probe = fmaf(r[m][e], 0.f, probe);
    if (!__any(probe != probe)) return false;
    const int at = 4 * ((threadIdx.x & 63) >> 4);
    first = 16 * M;
#pragma unroll
    for (int m = M - 1; m >= 0; m--)
#pragma unroll
        for (int e = 3; e >= 0; e--)
            if (!(fabsf(r[m][e]) < INFINITY)) first = 16 * m + at + e;
    first = min(first, __shfl_xor(first, 16));
    first = min(first, __shfl_xor(first, 32));
#pragma unroll
    for (int m = 0; m < M; m++) fill_from(r[m], m, first, 0.f);
    return true;
}
template <int M> __device__ __forceinline__ void put_back(acc_t (&r)[M], int first) {
#pragma unroll
    for (int m = 0; m < M; m++) fill_from(r[m], m, first, __builtin_nanf(""));
}

// ------------------------------------------------------------------------------------------------------ frame by frame

// Few frames, no training: 64 columns of a head, KP / 4 rows of the state in the registers of each of four waves.  The state is read and written once; with
// x = S^T k and y = S^T q of the state in front of a frame,  u = w (v - f x),  o = f y + (k.q) u.
template <typename T, int KP>
__global__ __launch_bounds__(kThreads, 4) void delta_frames(Args a) {
    constexpr int R = KP / 4;
    __shared__ __align__(16) float key[KP], query[KP], sums[4][2][64], dots[2][3];
    const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    const int len = len_of(a, b), g = h / (a.H / a.G);
    const int64_t head = (int64_t)b * a.H + h;
    const bool mine = col < a.V;
    // whole rows, as they mostly are: one address for all
    const int64_t from = (head * a.K + wave * R) * a.V + col;
    const bool whole = a.K == KP && blockIdx.x * 64 + 64 <= a.V;
    float state[R];
    if (a.initial && whole) {
        const float* p = a.initial + from;
#pragma unroll
        for (int i = 0; i < R; i++) {
            state[i] = *p;
            p += a.V;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; i++) state[i] = a.initial && mine && wave * R + i < a.K ? a.initial[from + (int64_t)i * a.V] : 0.f;
    }
    for (int t = 0; t < a.T; t++) {
        T* o = static_cast<T*>(a.o) + (((int64_t)b * a.T + t) * a.H + h) * a.V;
        if (t >= len) {
            if (wave == 0 && mine) o[col] = (T)0.f;
            continue;
        }
        const T* kr = static_cast<const T*>(a.k) + b * a.k_b + t * a.k_t + g * a.k_g;
        const T* qr = static_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + g * a.q_g;
        const float v = mine ? (float)static_cast<const T*>(a.v)[b * a.v_b + t * a.v_t + h * a.v_h + col] : 0.f;
        const float gate = (float)static_cast<const T*>(a.gate)[b * a.gate_b + t * a.gate_t + h * a.gate_h];
        const float beta = (float)static_cast<const T*>(a.beta)[b * a.beta_b + t * a.beta_t + h * a.beta_h];
        if (wave < 2) {                  // KP <= 128: two values a lane
            const int i = wave * 64 + lane;
            const float kv = i < a.K ? (float)kr[i] : 0.f, qv = i < a.K ? (float)qr[i] : 0.f;
            if (i < KP) {
                key[i] = kv;
                query[i] = qv;
            }
            const float kk = wave_sum(kv * kv), qq = wave_sum(qv * qv), kq = wave_sum(kv * qv);
            if (lane == 0) {
                dots[wave][0] = kk;
                dots[wave][1] = qq;
                dots[wave][2] = kq;
            }
        }
        __syncthreads();
        const float rk = 1.f / sqrtf(dots[0][0] + dots[1][0] + kNormEps), rq = 1.f / sqrtf(dots[0][1] + dots[1][1] + kNormEps);
        const float kq = (dots[0][2] + dots[1][2]) * rk * rq, f = expf(log_sigmoid(gate)), w = sigmoid(beta);
        float x = 0.f, y = 0.f, kv[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            kv[i] = key[wave * R + i];
            x = fmaf(state[i], kv[i], x);
            y = fmaf(state[i], query[wave * R + i], y);
        }
        sums[wave][0][lane] = x;
        sums[wave][1][lane] = y;
        __syncthreads();
        x = ((sums[0][0][lane] + sums[1][0][lane]) + (sums[2][0][lane] + sums[3][0][lane])) * rk;
        y = ((sums[0][1][lane] + sums[1][1][lane]) + (sums[2][1][lane] + sums[3][1][lane])) * rq;
        const float u = w * (v - f * x);
        if (wave == 0 && mine) o[col] = (T)fmaf(kq, u, f * y);
        const float uk = u * rk;
#pragma unroll
        for (int i = 0; i < R; i++) state[i] = fmaf(kv[i], uk, f * state[i]);
    }
    if (whole) {
        float* p = a.last + from;
#pragma unroll
        for (int i = 0; i < R; i++) {
            *p = state[i];
            p += a.V;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; i++)
            if (mine && wave * R + i < a.K) a.last[from + (int64_t)i * a.V] = state[i];
    }
}

// ------------------------------------------------------------------------------------------------------------ backward

// Sums over sixteen lanes of four values each: lanes with e in their last two bits get the sum of value e.
__device__ __forceinline__ float sum_of_16(acc_t v, int lane) {
#define I6_TURN(x, ctrl) __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), ctrl, 0xf, 0xf, false))
    const bool odd = lane & 1, high = lane & 2;
    const float lo = (odd ? v[1] : v[0]) + I6_TURN(odd ? v[0] : v[1], 0xb1), hi = (odd ? v[3] : v[2]) + I6_TURN(odd ? v[2] : v[3], 0xb1);      // with the neighbour
    float x = (high ? hi : lo) + I6_TURN(high ? lo : hi, 0x4e);                                                                               // with the one two further
    x += I6_TURN(x, 0x124);
    x += I6_TURN(x, 0x128);
#undef I6_TURN
    return x;
}

// The gradient of log f of a frame t is what decays over it:  what frames i >= t take from the state in front of the chunk, what frames j < t leave behind it, what goes from the one to
// the other, and M_ij of all pairs j < t <= i within the chunk.  Each of these is added up by itself, of terms that cross the frame and no others.  (Sums over all frames from t on
// of what decays with c_i, less what decays with -c_j, have the same value, but between frames of very different sizes, and where little is left of anything, what cancels
// there is far larger than the result.)
//
// Of a block of M, as an accumulator: on the diagonal the sums for its sixteen t; below it those of its rows, and of its columns.
__device__ __forceinline__ void store_crossing(acc_t v, bool diagonal, float* rows, float* columns) {
    const int lane = threadIdx.x & 63, group = lane >> 4, at = 4 * group;
    const float sum = (v[0] + v[1]) + (v[2] + v[3]);
    const float next = __shfl_down(sum, 16), second = __shfl_down(sum, 32), third = __shfl_down(sum, 48);
    if (diagonal) {
        float below = (group < 3 ? next : 0.f) + (group < 2 ? second : 0.f) + (group < 1 ? third : 0.f);
#pragma unroll
        for (int e = 3; e >= 0; e--) {
            below += v[e];
            v[e] = (lane & 15) < at + e ? below : 0.f;
        }
    } else if (lane < 16) {
        columns[lane] = (sum + next) + (second + third);
    }
    const float of_rows = sum_of_16(v, lane);
    if ((lane & 12) == 0) rows[at + (lane & 3)] = of_rows;
}
// What crosses frame t = lane of a chunk of M blocks; slot(which, block, 0: rows, 1: columns) is where sixteen of these sums are.
template <int M, typename F> __device__ __forceinline__ float crossing(F slot, int lane) {
    const int own = min(lane >> 4, M - 1), r = lane & 15;
    float rows = 0.f, columns = 0.f, across = 0.f, sum = 0.f;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        sum += slot(which, own * (own + 3) / 2, 0)[r];
#pragma unroll
        for (int i = 1; i < M; i++)
#pragma unroll
            for (int j = 0; j < i; j++) {
                const float of_row = slot(which, i * (i + 1) / 2 + j, 0)[r], of_column = slot(which, i * (i + 1) / 2 + j, 1)[r];
                rows += i == own ? of_row : 0.f;
                columns += j == own ? of_column : 0.f;
                across += j < own && own < i ? of_row : 0.f;
            }
    }
#pragma unroll
    for (int m = 1; m < 16; m *= 2) {
        const float behind = __shfl_down(rows, m), before = __shfl_up(columns, m);
        rows += r + m < 16 ? behind : 0.f;
        columns += r >= m ? before : 0.f;
        across += __shfl_xor(across, m);
    }
    const float in_front = __shfl_up(columns, 1);
    return (sum + across) + (rows + (r ? in_front : 0.f));
}
// And of what begins in front of the chunk or ends behind it: of frame t = lane what it takes from the state in front, what it leaves behind the chunk.
template <int C> __device__ __forceinline__ float reaching(float takes, float leaves, int lane) {
#pragma unroll
    for (int m = 1; m < C; m *= 2) {
        const float behind = __shfl_down(takes, m), before = __shfl_up(leaves, m);
        takes += lane + m < C ? behind : 0.f;
        leaves += lane >= m ? before : 0.f;
    }
    const float in_front = __shfl_up(leaves, 1);
    return takes + (lane ? in_front : 0.f);
}

// Four values of a row of a float matrix with V columns; zeros behind them.
__device__ __forceinline__ acc_t load_four(const float* row, int at, int n, bool whole) {
    if (whole) return at < n ? *reinterpret_cast<const acc_t*>(row + at) : acc_t{0.f, 0.f, 0.f, 0.f};
    acc_t v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = at + i < n ? row[at + i] : 0.f;
    return v;
}

// 32 bits: all other gradients of a chunk, from the state in front of it, the gradient of that behind it, U and dR:
//   dq^ = exp(c) dO S0^T + Z K^,   dk^ = exp(c_C - c) U G1^T - w exp(c) dR S0^T + Z^T Q^ + (E + E^T) K^,   Z = D (dO U^T),  E = - w D (dR U^T)
// (lower triangles, E's without its diagonal);  M_ij = Z_ij q_i.k_j + E_ij k_i.k_j.
template <int KP>
__global__ __launch_bounds__(kThreads, 2) void delta_gradients32(Args a, bool whole_k) {
    constexpr int M = kC / 16, N = KP == 128 ? 2 : 1, kV = 128 + 4, kSquare = kC + 4;
    __shared__ __align__(16) float s_o[kC * kV], s_u[kC * kV], s_r[kC * kV], s_z[kC * kSquare], s_e[kC * kSquare];
    __shared__ __align__(16) float s_c[kC], s_rest[kC], s_w[kC], s_rk[kC], s_rq[kC], s_start[kC], s_end[kC], s_dots[4][kC][4], s_whole[4], s_cross[2][M * (M + 1) / 2][2][16];
    const int b = blockIdx.z, h = blockIdx.y, n = blockIdx.x, first = n * kC;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = 4 * (lane >> 4);
    const int len = len_of(a, b), live = min(kC, len - first), rows = min(kC, a.T - first), g = h / (a.H / a.G);
    const int64_t head = (int64_t)b * a.H + h, frame = (int64_t)b * a.T + first;
    const int col = wave * 16 * N + (lane & 15) * N;
    float* dq = static_cast<float*>(a.d_q) + (frame * a.G + g) * a.K;
    float* dk = static_cast<float*>(a.d_k) + (frame * a.G + g) * a.K;
    float* dq_head = a.d_q_head + (frame * a.H + h) * a.K;
    float* dk_head = a.d_k_head + (frame * a.H + h) * a.K;
    const auto store = [&](const acc_t (&v)[M][N], bool keys) {
        if (a.d_q_head) store_columns<N, M>(v, keys ? dk_head : dq_head, (int64_t)a.H * a.K, rows, col, a.K);
        else store_columns<N, M>(v, keys ? dk : dq, (int64_t)a.G * a.K, rows, col, a.K);
    };
    float* d_gate = static_cast<float*>(a.d_gate) + frame * a.H + h;
    float* d_beta = static_cast<float*>(a.d_beta) + frame * a.H + h;
    if (live <= 0) {
        acc_t none[M][N] = {};
        if (col < KP) {
            store(none, false);
            store(none, true);
        }
        if ((int)threadIdx.x < rows) {
            d_gate[threadIdx.x * a.H] = 0.f;
            d_beta[threadIdx.x * a.H] = 0.f;
        }
        return;
    }

    const bool whole = a.V % 4 == 0;
    const int cols = (a.V + 15) / 16 * 16;
    Ahead<KP> in;                        // keys and queries, on their way to where dO and U are first
    in.fetch(a, b, h, first, len, whole_k);
    {
        constexpr int kPerRow = kThreads / kC;
        const int row = threadIdx.x / kPerRow, j = threadIdx.x % kPerRow;
        const float* u = a.u + (head * a.chunks * kC + first + row) * a.V;
        const float* r = a.dr + (head * a.chunks * kC + first + row) * a.V;
        const float* d_o = static_cast<const float*>(a.d_o) + b * a.do_b + (first + row) * a.do_t + h * a.do_h;
        float ru = 0.f;
        for (int c = j * 4; c < cols; c += kPerRow * 4) {
            const acc_t uv = load_four(u, c, a.V, whole), rv = load_four(r, c, a.V, whole);
            acc_t ov;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ov[i] = a.d_o && row < live && c + i < a.V ? d_o[c + i] : 0.f;
                ru = fmaf(uv[i], rv[i], ru);
            }
            *reinterpret_cast<acc_t*>(s_u + row * kV + c) = uv;
            *reinterpret_cast<acc_t*>(s_r + row * kV + c) = rv;
            *reinterpret_cast<acc_t*>(s_o + row * kV + c) = ov;
        }
#pragma unroll
        for (int m = 1; m < kPerRow; m *= 2) ru += __shfl_xor(ru, m);
        // u = w (v - ...), so dw = dR.u / w, times w (1 - w)
        if (j == 0 && row < rows) {
            const float beta = row < live ? static_cast<const float*>(a.beta)[b * a.beta_b + (first + row) * a.beta_t + h * a.beta_h] : 0.f;
            d_beta[row * a.H] = row < live ? ru * sigmoid(-beta) : 0.f;
        }
        if (threadIdx.x < kC) {
            const int i = threadIdx.x;
            const Rows x = a.rows[head * a.chunks * kC + first + i], end = a.rows[head * a.chunks * kC + first + kC - 1];
            s_c[i] = x.c; s_rest[i] = x.c_rest; s_w[i] = x.w; s_rk[i] = x.rk; s_rq[i] = x.rq;
            s_start[i] = exp_fast(x.c);
            s_end[i] = exp_fast((end.c - x.c) + (end.c_rest - x.c_rest));
        }
    }
    __syncthreads();
    const Tile<kV> to{s_o}, tu{s_u}, tr{s_r};
    const Tile<kSquare> tz{s_z}, te{s_e};
    const int blocks = cols / 16;
    acc_t yq[M][N] = {}, yp[M][N] = {}, ym[M][N] = {};
    float crossed = 0.f;                 // <S0, G1>, what decays with c_C
    if (col < KP) {
        const float* states = a.states + (head * a.chunks + n) * a.K * a.V;
        const float* ends = a.ends + (head * a.chunks + n) * a.K * a.V;
#pragma unroll 1
        for (int x = 0; x < blocks; x++) {
            acc_t sv[N], gv[N];
#pragma unroll
            for (int j = 0; j < N; j++) {
                const bool there = col + j < a.K;
                sv[j] = there ? load_four(states + (int64_t)(col + j) * a.V, 16 * x + at, a.V, whole) : acc_t{0.f, 0.f, 0.f, 0.f};
                gv[j] = there ? load_four(ends + (int64_t)(col + j) * a.V, 16 * x + at, a.V, whole) : acc_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; i++) crossed = fmaf(sv[j][i], gv[j][i], crossed);
            }
#pragma unroll
            for (int m = 0; m < M; m++) {
                const acc_t o = to.rows(m, x), r = tr.rows(m, x), u = tu.rows(m, x);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    yq[m][j] = product(o, sv[j], yq[m][j]);
                    yp[m][j] = product(r, sv[j], yp[m][j]);
                    ym[m][j] = product(u, gv[j], ym[m][j]);
                }
            }
        }
        crossed *= s_start[kC - 1];
    }
    acc_t square[2];                     // of Z and E, blocks of the lower triangles in turn
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const int c = wave + 4 * y, which = c & 1, i = block_row(c >> 1), j = (c >> 1) - i * (i + 1) / 2;
        if (c >= M * (M + 1)) continue;
        acc_t v = 0.f;
#pragma unroll 1
        for (int x = 0; x < blocks; x++) v = product(which ? tr.rows(i, x) : to.rows(i, x), tu.rows(j, x), v);
        const int column = 16 * j + (lane & 15), row = 16 * i + at;
        const float cc = s_c[column], rest = s_rest[column], rk = s_rk[column];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int t = row + e;
            const float decay = exp_fast((s_c[t] - cc) + (s_rest[t] - rest));
            const float by = which ? -s_w[t] * s_rk[t] : s_rq[t];
            v[e] = (which ? column < t : column <= t) ? v[e] * decay * rk * by : 0.f;
        }
        (which ? te : tz).put(i, j, v);
        square[y] = v;
    }
    __syncthreads();
    const Tile<kV> tk{s_o}, tq{s_u};     // of dO and U nothing is used any more
    {
        constexpr int kPerRow = Ahead<KP>::kThreadsPerRow;
        const int row = threadIdx.x / kPerRow, j = threadIdx.x % kPerRow;
#pragma unroll
        for (int i = 0; i < Ahead<KP>::kPer; i++) {
            const int c = (i * kPerRow + j) * 4;
            if (c >= KP) continue;
            *reinterpret_cast<acc_t*>(s_o + row * kV + c) = in.k[i];
            *reinterpret_cast<acc_t*>(s_u + row * kV + c) = in.q[i];
        }
    }
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; y++) {        // blocks of M
        const int c = wave + 4 * y, which = c & 1, i = block_row(c >> 1), j = (c >> 1) - i * (i + 1) / 2;
        if (c >= M * (M + 1)) continue;
        acc_t v = 0.f;
#pragma unroll
        for (int x = 0; x < KP / 16; x++) v = product(which ? tk.rows(i, x) : tq.rows(i, x), tk.rows(j, x), v);
        store_crossing(square[y] * v, i == j, s_cross[which][c >> 1][0], s_cross[which][c >> 1][1]);
    }
    acc_t kv[M][N], qv[M][N];
    if (col < KP) {
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int j = 0; j < N; j++) {
                    kv[m][j][e] = s_o[(16 * m + at + e) * kV + col + j];
                    qv[m][j][e] = s_u[(16 * m + at + e) * kV + col + j];
                }
#pragma unroll
        for (int m = 0; m < M; m++) {
            const acc_t start = four(s_start + 16 * m + at), rk = four(s_rk + 16 * m + at);
            const acc_t by_q = start * four(s_rq + 16 * m + at), by_p = -start * rk * four(s_w + 16 * m + at), by_m = four(s_end + 16 * m + at) * rk;
#pragma unroll
            for (int j = 0; j < N; j++) {
                yq[m][j] *= by_q;
                yp[m][j] *= by_p;
                ym[m][j] *= by_m;
            }
            const auto store_dots = [&](int which, acc_t v) {
                const float sum = sum_of_16(v, lane);
                if ((lane & 12) == 0) s_dots[wave][16 * m + at + (lane & 3)][which] = sum;
            };
            {
                acc_t takes = 0.f, leaves = 0.f;
#pragma unroll
                for (int j = 0; j < N; j++) {
                    takes += qv[m][j] * yq[m][j] + kv[m][j] * yp[m][j];
                    leaves += kv[m][j] * ym[m][j];
                }
                store_dots(2, takes);
                store_dots(3, leaves);
            }
#pragma unroll
            for (int x = 0; x <= m; x++) {
                const acc_t z = tz.rows(m, x), e = te.rows(m, x);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    yq[m][j] = product(z, kv[x][j], yq[m][j]);
                    yp[m][j] = product(e, kv[x][j], yp[m][j]);
                }
            }
#pragma unroll
            for (int x = m; x < M; x++) {
                const acc_t z = tz.columns(m, x), e = te.columns(m, x);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    ym[m][j] = product(z, qv[x][j], ym[m][j]);
                    ym[m][j] = product(e, kv[x][j], ym[m][j]);
                }
            }
            acc_t of_q = 0.f, of_k = 0.f;
#pragma unroll
            for (int j = 0; j < N; j++) {
                yp[m][j] += ym[m][j];
                of_q += qv[m][j] * yq[m][j];
                of_k += kv[m][j] * yp[m][j];
            }
            store_dots(0, of_q);
            store_dots(1, of_k);
        }
    } else if ((lane & 15) < 4) {
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) s_dots[wave][16 * m + at + e][lane & 15] = 0.f;
    }
    crossed = wave_sum(crossed);
    if (lane == 0) s_whole[wave] = crossed;
    __syncthreads();
    const auto dot = [&](int row, int i) { return (s_dots[0][row][i] + s_dots[1][row][i]) + (s_dots[2][row][i] + s_dots[3][row][i]); };
    if (col < KP) {
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = 16 * m + at + e;
                const float rq = s_rq[row], rk = s_rk[row];
                const float q_off = rq * rq * dot(row, 0), k_off = rk * rk * dot(row, 1);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    yq[m][j][e] = yq[m][j][e] - qv[m][j][e] * q_off;
                    yp[m][j][e] = yp[m][j][e] - kv[m][j][e] * k_off;
                }
            }
        store(yq, false);
        store(yp, true);
    }
    if (wave == 0) {
        const int t = lane & (kC - 1);
        const float whole_chunk = (s_whole[0] + s_whole[1]) + (s_whole[2] + s_whole[3]);
        const float d = (reaching<kC>(dot(t, 2), dot(t, 3), t) + whole_chunk) + crossing<M>([&](int which, int block, int part) { return s_cross[which][block][part]; }, t);
        if (lane < rows) {
            const float gate = lane < live ? static_cast<const float*>(a.gate)[b * a.gate_b + (first + lane) * a.gate_t + h * a.gate_h] : 0.f;
            d_gate[lane * a.H] = lane < live ? d * sigmoid(-gate) : 0.f;
        }
    }
}

// Gradients of keys and queries that heads share: the sum over these.
template <typename T> __global__ __launch_bounds__(kThreads) void delta_shared(Args a) {
    const int64_t n = (int64_t)a.B * a.T * a.G * a.K;
    const int each = a.H / a.G;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = i / a.K;
        const float* q = a.d_q_head + (row * each) * a.K + i % a.K;
        const float* k = a.d_k_head + (row * each) * a.K + i % a.K;
        float sq = 0.f, sk = 0.f;
        for (int j = 0; j < each; j++) {
            sq += q[(int64_t)j * a.K];
            sk += k[(int64_t)j * a.K];
        }
        static_cast<T*>(a.d_q)[i] = (T)sq;
        static_cast<T*>(a.d_k)[i] = (T)sk;
    }
}

#include "delta_16.inc"
#include "delta_32.inc"

// ---------------------------------------------------------------------------------------------------------------- host

constexpr int kMostFrames = 16;          // frame by frame up to this many, without training
constexpr int kCus = 256;

int checked(const i6delta_problem* p) {
    if (!p || p->B <= 0 || p->T <= 0 || p->H <= 0 || p->G <= 0 || p->K <= 0 || p->V <= 0 || p->H % p->G || !valid_dtype(p->dtype) || !p->q || !p->k || !p->v || !p->gate ||
        !p->beta)
        return I6TRAIN_ERR_INVALID_ARGUMENT;
    if (p->B > 65535 || p->H > 65535 || p->K > 128 || p->V > 128 || p->T > (1 << 28) || (int64_t)p->B * p->H * ceil_div(p->T, kC) > (1 << 23)) return I6TRAIN_ERR_TOO_LARGE;
    return I6TRAIN_OK;
}

Args args_of(const i6delta_problem& p) {
    Args a{};
    a.q = p.q; a.k = p.k; a.v = p.v; a.gate = p.gate; a.beta = p.beta;
    a.q_b = p.q_stride_b; a.q_t = p.q_stride_t; a.q_g = p.q_stride_g;
    a.k_b = p.k_stride_b; a.k_t = p.k_stride_t; a.k_g = p.k_stride_g;
    a.v_b = p.v_stride_b; a.v_t = p.v_stride_t; a.v_h = p.v_stride_h;
    a.gate_b = p.gate_stride_b; a.gate_t = p.gate_stride_t; a.gate_h = p.gate_stride_h;
    a.beta_b = p.beta_stride_b; a.beta_t = p.beta_stride_t; a.beta_h = p.beta_stride_h;
    a.lens = p.seq_lens; a.initial = p.initial;
    a.B = p.B; a.T = p.T; a.H = p.H; a.G = p.G; a.K = p.K; a.V = p.V;
    a.chunks = ceil_div(p.T, p.dtype == I6TRAIN_BF16 ? kC16 : kC);
    return a;
}

// 32 bits: whether rows begin where they can be read in pieces of 16 bytes.
bool whole_floats(const void* x, int64_t s0, int64_t s1, int64_t s2) { return (uintptr_t)x % 16 == 0 && s0 % 4 == 0 && s1 % 4 == 0 && s2 % 4 == 0; }

// bfloat16: whether rows of `cols` values can be read in pieces of 16 bytes; otherwise they are copied first, each in so many values.
bool whole_rows(const void* x, int64_t s0, int64_t s1, int64_t s2, int cols) { return (uintptr_t)x % 16 == 0 && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0 && cols % 8 == 0; }
int packed_row(int cols) { return ceil_div(cols, 8) * 8; }
size_t packed_bytes(const i6delta_problem& p, int heads, int cols) { return align256((size_t)p.B * p.T * heads * packed_row(cols) * sizeof(bf16)); }

int padded_keys(int K) { return K <= 32 ? 32 : (K <= 64 ? 64 : 128); }

// Where the parts of a call's memory are.
struct Places {
    size_t rows, states, u, blocks, kept;                            // kept; rows and blocks are in the forward workspace where nothing is
    size_t packed, forward;                                          // the forward workspace
    size_t ends, dr, d_q, d_k, back_packed, back;                    // the backward workspace
    size_t split, turns;                                             // of the forward workspace, and turns behind split
    size_t back_split;
    int pairs, segments = 1, per;
    Places(const i6delta_problem& p, bool train) {
        const bool x16 = p.dtype == I6TRAIN_BF16;
        const int C = x16 ? kC16 : kC, KP = padded_keys(p.K);
        const size_t n = (size_t)p.B * p.H * ceil_div(p.T, C);
        pairs = p.V > 64 ? 4 : 2;
        const size_t s = align256(x16 ? n * (KP / 16) * pairs * kKept * sizeof(bf16) : n * p.K * p.V * sizeof(float));
        const size_t r = align256(x16 ? n * (C / 16) * pairs * kKept * sizeof(bf16) : n * C * p.V * sizeof(float));
        const size_t heads = p.H > p.G ? align256((size_t)p.B * p.T * p.H * p.K * sizeof(float)) : 0;
        rows = 0;
        states = align256(n * C * sizeof(Rows));
        u = states + s;
        const size_t block_bytes = align256(x16 ? n * chunk_blocks(train) * sizeof(bf16) : n * kBlocks32 * 256 * sizeof(float));
        blocks = train ? u + r : states;
        kept = blocks + block_bytes;
        ends = 0;
        dr = s;
        d_q = dr + r;
        d_k = d_q + heads;
        // whatever their strides are: those of the incoming gradient are not known before it is there
        const size_t k = packed_bytes(p, p.G, p.K), v = packed_bytes(p, p.H, p.V);
        const size_t copy_k = whole_rows(p.k, p.k_stride_b, p.k_stride_t, p.k_stride_g, p.K) ? 0 : k, copy_q = whole_rows(p.q, p.q_stride_b, p.q_stride_t, p.q_stride_g, p.K) ? 0 : k;
        const size_t copy_v = whole_rows(p.v, p.v_stride_b, p.v_stride_t, p.v_stride_h, p.V) ? 0 : v;
        back_packed = d_k + heads;
        back_split = back_packed + (x16 ? copy_k + copy_q + v : 0);
        // Segments: as many as fill the card, and no more than pay for going along them one after the other; below three the second pass costs what the first one saves, and
        // a short sequence does not pay for the launches.  Without and with them, heads of 64 (128): 8 of 2048 frames 142 -> 54 us (225 -> 87), of 512 45 -> 37 (66 -> 52),
        // of 256 28.5 -> 29 (40.6 -> 41.6); 64 of 2048 frames 164 -> 108 (254 -> 208), of 1024 89 -> 67 (136 -> 134), of 512 53 -> 49 (76 -> 91).
        const int chunks = ceil_div(p.T, C);
        const int64_t heads_at_once = (int64_t)p.B * p.H;
        per = chunks;
        if (chunks >= (heads_at_once > 32 ? 16 : 8)) {
            const int most = (int)std::min<int64_t>(kCus / heads_at_once, (int64_t)sqrt(5.0 * chunks));
            if (most >= 3) {
                per = ceil_div(chunks, most);
                segments = ceil_div(chunks, per);
            }
        }
        const size_t slots = (size_t)p.B * p.H * (segments - 1);
        turns = align256(slots * p.K * p.V * sizeof(float));
        const size_t split_bytes = turns + align256(slots * KP * KP * sizeof(float));
        back = back_split + split_bytes;
        // frame by frame nothing is needed
        const bool chunked = train || p.T > kMostFrames;
        packed = chunked && !train ? kept : 0;
        split = chunked ? packed + (x16 ? copy_k + copy_q + copy_v : 0) : 0;
        forward = chunked ? split + split_bytes : 0;
    }
};

struct Call {
    Args a;
    Args16 k16;
    bool whole, whole_v, train;
    bf16* blocks;
};

// Whether a workgroup has all of a head's more than 64 columns: its waves share a unit two by two.  With half the card's units or fewer a head's columns are two workgroups'.
bool wide(const Call& c) { return c.a.V > 64 && (int64_t)c.a.B * c.a.H * c.k16.segments * 2 > kCus; }

template <int KP> void run_forward(const Call& c, hipStream_t s, float) {
    const Args16& k = c.k16;
    float* blocks = reinterpret_cast<float*>(c.blocks);
    delta_prepare32<KP><<<dim3(c.a.chunks, c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, blocks, c.whole);
    const int groups = ceil_div(32 * k.pairs + KP, 128);
    if (k.segments > 1) {
        delta_forward32<KP, 8, true><<<dim3(c.a.H * groups, c.a.B, k.segments - 1), dim3(512), 0, s>>>(c.a, k, blocks, c.whole, c.whole_v);
        delta_join16<KP, kC><<<dim3(ceil_div(c.a.V, 16), c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, k, false);
    }
    if (wide(c)) delta_forward32<KP, 8, false><<<dim3(c.a.H, c.a.B, k.segments), dim3(512), 0, s>>>(c.a, k, blocks, c.whole, c.whole_v);
    else delta_forward32<KP, 4, false><<<dim3(c.a.H * ceil_div(c.a.V, 64), c.a.B, k.segments), dim3(256), 0, s>>>(c.a, k, blocks, c.whole, c.whole_v);
}
template <int KP> void run_forward(const Call& c, hipStream_t s, bf16) {
    delta_prepare16<KP><<<dim3(c.a.chunks, c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, c.blocks, c.train);
    const int stride = chunk_blocks(c.train);
    const Args16& k = c.k16;
    const int groups = ceil_div(32 * k.pairs + KP, 128);
    if (k.segments > 1) {
        delta_forward16<KP, 8, true><<<dim3(c.a.H * groups, c.a.B, k.segments - 1), dim3(512), 0, s>>>(c.a, k, c.blocks, stride);
        delta_join16<KP, kC16><<<dim3(ceil_div(c.a.V, 16), c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, k, false);
    }
    if (wide(c)) delta_forward16<KP, 8, false><<<dim3(c.a.H, c.a.B, k.segments), dim3(512), 0, s>>>(c.a, k, c.blocks, stride);
    else delta_forward16<KP, 4, false><<<dim3(c.a.H * ceil_div(c.a.V, 64), c.a.B, k.segments), dim3(256), 0, s>>>(c.a, k, c.blocks, stride);
}
template <int KP> void run_backward(const Call& c, hipStream_t s, float) {
    const Args16& k = c.k16;
    float* blocks = reinterpret_cast<float*>(c.blocks);
    const int groups = ceil_div(32 * k.pairs + KP, 128);
    if (k.segments > 1) {
        delta_backward32<KP, 8, true><<<dim3(c.a.H * groups, c.a.B, k.segments - 1), dim3(512), 0, s>>>(c.a, k, blocks, c.whole, c.whole_v);
        delta_join16<KP, kC><<<dim3(ceil_div(c.a.V, 16), c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, k, true);
    }
    if (wide(c)) delta_backward32<KP, 8, false><<<dim3(c.a.H, c.a.B, k.segments), dim3(512), 0, s>>>(c.a, k, blocks, c.whole, c.whole_v);
    else delta_backward32<KP, 4, false><<<dim3(c.a.H * ceil_div(c.a.V, 64), c.a.B, k.segments), dim3(256), 0, s>>>(c.a, k, blocks, c.whole, c.whole_v);
    delta_gradients32<KP><<<dim3(c.a.chunks, c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, c.whole);
}
template <int KP> void run_backward(const Call& c, hipStream_t s, bf16) {
    const Args16& k = c.k16;
    const int groups = ceil_div(32 * k.pairs + KP, 128);
    if (k.segments > 1) {
        delta_backward16<KP, 8, true><<<dim3(c.a.H * groups, c.a.B, k.segments - 1), dim3(512), 0, s>>>(c.a, k, c.blocks);
        delta_join16<KP, kC16><<<dim3(ceil_div(c.a.V, 16), c.a.H, c.a.B), dim3(kThreads), 0, s>>>(c.a, k, true);
    }
    if (wide(c)) delta_backward16<KP, 8, false><<<dim3(c.a.H, c.a.B, k.segments), dim3(512), 0, s>>>(c.a, k, c.blocks);
    else delta_backward16<KP, 4, false><<<dim3(c.a.H * ceil_div(c.a.V, 64), c.a.B, k.segments), dim3(256), 0, s>>>(c.a, k, c.blocks);
    if (c.k16.pairs == 4) delta_gradients16<KP, 4><<<dim3(c.a.chunks, c.a.H, c.a.B), dim3(512), 0, s>>>(c.a, c.k16);
    else delta_gradients16<KP, 2><<<dim3(c.a.chunks, c.a.H, c.a.B), dim3(512), 0, s>>>(c.a, c.k16);
}

template <typename T, int KP> int forward(const Call& c, hipStream_t s) {
    const Args& a = c.a;
    if (!c.train && a.T <= kMostFrames) delta_frames<T, KP><<<dim3(ceil_div(a.V, 64), a.H, a.B), dim3(kThreads), 0, s>>>(a);
    else run_forward<KP>(c, s, T());
    return launched();
}

template <typename T, int KP> int backward(const Call& c, hipStream_t s) {
    const Args& a = c.a;
    run_backward<KP>(c, s, T());
    I6TRAIN_TRY(launched());
    if (a.d_q_head) {
        const int64_t n = (int64_t)a.B * a.T * a.G * a.K, groups = ceil_div(n, (int64_t)kThreads);
        delta_shared<T><<<dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(kThreads), 0, s>>>(a);
    }
    return launched();
}

template <typename T> int forward_of(const Call& c, hipStream_t s) {
    switch (padded_keys(c.a.K)) {
        case 32: return forward<T, 32>(c, s);
        case 64: return forward<T, 64>(c, s);
        default: return forward<T, 128>(c, s);
    }
}
template <typename T> int backward_of(const Call& c, hipStream_t s) {
    switch (padded_keys(c.a.K)) {
        case 32: return backward<T, 32>(c, s);
        case 64: return backward<T, 64>(c, s);
        default: return backward<T, 128>(c, s);
    }
}

// Takes the call to a copy of one of its tensors, if that is needed.
int pack(const Args& a, char*& to, const void*& x, int64_t& s0, int64_t& s1, int64_t& s2, int heads, int cols, hipStream_t s) {
    if (whole_rows(x, s0, s1, s2, cols)) return I6TRAIN_OK;
    const int row = packed_row(cols);
    const int64_t rows = (int64_t)a.B * a.T * heads, groups = ceil_div(rows * (row / 8), (int64_t)kThreads);
    delta_pack16<<<dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(kThreads), 0, s>>>(a, Strided{static_cast<const bf16*>(x), s0, s1, s2, heads, cols}, reinterpret_cast<bf16*>(to), row);
    x = to;
    s2 = row;
    s1 = (int64_t)heads * row;
    s0 = (int64_t)a.T * heads * row;
    to += align256((size_t)rows * row * sizeof(bf16));
    return launched();
}

Call call_of(const i6delta_problem& p, const Places& at, void* kept) {
    Call c{};
    c.a = args_of(p);
    c.whole = whole_floats(p.q, p.q_stride_b, p.q_stride_t, p.q_stride_g) && whole_floats(p.k, p.k_stride_b, p.k_stride_t, p.k_stride_g);
    c.whole_v = whole_floats(p.v, p.v_stride_b, p.v_stride_t, p.v_stride_h);
    c.k16.pairs = at.pairs;
    c.k16.segments = at.segments;
    c.k16.per = at.per;
    c.train = kept;
    if (kept) {
        char* base = static_cast<char*>(kept);
        c.a.rows = reinterpret_cast<Rows*>(base + at.rows);
        c.blocks = reinterpret_cast<bf16*>(base + at.blocks);
        c.a.states = reinterpret_cast<float*>(base + at.states);
        c.a.u = reinterpret_cast<float*>(base + at.u);
        c.k16.states = reinterpret_cast<Kept16>(base + at.states);
        c.k16.u = reinterpret_cast<Kept16>(base + at.u);
    }
    return c;
}

}  // namespace
}  // namespace i6train

using namespace i6train;

extern "C" {

int i6delta_sizes(const i6delta_problem* p, int train, size_t* kept_bytes, size_t* forward_bytes, size_t* backward_bytes) {
    I6TRAIN_TRY(checked(p));
    if (!kept_bytes || !forward_bytes || !backward_bytes) return I6TRAIN_ERR_INVALID_ARGUMENT;
    const Places at(*p, train);
    *kept_bytes = train ? at.kept : 0;
    *forward_bytes = at.forward;
    *backward_bytes = train ? at.back : 0;
    return I6TRAIN_OK;
}

int i6delta_forward(const i6delta_problem* p, void* o, float* last, void* kept, size_t kept_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    I6TRAIN_TRY(checked(p));
    if (!o || !last) return I6TRAIN_ERR_INVALID_ARGUMENT;
    const Places at(*p, kept);
    if ((kept && kept_bytes < at.kept) || (at.forward && (!workspace || workspace_bytes < at.forward))) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    Call c = call_of(*p, at, kept);
    c.a.o = o; c.a.last = last;
    if (at.forward) {
        if (!kept) {
            c.a.rows = static_cast<Rows*>(workspace);
            c.blocks = reinterpret_cast<bf16*>(static_cast<char*>(workspace) + at.blocks);
        }
        c.k16.ends = reinterpret_cast<float*>(static_cast<char*>(workspace) + at.split);
        c.k16.turns = reinterpret_cast<float*>(static_cast<char*>(workspace) + at.split + at.turns);
        if (p->dtype == I6TRAIN_BF16) {
            Args& a = c.a;
            char* to = static_cast<char*>(workspace) + at.packed;
            I6TRAIN_TRY(pack(a, to, a.k, a.k_b, a.k_t, a.k_g, a.G, a.K, (hipStream_t)stream));
            I6TRAIN_TRY(pack(a, to, a.q, a.q_b, a.q_t, a.q_g, a.G, a.K, (hipStream_t)stream));
            I6TRAIN_TRY(pack(a, to, a.v, a.v_b, a.v_t, a.v_h, a.H, a.V, (hipStream_t)stream));
        }
    }
    return p->dtype == I6TRAIN_F32 ? forward_of<float>(c, (hipStream_t)stream) : forward_of<bf16>(c, (hipStream_t)stream);
}

int i6delta_backward(const i6delta_problem* p, const void* grad_o, int64_t grad_stride_b, int64_t grad_stride_t, int64_t grad_stride_h, const float* grad_last, const void* kept,
                     size_t kept_bytes, void* grad_q, void* grad_k, void* grad_v, void* grad_gate, void* grad_beta, float* grad_initial, void* workspace,
                     size_t workspace_bytes, void* stream) {
    I6TRAIN_TRY(checked(p));
    if (!kept || !workspace || !grad_q || !grad_k || !grad_v || !grad_gate || !grad_beta) return I6TRAIN_ERR_INVALID_ARGUMENT;
    const Places at(*p, true);
    if (kept_bytes < at.kept || workspace_bytes < at.back) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
    Call c = call_of(*p, at, const_cast<void*>(kept));
    Args& a = c.a;
    a.d_o = grad_o; a.do_b = grad_stride_b; a.do_t = grad_stride_t; a.do_h = grad_stride_h;
    a.d_last = grad_last;
    c.whole_v = whole_floats(grad_o, grad_stride_b, grad_stride_t, grad_stride_h);
    a.d_q = grad_q; a.d_k = grad_k; a.d_v = grad_v; a.d_gate = grad_gate; a.d_beta = grad_beta; a.d_initial = grad_initial;
    char* base = static_cast<char*>(workspace);
    a.ends = reinterpret_cast<float*>(base + at.ends);
    a.dr = reinterpret_cast<float*>(base + at.dr);
    c.k16.left = reinterpret_cast<Kept16>(base + at.ends);
    c.k16.dr = reinterpret_cast<Kept16>(base + at.dr);
    c.k16.ends = reinterpret_cast<float*>(base + at.back_split);
    c.k16.turns = reinterpret_cast<float*>(base + at.back_split + at.turns);
    if (p->dtype == I6TRAIN_BF16) {
        char* to = base + at.back_packed;
        I6TRAIN_TRY(pack(a, to, a.k, a.k_b, a.k_t, a.k_g, a.G, a.K, (hipStream_t)stream));
        I6TRAIN_TRY(pack(a, to, a.q, a.q_b, a.q_t, a.q_g, a.G, a.K, (hipStream_t)stream));
        if (a.d_o) I6TRAIN_TRY(pack(a, to, a.d_o, a.do_b, a.do_t, a.do_h, a.H, a.V, (hipStream_t)stream));
    }
    if (p->H > p->G) {
        a.d_q_head = reinterpret_cast<float*>(base + at.d_q);
        a.d_k_head = reinterpret_cast<float*>(base + at.d_k);
    }
    return p->dtype == I6TRAIN_F32 ? backward_of<float>(c, (hipStream_t)stream) : backward_of<bf16>(c, (hipStream_t)stream);
}

}  // extern "C"
