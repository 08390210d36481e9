// Gated recurrence over the frames of a batch (include/i6train.h):  h_t = f_t h_{t-1} + (1 - f_t) x_t,  f = sigmoid(gate).
//
// A span of frames turns the state c in front of it into A c + H, where A is the product of its f and H its own result
// from c = 0; two neighbouring spans join as (A2 A1, A2 H1 + H2).  So frames need not wait for each other: each wave of a workgroup
// reduces L consecutive frames to (A, H) in registers, the waves exchange these pairs through LDS, every wave joins those of the
// waves before it, and then runs through its frames once more, in registers, from the right state.  A workgroup has 64 V
// channels of one sequence and walks along time, W L frames at a time, the loads of the next frames in flight
// while it works.  The recurrence is bound by memory: forward reads two and writes one value per frame and channel, backward
// reads three and writes two.  Nothing of the forward pass is kept but the state in front of every kStateSpan frames, from
// which backward forms the states again, in 32 bits.
//
// The gradient runs the other way: with d_t the gradient of h_t,  d_t = dh_t + f_{t+1} d_{t+1},  dx_t = (1 - f_t) d_t,
// dgate_t = d_t (h_{t-1} - x_t) f_t (1 - f_t): the same joins, from the end.
//
// Where there are too few (sequence, channel) groups for the chip, a sequence is cut into segments: a first launch reduces each
// segment to its pair (reading the inputs once more, from the caches as far as they fit), a second one starts every segment
// from the pairs of those before it.  No workgroup waits for another.
//
// 32 sequences, 28 800 frames, 1024 channels in bfloat16: forward 45 us (177 MB, 3.9 TB/s), backward 65 us (294 MB, 4.5 TB/s); the workgroups of the longest sequences end
// last.  One recording of 30 000 frames, 512 channels in 32 bits: 23 us for the pairs (123 MB, 5.3 TB/s) and 36 us for the states (184 MB, 5.2 TB/s).
#include "train_common.h"

// Multiply-adds are written out: the instances for single channels and for pairs round alike, so that a result
// does not depend on the strides of its inputs.
#pragma clang fp contract(off)

namespace i6train {
namespace {

constexpr int kStateSpan = 64;          // frames between two states kept for the backward pass

struct Args {
    const void *x, *gate, *dh;
    int64_t x_b, x_t, g_b, g_t, dh_b, dh_t;
    const int32_t* lens;
    const float *initial, *dlast;
    void *h, *dx, *dgate;
    float *last, *states, *dinitial;
    float *seg_a, *seg_h;               // [B][segments][D]
    int B, T, D, n_states, segments, seg_frames;
};

template <typename T, int V> struct Pack;
template <> struct Pack<float, 1> { using type = float; };
template <> struct Pack<float, 2> { using type = float __attribute__((ext_vector_type(2))); };
template <> struct Pack<bf16, 1> { using type = bf16; };
template <> struct Pack<bf16, 2> { using type = bf16 __attribute__((ext_vector_type(2))); };

template <typename T, int V> __device__ __forceinline__ float get(const typename Pack<T, V>::type& p, int v) {
    if constexpr (V == 1) return (float)p; else return (float)p[v];
}
template <typename T, int V> __device__ __forceinline__ void put(T* at, const float (&v)[V]) {
    if constexpr (V == 1) {
        *at = (T)v[0];
    } else {
        typename Pack<T, V>::type p;
        p[0] = (T)v[0]; p[1] = (T)v[1];
        *reinterpret_cast<typename Pack<T, V>::type*>(at) = p;
    }
}

// f and 1 - f, neither by subtraction: both keep their relative precision where the gate is large.  From the instructions for 2^x and 1 / x, each right to an ulp of 32
// bits: f is off by some ulp, which the sums over the frames leave as it is (19 x 437 x 321, all outputs: 2.7e-7 from 64 bits, 4.3e-7 with elementary operations), and a
// correctly rounded exponential and quotient would take several times as many instructions.
__device__ __forceinline__ void sigmoid2(float g, float& f, float& rest) {
    const float q = exp2_fast(-fabsf(g) * kLog2e), r = rcp_fast(1.f + q), s = q * r;
    f = g >= 0.f ? r : s;
    rest = g >= 0.f ? s : r;
}

__device__ __forceinline__ int clamp_len(const Args& a, int b) {
    if (!a.lens) return a.T;
    const int n = a.lens[b];
    return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// V channels of the state c after joining the pairs of `from` .. `to` - 1
template <int V, int W>
__device__ __forceinline__ void join(const float (*lds)[2 * V][64], int lane, int from, int to, float (&c)[V]) {
    for (int w = from; w < to; w++) {
#pragma unroll
        for (int v = 0; v < V; v++) c[v] = fmaf(lds[w][v][lane], c[v], lds[w][V + v][lane]);
    }
}

// kPairs: only the segment's pair (A, H) is wanted.
template <typename T, int V, int W, int L, bool kPairs>
__global__ __launch_bounds__(64 * W) void rec_forward(Args a) {
    using P = typename Pack<T, V>::type;
    __shared__ float lds[2][W][2 * V][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.y, seg = blockIdx.z;
    const int ch = (blockIdx.x * 64 + lane) * V;
    const bool mine = ch < a.D;
    const int at = mine ? ch : 0;
    const int len = clamp_len(a, b);
    const int begin = seg * a.seg_frames, stop = min(a.T, begin + a.seg_frames);
    const int end = min(len, stop);                       // frames of the sequence in this segment: begin .. end - 1
    // rows begin at addresses that are the same for a whole wave; the lanes add their channel
    const T* x = static_cast<const T*>(a.x) + (int64_t)b * a.x_b;
    const T* g = static_cast<const T*>(a.gate) + (int64_t)b * a.g_b;

    float c[V], total_a[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        c[v] = !kPairs && a.initial && mine ? a.initial[(int64_t)b * a.D + at + v] : 0.f;
        total_a[v] = 1.f;
    }
    if (!kPairs) {
        for (int s = 0; s < seg; s++) {
            const int64_t i = ((int64_t)b * a.segments + s) * a.D + at;
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = fmaf(a.seg_a[i + v], c[v], a.seg_h[i + v]);
        }
    }

    P xr[L], gr[L];
    const auto fetch = [&](int t0) {
#pragma unroll
        for (int l = 0; l < L; l++) {
            const int t = min(t0 + wave * L + l, len - 1);      // frames behind the end are not looked at
            xr[l] = *reinterpret_cast<const P*>(x + (int64_t)t * a.x_t + at);
            gr[l] = *reinterpret_cast<const P*>(g + (int64_t)t * a.g_t + at);
        }
    };
    if (begin < end) fetch(begin);
    int buf = 0;
    for (int t0 = begin; t0 < end; t0 += W * L, buf ^= 1) {
        float f[L][V], u[L][V], A[V], H[V];
#pragma unroll
        for (int v = 0; v < V; v++) { A[v] = 1.f; H[v] = 0.f; }
#pragma unroll
        for (int l = 0; l < L; l++) {
            const bool live = t0 + wave * L + l < end;
#pragma unroll
            for (int v = 0; v < V; v++) {
                float fv, rest;
                sigmoid2(get<T, V>(gr[l], v), fv, rest);
                f[l][v] = live ? fv : 1.f;
                u[l][v] = live ? rest * get<T, V>(xr[l], v) : 0.f;
                A[v] *= f[l][v];
                H[v] = fmaf(f[l][v], H[v], u[l][v]);
            }
        }
        if (t0 + W * L < end) fetch(t0 + W * L);
        float mine_c[V];
        if constexpr (W > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                lds[buf][wave][v][lane] = A[v];
                lds[buf][wave][V + v][lane] = H[v];
            }
            __syncthreads();        // one per turn: the other buffer is written in the next one, this one after its barrier
            join<V, W>(lds[buf], lane, 0, wave, c);
#pragma unroll
            for (int v = 0; v < V; v++) mine_c[v] = c[v];
            join<V, W>(lds[buf], lane, wave, W, c);
            if (kPairs) {
                for (int w = 0; w < W; w++)
#pragma unroll
                    for (int v = 0; v < V; v++) total_a[v] *= lds[buf][w][v][lane];
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) {
                mine_c[v] = c[v];
                c[v] = fmaf(A[v], c[v], H[v]);
                total_a[v] *= A[v];
            }
        }
        if (kPairs) continue;
        const int t1 = t0 + wave * L;
        if (a.states && mine && t1 % kStateSpan == 0 && t1 < a.T) {
            const int64_t i = ((int64_t)b * a.n_states + t1 / kStateSpan) * a.D + at;
#pragma unroll
            for (int v = 0; v < V; v++) a.states[i + v] = mine_c[v];
        }
        T* h = static_cast<T*>(a.h) + ((int64_t)b * a.T + t1) * a.D;
#pragma unroll
        for (int l = 0; l < L; l++) {
            const int t = t1 + l;
            float hv[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                mine_c[v] = fmaf(f[l][v], mine_c[v], u[l][v]);
                hv[v] = t < end ? mine_c[v] : 0.f;
            }
            if (mine && t < stop) put<T, V>(h + (int64_t)l * a.D + at, hv);
        }
    }
    if (kPairs) {
        if (mine && wave == 0) {
            const int64_t i = ((int64_t)b * a.segments + seg) * a.D + at;
#pragma unroll
            for (int v = 0; v < V; v++) { a.seg_a[i + v] = total_a[v]; a.seg_h[i + v] = c[v]; }
        }
        return;
    }
    if (!mine) return;
    // frames behind the end that no turn has written
    const int done = begin < end ? begin + ceil_div(end - begin, W * L) * (W * L) : begin;
    const float zero[V] = {};
    for (int t = done + wave; t < stop; t += W) put<T, V>(static_cast<T*>(a.h) + ((int64_t)b * a.T + t) * a.D + at, zero);
    if (seg == a.segments - 1 && wave == 0) {
#pragma unroll
        for (int v = 0; v < V; v++) a.last[(int64_t)b * a.D + at + v] = c[v];
    }
}

template <int V>
__device__ __forceinline__ void join_back(const float (*lds)[64], int lane, float (&c)[V], float (&total_a)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        c[v] = fmaf(lds[v][lane], c[v], lds[2 * V + v][lane]);
        total_a[v] *= lds[v][lane];
    }
}

// kPairs: the segment's pair (A, D) for the gradient that runs from its end to its beginning.
template <typename T, int V, int W, int L, bool kPairs>
__global__ __launch_bounds__(64 * W) void rec_backward(Args a) {
    using P = typename Pack<T, V>::type;
    static_assert(kStateSpan % (W * L) == 0, "a turn starts from a kept state, or from the one the last turn left");
    __shared__ float lds[2][W][3 * V][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.y, seg = blockIdx.z;
    const int ch = (blockIdx.x * 64 + lane) * V;
    const bool mine = ch < a.D;
    const int at = mine ? ch : 0;
    const int len = clamp_len(a, b);
    const int begin = seg * a.seg_frames, stop = min(a.T, begin + a.seg_frames);
    const int end = min(len, stop);
    // rows begin at addresses that are the same for a whole wave; the lanes add their channel
    const T* x = static_cast<const T*>(a.x) + (int64_t)b * a.x_b;
    const T* g = static_cast<const T*>(a.gate) + (int64_t)b * a.g_b;
    const bool has_dh = a.dh;                             // without: the gate is read in its place, and not used
    const T* dh = has_dh ? static_cast<const T*>(a.dh) + (int64_t)b * a.dh_b : g;
    const int64_t dh_t = has_dh ? a.dh_t : a.g_t;

    float c[V], total_a[V];        // c: the gradient of the state behind the frames that are still to come
#pragma unroll
    for (int v = 0; v < V; v++) {
        c[v] = !kPairs && a.dlast && mine ? a.dlast[(int64_t)b * a.D + at + v] : 0.f;
        total_a[v] = 1.f;
    }
    if (!kPairs) {
        for (int s = a.segments - 1; s > seg; s--) {
            const int64_t i = ((int64_t)b * a.segments + s) * a.D + at;
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = fmaf(a.seg_a[i + v], c[v], a.seg_h[i + v]);
        }
    }

    if (!kPairs && mine) {
        // behind the end: zeros
        const float zero[V] = {};
        for (int t = max(begin, end) + wave; t < stop; t += W) {
            const int64_t i = ((int64_t)b * a.T + t) * a.D + at;
            put<T, V>(static_cast<T*>(a.dx) + i, zero);
            put<T, V>(static_cast<T*>(a.dgate) + i, zero);
        }
    }

    P xr[L], gr[L], dr[L];
    float sr[V];
    const auto fetch = [&](int t0) {
#pragma unroll
        for (int l = 0; l < L; l++) {
            const int t = min(t0 + wave * L + l, len - 1);
            gr[l] = *reinterpret_cast<const P*>(g + (int64_t)t * a.g_t + at);
            if (!kPairs) xr[l] = *reinterpret_cast<const P*>(x + (int64_t)t * a.x_t + at);
            dr[l] = *reinterpret_cast<const P*>(dh + (int64_t)t * dh_t + at);
        }
        if (!kPairs) {
            const int64_t i = ((int64_t)b * a.n_states + t0 / kStateSpan) * a.D + at;
#pragma unroll
            for (int v = 0; v < V; v++) sr[v] = a.states[i + v];
        }
    };
    constexpr int kTurn = W * L;
    const int turns = begin < end ? ceil_div(end - begin, kTurn) : 0;
    if (turns) fetch(begin + (turns - 1) * kTurn);
    int buf = 0;
    for (int turn = turns - 1; turn >= 0; turn--, buf ^= 1) {
        const int t0 = begin + turn * kTurn;
        float f[L][V], rest[L][V], xv[L][V], d[L][V], A[V], H[V], G[V], hc[V];
#pragma unroll
        for (int v = 0; v < V; v++) { A[v] = 1.f; H[v] = 0.f; G[v] = 0.f; hc[v] = kPairs ? 0.f : sr[v]; }
#pragma unroll
        for (int l = 0; l < L; l++) {
            const bool live = t0 + wave * L + l < end;
#pragma unroll
            for (int v = 0; v < V; v++) {
                sigmoid2(get<T, V>(gr[l], v), f[l][v], rest[l][v]);
                if (!live) { f[l][v] = 1.f; rest[l][v] = 0.f; }
                xv[l][v] = !kPairs && live ? get<T, V>(xr[l], v) : 0.f;
                d[l][v] = has_dh && live ? get<T, V>(dr[l], v) : 0.f;
                A[v] *= f[l][v];
                H[v] = fmaf(f[l][v], H[v], rest[l][v] * xv[l][v]);
            }
        }
#pragma unroll
        for (int l = L - 1; l >= 0; l--)
#pragma unroll
            for (int v = 0; v < V; v++) G[v] = f[l][v] * (G[v] + d[l][v]);
        if (turn) fetch(t0 - kTurn);
        float mine_c[V];
        if constexpr (W > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                lds[buf][wave][v][lane] = A[v];
                lds[buf][wave][V + v][lane] = H[v];
                lds[buf][wave][2 * V + v][lane] = G[v];
            }
            __syncthreads();
            for (int w = W - 1; w > wave; w--) join_back<V>(lds[buf][w], lane, c, total_a);
#pragma unroll
            for (int v = 0; v < V; v++) mine_c[v] = c[v];
            for (int w = wave; w >= 0; w--) join_back<V>(lds[buf][w], lane, c, total_a);
            if (!kPairs) {
                for (int w = 0; w < wave; w++)
#pragma unroll
                    for (int v = 0; v < V; v++) hc[v] = fmaf(lds[buf][w][v][lane], hc[v], lds[buf][w][V + v][lane]);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) {
                mine_c[v] = c[v];
                c[v] = fmaf(A[v], c[v], G[v]);
                total_a[v] *= A[v];
            }
        }
        if (kPairs) continue;
        float before[L][V];
#pragma unroll
        for (int l = 0; l < L; l++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                before[l][v] = hc[v];
                hc[v] = fmaf(f[l][v], hc[v], rest[l][v] * xv[l][v]);
            }
        const int64_t row = ((int64_t)b * a.T + t0 + wave * L) * a.D;
#pragma unroll
        for (int l = L - 1; l >= 0; l--) {
            float dx[V], dg[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float dv = d[l][v] + mine_c[v];
                dx[v] = rest[l][v] * dv;
                dg[v] = dv * (before[l][v] - xv[l][v]) * (f[l][v] * rest[l][v]);
                mine_c[v] = f[l][v] * dv;
            }
            if (mine && t0 + wave * L + l < end) {
                put<T, V>(static_cast<T*>(a.dx) + row + (int64_t)l * a.D + at, dx);
                put<T, V>(static_cast<T*>(a.dgate) + row + (int64_t)l * a.D + at, dg);
            }
        }
    }
    if (!mine || wave != 0) return;
    if (kPairs) {
        const int64_t i = ((int64_t)b * a.segments + seg) * a.D + at;
#pragma unroll
        for (int v = 0; v < V; v++) { a.seg_a[i + v] = total_a[v]; a.seg_h[i + v] = c[v]; }
    } else if (seg == 0 && a.dinitial) {
#pragma unroll
        for (int v = 0; v < V; v++) a.dinitial[(int64_t)b * a.D + at + v] = c[v];
    }
}

// ------------------------------------------------------------------------------------------------------------- host

constexpr int kUnits = 256;             // compute units
constexpr int kMostSegments = 64, kLeastSegment = 128;

// Channels of a lane.  Pairs are for many workgroups, so their sequences are in one piece.  64 floats are a row of 256 bytes for a wave; of bfloat16, pairs are, unless the workgroups are then fewer than the compute
// units: single channels are twice as many with half the work each (training, 16 x 2000 x 1024: 147 us, pairs 164 us; 1 x 4000 x 512: 42 and 55 us; but
// 32 x 1000 x 1024: 124 and 110 us).
int vector_width(const i6train_rec_problem& p, const void* dh, int64_t dh_b, int64_t dh_t) {
    if (p.dtype != I6TRAIN_BF16 || (int64_t)p.B * ceil_div(p.D, 128) < kUnits) return 1;
    const auto even = [](const void* q, int64_t sb, int64_t st) { return (uintptr_t)q % 4 == 0 && sb % 2 == 0 && st % 2 == 0; };
    return p.D % 2 == 0 && even(p.x, p.x_stride_b, p.x_stride_t) && even(p.gate, p.gate_stride_b, p.gate_stride_t) && even(dh, dh_b, dh_t) ? 2 : 1;
}

// Segments of whole state spans: one, unless the (sequence, channel) groups leave compute units idle; then enough for two workgroups on each, of at least
// kLeastSegment frames, and at least three, as the first launch goes through all of them as well.  (Training, float, 1 x 1000 x 512: 27 us, 38 us with 256 frames at least, 66 us in one
// piece; 19 x 437 x 321, where there is little to gain: 44 us, and 40 us in one piece.)
void cut(const i6train_rec_problem& p, int& segments, int& seg_frames) {
    const int64_t groups = (int64_t)p.B * ceil_div(p.D, 64);
    int64_t n = 1;
    if (groups < kUnits) {
        n = ceil_div((int64_t)2 * kUnits, groups);
        n = n < kMostSegments ? n : kMostSegments;
        const int64_t room = ceil_div(p.T, kLeastSegment);
        n = n < room ? n : room;
        if (n < 3) n = 1;
    }
    seg_frames = (int)(ceil_div(ceil_div((int64_t)p.T, n), (int64_t)128) * 128);
    segments = (int)ceil_div(p.T, seg_frames);
}

bool valid(const i6train_rec_problem* p) {
    return p && p->B > 0 && p->T > 0 && p->D > 0 && p->B <= 65535 && valid_dtype(p->dtype) && p->x && p->gate && p->T <= (1 << 30);
}

int checked(const i6train_rec_problem* p) {
    if (!valid(p)) return I6TRAIN_ERR_INVALID_ARGUMENT;
    return launchable(ceil_div(p->D, 64), 512) ? I6TRAIN_OK : I6TRAIN_ERR_TOO_LARGE;
}

int n_states(const i6train_rec_problem& p) { return ceil_div(p.T, kStateSpan); }

Args args_of(const i6train_rec_problem& p) {
    Args a{};
    a.x = p.x; a.gate = p.gate;
    a.x_b = p.x_stride_b; a.x_t = p.x_stride_t; a.g_b = p.gate_stride_b; a.g_t = p.gate_stride_t;
    a.lens = p.seq_lens; a.initial = p.initial;
    a.B = p.B; a.T = p.T; a.D = p.D; a.n_states = n_states(p);
    return a;
}

template <typename T, int V> int forward(Args a, hipStream_t s) {
    const dim3 grid(ceil_div(a.D, 64 * V), a.B, a.segments);
    // few frames: one wave, no exchange
    if (a.T == 1) {
        rec_forward<T, V, 1, 1, false><<<grid, dim3(64), 0, s>>>(a);
    } else if (a.T <= 16) {
        rec_forward<T, V, 1, 4, false><<<grid, dim3(64), 0, s>>>(a);
    } else {
        if constexpr (V == 1)
            if (a.segments > 1) rec_forward<T, 1, 8, 16, true><<<grid, dim3(512), 0, s>>>(a);
        rec_forward<T, V, 8, 16, false><<<grid, dim3(512), 0, s>>>(a);
    }
    return launched();
}

template <typename T, int V> int backward(Args a, hipStream_t s) {
    const dim3 grid(ceil_div(a.D, 64 * V), a.B, a.segments);
    if constexpr (V == 1)
        if (a.segments > 1) rec_backward<T, 1, 8, 8, true><<<grid, dim3(512), 0, s>>>(a);
    rec_backward<T, V, 8, 8, false><<<grid, dim3(512), 0, s>>>(a);
    return launched();
}

size_t segment_bytes(const i6train_rec_problem& p) { return align256(sizeof(float) * (size_t)p.B * kMostSegments * p.D); }

}  // namespace
}  // namespace i6train

using namespace i6train;

extern "C" {

int i6train_rec_states_size(const i6train_rec_problem* p, size_t* bytes) {
    I6TRAIN_TRY(checked(p));
    if (!bytes) return I6TRAIN_ERR_INVALID_ARGUMENT;
    *bytes = sizeof(float) * (size_t)p->B * n_states(*p) * p->D;
    return I6TRAIN_OK;
}

int i6train_rec_workspace_size(const i6train_rec_problem* p, size_t* bytes) {
    I6TRAIN_TRY(checked(p));
    if (!bytes) return I6TRAIN_ERR_INVALID_ARGUMENT;
    int n, f;
    cut(*p, n, f);
    *bytes = n > 1 ? 2 * segment_bytes(*p) : 0;
    return I6TRAIN_OK;
}

int i6train_rec_forward(const i6train_rec_problem* p, void* h, float* last, float* states, void* workspace, size_t workspace_bytes, void* stream) {
    I6TRAIN_TRY(checked(p));
    if (!h || !last) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Args a = args_of(*p);
    a.h = h; a.last = last; a.states = states;
    const int V = vector_width(*p, nullptr, 0, 0);
    cut(*p, a.segments, a.seg_frames);
    if (a.segments > 1) {
        if (!workspace || workspace_bytes < 2 * segment_bytes(*p)) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
        a.seg_a = static_cast<float*>(workspace);
        a.seg_h = reinterpret_cast<float*>(static_cast<char*>(workspace) + segment_bytes(*p));
    }
    hipStream_t s = (hipStream_t)stream;
    if (p->dtype == I6TRAIN_F32) return forward<float, 1>(a, s);
    return V == 2 ? forward<bf16, 2>(a, s) : forward<bf16, 1>(a, s);
}

int i6train_rec_backward(const i6train_rec_problem* p, const void* grad_h, int64_t grad_stride_b, int64_t grad_stride_t,
                         const float* grad_last, const float* states, void* grad_x, void* grad_gate, float* grad_initial,
                         void* workspace, size_t workspace_bytes, void* stream) {
    I6TRAIN_TRY(checked(p));
    if (!states || !grad_x || !grad_gate) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Args a = args_of(*p);
    a.dh = grad_h; a.dh_b = grad_stride_b; a.dh_t = grad_stride_t;
    a.dlast = grad_last; a.states = const_cast<float*>(states);
    a.dx = grad_x; a.dgate = grad_gate; a.dinitial = grad_initial;
    const int V = vector_width(*p, grad_h, grad_stride_b, grad_stride_t);
    cut(*p, a.segments, a.seg_frames);
    if (a.segments > 1) {
        if (!workspace || workspace_bytes < 2 * segment_bytes(*p)) return I6TRAIN_ERR_WORKSPACE_TOO_SMALL;
        a.seg_a = static_cast<float*>(workspace);
        a.seg_h = reinterpret_cast<float*>(static_cast<char*>(workspace) + segment_bytes(*p));
    }
    hipStream_t s = (hipStream_t)stream;
    if (p->dtype == I6TRAIN_F32) return backward<float, 1>(a, s);
    return V == 2 ? backward<bf16, 2>(a, s) : backward<bf16, 1>(a, s);
}

}  // extern "C"
