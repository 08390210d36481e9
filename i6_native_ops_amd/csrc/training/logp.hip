// Log probabilities of given classes, entropy and best alternatives of every frame, from the scores of all classes (include/i6logp.h).
//
// Bound by memory: every score is read once and stays in the registers of the threads that share its row (a wave, or a workgroup for longer rows; rows beyond what
// 512 threads hold are read again for each of the passes below, from the caches).  Passes over the registers: the largest score m; the sums
// of e = exp(z - m) and e (z - m), the terms that are equal to the largest apart from the others, so that log p of a confident frame's class, log1p of the others'
// sum, and its entropy keep their relative precision; and the alternatives.
//
// Alternatives: the k-th largest of a wave's 64 lanes' largest scores is a bound that at least k scores of the row reach.  What reaches the
// largest such bound of the row's waves is a candidate; candidates go to LDS, and a candidate's place is the number of those before it.  Where more than
// kCandidates scores reach the bound, the k-th largest score itself is found bit by bit, and then the index up to
// which scores equal to it count: what is left are k candidates.  That is so for masked, equal and ordered scores, and also for any with many alternatives, as the bound is one
// wave's and more scores reach it the more waves a row has: from about 60 alternatives on where a row is one wave's, 45 at 12 001 classes, 30 at 20 000, 20 at 30 000 and more.  It
// takes some forty passes over the row: 4096 rows of 12 001 in 32 bits 43 us with 8 alternatives, 82 with 32 and 1000 with 48, of 30 000 257 with 16 and 2700 with 24.
//
// Backward, what every class has of the frame's sums is written, and then the classes that something comes in for are written again, by their numbers.
//
// 28 900 frames of 12 001 classes in 32 bits: 250 us, 5.5 TB/s, and all of the time vector instructions are issued, too.  Training on 44 800 frames of 5001 in 16 bits: 151 us
// forward (3 TB/s; ten instructions and an exponential a score) and 177 backward (5.4 TB/s with what is written).  The next frame of 64 streams: 15 us, most of which two barriers,
// the reductions and a row's first bytes take.  Rows of more than 24 576 classes (bfloat16 49 152) are not held: 4096 of 128 256 in 32 bits 855 us with 8 alternatives, 2.5 TB/s; 64 of them 44 us.
#include "train_common.h"
#include "../../../include/i6logp.h"

namespace i6train {
namespace {

constexpr int kCandidates = 256, kMany = 4096;
#define I6_INLINE __attribute__((always_inline))

struct Args {
    const void* logits;
    int64_t l_b, l_t;
    const int32_t* targets;
    int64_t t_b, t_t;
    const int32_t* lens;
    int B, T, F, k;
    float *log_prob, *entropy, *top;
    int32_t* top_class;
    float* statistics;                   // m, log of the sum, entropy, and whether there is a distribution
    int* report;
    const float *g_log_prob, *g_entropy, *g_top;
    void* grad;
};

// In statistics.
constexpr float kFine = 0.f, kEmpty = 1.f, kBad = 2.f;

// An order of whole numbers that is that of the floats, NaN aside; -0 and 0 are the same score.
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.f);
    return b ^ (uint32_t)((int32_t)b >> 31 | 0x80000000);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <typename T> constexpr int kPiece = 16 / sizeof(T);
template <typename T> using Vector = T __attribute__((ext_vector_type(16 / sizeof(T))));

// A row in pieces of 16 aligned bytes: `head` scores in front of the first, `pieces` of them, the rest behind.  A thread has pieces `thread`, `thread` + threads, ...
// and at most one of the scores in front and behind.
template <typename T> struct Row {
    const T* p;
    int head, pieces, rest, F;
    __device__ __forceinline__ Row(const T* row, int F) : p(row), F(F) {
        head = min(F, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
        pieces = (F - head) / kPiece<T>;
        rest = F - head - pieces * kPiece<T>;
    }
    // index of the single score of `thread`, or -1
    __device__ __forceinline__ int single(int thread) const { return thread < head ? thread : (thread < head + rest ? F - rest + (thread - head) : -1); }
    __device__ __forceinline__ Vector<T> piece(int i) const { return *reinterpret_cast<const Vector<T>*>(p + head + (int64_t)i * kPiece<T>); }
};

// Threads that share a row: one wave of four, or a whole workgroup.
template <int kThreads> struct Team {
    static constexpr int kWaves = kThreads / 64;
    static __device__ __forceinline__ int thread() { return kWaves == 1 ? threadIdx.x & 63 : threadIdx.x; }
    static __device__ __forceinline__ void meet() {
        if (kWaves == 1) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        } else {
            __syncthreads();
        }
    }
};

template <int kThreads> struct Shared {
    float part[3][16];
    uint32_t bound[16], count;
    float value[kCandidates];
    int index[kCandidates];
};

// kHeld: pieces of a thread that are kept in registers; 0: none, they are read again for every pass
template <typename T, int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void logp_forward(Args a) {
    using G = Team<kThreads>;
    constexpr int kWaves = G::kWaves, kTeams = kWaves == 1 ? 4 : 1, P = kPiece<T>;
    __shared__ Shared<kThreads> all[kTeams];
    const int team = kWaves == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    Shared<kThreads>& s = all[team];
    const int64_t frame = (int64_t)blockIdx.x * kTeams + team;
    if (frame >= (int64_t)a.B * a.T) return;
    const int thread = G::thread(), lane = threadIdx.x & 63, wave = kWaves == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = (int)((uint32_t)frame / (uint32_t)a.T), t = (int)((uint32_t)frame % (uint32_t)a.T), k = a.k;
    if (t >= a.lens[b]) {
        if (thread == 0) {
            a.log_prob[frame] = 0.f;
            a.entropy[frame] = 0.f;
        }
        if (thread < k) {
            a.top[frame * k + thread] = 0.f;
            a.top_class[frame * k + thread] = -1;
        }
        return;
    }
    const Row<T> row(static_cast<const T*>(a.logits) + b * a.l_b + t * a.l_t, a.F);
    Vector<T> held[kHeld ? kHeld : 1];
    const int single_at = row.single(thread);
    const float single = single_at >= 0 ? (float)row.p[single_at] : -INFINITY;
    if (kHeld) {
#pragma unroll
        for (int i = 0; i < kHeld; i++) {
            const int at = i * kThreads + thread;
            if (at < row.pieces) {
                held[i] = row.piece(at);
            } else {
#pragma unroll
                for (int e = 0; e < P; e++) held[i][e] = (T)-INFINITY;
            }
        }
    }
    const int y = a.targets[b * a.t_b + t * a.t_t];
    const float picked = thread == 0 && y >= 0 && y < a.F ? (float)row.p[y] : 0.f;

    // f(piece, index of its first score) for all pieces of this thread, those behind the row's end with index F and -inf; then the single score.  All lanes of a
    // wave together
    const auto read_pieces = [&](auto f) I6_INLINE {
        for (int first = 0; first < row.pieces; first += kThreads) {
            const int at = first + thread;
            Vector<T> v;
#pragma unroll
            for (int e = 0; e < P; e++) v[e] = (T)-INFINITY;
            if (at < row.pieces) v = row.piece(at);
            f(v, at < row.pieces ? row.head + at * P : a.F);
        }
    };
    const auto pieces = [&](auto f) I6_INLINE {
        if constexpr (kHeld > 0) {
#pragma unroll
            for (int i = 0; i < kHeld; i++) {
                const int at = i * kThreads + thread;
                f(held[i], at < row.pieces ? row.head + at * P : a.F, i);
                __builtin_amdgcn_sched_barrier(0);             // a few registers besides those of the row
            }
        } else {
            read_pieces([&](const Vector<T>& v, int at) I6_INLINE { f(v, at, 0); });
        }
    };
    // what one pass makes of the scores is not kept for the next
    const auto forget = [&] {
        if constexpr (kHeld > 0) {
#pragma unroll
            for (int i = 0; i < kHeld; i++) asm volatile("" : "+v"(held[i]));
        }
    };
    // the passes below look at a piece's largest first; it is kept for pieces of eight, of four it is formed again
    constexpr bool kKeep = kHeld > 0 && P == 8;
    float most = single, kept[kKeep ? kHeld : 1];              // (NaN is seen by the sums)
    const auto largest_of = [&](const Vector<T>& v) I6_INLINE {
        float x = fmaxf((float)v[0], (float)v[1]);
#pragma unroll
        for (int e = 2; e < P; e += 2) x = fmaxf(fmaxf((float)v[e], (float)v[e + 1]), x);
        return x;
    };
    pieces([&](const Vector<T>& v, int, int i) I6_INLINE {
        const float x = largest_of(v);
        if (kKeep) kept[i] = x;
        most = fmaxf(most, x);
    });
    const auto best_of = [&](const Vector<T>& v, int i) I6_INLINE { return kKeep ? kept[i] : largest_of(v); };

    // a bound that k scores reach: the k-th largest of the lanes' largest, to 16 bits
    uint32_t bound = 0;
    if (k > 0) {
        const uint32_t key = key_of(most);
#pragma unroll
        for (int bit = 31; bit >= 16; bit--) {
            const uint32_t more = bound | (1u << bit);
            if (__builtin_popcountll(__ballot(key >= more)) >= k) bound = more;
        }
    }
    const auto max_of = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    float m = of_key(wave_reduce(key_of(most), 0, max_of));
    if (kWaves > 1) {
        if (lane == 0) {
            s.part[0][wave] = m;
            s.bound[wave] = bound;
        }
        if (thread == 0) s.count = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            m = fmaxf(m, s.part[0][w]);
            bound = max_of(bound, s.bound[w]);
        }
    } else if (lane == 0) {
        s.count = 0;
    }

    // sums over the scores but the largest, and how many of those there are
    float rest = 0.f, more = 0.f, moment = 0.f, more_moment = 0.f;
    int n = 0;
    const auto add = [&](float z, float& sum, float& sum_moment) I6_INLINE {
        const float d = z - m;
        const bool largest = z == m;
        if (kWaves == 1) n += largest;                           // its lane's, or its wave's: by what is waited for
        else n += __builtin_popcountll(__ballot(largest));
        const float e = largest ? 0.f : exp2_fast(d * kLog2e);
        sum += e;
        sum_moment = fmaf(e, fmaxf(d, -1e30f), sum_moment);      // (0 times -inf)
    };
    const auto add_smaller = [&](float z, float& sum, float& sum_moment) I6_INLINE {
        const float d = z - m, e = exp2_fast(d * kLog2e);
        sum += e;
        sum_moment = fmaf(e, fmaxf(d, -1e30f), sum_moment);
    };
    forget();
    pieces([&](const Vector<T>& v, int, int i) I6_INLINE {
        // With the largest score in it: one piece of a wave, for the most part.  (32 bits by workgroups: asking costs more than it saves, 142 us for 16 384 rows of 12 001 instead
        // of 134; 16 bits 115 instead of 150.)
        if (kHeld == 0 || (P == 4 && kWaves > 1) || __any(best_of(v, i) == m)) {
#pragma unroll
            for (int e = 0; e < P; e += 2) {
                add((float)v[e], rest, moment);
                add((float)v[e + 1], more, more_moment);
            }
        } else {
#pragma unroll
            for (int e = 0; e < P; e += 2) {
                add_smaller((float)v[e], rest, moment);
                add_smaller((float)v[e + 1], more, more_moment);
            }
        }
    });
    add(single, rest, moment);
    rest += more;
    moment += more_moment;
    rest = wave_sum(rest);
    moment = wave_sum(moment);
    float equal = kWaves == 1 ? wave_sum((float)n) : (float)n; // (exact up to 2^24 a wave, that is, for all rows there are)
    if (kWaves > 1) {
        // part[0] is read by all before the waves meet below, and these are other places
        if (lane == 0) {
            s.part[1][wave] = rest;
            s.part[2][wave] = moment;
        }
        __syncthreads();
        if (lane == 0) s.part[0][wave] = equal;
        rest = moment = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            rest += s.part[1][w];
            moment += s.part[2][w];
        }
    }
    // Candidates, whichever lanes of a wave have one.
    const auto keep = [&](float z, int at, bool is) I6_INLINE {
        const uint64_t mask = __ballot(is);
        if (!mask) return;
        uint32_t slot = 0;
        if (lane == 0) slot = atomicAdd(&s.count, (uint32_t)__builtin_popcountll(mask));
        slot = __builtin_amdgcn_readfirstlane(slot) + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        if (is && slot < (uint32_t)kCandidates) {
            s.value[slot] = z;
            s.index[slot] = at;
        }
    };
    forget();
    if (k > 0) {
        const float least = of_key(bound < 0x007fffffu ? 0x007fffffu : bound);      // -inf at least
        if (kWaves == 1) G::meet();
        pieces([&](const Vector<T>& v, int at, int i) I6_INLINE {
            if (!__any(best_of(v, i) >= least)) return;
#pragma unroll
            for (int e = 0; e < P; e++) keep((float)v[e], at + e, (float)v[e] >= least && at < a.F);
        });
        keep(single, single_at, single >= least && single_at >= 0);
    }
    G::meet();
    if (kWaves > 1) {
        equal = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) equal += s.part[0][w];
    }
    // every thread has the same sums from here on
    float state = kFine;
    if (m == -INFINITY) state = kEmpty;
    if (m == INFINITY || rest != rest) state = kBad;
    const float ratio = rest / equal, log_total = log2_fast(equal) * kLn2 + log1pf(ratio), total = equal + rest;
    const float entropy = state == kFine ? log_total - moment / total : (state == kEmpty ? 0.f : __builtin_nanf(""));
    const auto log_p = [&](float z) I6_INLINE { return state == kFine ? (z - m) - log_total : (state == kEmpty ? -INFINITY : __builtin_nanf("")); };
    if (thread == 0) {
        float v = y < 0 ? 0.f : log_p(picked);
        if (y >= a.F) {
            v = __builtin_nanf("");
            if (a.report) {
                __hip_atomic_store(a.report + 1, b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
                __hip_atomic_store(a.report, I6TRAIN_ERR_BAD_TARGET, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
            }
        }
        a.log_prob[frame] = v;
        a.entropy[frame] = entropy;
        if (a.statistics) {
            float* to = a.statistics + frame * 4;
            to[0] = m; to[1] = log_total; to[2] = entropy; to[3] = state;
        }
    }
    if (k == 0) return;
    if (state == kBad) {
        if (thread < k) {
            a.top[frame * k + thread] = __builtin_nanf("");
            a.top_class[frame * k + thread] = -1;
        }
        return;
    }
    int count = (int)s.count;
    if (count > kCandidates) {
        // from memory, all scores: with what this needs, rows that never come here would not keep theirs in registers
        const auto each = [&](auto f) I6_INLINE {
            read_pieces([&](const Vector<T>& v, int at) I6_INLINE {
#pragma unroll
                for (int e = 0; e < P; e++) f((float)v[e], at + e);
            });
            f(single, single_at >= 0 ? single_at : a.F);
        };
        const auto counted = [&](auto f) I6_INLINE {                     // of the row's scores, those with f
            uint32_t sum = 0;
            each([&](float z, int at) I6_INLINE { sum += __builtin_popcountll(__ballot(at < a.F && f(z, at))); });
            if (kWaves > 1) {
                __syncthreads();
                if (lane == 0) s.bound[wave] = sum;
                __syncthreads();
                sum = 0;
#pragma unroll
                for (int w = 0; w < kWaves; w++) sum += s.bound[w];
            }
            return (int)sum;
        };
        // between the bound and the largest score; with fewer than k scores above -inf it is that
        const uint32_t lowest = 0x007fffffu, top = key_of(m);
        uint32_t kth = lowest;
        if (bound > lowest || counted([&](float z, int) I6_INLINE { return key_of(z) > lowest; }) >= k) {
            const int same = bound == top ? 0 : 32 - __builtin_clz(bound ^ top);      // bits in which the two differ, and those behind
            kth = same == 32 ? 0 : bound >> same << same;
            for (int bit = same - 1; bit >= 0; bit--) {
                const uint32_t next = kth | (1u << bit);
                if (counted([&](float z, int) I6_INLINE { return key_of(z) >= next; }) >= k) kth = next;
            }
        }
        // the scores that are larger, and equal ones up to the index `last`
        const int ties = k - counted([&](float z, int) I6_INLINE { return key_of(z) > kth; });
        int last = 0;
        for (int bit = 31 - __builtin_clz(a.F); bit >= 0; bit--) {
            const int next = last + (1 << bit);
            if (next < a.F && counted([&](float z, int at) I6_INLINE { return key_of(z) == kth && at < next; }) < ties) last = next;
        }
        G::meet();
        if (thread == 0) s.count = 0;
        G::meet();
        each([&](float z, int at) I6_INLINE {
            const uint32_t key = key_of(z);
            keep(z, at, at < a.F && (key > kth || (key == kth && at <= last)));
        });
        G::meet();
        count = min((int)s.count, kCandidates);
    }
    for (int c = thread; c < count; c += kThreads) {
        const float z = s.value[c];
        const int at = s.index[c];
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < count; i++) {
            const float other = s.value[i];
            place += other > z || (other == z && s.index[i] < at);
        }
        if (place < k) {
            a.top[frame * k + place] = log_p(z);
            a.top_class[frame * k + place] = at;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ backward

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void logp_backward(Args a) {
    using G = Team<kThreads>;
    constexpr int kTeams = G::kWaves == 1 ? 4 : 1, P = kPiece<T>, kList = I6LOGP_MOST_ALTERNATIVES + 1;
    __shared__ int all_class[kTeams][kList];
    __shared__ float all_more[kTeams][kList];
    const int team = kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t frame = (int64_t)blockIdx.x * kTeams + team;
    if (frame >= (int64_t)a.B * a.T) return;
    int* classes = all_class[team];
    float* mores = all_more[team];
    const int thread = G::thread(), b = (int)((uint32_t)frame / (uint32_t)a.T), t = (int)((uint32_t)frame % (uint32_t)a.T), k = a.k;
    T* to = static_cast<T*>(a.grad) + frame * a.F;
    const Row<T> out(to, a.F);
    const int single = out.single(thread);
    const auto fill = [&](float v) {
        Vector<T> p;
#pragma unroll
        for (int e = 0; e < P; e++) p[e] = (T)v;
        for (int i = thread; i < out.pieces; i += kThreads) *reinterpret_cast<Vector<T>*>(to + out.head + (int64_t)i * P) = p;
        if (single >= 0) to[single] = (T)v;
    };
    if (t >= a.lens[b]) return fill(0.f);
    const float* statistics = a.statistics + frame * 4;
    const float m = statistics[0], log_total = statistics[1], entropy = statistics[2], state = statistics[3];
    const int y = a.targets[b * a.t_b + t * a.t_t];
    if (state == kEmpty && y < a.F) return fill(0.f);
    if (state != kFine || y >= a.F) return fill(__builtin_nanf(""));
    const float gl = a.g_log_prob && y >= 0 ? a.g_log_prob[frame] : 0.f, ge = a.g_entropy ? a.g_entropy[frame] : 0.f;
    const int lane = threadIdx.x & 63;
    const float gt = a.g_top && lane < k ? a.g_top[frame * k + lane] : 0.f, sum = gl + wave_sum(gt);
    if (thread < k) {
        classes[thread] = a.top_class[frame * k + thread];
        mores[thread] = gt;
    }
    if (thread == 0) {
        classes[k] = y;
        mores[k] = gl;
    }
    // - p (gl + sum gt + ge (log p + entropy)).  Below -200 p is 0 and log p only has to be a number whose product with ge is one, too
    const auto share = [&](float z) {
        const float log_p = (z - m) - log_total, p = exp2_fast(log_p * kLog2e);
        return -p * fmaf(ge, fmaxf(log_p, -200.f) + entropy, sum);
    };
    const T* from = static_cast<const T*>(a.logits) + b * a.l_b + t * a.l_t;
    if ((((uintptr_t)from ^ (uintptr_t)to) & 15) == 0) {
#pragma unroll 4
        for (int i = thread; i < out.pieces; i += kThreads) {
            const int at = out.head + i * P;
            const Vector<T> z = *reinterpret_cast<const Vector<T>*>(from + at);
            Vector<T> v;
#pragma unroll
            for (int e = 0; e < P; e++) v[e] = (T)share((float)z[e]);
            *reinterpret_cast<Vector<T>*>(to + at) = v;
        }
        if (single >= 0) to[single] = (T)share((float)from[single]);
    } else {
        for (int i = thread; i < a.F; i += kThreads) to[i] = (T)share((float)from[i]);
    }
    G::meet();
    for (int i = thread; i <= k; i += kThreads) {
        const int c = classes[i];
        if (c < 0 || c >= a.F) continue; // (none: a caller's alternatives may be anything)
        float more = 0.f;                // a target may be an alternative; then both write the same
        for (int j = 0; j <= k; j++) more += classes[j] == c ? mores[j] : 0.f;
        // Where p is next to 1 with 1 - p from log p, so that a confident frame's difference keeps its relative precision; below one half more - p (...) is one rounding and
        // nothing cancels
        const float log_p = ((float)from[c] - m) - log_total, p = exp2_fast(log_p * kLog2e), of_entropy = fmaxf(log_p, -200.f) + entropy;
        to[c] = (T)(p > 0.5f ? fmaf(-p, fmaf(ge, of_entropy, sum - more), -more * expm1f(log_p)) : fmaf(-p, fmaf(ge, of_entropy, sum), more));
    }
}

// ---------------------------------------------------------------------------------------------------------------- host

int checked(const i6logp_problem* p) {
    if (!p || p->B <= 0 || p->T <= 0 || p->F <= 0 || p->k < 0 || p->k > p->F || p->k > I6LOGP_MOST_ALTERNATIVES || !valid_dtype(p->dtype) || !p->logits || !p->targets || !p->seq_lens)
        return I6TRAIN_ERR_INVALID_ARGUMENT;
    const int64_t frames = (int64_t)p->B * p->T;
    if (p->F > (1 << 28) || !launchable(frames, p->F <= 512 ? 64 : 1024)) return I6TRAIN_ERR_TOO_LARGE;      // short rows have a wave each
    return I6TRAIN_OK;
}

Args args_of(const i6logp_problem& p) {
    Args a{};
    a.logits = p.logits; a.l_b = p.logits_stride_b; a.l_t = p.logits_stride_t;
    a.targets = p.targets; a.t_b = p.targets_stride_b; a.t_t = p.targets_stride_t;
    a.lens = p.seq_lens;
    a.B = p.B; a.T = p.T; a.F = p.F; a.k = p.k;
    return a;
}

// Rows for several waves on each of the card's 1024 SIMDs.
bool many(const Args& a) { return (int64_t)a.B * a.T >= kMany; }

template <typename T, int kThreads, int kHeld> void forward_with(const Args& a, hipStream_t s) {
    constexpr int kTeams = kThreads == 64 ? 4 : 1;
    const int64_t frames = (int64_t)a.B * a.T;
    logp_forward<T, kThreads, kHeld><<<dim3((unsigned)ceil_div(frames, (int64_t)kTeams)), dim3(kThreads < 256 ? 256 : kThreads), 0, s>>>(a);
}

// The fewest threads that hold a row in 48 registers each; with many rows, the fewest that do so in 80, as what a row needs besides its scores is done by every wave
// (16 384 rows of 5001 in 16 bits: 94 us by workgroups, 77 by waves; 1024 rows 12.6 either way).
template <typename T> int forward(const Args& a, hipStream_t s) {
    constexpr int64_t kPer = kPiece<T>, kMost = 48 / sizeof(float) * 4 / kPer;      // pieces of a thread
    const int64_t pieces = ceil_div((int64_t)a.F, kPer);
    if (pieces <= 64 * 2) forward_with<T, 64, 2>(a, s);
    else if (pieces <= 64 * 6) forward_with<T, 64, 6>(a, s);
    else if (pieces <= 64 * 12 && many(a)) forward_with<T, 64, 12>(a, s);
    else if (pieces <= 64 * 20 && many(a)) forward_with<T, 64, 20>(a, s);
    else if (pieces <= 256 * 3) forward_with<T, 256, 3>(a, s);
    else if (pieces <= 256 * 6) forward_with<T, 256, 6>(a, s);
    else if (pieces <= 256 * kMost) forward_with<T, 256, kMost>(a, s);
    else if (pieces <= 512 * kMost) forward_with<T, 512, kMost>(a, s);
    else forward_with<T, 1024, 0>(a, s);
    return launched();
}

template <typename T> int backward(const Args& a, hipStream_t s) {
    const int64_t frames = (int64_t)a.B * a.T;
    // many rows of up to 10 KB have a wave each: 16 384 of 5001 in 16 bits 72 us by workgroups, 68 by waves, of 1000 27 and 15, but of 5001 in 32 bits 124 and 175, and 1024 of 1000 4.7 and 5.9
    if (many(a) && a.F * sizeof(T) <= 10240) logp_backward<T, 64><<<dim3((unsigned)ceil_div(frames, (int64_t)4)), dim3(256), 0, s>>>(a);
    else logp_backward<T, 256><<<dim3((unsigned)frames), dim3(256), 0, s>>>(a);
    return launched();
}

}  // namespace
}  // namespace i6train

using namespace i6train;

extern "C" {

int i6logp_forward(const i6logp_problem* p, float* log_prob, float* entropy, float* top, int32_t* top_class, float* statistics, void* stream) {
    I6TRAIN_TRY(checked(p));
    if (!log_prob || !entropy || (p->k > 0 && (!top || !top_class))) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Args a = args_of(*p);
    a.log_prob = log_prob; a.entropy = entropy; a.top = top; a.top_class = top_class; a.statistics = statistics;
    a.report = status_slot();
    return p->dtype == I6TRAIN_F32 ? forward<float>(a, (hipStream_t)stream) : forward<bf16>(a, (hipStream_t)stream);
}

int i6logp_backward(const i6logp_problem* p, const float* statistics, const int32_t* top_class, const float* grad_log_prob, const float* grad_entropy, const float* grad_top,
                    void* grad_logits, void* stream) {
    I6TRAIN_TRY(checked(p));
    if (!statistics || !grad_logits || (p->k > 0 && !top_class)) return I6TRAIN_ERR_INVALID_ARGUMENT;
    Args a = args_of(*p);
    a.statistics = const_cast<float*>(statistics); a.top_class = const_cast<int32_t*>(top_class);
    a.g_log_prob = grad_log_prob; a.g_entropy = grad_entropy; a.g_top = grad_top; a.grad = grad_logits;
    return p->dtype == I6TRAIN_F32 ? backward<float>(a, (hipStream_t)stream) : backward<bf16>(a, (hipStream_t)stream);
}

}  // extern "C"
