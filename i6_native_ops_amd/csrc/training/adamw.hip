// AdamW over many tensors in one launch, states in 32 bits or in 8 (include/i6train.h).
//
// Bound by memory: a value in 32 bits moves 28 bytes (parameter and two states both ways, gradient one way), with
// states in 8 bits 16.06.  The table of tensors travels in the kernel's arguments, so a step is one launch for up to kMaxTensors
// tensors, copies nothing to the device and can be captured into a graph.  A workgroup takes kChunk consecutive values of one
// tensor; which tensor, it finds by bisection over the first workgroup of each.  38 tensors of 37 M values in 32 bits: 187 us (1.05 GB, 5.6 TB/s); 74 tensors of
// 226 M values with states in 8 bits: 650 us (3.63 GB, 5.6 TB/s).
#include <cmath>

#include "train_common.h"

// Sums and products are rounded one by one, as the definition states them: what is stored in 8 bits depends on
// comparisons, and a contracted multiply-add would make them depend on the compiler.
#pragma clang fp contract(off)

namespace i6train {
namespace {

constexpr int kMaxTensors = 56;          // x 64 bytes: the arguments of a kernel may have 4 KB
constexpr int kChunk = 4096;
constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.f, kPerMax = 1.f / 448.f;
constexpr float kLeastScale = 0x1p-100f;
constexpr uint32_t kPhi = 2654435769u, kRoot = 1779033703u;

struct Table {
    i6train_adamw_tensor t[kMaxTensors];
    int first[kMaxTensors];              // first workgroup of each tensor
    int n;
};
static_assert(sizeof(Table) <= 3800, "kernel arguments");

struct Factors {
    float beta1, rest1, beta2, rest2, keep, rate, root_correction, eps;
    uint32_t turn_m, turn_v;             // step ROOT and step PHI
};

__device__ __forceinline__ int find(const Table& tab, int wg) {
    int lo = 0, hi = tab.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= wg) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename T> using vec4 = T __attribute__((ext_vector_type(4)));
using f32x4 = vec4<float>;

// How tensors are accessed.  kAligned: their addresses allow one access for four values.  kStream: past the caches.  A step that moves more than kStreamBytes finds
// nothing of the last one in the 256 MB in front of the memory, and is faster when it leaves nothing there either (float, states in 32 bits: 40 M values
// 199 us, 215 us without; states in 8 bits, 64 M values 190 and 203 us); a smaller one finds part of its tensors (16 M values: 68 us, 83 us past the caches; 8 bits, 32 M values: 92 and
// 99 us).  The two meet at 22 M and 38 M values, 610 MB in both formats.
constexpr int64_t kStreamBytes = 610000000;
template <bool kAligned_, bool kStream_> struct Access { static constexpr bool kAligned = kAligned_, kStream = kStream_; };

template <typename A, typename V> __device__ __forceinline__ V get(const V* p) { return A::kStream ? __builtin_nontemporal_load(p) : *p; }
template <typename A, typename V> __device__ __forceinline__ void put(V* p, V v) {
    if (A::kStream) __builtin_nontemporal_store(v, p); else *p = v;
}

// Four consecutive values; `left` of them are there.
template <typename A, typename T> __device__ __forceinline__ f32x4 load4(const T* p, int64_t left) {
    if (A::kAligned && left >= 4) {
        const vec4<T> v = get<A>(reinterpret_cast<const vec4<T>*>(p));
        return f32x4{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
    }
    f32x4 v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) v[i] = (float)p[i];
    return v;
}

template <typename A, typename T> __device__ __forceinline__ void store4(T* p, f32x4 v, int64_t left) {
    if (A::kAligned && left >= 4) {
        put<A>(reinterpret_cast<vec4<T>*>(p), vec4<T>{(T)v.x, (T)v.y, (T)v.z, (T)v.w});
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) p[i] = (T)v[i];
}

// m, v and p of one value.
__device__ __forceinline__ void update(const Factors& k, float g, float& p, float& m, float& v, float& root) {
    m = m * k.beta1 + g * k.rest1;
    v = v * k.beta2 + g * g * k.rest2;
    root = sqrtf(v);
    const float size = root * k.root_correction + k.eps;
    p = p * k.keep - m / size * k.rate;
}

template <typename T, typename A>
__device__ __forceinline__ void chunk32(const i6train_adamw_tensor& t, const Factors& k, int64_t base) {
    T* p = static_cast<T*>(t.param);
    const T* g = static_cast<const T*>(t.grad);
    float* m = static_cast<float*>(t.exp_avg);
    float* v = static_cast<float*>(t.exp_avg_sq);
#pragma unroll
    for (int r = 0; r < kChunk / (4 * kThreads); r++) {
        const int64_t at = base + (r * kThreads + threadIdx.x) * 4, left = t.n - at;
        if (left <= 0) continue;
        f32x4 pv = load4<A>(p + at, left), mv = load4<A>(m + at, left), vv = load4<A>(v + at, left);
        const f32x4 gv = load4<A>(g + at, left);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float pi = pv[i], mi = mv[i], vi = vv[i], root;
            update(k, gv[i], pi, mi, vi, root);
            pv[i] = pi; mv[i] = mi; vv[i] = vi;
        }
        store4<A>(p + at, pv, left);
        store4<A>(m + at, mv, left);
        store4<A>(v + at, vv, left);
    }
}

__device__ __forceinline__ float scale_of(uint32_t bits) {
    const float s = __uint_as_float(bits) * kPerMax;
    return s < kLeastScale ? kLeastScale : s;
}

// The scales of a wave's block from its largest magnitudes as bit patterns.  Infinities and NaN are on top of these; they say nothing about
// the others of their block, so where there are any, the largest of those that are numbers is looked for.
constexpr uint32_t kInfinity = 0x7f800000u;
__device__ __forceinline__ float scale_of_block(uint32_t most, f32x4 v) {
    most = wave_max(most);
    if (most >= kInfinity) {
        most = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t b = __float_as_uint(fabsf(v[i]));
            most = b < kInfinity && b > most ? b : most;
        }
        most = wave_max(most);
    }
    return scale_of(most);
}

// Distance of the 8-bit values around y >= 0: 2^(e - 3), e the exponent, -6 at least.
__device__ __forceinline__ float quantum(float y) {
    uint32_t e = (__float_as_uint(y) >> 23) & 255u;
    e = e < 121u ? 121u : e;
    return __uint_as_float((e - 3u) << 23);
}
// 1 / quantum(y), a power of two as well
__device__ __forceinline__ float per_quantum(float y) {
    uint32_t e = (__float_as_uint(y) >> 23) & 255u;
    e = e < 121u ? 121u : e;
    return __uint_as_float((257u - e) << 23);
}

// m / scale rounded up with the probability that keeps its mean: floor(|y| / q + u) q.
__device__ __forceinline__ float round_m(float y, float u) {
    const float a = fabsf(y), q = quantum(a);
    float k = floorf(a * per_quantum(a) + u) * q;
    k = k > kE4m3Max ? kE4m3Max : k;
    return copysignf(fmaf(a, 0.f, k), y);      // NaN for infinities, which the format does not have
}

// The root so that its square keeps its mean: up where y^2 - low^2 > u (high^2 - low^2).  The square would otherwise grow by the variance of
// the rounding, up to 0.4 %, at every step, more than a step with beta2 = 0.999 forgets.  A root under the smallest value is rounded up:
// what divides by it stays bounded.
__device__ __forceinline__ float round_root(float y, float u) {
    const float q = quantum(y);
    const float low = floorf(y * per_quantum(y)) * q;
    const bool up = (y * y - low * low > u * (q * (low + low + q))) || (low == 0.f && y > 0.f);
    float k = up ? low + q : low;
    k = k > kE4m3Max ? kE4m3Max : k;
    return fmaf(y, 0.f, k);
}

__device__ __forceinline__ f32x4 from_fp8(uint32_t w) {
    return f32x4{__builtin_amdgcn_cvt_f32_fp8((int)w, 0), __builtin_amdgcn_cvt_f32_fp8((int)w, 1), __builtin_amdgcn_cvt_f32_fp8((int)w, 2),
                 __builtin_amdgcn_cvt_f32_fp8((int)w, 3)};
}
__device__ __forceinline__ uint32_t to_fp8(f32x4 v) {        // values of the format: nothing is rounded here
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v.x, v.y, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v.z, v.w, w, true);
}

template <typename A> __device__ __forceinline__ uint32_t load_bytes(const uint8_t* p, int64_t left) {
    if (A::kAligned && left >= 4) return get<A>(reinterpret_cast<const uint32_t*>(p));
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) w |= (uint32_t)p[i] << (8 * i);
    return w;
}
template <typename A> __device__ __forceinline__ void store_bytes(uint8_t* p, uint32_t w, int64_t left) {
    if (A::kAligned && left >= 4) {
        put<A>(reinterpret_cast<uint32_t*>(p), w);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) p[i] = (uint8_t)(w >> (8 * i));
}

// A wave has a block of 256 values, four in each lane: the scale of a block is a reduction within the wave.
template <typename T, typename A>
__device__ __forceinline__ void chunk8(const i6train_adamw_tensor& t, const Factors& k, int64_t base) {
    T* p = static_cast<T*>(t.param);
    const T* g = static_cast<const T*>(t.grad);
    uint8_t* m8 = static_cast<uint8_t*>(t.exp_avg);
    uint8_t* v8 = static_cast<uint8_t*>(t.exp_avg_sq);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    f32x4 um, uv;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t j = lane * 4 + i;
        um[i] = (float)((j * kPhi + k.turn_m) >> 16) * 0x1p-16f;
        uv[i] = (float)((j * kRoot + k.turn_v) >> 16) * 0x1p-16f;
    }
#pragma unroll
    for (int r = 0; r < kChunk / (4 * kThreads); r++) {
        const int64_t block = base / I6TRAIN_BLOCK + r * (kThreads / kWave) + wave;
        if (block * I6TRAIN_BLOCK >= t.n) continue;          // the same for the whole wave
        const int64_t at = block * I6TRAIN_BLOCK + lane * 4, left = t.n - at;
        f32x4 pv = load4<A>(p + at, left), gv = load4<A>(g + at, left);
        f32x4 mv = from_fp8(load_bytes<A>(m8 + at, left)) * t.exp_avg_scale[block];
        f32x4 vv = from_fp8(load_bytes<A>(v8 + at, left)) * t.exp_avg_sq_scale[block];
        f32x4 rv;
        uint32_t most_m = 0, most_r = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float pi = pv[i], mi = mv[i], vi = vv[i] * vv[i], root;
            update(k, gv[i], pi, mi, vi, root);
            pv[i] = pi; mv[i] = mi; rv[i] = root;
            const uint32_t bm = __float_as_uint(fabsf(mi)), br = __float_as_uint(fabsf(root));
            most_m = bm > most_m ? bm : most_m;
            most_r = br > most_r ? br : most_r;
        }
        const float sm = scale_of_block(most_m, mv), sr = scale_of_block(most_r, rv);
        const float per_m = 1.f / sm, per_r = 1.f / sr;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mv[i] = round_m(mv[i] * per_m, um[i]);
            rv[i] = round_root(rv[i] * per_r, uv[i]);
        }
        store4<A>(p + at, pv, left);
        store_bytes<A>(m8 + at, to_fp8(mv), left);
        store_bytes<A>(v8 + at, to_fp8(rv), left);
        if (lane == 0) {
            t.exp_avg_scale[block] = sm;
            t.exp_avg_sq_scale[block] = sr;
        }
    }
}

template <typename T, int BITS, bool kStream>
__global__ __launch_bounds__(kThreads) void adamw_step(Table tab, Factors k) {
    const int i = find(tab, blockIdx.x);
    const i6train_adamw_tensor& t = tab.t[i];
    const int64_t base = (int64_t)(blockIdx.x - tab.first[i]) * kChunk;
    // one access for four values needs their size as alignment; views into a larger buffer may not have it
    const uintptr_t whole = (uintptr_t)t.param | (uintptr_t)t.grad, state = (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq;
    const bool aligned = whole % (4 * sizeof(T)) == 0 && state % (BITS == 8 ? 4 : 16) == 0;
    if (BITS == 8) {
        if (aligned) chunk8<T, Access<true, kStream>>(t, k, base); else chunk8<T, Access<false, kStream>>(t, k, base);
    } else {
        if (aligned) chunk32<T, Access<true, kStream>>(t, k, base); else chunk32<T, Access<false, kStream>>(t, k, base);
    }
}

template <typename T, bool kStream> void launch(const Table& tab, const Factors& k, int bits, int wgs, hipStream_t s) {
    if (bits == 8) adamw_step<T, 8, kStream><<<dim3(wgs), dim3(kThreads), 0, s>>>(tab, k);
    else adamw_step<T, 32, kStream><<<dim3(wgs), dim3(kThreads), 0, s>>>(tab, k);
}

}  // namespace
}  // namespace i6train

extern "C" int i6train_adamw(const i6train_adamw_tensor* tensors, int n_tensors, int dtype, int state_bits, int64_t step, double lr,
                             double beta1, double beta2, double eps, double weight_decay, void* stream) {
    using namespace i6train;
    if (n_tensors < 0 || (n_tensors > 0 && !tensors) || !valid_dtype(dtype) || (state_bits != 8 && state_bits != 32) || step < 1 ||
        !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !std::isfinite(lr) || !std::isfinite(weight_decay))
        return I6TRAIN_ERR_INVALID_ARGUMENT;
    int64_t values = 0;
    for (int i = 0; i < n_tensors; i++) {
        const i6train_adamw_tensor& t = tensors[i];
        if (t.n < 0) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return I6TRAIN_ERR_INVALID_ARGUMENT;
        if (!launchable(ceil_div(t.n, (int64_t)kChunk), kThreads)) return I6TRAIN_ERR_TOO_LARGE;
        values += t.n;
    }
    const bool stream_past = values * (3 * (int64_t)elem_size(dtype) + (state_bits == 8 ? 4 : 16)) > kStreamBytes;
    Factors k;
    k.beta1 = (float)beta1; k.rest1 = (float)(1.0 - beta1);
    k.beta2 = (float)beta2; k.rest2 = (float)(1.0 - beta2);
    k.keep = (float)(1.0 - lr * weight_decay);
    k.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    k.root_correction = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    k.eps = (float)eps;
    k.turn_m = (uint32_t)step * kRoot;
    k.turn_v = (uint32_t)step * kPhi;
    Table tab;
    tab.n = 0;
    int64_t wgs = 0;
    const auto flush = [&]() {
        if (tab.n == 0) return I6TRAIN_OK;
        const auto run = dtype == I6TRAIN_BF16 ? (stream_past ? launch<bf16, true> : launch<bf16, false>) : (stream_past ? launch<float, true> : launch<float, false>);
        run(tab, k, state_bits, (int)wgs, (hipStream_t)stream);
        tab.n = 0;
        wgs = 0;
        return launched();
    };
    for (int i = 0; i < n_tensors; i++) {
        if (tensors[i].n == 0) continue;
        const int64_t need = ceil_div(tensors[i].n, (int64_t)kChunk);
        if (tab.n == kMaxTensors || !launchable(wgs + need, kThreads)) I6TRAIN_TRY(flush());
        tab.t[tab.n] = tensors[i];
        tab.first[tab.n] = (int)wgs;
        tab.n++;
        wgs += need;
    }
    return flush();
}
