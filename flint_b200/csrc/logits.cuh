// Pieces that the kernels over rows of logits share: maxima of 16-byte words, and numbers that order logits by value and place.
#pragma once

#include <cstdint>
#include <type_traits>

#include <cuda_fp16.h>

#include "device_utils.cuh"

namespace {

using Key = unsigned long long;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The running maximum of words, whose NaN stays, and a word's, in which a NaN is passed over.
struct MaxF {
    float m = -INFINITY;
    __device__ __forceinline__ void add(const uint4& q) {
        m = max_nan(m, max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)),
                               max_nan(__uint_as_float(q.z), __uint_as_float(q.w))));
    }
    __device__ __forceinline__ void add(const MaxF& other) { m = max_nan(m, other.m); }
    __device__ __forceinline__ float value() const { return m; }
    __device__ static __forceinline__ float word(const uint4& q) {
        return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
};
struct MaxH {
    __half2 m = __half2half2(__ushort_as_half(0xfc00));
    __device__ __forceinline__ void add(const uint4& q) {
        const __half2* h = reinterpret_cast<const __half2*>(&q);
        m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    }
    __device__ __forceinline__ void add(const MaxH& other) { m = __hmax2_nan(m, other.m); }
    __device__ __forceinline__ float value() const { return max_nan(__low2float(m), __high2float(m)); }
    __device__ static __forceinline__ float word(const uint4& q) {
        const __half2* h = reinterpret_cast<const __half2*>(&q);
        const __half2 w = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return __half2float(__hmax(__low2half(w), __high2half(w)));
    }
};
template <typename T>
using Max = typename std::conditional<sizeof(T) == 2, MaxH, MaxF>::type;

// A word's values from the `count`-th on become minus infinity, which counts for nothing.
__device__ __forceinline__ void cut_word(uint4& q, int count, float) {
    unsigned* w = reinterpret_cast<unsigned*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = i < count ? w[i] : 0xff800000u;
    }
}
__device__ __forceinline__ void cut_word(uint4& q, int count, __half) {
    unsigned* w = reinterpret_cast<unsigned*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = 2 * i >= count ? 0xfc00fc00u : 2 * i + 1 >= count ? (w[i] & 0xffffu) | 0xfc000000u : w[i];
    }
}

// A number that orders logits by value (both zeros alike, NaN above all) and equal ones by place,
// the lowest first. No two columns have the same; none has 0.
__device__ __forceinline__ Key order_key(float v, int column) {
    const unsigned bits = __float_as_uint(__fadd_rn(v, 0.0f));
    const unsigned ordered = v != v ? 0xffffffffu : (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
    return (static_cast<Key>(ordered) << 32) | (0xffffffffu - static_cast<unsigned>(column));
}
__device__ __forceinline__ int key_column(Key key) {
    return static_cast<int>(0xffffffffu - static_cast<unsigned>(key));
}
__device__ __forceinline__ float key_value(Key key) {
    const unsigned ordered = static_cast<unsigned>(key >> 32);
    return __uint_as_float((ordered & 0x80000000u) != 0 ? ordered ^ 0x80000000u : ~ordered);
}

}  // namespace
