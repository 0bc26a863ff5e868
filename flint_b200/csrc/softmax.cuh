// Pieces that the attention kernels share: exponentials in base 2, the running maximum's
// constants and the descriptors of 64-column tiles.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "device_utils.cuh"
#include "sm100.cuh"

namespace fb {

// 2^x on the special-function unit (relative error about 2^-22, flushes denormals).
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The larger of two values; a NaN among them gives NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// How far (in base-2 exponent units) a tile's maximum may exceed the reference exponent
// before the forward kernel moves the reference and rescales its accumulator:
// probabilities then stay below 2^8, well inside FP16.
constexpr float kLazyShift = 8.0f;

// The reference exponent of a row for which no key has counted so far: the least finite value, so that
// keys of minus infinity (an infinity in K, or a mask) give probabilities of 2^-inf where -inf - -inf would be
// NaN, and the first key that counts moves it.
constexpr float kNoKey = -3.402823466e38f;

// 2^x for two values at once on the FMA pipe, for the share of the kernels'
// exponentials that the special-function unit has no time for: x = n + f with n the
// nearest integer (taken from the low mantissa bits of x + 1.5 * 2^23), 2^f by a
// degree-4 polynomial on [-0.5, 0.5] (relative error 2.7e-6, two orders below the FP16
// rounding of the probabilities), n added into the exponent field. x must be at most
// 127 - 1; anything below -120 counts as -120 (2^-120 is zero in FP16).
// kKeepNan: a NaN stays one, where else it counts as -120 too. 2 2^f is then multiplied by 2^(n - 1), whose exponent field,
// n + 126, is what the low bits of x + 1.5 * 2^23 + 126 hold: the same bits otherwise. (The forward kernels have no
// need of it, as the maximum of a row with a NaN is NaN and so are the row's other exponentials: 150 heads of 1,024 tokens take
// 43.5 us without, 44.1 with it. Backward, 24 heads: 26.05 and 26.1.)
template <bool kKeepNan>
__device__ __forceinline__ void exp2_pair_fma(F2 x, float& lo, float& hi) {
    auto both = [](float c) { return f2_pack(c, c); };
    auto coefficient = [&](float c) { return both(kKeepNan ? 2.0f * c : c); };
    float x0, x1;
    f2_unpack(x, x0, x1);
    const F2 clamped = kKeepNan ? f2_pack(max_nan(x0, -120.0f), max_nan(x1, -120.0f))
                                : f2_pack(fmaxf(x0, -120.0f), fmaxf(x1, -120.0f));
    const F2 magic = both(kKeepNan ? 12582912.0f + 126.0f : 12582912.0f);
    const F2 z = f2_add(clamped, magic);
    const F2 f = f2_sub(clamped, f2_sub(z, magic));
    F2 poly = f2_fma(f, coefficient(0.009570090100169182f), coefficient(0.05591785907745361f));
    poly = f2_fma(poly, f, coefficient(0.2402474582195282f));
    poly = f2_fma(poly, f, coefficient(0.6931217908859253f));
    poly = f2_fma(poly, f, coefficient(0.9999992847442627f));
    float z0, z1;
    f2_unpack(z, z0, z1);
    const int n0 = __float_as_int(z0) << 23, n1 = __float_as_int(z1) << 23;
    if constexpr (kKeepNan) {
        f2_unpack(f2_mul(poly, f2_pack(__int_as_float(n0), __int_as_float(n1))), lo, hi);
    } else {
        float p0, p1;
        f2_unpack(poly, p0, p1);
        lo = __int_as_float(__float_as_int(p0) + n0);
        hi = __int_as_float(__float_as_int(p1) + n1);
    }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Descriptors for the three ways a tile is read.
// K-major tile [128 rows][64 cols] (rows = M or N index): 16-column step = 32 bytes.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t tile, int kstep) {
    return sm100::smem_desc_sw128(tile + kstep * 32, 16, 1024);
}
// MN-major view of the same memory: rows are the K index, 16 rows = 2,048 bytes;
// 64-column blocks (panels) are `lbo` bytes apart.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t tile, int kstep, uint32_t lbo) {
    return sm100::smem_desc_sw128(tile + kstep * 2048, lbo, 1024);
}

}  // namespace fb
