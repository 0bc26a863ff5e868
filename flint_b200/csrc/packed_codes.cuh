// 8-bit codes as FP16.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace fb {

// Bytes kLow and kLow + 1 of x, which are codes + 128, as FP16: 1,024 + byte has the byte as its low bits.
template <int kLow>
__device__ __forceinline__ unsigned two_codes(unsigned x) {
    const unsigned biased = __byte_perm(x, 0x64646464u, kLow == 0 ? 0x4140 : 0x4342);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const unsigned*>(&h);
}

}  // namespace fb
