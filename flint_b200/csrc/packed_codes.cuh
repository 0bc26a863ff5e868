// Pages of 8 bits: codes as FP16, and the weight of blocks of zeros.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace fb {

// What stands for V's scale where that is 0, and all codes are. Any number would do for its keys' part of the sum (it is divided
// out again); one far below every scale that storing leaves (2^-31 or more) keeps its probabilities from pushing those of
// blocks that have values below what FP16 holds. (With 1, values of 10^-3 beside zeros gave results 5 to 9 times their rounding off.)
constexpr float kWeightOfZeros = 0x1p-40f;

// Bytes kLow and kLow + 1 of x, which are codes + 128, as FP16: 1,024 + byte has the byte as its low bits.
template <int kLow>
__device__ __forceinline__ unsigned two_codes(unsigned x) {
    const unsigned biased = __byte_perm(x, 0x64646464u, kLow == 0 ? 0x4140 : 0x4342);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const unsigned*>(&h);
}

}  // namespace fb
