// Device pieces of the attention kernels for sequences of different lengths: a sequence's place, its
// pages, and the error word.
#pragma once

#include "packed.h"
#include "packed_schedule.h"

namespace fb {

// Each file of kernels has its own error word.
static __device__ int g_packed_error = 0;

__device__ __forceinline__ void report() { atomicExch(&g_packed_error, 1); }

static inline cudaError_t read_error_word(int* value, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(value, g_packed_error, sizeof(int));
    if (e == cudaSuccess && reset && *value != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_packed_error, &zero, sizeof(int));
    }
    return e;
}

// Values outside their ranges are clamped and reported.
__device__ __forceinline__ Sequence sequence_at(const PackedArgs& p, int s) {
    const int a = p.starts[s], b = p.starts[s + 1];
    Sequence out;
    out.first = min(max(a, 0), p.rows);
    out.count = min(max(b, out.first), p.rows) - out.first;
    bool good = out.first == a && out.first + out.count == b;
    out.keys = out.count;
    if (p.lengths != nullptr) {
        const int given = p.lengths[s];
        const long long most = static_cast<long long>(p.table_stride) * p.page_size;
        out.keys = static_cast<int>(min(static_cast<long long>(max(given, 0)), most));
        good = good && out.keys == given;
    }
    if (!good) {
        report();
    }
    return out;
}

// The page that holds a key of sequence s, or -1 (reported) where the table names none.
__device__ __forceinline__ long long page_of(const PackedArgs& p, int s, int key) {
    const int page = p.table[static_cast<long long>(s) * p.table_stride + key / p.page_size];
    if (page < 0 || page >= p.pages) {
        report();
        return -1;
    }
    return page;
}

}  // namespace fb
