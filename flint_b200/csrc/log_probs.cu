// Log-probabilities of given tokens with the entropy and the most likely alternatives, and the
// gradient of the first two (extensions: the reference's loss, src/kernels/cross_entropy.cu:106-172,
// gives neither).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include <cuda_fp16.h>

#include "common.h"
#include "device_utils.cuh"
#include "flint/flint_b200.h"

namespace {

constexpr int kThreads = 512;
constexpr int kMostTop = 32;
constexpr float kLowest = -200.0f;   // e^-200 is 0 in FP32, and 0 * -200 a number

struct LogProbArgs {
    float* log_probs;
    float* entropy;
    float* lse;
    float* top_log_probs;
    uint16_t* top_tokens;
    const void* logits;
    const uint16_t* targets;
    size_t rows;
    int vocab, cols, top;
};

__device__ __forceinline__ float value_at(const float* row, int c) { return row[c]; }
__device__ __forceinline__ float value_at(const __half* row, int c) { return __half2float(row[c]); }

// A number that orders logits by value (both zeros alike, NaN above all) and equal ones by place,
// the lowest first. No two columns have the same.
__device__ __forceinline__ unsigned long long order_key(float v, int column) {
    const unsigned bits = __float_as_uint(__fadd_rn(v, 0.0f));
    const unsigned ordered = v != v ? 0xffffffffu : (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
    return (static_cast<unsigned long long>(ordered) << 32) | (0xffffffffu - static_cast<unsigned>(column));
}

__device__ __forceinline__ float combine(float a, float b) { return a + b; }
__device__ __forceinline__ unsigned long long combine(unsigned long long a, unsigned long long b) {
    return a > b ? a : b;
}

// The block's sum (float) or maximum (keys), for every thread.
template <typename Value>
__device__ Value block_reduce(Value v, Value* scratch) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        v = combine(v, __shfl_xor_sync(fb::kFullMask, v, off));
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) {
        scratch[threadIdx.x / 32] = v;
    }
    __syncthreads();
    v = scratch[threadIdx.x % (kThreads / 32)];
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
        v = combine(v, __shfl_xor_sync(fb::kFullMask, v, off));
    }
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) fb_token_log_probs_rows(const LogProbArgs p) {
    __shared__ float sums[kThreads / 32];
    __shared__ unsigned long long keys[kThreads / 32];
    fb::dependency_wait();
    fb::dependency_release();
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.logits) + row * p.cols;
        unsigned long long best = 0;
        for (int c = threadIdx.x; c < p.vocab; c += kThreads) {
            best = combine(best, order_key(value_at(x, c), c));
        }
        best = block_reduce(best, keys);
        const float top = value_at(x, static_cast<int>(0xffffffffu - static_cast<unsigned>(best)));
        float total = 0.0f, weighted = 0.0f;
        for (int c = threadIdx.x; c < p.vocab && top != -INFINITY; c += kThreads) {
            const float d = value_at(x, c) - top;
            const float e = expf(d);
            total += e;
            weighted += e * (d < kLowest ? kLowest : d);
        }
        total = block_reduce(total, sums);
        weighted = block_reduce(weighted, sums);
        const float log_total = logf(total);
        const bool none = top == -INFINITY;
        auto log_prob = [&](float v) { return none ? -INFINITY : (v - top) - log_total; };
        if (threadIdx.x == 0) {
            if (p.log_probs != nullptr) {
                const int target = p.targets[row];
                p.log_probs[row] = target < p.vocab ? log_prob(value_at(x, target)) : 0.0f;
            }
            if (p.entropy != nullptr) {
                p.entropy[row] = none ? 0.0f : log_total - weighted / total;
            }
            if (p.lse != nullptr) {
                p.lse[row] = none ? -INFINITY : top + log_total;
            }
        }
        for (int k = 0; k < p.top; ++k) {
            const int column = static_cast<int>(0xffffffffu - static_cast<unsigned>(best));
            if (threadIdx.x == 0) {
                p.top_tokens[row * p.top + k] = static_cast<uint16_t>(column);
                p.top_log_probs[row * p.top + k] = log_prob(value_at(x, column));
            }
            if (k + 1 < p.top) {
                unsigned long long next = 0;
                for (int c = threadIdx.x; c < p.vocab; c += kThreads) {
                    const unsigned long long key = order_key(value_at(x, c), c);
                    next = key < best ? combine(next, key) : next;
                }
                best = block_reduce(next, keys);
            }
        }
    }
}

struct LogProbGradientArgs {
    void* dlogits;
    const void* logits;
    const uint16_t* targets;
    const float* lse;
    const float* entropy;
    const float* d_log_probs;
    const float* d_entropy;
    size_t rows;
    int vocab, cols;
};

__device__ __forceinline__ void store_value(float* row, int c, float v) { row[c] = v; }
__device__ __forceinline__ void store_value(__half* row, int c, float v) { row[c] = __float2half_rn(v); }

template <typename T>
__global__ void __launch_bounds__(kThreads) fb_token_log_probs_backward_rows(const LogProbGradientArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.logits) + row * p.cols;
        T* out = static_cast<T*>(p.dlogits) + row * p.cols;
        const int target = p.targets != nullptr ? p.targets[row] : p.vocab;
        const float a = p.d_log_probs != nullptr && target < p.vocab ? p.d_log_probs[row] : 0.0f;
        const float b = p.d_entropy != nullptr ? p.d_entropy[row] : 0.0f;
        const float lse = p.lse[row], entropy = p.d_entropy != nullptr ? p.entropy[row] : 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += kThreads) {
            float grad = 0.0f;
            if (c < p.vocab && lse != -INFINITY) {
                const float d = value_at(x, c) - lse;
                const float e = expf(d);
                grad = (c == target ? a : 0.0f) - e * (a + b * ((d < kLowest ? kLowest : d) + entropy));
            }
            store_value(out, c, grad);
        }
    }
}

constexpr flint_status kBad = FLINT_ERROR_INVALID_ARGUMENT;
constexpr size_t kMostRows = size_t{1} << 31;

flint_status check_logits(const char* name, size_t rows, size_t vocab, size_t cols) {
    constexpr size_t kMaxCols = size_t{1} << 16;
    if (cols == 0 || cols % 8 != 0 || cols > kMaxCols) {
        return fb::fail(kBad, "%s: cols (%zu) must be a multiple of 8 from 8 to %zu", name, cols, kMaxCols);
    }
    if (vocab == 0 || vocab > cols) {
        return fb::fail(kBad, "%s: vocab (%zu) must be from 1 to cols (%zu)", name, vocab, cols);
    }
    if (rows > kMostRows) {
        return fb::fail(kBad, "%s: rows (%zu) can be up to %zu", name, rows, kMostRows);
    }
    return FLINT_OK;
}

// An array that may be left out stands in the list of spans as `instead`, with no bytes, which
// overlaps nothing.
fb::Span span_or(const char* what, const void* pointer, size_t bytes, const void* instead) {
    return pointer != nullptr ? fb::Span{what, pointer, bytes} : fb::Span{what, instead, 0};
}

}  // namespace

extern "C" {

flint_status flint_b200_token_log_probs(void* log_probs, void* entropy, void* lse, void* top_log_probs,
                                        void* top_tokens, const void* logits, const void* targets, int fp32_logits,
                                        size_t rows, size_t vocab, size_t cols, size_t top, flint_stream stream) {
    constexpr const char* name = "flint_b200_token_log_probs";
    FB_TRY(check_logits(name, rows, vocab, cols));
    if (top > static_cast<size_t>(kMostTop) || top > vocab) {
        return fb::fail(kBad, "%s: top (%zu) can be up to %d and up to vocab (%zu)", name, top, kMostTop, vocab);
    }
    if (rows == 0) {
        return FLINT_OK;
    }
    if ((log_probs == nullptr) != (targets == nullptr)) {
        return fb::fail(kBad, "%s: log_probs and targets go together: %s is null", name,
                        log_probs == nullptr ? "log_probs" : "targets");
    }
    const void* none = logits;
    const fb::Span spans[] = {
        span_or("log_probs", log_probs, rows * 4, none),
        span_or("entropy", entropy, rows * 4, none),
        span_or("lse", lse, rows * 4, none),
        span_or("top_log_probs", top_log_probs, rows * top * 4, top != 0 ? nullptr : none),
        span_or("top_tokens", top_tokens, rows * top * 2, top != 0 ? nullptr : none),
        {"logits", logits, rows * cols * (fp32_logits != 0 ? 4 : 2)},
        span_or("targets", targets, rows * 2, none),
    };
    if (logits == nullptr) {
        return fb::fail(kBad, "%s: logits is null", name);
    }
    FB_TRY(fb::check_spans(name, spans, 5));
    LogProbArgs p = {};
    p.log_probs = static_cast<float*>(log_probs);
    p.entropy = static_cast<float*>(entropy);
    p.lse = static_cast<float*>(lse);
    p.top_log_probs = static_cast<float*>(top_log_probs);
    p.top_tokens = static_cast<uint16_t*>(top_tokens);
    p.logits = logits;
    p.targets = static_cast<const uint16_t*>(targets);
    p.rows = rows;
    p.vocab = static_cast<int>(vocab);
    p.cols = static_cast<int>(cols);
    p.top = static_cast<int>(top);
    int sms = 148;
    FB_CUDA(fb::sm_count(&sms));
    const unsigned blocks = static_cast<unsigned>(std::min<size_t>(rows, 4 * static_cast<size_t>(sms)));
    FB_CUDA(fb::launch_dependent(fp32_logits != 0 ? fb_token_log_probs_rows<float> : fb_token_log_probs_rows<__half>,
                                 dim3(blocks), dim3(kThreads), 0, stream, p));
    return FLINT_OK;
}

flint_status flint_b200_token_log_probs_backward(void* dlogits, const void* logits, const void* targets,
                                                 const void* lse, const void* entropy, const void* d_log_probs,
                                                 const void* d_entropy, int fp32_logits, size_t rows, size_t vocab,
                                                 size_t cols, flint_stream stream) {
    constexpr const char* name = "flint_b200_token_log_probs_backward";
    FB_TRY(check_logits(name, rows, vocab, cols));
    if (rows == 0) {
        return FLINT_OK;
    }
    if (d_log_probs == nullptr && d_entropy == nullptr) {
        return fb::fail(kBad, "%s: d_log_probs and d_entropy are both null", name);
    }
    if (d_log_probs != nullptr && targets == nullptr) {
        return fb::fail(kBad, "%s: targets is null", name);
    }
    if (d_entropy != nullptr && entropy == nullptr) {
        return fb::fail(kBad, "%s: entropy is null", name);
    }
    const size_t bytes = rows * cols * (fp32_logits != 0 ? 4 : 2);
    // The gradient may take the logits' place: a thread reads a logit before it writes there.
    const bool in_place = dlogits == logits;
    const fb::Span spans[] = {
        {"dlogits", dlogits, bytes},
        {"logits", logits, in_place && logits != nullptr ? 0 : bytes},
        {"lse", lse, rows * 4},
        span_or("targets", targets, rows * 2, lse),
        span_or("entropy", entropy, rows * 4, lse),
        span_or("d_log_probs", d_log_probs, rows * 4, lse),
        span_or("d_entropy", d_entropy, rows * 4, lse),
    };
    FB_TRY(fb::check_spans(name, spans, 1));
    LogProbGradientArgs p = {};
    p.dlogits = dlogits;
    p.logits = logits;
    p.targets = static_cast<const uint16_t*>(targets);
    p.lse = static_cast<const float*>(lse);
    p.entropy = static_cast<const float*>(entropy);
    p.d_log_probs = static_cast<const float*>(d_log_probs);
    p.d_entropy = static_cast<const float*>(d_entropy);
    p.rows = rows;
    p.vocab = static_cast<int>(vocab);
    p.cols = static_cast<int>(cols);
    int sms = 148;
    FB_CUDA(fb::sm_count(&sms));
    const unsigned blocks = static_cast<unsigned>(std::min<size_t>(rows, 4 * static_cast<size_t>(sms)));
    FB_CUDA(fb::launch_dependent(
        fp32_logits != 0 ? fb_token_log_probs_backward_rows<float> : fb_token_log_probs_backward_rows<__half>,
        dim3(blocks), dim3(kThreads), 0, stream, p));
    return FLINT_OK;
}

}  // extern "C"
