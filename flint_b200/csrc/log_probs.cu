// Log-probabilities of given tokens with the entropy and the most likely alternatives, and the
// gradient of the first two (extensions: the reference's loss, src/kernels/cross_entropy.cu:106-172,
// gives neither).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.h"
#include "device_utils.cuh"
#include "flint/flint_b200.h"
#include "sm100.cuh"

namespace {

constexpr int kMostTop = 32;
constexpr int kCandidates = 512;
constexpr int kMostRanks = 8;        // CTAs of a cluster
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -200.0f;   // e^-200 is 0 in FP32, and 0 * -200 a number
// FP16: minus infinity may stand as the lowest finite value, -65,504, where the row's largest logit (or log-sum-exp) is so
// far above it that e^(the difference) is 0. Rows below this bound are low: their logits are raised first.
constexpr float kLowRow = -65000.0f;

using Key = unsigned long long;

__device__ int g_log_probs_error = 0;

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
    int slice;      // 16-byte words per CTA of a cluster
    int ranks;      // CTAs of a cluster
};

// Eight FP16 or four FP32 logits: a 16-byte word.
template <typename T>
struct Word {
    static constexpr int kValues = 16 / sizeof(T);
    __device__ static float value(const T* row, int c);
    __device__ static void unpack(float (&v)[kValues], const uint4& q);
    __device__ static uint4 pack(const float (&v)[kValues]);
    // As unpack, but that FP16's minus infinity becomes the lowest finite value (its exponential is 0, and 0 times
    // it a number); and for FP32, whose lowest value would not do, the same for differences.
    __device__ static void unpack_finite(float (&v)[kValues], const uint4& q);
    __device__ static fb::F2 clamp(fb::F2 d);
};
template <>
__device__ __forceinline__ float Word<float>::value(const float* row, int c) {
    return row[c];
}
template <>
__device__ __forceinline__ float Word<__half>::value(const __half* row, int c) {
    return __half2float(row[c]);
}
template <>
__device__ __forceinline__ void Word<float>::unpack(float (&v)[4], const uint4& q) {
    v[0] = __uint_as_float(q.x);
    v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z);
    v[3] = __uint_as_float(q.w);
}
template <>
__device__ __forceinline__ void Word<__half>::unpack(float (&v)[8], const uint4& q) {
    fb::unpack8(v, q);
}
template <>
__device__ __forceinline__ uint4 Word<float>::pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <>
__device__ __forceinline__ uint4 Word<__half>::pack(const float (&v)[8]) {
    return fb::pack8(v);
}

template <>
__device__ __forceinline__ void Word<float>::unpack_finite(float (&v)[4], const uint4& q) {
    unpack(v, q);
}
template <>
__device__ __forceinline__ void Word<__half>::unpack_finite(float (&v)[8], const uint4& q) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hmax2_nan(*reinterpret_cast<const __half2*>(&w[i]), __half2half2(__ushort_as_half(0xfbff)));
        const float2 x = __half22float2(h);
        v[2 * i] = x.x;
        v[2 * i + 1] = x.y;
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <>
__device__ __forceinline__ fb::F2 Word<float>::clamp(fb::F2 d) {
    float a, b;
    fb::f2_unpack(d, a, b);
    return fb::f2_pack(max_nan(a, kLowest), max_nan(b, kLowest));
}
template <>
__device__ __forceinline__ fb::F2 Word<__half>::clamp(fb::F2 d) {
    return d;
}

// The running maximum of words, whose NaN stays, and a word's, in which a NaN is passed over.
struct MaxF {
    float m = -INFINITY;
    __device__ __forceinline__ void add(const uint4& q) {
        m = max_nan(m, max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)),
                               max_nan(__uint_as_float(q.z), __uint_as_float(q.w))));
    }
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
    __device__ __forceinline__ float value() const { return max_nan(__low2float(m), __high2float(m)); }
    __device__ static __forceinline__ float word(const uint4& q) {
        const __half2* h = reinterpret_cast<const __half2*>(&q);
        const __half2 w = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return __half2float(__hmax(__low2half(w), __high2half(w)));
    }
};
template <typename T>
using Max = typename std::conditional<sizeof(T) == 2, MaxH, MaxF>::type;

// Sums of 2^y and of 2^y y with y = (x - m) log2 e, over the words given to add().
// (One value at a time from the exponential on: packed sums cost as many moves into register pairs as they save.)
struct SumsBase {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, weighted[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ void pair(int i, fb::F2 y) {
        float y0, y1, e0, e1;
        fb::f2_unpack(y, y0, y1);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(y0));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(y1));
        const int at = 2 * (i & 1);
        sum[at] += e0;
        sum[at + 1] += e1;
        weighted[at] = fmaf(e0, y0, weighted[at]);
        weighted[at + 1] = fmaf(e1, y1, weighted[at + 1]);
    }
    __device__ __forceinline__ void totals(float& total, float& mean) const {
        total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        mean = (weighted[0] + weighted[1]) + (weighted[2] + weighted[3]);
    }
};
// (The difference first: it is exact near m, so that a row of one possible token has an entropy of exactly 0. One
// instruction less, fma(x, log2 e, -m log2 e), is not.) 2^y y has to be a number for y of minus infinity.
struct SumsF : SumsBase {
    fb::F2 minus_m;
    __device__ __forceinline__ explicit SumsF(float m) : minus_m(fb::f2_pack(-m, -m)) {}
    __device__ __forceinline__ void add(const uint4& q) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float d0, d1;
            fb::f2_unpack(fb::f2_add(fb::f2_pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])), minus_m), d0, d1);
            pair(i, fb::f2_mul(fb::f2_pack(max_nan(d0, kLowest), max_nan(d1, kLowest)), fb::f2_pack(kLog2e, kLog2e)));
        }
    }
};
struct SumsH : SumsBase {
    float minus_m;
    __device__ __forceinline__ explicit SumsH(float m) : minus_m(-m) {}
    // x - m in FP32 from x in FP16, one instruction.
    __device__ __forceinline__ float difference(__half x) const {
        float d;
        asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d) : "h"(__half_as_ushort(x)), "f"(minus_m));
        return d;
    }
    __device__ __forceinline__ void add(const uint4& q) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (The lowest finite value does for minus infinity: low rows are raised.)
            const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&w[i]), __half2half2(__ushort_as_half(0xfbff)));
            pair(i, fb::f2_mul(fb::f2_pack(difference(__low2half(h)), difference(__high2half(h))), fb::f2_pack(kLog2e, kLog2e)));
        }
    }
};
template <typename T>
using Sums = typename std::conditional<sizeof(T) == 2, SumsH, SumsF>::type;

// Low rows of FP16 (their values are multiples of 32 from -65,504 on, or minus infinity) are taken 32,768 higher: that is
// exact, as it is for their FP32 log-sum-exps, and far above the lowest finite value.
constexpr float kRaise = 32768.0f;
__device__ __forceinline__ void raise_word(uint4&, float) {}
__device__ __forceinline__ void raise_word(uint4& q, __half) {
    unsigned* w = reinterpret_cast<unsigned*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hadd2(*reinterpret_cast<const __half2*>(&w[i]), __float2half2_rn(kRaise));
        w[i] = *reinterpret_cast<const unsigned*>(&h);
    }
}

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

// ---- forward ---------------------------------------------------------------------------------------
//
// With m the row's largest logit, d = x - m and S = sum e^d, D = sum d e^d:
//   lse = m + log S,  log p = d - log S,  entropy = log S - D / S   (all terms of one sign: nothing cancels)
// A thread holds its words of the row in registers: one pass finds the maxima, the second takes
// the exponentials while it asks for the next row's words, so that memory never waits. Long
// rows, and few of them, are divided over a cluster's CTAs: each takes sums against its own maximum, and the
// first puts them together.
// The alternatives: the slice falls into 64 (or 32) bins of neighbouring lanes. The k-th largest of the bins' maxima
// is a lower bound of the k-th largest logit; what is not below it (about k values) is collected in the
// second pass and put in order by counting. Where too many qualify (rows of equal logits, or fewer bins with words in them
// than there are alternatives), or a NaN is among them, the row is gone through once per alternative.
// Measured on rows of GPT-2's 50,257 words: 8,192 FP16 rows with five alternatives 206 us (4.0 TB/s), 4,096 without 88 us;
// 1,000 FP32 rows, a pair of CTAs each, 56 us; one FP32 row on eight CTAs with twenty alternatives 7.6 us with its
// launch. Bound by issue slots (40 instructions per eight logits for the sums) and what a row costs besides. (Rows held in
// registers, one CTA per SM: 355 us where shared memory takes 206.)
constexpr int blocks_per_sm(int threads, int held) { return (threads == 128 ? 4 : 1) * (held > 4 ? 1 : 2); }

constexpr int kChunks = 2;      // pieces in which a slice is copied into shared memory

// What a block keeps of two rows in turn, besides staged words.
template <int kWarps, int kBins>
struct RowMemory {
    union Lists {
        float bins[kBins];               // read before the first candidate of the row is written, and
        Key candidates[kCandidates];     // written when all are done with those of two rows before
    } lists[2];
    Key best[2][kMostRanks * kMostTop];
    Key reduced[kWarps];
    unsigned long long barriers[kChunks];
    float maxima[2][kWarps];
    float sums[2][2 * kWarps];
    float parts[2][kMostRanks][3];     // the first CTA's: every CTA's m, S, D
    float least[2];
    int counts[2];
    int abort_flag;
};

constexpr int kStagedThreads = 512;    // 256 are 6 % faster without alternatives, 5 % slower with five of them
constexpr int kStagedBins = 64;
// Words of a slice in shared memory: two CTAs per SM. An SM has 228 KB, of which a CTA costs 1 KB more than it asks for.
// (One CTA where 6,400 words did not fit twice: 8,192 rows of 51,200 FP16 logits with five alternatives 267 us, 197 with two.)
constexpr int kStagedWords = 6400;
static_assert(2 * (kStagedWords * 16 + (sizeof(RowMemory<kStagedThreads / 32, kStagedBins>) + 127) / 128 * 128 + 1024) <= 228 * 1024,
              "two CTAs fit on an SM");

// kHeld > 0: a thread holds that many words of the row in registers, and asks for the next row's while it takes
// the exponentials. kHeld == 0: the slice is copied into shared memory, and the CTA beside it on the SM computes
// meanwhile.
template <typename T, int kThreads, int kHeld>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(kThreads, kHeld)) fb_token_log_probs(const LogProbArgs p) {
    using W = Word<T>;
    constexpr bool kStaged = kHeld == 0;
    constexpr int kWarps = kThreads / 32;
    constexpr int kBins = kThreads >= 512 ? kStagedBins : 32;     // parts whose maxima bound the alternatives (up to 32) from below
    constexpr int kLanes = kThreads / kBins;      // of a bin
    extern __shared__ __align__(128) uint4 staged[];
    __shared__ RowMemory<kWarps, kBins> shared;
    auto& least = shared.least;
    auto& maxima = shared.maxima;
    auto& sums = shared.sums;
    auto& reduced = shared.reduced;
    auto& counts = shared.counts;
    auto& parts = shared.parts;
    auto& best = shared.best;
    auto& barriers = shared.barriers;
    int& abort_flag = shared.abort_flag;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    const int rank = p.ranks > 1 ? static_cast<int>(sm100::cluster_cta_rank()) : 0;
    const size_t stride = gridDim.x / p.ranks;
    const int row_words = p.cols / W::kValues;
    const int all_words = (p.vocab + W::kValues - 1) / W::kValues;
    const int first_word = rank * p.slice;
    const int words = max(0, min(p.slice, all_words - first_word));
    const int last_word = all_words - 1 - first_word;     // of the row, counted from the slice's first
    const int last_count = p.vocab - (all_words - 1) * W::kValues;
    const int full = last_word == words - 1 && last_count < W::kValues ? words - 1 : words;   // words that count whole
    const int top = p.top;
    // Threads of different warps have what one thread does per row: start copies, fetch the target and write results.
    constexpr int kCopier = kThreads / 2, kScribe = kThreads - 32;

    if (tid < 2) {
        counts[tid] = 0;
    }
    if (kStaged && tid == 0) {
        abort_flag = 0;
        for (int c = 0; c < kChunks; ++c) {
            sm100::mbar_init(sm100::smem_u32(&barriers[c]), 1);
        }
        sm100::mbar_fence_init();
    }
    fb::dependency_wait();
    if (p.ranks > 1) {
        sm100::cluster_sync_all();    // every CTA of the cluster runs before any writes to the first one's memory
    } else {
        __syncthreads();
    }
    if (tid == 0) {
        fb::dependency_release();
    }
    // (Plain loads, which the wait holds back: after_wait() pointers take registers, 214 -> 217 us for 8,192 rows of 51,200.)
    auto row_of = [&](size_t row) { return static_cast<const uint4*>(p.logits) + row * row_words + first_word; };
    size_t row = blockIdx.x / p.ranks;
    if (row >= p.rows) {
        return;     // (the whole cluster)
    }
    const int chunk = ((words + kChunks - 1) / kChunks + kThreads - 1) / kThreads * kThreads;
    auto copy_row = [&](size_t from) {     // one thread
        for (int c = 0; c < kChunks && c * chunk < words; ++c) {
            const uint32_t bytes = static_cast<uint32_t>(min(chunk, words - c * chunk)) * 16u;
            const uint32_t bar = sm100::smem_u32(&barriers[c]);
            sm100::mbar_expect_tx(bar, bytes);
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                ::"r"(sm100::smem_u32(staged + c * chunk)), "l"(row_of(from) + c * chunk), "r"(bytes), "r"(bar)
                : "memory");
        }
    };
    uint4 held[kStaged ? 1 : kHeld];
    if constexpr (kStaged) {
        if (tid == kCopier) {
            copy_row(row);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = tid + j * kThreads;
            if (i < words) {
                held[j] = row_of(row)[i];
            }
        }
    }
    // The scribe's: this row's target and its logit, fetched while the row before was worked on.
    auto target_of = [&](size_t from) { return p.targets != nullptr ? static_cast<int>(p.targets[from]) : 0; };
    auto target_value_of = [&](size_t from, int column) {
        return column < p.vocab ? W::value(static_cast<const T*>(p.logits) + from * p.cols, column) : 0.0f;
    };
    const bool scribe = tid == kScribe && rank == 0;
    int target = scribe ? target_of(row) : 0;
    float target_value = scribe ? target_value_of(row, target) : 0.0f;
    bool gave_up = false;
    uint32_t phase = 0;
    for (int parity = 0; row < p.rows; row += stride, parity ^= 1) {
        const T* values = static_cast<const T*>(p.logits) + row * p.cols;
        const size_t next = row + stride;
        const size_t soon = kStaged ? next : next + stride;
        if (tid == kCopier && soon < p.rows && words > 0) {
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row_of(soon)),
                         "r"(static_cast<uint32_t>(words) * 16u)
                         : "memory");
        }
        const int next_target = scribe && next < p.rows ? target_of(next) : 0;

        Max<T> running;
        bool there = true;
        if constexpr (kStaged) {
            for (int c = 0; c < kChunks && c * chunk < words; ++c) {
                there = sm100::mbar_wait(sm100::smem_u32(&barriers[c]), phase, &abort_flag) && there;
                const int end = min(full, (c + 1) * chunk);
#pragma unroll 4
                for (int i = c * chunk + tid; i < end; i += kThreads) {
                    running.add(staged[i]);
                }
            }
            phase ^= 1u;
            if (full < words && tid == full % kThreads) {
                // The last word, cut for good: this thread reads it again below.
                uint4 q = staged[full];
                cut_word(q, last_count, T());
                staged[full] = q;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // ahead of the next row's copy
                running.add(q);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int i = tid + j * kThreads;
                if (i < words) {
                    if (i >= full) {
                        cut_word(held[j], last_count, T());
                    }
                    running.add(held[j]);
                }
            }
        }
        float mx = running.value();
        const float my_max = mx;
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) {
            mx = max_nan(mx, __shfl_xor_sync(fb::kFullMask, mx, off));
        }
        if (tid % kLanes == 0) {
            shared.lists[parity].bins[tid / kLanes] = mx;
        }
#pragma unroll
        for (int off = kLanes; off < 32; off <<= 1) {
            mx = max_nan(mx, __shfl_xor_sync(fb::kFullMask, mx, off));
        }
        if (lane == 0) {
            maxima[parity][warp] = mx;
        }
        // One outcome for the whole CTA: who has seen its data must not wait for who has not. (A cluster's
        // CTAs go on in step, to the end: the others still write into the first one's memory.)
        if (kStaged ? __syncthreads_or(there ? 0 : 1) != 0 : (__syncthreads(), false)) {
            gave_up = true;
        }
        if (tid == 0) {
            counts[parity ^ 1] = 0;     // (of the row before, which everybody is done with)
        }
        mx = maxima[parity][lane % kWarps];
#pragma unroll
        for (int off = 1; off < kWarps; off <<= 1) {
            mx = max_nan(mx, __shfl_xor_sync(fb::kFullMask, mx, off));
        }
        // Whether a value can be among the `top` largest of the slice: the top-th largest of the bins' maxima, equal
        // ones counted each.
        float bound = INFINITY;
        if (top > 0) {
            // A warp ranks its share of the bins, each against all of them, one or two per lane.
            const float low = shared.lists[parity].bins[lane], high = kBins > 32 ? shared.lists[parity].bins[lane + kBins - 32] : 0.0f;
#pragma unroll 4
            for (int i = 0; i < kBins / kWarps; ++i) {
                const int bin = warp * (kBins / kWarps) + i;
                const float value = shared.lists[parity].bins[bin];
                int larger = __popc(__ballot_sync(fb::kFullMask, low > value || (low == value && lane < bin)));
                if (kBins > 32) {
                    larger += __popc(__ballot_sync(fb::kFullMask, high > value || (high == value && lane + 32 < bin)));
                }
                if (larger == top - 1 && lane == 0) {
                    least[parity] = value;      // (none is where bins are NaN)
                }
            }
            __syncthreads();
            bound = least[parity];
        }
        const bool none = mx == -INFINITY;
        auto collect = [&](const uint4& q, int i) {
            float v[W::kValues];
            W::unpack(v, q);
#pragma unroll
            for (int c = 0; c < W::kValues; ++c) {
                if (v[c] >= bound && v[c] > -INFINITY) {
                    const int at = atomicAdd(&counts[parity], 1);
                    if (at < kCandidates) {
                        shared.lists[parity].candidates[at] = order_key(v[c], (first_word + i) * W::kValues + c);
                    }
                }
            }
        };
        const bool collects = top > 0 && __any_sync(fb::kFullMask, my_max >= bound);
        const bool low = sizeof(T) == 2 && mx < kLowRow;
        Sums<T> sums_of(low ? mx + kRaise : mx);
        if constexpr (kStaged) {
            if (collects) {
#pragma unroll 4
                for (int i = tid; i < words; i += kThreads) {
                    const uint4 q = staged[i];
                    if (Max<T>::word(q) >= bound) {
                        collect(q, i);
                    }
                }
            }
            if (low) {
                for (int i = tid; i < words; i += kThreads) {     // (this thread's words, here and below)
                    uint4 q = staged[i];
                    raise_word(q, T());
                    staged[i] = q;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // ahead of the next row's copy
            }
#pragma unroll 4
            for (int i = tid; i < words; i += kThreads) {
                sums_of.add(staged[i]);
            }
        } else {
            if (collects) {
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    const int i = tid + j * kThreads;
                    if (i < words && Max<T>::word(held[j]) >= bound) {
                        collect(held[j], i);
                    }
                }
            }
            if (low) {
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    raise_word(held[j], T());
                }
            }
            const uint4* next_in = row_of(next < p.rows ? next : row);
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int i = tid + j * kThreads;
                if (i < words) {
                    sums_of.add(held[j]);
                    held[j] = next_in[i];
                }
            }
        }
        float total, mean;
        sums_of.totals(total, mean);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            total += __shfl_xor_sync(fb::kFullMask, total, off);
            mean += __shfl_xor_sync(fb::kFullMask, mean, off);
        }
        if (lane == 0) {
            sums[parity][2 * warp] = total;
            sums[parity][2 * warp + 1] = mean;
        }
        __syncthreads();
        if (kStaged && tid == kCopier && next < p.rows && !gave_up) {
            copy_row(next);     // everybody has read this row's words
        }
        const float next_value = scribe && next < p.rows ? target_value_of(next, next_target) : 0.0f;
        // Only the warps that write results go on: the scribe's, those with candidates, and all where the
        // alternatives take the long way. (A cluster's CTAs meet below.)
        const int found = top > 0 ? counts[parity] : 0;
        const bool collected = found <= kCandidates && mx == mx;
        const bool goes_on = warp == kScribe / 32 || (p.ranks > 1 && warp == 0) ||
                             (top > 0 && (!collected || warp * 32 < max(found, 1)));
        if (!goes_on && p.ranks == 1) {
            continue;
        }
        float log_total = 0.0f;
        if (goes_on) {
            total = sums[parity][2 * (lane % kWarps)];
            mean = sums[parity][2 * (lane % kWarps) + 1];
#pragma unroll
            for (int off = 1; off < kWarps; off <<= 1) {
                total += __shfl_xor_sync(fb::kFullMask, total, off);
                mean += __shfl_xor_sync(fb::kFullMask, mean, off);
            }
            mean *= kLn2;
            if (none) {
                total = mean = 0.0f;
            }
            log_total = logf(total);
        }
        auto log_prob = [&](float v) { return mx == -INFINITY ? -INFINITY : (v - mx) - log_total; };
        auto emit = [&](int place, Key key) {
            p.top_tokens[row * top + place] = static_cast<uint16_t>(key_column(key));
            p.top_log_probs[row * top + place] = log_prob(key_value(key));
        };
        // The slice's `top` largest: written out, or into the first CTA's memory.
        auto place_key = [&](int place, Key key) {
            if (p.ranks == 1) {
                emit(place, key);
            } else {
                const uint32_t to = sm100::map_to_cta(sm100::smem_u32(&best[parity][rank * kMostTop + place]), 0);
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
            }
        };
        if (top > 0 && goes_on) {
            if (collected) {
                for (int c = tid; c < found; c += kThreads) {
                    const Key key = shared.lists[parity].candidates[c];
                    int larger = 0;
#pragma unroll 8
                    for (int other = 0; other < found; ++other) {
                        larger += shared.lists[parity].candidates[other] > key ? 1 : 0;
                    }
                    if (larger < top) {
                        place_key(larger, key);
                    }
                }
                if (found < top && warp == 0) {
                    // Fewer than that are above minus infinity: the first columns that are not.
                    int place = found;
                    const int end = min((first_word + words) * W::kValues, p.vocab);
                    for (int c = first_word * W::kValues; place < top && c < end; c += 32) {
                        const bool mine = c + lane < end && W::value(values, c + lane) == -INFINITY;
                        const unsigned those = __ballot_sync(fb::kFullMask, mine);
                        const int at = place + __popc(those & ((1u << lane) - 1));
                        if (mine && at < top) {
                            place_key(at, order_key(-INFINITY, c + lane));
                        }
                        place += __popc(those);
                    }
                    for (int at = place + lane; at < top; at += 32) {
                        place_key(at, 0);     // (the slice has no more columns; another CTA's has)
                    }
                }
            } else {
                Key before = ~Key{0};
                for (int k = 0; k < top; ++k) {
                    Key mine = 0;
                    const int end = min((first_word + words) * W::kValues, p.vocab);
                    for (int c = first_word * W::kValues + tid; c < end; c += kThreads) {
                        const Key key = order_key(W::value(values, c), c);
                        mine = key < before && key > mine ? key : mine;
                    }
#pragma unroll
                    for (int off = 16; off > 0; off >>= 1) {
                        const Key other = __shfl_xor_sync(fb::kFullMask, mine, off);
                        mine = other > mine ? other : mine;
                    }
                    __syncthreads();
                    if (lane == 0) {
                        reduced[warp] = mine;
                    }
                    __syncthreads();
                    for (int w = 0; w < kWarps; ++w) {
                        mine = reduced[w] > mine ? reduced[w] : mine;
                    }
                    before = mine;
                    if (tid == 0) {
                        place_key(k, mine);
                    }
                }
            }
        }
        if (p.ranks > 1) {
            if (tid == 0) {
                const float mine[3] = {mx, total, mean};
                for (int i = 0; i < 3; ++i) {
                    const uint32_t to = sm100::map_to_cta(sm100::smem_u32(&parts[parity][rank][i]), 0);
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(mine[i]) : "memory");
                }
            }
            sm100::cluster_sync_all();
            if (rank != 0) {
                continue;
            }
            mx = -INFINITY;
            for (int r = 0; r < p.ranks; ++r) {
                mx = max_nan(mx, parts[parity][r][0]);
            }
            total = mean = 0.0f;
            for (int r = 0; r < p.ranks; ++r) {
                const float m = parts[parity][r][0];
                if (m != -INFINITY) {
                    const float below = max_nan(m - mx, kLowest), weight = expf(below);
                    total = fmaf(weight, parts[parity][r][1], total);
                    mean = fmaf(weight, fmaf(parts[parity][r][1], below, parts[parity][r][2]), mean);
                }
            }
            log_total = logf(total);
            for (int c = tid; c < p.ranks * top; c += kThreads) {
                const Key key = best[parity][c / top * kMostTop + c % top];
                int larger = 0;
                for (int r = 0; r < p.ranks; ++r) {
                    for (int k = 0; k < top; ++k) {
                        larger += best[parity][r * kMostTop + k] > key ? 1 : 0;
                    }
                }
                if (key != 0 && larger < top) {
                    emit(larger, key);
                }
            }
        }
        if (scribe) {
            if (p.log_probs != nullptr) {
                p.log_probs[row] = target < p.vocab ? log_prob(target_value) : 0.0f;
            }
            if (p.entropy != nullptr) {
                p.entropy[row] = mx == -INFINITY ? 0.0f : log_total - mean / total;
            }
            if (p.lse != nullptr) {
                p.lse[row] = mx == -INFINITY ? -INFINITY : mx + log_total;
            }
            target = next_target;
            target_value = next_value;
        }
    }
    if (gave_up && tid == 0) {
        // Copies that were started get a second, equally bounded chance to land before the memory goes.
        atomicExch(&g_log_probs_error, 1);
        const long long start = clock64();
        while (clock64() - start < 2000000LL) {
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------

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
    int chunk;          // words of a row, or of several rows, that a block takes at a time
    int row_chunks;     // chunks of a row; 1 where a block takes several rows
    int chunk_rows;     // rows that a block takes at a time
};

// dx_c = a ([c = target] - p_c) - b p_c (log p_c + entropy) with log p_c = x_c - lse: one pass, bound by what it
// reads and writes (4,096 FP16 rows of 50,304: 140 us, 0.90 of the copy rate). A thread has four 16-byte words on
// their way at a time.
constexpr int kGradientThreads = 512;
constexpr int kGradientWords = 4;

// What a row's gradient needs: e^d (slope d + constant), and `a` more at the target; zeros for a row without tokens.
template <typename T>
struct RowGradient {
    fb::F2 minus_lse, slope, constant;
    float a;
    int target;
    bool low;      // its logits are to be raised
    __device__ __forceinline__ RowGradient(const LogProbGradientArgs& p, size_t row) {
        target = p.targets != nullptr ? p.targets[row] : p.vocab;
        a = p.d_log_probs != nullptr && target < p.vocab ? p.d_log_probs[row] : 0.0f;
        float b = p.d_entropy != nullptr ? p.d_entropy[row] : 0.0f;
        float lse = p.lse[row], entropy = p.d_entropy != nullptr ? p.entropy[row] : 0.0f;
        if (lse == -INFINITY) {
            lse = a = b = entropy = 0.0f;
            target = -1;
        }
        low = sizeof(T) == 2 && lse < kLowRow;
        lse += low ? kRaise : 0.0f;
        minus_lse = fb::f2_pack(-lse, -lse);
        slope = fb::f2_pack(-b, -b);
        const float rest = -fmaf(b, entropy, a);
        constant = fb::f2_pack(rest, rest);
    }
    __device__ __forceinline__ uint4 word(const uint4& q, int column, int vocab) const {
        using W = Word<T>;
        float v[W::kValues], out[W::kValues];
        W::unpack_finite(v, q);
#pragma unroll
        for (int c = 0; c < W::kValues; c += 2) {
            const fb::F2 d = W::clamp(fb::f2_add(fb::f2_pack(v[c], v[c + 1]), minus_lse));
            float y0, y1, e0, e1;
            fb::f2_unpack(fb::f2_mul(d, fb::f2_pack(kLog2e, kLog2e)), y0, y1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(y0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(y1));
            fb::f2_unpack(fb::f2_mul(fb::f2_pack(e0, e1), fb::f2_fma(slope, d, constant)), out[c], out[c + 1]);
        }
        // (Rare, and so kept out of the way as a branch.)
        if (static_cast<unsigned>(target - column) < W::kValues || column + W::kValues > vocab) {
#pragma unroll 1
            for (int c = 0; c < W::kValues; ++c) {
                const float at_target = column + c == target ? a : 0.0f;
#pragma unroll
                for (int k = 0; k < W::kValues; ++k) {
                    out[k] = k == c ? (column + c < vocab ? out[k] + at_target : 0.0f) : out[k];
                }
            }
        }
        return W::pack(out);
    }
};

// kLong: a block takes pieces of one row, whose numbers all its threads share; else whole rows.
template <typename T, bool kLong>
__global__ void __launch_bounds__(kGradientThreads) fb_token_log_probs_backward(const LogProbGradientArgs p) {
    using W = Word<T>;
    fb::dependency_wait();
    fb::dependency_release();
    const uint4* logits = fb::after_wait(static_cast<const uint4*>(p.logits));
    const int row_words = p.cols / W::kValues;
    const int read_words = (p.vocab + W::kValues - 1) / W::kValues;
    const size_t groups = (p.rows + p.chunk_rows - 1) / p.chunk_rows;
    for (size_t item = blockIdx.x; item < groups * p.row_chunks; item += gridDim.x) {
        const size_t first_row = kLong ? item / p.row_chunks : item * p.chunk_rows;
        const int first_word = kLong ? static_cast<int>(item - first_row * p.row_chunks) * p.chunk : 0;
        const int here = kLong ? min(p.chunk, row_words - first_word)
                               : static_cast<int>(min(static_cast<size_t>(p.chunk_rows), p.rows - first_row)) * row_words;
        const uint4* in = logits + first_row * row_words + first_word;
        uint4* out = static_cast<uint4*>(p.dlogits) + first_row * row_words + first_word;
        uint4 held[kGradientWords];
#pragma unroll
        for (int j = 0; j < kGradientWords; ++j) {
            const int i = static_cast<int>(threadIdx.x) + j * kGradientThreads;
            const int word = kLong ? first_word + i : i % row_words;
            held[j] = make_uint4(0u, 0u, 0u, 0u);
            if (i < here && word < read_words) {
                held[j] = in[i];       // (not load_input: dlogits may be logits)
            }
        }
        if constexpr (kLong) {
            const RowGradient<T> row(p, first_row);
            if (row.low) {
#pragma unroll
                for (int j = 0; j < kGradientWords; ++j) {
                    raise_word(held[j], T());
                }
            }
#pragma unroll
            for (int j = 0; j < kGradientWords; ++j) {
                const int i = static_cast<int>(threadIdx.x) + j * kGradientThreads;
                if (i < here) {
                    __stcs(out + i, row.word(held[j], (first_word + i) * W::kValues, p.vocab));
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kGradientWords; ++j) {
                const int i = static_cast<int>(threadIdx.x) + j * kGradientThreads;
                if (i < here) {
                    const int r = i / row_words;
                    const RowGradient<T> row(p, first_row + r);
                    if (row.low) {
                        raise_word(held[j], T());
                    }
                    __stcs(out + i, row.word(held[j], (i - r * row_words) * W::kValues, p.vocab));
                }
            }
        }
    }
}

template <typename T, int kThreads, int kHeld>
cudaError_t launch_form(LogProbArgs p, int ranks, int sms, cudaStream_t stream) {
    const int words = (p.vocab + Word<T>::kValues - 1) / Word<T>::kValues;
    p.ranks = ranks;
    p.slice = (words + ranks - 1) / ranks;
    const size_t smem = kHeld == 0 ? static_cast<size_t>(p.slice) * 16 : 0;
    if (kHeld == 0) {
        static std::atomic<bool> configured[64] = {};
        const cudaError_t e = fb::allow_shared_memory(fb_token_log_probs<T, kThreads, kHeld>, kStagedWords * 16, configured);
        if (e != cudaSuccess) {
            return e;
        }
    }
    const size_t resident = static_cast<size_t>(blocks_per_sm(kThreads, kHeld)) * sms;
    const size_t clusters = std::max<size_t>(1, std::min(p.rows, resident / ranks));
    const dim3 grid(static_cast<unsigned>(clusters * ranks));
    if (ranks == 1) {
        return fb::launch_dependent(fb_token_log_probs<T, kThreads, kHeld>, grid, dim3(kThreads), smem, stream, p);
    }
    return fb::launch_dependent_cluster(fb_token_log_probs<T, kThreads, kHeld>, grid, dim3(kThreads),
                                        static_cast<unsigned>(ranks), smem, stream, p);
}

// Rows of up to 1,664 words (13,312 FP16 columns) take blocks of 128 threads, so that several rows are on an SM;
// longer ones 512 threads, and as many CTAs of a cluster as have room for them in half an SM's shared memory.
// Few rows are divided further, as long as the GPU has CTAs for it and each keeps 512 words.
template <typename T>
cudaError_t launch_forward(const LogProbArgs& p, int sms, cudaStream_t stream) {
    const int words = (p.vocab + Word<T>::kValues - 1) / Word<T>::kValues;
    if (words <= 4 * 128) {
        return launch_form<T, 128, 4>(p, 1, sms, stream);
    }
    if (words <= 13 * 128 && p.rows * 2 > static_cast<size_t>(sms)) {
        return launch_form<T, 128, 13>(p, 1, sms, stream);
    }
    int ranks = 1;
    while ((words + ranks - 1) / ranks > kStagedWords ||
           (ranks < kMostRanks && p.rows * ranks * 2 <= static_cast<size_t>(sms) && words / ranks >= 2 * 512)) {
        ranks *= 2;
    }
    return (words + ranks - 1) / ranks <= 4 * 512 ? launch_form<T, 512, 4>(p, ranks, sms, stream)
                                                  : launch_form<T, kStagedThreads, 0>(p, ranks, sms, stream);
}

template <typename T>
cudaError_t launch_backward(LogProbGradientArgs p, int sms, cudaStream_t stream) {
    const int words = p.cols / Word<T>::kValues;
    p.chunk = kGradientThreads * kGradientWords;
    p.row_chunks = words > p.chunk ? (words + p.chunk - 1) / p.chunk : 1;
    p.chunk_rows = p.row_chunks > 1 ? 1 : p.chunk / words;
    const size_t items = (p.rows + p.chunk_rows - 1) / p.chunk_rows * p.row_chunks;
    const unsigned blocks = static_cast<unsigned>(std::min<size_t>(items, 4 * static_cast<size_t>(sms)));
    return fb::launch_dependent(p.row_chunks > 1 ? fb_token_log_probs_backward<T, true> : fb_token_log_probs_backward<T, false>,
                                dim3(blocks), dim3(kGradientThreads), 0, stream, p);
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

namespace fb {

cudaError_t log_probs_error_flag(int* value, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(value, g_log_probs_error, sizeof(int));
    if (e == cudaSuccess && reset && *value != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_log_probs_error, &zero, sizeof(int));
    }
    return e;
}

}  // namespace fb

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
    FB_CUDA(fp32_logits != 0 ? launch_forward<float>(p, sms, stream) : launch_forward<__half>(p, sms, stream));
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
    FB_CUDA(fp32_logits != 0 ? launch_backward<float>(p, sms, stream) : launch_backward<__half>(p, sms, stream));
    return FLINT_OK;
}

}  // extern "C"
