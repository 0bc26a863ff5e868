// Beam search's selection: the best continuations of each group of beams over beams and vocabulary (an extension: the
// reference has no decoding).
//
// A beam's continuation by token c has the total  score + x_c - lse.  Within a beam the order is that of the logits, so a row
// needs its log-sum-exp and its `beams` largest logits alone. The first launch reads the logits once: a row falls into parts, a
// part into 64 bins of neighbouring lanes, and what is not below the beams-th largest of the bins' maxima (a lower
// bound of the beams-th largest logit; about `beams` values) is collected and put in order by counting. The second launch
// has a block per group: the beams-th largest of its lists' heads bounds the totals in the same way, and few are left to be
// ordered. Totals are FP64 there, because two beams' continuations can be closer than FP32 tells apart; a tie goes to the
// lower beam, then the lower token.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.h"
#include "device_utils.cuh"
#include "flint/flint_b200.h"
#include "logits.cuh"
#include "pages.h"

namespace {

constexpr int kMostBeams = 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 64;
constexpr int kLanes = kThreads / kBins;
constexpr int kCandidates = 512;
constexpr int kMostLists = 256;      // of a group
constexpr int kHeldWords = 8;        // 16-byte words of a part per thread
constexpr float kLog2e = 1.4426950408889634f;

__device__ int g_beams_error = 0;

struct RowArgs {
    const void* logits;
    const int* finished;      // may be null
    float2* stats;            // [row][part] the part's maximum m and its sum of e^(x - m)
    Key* best;                // [row][part][beams] its largest logits in order; 0 where it has no more above minus infinity
    long long items;          // rows * parts
    int vocab, cols, beams;
    int parts, slice;         // words of a part
};

template <typename T>
struct Row;
template <>
struct Row<float> {
    static constexpr int kValues = 4;
    __device__ static __forceinline__ float value(const void* row, int c) { return static_cast<const float*>(row)[c]; }
    __device__ static __forceinline__ void unpack(float (&v)[4], const uint4& q) {
        v[0] = __uint_as_float(q.x);
        v[1] = __uint_as_float(q.y);
        v[2] = __uint_as_float(q.z);
        v[3] = __uint_as_float(q.w);
    }
};
template <>
struct Row<__half> {
    static constexpr int kValues = 8;
    __device__ static __forceinline__ float value(const void* row, int c) {
        return __half2float(static_cast<const __half*>(row)[c]);
    }
    __device__ static __forceinline__ void unpack(float (&v)[8], const uint4& q) { fb::unpack8(v, q); }
};

// Sums of e^(x - m): the difference first, which is exact near m.
struct Exponentials {
    float minus_m, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ explicit Exponentials(float m) : minus_m(-m) {}
    template <int kValues>
    __device__ __forceinline__ void add(const float (&v)[kValues]) {
        const fb::F2 minus = fb::f2_pack(minus_m, minus_m), log2e = fb::f2_pack(kLog2e, kLog2e);
#pragma unroll
        for (int c = 0; c < kValues; c += 2) {
            float y0, y1, e0, e1;
            fb::f2_unpack(fb::f2_mul(fb::f2_add(fb::f2_pack(v[c], v[c + 1]), minus), log2e), y0, y1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(y0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(y1));
            sum[c & 2] += e0;
            sum[(c & 2) + 1] += e1;
        }
    }
    __device__ __forceinline__ float total() const { return (sum[0] + sum[1]) + (sum[2] + sum[3]); }
};

template <typename T, int kHeld>
__global__ void __launch_bounds__(kThreads, kHeld > 2 ? 3 : 4) fb_beam_rows(const RowArgs p) {
    using R = Row<T>;
    // Two of each, for parts in turn: one barrier less at a part's end.
    __shared__ float bins[2][kBins];
    __shared__ Key candidates[2][kCandidates];
    __shared__ float maxima[2][kWarps], sums[2][kWarps], least[2];
    __shared__ int counts[2];
    __shared__ Key reduced[kWarps];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    const int row_words = p.cols / R::kValues;
    const int all_words = (p.vocab + R::kValues - 1) / R::kValues;
    const int last_count = p.vocab - (all_words - 1) * R::kValues;
    if (tid < 2) {
        counts[tid] = 0;
    }
    fb::dependency_wait();
    fb::dependency_release();
    __syncthreads();
    struct Part {
        long long row;
        int first, words;      // 0 words: the beam is finished, or there is no part
    };
    auto part_at = [&](long long item) {
        Part part = {0, 0, 0};
        if (item < p.items) {
            part.row = item / p.parts;
            part.first = static_cast<int>(item - part.row * p.parts) * p.slice;
            part.words = p.finished != nullptr && p.finished[part.row] != 0 ? 0 : max(0, min(p.slice, all_words - part.first));
        }
        return part;
    };
    auto words_of = [&](const Part& part) { return static_cast<const uint4*>(p.logits) + part.row * row_words + part.first; };
    const long long stride = gridDim.x;
    Part part = part_at(blockIdx.x), next = part_at(blockIdx.x + stride);
    uint4 held[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        if (tid + j * kThreads < part.words) {
            held[j] = words_of(part)[tid + j * kThreads];
        }
    }
    int parity = 0;
    for (long long item = blockIdx.x; item < p.items; item += stride) {
        const Part after = part_at(item + 2 * stride);
        const uint4* next_words = words_of(next);
        if (part.words == 0) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                if (tid + j * kThreads < next.words) {
                    held[j] = next_words[tid + j * kThreads];
                }
            }
            part = next;
            next = after;
            continue;
        }
        Max<T> running;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = tid + j * kThreads;
            if (i < part.words) {
                if (part.first + i == all_words - 1) {
                    cut_word(held[j], last_count, T());
                }
                running.add(held[j]);
            }
        }
        const float my_max = running.value();
        float mx = my_max;
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) {
            mx = max_nan(mx, __shfl_xor_sync(fb::kFullMask, mx, off));
        }
        if (tid % kLanes == 0) {
            bins[parity][tid / kLanes] = mx;
        }
#pragma unroll
        for (int off = kLanes; off < 32; off <<= 1) {
            mx = max_nan(mx, __shfl_xor_sync(fb::kFullMask, mx, off));
        }
        if (lane == 0) {
            maxima[parity][warp] = mx;
        }
        __syncthreads();
        if (tid == 0) {
            counts[parity ^ 1] = 0;      // (of the part before, which everybody is done with)
        }
        mx = maxima[parity][lane % kWarps];
#pragma unroll
        for (int off = 1; off < kWarps; off <<= 1) {
            mx = max_nan(mx, __shfl_xor_sync(fb::kFullMask, mx, off));
        }
        // The beams-th largest of the bins' maxima, equal ones counted each: a warp ranks its share of the bins.
        const float low = bins[parity][lane], high = bins[parity][lane + 32];
#pragma unroll
        for (int i = 0; i < kBins / kWarps; ++i) {
            const int bin = warp * (kBins / kWarps) + i;
            const float value = bins[parity][bin];
            const int larger = __popc(__ballot_sync(fb::kFullMask, low > value || (low == value && lane < bin))) +
                               __popc(__ballot_sync(fb::kFullMask, high > value || (high == value && lane + 32 < bin)));
            if (larger == p.beams - 1 && lane == 0) {
                least[parity] = value;      // (none is where bins are NaN)
            }
        }
        __syncthreads();
        const float bound = least[parity];
        const bool counts_for_nothing = !(mx > -INFINITY && mx < INFINITY);      // NaN, plus infinity, or nothing there
        if (!counts_for_nothing && __any_sync(fb::kFullMask, my_max >= bound)) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int i = tid + j * kThreads;
                if (i < part.words && Max<T>::word(held[j]) >= bound) {
                    float v[R::kValues];
                    R::unpack(v, held[j]);
#pragma unroll
                    for (int c = 0; c < R::kValues; ++c) {
                        if (v[c] >= bound && v[c] > -INFINITY) {
                            const int at = atomicAdd(&counts[parity], 1);
                            if (at < kCandidates) {
                                candidates[parity][at] = order_key(v[c], (part.first + i) * R::kValues + c);
                            }
                        }
                    }
                }
            }
        }
        Exponentials exponentials(mx);
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = tid + j * kThreads;
            if (i < part.words) {
                float v[R::kValues];
                R::unpack(v, held[j]);
                exponentials.add(v);
            }
            if (i < next.words) {
                held[j] = next_words[i];
            }
        }
        float total = exponentials.total();
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            total += __shfl_xor_sync(fb::kFullMask, total, off);
        }
        if (lane == 0) {
            sums[parity][warp] = total;
        }
        __syncthreads();
        Key* best = p.best + item * p.beams;
        const int found = counts[parity];
        if (warp == kWarps - 1) {
            total = sums[parity][lane % kWarps];
#pragma unroll
            for (int off = 1; off < kWarps; off <<= 1) {
                total += __shfl_xor_sync(fb::kFullMask, total, off);
            }
            if (lane == 0) {
                // (A part of nothing but minus infinity adds nothing, one with a NaN or plus infinity makes the row NaN.)
                p.stats[item] = make_float2(mx, mx == -INFINITY ? 0.0f : total);
            }
        }
        if (found <= kCandidates) {
            for (int c = tid; c < found; c += kThreads) {
                const Key key = candidates[parity][c];
                int larger = 0;
#pragma unroll 8
                for (int other = 0; other < found; ++other) {
                    larger += candidates[parity][other] > key ? 1 : 0;
                }
                if (larger < p.beams) {
                    best[larger] = key;
                }
            }
            for (int c = found + tid; c < p.beams; c += kThreads) {
                best[c] = 0;
            }
        } else {
            // Many equal ones: the part is gone through once for every place.
            const char* row = static_cast<const char*>(p.logits) + part.row * p.cols * sizeof(T);
            const int begin = part.first * R::kValues, end = min((part.first + part.words) * R::kValues, p.vocab);
            Key before = ~Key{0};
            for (int k = 0; k < p.beams; ++k) {
                Key mine = 0;
                for (int c = begin + tid; c < end; c += kThreads) {
                    const float v = R::value(row, c);
                    const Key key = v > -INFINITY ? order_key(v, c) : 0;
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
                    best[k] = mine;
                }
            }
        }
        parity ^= 1;
        part = next;
        next = after;
    }
}

struct GroupArgs {
    float* next_scores;
    int* parents;
    uint16_t* tokens;
    int* next_finished;       // may be null, as all below
    int* next_lengths;
    uint16_t* next_histories;
    const float* scores;
    const int* finished;
    const int* lengths;
    const uint16_t* histories;
    const float2* stats;
    const Key* best;
    long long history_stride;
    int beams, parts, end_token;
    float power;
};

// A number that orders totals; 0 for none.
__device__ __forceinline__ Key order_total(double v) {
    if (!(v > -INFINITY)) {
        return 0;
    }
    const Key bits = static_cast<Key>(__double_as_longlong(v + 0.0));
    return (bits >> 63) != 0 ? ~bits : bits | (Key{1} << 63);
}

struct Candidate {
    Key rank;
    unsigned place;      // beam, token
    __device__ __forceinline__ bool above(const Candidate& other) const {
        return rank > other.rank || (rank == other.rank && place < other.place);
    }
};

__global__ void __launch_bounds__(kThreads) fb_beam_groups(const GroupArgs p) {
    __shared__ double score_of[kMostBeams], lse_of[kMostBeams], norm_of[kMostBeams];
    __shared__ int over_of[kMostBeams], length_of[kMostBeams];
    __shared__ float2 stats[kMostLists];
    __shared__ Candidate heads[kMostLists];
    __shared__ Candidate bound;
    __shared__ Candidate left[kMostBeams * kMostBeams];
    __shared__ double left_total[kMostBeams * kMostBeams];
    __shared__ int left_count;
    __shared__ unsigned chosen[kMostBeams];
    __shared__ double chosen_total[kMostBeams];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    fb::dependency_wait();
    fb::dependency_release();
    const long long first = static_cast<long long>(blockIdx.x) * p.beams;
    const int lists = p.beams * p.parts;
    if (tid < lists) {
        stats[tid] = p.stats[first * p.parts + tid];
    }
    if (tid == 0) {
        left_count = 0;
        bound = Candidate{1, ~0u};      // anything that is a continuation
    }
    if (tid < p.beams) {
        chosen[tid] = ~0u;
        const float score = p.scores[first + tid];
        over_of[tid] = p.finished != nullptr && p.finished[first + tid] != 0 ? 1 : 0;
        int length = p.lengths != nullptr ? p.lengths[first + tid] : 0;
        if (length < 0 || (p.histories != nullptr && length > p.history_stride)) {
            atomicExch(&g_beams_error, 1);
            length = length < 0 ? 0 : static_cast<int>(p.history_stride);
        }
        length_of[tid] = length;
        score_of[tid] = fabsf(score) < INFINITY ? static_cast<double>(score) : -INFINITY;
        const double grown = over_of[tid] != 0 ? max(length, 1) : static_cast<double>(length) + 1.0;
        norm_of[tid] = p.power == 0.0f ? 1.0 : pow(grown, static_cast<double>(p.power));
    }
    __syncthreads();
    if (tid < p.beams) {
        // (A finished beam's row was not read.)
        double lse = 0.0;
        if (over_of[tid] == 0) {
            float m = -INFINITY, sum = 0.0f;
            for (int i = 0; i < p.parts; ++i) {
                m = max_nan(m, stats[tid * p.parts + i].x);
            }
            for (int i = 0; i < p.parts; ++i) {
                const float2 part = stats[tid * p.parts + i];
                sum += part.x == -INFINITY ? 0.0f : part.y * expf(part.x - m);
            }
            lse = static_cast<double>(m) + log(static_cast<double>(sum));
        }
        lse_of[tid] = lse;
    }
    __syncthreads();
    auto candidate_at = [&](int list, int i, double& total) {
        const int beam = list / p.parts;
        if (over_of[beam] != 0) {
            total = list % p.parts == 0 && i == 0 ? score_of[beam] : -INFINITY;
            return Candidate{order_total(total / norm_of[beam]), static_cast<unsigned>(beam) << 16 | static_cast<unsigned>(max(p.end_token, 0))};
        }
        const Key key = p.best[(first * p.parts + list) * p.beams + i];
        // (An lse that is not a number, or minus infinity, gives none.)
        total = key != 0 ? score_of[beam] + (static_cast<double>(key_value(key)) - lse_of[beam]) : -INFINITY;
        total = total < INFINITY ? total : -INFINITY;
        return Candidate{order_total(total / norm_of[beam]), static_cast<unsigned>(beam) << 16 | static_cast<unsigned>(key_column(key) & 0xffff)};
    };
    double total;
    if (tid < lists) {
        heads[tid] = candidate_at(tid, 0, total);
    }
    __syncthreads();
    if (tid < lists && heads[tid].rank != 0) {
        int larger = 0;
        for (int other = 0; other < lists; ++other) {
            larger += heads[other].above(heads[tid]) ? 1 : 0;
        }
        if (larger == p.beams - 1) {
            bound = heads[tid];
        }
    }
    __syncthreads();
    for (int i = tid; i < lists * p.beams; i += kThreads) {
        const int list = i / p.beams;
        if (heads[list].rank == 0 || bound.above(heads[list])) {
            continue;
        }
        const Candidate mine = candidate_at(list, i - list * p.beams, total);
        if (mine.rank != 0 && !bound.above(mine)) {
            const int at = atomicAdd(&left_count, 1);
            left[at] = mine;
            left_total[at] = total;
        }
    }
    __syncthreads();
    const int count = left_count;
    for (int i = tid; i < count; i += kThreads) {
        int larger = 0;
        for (int other = 0; other < count; ++other) {
            larger += left[other].above(left[i]) ? 1 : 0;
        }
        if (larger < p.beams) {
            chosen[larger] = left[i].place;
            chosen_total[larger] = left_total[i];
        }
    }
    __syncthreads();
    // A warp per beam: its numbers, and its history.
    for (int t = warp; t < p.beams; t += kWarps) {
        const bool none = chosen[t] == ~0u;
        const int parent = none ? t : static_cast<int>(chosen[t] >> 16);
        const bool over = over_of[parent] != 0;
        const int token = none ? (over ? max(p.end_token, 0) : 0) : static_cast<int>(chosen[t] & 0xffffu);
        int length = length_of[parent];
        const long long row = first + t;
        if (p.next_histories != nullptr) {
            const uint16_t* from = p.histories + (first + parent) * p.history_stride;
            uint16_t* to = p.next_histories + row * p.history_stride;
            for (int c = lane; c < length; c += 32) {
                to[c] = from[c];
            }
            if (!over && length == p.history_stride) {
                atomicExch(&g_beams_error, 1);
                --length;      // (stays as long as it is, and keeps its last token)
            } else if (!over && lane == 0) {
                to[length] = static_cast<uint16_t>(token);
            }
        }
        if (lane == 0) {
            p.next_scores[row] = none ? -INFINITY : static_cast<float>(chosen_total[t]);
            p.parents[row] = static_cast<int>(first) + parent;
            p.tokens[row] = static_cast<uint16_t>(token);
            if (p.next_finished != nullptr) {
                p.next_finished[row] = over || token == p.end_token ? 1 : 0;
            }
            if (p.next_lengths != nullptr) {
                p.next_lengths[row] = over ? length : length + 1;
            }
        }
    }
}

// Parts of a row: as many as have room in a block's registers, and where rows are few as many as give two blocks to every
// SM something to do, but each at least a word per thread.
int parts_of(int words, size_t rows, int beams, int sms) {
    const int least = (words + kThreads * kHeldWords - 1) / (kThreads * kHeldWords);
    const size_t wanted = std::min<size_t>(2 * static_cast<size_t>(sms) / std::max<size_t>(rows, 1),
                                           static_cast<size_t>((words + kThreads - 1) / kThreads));
    return std::max(least, static_cast<int>(std::min<size_t>(wanted, static_cast<size_t>(kMostLists / beams))));
}

// Rows' parts are at most eight, or two per SM together.
size_t most_lists(size_t rows, int sms) { return 8 * rows + 2 * static_cast<size_t>(sms); }
size_t stats_bytes(size_t lists) { return (lists * sizeof(float2) + 255) / 256 * 256; }

template <typename T>
cudaError_t launch_rows(RowArgs p, size_t rows, int sms, cudaStream_t stream) {
    const int words = (p.vocab + Row<T>::kValues - 1) / Row<T>::kValues;
    p.parts = parts_of(words, rows, p.beams, sms);
    p.slice = (words + p.parts - 1) / p.parts;
    p.items = static_cast<long long>(rows) * p.parts;
    const bool few = p.slice <= 2 * kThreads;
    const unsigned blocks = static_cast<unsigned>(std::min<long long>(p.items, (few ? 4LL : 3LL) * sms));
    return fb::launch_dependent(few ? fb_beam_rows<T, 2> : fb_beam_rows<T, kHeldWords>, dim3(blocks), dim3(kThreads), 0,
                                stream, p);
}

constexpr flint_status kBad = FLINT_ERROR_INVALID_ARGUMENT;
constexpr size_t kMostRows = size_t{1} << 20;

flint_status check_beams(const char* name, size_t groups, size_t beams) {
    if (beams == 0 || beams > static_cast<size_t>(kMostBeams)) {
        return fb::fail(kBad, "%s: beams (%zu) must be from 1 to %d", name, beams, kMostBeams);
    }
    if (groups > kMostRows / beams) {
        return fb::fail(kBad, "%s: groups (%zu) times beams (%zu) can be up to %zu", name, groups, beams, kMostRows);
    }
    return FLINT_OK;
}

}  // namespace

namespace fb {

cudaError_t beams_error_flag(int* value, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(value, g_beams_error, sizeof(int));
    if (e == cudaSuccess && reset && *value != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_beams_error, &zero, sizeof(int));
    }
    return e;
}

}  // namespace fb

extern "C" {

flint_status flint_b200_beam_select_workspace(size_t groups, size_t beams, size_t* bytes) {
    constexpr const char* name = "flint_b200_beam_select_workspace";
    FB_TRY(check_beams(name, groups, beams));
    if (bytes == nullptr) {
        return fb::fail(kBad, "%s: bytes is null", name);
    }
    int sms = 148;
    FB_CUDA(fb::sm_count(&sms));
    const size_t lists = most_lists(groups * beams, sms);
    *bytes = stats_bytes(lists) + lists * beams * sizeof(Key);
    return FLINT_OK;
}

flint_status flint_b200_beam_select(void* next_scores, void* parents, void* tokens, void* next_finished,
                                    void* next_lengths, void* next_histories, const void* logits, const void* scores,
                                    const void* finished, const void* lengths, const void* histories,
                                    int fp32_logits, size_t groups, size_t beams, size_t vocab, size_t cols,
                                    size_t history_stride, int end_token, float length_power, void* workspace,
                                    size_t workspace_bytes, flint_stream stream) {
    constexpr const char* name = "flint_b200_beam_select";
    FB_TRY(check_beams(name, groups, beams));
    constexpr size_t kMaxCols = size_t{1} << 16;
    if (cols == 0 || cols % 8 != 0 || cols > kMaxCols) {
        return fb::fail(kBad, "%s: cols (%zu) must be a multiple of 8 from 8 to %zu", name, cols, kMaxCols);
    }
    if (vocab == 0 || vocab > cols) {
        return fb::fail(kBad, "%s: vocab (%zu) must be from 1 to cols (%zu)", name, vocab, cols);
    }
    if (end_token < -1 || (end_token >= 0 && static_cast<size_t>(end_token) >= vocab)) {
        return fb::fail(kBad, "%s: end_token (%d) must be -1 or below vocab (%zu)", name, end_token, vocab);
    }
    if (!std::isfinite(length_power) || length_power < 0.0f) {
        return fb::fail(kBad, "%s: length_power (%g) must be finite and not negative", name,
                        static_cast<double>(length_power));
    }
    const struct {
        const char* names;
        bool all, none, needed;
    } groups_of[] = {
        {"finished and next_finished", finished != nullptr && next_finished != nullptr,
         finished == nullptr && next_finished == nullptr, end_token >= 0},
        {"lengths and next_lengths", lengths != nullptr && next_lengths != nullptr,
         lengths == nullptr && next_lengths == nullptr, histories != nullptr || length_power > 0.0f},
        {"histories and next_histories", histories != nullptr && next_histories != nullptr,
         histories == nullptr && next_histories == nullptr, false},
    };
    for (const auto& g : groups_of) {
        if (!g.all && (!g.none || g.needed)) {
            return fb::fail(kBad, g.none ? "%s: %s must be given with these arguments" : "%s: %s go together", name, g.names);
        }
    }
    constexpr size_t kMostHistory = size_t{1} << 24;
    if (histories != nullptr && (history_stride == 0 || history_stride > kMostHistory)) {
        return fb::fail(kBad, "%s: history_stride (%zu) must be from 1 to %zu", name, history_stride, kMostHistory);
    }
    if (groups == 0) {
        return FLINT_OK;
    }
    size_t needed = 0;
    FB_TRY(flint_b200_beam_select_workspace(groups, beams, &needed));
    if (workspace_bytes < needed) {
        return fb::fail(kBad, "%s: needs %zu bytes of workspace, given %zu", name, needed, workspace_bytes);
    }
    if (logits == nullptr) {
        return fb::fail(kBad, "%s: logits is null", name);
    }
    const size_t rows = groups * beams;
    auto optional = [&](const char* what, const void* pointer, size_t bytes) {
        return pointer != nullptr ? fb::Span{what, pointer, bytes} : fb::Span{what, logits, 0};
    };
    const fb::Span spans[] = {
        {"next_scores", next_scores, rows * 4},
        {"parents", parents, rows * 4},
        {"tokens", tokens, rows * 2},
        optional("next_finished", next_finished, rows * 4),
        optional("next_lengths", next_lengths, rows * 4),
        optional("next_histories", next_histories, rows * history_stride * 2),
        {"workspace", workspace, needed},
        {"logits", logits, rows * cols * (fp32_logits != 0 ? 4 : 2)},
        {"scores", scores, rows * 4},
        optional("finished", finished, rows * 4),
        optional("lengths", lengths, rows * 4),
        optional("histories", histories, rows * history_stride * 2),
    };
    FB_TRY(fb::check_spans(name, spans, 7));
    int sms = 148;
    FB_CUDA(fb::sm_count(&sms));
    RowArgs p = {};
    p.logits = logits;
    p.finished = static_cast<const int*>(finished);
    p.stats = static_cast<float2*>(workspace);
    p.best = reinterpret_cast<Key*>(static_cast<char*>(workspace) + stats_bytes(most_lists(rows, sms)));
    p.vocab = static_cast<int>(vocab);
    p.cols = static_cast<int>(cols);
    p.beams = static_cast<int>(beams);
    GroupArgs g = {};
    g.next_scores = static_cast<float*>(next_scores);
    g.parents = static_cast<int*>(parents);
    g.tokens = static_cast<uint16_t*>(tokens);
    g.next_finished = static_cast<int*>(next_finished);
    g.next_lengths = static_cast<int*>(next_lengths);
    g.next_histories = static_cast<uint16_t*>(next_histories);
    g.scores = static_cast<const float*>(scores);
    g.finished = p.finished;
    g.lengths = static_cast<const int*>(lengths);
    g.histories = static_cast<const uint16_t*>(histories);
    g.stats = p.stats;
    g.best = p.best;
    g.history_stride = static_cast<long long>(history_stride);
    g.beams = p.beams;
    const int values = fp32_logits != 0 ? Row<float>::kValues : Row<__half>::kValues;
    g.parts = parts_of((p.vocab + values - 1) / values, rows, p.beams, sms);
    g.end_token = end_token;
    g.power = length_power;
    FB_CUDA(fp32_logits != 0 ? launch_rows<float>(p, rows, sms, stream) : launch_rows<__half>(p, rows, sms, stream));
    FB_CUDA(fb::launch_dependent(fb_beam_groups, dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream, g));
    return FLINT_OK;
}

}  // extern "C"
