// Beam search's selection: the best continuations of each group of beams over beams and vocabulary (an extension: the
// reference has no decoding).
//
// A beam's continuation by token c has the total  score + x_c - lse.  Within a beam the order is that of the logits, so a row
// needs its log-sum-exp and its `beams` largest logits alone. The first launch reads the logits once: a warp has a
// part of a row to itself, so that nothing waits for anything but memory. It takes sums against each lane's own running maximum and
// notes the maxima of groups of a few words. The beams-th largest of the lanes' two largest groups bounds the beams-th largest logit
// from below; the groups that reach it (about `beams`) are read again, from L2, and what reaches it is put in order by counting. The
// second launch has a block per group of beams and does the same with totals, in FP64, because two beams'
// continuations can be closer than FP32 tells apart; a tie goes to the lower beam, then the lower token.
//
// 5,000 rows of 50,257 FP16 logits take 99 to 102 us (4.3 TB/s): no unit is full (DRAM 57 %, special-function unit 57 %, issue slots 58 %); warps wait for
// memory most, with one chunk on its way while they sum the one before and room for 42 % of an SM's warps. 1,240 rows of 32,001 FP32 logits and 31 beams 49 us,
// where two parts of a row each leave 30 % of the warps without one, and a part's 31 candidates count as well; 512 rows 24 us and 4 rows 10.5 us,
// which are a warp's chain of loads and two launches' beginnings.
#include <algorithm>
#include <atomic>
#include <climits>
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
// Of rows of values of 16 / `values` bytes: 16-byte words that a lane has on their way (its values have a bit each), words that a
// warp works on at a time, and blocks per SM.
struct Form {
    int held, chunk, blocks;
};
__host__ __device__ constexpr Form form_of(int values) { return Form{32 / values, 32 * 32 / values, values == 4 ? 3 : 4}; }
constexpr int kCandidates = 128;     // of a warp
constexpr int kMany = 96;            // from which on the bound rises
constexpr int kGroups = 32;          // of a lane's words, whose maxima are noted
constexpr int kMostLists = 256;      // of a group
constexpr float kMostPower = 16.0f;  // of a length: what scores are divided by, and the quotients, are FP64 numbers then
constexpr float kLog2e = 1.4426950408889634f;

__device__ int g_beams_error = 0;

struct RowArgs {
    const void* logits;
    const int* finished;      // may be null
    float2* stats;            // [row][part] the part's maximum m and its sum of e^(x - m)
    Key* best;                // [row][part][beams] its largest logits in order; 0 where it has no more above minus infinity
    unsigned items;           // rows * parts
    int vocab, cols, beams;
    int parts, slice;         // words of a part
};

template <typename T>
struct Row;
template <>
struct Row<float> {
    static constexpr int kValues = 4;
    static constexpr float kLowestValue = -3.402823466e38f;
    __device__ static __forceinline__ float value(const void* row, int c) { return static_cast<const float*>(row)[c]; }
    // A bit for each of a word's values that is not below the bound, or (kAbove) that is above it.
    template <bool kAbove = false>
    __device__ static __forceinline__ unsigned reaching(const uint4& q, float bound) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
        unsigned those = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float v = __uint_as_float(w[c]);
            those |= (kAbove ? v > bound : v >= bound) ? 1u << c : 0u;
        }
        return those;
    }
};
template <>
struct Row<__half> {
    static constexpr int kValues = 8;
    static constexpr float kLowestValue = -65504.0f;
    __device__ static __forceinline__ float value(const void* row, int c) {
        return __half2float(static_cast<const __half*>(row)[c]);
    }
    // (A bound from upper bits is rounded to FP16 here if it is negative. Rounding is monotone, so that no value that is not below the bound
    // is left out; one that is below it can be among those, and is compared again in FP32. kAbove: the bound is one of the values.)
    template <bool kAbove = false>
    __device__ static __forceinline__ unsigned reaching(const uint4& q, float bound) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
        const __half2 both = __float2half2_rn(bound);
        unsigned those = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const __half2 v = *reinterpret_cast<const __half2*>(&w[c]);
            those |= (kAbove ? __hgt2_mask(v, both) : __hge2_mask(v, both)) & (0x20001u << (2 * c));
        }
        // Bits 2 c and 2 c + 17: the upper halves' go beside the lower ones'.
        return (those & 0xffffu) | (those >> 16);
    }
};

// A lane's sum of e^(x - m) against its running maximum m. It begins at the lowest number, so that minus infinity adds nothing.
// The difference comes first, which is exact near m; from FP16 it is one instruction.
constexpr float kLowest = -3.402823466e38f;
struct LaneSum {
    float m = kLowest;
    fb::F2 sum[2] = {0, 0};
    __device__ __forceinline__ void raise(float next) {
        const float factor = exp2f((m - next) * kLog2e);
        sum[0] = fb::f2_mul(sum[0], fb::f2_pack(factor, factor));
        sum[1] = fb::f2_mul(sum[1], fb::f2_pack(factor, factor));
        m = next;
    }
    __device__ __forceinline__ void add(const uint4& q, float) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            pair(i, __uint_as_float(w[i]) - m, __uint_as_float(w[i + 1]) - m);
        }
    }
    __device__ __forceinline__ void add(const uint4& q, __half) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float d0, d1;
            asm("{\n.reg .f16 lo, hi;\nmov.b32 {lo, hi}, %2;\nadd.rn.f32.f16 %0, lo, %3;\nadd.rn.f32.f16 %1, hi, %3;\n}"
                : "=f"(d0), "=f"(d1)
                : "r"(w[i]), "f"(-m));
            pair(2 * i, d0, d1);
        }
    }
    __device__ __forceinline__ void pair(int i, float d0, float d1) {
        float y0, y1, e0, e1;
        fb::f2_unpack(fb::f2_mul(fb::f2_pack(d0, d1), fb::f2_pack(kLog2e, kLog2e)), y0, y1);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(y0));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(y1));
        sum[i / 2 & 1] = fb::f2_add(sum[i / 2 & 1], fb::f2_pack(e0, e1));
    }
    __device__ __forceinline__ float total() const {
        float a, b;
        fb::f2_unpack(fb::f2_add(sum[0], sum[1]), a, b);
        return a + b;
    }
};

__device__ __forceinline__ unsigned upper(Key key) { return static_cast<unsigned>(key >> 32); }

// The largest number of kBits upper bits that k of the warp's values (kEach per lane, order_key's upper halves) reach.
template <int kBits, int kEach>
__device__ __forceinline__ unsigned reached_by(const unsigned (&mine)[kEach], int k) {
    unsigned least = 0;
#pragma unroll 4
    for (int bit = 31; bit >= 32 - kBits; --bit) {
        const unsigned trial = least | (1u << bit);
        int reach = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            reach += mine[i] >= trial ? 1 : 0;
        }
        if (__reduce_add_sync(fb::kFullMask, reach) >= k) {
            least = trial;
        }
    }
    return least;
}

// What is not below the k-th largest value of a warp's `count` candidates (up to kCandidates) stays, in order; how many that are,
// and the value. `exact`: of those equal to it the first columns only, k in all.
__device__ __noinline__ int keep_largest(Key* list, int count, int k, float& bound, int lane, bool exact) {
    Key mine[kCandidates / 32];
#pragma unroll
    for (int i = 0; i < kCandidates / 32; ++i) {
        mine[i] = lane + 32 * i < count ? list[lane + 32 * i] : 0;
    }
    unsigned values[kCandidates / 32];
#pragma unroll
    for (int i = 0; i < kCandidates / 32; ++i) {
        values[i] = upper(mine[i]);
    }
    const unsigned least = reached_by<32>(values, k);
    unsigned first = 0;      // of the equal ones, by their columns' places from the end
    if (exact) {
        int above = 0;
#pragma unroll
        for (int i = 0; i < kCandidates / 32; ++i) {
            above += values[i] > least ? 1 : 0;
            // (0xffffffff less the column, which has 16 bits.)
            values[i] = values[i] == least ? static_cast<unsigned>(mine[i]) << 16 | 1u : 0u;
        }
        first = reached_by<16>(values, k - __reduce_add_sync(fb::kFullMask, above));
    }
    __syncwarp();
    int kept = 0;
#pragma unroll
    for (int i = 0; i < kCandidates / 32; ++i) {
        const bool stays = mine[i] != 0 && (upper(mine[i]) > least || (upper(mine[i]) == least && (!exact || values[i] >= first)));
        const unsigned those = __ballot_sync(fb::kFullMask, stays);
        if (stays) {
            list[kept + __popc(those & ((1u << lane) - 1))] = mine[i];
        }
        kept += __popc(those);
    }
    __syncwarp();
    bound = fmaxf(bound, key_value(static_cast<Key>(least) << 32));
    return kept;
}

// What is among the `k` largest of a part (words [0, words) of `from`, its columns from `begin` on, those of the row's last word up to
// `end`), none of which is below the bound, where many are equal to the k-th largest: one pass in the order of columns. Behind
// a chunk with which k candidates reach the bound, only larger ones count. (Rows masked by a finite number, three tokens left: 512 rows
// of 50,257 49 us, 1,240 rows of 32,001 and 31 beams 123; with a pass per place 186 and 2,280. Without the mask 21 and 46.)
template <typename T>
__device__ __noinline__ int among_equals(Key* list, const uint4* from, int words, int begin, int end, int k, float bound, int lane) {
    using R = Row<T>;
    int count = 0;
    for (int chunk = 0; chunk < words; chunk += 32) {
        const int column = begin + (chunk + lane) * R::kValues;
        const bool all = count >= k;
        unsigned those = 0;
        if (chunk + lane < words) {
            uint4 q = from[chunk + lane];
            if (column + R::kValues > end) {
                cut_word(q, end - column, T());
            }
            those = all ? R::template reaching<true>(q, bound) : R::reaching(q, bound);
        }
        while (__any_sync(fb::kFullMask, those != 0)) {
            const int c = __ffs(those) - 1;
            const float v = c >= 0 ? R::value(from, (chunk + lane) * R::kValues + c) : -INFINITY;
            const bool reaches = c >= 0 && v >= bound;      // (which may have risen)
            const unsigned lanes = __ballot_sync(fb::kFullMask, reaches);
            those &= those - 1;
            if (reaches) {
                list[count + __popc(lanes & ((1u << lane) - 1))] = order_key(v, column + c);
            }
            count += __popc(lanes);
            if (count > kMany) {
                __syncwarp();
                count = keep_largest(list, count, k, bound, lane, true);
            }
        }
    }
    return count;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, form_of(Row<T>::kValues).blocks) fb_beam_rows(const RowArgs p) {
    using R = Row<T>;
    constexpr int kHeld = form_of(R::kValues).held, kChunk = form_of(R::kValues).chunk;
    __shared__ Key lists[kWarps][kCandidates];
    __shared__ T group_max[kWarps][kGroups][32];      // (a maximum of FP16 values is one)
    __shared__ int claimed;
    const int lane = static_cast<int>(threadIdx.x) % 32, warp = __shfl_sync(fb::kFullMask, static_cast<int>(threadIdx.x) / 32, 0);
    const int all_words = (p.vocab + R::kValues - 1) / R::kValues;
    const int last_count = p.vocab - (all_words - 1) * R::kValues;
    Key* list = lists[warp];
    // Chunks whose words make up a group, and the chunks in a part.
    const int chunks = (p.slice + kChunk - 1) / kChunk, of_group = (chunks + kGroups - 1) / kGroups;
    if (threadIdx.x == 0) {
        claimed = 0;
    }
    fb::dependency_wait();
    fb::dependency_release();
    __syncthreads();
    // A block's warps take its parts as they come to them (finished beams have nothing to read); neighbouring parts go to
    // different SMs.
    struct Part {
        unsigned item;           // p.items: there is none
        int first, words;        // its first word's place in the row, and how many
        const char* values;      // of the row
    };
    auto claim = [&]() {
        for (;;) {
            int turn = 0;
            if (lane == 0) {
                turn = atomicAdd(&claimed, 1);
            }
            turn = __shfl_sync(fb::kFullMask, turn, 0);
            const unsigned item = static_cast<unsigned>(turn) * gridDim.x + blockIdx.x;
            if (item >= p.items) {
                return Part{p.items, 0, 0, nullptr};
            }
            const unsigned row = item / static_cast<unsigned>(p.parts);
            if (p.finished == nullptr || p.finished[row] == 0) {
                const int first = static_cast<int>(item - row * p.parts) * p.slice;
                return Part{item, first, max(0, min(p.slice, all_words - first)),
                            static_cast<const char*>(p.logits) + static_cast<size_t>(row) * p.cols * sizeof(T)};
            }
        }
    };
    // Word i of a part; minus infinity, which counts for nothing, behind its end.
    auto word_at = [&](const Part& part, int i) {
        uint4 q = make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
        if (sizeof(T) == 4) {
            q = make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
        }
        if (i < part.words) {
            q = reinterpret_cast<const uint4*>(part.values)[part.first + i];
        }
        return q;
    };
    uint4 held[kHeld];
    Part part = claim();
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        held[j] = word_at(part, lane + 32 * j);
    }
    while (part.item < p.items) {
        const int first = part.first, words = part.words;
        const uint4* from = reinterpret_cast<const uint4*>(part.values) + first;
        auto cut = [&](uint4& q, int i) {
            if (first + i == all_words - 1) {
                cut_word(q, last_count, T());
            }
        };
        LaneSum sum;
        float best_group = -INFINITY, second_group = -INFINITY;
        int group = 0;
        for (int c = 0; c * kChunk < words;) {
            Max<T> running;
            for (int end = c + of_group; c < end && c * kChunk < words; ++c) {
                const int at = c * kChunk + lane;
                if (first + (c + 1) * kChunk >= all_words) {
#pragma unroll
                    for (int j = 0; j < kHeld; ++j) {
                        cut(held[j], at + 32 * j);
                    }
                }
                Max<T> here;
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    here.add(held[j]);
                }
                running.add(here);
                const float mx = here.value();
                if (!(mx <= sum.m)) {       // (a NaN stays)
                    sum.raise(mx);
                }
                if ((c + 2) * kChunk <= words) {
#pragma unroll
                    for (int j = 0; j < kHeld; ++j) {
                        sum.add(held[j], T());
                        held[j] = from[at + kChunk + 32 * j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kHeld; ++j) {
                        sum.add(held[j], T());
                        held[j] = word_at(part, at + kChunk + 32 * j);
                    }
                }
            }
            const float mx = running.value();
            group_max[warp][group++][lane] = static_cast<T>(mx);
            second_group = fmaxf(second_group, fminf(best_group, mx));
            best_group = fmaxf(best_group, mx);
        }
        // The next part's first words come while this one's largest are sought.
        const Part next = claim();
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            held[j] = word_at(next, lane + 32 * j);
        }
        float m = sum.m;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            m = max_nan(m, __shfl_xor_sync(fb::kFullMask, m, off));
        }
        float total = sum.total() * exp2f((sum.m - m) * kLog2e);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            total += __shfl_xor_sync(fb::kFullMask, total, off);
        }
        if (lane == 0) {
            // (A part of nothing but minus infinity adds nothing, one with a NaN or plus infinity makes the row NaN.)
            p.stats[part.item] = make_float2(m, total);
        }
        // 16 bits are sign, exponent and 7 bits of the fraction: enough for a bound. Minus infinity does not reach it.
        const unsigned tops[2] = {upper(order_key(best_group, 0)), upper(order_key(second_group, 0))};
        float bound = key_value(static_cast<Key>(reached_by<16>(tops, p.beams)) << 32);
        bound = bound >= R::kLowestValue ? bound : R::kLowestValue;      // (a NaN: fewer groups than beams)
        unsigned mask = 0;
#pragma unroll 4
        for (int g = 0; g < group; ++g) {
            mask |= static_cast<float>(group_max[warp][g][lane]) >= bound ? 1u << g : 0u;
        }
        int count = 0;
        bool overflow = false;
        while (!overflow && __any_sync(fb::kFullMask, mask != 0)) {
            const int g = __ffs(mask) - 1;
            mask &= mask - 1;
            for (int of = 0; of < of_group && !overflow; ++of) {
                const int at = (g * of_group + of) * kChunk + lane;
                uint4 q[kHeld];
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    q[j] = word_at(part, g >= 0 ? at + 32 * j : words);
                }
                if (__any_sync(fb::kFullMask, first + at + 32 * (kHeld - 1) >= all_words - 1)) {
#pragma unroll
                    for (int j = 0; j < kHeld; ++j) {
                        cut(q[j], at + 32 * j);
                    }
                }
                unsigned those = 0;      // of this lane's values, that reach the bound
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    those |= R::reaching(q[j], bound) << (j * R::kValues);
                }
                while (!overflow && __any_sync(fb::kFullMask, those != 0)) {
                    const int k = __ffs(those) - 1;
                    const int column = (first + at + 32 * (k / R::kValues)) * R::kValues + k % R::kValues;
                    const float v = k >= 0 ? R::value(part.values, column) : -INFINITY;
                    const bool reaches = k >= 0 && v >= bound;      // (which may have risen)
                    const unsigned lanes = __ballot_sync(fb::kFullMask, reaches);
                    those &= those - 1;
                    if (reaches) {
                        list[count + __popc(lanes & ((1u << lane) - 1))] = order_key(v, column);
                    }
                    count += __popc(lanes);
                    if (count > kMany) {
                        __syncwarp();
                        count = keep_largest(list, count, p.beams, bound, lane, false);
                        overflow = count > kMany;      // many equal ones
                    }
                }
            }
        }
        if (overflow) {
            __syncwarp();
            count = among_equals<T>(list, from, words, first * R::kValues, p.vocab, p.beams, bound, lane);
        }
        __syncwarp();
        Key* best = p.best + static_cast<size_t>(part.item) * p.beams;
        for (int c = lane; c < count; c += 32) {
            const Key key = list[c];
            int larger = 0;
#pragma unroll 4
            for (int other = 0; other < count; ++other) {
                larger += list[other] > key ? 1 : 0;
            }
            if (larger < p.beams) {
                best[larger] = key;
            }
        }
        for (int c = count + lane; c < p.beams; c += 32) {
            best[c] = 0;
        }
        __syncwarp();      // (the list is read)
        part = next;
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

// length^power. Whole powers by products, which are exact up to 2^53: equal quotients of totals are equal numbers then.
__device__ __forceinline__ double power_of(double length, float power) {
    if (power != rintf(power)) {
        return pow(length, static_cast<double>(power));
    }
    double product = 1.0;
    for (int rest = static_cast<int>(power); rest != 0; rest >>= 1, length *= length) {
        product *= (rest & 1) != 0 ? length : 1.0;
    }
    return product;
}

constexpr int kBins = 64;
constexpr int kMostEntries = 4096;   // of a group's lists

// The bound leaves entries of at most `beams` bins, each with those of its threads.
__host__ __device__ constexpr int most_left(int entries, int beams, int threads) {
    return beams * (threads / kBins) * ((entries + threads - 1) / threads);
}

struct Candidate {
    Key rank;
    unsigned place;      // beam, token
    __device__ __forceinline__ bool above(const Candidate& other) const {
        return rank > other.rank || (rank == other.rank && place < other.place);
    }
};

// What is known of a group's beams.
struct Beams {
    // A row's log-sum-exp is top + log_sum, which stay apart: of the lowest FP32 number as the largest logit their sum would be the former.
    double score[kMostBeams], top[kMostBeams], log_sum[kMostBeams], divisor[kMostBeams];     // divisor: length^power
    int over[kMostBeams], length[kMostBeams];
};

// Histories of a warp's new beams, kBeams of them at a time. (Loads first: to the compiler a store may change what is
// loaded next, and each would wait for the one before.)
template <int kWarps, int kBeams, int kAtOnce>
__device__ __forceinline__ void copy_histories(const GroupArgs& p, long long first, const Beams& of,
                                               const unsigned (&chosen)[kMostBeams], int warp, int lane) {
    for (int t0 = warp; t0 < p.beams; t0 += kBeams * kWarps) {
        const uint16_t* from[kBeams];
        int lengths[kBeams], longest = 0;
#pragma unroll
        for (int b = 0; b < kBeams; ++b) {
            const int t = t0 + b * kWarps;
            const int parent = t >= p.beams ? 0 : chosen[t] == ~0u ? t : static_cast<int>(chosen[t] >> 16);
            from[b] = p.histories + (first + parent) * p.history_stride;
            lengths[b] = t < p.beams ? of.length[parent] : 0;
            longest = max(longest, lengths[b]);
        }
        for (int c = lane; c < longest; c += 32 * kAtOnce) {
            uint16_t some[kBeams][kAtOnce];
#pragma unroll
            for (int b = 0; b < kBeams; ++b) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    some[b][i] = c + 32 * i < lengths[b] ? from[b][c + 32 * i] : 0;
                }
            }
#pragma unroll
            for (int b = 0; b < kBeams; ++b) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (c + 32 * i < lengths[b]) {
                        p.next_histories[(first + t0 + b * kWarps) * p.history_stride + c + 32 * i] = some[b][i];
                    }
                }
            }
        }
    }
}

// kHeldEntries: of a group's lists, per thread.
// (Blocks of 128 threads for few entries: 1,000 groups of 5 beams are on the GPU at once then, 11 us where 256 threads take 13.6.)
template <int kThreads, int kHeldEntries>
__global__ void __launch_bounds__(kThreads, kHeldEntries > 4 ? 2 : 1280 / kThreads) fb_beam_groups(const GroupArgs p) {
    constexpr int kWarps = kThreads / 32;
    extern __shared__ __align__(16) unsigned char left_memory[];
    __shared__ Beams of;
    __shared__ float2 stats[kMostLists];
    __shared__ Candidate bins[kBins];
    __shared__ Candidate bound;
    __shared__ int left_count;
    __shared__ unsigned chosen[kMostBeams];
    __shared__ double chosen_total[kMostBeams];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    fb::dependency_wait();
    fb::dependency_release();
    const long long first = static_cast<long long>(blockIdx.x) * p.beams;
    const int lists = p.beams * p.parts, entries = lists * p.beams, of_beam = p.parts * p.beams;
    const int most = most_left(entries, p.beams, kThreads);
    Key* left_rank = reinterpret_cast<Key*>(left_memory);
    double* left_total = reinterpret_cast<double*>(left_rank + most);
    unsigned* left_place = reinterpret_cast<unsigned*>(left_total + most);
    const Key* keys = p.best + first * p.parts * p.beams;
    Key held[kHeldEntries];       // this thread's first entries
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
        held[i] = tid + i * kThreads < entries ? keys[tid + i * kThreads] : 0;
    }
    for (int i = tid; i < lists; i += kThreads) {
        stats[i] = p.stats[first * p.parts + i];
    }
    // A warp takes the beams' lengths while others wait for statistics.
    if (warp == kWarps - 1 && lane < p.beams) {
        const int over = p.finished != nullptr && p.finished[first + lane] != 0 ? 1 : 0;
        int length = p.lengths != nullptr ? p.lengths[first + lane] : 0;
        const int most = p.histories != nullptr ? static_cast<int>(p.history_stride) : INT_MAX - 1;
        if (length < 0 || length > most) {
            atomicExch(&g_beams_error, 1);
            length = min(max(length, 0), most);
        }
        const float score = p.scores[first + lane];
        of.over[lane] = over;
        of.length[lane] = length;
        of.score[lane] = fabsf(score) < INFINITY ? static_cast<double>(score) : -INFINITY;
        chosen[lane] = ~0u;
    }
    if (tid == 0) {
        left_count = 0;
        bound = Candidate{1, ~0u};      // anything that is a continuation
    }
    __syncthreads();
    // Four lanes take a beam's log-sum-exp, and a warp the powers of lengths meanwhile. (FP64 throughout: powers that were off by
    // FP32's roundings would move totals past each other.)
    constexpr int kLanes = 4;
    const int beam = tid / kLanes;
    if (warp == kWarps - 1) {
        if (lane < p.beams) {
            const double grown = of.over[lane] != 0 ? max(of.length[lane], 1) : static_cast<double>(of.length[lane]) + 1.0;
            of.divisor[lane] = power_of(grown, p.power);
        }
    } else if (warp * (32 / kLanes) < p.beams) {
        float m = kLowest, sum = 0.0f;
        const int its = min(beam, p.beams - 1) * p.parts;
        for (int i = tid % kLanes; i < p.parts; i += kLanes) {
            m = max_nan(m, stats[its + i].x);
        }
        m = max_nan(m, __shfl_xor_sync(fb::kFullMask, m, 1));
        m = max_nan(m, __shfl_xor_sync(fb::kFullMask, m, 2));
        for (int i = tid % kLanes; i < p.parts; i += kLanes) {
            const float2 part = stats[its + i];
            sum += part.y * expf(part.x - m);
        }
        sum += __shfl_xor_sync(fb::kFullMask, sum, 1);
        sum += __shfl_xor_sync(fb::kFullMask, sum, 2);
        if (tid % kLanes == 0 && beam < p.beams) {
            of.top[beam] = static_cast<double>(m);
            of.log_sum[beam] = log(static_cast<double>(sum));
        }
    }
    __syncthreads();
    // Entry i, of beam i / of_beam: its total, and its place.
    auto total_of = [&](int i, Key key, unsigned& place) {
        const int its = static_cast<int>(static_cast<unsigned>(i) / static_cast<unsigned>(of_beam));
        const unsigned high = static_cast<unsigned>(its) << 16;
        if (of.over[its] != 0) {
            // (A finished beam's row was not read; it has one continuation.)
            place = high | static_cast<unsigned>(max(p.end_token, 0));
            return i == its * of_beam ? of.score[its] : -INFINITY;
        }
        place = high | static_cast<unsigned>(key_column(key) & 0xffff);
        // (A sum that is not a number gives none, nor does one of 0.)
        const double total = key != 0 ? of.score[its] + (static_cast<double>(key_value(key)) - of.top[its] - of.log_sum[its]) : -INFINITY;
        return total < INFINITY ? total : -INFINITY;
    };
    // (A reciprocal in the quotient's place would be rounded once more, and equal quotients not be equal.)
    auto rank_of = [&](double total, unsigned place) {
        return order_total(p.power == 0.0f ? total : total / of.divisor[place >> 16]);
    };
    Candidate top = {0, ~0u};
    Key ranks[kHeldEntries];
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
        ranks[i] = 0;
        if (tid + i * kThreads < entries) {
            unsigned place;
            const double total = total_of(tid + i * kThreads, held[i], place);
            const Candidate mine = {rank_of(total, place), place};
            ranks[i] = mine.rank;
            top = mine.above(top) ? mine : top;
        }
    }
    const Candidate own_top = top;
#pragma unroll
    for (int off = 1; off < kThreads / kBins; off <<= 1) {
        const Candidate other = {__shfl_xor_sync(fb::kFullMask, top.rank, off), __shfl_xor_sync(fb::kFullMask, top.place, off)};
        top = other.above(top) ? other : top;
    }
    if (tid % (kThreads / kBins) == 0) {
        bins[tid / (kThreads / kBins)] = top;
    }
    __syncthreads();
    // The beams-th largest of the bins' tops: a warp ranks its share of the bins.
    const Candidate low = bins[lane], high = bins[lane + 32];
#pragma unroll
    for (int i = 0; i < kBins / kWarps; ++i) {
        const Candidate bin = bins[warp * (kBins / kWarps) + i];
        const int larger = __popc(__ballot_sync(fb::kFullMask, low.above(bin))) + __popc(__ballot_sync(fb::kFullMask, high.above(bin)));
        if (larger == p.beams - 1 && bin.rank != 0 && lane == 0) {
            bound = bin;
        }
    }
    __syncthreads();
    if (own_top.rank != 0 && !bound.above(own_top)) {
#pragma unroll
        for (int i = 0; i < kHeldEntries; ++i) {
            if (ranks[i] != 0 && ranks[i] >= bound.rank) {
                unsigned place;
                const double total = total_of(tid + i * kThreads, held[i], place);
                const Candidate mine = {ranks[i], place};
                if (!bound.above(mine)) {
                    const int at = atomicAdd(&left_count, 1);
                    left_rank[at] = mine.rank;
                    left_place[at] = mine.place;
                    left_total[at] = total;
                }
            }
        }
    }
    __syncthreads();
    const int count = left_count;
    for (int i = tid / kLanes; i < count; i += kThreads / kLanes) {
        const Candidate its = {left_rank[i], left_place[i]};
        int larger = 0;
#pragma unroll 4
        for (int other = tid % kLanes; other < count; other += kLanes) {
            larger += Candidate{left_rank[other], left_place[other]}.above(its) ? 1 : 0;
        }
        const unsigned four = 0xfu << (lane / kLanes * kLanes);
        larger += __shfl_xor_sync(four, larger, 1);
        larger += __shfl_xor_sync(four, larger, 2);
        if (larger < p.beams && tid % kLanes == 0) {
            chosen[larger] = its.place;
            chosen_total[larger] = left_total[i];
        }
    }
    __syncthreads();
    // The new beams, a warp each in turn: their histories, and their numbers.
    if (p.next_histories != nullptr) {
        if (p.beams <= kWarps) {
            copy_histories<kWarps, 1, 16>(p, first, of, chosen, warp, lane);
        } else {
            copy_histories<kWarps, 4, 4>(p, first, of, chosen, warp, lane);
        }
    }
    if (tid < p.beams) {
        const int t = tid;
        const bool none = chosen[t] == ~0u;
        const int parent = none ? t : static_cast<int>(chosen[t] >> 16);
        const bool over = of.over[parent] != 0;
        const int token = none ? (over ? max(p.end_token, 0) : 0) : static_cast<int>(chosen[t] & 0xffffu);
        int length = of.length[parent];
        const long long row = first + t;
        if (!over && p.next_histories != nullptr) {
            if (length == p.history_stride) {
                atomicExch(&g_beams_error, 1);
                --length;      // (stays as long as it is, and keeps its last token)
            } else {
                p.next_histories[row * p.history_stride + length] = static_cast<uint16_t>(token);
            }
        }
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

// Parts of a row: those with which the warps are done soonest, each part costing three chunks more than it has; never so many that
// a group has more than kMostLists or kMostEntries, or the GPU more than kMostRounds parts per warp on their account.
constexpr int kMostRounds = 8;
unsigned warps_of(const Form& form, int sms) { return static_cast<unsigned>(sms * form.blocks * kWarps); }

int parts_of(const Form& form, int words, size_t rows, int beams, int sms) {
    const unsigned warps = warps_of(form, sms), chunk = static_cast<unsigned>(form.chunk);
    const size_t most = std::min<size_t>(std::min(kMostLists / beams, kMostEntries / (beams * beams)),
                                         kMostRounds * static_cast<size_t>(warps) / std::max<size_t>(rows, 1));
    unsigned best = 1;
    float least = 0.0f;
    for (unsigned parts = 1; parts == 1 || (parts <= most && words / parts >= 32); ++parts) {
        // (A block's warps are done about a part apart: 5,000 rows 102.6 us so, 106.1 with half a part.)
        const float items = static_cast<float>(rows) * parts / static_cast<float>(warps);
        const unsigned chunks = ((words + parts - 1) / parts + chunk - 1) / chunk;
        const float cost = (items <= 1.0f ? 1.0f : items + 1.0f) * static_cast<float>(chunks + 3);
        if (parts == 1 || cost < least) {
            best = parts;
            least = cost;
        }
    }
    return static_cast<int>(best);
}
size_t most_lists(size_t rows, int sms) { return rows + kMostRounds * static_cast<size_t>(warps_of(form_of(8), sms)); }

size_t stats_bytes(size_t lists) { return (lists * sizeof(float2) + 255) / 256 * 256; }

template <typename T>
cudaError_t launch_rows(RowArgs p, size_t rows, int sms, cudaStream_t stream) {
    const int words = (p.vocab + Row<T>::kValues - 1) / Row<T>::kValues;
    p.slice = (words + p.parts - 1) / p.parts;
    p.items = static_cast<unsigned>(rows * p.parts);
    const size_t blocks = std::min<size_t>(p.items, static_cast<size_t>(form_of(Row<T>::kValues).blocks) * sms);
    return fb::launch_dependent(fb_beam_rows<T>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, p);
}

template <int kThreads, int kHeldEntries>
cudaError_t launch_groups(const GroupArgs& g, size_t groups, int entries, cudaStream_t stream) {
    constexpr size_t kEach = sizeof(Key) + sizeof(double) + sizeof(unsigned);
    constexpr int kMostSmem = static_cast<int>(most_left(kThreads * kHeldEntries, kMostBeams, kThreads) * kEach);
    static std::atomic<bool> configured[64] = {};
    const auto kernel = fb_beam_groups<kThreads, kHeldEntries>;
    const cudaError_t e = fb::allow_shared_memory(kernel, kMostSmem, configured);
    return e != cudaSuccess ? e
                            : fb::launch_dependent(kernel, dim3(static_cast<unsigned>(groups)), dim3(kThreads),
                                                   most_left(entries, g.beams, kThreads) * kEach, stream, g);
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
    if (!(length_power >= 0.0f && length_power <= kMostPower)) {
        return fb::fail(kBad, "%s: length_power (%g) must be from 0 to %g", name, static_cast<double>(length_power),
                        static_cast<double>(kMostPower));
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
    g.parts = p.parts = parts_of(form_of(values), (p.vocab + values - 1) / values, rows, p.beams, sms);
    g.end_token = end_token;
    g.power = length_power;
    FB_CUDA(fp32_logits != 0 ? launch_rows<float>(p, rows, sms, stream) : launch_rows<__half>(p, rows, sms, stream));
    const int entries = p.parts * p.beams * p.beams;
    FB_CUDA(entries <= 256    ? (launch_groups<128, 2>(g, groups, entries, stream))
            : entries <= 512  ? (launch_groups<256, 2>(g, groups, entries, stream))
            : entries <= 1024 ? (launch_groups<256, 4>(g, groups, entries, stream))
                              : (launch_groups<256, kMostEntries / 256>(g, groups, entries, stream)));
    return FLINT_OK;
}

}  // extern "C"
