// How a CTA of the attention kernels for sequences of different lengths finds its part of the batch
// (packed_schedule.h): the place of its two cuts on the line of key tiles, or that tiles are dealt out whole. P is a
// kernel's parameters: `a` (PackedArgs), `log_tokens` and `splits` (tiles may be split between CTAs).
#pragma once

#include "device_utils.cuh"
#include "packed.cuh"

namespace fb {
namespace {

constexpr int kLeastPart = 4;   // of the line of key tiles, per CTA
constexpr int kSplitCost = 6;      // about what splits and their join cost, in key tiles
constexpr int kMostDealt = 128;    // sequences whose tiles can be dealt out

struct SequenceOf {
    const PackedArgs& a;
    __device__ __forceinline__ Sequence operator()(int s) const { return sequence_at(a, s); }
};

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        v += __shfl_xor_sync(kFullMask, v, off);
    }
    return v;
}
__device__ __forceinline__ long long warp_prefix(long long v, int lane) {     // inclusive
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long other = __shfl_up_sync(kFullMask, v, off);
        v += lane >= off ? other : 0;
    }
    return v;
}

// The place of one of this CTA's two cuts (0 its part's beginning, 1 its end; both the line's end for a CTA without a
// part), and how far it may move.
struct Place {
    long long at, tolerance;
    template <typename P>
    __device__ __forceinline__ Place(const P& p, long long total, int which) {
        const int parts = part_count(total, static_cast<int>(gridDim.x), kLeastPart);
        const int cta = static_cast<int>(blockIdx.x);
        at = cta < parts ? cut_place(total, parts, cta + which) : total;
        tolerance = cta >= parts ? 0 : p.splits ? cut_tolerance(total, parts) : total;
    }
};

template <typename P>
__device__ __forceinline__ long long length_of(const P& p, int s, int& before, int& tokens) {
    before = tokens = 0;
    if (s >= p.a.sequences) {
        return 0;
    }
    const Sequence q = sequence_at(p.a, s);
    before = q.before();
    tokens = q.count;
    return head_length(before, tokens, p.log_tokens);
}

template <typename P>
__device__ __forceinline__ int most_key_tiles(const P& p, int before, int tokens) {
    return tokens == 0 ? 0 : key_tiles(before, tokens, p.log_tokens, tile_count(tokens, p.log_tokens) - 1);
}

// Whether tiles stay whole and are dealt out: none has more key tiles than a part of the line is long and splits cost.
// The longest CTA then works on 14 key tiles and ends instead of 17 (24 sequences of up to 700 tokens, 12 heads:
// 32.4 -> 27.3 us with the join, which finds nothing to do; 16 of up to 1,024: 29.4 -> 21.8; 5 of up to 4,096: 82 -> 73).
// Tiles longer than a part: 6 more key tiles 24.1 -> 20.6, 28.7 -> 24.9 and 21.7 -> 21.0 us (three batches), 9 more 20.2 ->
// 21.0 and 22.8 -> 25.1, 11 more 24.0 -> 29.5.
template <typename P>
__device__ __forceinline__ bool deals_out(const P& p, long long total, int longest) {
    return p.a.sequences <= kMostDealt && total < 1LL << 30 &&
           (!p.splits || longest <= (static_cast<int>(total) - 1) / static_cast<int>(gridDim.x) + 1 + kSplitCost);
}

// Tiles dealt out whole. One warp, lane l with the sequences l, l + 32, ...
struct Dealt {
    static constexpr int kEach = kMostDealt / 32;
    Sequence of[kEach];
    int each = 1;
    int count = 0;        // tiles
    int longest = 0;      // key tiles of the next one at most
    int round = 0;

    template <typename P>
    __device__ __forceinline__ void load(const P& p, int lane) {
        each = (p.a.sequences + 31) / 32;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            of[i] = Sequence{0, 0, 0};
            if (lane + 32 * i < p.a.sequences) {
                of[i] = sequence_at(p.a, lane + 32 * i);
            }
        }
    }
    template <typename P>
    __device__ __forceinline__ int of_lane(const P& p, int least) const {
        int those = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i < each) {
                those += tiles_of_at_least(of[i].before(), of[i].count, p.log_tokens, least);
            }
        }
        return those;
    }
    template <typename P>
    __device__ __forceinline__ int at_least(const P& p, int least) const {
        return __reduce_add_sync(kFullMask, of_lane(p, least)) * p.a.kv_heads;
    }
    template <typename P>
    __device__ __forceinline__ void begin(const P& p, int most) {
        longest = most;
        count = at_least(p, 1);
    }
    // The next tile of this CTA, if there is one.
    template <typename P>
    __device__ __forceinline__ bool next(const P& p, int lane, Piece& out) {
        const long long rank = dealt_rank(round, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
        ++round;
        if (rank >= count) {
            return false;
        }
        int low = 1;      // the most key tiles that more than `rank` tiles have
        while (low < longest) {
            const int middle = low + (longest - low + 1) / 2;
            if (at_least(p, middle) > rank) {
                low = middle;
            } else {
                longest = middle - 1;
            }
        }
        // Among those of as many key tiles: by lane, the lane's sequences, heads, tiles.
        const int more = of_lane(p, low + 1);
        const int mine = (of_lane(p, low) - more) * p.a.kv_heads;
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int other = __shfl_up_sync(kFullMask, upto, off);
            upto += lane >= off ? other : 0;
        }
        int at = static_cast<int>(rank) - __reduce_add_sync(kFullMask, more) * p.a.kv_heads - (upto - mine);
        const int owner = __ffs(__ballot_sync(kFullMask, at >= 0 && at < mine)) - 1;
        Sequence q = of[0];
        int s = lane;
#pragma unroll
        for (int i = 0; i + 1 < kEach; ++i) {
            if (s == lane + 32 * i && i + 1 < each) {
                const int those = (tiles_of_at_least(q.before(), q.count, p.log_tokens, low) -
                                   tiles_of_at_least(q.before(), q.count, p.log_tokens, low + 1)) * p.a.kv_heads;
                if (at >= those) {
                    at -= those;
                    q = of[i + 1];
                    s += 32;
                }
            }
        }
        at = __shfl_sync(kFullMask, at, owner);
        out.index = __shfl_sync(kFullMask, s, owner);
        out.sequence.first = __shfl_sync(kFullMask, q.first, owner);
        out.sequence.count = __shfl_sync(kFullMask, q.count, owner);
        out.sequence.keys = __shfl_sync(kFullMask, q.keys, owner);
        const int of_low = tiles_of_at_least(out.sequence.before(), out.sequence.count, p.log_tokens, low);
        const int these = of_low - tiles_of_at_least(out.sequence.before(), out.sequence.count, p.log_tokens, low + 1);
        out.head = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(these));
        out.first_token = (tile_count(out.sequence.count, p.log_tokens) - of_low + at - out.head * these) << p.log_tokens;
        out.tokens = min(out.sequence.count - out.first_token, 1 << p.log_tokens);
        out.from = 0;
        out.to = out.tiles = low;
        return true;
    }
};

// Which part of the line this CTA works on, for up to 32 sequences: one warp, its even lanes for one cut and the odd
// ones for the other.
template <bool kDeals, typename P>
__device__ __forceinline__ void locate_in_warp(const P& p, Cut (&cuts)[2], int& whole, int lane) {
    int before, tokens;
    const long long length = length_of(p, lane, before, tokens);
    const long long mine = length * p.a.kv_heads;
    const long long upto = warp_prefix(mine, lane);
    const long long total = __shfl_sync(kFullMask, upto, 31);
    if constexpr (kDeals) {
        const int longest = __reduce_max_sync(kFullMask, most_key_tiles(p, before, tokens));
        const bool deals = deals_out(p, total, longest);
        if (lane == 0) {
            whole = deals ? longest : 0;
        }
        if (deals) {
            if (lane < 2) {
                cuts[lane] = Cut{total, p.a.sequences, 0, 0, 0};
            }
            return;
        }
    }
    const Place place(p, total, lane & 1);
    const long long begins = upto - mine;
    const long long first = __shfl_sync(kFullMask, place.at, 0), second = __shfl_sync(kFullMask, place.at, 1);
    const unsigned has_first = __ballot_sync(kFullMask, first >= begins && first < upto);
    const unsigned has_second = __ballot_sync(kFullMask, second >= begins && second < upto);
    const unsigned has = (lane & 1) == 0 ? has_first : has_second;
    const int owner = has != 0 ? __ffs(has) - 1 : 0;
    const int its_before = __shfl_sync(kFullMask, before, owner), its_tokens = __shfl_sync(kFullMask, tokens, owner);
    const long long its_length = __shfl_sync(kFullMask, length, owner), its_begin = __shfl_sync(kFullMask, begins, owner);
    if (lane < 2) {
        cuts[lane] = has == 0 ? Cut{total, p.a.sequences, 0, 0, 0}
                              : cut_at(place.at, place.at - its_begin, owner, its_before, its_tokens, p.log_tokens,
                                       its_length, place.tolerance);
    }
}

// The same for up to 32 kEach sequences, lane l having a run of them, where tiles are not dealt out.
template <int kEach, typename P>
__device__ __forceinline__ void locate_runs_in_warp(const P& p, Cut (&cuts)[2], int lane) {
    const int each = (p.a.sequences + 31) / 32;
    int before[kEach], tokens[kEach];
    long long length[kEach], mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        length[i] = length_of(p, i < each ? lane * each + i : p.a.sequences, before[i], tokens[i]);
        mine += length[i] * p.a.kv_heads;
    }
    const long long upto = warp_prefix(mine, lane);
    const long long total = __shfl_sync(kFullMask, upto, 31);
    const Place place(p, total, lane & 1);
    int owner[2], its_sequence[2], its_before[2], its_tokens[2];
    long long its_length[2], its_begin[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const long long at = __shfl_sync(kFullMask, place.at, c);
        const unsigned has = __ballot_sync(kFullMask, at >= upto - mine && at < upto);
        owner[c] = has != 0 ? __ffs(has) - 1 : -1;
        // This lane's sequence that it would be.
        long long begin = upto - mine;
        int k = 0;
        its_before[c] = before[0];
        its_tokens[c] = tokens[0];
        its_length[c] = length[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) {
            const long long next = begin + length[i - 1] * p.a.kv_heads;
            if (k == i - 1 && at >= next) {
                k = i;
                begin = next;
                its_before[c] = before[i];
                its_tokens[c] = tokens[i];
                its_length[c] = length[i];
            }
        }
        const int from = max(owner[c], 0);
        its_sequence[c] = __shfl_sync(kFullMask, lane * each + k, from);
        its_before[c] = __shfl_sync(kFullMask, its_before[c], from);
        its_tokens[c] = __shfl_sync(kFullMask, its_tokens[c], from);
        its_length[c] = __shfl_sync(kFullMask, its_length[c], from);
        its_begin[c] = __shfl_sync(kFullMask, begin, from);
    }
    if (lane < 2) {
        const bool second = lane == 1;
        cuts[lane] = (second ? owner[1] : owner[0]) < 0
                         ? Cut{total, p.a.sequences, 0, 0, 0}
                         : cut_at(place.at, place.at - (second ? its_begin[1] : its_begin[0]), second ? its_sequence[1] : its_sequence[0],
                                  second ? its_before[1] : its_before[0], second ? its_tokens[1] : its_tokens[0], p.log_tokens,
                                  second ? its_length[1] : its_length[0], place.tolerance);
    }
}

// The same for any number: every thread of the block takes part.
template <bool kDeals, int kThreads, typename P>
__device__ __noinline__ void locate(const P& p, Cut (&cuts)[2], int& whole, long long (&scan)[kThreads / 32 + 1],
                                    int (&scan_longest)[kThreads / 32]) {
    constexpr int kWarps = kThreads / 32;
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    int before = 0, tokens = 0;
    long long sum = 0;
    int longest = 0;
    for (int s = tid; s < p.a.sequences; s += kThreads) {
        sum += length_of(p, s, before, tokens);
        longest = kDeals ? max(longest, most_key_tiles(p, before, tokens)) : 0;
    }
    sum = warp_sum(sum);
    longest = __reduce_max_sync(kFullMask, longest);
    if (lane == 0) {
        scan[warp] = sum;
        scan_longest[warp] = longest;
    }
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < kWarps; ++w) {
        total += scan[w];
        longest = max(longest, scan_longest[w]);
    }
    total *= p.a.kv_heads;
    if constexpr (kDeals) {
        const bool deals = deals_out(p, total, longest);
        if (tid == 0) {
            whole = deals ? longest : 0;
        }
        if (deals) {
            if (tid < 2) {
                cuts[tid] = Cut{total, p.a.sequences, 0, 0, 0};
            }
            return;
        }
    }
    const Place place[2] = {Place(p, total, 0), Place(p, total, 1)};
    if (tid < 2 && place[tid].at == total) {
        cuts[tid] = Cut{total, p.a.sequences, 0, 0, 0};
    }
    long long running = 0;
    for (int first = 0; first < p.a.sequences; first += kThreads) {
        const long long length = length_of(p, first + tid, before, tokens);
        const long long mine = length * p.a.kv_heads;
        long long upto = warp_prefix(mine, lane);
        __syncthreads();
        if (lane == 31) {
            scan[warp] = upto;
        }
        __syncthreads();
        long long all = 0;
        for (int w = 0; w < kWarps; ++w) {
            upto += w < warp ? scan[w] : 0;
            all += scan[w];
        }
        const long long begins = running + upto - mine;
        for (int c = 0; c < 2; ++c) {
            if (place[c].at >= begins && place[c].at < begins + mine) {
                cuts[c] = cut_at(place[c].at, place[c].at - begins, first + tid, before, tokens, p.log_tokens, length,
                                 place[c].tolerance);
            }
        }
        running += all;
    }
}

}  // namespace
}  // namespace fb
