// Causal attention over sequences of different lengths, packed or in the pages of a cache, on the
// 5th-generation tensor cores (head width 64).
//
// A tile is the 128 rows of (token, query head) that one K/V head's group makes of 128 / group
// consecutive tokens (rounded down to a power of two): one load of keys and values serves the whole
// group. S = Q K^T goes to tensor memory, two threads take the softmax of a row in base 2, P goes
// back as FP16 pairs and is the A operand of O += P V, which accumulates in tensor memory over the
// row of key tiles; the exponent that probabilities are taken against moves only when a row's
// maximum exceeds it by more than 2^8, so that O is rarely rescaled.
// The batch is shared out evenly however ragged it is (packed_schedule.h): whole tiles, sorted by their length and dealt
// out, or where a tile is too long for that a line of tiles cut into equal parts; a tile split between CTAs
// leaves its parts (O before the division, row maxima and sums, FP32) in the workspace, and a second,
// dependent launch joins them in the order of the keys.
//
// Two CTAs per SM with one tile each: one's matrix products, loads and ends run under the other's
// exponentials. Those bound long sequences: 128 x 128 of them take the SM's special-function unit 1,024 clocks
// and the products 512; a quarter of them runs on the FMA pipe instead (half of them: 10 % slower, none: 9 %). A key tile
// takes 1,350 clocks of an SM; short sequences are bound by what a tile's beginning and end cost, about two key tiles.
// Measured, with the join: 5 sequences of up to 4,096 tokens, 16 query heads on 4, 73 us (570 TFLOP/s); 24 of up to 700,
// 12 heads, 28.7 us; 64 single tokens on caches of up to 8,192, 32 heads on 8, 77 us (5.1 TB/s).
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>

#include <cuda.h>
#include <cuda_fp16.h>

#include "common.h"
#include "device_utils.cuh"
#include "packed.cuh"
#include "packed_maps.h"
#include "sm100.cuh"
#include "softmax.cuh"

namespace fb {
namespace {

constexpr int kRows = 128;      // (token, head) rows of a tile
constexpr int kHead = 64;
constexpr int kTileBytes = 128 * kHead * 2;   // Q, K or V: 16 KB
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

constexpr int kThreads = 320;   // TMA warp, MMA warp, eight softmax warps with two threads per row
constexpr int kWarps = kThreads / 32;
constexpr int kSlots = 4;       // ring of K and V tiles
constexpr int kSoftmaxWarps = 8;
constexpr int kStaging = 1024;     // bytes per softmax warp
constexpr int kStagingBytes = kSoftmaxWarps * kStaging;
constexpr int kPieces = 8;      // ring of piece descriptions
constexpr int kSmem = 1024 + (2 + kSlots) * kTileBytes + kStagingBytes + 256;
constexpr int kLeastPart = 4;   // of the line of key tiles, per CTA
constexpr int kWholeKeys = 1024;   // up to which a tile is never split
constexpr int kSplitCost = 6;      // about what splits and their join cost, in key tiles
constexpr int kMostDealt = 128;    // sequences whose tiles can be dealt out

constexpr size_t kPartFloats = size_t{kRows} * kHead + 2 * kRows;   // O [column / 4][row][4], maxima, sums

struct TileParams {
    CUtensorMap map_q, map_k, map_v;
    PackedArgs a;
    Record* records;    // [CTA]
    float* parts;       // [CTA][head part, tail part]
    int group, log_tokens;
    int boxes;          // loads per K or V tile
    int box_rows;
    bool splits;        // tiles may be split between CTAs
};

struct Barriers {
    uint32_t base;
    __device__ uint32_t q_full(int b) const { return base + 8u * b; }
    __device__ uint32_t q_empty(int b) const { return base + 16 + 8u * b; }
    __device__ uint32_t s_full() const { return base + 32; }
    __device__ uint32_t s_free() const { return base + 40; }
    __device__ uint32_t p_ready() const { return base + 48; }
    __device__ uint32_t pv_done() const { return base + 56; }
    __device__ uint32_t meeting() const { return base + 64; }
    __device__ uint32_t pair(int quadrant) const { return base + 72 + 8u * quadrant; }
    __device__ uint32_t piece_full(int i) const { return base + 104 + 8u * i; }
    __device__ uint32_t slot_full(int s) const { return base + 104 + 8u * (kPieces + s); }
    __device__ uint32_t slot_empty(int s) const { return base + 104 + 8u * (kPieces + kSlots + s); }
};

constexpr uint32_t kIdescS = sm100::instr_desc_f16(128, 128, false, false);
constexpr uint32_t kIdescPV = sm100::instr_desc_f16(128, 64, false, true);

// A NaN among the three gives NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

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
    __device__ __forceinline__ Place(const TileParams& p, long long total, int which) {
        const int parts = part_count(total, static_cast<int>(gridDim.x), kLeastPart);
        const int cta = static_cast<int>(blockIdx.x);
        at = cta < parts ? cut_place(total, parts, cta + which) : total;
        tolerance = cta >= parts ? 0 : p.splits ? cut_tolerance(total, parts) : total;
    }
};

__device__ __forceinline__ long long length_of(const TileParams& p, int s, int& before, int& tokens) {
    before = tokens = 0;
    if (s >= p.a.sequences) {
        return 0;
    }
    const Sequence q = sequence_at(p.a, s);
    before = q.before();
    tokens = q.count;
    return head_length(before, tokens, p.log_tokens);
}

__device__ __forceinline__ int most_key_tiles(const TileParams& p, int before, int tokens) {
    return tokens == 0 ? 0 : key_tiles(before, tokens, p.log_tokens, tile_count(tokens, p.log_tokens) - 1);
}

// Whether tiles stay whole and are dealt out: none has more key tiles than a part of the line is long and splits cost.
// The longest CTA then works on 14 key tiles and ends instead of 17 (24 sequences of up to 700 tokens, 12 heads:
// 32.4 -> 27.3 us with the join, which finds nothing to do; 16 of up to 1,024: 29.4 -> 21.8; 5 of up to 4,096: 82 -> 73).
// Tiles longer than a part: 6 more key tiles 24.1 -> 20.6, 28.7 -> 24.9 and 21.7 -> 21.0 us (three batches), 9 more 20.2 ->
// 21.0 and 22.8 -> 25.1, 11 more 24.0 -> 29.5.
__device__ __forceinline__ bool deals_out(const TileParams& p, long long total, int longest) {
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

    __device__ __forceinline__ void load(const TileParams& p, int lane) {
        each = (p.a.sequences + 31) / 32;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            of[i] = Sequence{0, 0, 0};
            if (lane + 32 * i < p.a.sequences) {
                of[i] = sequence_at(p.a, lane + 32 * i);
            }
        }
    }
    __device__ __forceinline__ int of_lane(const TileParams& p, int least) const {
        int those = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i < each) {
                those += tiles_of_at_least(of[i].before(), of[i].count, p.log_tokens, least);
            }
        }
        return those;
    }
    __device__ __forceinline__ int at_least(const TileParams& p, int least) const {
        return __reduce_add_sync(kFullMask, of_lane(p, least)) * p.a.kv_heads;
    }
    __device__ __forceinline__ void begin(const TileParams& p, int most) {
        longest = most;
        count = at_least(p, 1);
    }
    // The next tile of this CTA, if there is one.
    __device__ __forceinline__ bool next(const TileParams& p, int lane, Piece& out) {
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
template <bool kDeals>
__device__ __forceinline__ void locate_in_warp(const TileParams& p, Cut (&cuts)[2], int& whole, int lane) {
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

// The same for any number: every thread of the block takes part.
template <bool kDeals>
__device__ __noinline__ void locate(const TileParams& p, Cut (&cuts)[2], int& whole, long long (&scan)[kWarps + 1],
                                    int (&scan_longest)[kWarps]) {
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

// A piece as the TMA warp hands it to the others; `to` of 0 ends the list.
struct PieceInfo {
    int from, to, tiles;
    int position;      // of the tile's first token
    int tokens;        // in the tile
    int first_row;     // of its first token
    int head;          // K/V head
    int keys;          // of the sequence
};

// Softmax warps that share rows meet here (bounded, like every wait).
struct Meeting {
    uint32_t bar;
    uint32_t count;
    volatile int* abort;
    int lane;
    __device__ __forceinline__ bool meet() {
        __syncwarp();
        if (lane == 0) {
            sm100::mbar_arrive(bar);
        }
        return sm100::mbar_wait_warp(bar, count++ & 1, abort);
    }
};

// kSubsets > 1 (single tokens and few of them): a tile has 128 / kSubsets rows, which lie kSubsets times in the 128
// lanes, and each copy takes its share of a key tile's columns (its other probabilities are zeros, written once),
// with its own maxima and sums. A step's softmax then takes a kSubsets-th of the time, and all four warps
// work where one would; the copies are put together at the end of a piece.
template <bool kPaged, int kSubsets>
__global__ void __launch_bounds__(kThreads, 2) fb_packed_forward_tiles(const __grid_constant__ TileParams p) {
    // Few rows' tiles are not dealt out: finding one takes longer than what it gains (8 single tokens on up to 1,000 keys
    // 14.2 -> 15.2 us, 64 on up to 8,192 78 -> 82 us with the code alone).
    constexpr bool kDeals = kSubsets == 1;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_tiles = base;
    const uint32_t ring = base + 2 * kTileBytes;
    const uint32_t staging = ring + kSlots * kTileBytes;
    const Barriers bar{staging + kStagingBytes};
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ Cut cuts[2];
    __shared__ long long scan[kWarps + 1];
    __shared__ int scan_longest[kWarps];
    __shared__ int whole_tiles;      // the longest tile's key tiles where tiles are dealt out, else 0
    __shared__ PieceInfo pieces[kPieces];
    __shared__ float pair_max[2][2][kRows];           // [step parity][half of the columns][row]
    __shared__ float merge_max[4][32], merge_sum[kSoftmaxWarps][32];

    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x / 32), 0);
    const int lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int b = 0; b < 2; ++b) {
            sm100::mbar_init(bar.q_full(b), 1);
            sm100::mbar_init(bar.q_empty(b), 1);
        }
        sm100::mbar_init(bar.s_full(), 1);
        sm100::mbar_init(bar.s_free(), kSoftmaxWarps);     // one arrival per softmax warp
        sm100::mbar_init(bar.p_ready(), kSoftmaxWarps);
        sm100::mbar_init(bar.pv_done(), 1);
        sm100::mbar_init(bar.meeting(), kSoftmaxWarps);
        for (int q = 0; q < 4; ++q) {
            sm100::mbar_init(bar.pair(q), 2);
        }
        for (int i = 0; i < kPieces; ++i) {
            sm100::mbar_init(bar.piece_full(i), 1);
        }
        for (int s = 0; s < kSlots; ++s) {
            sm100::mbar_init(bar.slot_full(s), 1);
            sm100::mbar_init(bar.slot_empty(s), 1);
        }
        sm100::mbar_fence_init();
        sm100::tma_prefetch_descriptor(&p.map_q);
        sm100::tma_prefetch_descriptor(&p.map_k);
        sm100::tma_prefetch_descriptor(&p.map_v);
    }
    if (warp == 1) {
        sm100::tmem_alloc(sm100::smem_u32(&tmem_slot), 256);
    }
    dependency_wait();
    Dealt dealt;
    if (kDeals && warp == 0 && p.a.sequences <= kMostDealt) {
        dealt.load(p, lane);
    }
    if (p.a.sequences > 32) {
        locate<kDeals>(p, cuts, whole_tiles, scan, scan_longest);
    } else if (warp == 2) {
        locate_in_warp<kDeals>(p, cuts, whole_tiles, lane);
    }
    sm100::tc_fence_before_sync();
    __syncthreads();
    sm100::tc_fence_after_sync();
    if (threadIdx.x == 0) {
        dependency_release();    // (the join's blocks take the place of this kernel's as they end)
    }
    const uint32_t tmem_s = tmem_slot, tmem_o = tmem_slot + 128, tmem_p = tmem_slot + 192;
    volatile int* abort = &abort_flag;

    if (warp == 0) {
        Walk walk;
        Piece piece = {};
        walk.begin(SequenceOf{p.a}, cuts[0], cuts[1].at);
        int round = 0;
        const bool whole = kDeals && whole_tiles > 0;
        if (whole) {
            dealt.begin(p, whole_tiles);
        }
        bool fetch = true, more = false;     // whether the next piece is to be found, and whether there was one
        int j = 0;
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        // 32 of the sequence's page numbers, one per lane, and where each lane's part of the key tile at hand and of
        // the one before lies.
        int page_entries = 0, entries_from = -1, entries_of = -1;
        int at_now = 0, head_now = 0, at_before = 0, head_before = 0;
        auto find = [&]() {
            at_before = at_now;
            head_before = head_now;
            head_now = piece.head;
            if constexpr (kPaged) {
                const int first = j * kKeyTile / p.a.page_size;     // page of the tile's first key
                if (entries_of != piece.index || first < entries_from || first + p.boxes > entries_from + 32) {
                    const int index = first + lane;
                    entries_of = piece.index;
                    entries_from = first;
                    page_entries = -1;
                    if (index < (piece.sequence.keys + p.a.page_size - 1) / p.a.page_size) {
                        page_entries = static_cast<int>(page_of(p.a, piece.index, index * p.a.page_size));
                    }
                }
                const int box = min(lane, p.boxes - 1);
                const int page = __shfl_sync(kFullMask, page_entries, first - entries_from + box);
                // A page that is not there is read from outside the cache, as zeros.
                const int key = j * kKeyTile + box * p.box_rows;
                at_now = page < 0 || key >= piece.sequence.keys
                             ? static_cast<int>(p.a.pages * p.a.kv_heads * p.a.page_size)
                             : (page * p.a.kv_heads + piece.head) * p.a.page_size + (key & (p.a.page_size - 1));
            } else {
                at_now = piece.sequence.first + j * kKeyTile;
            }
        };
        auto load = [&](const CUtensorMap* map, int at, int head) {
            if (!sm100::mbar_wait_warp(bar.slot_empty(slot), phase ^ 1u, abort)) {
                ok = false;
                return;
            }
            const uint32_t full = bar.slot_full(slot), dst = ring + slot * kTileBytes;
            if (lane == 0) {
                sm100::mbar_expect_tx(full, kTileBytes);
            }
            __syncwarp();
            if constexpr (kPaged) {
                if (lane < p.boxes) {
                    sm100::tma_load_2d(dst + lane * p.box_rows * (kHead * 2), map, full, 0, at);
                }
            } else if (lane == 0) {
                sm100::tma_load_3d(dst, map, full, 0, head, at);
            }
            __syncwarp();
            if (++slot == kSlots) {
                slot = 0;
                phase ^= 1u;
            }
        };
        int waiting = 0;     // K tiles whose V tile has not been asked for
        while (ok) {
            if (fetch) {
                fetch = false;
                more = whole ? dealt.next(p, lane, piece)
                             : walk.next(SequenceOf{p.a}, p.a.sequences, p.a.kv_heads, p.log_tokens, piece);
                j = piece.from;
                if (!more && lane == 0) {
                    pieces[round % kPieces].to = 0;
                    sm100::mbar_arrive(bar.piece_full(round % kPieces));
                }
            }
            if (more) {
                if (j == piece.from) {
                    // A new piece. Its description's place was read long ago: the ring of tiles keeps this
                    // warp within a few steps, and so within fewer than kPieces pieces, of the softmax warps.
                    // Its queries go into the buffer of its parity, free once the piece two rounds
                    // back has issued its last scores.
                    const int b = round & 1;
                    if (round >= 2 && !sm100::mbar_wait_warp(bar.q_empty(b), ((round >> 1) - 1) & 1, abort)) {
                        break;
                    }
                    if (lane == 0) {
                        pieces[round % kPieces] = PieceInfo{piece.from, piece.to, piece.tiles, piece.position(),
                                                            piece.tokens, piece.sequence.first + piece.first_token,
                                                            piece.head, piece.sequence.keys};
                        sm100::mbar_arrive(bar.piece_full(round % kPieces));
                        sm100::mbar_expect_tx(bar.q_full(b), kSubsets * static_cast<uint32_t>(p.group << p.log_tokens) *
                                                                 (kHead * 2));
#pragma unroll
                        for (int copy = 0; copy < kSubsets; ++copy) {
                            sm100::tma_load_3d(q_tiles + b * kTileBytes + copy * (kTileBytes / kSubsets), &p.map_q,
                                               bar.q_full(b), 0, piece.head * p.group,
                                               piece.sequence.first + piece.first_token);
                        }
                    }
                    __syncwarp();
                }
                find();
                load(&p.map_k, at_now, head_now);
                ++waiting;
                if (++j == piece.to) {
                    ++round;
                    fetch = true;
                }
                if (waiting < 2) {
                    continue;
                }
                if (ok) {
                    load(&p.map_v, at_before, head_before);
                    --waiting;
                }
            } else {
                if (waiting > 0) {
                    load(&p.map_v, at_now, head_now);
                }
                break;
            }
        }
    } else if (warp == 1) {
        // The whole warp runs this loop, so that its state stays uniform; one elected lane issues.
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        auto next_tile = [&]() -> uint32_t {
            if (!sm100::mbar_wait_warp(bar.slot_full(slot), phase, abort)) {
                ok = false;
                return 0u;
            }
            sm100::tc_fence_after_sync();
            return ring + slot * kTileBytes;
        };
        auto step_ring = [&]() {
            if (++slot == kSlots) {
                slot = 0;
                phase ^= 1u;
            }
        };
        // Where the next scores to issue stand, and how far the piece goes.
        int round = 0, j = 0, to = 0, from = 0, keys = 0;
        auto enter = [&]() {
            if (!sm100::mbar_wait_warp(bar.piece_full(round % kPieces), (round / kPieces) & 1, abort)) {
                ok = false;
                to = 0;
                return;
            }
            const PieceInfo& info = pieces[round % kPieces];
            from = j = info.from;
            to = info.to;
            keys = info.keys;
        };
        bool at_end = true;      // of a piece: the next one's description comes first
        uint32_t issued = 0;
        // Of the step whose scores were issued last: whether its piece begins with it, and the keys in its tile.
        bool begins_ahead = false;
        int present_ahead = 0;
        auto issue_scores = [&]() {
            if (ok && at_end) {
                enter();
                at_end = false;
            }
            if (!ok || to == 0) {
                return;
            }
            const int b = round & 1;
            if (j == from && !sm100::mbar_wait_warp(bar.q_full(b), (round >> 1) & 1, abort)) {
                ok = false;
                return;
            }
            const uint32_t k_tile = next_tile();
            if (k_tile == 0) {
                return;
            }
            if (issued > 0 && !sm100::mbar_wait_warp(bar.s_free(), (issued - 1) & 1, abort)) {
                ok = false;
                return;
            }
            sm100::tc_fence_after_sync();
            const uint64_t q_desc = desc_kmajor(q_tiles + b * kTileBytes, 0);
            const uint64_t k_desc = desc_kmajor(k_tile, 0);
            const bool last = j + 1 == to;
            if (sm100::elect_one()) {
                sm100::mma_f16_ss_at<0>(tmem_s, q_desc, 0, k_desc, 0, kIdescS);
                sm100::mma_f16_ss_at<1>(tmem_s, q_desc, 2, k_desc, 2, kIdescS);
                sm100::mma_f16_ss_at<1>(tmem_s, q_desc, 4, k_desc, 4, kIdescS);
                sm100::mma_f16_ss_at<1>(tmem_s, q_desc, 6, k_desc, 6, kIdescS);
                sm100::mma_commit(bar.s_full());
                sm100::mma_commit(bar.slot_empty(slot));
                if (last) {
                    sm100::mma_commit(bar.q_empty(b));
                }
            }
            __syncwarp();
            step_ring();
            ++issued;
            begins_ahead = j == from;
            present_ahead = keys - j * kKeyTile;
            ++j;
            if (last) {
                ++round;
                at_end = true;
            }
        };
        issue_scores();
        for (uint32_t n = 0; ok && n < issued; ++n) {
            const bool begins = begins_ahead;
            const int present = present_ahead;
            issue_scores();    // of the next step, as soon as this step's have been read
            const uint32_t v_tile = ok ? next_tile() : 0u;
            if (v_tile == 0) {
                break;
            }
            if (present < kKeyTile) {
                // Rows behind the sequence's last key hold anything, and 0 times that need not be 0.
                for (int at = max(present, 0) * (kHead * 2) + lane * 16; at < kTileBytes; at += 512) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_tile + at), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            if (!sm100::mbar_wait_warp(bar.p_ready(), n & 1, abort)) {
                break;
            }
            sm100::tc_fence_after_sync();
            const uint64_t v_desc = desc_mnmajor(v_tile, 0, 16);
            if (sm100::elect_one()) {
                sm100::mma_f16_ts_at<-1>(tmem_o, tmem_p, v_desc, 0, kIdescPV, begins ? 0u : 1u);
#pragma unroll
                for (int ks = 1; ks < 8; ++ks) {
                    sm100::mma_f16_ts_at<1>(tmem_o, tmem_p + ks * 8, v_desc, ks * 128, kIdescPV);
                }
                sm100::mma_commit(bar.pv_done());
                sm100::mma_commit(bar.slot_empty(slot));
            }
            __syncwarp();
            step_ring();
        }
    } else {
        constexpr int kColumns = kKeyTile / kSubsets / 2;    // of a key tile, that this thread works on
        constexpr int kChunk = kColumns < 32 ? kColumns : 32;
        constexpr int kChunks = kColumns / kChunk;
        constexpr int kOut = kHead / kSubsets / 2;           // columns of O that it writes
        constexpr int kCopyRows = kRows / kSubsets;
        const int quadrant = warp % 4;
        const int half = (warp - 2) / 4;
        const int subset = quadrant * kSubsets / 4;
        const int row = (quadrant * 32 + lane) % kCopyRows;  // of the tile
        const int lane_row = quadrant * 32 + lane;           // of the 128 lanes
        const uint32_t lane_base = static_cast<uint32_t>(quadrant * 32) << 16;
        const int first_column = (subset * 2 + half) * kColumns;
        const uint32_t my_scores = tmem_s + lane_base + first_column;
        const uint32_t my_weights = tmem_p + lane_base + first_column / 2;
        const uint32_t my_output = tmem_o + lane_base;
        const uint32_t my_staging = staging + (half * 4 + quadrant) * kStaging;
        const int token = row / p.group;
        const int head_of_group = row - token * p.group;
        const float scale2 = p.a.scale * kLog2e;
        const F2 scale_pair = f2_pack(scale2, scale2);
        Meeting meeting{bar.meeting(), 0, abort, lane};
        Meeting pair{bar.pair(quadrant), 0, abort, lane};
        if (quadrant == 0 && half == 0 && lane == 0) {
            p.records[blockIdx.x] = make_record(SequenceOf{p.a}, p.log_tokens, cuts[0], cuts[1]);
        }
        if (kSubsets > 1) {
            const uint32_t zeros[16] = {};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                sm100::tmem_st_32x16(tmem_p + lane_base + 32 * half + 16 * c, zeros);
            }
            sm100::tmem_st_wait();
        }
        uint32_t n = 0;
        bool ok = true;
        for (int round = 0; ok; ++round) {
            if (!sm100::mbar_wait_warp(bar.piece_full(round % kPieces), (round / kPieces) & 1, abort)) {
                break;
            }
            const PieceInfo& info = pieces[round % kPieces];
            const int from = info.from, to = info.to;
            if (to == 0) {
                break;
            }
            const bool whole = from == 0 && to == info.tiles;
            const int first_position = info.position;
            const bool valid = token < info.tokens;
            const int position = valid ? first_position + token : -1;
            const int info_row = info.first_row, info_head = info.head * p.group, info_tokens = info.tokens;
            const bool active = __any_sync(kFullMask, valid);    // (the same for a quadrant's two warps)
            float m = kNoKey;     // reference exponent of the row (base 2), shared by its two threads
            F2 l = 0;             // this thread's share of the row sum, in two partial sums
            for (int j = from; j < to; ++j, ++n) {
                if (!sm100::mbar_wait_warp(bar.s_full(), n & 1, abort)) {
                    ok = false;
                    break;
                }
                sm100::tc_fence_after_sync();
                // One copy of 64 columns is read twice, 32 at a time (64 bytes spilled; all at once, 500: two threads'
                // registers do not hold them beside everything else); up to 32 once.
                uint32_t raw[kChunk];
                auto read = [&](int c) {
                    if constexpr (kChunk == 32) {
                        sm100::tmem_ld_32x32(my_scores + 32 * c, raw);
                    } else {
                        sm100::tmem_ld_32x16(my_scores, raw);
                    }
                    sm100::tmem_ld_wait();
                };
                const bool masked = j * kKeyTile + kKeyTile - 1 > first_position;
                const int visible = position - j * kKeyTile - first_column;
                auto mask = [&](int c) {
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) {
                            raw[i] = kChunk * c + i <= visible ? raw[i] : 0xff800000u;
                        }
                    }
                };
                auto scores_are_read = [&]() {     // the next step's may come
                    sm100::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        sm100::mbar_arrive(bar.s_free());
                    }
                };
                float alpha = 1.0f;
                bool moved = false;
                if (active) {
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        read(c);
                        mask(c);
#pragma unroll
                        for (int i = 0; i < kChunk; i += 8) {
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                top[t] = max3_nan(top[t], __uint_as_float(raw[i + t]), __uint_as_float(raw[i + 4 + t]));
                            }
                        }
                    }
                    if (kChunks == 1) {
                        scores_are_read();
                    }
                    // The scale is positive, so the maximum may be scaled after it is taken.
                    const float local = max3_nan(top[0], top[1], max3_nan(top[2], top[3], top[3])) * scale2;
                    pair_max[n & 1][half][lane_row] = local;
                    if (!pair.meet()) {
                        ok = false;
                        break;
                    }
                    const float mx = max3_nan(m, local, pair_max[n & 1][half ^ 1][lane_row]);
                    moved = valid && !(mx - m <= kLazyShift);   // (a NaN moves it too)
                    if (moved) {
                        alpha = fast_exp2(m - mx);
                        m = mx;
                        l = f2_mul(l, f2_pack(alpha, alpha));
                    }
                }
                // O is complete up to the step before, and P's columns are free.
                if (n > 0 && !sm100::mbar_wait_warp(bar.pv_done(), (n - 1) & 1, abort)) {
                    ok = false;
                    break;
                }
                sm100::tc_fence_after_sync();
                if (active) {
                    if (j > from && __any_sync(kFullMask, moved)) {
                        const F2 a2 = f2_pack(alpha, alpha);
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            uint32_t acc[16];
                            sm100::tmem_ld_32x16(my_output + 32 * half + c * 16, acc);
                            sm100::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                float x, y;
                                f2_unpack(f2_mul(f2_pack(__uint_as_float(acc[i]), __uint_as_float(acc[i + 1])), a2), x, y);
                                acc[i] = __float_as_uint(x);
                                acc[i + 1] = __float_as_uint(y);
                            }
                            sm100::tmem_st_32x16(my_output + 32 * half + c * 16, acc);
                        }
                    }
                    const F2 shift = f2_pack(-m, -m);
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        if (kChunks > 1) {
                            read(c);
                            if (c + 1 == kChunks) {
                                scores_are_read();
                            }
                            mask(c);
                        }
                        uint32_t packed[kChunk / 2];
#pragma unroll
                        for (int i = 0; i < kChunk / 2; ++i) {
                            float x, y;
                            const F2 t = f2_fma(f2_pack(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1])),
                                                scale_pair, shift);
                            if (kSubsets == 1 && (i & 3) == 0) {
                                exp2_pair_fma<false>(t, x, y);
                            } else {
                                f2_unpack(t, x, y);
                                x = fast_exp2(x);
                                y = fast_exp2(y);
                            }
                            l = f2_add(l, f2_pack(x, y));
                            packed[i] = pack2(x, y);
                        }
                        if constexpr (kChunk == 32) {
                            sm100::tmem_st_32x16(my_weights + c * 16, packed);
                        } else {
                            sm100::tmem_st_32x8(my_weights, packed);
                        }
                    }
                    sm100::tmem_st_wait();
                } else {
                    scores_are_read();
                }
                sm100::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    sm100::mbar_arrive(bar.p_ready());
                }
            }
            if (!ok || !sm100::mbar_wait_warp(bar.pv_done(), (n - 1) & 1, abort)) {
                break;
            }
            sm100::tc_fence_after_sync();
            float sum_x, sum_y;
            f2_unpack(l, sum_x, sum_y);
            float total = m == kNoKey ? 0.0f : sum_x + sum_y;    // (the polynomial's least power of two is not 0)
            merge_sum[half * 4 + quadrant][lane] = total;
            if (kSubsets > 1 && half == 0) {
                merge_max[quadrant][lane] = m;
            }
            float acc[kOut];
            if constexpr (kSubsets == 1) {
                if (active) {
                    sm100::tmem_ld_32x32(my_output + 32 * half, reinterpret_cast<uint32_t(&)[32]>(acc));
                    sm100::tmem_ld_wait();
                }
                if (!pair.meet()) {
                    break;
                }
                total = merge_sum[quadrant][lane] + merge_sum[4 + quadrant][lane];
            } else {
                // The copies of a row: one reference exponent, one sum, and O's columns 16 at a time.
                if (!meeting.meet()) {
                    break;
                }
                constexpr int kApart = 4 / kSubsets;          // quadrants between a row's copies
                float top = kNoKey;
#pragma unroll
                for (int s = 0; s < kSubsets; ++s) {
                    top = max3_nan(top, merge_max[(quadrant % kApart) + s * kApart][lane], kNoKey);
                }
                const float mine = m == kNoKey ? 0.0f : fast_exp2(m - top);
                total = 0.0f;
#pragma unroll
                for (int s = 0; s < kSubsets; ++s) {
                    const int other = (quadrant % kApart) + s * kApart;
                    total += merge_max[other][lane] == kNoKey
                                 ? 0.0f
                                 : (merge_sum[other][lane] + merge_sum[4 + other][lane]) *
                                       fast_exp2(merge_max[other][lane] - top);
                }
                // In four rounds a quadrant's two warps hand over 8 of their 32 columns of O each.
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    uint32_t part[8];
                    sm100::tmem_ld_32x8(my_output + 32 * half + 8 * r, part);
                    sm100::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {     // (a copy that saw no key may hold 0 times anything)
                        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(my_staging + i * 256 + lane * 8),
                                     "f"(m == kNoKey ? 0.0f : __uint_as_float(part[2 * i]) * mine),
                                     "f"(m == kNoKey ? 0.0f : __uint_as_float(part[2 * i + 1]) * mine)
                                     : "memory");
                    }
                    ok = meeting.meet() && ok;
                    // Of these 8 columns, in pairs, this copy adds up its share: 8 / kSubsets.
#pragma unroll
                    for (int i = 0; i < 4 / kSubsets; ++i) {
                        float sum[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int s = 0; s < kSubsets; ++s) {
                            float v[2];
                            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                                         : "=f"(v[0]), "=f"(v[1])
                                         : "r"(staging + (half * 4 + (quadrant % kApart) + s * kApart) * kStaging +
                                               (subset * (4 / kSubsets) + i) * 256 + lane * 8)
                                         : "memory");
                            sum[0] += v[0];
                            sum[1] += v[1];
                        }
                        acc[r * (kOut / 4) + 2 * i] = sum[0];
                        acc[r * (kOut / 4) + 2 * i + 1] = sum[1];
                    }
                    ok = meeting.meet() && ok;     // (the staging is read)
                }
                m = top;
                if (!ok) {
                    break;
                }
            }
            sm100::tc_fence_before_sync();
            // This thread's columns of O: runs of kRun from 32 half + 8 r + its copy's share.
            constexpr int kRun = kSubsets == 1 ? 32 : 8 / kSubsets;
            auto column_of = [&](int i) {
                return kSubsets == 1 ? 32 * half + i : 32 * half + 8 * (i / kRun) + subset * kRun + i % kRun;
            };
            const long long out_row = static_cast<long long>(info_row) + token;
            const int head = info_head + head_of_group;
            if (whole) {
                const float inv = position < 0 ? 0.0f : 1.0f / total;   // no key at all gives zeros
#pragma unroll
                for (int i = 0; i < kOut; ++i) {
                    acc[i] = kPaged && position < 0 ? 0.0f : acc[i] * inv;
                }
                if constexpr (kSubsets == 1) {
                    // Through shared memory, 16 columns at a time, so that a row's 32 bytes leave by two lanes: rows are
                    // apart in memory, and 32 of them at 16 bytes each took three times as long.
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            float v[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                v[i] = acc[16 * r + 8 * b + i];
                            }
                            const uint4 q = pack8(v);
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                             my_staging + lane * 32 + ((b ^ ((lane >> 2) & 1)) << 4)),
                                         "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w)
                                         : "memory");
                        }
                        __syncwarp();
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int its = 16 * b + lane / 2;
                            uint4 q;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                                         : "r"(my_staging + its * 32 + (((lane & 1) ^ ((its >> 2) & 1)) << 4))
                                         : "memory");
                            const int there = quadrant * 32 + its, token_there = there / p.group;
                            if (token_there < info_tokens) {
                                __half* to_row = p.a.o + (static_cast<long long>(info_row) + token_there) * p.a.o_stride +
                                                 (info_head + there - token_there * p.group) * kHead + 32 * half + 16 * r;
                                reinterpret_cast<uint4*>(to_row)[lane & 1] = q;
                            }
                        }
                        __syncwarp();
                    }
                } else if (valid) {
                    __half* out = p.a.o + out_row * p.a.o_stride + head * kHead;
#pragma unroll
                    for (int i = 0; i < kOut; i += 2) {
                        *reinterpret_cast<unsigned*>(out + column_of(i)) = pack2(acc[i], acc[i + 1]);
                    }
                }
                if (valid && subset == 0 && half == 0 && p.a.lse != nullptr) {
                    p.a.lse[static_cast<long long>(head) * p.a.rows + out_row] =
                        position < 0 ? -INFINITY : (m + log2f(total)) * kLn2;
                }
            } else if (valid) {
                float* part = p.parts + (2 * size_t{blockIdx.x} + (from == 0 ? 1 : 0)) * kPartFloats;
#pragma unroll
                for (int i = 0; i < kOut; i += 2) {
                    const int column = column_of(i);
                    *reinterpret_cast<float2*>(part + (column / 4 * kRows + row) * 4 + column % 4) =
                        make_float2(acc[i], acc[i + 1]);
                }
                if (subset == 0 && half == 0) {
                    part[kRows * kHead + row] = m;
                    part[kRows * kHead + kRows + row] = total;
                }
            }
        }
    }
    __syncthreads();
    if (abort_flag != 0) {
        if (threadIdx.x == 0) {
            report();
        }
        const long long start = clock64();
        while (clock64() - start < 2000000LL) {
        }
        __syncthreads();
    }
    if (warp == 1) {
        sm100::tc_fence_after_sync();
        sm100::tmem_dealloc(tmem_slot, 256);
    }
}

// ---- the join -------------------------------------------------------------------------------------

struct JoinParams {
    PackedArgs a;
    const Record* records;
    const float* parts;
    int ctas, group;
};

constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kMostCtas = 1024;
// Caches of more than kManyKeys keys per sequence can make tiles of many parts. Those of more than kFewParts are then
// left to kHelpers other blocks (of shorter ones the block that has the tile joins them all, two at a time).
constexpr int kFewParts = 8;
constexpr int kManyKeys = 16384;
constexpr int kHelpers = 148;

// A row's sum over parts in the order of the keys, for kColumns of its columns: a running reference exponent, as in
// the softmax itself. A part of no key (m = kNoKey) may hold 0 times anything and is passed over.
template <int kColumns>
struct JoinSum {
    float m = kNoKey, total = 0.0f;
    float acc[kColumns] = {};
    __device__ __forceinline__ void add(float part_m, float part_total, const float4 (&x)[kColumns / 4]) {
        if (part_m == kNoKey) {
            return;
        }
        const float top = max3_nan(m, part_m, part_m);
        const float mine = fast_exp2(m - top), other = fast_exp2(part_m - top);
        m = top;
        total = total * mine + part_total * other;
#pragma unroll
        for (int i = 0; i < kColumns / 4; ++i) {
            const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                acc[4 * i + c] = acc[4 * i + c] * mine + v[c] * other;
            }
        }
    }
};

// Block k joins the tile that CTA k began and did not end, if there is one: a warp has 32 rows and 32 columns, a
// row per lane, and two parts on their way at a time. The helpers, which come first, take the tiles in many
// parts, 32 rows and four columns at a time, a warp's share of the parts each.
__global__ void __launch_bounds__(kJoinThreads) fb_packed_join(const JoinParams p) {
    __shared__ uint4 staged[kJoinWarps][128];
    __shared__ float sums[kJoinWarps][32][7];
    __shared__ unsigned ends[kMostCtas / 32 + 1];      // bit k: CTA k's first piece is not the middle of a tile
    __shared__ int many[kMostCtas / kFewParts + 1], many_last[kMostCtas / kFewParts + 1];
    __shared__ int many_count;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    dependency_wait();
    dependency_release();
    auto rows_of = [&](const Record& r) { return r.tokens * p.group; };
    // Where a row of a tile goes.
    auto out_of = [&](const Record& r, int row) {
        const int token = row / p.group;
        return p.a.o + (static_cast<long long>(r.first_row) + token) * p.a.o_stride +
               (r.kv_head * p.group + row - token * p.group) * kHead;
    };
    auto none_of = [&](const Record& r, int row) { return r.position + row / p.group < 0; };
    auto store_lse = [&](const Record& r, int row, float m, float total) {
        const int token = row / p.group;
        p.a.lse[static_cast<long long>(r.kv_head * p.group + row - token * p.group) * p.a.rows + r.first_row + token] =
            none_of(r, row) ? -INFINITY : (m + log2f(total)) * kLn2;
    };
    // Part i of the tile that CTA k began.
    auto part_of = [&](int k, int i) {
        return p.parts + (2 * static_cast<size_t>(k + i) + (i == 0 ? 1 : 0)) * kPartFloats;
    };
    const int helpers = static_cast<int>(gridDim.x) - p.ctas;
    if (static_cast<int>(blockIdx.x) >= helpers) {
        const int k = static_cast<int>(blockIdx.x) - helpers;
        // Own record, and whether the CTAs behind go on with the tile.
        const Record mine = p.records[k];
        int count = 0;      // of parts
        for (int from = k + 1; count == 0; from += 32) {
            const unsigned found =
                __ballot_sync(kFullMask, from + lane >= p.ctas || p.records[from + lane].head_part != 2);
            if (mine.tail_part == 0) {
                return;
            }
            count = found != 0 ? min(from + __ffs(found) - 1, p.ctas - 1) - k + 1 : 0;
        }
        if (count > kFewParts && helpers > 0) {
            return;
        }
        const int row = warp % 4 * 32 + lane, half = warp / 4;
        if (warp % 4 * 32 >= rows_of(mine)) {
            return;
        }
        JoinSum<32> sum;
        for (int i = 0; i < count; i += 2) {
            float4 x[2][8];
            float m[2], total[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[c] = kNoKey;
                total[c] = 0.0f;
                if (i + c < count) {
                    const float* part = part_of(k, i + c);
                    m[c] = part[kRows * kHead + row];
                    total[c] = part[kRows * kHead + kRows + row];
#pragma unroll
                    for (int b = 0; b < 8; ++b) {
                        x[c][b] = reinterpret_cast<const float4*>(part)[(8 * half + b) * kRows + row];
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                sum.add(m[c], total[c], x[c]);
            }
        }
        const bool none = none_of(mine, row);
        const float inv = 1.0f / sum.total;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                v[c] = none ? 0.0f : sum.acc[8 * b + c] * inv;
            }
            staged[warp][lane * 4 + (b ^ ((lane >> 1) & 3))] = pack8(v);
        }
        __syncwarp();
        // A row's 64 bytes leave by four lanes.
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int r = 8 * b + lane / 4, its = warp % 4 * 32 + r;
            const uint4 q = staged[warp][r * 4 + ((lane & 3) ^ ((r >> 1) & 3))];
            if (its < rows_of(mine)) {
                reinterpret_cast<uint4*>(out_of(mine, its) + 32 * half)[lane & 3] = q;
            }
        }
        if (half == 0 && row < rows_of(mine) && p.a.lse != nullptr) {
            store_lse(mine, row, sum.m, sum.total);
        }
        return;
    }
    // A helper: the tiles of many parts, in the order of their CTAs.
    const int words = (p.ctas + 31) / 32;
    for (int k = threadIdx.x; k < words * 32; k += kJoinThreads) {
        const unsigned bits = __ballot_sync(kFullMask, k >= p.ctas || p.records[k].head_part != 2);
        if (lane == 0) {
            ends[k / 32] = bits;
        }
    }
    if (threadIdx.x == 0) {
        many_count = 0;
    }
    __syncthreads();
    if (warp == 0) {
        int listed = 0;
        for (int from = 0; from < p.ctas; from += 32) {
            // The first CTA behind this one whose piece of the tile is its last.
            const int k = from + lane;
            int last = p.ctas;
            if (k + 1 < p.ctas) {
                int word = (k + 1) / 32;
                unsigned bits = ends[word] & (kFullMask << ((k + 1) % 32));
                while (bits == 0 && word + 1 < words) {
                    bits = ends[++word];
                }
                last = bits != 0 ? word * 32 + __ffs(bits) - 1 : p.ctas;
            }
            const bool is = k + 1 < p.ctas && last < p.ctas && last - k + 1 > kFewParts && p.records[k].tail_part != 0;
            const unsigned those = __ballot_sync(kFullMask, is);
            if (is) {
                const int place = listed + __popc(those & ((1u << lane) - 1));
                many[place] = k;
                many_last[place] = last;
            }
            listed += __popc(those);
        }
        if (lane == 0) {
            many_count = listed;
        }
    }
    __syncthreads();
    constexpr int kEach = (kRows / 32) * (kHead / 4);
    for (int item = static_cast<int>(blockIdx.x); item < many_count * kEach; item += helpers) {
        // (The row groups outermost: few rows have the first one only.)
        const int at = item % (many_count * (kHead / 4));
        const int first_row = item / (many_count * (kHead / 4)) * 32;
        const int k = many[at / (kHead / 4)], column = at % (kHead / 4);     // by four
        const Record mine = p.records[k];
        if (first_row >= rows_of(mine)) {
            continue;
        }
        const int count = many_last[at / (kHead / 4)] - k + 1;
        const int row = first_row + lane;
        JoinSum<4> sum;
        for (int i = warp; i < count; i += 8 * kJoinWarps) {
            float4 x[8][1];
            float m[8], total[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                m[c] = kNoKey;
                total[c] = 0.0f;
                if (i + c * kJoinWarps < count) {
                    const float* part = part_of(k, i + c * kJoinWarps);
                    m[c] = part[kRows * kHead + row];
                    total[c] = part[kRows * kHead + kRows + row];
                    x[c][0] = reinterpret_cast<const float4*>(part)[column * kRows + row];
                }
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                sum.add(m[c], total[c], x[c]);
            }
        }
        sums[warp][lane][4] = sum.m;
        sums[warp][lane][5] = sum.total;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            sums[warp][lane][c] = sum.acc[c];
        }
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < kJoinWarps; ++w) {
                const float* from = sums[w][lane];
                const float4 x[1] = {make_float4(from[0], from[1], from[2], from[3])};
                sum.add(from[4], from[5], x);
            }
            if (row < rows_of(mine)) {
                const float inv = 1.0f / sum.total;
                reinterpret_cast<uint2*>(out_of(mine, row))[column] =
                    none_of(mine, row) ? make_uint2(0u, 0u)
                                       : make_uint2(pack2(sum.acc[0] * inv, sum.acc[1] * inv),
                                                    pack2(sum.acc[2] * inv, sum.acc[3] * inv));
                if (column == 0 && p.a.lse != nullptr) {
                    store_lse(mine, row, sum.m, sum.total);
                }
            }
        }
        __syncthreads();      // (the sums are read)
    }
}

// ---- host -------------------------------------------------------------------------------------------

size_t records_bytes(int ctas) { return (static_cast<size_t>(ctas) * sizeof(Record) + 255) / 256 * 256; }

}  // namespace

cudaError_t packed_forward_error_flag(int* value, bool reset) { return read_error_word(value, reset); }

cudaError_t packed_forward_workspace(size_t* bytes) {
    int sms = 148;
    const cudaError_t e = sm_count(&sms);
    const int ctas = std::min(2 * sms, kMostCtas);
    *bytes = records_bytes(ctas) + 2 * static_cast<size_t>(ctas) * kPartFloats * sizeof(float);
    return e;
}

cudaError_t packed_forward(const PackedArgs& args, int longest, void* workspace, cudaStream_t stream) {
    TileParams p;
    std::memset(&p, 0, sizeof p);
    p.a = args;
    p.group = args.heads / args.kv_heads;
    const bool paged = args.table != nullptr;
    // Few rows per K/V head and sequence: in two or four copies.
    const long long rows = static_cast<long long>(longest) * p.group;
    const int subsets = !paged || rows > 64 ? 1 : rows > 32 ? 2 : 4;
    while ((2 << p.log_tokens) * p.group <= kRows / subsets) {
        ++p.log_tokens;
    }
    int sms = 148;
    cudaError_t e = sm_count(&sms);
    const int ctas = std::min(2 * sms, kMostCtas);
    if (e == cudaSuccess) {
        e = encode_rows(&p.map_q, args.q, args.heads, args.rows, args.q_stride, p.group, 1 << p.log_tokens);
    }
    if (paged) {
        p.box_rows = std::min(args.page_size, kKeyTile);
        p.boxes = kKeyTile / p.box_rows;
        const long long cache_rows = args.pages * args.kv_heads * args.page_size;
        if (e == cudaSuccess) e = encode_pages(&p.map_k, args.k, cache_rows, p.box_rows);
        if (e == cudaSuccess) e = encode_pages(&p.map_v, args.v, cache_rows, p.box_rows);
    } else {
        if (e == cudaSuccess) e = encode_rows(&p.map_k, args.k, args.kv_heads, args.rows, args.kv_stride, 1, kKeyTile);
        if (e == cudaSuccess) e = encode_rows(&p.map_v, args.v, args.kv_heads, args.rows, args.kv_stride, 1, kKeyTile);
    }
    if (e != cudaSuccess) {
        return e;
    }
    // Few rows have few key tiles each: whole tiles for every CTA, and no join.
    const long long most_keys = paged ? static_cast<long long>(args.table_stride) * args.page_size : args.rows;
    p.splits = most_keys > kWholeKeys;
    p.records = static_cast<Record*>(workspace);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + records_bytes(ctas));
    const int form = !paged ? 0 : subsets == 1 ? 1 : subsets == 2 ? 2 : 3;
    const auto kernel = form == 0   ? fb_packed_forward_tiles<false, 1>
                        : form == 1 ? fb_packed_forward_tiles<true, 1>
                        : form == 2 ? fb_packed_forward_tiles<true, 2>
                                    : fb_packed_forward_tiles<true, 4>;
    static std::atomic<bool> configured[4][64] = {};
    e = allow_shared_memory(kernel, kSmem, configured[form]);
    if (e != cudaSuccess) {
        return e;
    }
    e = launch_dependent(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmem, stream, p);
    if (e != cudaSuccess || !p.splits) {
        return e;
    }
    JoinParams j = {args, p.records, p.parts, ctas, p.group};
    return launch_dependent(fb_packed_join, dim3(static_cast<unsigned>(ctas + (most_keys > kManyKeys ? kHelpers : 0))),
                            dim3(kJoinThreads), 0, stream, j);
}

}  // namespace fb
