// Gradients of packed attention (head width 64) on the 5th-generation tensor cores.
//
//   P = exp2(scale log2(e) Q K^T - lse),  dV = sum over the group's heads of P^T dO,
//   dS = P (dO V^T - delta),  delta = rowsum(dO O),  dQ = scale dS K,  dK = scale sum over the group of dS^T Q
//
// Two launches. The first takes delta and the log-sum-exps into rows that start on 16 bytes for every
// sequence (bulk copies need that), and one of its blocks lists the batch's blocks of 128 tokens, those with
// the most work first. In the second, persistent CTAs work through (block, K/V head) items for
// dK and dV, the others through (block, query head) items for dQ: scores are recomputed by both, so that every
// output element has one CTA, which adds in a fixed order; the heads that share keys add up in
// tensor memory. The A operands of all products are in tensor memory and shared memory feeds
// the streamed 64-row tiles only, as in the kernels for equal lengths (attention.cu). A sub-step of 128 x 64 takes a CTA
// about a thousand clocks: chains between the compute warps and products of N = 64, not a pipe, bound it.
// Measured, all launches: 16 sequences of up to 1,024 tokens, 12 heads, 53 us; 5 of up to 4,096, 16 heads on 4,
// 187 us (550 TFLOP/s of the seven products). Two launches because delta needs O's whole rows; a third, which adds
// up divided groups, only where blocks are few.
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

constexpr int kBlock = 128;      // tokens of an item
constexpr int kHead = 64;
constexpr int kTileBytes = kBlock * kHead * 2;
constexpr int kSub = 64;         // streamed rows (queries for dK and dV, keys for dQ) per sub-step
constexpr int kSubBytes = kSub * kHead * 2;
constexpr int kThreads = 576;    // TMA warp, MMA warp, 16 compute warps
constexpr int kComputeWarps = 16;
constexpr int kPart = 16;        // accumulator columns per compute thread and sub-step
constexpr int kStages = 4;
constexpr int kStatBytes = kSub * 4;
constexpr int kUsed = 1024 + 2 * kTileBytes + kStages * 2 * kSubBytes + kStages * 2 * kStatBytes + 256;
// More than half of an SM's shared memory keeps two CTAs, each of which wants all of tensor
// memory, from landing on one SM.
constexpr int kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
constexpr double kKeyShare = 0.575;   // of the CTAs, for dK and dV (four products and row statistics against three)
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kListThreads = 256;
constexpr int kLevels = 1024;    // of work that the list tells apart
constexpr int kItems = 8;        // ring of items that the TMA warp has taken

// A block of 128 tokens of a sequence of `count`: `level` blocks from the sequence's end (for dK and dV), the
// level-th from its beginning (for dQ), so that the work is proportional to it in either.
struct Entry {
    int first, count, level, stats;   // row of the sequence's first token; where its statistics begin
};

struct BackwardParams {
    CUtensorMap map_q, map_k, map_v, map_do;    // boxes of 64 rows
    PackedArgs a;
    PackedGradients g;
    const Entry* entries;
    int* counts;              // of the entries; of the items taken so far, for dK and dV and for dQ
    const float* lse2;        // [heads, stats_stride]: log2(e) times the log-sum-exps
    const float* delta;
    long long stats_stride;
    int group;
    // Few blocks: a group's heads are divided among `slices` items, whose sums (FP32 [slice][row][K/V head][dK, dV][64])
    // a third launch adds up.
    int slices;
    float* partial;
};

struct Barriers {
    uint32_t base;
    __device__ uint32_t resident() const { return base; }
    __device__ uint32_t done() const { return base + 8; }
    __device__ uint32_t a_ready() const { return base + 16; }
    __device__ uint32_t scores_full(int b) const { return base + 32 + 8u * b; }
    __device__ uint32_t operands_ready(int b) const { return base + 48 + 8u * b; }
    __device__ uint32_t stage_full(int s) const { return base + 64 + 8u * s; }
    __device__ uint32_t stage_empty(int s) const { return base + 96 + 8u * s; }
    __device__ uint32_t item_full(int i) const { return base + 128 + 8u * i; }
};

constexpr uint32_t kIdescSub = sm100::instr_desc_f16(128, 64, false, false);
constexpr uint32_t kIdescOut = sm100::instr_desc_f16(128, 64, false, true);

// Where a sequence's statistics begin: on 16 bytes, and never before the sequence before ends.
__device__ __forceinline__ int stats_at(int first, int s) { return (first & ~3) + 4 * s; }

// ---- the first launch --------------------------------------------------------------------------

struct PrepareParams {
    PackedArgs a;
    const __half* d_o;
    Entry* entries;
    int* counts;
    float* lse2;
    float* delta;
    long long stats_stride;
    int capacity;             // of the entries: enough for any sequences that do not overlap
};

// One block lists the blocks of 128 tokens by their work, descending (a counting sort).
__device__ void list_blocks(const PrepareParams& p) {
    __shared__ int counts[kLevels];
    __shared__ int sums[kListThreads / 32];
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    for (int i = tid; i < kLevels; i += kListThreads) {
        counts[i] = 0;
    }
    __syncthreads();
    for (int s = warp; s < p.a.sequences; s += kListThreads / 32) {
        const Sequence q = sequence_at(p.a, s);
        for (int level = 1 + lane; level <= (q.count + kBlock - 1) / kBlock; level += 32) {
            atomicAdd(&counts[kLevels - 1 - min(level, kLevels - 1)], 1);
        }
    }
    __syncthreads();
    // Exclusive sums over the levels, the largest first: four per thread.
    static_assert(kLevels == 4 * kListThreads, "four levels per thread");
    int mine[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        mine[i] = counts[4 * tid + i];
        sum += mine[i];
    }
    int upto = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int other = __shfl_up_sync(kFullMask, upto, off);
        upto += lane >= off ? other : 0;
    }
    if (lane == 31) {
        sums[warp] = upto;
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
        upto += sums[w];
    }
    if (tid == kListThreads - 1) {
        p.counts[0] = min(upto, p.capacity);
        p.counts[1] = p.counts[2] = 0;
    }
    int at = upto - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        counts[4 * tid + i] = at;
        at += mine[i];
    }
    __syncthreads();
    for (int s = warp; s < p.a.sequences; s += kListThreads / 32) {
        const Sequence q = sequence_at(p.a, s);
        for (int level = 1 + lane; level <= (q.count + kBlock - 1) / kBlock; level += 32) {
            const int place = atomicAdd(&counts[kLevels - 1 - min(level, kLevels - 1)], 1);
            if (place < p.capacity) {
                p.entries[place] = Entry{q.first, q.count, level, stats_at(q.first, s)};
            }
        }
    }
}

// A warp per row: eight lanes per head, 16 bytes of dO and of O each. (The order of the entries of
// one level is not fixed; it decides only which CTA an item goes to.)
__global__ void __launch_bounds__(kListThreads) fb_packed_backward_prepare(const PrepareParams p) {
    dependency_wait();
    dependency_release();
    if (blockIdx.x == 0) {
        list_blocks(p);
        return;
    }
    const uint4* d_o = reinterpret_cast<const uint4*>(after_wait(p.d_o));
    const uint4* o = reinterpret_cast<const uint4*>(after_wait(static_cast<const __half*>(p.a.o)));
    const int lane = threadIdx.x % 32;
    const int warps = (gridDim.x - 1) * (kListThreads / 32);
    for (int row = (blockIdx.x - 1) * (kListThreads / 32) + threadIdx.x / 32; row < p.a.rows; row += warps) {
        // The last sequence that begins at or before the row: 32 of them looked at in one step.
        int low = 0;
        for (int count = p.a.sequences; count > 1;) {
            const int step = (count + 31) / 32;
            const bool before = lane * step < count && p.a.starts[low + min(lane * step, count - 1)] <= row;
            const int which = max(__popc(__ballot_sync(kFullMask, before)) - 1, 0);
            low += which * step;
            count = min(step, count - which * step);
        }
        const Sequence q = sequence_at(p.a, low);
        if (row < q.first || row >= q.first + q.count) {
            continue;
        }
        const long long at = stats_at(q.first, low) + (row - q.first);
        const long long o_row = static_cast<long long>(row) * p.a.o_stride / 8;      // in words of eight values
        // Four heads at a time, and four times that on their way.
        for (int first_head = 0; first_head < p.a.heads; first_head += 16) {
            uint4 x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int head = first_head + 4 * i + lane / 8;
                x[i] = y[i] = make_uint4(0u, 0u, 0u, 0u);
                if (head < p.a.heads) {
                    x[i] = load_input(d_o + o_row + head * (kHead / 8) + lane % 8);
                    y[i] = load_input(o + o_row + head * (kHead / 8) + lane % 8);
                }
            }
            const int stat_head = first_head + lane;
            const float lse = lane < 16 && stat_head < p.a.heads ? p.a.lse[static_cast<long long>(stat_head) * p.a.rows + row] : 0.0f;
            float sums[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float a[8], b[8];
                unpack8(a, x[i]);
                unpack8(b, y[i]);
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    sum = fmaf(a[c], b[c], sum);
                }
                sum += __shfl_xor_sync(kFullMask, sum, 4);
                sum += __shfl_xor_sync(kFullMask, sum, 2);
                sums[i] = sum + __shfl_xor_sync(kFullMask, sum, 1);
            }
            // Lane h of the first 16 has head first_head + h: of quarter h / 4, from the eight lanes 8 (h % 4).
            float delta = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float other = __shfl_sync(kFullMask, sums[i], 8 * (lane % 4));
                delta = lane / 4 == i ? other : delta;
            }
            if (lane < 16 && stat_head < p.a.heads) {
                p.delta[stat_head * p.stats_stride + at] = delta;
                p.lse2[stat_head * p.stats_stride + at] = lse * kLog2e;
            }
        }
    }
}

// ---- pieces of the second launch ------------------------------------------------------------------

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}

// Two exponentials; a quarter of the pairs takes the FMA pipe.
__device__ __forceinline__ void exp2_two(int pair, float x0, float x1, float& e0, float& e1) {
    if ((pair & 3) == 0) {
        exp2_pair_fma<true>(f2_pack(x0, x1), e0, e1);
    } else {
        e0 = fast_exp2(x0);
        e1 = fast_exp2(x1);
    }
}

// This thread's 16 columns of a row of a resident tile (swizzled as TMA wrote it) into tensor
// memory as part of an A operand.
__device__ __forceinline__ void tile_row_to_tmem(uint32_t dst, uint32_t tile, int row, int part) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int chunk = part * 2 + i;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[4 * i]), "=r"(r[4 * i + 1]), "=r"(r[4 * i + 2]), "=r"(r[4 * i + 3])
                     : "r"(tile + row * 128 + ((chunk ^ (row & 7)) << 4)));
    }
    sm100::tmem_st_32x8(dst + 8 * part, r);
}

__device__ __forceinline__ void pack_pairs(uint32_t (&w)[8], const float (&v)[kPart]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        w[i] = pack2(v[2 * i], v[2 * i + 1]);
    }
}

__device__ __forceinline__ void warp_arrive_after_stores(uint32_t bar, int lane) {
    sm100::tmem_st_wait();
    sm100::tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) {
        sm100::mbar_arrive(bar);
    }
}

// Zeros the rows of a 64-row tile from `present` on (a whole warp): behind a sequence's end lies anything, and 0 times
// that need not be 0.
__device__ __forceinline__ void zero_rows(uint32_t tile, int present, int lane) {
    for (int at = max(present, 0) * (kHead * 2) + lane * 16; at < kSubBytes; at += 512) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + at), "r"(0) : "memory");
    }
}

struct Shared {
    uint32_t base;
    Barriers bar;
    uint32_t tmem;
    volatile int* abort;
    int warp;
};

// The items of a kind, which CTAs take one after the other from the list, the longest first: whoever is done takes
// the next one. (Dealt out in advance, the CTAs' sums differed by 30 % where a group of four shares keys.) The TMA warp
// takes an item when the loads of the one before are issued (not earlier: an item taken ahead is one that another CTA
// would have had time for) and leaves its number in a ring for the others.
struct Items {
    int* taken;
    int count;
    volatile int* ring;
    Barriers bar;
    volatile int* abort;
    // TMA warp, one lane.
    __device__ __forceinline__ int take(int round) const {
        const int item = atomicAdd(taken, 1);
        ring[round % kItems] = item < count ? item : -1;
        sm100::mbar_arrive(bar.item_full(round % kItems));
        return item < count ? item : -1;
    }
    // A whole warp: the item of this round, or -1 behind the last one.
    __device__ __forceinline__ int of(int round) const {
        if (!sm100::mbar_wait_warp(bar.item_full(round % kItems), (round / kItems) & 1, abort)) {
            return -1;
        }
        return ring[round % kItems];
    }
};

// An item for dK and dV: keys [key, key + 128) of an entry's sequence; per head of the group, sub-steps of 64
// queries from the diagonal on.
struct KeyItem {
    Entry e;
    int head, slice, first_head, heads, key, subs, steps;     // of the group's heads: those of the slice
    __device__ __forceinline__ KeyItem(const BackwardParams& p, int item) {
        const int each = p.a.kv_heads * p.slices;
        const int at = item / each;
        e = p.entries[at];
        slice = (item - at * each) / p.a.kv_heads;
        head = (item - at * each) % p.a.kv_heads;
        const int from = slice * p.group / p.slices;
        first_head = head * p.group + from;
        heads = (slice + 1) * p.group / p.slices - from;
        key = ((e.count + kBlock - 1) / kBlock - e.level) * kBlock;
        subs = (e.count - key + kSub - 1) / kSub;
        steps = subs * heads;
    }
};

// An item for dQ: queries [query, query + 128), sub-steps of 64 keys up to the diagonal.
struct QueryItem {
    Entry e;
    int head, query, steps;
    __device__ __forceinline__ QueryItem(const BackwardParams& p, int item) {
        const int at = item / p.a.heads;
        e = p.entries[at];
        head = item - at * p.a.heads;
        query = (e.level - 1) * kBlock;
        steps = (min(e.count, query + kBlock) + kSub - 1) / kSub;
    }
};

// ---- dK and dV --------------------------------------------------------------------------------------
//
// Scores are formed transposed, S^T = K Q^T and dP^T = V dO^T with keys on the lanes (A = K, V from tensor
// memory), so that P^T and dS^T are already the A operands of dV += P^T dO and dK += dS^T Q. The MMA
// warp issues a sub-step's score products before it waits for the probabilities of the one
// before; items overlap as well. Sub-steps are counted through all items, and a count's low bit names its accumulators.
// Tensor memory: S^T at 0/64, dP^T at 128/192 (P^T and dS^T overwrite 4 x 8 columns of each), dV 256,
// dK 320, K 384, V 416.

__device__ __forceinline__ void key_items(const BackwardParams& p, const Shared& shared, const Items& items) {
    const uint32_t k_tile = shared.base, v_tile = shared.base + kTileBytes;
    const uint32_t ring = shared.base + 2 * kTileBytes;           // stage: Q then dO
    const uint32_t stats = ring + kStages * 2 * kSubBytes;        // stage: lse2[64] then delta[64]
    const Barriers bar = shared.bar;
    volatile int* abort = shared.abort;
    const int warp = shared.warp;
    const int lane = threadIdx.x % 32;
    const uint32_t tmem = shared.tmem;
    auto tmem_st = [&](uint32_t count) { return tmem + 64u * (count & 1); };
    auto tmem_dpt = [&](uint32_t count) { return tmem + 128u + 64u * (count & 1); };
    const uint32_t tmem_dv = tmem + 256, tmem_dk = tmem + 320, tmem_k = tmem + 384, tmem_v = tmem + 416;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            int round = 0;
            for (int item = items.take(0); ok && item >= 0; item = items.take(++round)) {
                const KeyItem it(p, item);
                // The K and V buffers are free once the item before was copied to tensor memory.
                if (round > 0 && !sm100::mbar_wait(bar.a_ready(), (round - 1) & 1, abort)) {
                    break;
                }
                sm100::mbar_expect_tx(bar.resident(), 2 * kTileBytes);
                for (int half = 0; half < 2; ++half) {
                    const int row = it.e.first + it.key + half * kSub;
                    sm100::tma_load_3d(k_tile + half * kSubBytes, &p.map_k, bar.resident(), 0, it.head, row);
                    sm100::tma_load_3d(v_tile + half * kSubBytes, &p.map_v, bar.resident(), 0, it.head, row);
                }
                for (int g = 0; ok && g < it.heads; ++g) {
                    const int head = it.first_head + g;
                    for (int h = 0; h < it.subs; ++h) {
                        if (!sm100::mbar_wait(bar.stage_empty(stage), phase ^ 1u, abort)) {
                            ok = false;
                            break;
                        }
                        const int query = it.key + h * kSub;
                        const uint32_t dst = ring + stage * 2 * kSubBytes, full = bar.stage_full(stage);
                        sm100::mbar_expect_tx(full, 2 * kSubBytes + 2 * kStatBytes);
                        sm100::tma_load_3d(dst, &p.map_q, full, 0, head, it.e.first + query);
                        sm100::tma_load_3d(dst + kSubBytes, &p.map_do, full, 0, head, it.e.first + query);
                        const long long at = head * p.stats_stride + it.e.stats + query;
                        const uint32_t slot = stats + stage * 2 * kStatBytes;
                        bulk_load(slot, p.lse2 + at, kStatBytes, full);
                        bulk_load(slot + kStatBytes, p.delta + at, kStatBytes, full);
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        const uint64_t q_desc = sm100::smem_desc_sw128(ring, 16, 1024);
        const uint64_t do_desc = sm100::smem_desc_sw128(ring + kSubBytes, 16, 1024);
        uint32_t before = 0;   // sub-steps of earlier items
        bool ok = true;
        int round = 0;
        for (int item = items.of(0); ok && item >= 0; item = items.of(++round)) {
            const KeyItem it(p, item);
            ok = sm100::mbar_wait_warp(bar.a_ready(), round & 1, abort);
            sm100::tc_fence_after_sync();
            int sub_ahead = 0;
            auto issue_scores = [&](int step) -> bool {
                const uint32_t count = before + step;
                const int stage = count % kStages;
                if (!sm100::mbar_wait_warp(bar.stage_full(stage), (count / kStages) & 1, abort)) {
                    return false;
                }
                sm100::tc_fence_after_sync();
                const int present = it.e.count - (it.key + sub_ahead * kSub);
                if (present < kSub) {
                    const uint32_t tile = ring + stage * 2 * kSubBytes;
                    zero_rows(tile, present, lane);
                    zero_rows(tile + kSubBytes, present, lane);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                sub_ahead = sub_ahead + 1 == it.subs ? 0 : sub_ahead + 1;
                const uint64_t q_sub = q_desc + stage * (2 * kSubBytes >> 4);
                const uint64_t do_sub = do_desc + stage * (2 * kSubBytes >> 4);
                if (sm100::elect_one()) {
                    const uint32_t st_at = tmem_st(count), dpt_at = tmem_dpt(count);
                    sm100::mma_f16_ts_at<0>(st_at, tmem_k, q_sub, 0, kIdescSub);
                    sm100::mma_f16_ts_at<1>(st_at, tmem_k + 8, q_sub, 2, kIdescSub);
                    sm100::mma_f16_ts_at<1>(st_at, tmem_k + 16, q_sub, 4, kIdescSub);
                    sm100::mma_f16_ts_at<1>(st_at, tmem_k + 24, q_sub, 6, kIdescSub);
                    sm100::mma_f16_ts_at<0>(dpt_at, tmem_v, do_sub, 0, kIdescSub);
                    sm100::mma_f16_ts_at<1>(dpt_at, tmem_v + 8, do_sub, 2, kIdescSub);
                    sm100::mma_f16_ts_at<1>(dpt_at, tmem_v + 16, do_sub, 4, kIdescSub);
                    sm100::mma_f16_ts_at<1>(dpt_at, tmem_v + 24, do_sub, 6, kIdescSub);
                    sm100::mma_commit(bar.scores_full(count & 1));
                }
                __syncwarp();
                return true;
            };
            ok = ok && issue_scores(0);
            for (int step = 0; ok && step < it.steps; ++step) {
                const uint32_t count = before + step;
                if (step + 1 < it.steps && !issue_scores(step + 1)) {
                    ok = false;
                    break;
                }
                if (!sm100::mbar_wait_warp(bar.operands_ready(count & 1), (count >> 1) & 1, abort)) {
                    ok = false;
                    break;
                }
                sm100::tc_fence_after_sync();
                const int stage = count % kStages;
                const uint64_t q_sub = q_desc + stage * (2 * kSubBytes >> 4);
                const uint64_t do_sub = do_desc + stage * (2 * kSubBytes >> 4);
                // Queries 16 part + [0, 16) sit in columns 16 part + [0, 8) of the accumulators.
                if (sm100::elect_one()) {
                    const uint32_t st_at = tmem_st(count), dpt_at = tmem_dpt(count);
                    sm100::mma_f16_ts_at<-1>(tmem_dv, st_at, do_sub, 0, kIdescOut, step != 0);
                    sm100::mma_f16_ts_at<1>(tmem_dv, st_at + 16, do_sub, 128, kIdescOut);
                    sm100::mma_f16_ts_at<1>(tmem_dv, st_at + 32, do_sub, 256, kIdescOut);
                    sm100::mma_f16_ts_at<1>(tmem_dv, st_at + 48, do_sub, 384, kIdescOut);
                    sm100::mma_f16_ts_at<-1>(tmem_dk, dpt_at, q_sub, 0, kIdescOut, step != 0);
                    sm100::mma_f16_ts_at<1>(tmem_dk, dpt_at + 16, q_sub, 128, kIdescOut);
                    sm100::mma_f16_ts_at<1>(tmem_dk, dpt_at + 32, q_sub, 256, kIdescOut);
                    sm100::mma_f16_ts_at<1>(tmem_dk, dpt_at + 48, q_sub, 384, kIdescOut);
                    sm100::mma_commit(bar.stage_empty(stage));
                    if (step + 1 == it.steps) {
                        sm100::mma_commit(bar.done());
                    }
                }
                __syncwarp();
            }
            before += it.steps;
        }
    } else {
        const int quadrant = warp % 4;
        const int part = (warp - 2) / 4;               // which 16 of the 64 query columns
        const int row = quadrant * 32 + lane;          // key row in the block
        const uint32_t lane_base = static_cast<uint32_t>(quadrant * 32) << 16;
        const float scale2 = p.a.scale * kLog2e;
        auto install = [&](int round) -> bool {
            if (!sm100::mbar_wait_warp(bar.resident(), round & 1, abort)) {
                return false;
            }
            tile_row_to_tmem(tmem_k + lane_base, k_tile, row, part);
            tile_row_to_tmem(tmem_v + lane_base, v_tile, row, part);
            warp_arrive_after_stores(bar.a_ready(), lane);
            return true;
        };
        uint32_t before = 0;
        int round = 0;
        int item = items.of(0);
        bool ok = item >= 0 && install(0);
        for (; ok && item >= 0; item = items.of(++round)) {
            const KeyItem it(p, item);
            const int key = it.key + row;
            int sub = 0;
            for (int step = 0; ok && step < it.steps; ++step) {
                const uint32_t count = before + step;
                const int stage = count % kStages;
                const int query = it.key + sub * kSub + part * kPart;   // first one of my columns
                // (A lane that gives up goes along to the end of the sub-step, where the warp agrees.)
                bool there = sm100::mbar_wait(bar.scores_full(count & 1), (count >> 1) & 1, abort);
                sm100::tc_fence_after_sync();
                const uint32_t my_scores = tmem_st(count) + lane_base + part * kPart;
                const uint32_t my_weights = tmem_dpt(count) + lane_base + part * kPart;
                uint32_t s_raw[kPart], dp_raw[kPart];
                sm100::tmem_ld_32x16(my_scores, s_raw);
                sm100::tmem_ld_32x16(my_weights, dp_raw);
                there = sm100::mbar_wait(bar.stage_full(stage), (count / kStages) & 1, abort) && there;
                const uint32_t stat = stats + stage * 2 * kStatBytes + part * kPart * 4;
                float lse2[kPart], delta[kPart];
#pragma unroll
                for (int c = 0; c < kPart / 4; ++c) {
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(lse2[4 * c]), "=f"(lse2[4 * c + 1]), "=f"(lse2[4 * c + 2]), "=f"(lse2[4 * c + 3])
                                 : "r"(stat + c * 16));
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(delta[4 * c]), "=f"(delta[4 * c + 1]), "=f"(delta[4 * c + 2]), "=f"(delta[4 * c + 3])
                                 : "r"(stat + kStatBytes + c * 16));
                }
                sm100::tmem_ld_wait();
                float pv[kPart], dsv[kPart];
                if (sub < 2 || it.key + (sub + 1) * kSub > it.e.count) {
                    // The diagonal, or queries behind the sequence's end: both tests select.
                    const int first_visible = sub < 2 ? key : 0;
#pragma unroll
                    for (int i = 0; i < kPart; ++i) {
                        const bool visible = first_visible <= query + i && query + i < it.e.count;
                        const float e = fast_exp2(fmaf(__uint_as_float(s_raw[i]), scale2, -lse2[i]));
                        pv[i] = visible ? e : 0.0f;
                        dsv[i] = visible ? e * (__uint_as_float(dp_raw[i]) - delta[i]) : 0.0f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kPart; i += 2) {
                        exp2_two(i / 2, fmaf(__uint_as_float(s_raw[i]), scale2, -lse2[i]),
                                 fmaf(__uint_as_float(s_raw[i + 1]), scale2, -lse2[i + 1]), pv[i], pv[i + 1]);
                        dsv[i] = pv[i] * (__uint_as_float(dp_raw[i]) - delta[i]);
                        dsv[i + 1] = pv[i + 1] * (__uint_as_float(dp_raw[i + 1]) - delta[i + 1]);
                    }
                }
                // P^T and dS^T go back over the first 8 of the 16 columns this thread read.
                uint32_t packed[8];
                pack_pairs(packed, pv);
                sm100::tmem_st_32x8(my_scores, packed);
                pack_pairs(packed, dsv);
                sm100::tmem_st_32x8(my_weights, packed);
                warp_arrive_after_stores(bar.operands_ready(count & 1), lane);
                sub = sub + 1 == it.subs ? 0 : sub + 1;
                ok = __all_sync(kFullMask, there);
            }
            before += it.steps;
            if (!ok) {
                break;
            }
            // The next item's K and V go in now, so that its first products run while this item's
            // gradients are written out.
            if (items.of(round + 1) >= 0 && !install(round + 1)) {
                ok = false;
                break;
            }
            if (!sm100::mbar_wait_warp(bar.done(), round & 1, abort)) {
                ok = false;
                break;
            }
            sm100::tc_fence_after_sync();
            uint32_t dv_raw[kPart], dk_raw[kPart];
            sm100::tmem_ld_32x16(tmem_dv + lane_base + part * kPart, dv_raw);
            sm100::tmem_ld_32x16(tmem_dk + lane_base + part * kPart, dk_raw);
            sm100::tmem_ld_wait();
            if (key < it.e.count && p.slices > 1) {
                const long long row_there = it.slice * static_cast<long long>(p.a.rows) + it.e.first + key;
                float* to = p.partial + ((row_there * p.a.kv_heads + it.head) * 2) * kHead + part * kPart;
#pragma unroll
                for (int c = 0; c < kPart; c += 4) {
                    *reinterpret_cast<uint4*>(to + c) = make_uint4(dk_raw[c], dk_raw[c + 1], dk_raw[c + 2], dk_raw[c + 3]);
                    *reinterpret_cast<uint4*>(to + kHead + c) =
                        make_uint4(dv_raw[c], dv_raw[c + 1], dv_raw[c + 2], dv_raw[c + 3]);
                }
            } else if (key < it.e.count) {
                const long long at = (it.e.first + static_cast<long long>(key)) * p.a.kv_stride + it.head * kHead +
                                     part * kPart;
#pragma unroll
                for (int c = 0; c < kPart / 8; ++c) {
                    float a[8], b[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        a[i] = __uint_as_float(dk_raw[c * 8 + i]) * p.a.scale;   // (dS was kept unscaled)
                        b[i] = __uint_as_float(dv_raw[c * 8 + i]);
                    }
                    *reinterpret_cast<uint4*>(p.g.dk + at + c * 8) = pack8(a);
                    *reinterpret_cast<uint4*>(p.g.dv + at + c * 8) = pack8(b);
                }
            }
            sm100::tc_fence_before_sync();
        }
    }
}

// ---- dQ ---------------------------------------------------------------------------------------------
//
// S = Q K^T and dP = dO V^T (A = Q, dO from tensor memory), dS written back over dP, dQ += dS K.
// Tensor memory: S at 0/64, dP at 128/192, dQ 256, Q 320, dO 352.

__device__ __forceinline__ void query_items(const BackwardParams& p, const Shared& shared, const Items& items) {
    const uint32_t q_tile = shared.base, do_tile = shared.base + kTileBytes;
    const uint32_t ring = shared.base + 2 * kTileBytes;           // stage: K then V
    const Barriers bar = shared.bar;
    volatile int* abort = shared.abort;
    const int warp = shared.warp;
    const int lane = threadIdx.x % 32;
    const uint32_t tmem = shared.tmem;
    auto tmem_s = [&](uint32_t count) { return tmem + 64u * (count & 1); };
    auto tmem_dp = [&](uint32_t count) { return tmem + 128u + 64u * (count & 1); };
    const uint32_t tmem_dq = tmem + 256, tmem_q = tmem + 320, tmem_do = tmem + 352;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            int round = 0;
            for (int item = items.take(0); ok && item >= 0; item = items.take(++round)) {
                const QueryItem it(p, item);
                if (round > 0 && !sm100::mbar_wait(bar.a_ready(), (round - 1) & 1, abort)) {
                    break;
                }
                sm100::mbar_expect_tx(bar.resident(), 2 * kTileBytes);
                for (int half = 0; half < 2; ++half) {
                    const int row = it.e.first + it.query + half * kSub;
                    sm100::tma_load_3d(q_tile + half * kSubBytes, &p.map_q, bar.resident(), 0, it.head, row);
                    sm100::tma_load_3d(do_tile + half * kSubBytes, &p.map_do, bar.resident(), 0, it.head, row);
                }
                const int kv_head = it.head / p.group;
                for (int step = 0; step < it.steps; ++step) {
                    if (!sm100::mbar_wait(bar.stage_empty(stage), phase ^ 1u, abort)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = ring + stage * 2 * kSubBytes, full = bar.stage_full(stage);
                    sm100::mbar_expect_tx(full, 2 * kSubBytes);
                    sm100::tma_load_3d(dst, &p.map_k, full, 0, kv_head, it.e.first + step * kSub);
                    sm100::tma_load_3d(dst + kSubBytes, &p.map_v, full, 0, kv_head, it.e.first + step * kSub);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        const uint64_t k_desc = sm100::smem_desc_sw128(ring, 16, 1024);
        const uint64_t v_desc = sm100::smem_desc_sw128(ring + kSubBytes, 16, 1024);
        uint32_t before = 0;
        bool ok = true;
        int round = 0;
        for (int item = items.of(0); ok && item >= 0; item = items.of(++round)) {
            const QueryItem it(p, item);
            ok = sm100::mbar_wait_warp(bar.a_ready(), round & 1, abort);
            sm100::tc_fence_after_sync();
            auto issue_scores = [&](int step) -> bool {
                const uint32_t count = before + step;
                const int stage = count % kStages;
                if (!sm100::mbar_wait_warp(bar.stage_full(stage), (count / kStages) & 1, abort)) {
                    return false;
                }
                sm100::tc_fence_after_sync();
                const int present = it.e.count - step * kSub;
                if (present < kSub) {
                    zero_rows(ring + stage * 2 * kSubBytes, present, lane);   // (V's rows meet dP's masked columns only)
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                const uint64_t k_sub = k_desc + stage * (2 * kSubBytes >> 4);
                const uint64_t v_sub = v_desc + stage * (2 * kSubBytes >> 4);
                if (sm100::elect_one()) {
                    const uint32_t s_at = tmem_s(count), dp_at = tmem_dp(count);
                    sm100::mma_f16_ts_at<0>(s_at, tmem_q, k_sub, 0, kIdescSub);
                    sm100::mma_f16_ts_at<1>(s_at, tmem_q + 8, k_sub, 2, kIdescSub);
                    sm100::mma_f16_ts_at<1>(s_at, tmem_q + 16, k_sub, 4, kIdescSub);
                    sm100::mma_f16_ts_at<1>(s_at, tmem_q + 24, k_sub, 6, kIdescSub);
                    sm100::mma_f16_ts_at<0>(dp_at, tmem_do, v_sub, 0, kIdescSub);
                    sm100::mma_f16_ts_at<1>(dp_at, tmem_do + 8, v_sub, 2, kIdescSub);
                    sm100::mma_f16_ts_at<1>(dp_at, tmem_do + 16, v_sub, 4, kIdescSub);
                    sm100::mma_f16_ts_at<1>(dp_at, tmem_do + 24, v_sub, 6, kIdescSub);
                    sm100::mma_commit(bar.scores_full(count & 1));
                }
                __syncwarp();
                return true;
            };
            ok = ok && issue_scores(0);
            for (int step = 0; ok && step < it.steps; ++step) {
                const uint32_t count = before + step;
                if (step + 1 < it.steps && !issue_scores(step + 1)) {
                    ok = false;
                    break;
                }
                if (!sm100::mbar_wait_warp(bar.operands_ready(count & 1), (count >> 1) & 1, abort)) {
                    ok = false;
                    break;
                }
                sm100::tc_fence_after_sync();
                const int stage = count % kStages;
                const uint64_t k_sub = k_desc + stage * (2 * kSubBytes >> 4);
                if (sm100::elect_one()) {
                    const uint32_t dp_at = tmem_dp(count);
                    sm100::mma_f16_ts_at<-1>(tmem_dq, dp_at, k_sub, 0, kIdescOut, step != 0);
                    sm100::mma_f16_ts_at<1>(tmem_dq, dp_at + 16, k_sub, 128, kIdescOut);
                    sm100::mma_f16_ts_at<1>(tmem_dq, dp_at + 32, k_sub, 256, kIdescOut);
                    sm100::mma_f16_ts_at<1>(tmem_dq, dp_at + 48, k_sub, 384, kIdescOut);
                    sm100::mma_commit(bar.stage_empty(stage));
                    if (step + 1 == it.steps) {
                        sm100::mma_commit(bar.done());
                    }
                }
                __syncwarp();
            }
            before += it.steps;
        }
    } else {
        const int quadrant = warp % 4;
        const int part = (warp - 2) / 4;               // which 16 of the 64 key columns
        const int row = quadrant * 32 + lane;          // query row in the block
        const uint32_t lane_base = static_cast<uint32_t>(quadrant * 32) << 16;
        const float scale2 = p.a.scale * kLog2e;
        auto install = [&](int round) -> bool {
            if (!sm100::mbar_wait_warp(bar.resident(), round & 1, abort)) {
                return false;
            }
            tile_row_to_tmem(tmem_q + lane_base, q_tile, row, part);
            tile_row_to_tmem(tmem_do + lane_base, do_tile, row, part);
            warp_arrive_after_stores(bar.a_ready(), lane);
            return true;
        };
        uint32_t before = 0;
        int round = 0;
        int item = items.of(0);
        bool ok = item >= 0 && install(0);
        for (; ok && item >= 0; item = items.of(++round)) {
            const QueryItem it(p, item);
            const int query = it.query + row;
            const bool valid = query < it.e.count;
            float lse2 = INFINITY, delta = 0.0f;
            if (valid) {
                const long long at = it.head * p.stats_stride + it.e.stats + query;
                lse2 = p.lse2[at];
                delta = p.delta[at];
            }
            for (int step = 0; ok && step < it.steps; ++step) {
                const uint32_t count = before + step;
                const bool there = sm100::mbar_wait(bar.scores_full(count & 1), (count >> 1) & 1, abort);
                sm100::tc_fence_after_sync();
                const uint32_t my_weights = tmem_dp(count) + lane_base + part * kPart;
                uint32_t s_raw[kPart], dp_raw[kPart];
                sm100::tmem_ld_32x16(tmem_s(count) + lane_base + part * kPart, s_raw);
                sm100::tmem_ld_32x16(my_weights, dp_raw);
                sm100::tmem_ld_wait();
                const int key = step * kSub + part * kPart;    // first one of my columns
                float dsv[kPart];
                if ((step + 1) * kSub > it.query) {
                    // The diagonal: keys after the query are masked.
#pragma unroll
                    for (int i = 0; i < kPart; ++i) {
                        const float e = fast_exp2(fmaf(__uint_as_float(s_raw[i]), scale2, -lse2));
                        dsv[i] = key + i <= query ? e * (__uint_as_float(dp_raw[i]) - delta) : 0.0f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kPart; i += 2) {
                        float e0, e1;
                        exp2_two(i / 2, fmaf(__uint_as_float(s_raw[i]), scale2, -lse2),
                                 fmaf(__uint_as_float(s_raw[i + 1]), scale2, -lse2), e0, e1);
                        dsv[i] = e0 * (__uint_as_float(dp_raw[i]) - delta);
                        dsv[i + 1] = e1 * (__uint_as_float(dp_raw[i + 1]) - delta);
                    }
                }
                uint32_t packed[8];
                pack_pairs(packed, dsv);
                sm100::tmem_st_32x8(my_weights, packed);
                warp_arrive_after_stores(bar.operands_ready(count & 1), lane);
                ok = __all_sync(kFullMask, there);
            }
            before += it.steps;
            if (!ok) {
                break;
            }
            if (items.of(round + 1) >= 0 && !install(round + 1)) {
                ok = false;
                break;
            }
            if (!sm100::mbar_wait_warp(bar.done(), round & 1, abort)) {
                ok = false;
                break;
            }
            sm100::tc_fence_after_sync();
            uint32_t raw[kPart];
            sm100::tmem_ld_32x16(tmem_dq + lane_base + part * kPart, raw);
            sm100::tmem_ld_wait();
            if (valid) {
                __half* out = p.g.dq + (it.e.first + static_cast<long long>(query)) * p.a.q_stride + it.head * kHead +
                              part * kPart;
#pragma unroll
                for (int c = 0; c < kPart / 8; ++c) {
                    float a[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        a[i] = __uint_as_float(raw[c * 8 + i]) * p.a.scale;
                    }
                    *reinterpret_cast<uint4*>(out + c * 8) = pack8(a);
                }
            }
            sm100::tc_fence_before_sync();
        }
    }
}

__global__ void __launch_bounds__(kThreads, 1) fb_packed_backward(const __grid_constant__ BackwardParams p) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
    const Barriers bar{base + kUsed - 1024 - 256};
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ int ring[kItems];
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x / 32), 0);
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < kItems; ++i) {
            sm100::mbar_init(bar.item_full(i), 1);
        }
        sm100::mbar_init(bar.resident(), 1);
        sm100::mbar_init(bar.done(), 1);
        sm100::mbar_init(bar.a_ready(), kComputeWarps);
        for (int i = 0; i < 2; ++i) {
            sm100::mbar_init(bar.scores_full(i), 1);
            sm100::mbar_init(bar.operands_ready(i), kComputeWarps);
        }
        for (int s = 0; s < kStages; ++s) {
            sm100::mbar_init(bar.stage_full(s), 1);
            sm100::mbar_init(bar.stage_empty(s), 1);
        }
        sm100::mbar_fence_init();
    }
    if (warp == 1) {
        sm100::tmem_alloc(sm100::smem_u32(&tmem_slot), 512);
    }
    sm100::tc_fence_before_sync();
    __syncthreads();
    sm100::tc_fence_after_sync();
    const Shared shared{base, bar, tmem_slot, &abort_flag, warp};
    dependency_wait();

    // Both gradients have as many sub-steps; dK's and dV's take longer, which sets their share of the CTAs.
    const int count = *static_cast<volatile int*>(p.counts);
    const int cta = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
    const int key_count = count * p.a.kv_heads * p.slices;
    const int share = min(key_count, max(1, static_cast<int>(ctas * kKeyShare + 0.5)));
    if (cta < share) {
        key_items(p, shared, Items{p.counts + 1, key_count, ring, bar, &abort_flag});
    } else {
        query_items(p, shared, Items{p.counts + 2, count * p.a.heads, ring, bar, &abort_flag});
    }
    if (threadIdx.x == 0) {
        dependency_release();
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
        sm100::tmem_dealloc(tmem_slot, 512);
    }
}

// ---- the third launch, where groups were divided -----------------------------------------------------

// Eight values of dK or dV per thread, the slices in order.
__global__ void __launch_bounds__(256) fb_packed_backward_join(const BackwardParams p) {
    dependency_wait();
    dependency_release();
    const float4* partial = reinterpret_cast<const float4*>(after_wait(static_cast<const float*>(p.partial)));
    const int first = max(p.a.starts[0], 0), end = min(p.a.starts[p.a.sequences], p.a.rows);
    const long long per_row = static_cast<long long>(p.a.kv_heads) * 16;     // 16-byte pieces of dK and dV
    const long long slice = static_cast<long long>(p.a.rows) * p.a.kv_heads * 2 * kHead / 4;   // in words of four values
    for (long long i = first * per_row + blockIdx.x * 256ll + threadIdx.x; i < end * per_row; i += gridDim.x * 256ll) {
        float sum[8] = {};
        for (int s = 0; s < p.slices; ++s) {
            float v[8];
            load8_input(v, partial + s * slice + i * 2);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                sum[c] += v[c];
            }
        }
        const long long row = i / per_row;
        const int rest = static_cast<int>(i - row * per_row);
        const int head = rest / 16, which = rest / 8 % 2, piece = rest % 8;
        if (which == 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                sum[c] *= p.a.scale;
            }
        }
        *reinterpret_cast<uint4*>((which == 0 ? p.g.dk : p.g.dv) + row * p.a.kv_stride + head * kHead + piece * 8) = pack8(sum);
    }
}

// ---- host ---------------------------------------------------------------------------------------------

constexpr int kMostSlices = 8;

// Into how many items a group's heads are divided: until there are about two (block, K/V head) items for every CTA that
// works on dK and dV. 8 heads on 1, two sequences of up to 1,500 tokens: 132 -> 29 us.
int slices_of(size_t rows, size_t heads, size_t kv_heads, int sms) {
    const size_t items = std::max<size_t>(1, rows / kBlock) * kv_heads;
    const size_t wanted = (static_cast<size_t>(sms) + items - 1) / items;
    return static_cast<int>(std::max<size_t>(1, std::min({wanted, heads / kv_heads, size_t{kMostSlices}})));
}

struct Layout {
    size_t count, entries, lse2, delta, partial, bytes;   // offsets
    long long stride;
    int capacity, slices;
};

Layout layout_of(size_t sequences, size_t rows, size_t heads, size_t kv_heads, int sms) {
    auto up = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    Layout l;
    // A sub-step's copy takes 64 values from a multiple of 64 behind a sequence's beginning.
    l.stride = static_cast<long long>((rows + 4 * sequences + kSub + 3) / 4 * 4);
    l.capacity = static_cast<int>(rows / kBlock + sequences + 1);
    l.count = 0;
    l.entries = 256;
    l.lse2 = l.entries + up(l.capacity * sizeof(Entry));
    l.delta = l.lse2 + up(heads * l.stride * sizeof(float));
    l.partial = l.delta + up(heads * l.stride * sizeof(float));
    l.slices = slices_of(rows, heads, kv_heads, sms);
    l.bytes = l.partial + (l.slices > 1 ? l.slices * rows * kv_heads * 2 * kHead * sizeof(float) : 0);
    return l;
}

}  // namespace

cudaError_t packed_backward_error_flag(int* value, bool reset) { return read_error_word(value, reset); }

cudaError_t packed_backward_workspace(size_t sequences, size_t rows, size_t heads, size_t kv_heads, size_t* bytes) {
    int sms = 148;
    const cudaError_t e = sm_count(&sms);
    *bytes = layout_of(sequences, rows, heads, kv_heads, sms).bytes;
    return e;
}

cudaError_t packed_backward(const PackedArgs& args, const PackedGradients& gradients, void* workspace,
                            cudaStream_t stream) {
    BackwardParams p;
    std::memset(&p, 0, sizeof p);
    cudaError_t e = encode_rows(&p.map_q, args.q, args.heads, args.rows, args.q_stride, 1, kSub);
    if (e == cudaSuccess) e = encode_rows(&p.map_k, args.k, args.kv_heads, args.rows, args.kv_stride, 1, kSub);
    if (e == cudaSuccess) e = encode_rows(&p.map_v, args.v, args.kv_heads, args.rows, args.kv_stride, 1, kSub);
    if (e == cudaSuccess) e = encode_rows(&p.map_do, gradients.d_o, args.heads, args.rows, args.o_stride, 1, kSub);
    int sms = 148;
    if (e == cudaSuccess) e = sm_count(&sms);
    if (e != cudaSuccess) {
        return e;
    }
    const Layout l = layout_of(args.sequences, args.rows, args.heads, args.kv_heads, sms);
    char* at = static_cast<char*>(workspace);
    PrepareParams prepare = {args, gradients.d_o, reinterpret_cast<Entry*>(at + l.entries),
                             reinterpret_cast<int*>(at + l.count), reinterpret_cast<float*>(at + l.lse2),
                             reinterpret_cast<float*>(at + l.delta), l.stride, l.capacity};
    const unsigned blocks = static_cast<unsigned>(std::min((args.rows + 7) / 8, 8 * sms)) + 1;
    e = launch_dependent(fb_packed_backward_prepare, dim3(blocks), dim3(kListThreads), 0, stream, prepare);
    if (e != cudaSuccess) {
        return e;
    }
    p.a = args;
    p.g = gradients;
    p.entries = prepare.entries;
    p.counts = prepare.counts;
    p.lse2 = prepare.lse2;
    p.delta = prepare.delta;
    p.stats_stride = l.stride;
    p.group = args.heads / args.kv_heads;
    static std::atomic<bool> configured[64] = {};
    e = allow_shared_memory(fb_packed_backward, kSmem, configured);
    if (e != cudaSuccess) {
        return e;
    }
    p.slices = l.slices;
    p.partial = reinterpret_cast<float*>(at + l.partial);
    e = launch_dependent(fb_packed_backward, dim3(static_cast<unsigned>(std::max(2, sms))), dim3(kThreads), kSmem, stream,
                         p);
    if (e != cudaSuccess || l.slices == 1) {
        return e;
    }
    const long long pieces = static_cast<long long>(args.rows) * args.kv_heads * 16;
    return launch_dependent(fb_packed_backward_join,
                            dim3(static_cast<unsigned>(std::min<long long>((pieces + 255) / 256, 8LL * sms))), dim3(256), 0,
                            stream, p);
}

}  // namespace fb
