// A paged cache of 8 bits (int8 codes, an FP32 scale for each block of 16 positions of a head): storing new tokens, and their
// attention over it while they are few.
//
// With b the block of key j:  t_j = (q . k_j) s_b + log2 w_b  (k_j the codes, s_b K's scale times `scale` and log2 e, w_b V's
// scale),  P_j = 2^(t_j - m),  O = sum P_j v_j over V's codes,  l = sum_b (sum_j P_j) / w_b,  o = O / l. Both scales thus
// cost one multiplication and addition per score and one per block and row; codes are exact in FP16, so the products take
// them as they are, and P_j, rounded to FP16 for the second one, stays below 2^8 whatever V's scales are.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>

#include <cuda_fp16.h>

#include "common.h"
#include "device_utils.cuh"
#include "packed.cuh"
#include "packed_codes.cuh"
#include "packed_locate.cuh"
#include "sm100.cuh"
#include "softmax.cuh"

namespace fb {
namespace {

constexpr int kHead = 64;
constexpr int kBlock = 16;      // positions that share a scale
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ---- storing ------------------------------------------------------------------------------------------

// A warp stores one block of one head of K or V: its lanes take 8 values of 4 rows at a time. Bound by three loads one behind the
// other (lengths, a page's number, the block's scale) and the launch: one token of 1 or 64 sequences 3.0 and 3.5 us, four chunks of 512 tokens and
// two single ones, 4 heads, 7.2 us.
__global__ void __launch_bounds__(256) fb_paged8_store(const PackedArgs p, const Cache8 cache) {
    dependency_wait();
    dependency_release();
    const int lane = threadIdx.x % 32, piece = lane % 8, of_four = lane / 8;
    const long long first = static_cast<long long>(blockIdx.x) * 8 + threadIdx.x / 32;
    const long long stride = static_cast<long long>(gridDim.x) * 8;
    for (int s = blockIdx.y; s < p.sequences; s += gridDim.y) {
        const Sequence q = sequence_at(p, s);
        const int begins = q.keys - q.count;       // position of the first new token, which may be negative
        const int low = max(begins, 0) / kBlock;
        const int blocks = q.keys > max(begins, 0) && q.count > 0 ? (q.keys - 1) / kBlock - low + 1 : 0;
        for (long long item = first; item < static_cast<long long>(blocks) * p.kv_heads * 2; item += stride) {
            const int which = static_cast<int>(item % 2);
            const int head = static_cast<int>(item / 2 % p.kv_heads);
            const int key = (low + static_cast<int>(item / 2 / p.kv_heads)) * kBlock;      // the block's first
            const __half* from = (which == 0 ? p.k : p.v) + head * kHead;
            // What the steps below need is asked for at once: the new rows beside the page's number, what the block holds
            // beside its scale.
            uint4 held[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = key + 4 * r + of_four - begins;      // of the new tokens
                held[r] = make_uint4(0u, 0u, 0u, 0u);
                if (i >= 0 && i < q.count) {
                    held[r] = reinterpret_cast<const uint4*>(from + (q.first + static_cast<long long>(i)) * p.kv_stride)[piece];
                }
            }
            const long long page = page_of(p, s, key);
            if (page < 0) {
                continue;
            }
            const long long row = (page * p.kv_heads + head) * p.page_size + key % p.page_size;
            int8_t* codes = (which == 0 ? cache.k : cache.v) + row * kHead;
            float* scale_at = (which == 0 ? cache.k_scales : cache.v_scales) + row / kBlock;
            const bool kept = begins > key;
            const float before = kept ? *scale_at : 0.0f;
            uint2 old[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                old[r] = make_uint2(0u, 0u);
                if (key + 4 * r + of_four < begins) {
                    old[r] = reinterpret_cast<const uint2*>(codes + (4 * r + of_four) * kHead)[piece];
                }
            }
            float largest = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v[8];
                unpack8(v, held[r]);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    largest = max_nan(largest, fabsf(v[c]));
                }
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) {
                largest = max_nan(largest, __shfl_xor_sync(kFullMask, largest, off));
            }
            // (An infinity counts as NaN.)
            float scale = largest <= 65504.0f ? __fdiv_rn(largest, 127.0f) : __int_as_float(0x7fffffff);
            scale = kept ? max_nan(before, scale) : scale;
            const bool grows = kept && scale != before;     // (a NaN grows: codes of it are 0)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = key + 4 * r + of_four - begins;
                const bool fresh = i >= 0 && i < q.count;
                uint2* to = reinterpret_cast<uint2*>(codes + (4 * r + of_four) * kHead) + piece;
                if (!fresh && !(grows && i < 0)) {
                    continue;
                }
                float v[8];
                if (fresh) {
                    unpack8(v, held[r]);
                } else {
                    const unsigned w[2] = {old[r].x, old[r].y};
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        v[c] = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[c / 4] >> (8 * (c % 4)))), before);
                    }
                }
                unsigned w[2] = {0u, 0u};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    // At most 127 in size: |v| <= 127 scale but for roundings, which a half step holds.
                    const int code = scale > 0.0f ? __float2int_rn(__fdiv_rn(v[c], scale)) : 0;
                    w[c / 4] |= (static_cast<unsigned>(code) & 0xffu) << (8 * (c % 4));
                }
                *to = make_uint2(w[0], w[1]);
            }
            __syncwarp();      // (everybody has the scale before)
            if (lane == 0) {
                *scale_at = scale;
            }
        }
    }
}

// ---- attention of few rows ------------------------------------------------------------------------------

// Bound by what it reads and by what turning codes into FP16 takes, so a warp's own product is the right one: mma.sync takes codes
// that a lane has just turned into FP16 in its registers, where the tensor cores' larger instruction would want
// them written to shared memory first. Keys are the products' rows and queries their columns, eight of them to a
// product: S^T = K Q^T, O^T = V^T P^T. With 16 rows of queries instead, a group of four heads would leave three quarters of the
// exponentials to nobody. A tile (packed_schedule.h) has up to 8 kTiles rows; a warp takes every eighth unit of one or two blocks of 16
// keys, whose codes come to it alone through stages of asynchronous copies, and the warps' sums meet at the end of a piece. (Two blocks
// at a time where registers allow: one's products run under the other's conversions.)
// Measured with the join, as part of a graph: one sequence of 1,000 keys, 12 heads, 7.8 us; 64 sequences of up to 8,192, 32 heads on 8, 48 us (196 MB,
// 4.1 TB/s). There no pipe is full (47 % of the issue slots, DRAM 51 %, the tensor pipe 18 %): sixteen warps on an SM, each a chain
// of copies, conversions and two products, and the pieces' uneven ends, at which the warps wait for each other.
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBlockBytes = 2 * kBlock * kHead;       // K and V of a block
constexpr int kMergeStride = kHead + 4;               // floats between rows that meet

struct FewParams {
    PackedArgs a;
    Cache8 cache;
    Record* records;
    float* parts;
    int group, log_tokens, log_page;
    bool splits;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The transpose of 8 x 8 values of 16 bits, a row to four lanes.
__device__ __forceinline__ unsigned transposed(unsigned x) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

constexpr int kFewPerSm = 2;     // CTAs on an SM (registers)

template <int kTiles>
struct FewMemory {
    static constexpr int kRows = 8 * kTiles;
    static constexpr int kUnit = kTiles == 1 ? 2 : 1;        // blocks at a time
    static constexpr int kStages = kUnit == 2 ? 3 : 5;
    union {      // a warp's
        unsigned char ring[kStages][kUnit][kBlockBytes];
        float merge[kRows][kMergeStride];       // (at the end of a piece)
    } of[kWarps];
    float merge_max[kWarps][kRows], merge_sum[kWarps][kRows];
    Cut cuts[2];
    long long scan[kWarps + 1];
    int scan_longest[kWarps];
    int whole_tiles;
};

template <int kTiles>
__global__ void __launch_bounds__(kThreads, kFewPerSm) fb_paged8_few(const __grid_constant__ FewParams p) {
    using Memory = FewMemory<kTiles>;
    constexpr int kUnit = Memory::kUnit, kStages = Memory::kStages;
    constexpr int kBatch = 32 / kUnit;           // units whose places the lanes hold
    constexpr int kUnitKeys = kUnit * kBlock;
    extern __shared__ __align__(128) unsigned char memory[];
    Memory& shared = *reinterpret_cast<Memory*>(memory);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x / 32), 0), lane = threadIdx.x % 32;
    const int g = lane / 4, t = lane % 4;        // row and column of the products' fragments
    dependency_wait();
    if (p.a.sequences > 128) {
        locate<false, kThreads>(p, shared.cuts, shared.whole_tiles, shared.scan, shared.scan_longest);
    } else if (warp == 0) {
        if (p.a.sequences > 32) {
            locate_runs_in_warp<4>(p, shared.cuts, lane);
        } else {
            locate_in_warp<false>(p, shared.cuts, shared.whole_tiles, lane);
        }
    }
    __syncthreads();
    dependency_release();
    if (threadIdx.x == 0) {
        p.records[blockIdx.x] = make_record(SequenceOf{p.a}, p.log_tokens, shared.cuts[0], shared.cuts[1]);
    }
    const unsigned char* stages = &shared.of[warp].ring[0][0][0];
    const uint32_t stages_at = sm100::smem_u32(stages);
    const float scale2 = p.a.scale * kLog2e;
    Walk walk;
    Piece piece;
    walk.begin(SequenceOf{p.a}, shared.cuts[0], shared.cuts[1].at);
    while (walk.next(SequenceOf{p.a}, p.a.sequences, p.a.kv_heads, p.log_tokens, piece)) {
        const int first_position = piece.position();
        const int first_block = piece.from * (kKeyTile / kBlock);
        const int blocks = min(piece.to * (kKeyTile / kBlock), (piece.sequence.keys + kBlock - 1) / kBlock) - first_block;
        const int rows = piece.tokens * p.group;
        const int tiles = (rows + 7) / 8;        // of eight rows
        // This warp's units: warp + 8 i.
        const int count = max(0, ((blocks + kUnit - 1) / kUnit - warp + kWarps - 1) / kWarps);
        // Lane i has the place of the i-th block of a batch (the row of its first key in the cache, -1 for none) and what its
        // scales come to.
        auto place_of = [&](int i) {
            const int block = (warp + i / kUnit * kWarps) * kUnit + i % kUnit;
            if (block >= blocks) {
                return -1;
            }
            const int key = (first_block + block) * kBlock;
            const long long page = page_of(p.a, piece.index, key);
            return page < 0 ? -1
                            : static_cast<int>((page * p.a.kv_heads + piece.head) << p.log_page) + (key & (p.a.page_size - 1));
        };
        int place_next = place_of(lane), place = -1;
        float k_next = 0.0f, v_next = 0.0f, slope_of = 0.0f, offset_of = 0.0f, inverse_of = 0.0f;
        auto fetch = [&](int i, int stage) {
            if (i < count) {
                if (i % kBatch == 0) {
                    place = place_next;
                    k_next = v_next = 0.0f;
                    if (place >= 0) {
                        k_next = p.cache.k_scales[place / kBlock];
                        v_next = p.cache.v_scales[place / kBlock];
                    }
                    place_next = place_of(i * kUnit + 32 + lane);
                }
#pragma unroll
                for (int b = 0; b < kUnit; ++b) {
                    const int from = __shfl_sync(kFullMask, place, i % kBatch * kUnit + b);
                    const uint32_t to = stages_at + (stage * kUnit + b) * kBlockBytes + lane * 16;
                    const unsigned bytes = from >= 0 ? 16u : 0u;       // zeros for a page that is not there
                    const long long at = static_cast<long long>(max(from, 0)) * kHead + lane * 16;
                    const int8_t* k = p.cache.k + at;
                    const int8_t* v = p.cache.v + at;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(k), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 512), "l"(k + 512), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 1024), "l"(v), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 1536), "l"(v + 512), "r"(bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            fetch(i, i);
        }
        // Queries as they are multiplied: of eight rows, lane (g, t) has the 16 values from 16 t on of row g, four of
        // which are a product's term with the four codes that lie beside each other in a key. Its scores are of rows 2 t and
        // 2 t + 1, whose positions it has.
        uint4 query[kTiles][2];
        int position[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int row = 8 * n + g, token = row / p.group;
            query[n][0] = query[n][1] = make_uint4(0u, 0u, 0u, 0u);
            if (row < rows) {
                const __half* from = p.a.q + (static_cast<long long>(piece.sequence.first) + piece.first_token + token) * p.a.q_stride +
                                     (piece.head * p.group + row - token * p.group) * kHead + 16 * t;
                query[n][0] = reinterpret_cast<const uint4*>(from)[0];
                query[n][1] = reinterpret_cast<const uint4*>(from)[1];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                position[n][c] = 8 * n + 2 * t + c < rows ? first_position + (8 * n + 2 * t + c) / p.group : -1;
            }
        }
        float m[kTiles][2], l[kTiles][2];
        float out[kTiles][4][4];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            m[n][0] = m[n][1] = kNoKey;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                out[n][j][0] = out[n][j][1] = out[n][j][2] = out[n][j][3] = 0.0f;
            }
        }
        // Of the products' rows the even ones are keys 0 to 3 and the odd ones 4 to 7, and so on: V's are then read four in
        // a row at a time below.
        const int low = (g & 1) * 4 + (g >> 1);      // key of the product's row g; 8 more for row g + 8
        int stage = 0;
        for (int i = 0; i < count; ++i) {
            if (i % kBatch == 0) {
                const float v = v_next == 0.0f ? kWeightOfZeros : v_next;
                slope_of = k_next * scale2;
                offset_of = __log2f(v);
                inverse_of = 1.0f / v;
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();       // everybody's copies have landed, and the stage before is read
            fetch(i + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
            const unsigned char* codes = stages + stage * (kUnit * kBlockBytes);
            const int key = first_block * kBlock + (warp + i * kWarps) * kUnitKeys;
            const bool masked = key + kUnitKeys - 1 > first_position;
            float slope[kUnit], offset[kUnit], inverse[kUnit];
            float scores[kTiles][kUnit][4];
#pragma unroll
            for (int b = 0; b < kUnit; ++b) {
                const int of = i % kBatch * kUnit + b;
                slope[b] = __shfl_sync(kFullMask, slope_of, of);
                offset[b] = __shfl_sync(kFullMask, offset_of, of);
                inverse[b] = __shfl_sync(kFullMask, inverse_of, of);
                const unsigned char* k = codes + b * kBlockBytes;
                const uint4 first = *reinterpret_cast<const uint4*>(k + low * kHead + 16 * t);
                const uint4 second = *reinterpret_cast<const uint4*>(k + (8 + low) * kHead + 16 * t);
                const unsigned x[4] = {first.x ^ 0x80808080u, first.y ^ 0x80808080u, first.z ^ 0x80808080u, first.w ^ 0x80808080u};
                const unsigned y[4] = {second.x ^ 0x80808080u, second.y ^ 0x80808080u, second.z ^ 0x80808080u,
                                       second.w ^ 0x80808080u};
                unsigned keys[4][4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    keys[s][0] = two_codes<0>(x[s]);
                    keys[s][1] = two_codes<0>(y[s]);
                    keys[s][2] = two_codes<2>(x[s]);
                    keys[s][3] = two_codes<2>(y[s]);
                }
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    scores[n][b][0] = scores[n][b][1] = scores[n][b][2] = scores[n][b][3] = 0.0f;
                    if (kTiles == 1 || n < tiles) {
                        mma_16816(scores[n][b], keys[0], query[n][0].x, query[n][0].y);
                        mma_16816(scores[n][b], keys[1], query[n][0].z, query[n][0].w);
                        mma_16816(scores[n][b], keys[2], query[n][1].x, query[n][1].y);
                        mma_16816(scores[n][b], keys[3], query[n][1].z, query[n][1].w);
                    }
                }
            }
            unsigned values[kUnit][4][4];    // of the products with V: rows g and g + 8 are columns 8 g + 2 j and 8 g + 2 j + 1
#pragma unroll
            for (int b = 0; b < kUnit; ++b) {
                uint2 read[4];               // keys t, t + 4, t + 8 and t + 12
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    read[k] = *reinterpret_cast<const uint2*>(codes + b * kBlockBytes + kBlock * kHead + (4 * k + t) * kHead + 8 * g);
                    read[k].x ^= 0x80808080u;
                    read[k].y ^= 0x80808080u;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // Two columns of two keys side by side.
                    const unsigned first = j < 2 ? __byte_perm(read[0].x, read[1].x, j % 2 == 0 ? 0x5140 : 0x7362)
                                                 : __byte_perm(read[0].y, read[1].y, j % 2 == 0 ? 0x5140 : 0x7362);
                    const unsigned second = j < 2 ? __byte_perm(read[2].x, read[3].x, j % 2 == 0 ? 0x5140 : 0x7362)
                                                  : __byte_perm(read[2].y, read[3].y, j % 2 == 0 ? 0x5140 : 0x7362);
                    values[b][j][0] = two_codes<0>(first);
                    values[b][j][1] = two_codes<2>(first);
                    values[b][j][2] = two_codes<0>(second);
                    values[b][j][3] = two_codes<2>(second);
                }
            }
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                if (kTiles > 1 && n >= tiles) {
                    break;
                }
                // Lane (g, t) has keys `low` and low + 8 of each block, of rows 2 t and 2 t + 1.
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int b = 0; b < kUnit; ++b) {
                    float (&x)[4] = scores[n][b];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        x[c] = fmaf(x[c], slope[b], offset[b]);
                    }
                    if (masked) {
                        const int here = key + b * kBlock + low;
                        x[0] = here <= position[n][0] ? x[0] : -INFINITY;
                        x[1] = here <= position[n][1] ? x[1] : -INFINITY;
                        x[2] = here + 8 <= position[n][0] ? x[2] : -INFINITY;
                        x[3] = here + 8 <= position[n][1] ? x[3] : -INFINITY;
                    }
                    top[0] = max_nan(top[0], max_nan(x[0], x[2]));
                    top[1] = max_nan(top[1], max_nan(x[1], x[3]));
                }
                if (__any_sync(kFullMask, !(top[0] - m[n][0] <= kLazyShift) || !(top[1] - m[n][1] <= kLazyShift))) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        top[c] = max_nan(top[c], __shfl_xor_sync(kFullMask, top[c], 4));
                        top[c] = max_nan(top[c], __shfl_xor_sync(kFullMask, top[c], 8));
                        top[c] = max_nan(top[c], __shfl_xor_sync(kFullMask, top[c], 16));
                        const float next = max_nan(m[n][c], top[c]);
                        const float alpha = fast_exp2(m[n][c] - next);
                        m[n][c] = next;
                        l[n][c] *= alpha;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            out[n][j][c] *= alpha;
                            out[n][j][2 + c] *= alpha;
                        }
                    }
                }
#pragma unroll
                for (int b = 0; b < kUnit; ++b) {
                    float (&x)[4] = scores[n][b];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        x[c] = fast_exp2(x[c] - m[n][c % 2]);
                    }
                    const float sum0 = x[0] + x[2], sum1 = x[1] + x[3];
                    // (A row that sees nothing of the block has nothing to do with its scale, whatever that is.)
                    l[n][0] = fmaf(sum0, masked && sum0 == 0.0f ? 0.0f : inverse[b], l[n][0]);
                    l[n][1] = fmaf(sum1, masked && sum1 == 0.0f ? 0.0f : inverse[b], l[n][1]);
                    // Probabilities go into the product in two parts, FP16 and what that leaves: with the first alone results are
                    // off by half as much again as their own rounding (sqrt 2 times it), and 64 single tokens take 52.2 us instead of 54.0.
                    unsigned part[2][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const unsigned first = pack2(x[2 * h], x[2 * h + 1]);
                        const float2 is = __half22float2(*reinterpret_cast<const __half2*>(&first));
                        part[h][0] = transposed(first);
                        part[h][1] = transposed(pack2(x[2 * h] - is.x, x[2 * h + 1] - is.y));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma_16816(out[n][j], values[b][j], part[0][0], part[1][0]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma_16816(out[n][j], values[b][j], part[0][1], part[1][1]);
                    }
                }
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();          // this warp's part of the ring is read
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            if (n < tiles) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int row = 8 * n + 2 * t + c;
                    l[n][c] += __shfl_xor_sync(kFullMask, l[n][c], 4);
                    l[n][c] += __shfl_xor_sync(kFullMask, l[n][c], 8);
                    l[n][c] += __shfl_xor_sync(kFullMask, l[n][c], 16);
                    if (g == 0) {
                        shared.merge_max[warp][row] = m[n][c];
                        shared.merge_sum[warp][row] = l[n][c];
                    }
                    // Column 8 g + 2 j of the row is out[j][c], column 8 g + 2 j + 1 out[j][2 + c].
                    float4* to = reinterpret_cast<float4*>(&shared.of[warp].merge[row][8 * g]);
                    to[0] = make_float4(out[n][0][c], out[n][0][2 + c], out[n][1][c], out[n][1][2 + c]);
                    to[1] = make_float4(out[n][2][c], out[n][2][2 + c], out[n][3][c], out[n][3][2 + c]);
                }
            }
        }
        __syncthreads();
        const bool whole = piece.from == 0 && piece.to == piece.tiles;
        for (int row = threadIdx.x / 16; row < rows; row += kThreads / 16) {
            const int column = threadIdx.x % 16 * 4;
            float all = kNoKey;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                all = max_nan(all, shared.merge_max[w][row]);
            }
            float total = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float top = shared.merge_max[w][row], factor = fast_exp2(top - all);
                const float4 x = *reinterpret_cast<const float4*>(&shared.of[w].merge[row][column]);
                if (top != kNoKey) {
                    total = fmaf(shared.merge_sum[w][row], factor, total);
                    sum.x = fmaf(x.x, factor, sum.x);
                    sum.y = fmaf(x.y, factor, sum.y);
                    sum.z = fmaf(x.z, factor, sum.z);
                    sum.w = fmaf(x.w, factor, sum.w);
                }
            }
            const int token = row / p.group, head = piece.head * p.group + row - token * p.group;
            const long long out_row = static_cast<long long>(piece.sequence.first) + piece.first_token + token;
            if (whole) {
                const bool none = first_position + token < 0;       // no key at all gives zeros
                const float inv = none ? 0.0f : 1.0f / total;
                *reinterpret_cast<uint2*>(p.a.o + out_row * p.a.o_stride + head * kHead + column) =
                    none ? make_uint2(0u, 0u) : make_uint2(pack2(sum.x * inv, sum.y * inv), pack2(sum.z * inv, sum.w * inv));
                if (column == 0 && p.a.lse != nullptr) {
                    p.a.lse[static_cast<long long>(head) * p.a.rows + out_row] =
                        none ? -INFINITY : (all + log2f(total)) * kLn2;
                }
            } else {
                float* part = p.parts + (2 * size_t{blockIdx.x} + (piece.from == 0 ? 1 : 0)) * kPartFloats;
                *reinterpret_cast<float4*>(part + (column / 4 * 128 + row) * 4) = sum;
                if (column == 0) {
                    part[128 * kHead + row] = all;
                    part[128 * kHead + 128 + row] = total;
                }
            }
        }
        __syncthreads();       // the rings are the copies' again
    }
}

template <int kTiles>
cudaError_t launch_few(FewParams p, int sms, void* workspace, long long most_keys, cudaStream_t stream) {
    const int ctas = std::min(kFewPerSm * sms, kMostPackedCtas);
    p.records = packed_records(workspace);
    p.parts = packed_parts(workspace, ctas);
    p.splits = most_keys > 1024;
    constexpr int kBytes = sizeof(FewMemory<kTiles>);
    while ((2 << p.log_tokens) * p.group <= FewMemory<kTiles>::kRows) {
        ++p.log_tokens;
    }
    static std::atomic<bool> configured[64] = {};
    cudaError_t e = allow_shared_memory(fb_paged8_few<kTiles>, kBytes, configured);
    if (e == cudaSuccess) {
        e = launch_dependent(fb_paged8_few<kTiles>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kBytes, stream, p);
    }
    if (e != cudaSuccess || !p.splits) {
        return e;
    }
    return packed_join(p.a, p.records, p.parts, ctas, most_keys, stream);
}

}  // namespace

cudaError_t paged8_error_flag(int* value, bool reset) { return read_error_word(value, reset); }

cudaError_t paged8_store(const PackedArgs& args, const Cache8& cache, cudaStream_t stream) {
    int sms = 148;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) {
        return e;
    }
    // Blocks of 16 tokens, one more than a sequence's share of the rows fills, shared out to warps.
    const long long items = (static_cast<long long>(args.rows) / args.sequences / kBlock + 2) * args.kv_heads * 2;
    const unsigned y = static_cast<unsigned>(std::min(args.sequences, 65535));
    const long long most = std::max<long long>(1, 16LL * sms / y + 1);
    const dim3 grid(static_cast<unsigned>(std::min((items + 7) / 8, most)), y);
    return launch_dependent(fb_paged8_store, grid, dim3(256), 0, stream, args, cache);
}

cudaError_t paged8_attention(const PackedArgs& args, const Cache8& cache, int longest, void* workspace,
                             cudaStream_t stream) {
    FewParams p;
    std::memset(&p, 0, sizeof p);
    p.a = args;
    p.cache = cache;
    p.group = args.heads / args.kv_heads;
    const long long rows = static_cast<long long>(longest) * p.group;
    while ((1 << p.log_page) < args.page_size) {
        ++p.log_page;
    }
    int sms = 148;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) {
        return e;
    }
    const long long most_keys = static_cast<long long>(args.table_stride) * args.page_size;
    // 64 sequences of up to 8,192 keys, 32 heads on 8, with 1, 2, 4, 5, 8 and 16 new tokens (4 to 64 rows): tiles of eight rows 47, 48, 80, 115, 150
    // and 292 us; of 16 rows 52, 52, 66, 104, 116 and 220; the tensor cores' of 32 rows 105, 105, 105, 106, 106 and 190, of 64 rows 106 to 107
    // and 119. Two sequences of 100,000 and 7,200, 16 heads on 2, with 8, 16, 24, 32 and 40 rows: 19, 23, 26, 30 and 36 us; 21, 23, 28, 29 and 34; 31 up to
    // 32 rows and 42; 32 up to 32 rows and 34. From 17 rows on both take about as long.
    return rows <= 8    ? launch_few<1>(p, sms, workspace, most_keys, stream)
           : rows <= 16 ? launch_few<2>(p, sms, workspace, most_keys, stream)
                        : packed_forward(args, &cache, longest, workspace, stream);
}

cudaError_t paged8_workspace(size_t* bytes) {
    int sms = 148;
    const cudaError_t e = sm_count(&sms);
    *bytes = packed_workspace(std::min(kFewPerSm * sms, kMostPackedCtas));
    return e;
}

}  // namespace fb
