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

// A warp stores one block of one head of K or V: its lanes take 8 values of 4 rows at a time.
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
            const long long page = page_of(p, s, key);
            if (page < 0) {
                continue;
            }
            const __half* from = (which == 0 ? p.k : p.v) + head * kHead;
            const long long row = (page * p.kv_heads + head) * p.page_size + key % p.page_size;
            int8_t* codes = (which == 0 ? cache.k : cache.v) + row * kHead;
            float* scale_at = (which == 0 ? cache.k_scales : cache.v_scales) + row / kBlock;
            uint4 held[4];
            float largest = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = key + 4 * r + of_four - begins;      // of the new tokens
                held[r] = make_uint4(0u, 0u, 0u, 0u);
                if (i >= 0 && i < q.count) {
                    held[r] = reinterpret_cast<const uint4*>(from + (q.first + static_cast<long long>(i)) * p.kv_stride)[piece];
                }
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
            float before = 0.0f;
            if (begins > key) {
                before = *scale_at;
                scale = max_nan(before, scale);
            }
            const bool grows = begins > key && scale != before;     // (a NaN grows: codes of it are 0)
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
                    const uint2 old = *to;
                    const unsigned w[2] = {old.x, old.y};
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

// Bound by what it reads, so the warp-wide product is the right one: mma.sync takes codes that a lane has just turned into FP16
// in its registers, where the tensor cores' larger instruction would want them written to shared memory first. A tile
// (packed_schedule.h) has up to 16 kTiles rows; a warp takes 16 of them and every (8 / kTiles)-th block of 16 keys, whose codes
// come to it alone through four stages of asynchronous copies, and the warps' sums meet at the end of a piece.
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kStages = 4;
constexpr int kStageBytes = 2 * kBlock * kHead;       // K and V of a block
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kMergeStride = kHead + 4;               // floats between rows that meet
static_assert(kWarps * 16 * kMergeStride * 4 <= kRingBytes, "the rows that meet take the ring's place");

struct FewParams {
    PackedArgs a;
    Cache8 cache;
    Record* records;
    float* parts;
    int group, log_tokens, log_page;
    bool splits;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                          unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bytes kLow and kLow + 1 of x, which are codes + 128, as FP16: 1,024 + byte has the byte as its low bits.
template <int kLow>
__device__ __forceinline__ unsigned two_codes(unsigned x) {
    const unsigned biased = __byte_perm(x, 0x64646464u, kLow == 0 ? 0x4140 : 0x4342);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const unsigned*>(&h);
}

template <int kTiles>
__global__ void __launch_bounds__(kThreads, 2) fb_paged8_few(const FewParams p) {
    constexpr int kApart = kWarps / kTiles;      // warps that share rows
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ Cut cuts[2];
    __shared__ long long scan[kWarps + 1];
    __shared__ int scan_longest[kWarps];
    __shared__ int whole_tiles;
    __shared__ float merge_max[kWarps][16], merge_sum[kWarps][16];
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x / 32), 0), lane = threadIdx.x % 32;
    const int g = lane / 4, t = lane % 4;        // row and column of the products' fragments
    dependency_wait();
    if (p.a.sequences > 32) {
        locate<false, kThreads>(p, cuts, whole_tiles, scan, scan_longest);
    } else if (warp == 0) {
        locate_in_warp<false>(p, cuts, whole_tiles, lane);
    }
    __syncthreads();
    dependency_release();
    if (threadIdx.x == 0) {
        p.records[blockIdx.x] = make_record(SequenceOf{p.a}, p.log_tokens, cuts[0], cuts[1]);
    }
    const int tile = warp % kTiles, share = warp / kTiles;
    unsigned char* stages = ring + warp * (kStages * kStageBytes);
    const uint32_t stages_at = sm100::smem_u32(stages);
    const float scale2 = p.a.scale * kLog2e;
    Walk walk;
    Piece piece;
    walk.begin(SequenceOf{p.a}, cuts[0], cuts[1].at);
    while (walk.next(SequenceOf{p.a}, p.a.sequences, p.a.kv_heads, p.log_tokens, piece)) {
        const int first_position = piece.position();
        const int first_block = piece.from * (kKeyTile / kBlock);
        const int end_block = min(piece.to * (kKeyTile / kBlock), (piece.sequence.keys + kBlock - 1) / kBlock);
        const int rows = piece.tokens * p.group;
        // This warp's blocks: first_block + share + i kApart.
        const int count = tile * 16 >= rows ? 0 : max(0, (end_block - first_block - share + kApart - 1) / kApart);
        // Its rows g and g + 8: queries as they are multiplied, and positions.
        uint4 query[2][2];
        int position[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = tile * 16 + g + 8 * h, token = row / p.group;
            position[h] = -1;
            query[h][0] = query[h][1] = make_uint4(0u, 0u, 0u, 0u);
            if (row < rows) {
                position[h] = first_position + token;
                const __half* from = p.a.q + (static_cast<long long>(piece.sequence.first) + piece.first_token + token) * p.a.q_stride +
                                     (piece.head * p.group + row - token * p.group) * kHead + 16 * t;
                query[h][0] = reinterpret_cast<const uint4*>(from)[0];
                query[h][1] = reinterpret_cast<const uint4*>(from)[1];
            }
        }
        float m[2] = {kNoKey, kNoKey}, l[2] = {0.0f, 0.0f};
        float out[8][4] = {};
        // Lane i has the place of block 32 batch + i (the row of its first key in the cache, -1 for none) and its scales.
        auto place_of = [&](int i) {
            if (i >= count) {
                return -1;
            }
            const int key = (first_block + share + i * kApart) * kBlock;
            const long long page = page_of(p.a, piece.index, key);
            return page < 0 ? -1
                            : static_cast<int>((page * p.a.kv_heads + piece.head) << p.log_page) + (key & (p.a.page_size - 1));
        };
        int place_next = place_of(lane), place = -1;
        float k_scale_next = 0.0f, v_scale_next = 0.0f, k_scale = 0.0f, v_scale = 0.0f;
        auto fetch = [&](int i) {
            if (i < count) {
                if (i % 32 == 0) {
                    place = place_next;
                    k_scale_next = v_scale_next = 0.0f;
                    if (place >= 0) {
                        k_scale_next = p.cache.k_scales[place / kBlock];
                        v_scale_next = p.cache.v_scales[place / kBlock];
                    }
                    place_next = place_of(i + 32 + lane);
                }
                const int from = __shfl_sync(kFullMask, place, i % 32);
                const uint32_t to = stages_at + (i % kStages) * kStageBytes + lane * 16;
                const unsigned bytes = from >= 0 ? 16u : 0u;       // zeros for a page that is not there
                const long long at = static_cast<long long>(max(from, 0)) * kHead + lane * 16;
                const int8_t* k = p.cache.k + at;
                const int8_t* v = p.cache.v + at;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(k), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 512), "l"(k + 512), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 1024), "l"(v), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 1536), "l"(v + 512), "r"(bytes) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            fetch(i);
        }
        for (int i = 0; i < count; ++i) {
            if (i % 32 == 0) {
                k_scale = k_scale_next;
                v_scale = v_scale_next;
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();       // everybody's copies have landed, and the stage before is read
            fetch(i + kStages - 1);
            const unsigned char* stage = stages + (i % kStages) * kStageBytes;
            const int key = (first_block + share + i * kApart) * kBlock;
            // Scores: of the products' eight columns the even ones are keys 0 to 3 and the odd ones 4 to 7, which is the order that
            // V's rows below are read in, four in a row at a time; a lane's four terms of a product are
            // neighbours, as they lie in its 16 bytes of a key.
            float scores[2][4] = {};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint4 codes = *reinterpret_cast<const uint4*>(stage + (8 * u + (g & 1) * 4 + (g >> 1)) * kHead + 16 * t);
                const unsigned w[4] = {codes.x ^ 0x80808080u, codes.y ^ 0x80808080u, codes.z ^ 0x80808080u, codes.w ^ 0x80808080u};
                const unsigned low[8] = {query[0][0].x, query[0][0].y, query[0][0].z, query[0][0].w,
                                         query[0][1].x, query[0][1].y, query[0][1].z, query[0][1].w};
                const unsigned high[8] = {query[1][0].x, query[1][0].y, query[1][0].z, query[1][0].w,
                                          query[1][1].x, query[1][1].y, query[1][1].z, query[1][1].w};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    mma_16816(scores[u], low[2 * s], high[2 * s], low[2 * s + 1], high[2 * s + 1], two_codes<0>(w[s]),
                              two_codes<2>(w[s]));
                }
            }
            const float weight = __shfl_sync(kFullMask, v_scale, i % 32);
            const float v_here = weight == 0.0f ? 1.0f : weight;      // (codes are 0 then)
            const float slope = __shfl_sync(kFullMask, k_scale, i % 32) * scale2, offset = __log2f(v_here);
            const float inverse = 1.0f / v_here;
            bool moves = false;
            float top[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& x = scores[u][2 * h + c];
                        x = fmaf(x, slope, offset);
                        if (key + kBlock - 1 > first_position) {
                            x = key + 8 * u + 4 * c + t <= position[h] ? x : -INFINITY;
                        }
                        top[h] = max_nan(top[h], x);
                    }
                }
                moves = moves || !(top[h] - m[h] <= kLazyShift);
            }
            if (__any_sync(kFullMask, moves)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = max_nan(top[h], __shfl_xor_sync(kFullMask, top[h], 1));
                    top[h] = max_nan(top[h], __shfl_xor_sync(kFullMask, top[h], 2));
                    const float next = max_nan(m[h], top[h]);
                    const float alpha = fast_exp2(m[h] - next);
                    m[h] = next;
                    l[h] *= alpha;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        out[j][2 * h] *= alpha;
                        out[j][2 * h + 1] *= alpha;
                    }
                }
            }
            unsigned weights[2][2];        // [half of the keys][row]
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float sum = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float x = fast_exp2(scores[u][2 * h] - m[h]), y = fast_exp2(scores[u][2 * h + 1] - m[h]);
                    sum += x + y;
                    weights[u][h] = pack2(x, y);
                }
                // (A row that sees nothing of the block has nothing to do with its scale, whatever that is.)
                l[h] = fmaf(sum, sum == 0.0f ? 0.0f : inverse, l[h]);
            }
            uint2 values[4];       // of keys t, t + 4, t + 8 and t + 12, columns 8 g to 8 g + 7
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                values[k] = *reinterpret_cast<const uint2*>(stage + kBlock * kHead + (4 * k + t) * kHead + 8 * g);
                values[k].x ^= 0x80808080u;
                values[k].y ^= 0x80808080u;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const unsigned w[4] = {half == 0 ? values[0].x : values[0].y, half == 0 ? values[1].x : values[1].y,
                                       half == 0 ? values[2].x : values[2].y, half == 0 ? values[3].x : values[3].y};
#pragma unroll
                for (int pair = 0; pair < 2; ++pair) {
                    // Two columns of two keys side by side.
                    const unsigned first = __byte_perm(w[0], w[1], pair == 0 ? 0x5140 : 0x7362);
                    const unsigned second = __byte_perm(w[2], w[3], pair == 0 ? 0x5140 : 0x7362);
                    const int j = 4 * half + 2 * pair;
                    mma_16816(out[j], weights[0][0], weights[0][1], weights[1][0], weights[1][1], two_codes<0>(first),
                              two_codes<0>(second));
                    mma_16816(out[j + 1], weights[0][0], weights[0][1], weights[1][0], weights[1][1], two_codes<2>(first),
                              two_codes<2>(second));
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();       // the ring is everybody's from here on
        float* mine = reinterpret_cast<float*>(ring) + warp * 16 * kMergeStride;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
            l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
            if (t == 0) {
                merge_max[warp][g + 8 * h] = m[h];
                merge_sum[warp][g + 8 * h] = l[h];
            }
            // Column 16 t + j of the row is out[j][2 h], column 16 t + 8 + j out[j][2 h + 1].
            float4* to = reinterpret_cast<float4*>(mine + (g + 8 * h) * kMergeStride + 16 * t);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                to[2 * c] = make_float4(out[0][2 * h + c], out[1][2 * h + c], out[2][2 * h + c], out[3][2 * h + c]);
                to[2 * c + 1] = make_float4(out[4][2 * h + c], out[5][2 * h + c], out[6][2 * h + c], out[7][2 * h + c]);
            }
        }
        __syncthreads();
        const bool whole = piece.from == 0 && piece.to == piece.tiles;
        for (int row = threadIdx.x / 16; row < rows; row += kThreads / 16) {
            const int column = threadIdx.x % 16 * 4;
            float all = kNoKey;
#pragma unroll
            for (int w = 0; w < kApart; ++w) {
                all = max_nan(all, merge_max[w * kTiles + row / 16][row % 16]);
            }
            float total = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kApart; ++w) {
                const int its = w * kTiles + row / 16;
                const float factor = fast_exp2(merge_max[its][row % 16] - all);
                const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(ring) +
                                                                  (its * 16 + row % 16) * kMergeStride + column);
                if (merge_max[its][row % 16] != kNoKey) {
                    total = fmaf(merge_sum[its][row % 16], factor, total);
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
        __syncthreads();       // the ring is the copies' again
    }
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
    const int form = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
    while ((2 << p.log_tokens) * p.group <= 16 << form) {
        ++p.log_tokens;
    }
    while ((1 << p.log_page) < args.page_size) {
        ++p.log_page;
    }
    int sms = 148;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) {
        return e;
    }
    const int ctas = packed_ctas(sms);
    const long long most_keys = static_cast<long long>(args.table_stride) * args.page_size;
    p.splits = most_keys > 1024;
    p.records = packed_records(workspace);
    p.parts = packed_parts(workspace, ctas);
    const auto kernel = form == 0   ? fb_paged8_few<1>
                        : form == 1 ? fb_paged8_few<2>
                        : form == 2 ? fb_paged8_few<4>
                                    : fb_paged8_few<8>;
    static std::atomic<bool> configured[4][64] = {};
    e = allow_shared_memory(kernel, kRingBytes, configured[form]);
    if (e == cudaSuccess) {
        e = launch_dependent(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kRingBytes, stream, p);
    }
    if (e != cudaSuccess || !p.splits) {
        return e;
    }
    return packed_join(args, p.records, p.parts, ctas, most_keys, stream);
}

}  // namespace fb
