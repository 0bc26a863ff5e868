// Causal attention over sequences of different lengths, packed or in the pages of a cache, on the
// 5th-generation tensor cores (head width 64).
//
// A tile is the 128 rows of (token, query head) that one K/V head's group makes of 128 / group
// consecutive tokens (rounded down to a power of two): one load of keys and values serves the whole
// group. S = Q K^T goes to tensor memory, a thread takes the softmax of a row in base 2, P goes
// back as FP16 pairs and is the A operand of O += P V, which accumulates in tensor memory over the
// row of key tiles; the exponent that probabilities are taken against moves only when a row's
// maximum exceeds it by more than 2^8, so that O is rarely rescaled.
// The batch is shared out evenly however ragged it is (packed_schedule.h); a tile split between CTAs
// leaves its parts (O before the division, row maxima and sums, FP32) in the workspace, and a second,
// dependent launch joins them in the order of the keys.
//
// Two CTAs per SM with one tile each: one's matrix products, loads and ends run under the other's
// exponentials, which bound the kernel (128 x 128 of them per key tile take the SM's special-function
// unit 1,024 clocks and the products 512; a quarter of them runs on the FMA pipe instead).
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

constexpr int kThreads = 192;   // TMA warp, MMA warp, four softmax warps with a row per thread
constexpr int kWarps = kThreads / 32;
constexpr int kSlots = 4;       // ring of K and V tiles
constexpr int kSmem = 1024 + (2 + kSlots) * kTileBytes + 256;
constexpr int kLeastPart = 2;   // of the line of key tiles, per CTA

constexpr size_t kPartFloats = size_t{kRows} * kHead + 2 * kRows;   // O [column / 4][row][4], maxima, sums

struct TileParams {
    CUtensorMap map_q, map_k, map_v;
    PackedArgs a;
    Record* records;    // [CTA]
    float* parts;       // [CTA][head part, tail part]
    int group, log_tokens;
    int boxes;          // loads per K or V tile
    int box_rows;
};

struct Barriers {
    uint32_t base;
    __device__ uint32_t q_full(int b) const { return base + 8u * b; }
    __device__ uint32_t q_empty(int b) const { return base + 16 + 8u * b; }
    __device__ uint32_t s_full() const { return base + 32; }
    __device__ uint32_t s_free() const { return base + 40; }
    __device__ uint32_t p_ready() const { return base + 48; }
    __device__ uint32_t pv_done() const { return base + 56; }
    __device__ uint32_t slot_full(int s) const { return base + 64 + 8u * s; }
    __device__ uint32_t slot_empty(int s) const { return base + 64 + 8u * (kSlots + s); }
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

// Which part of the line this CTA works on: every thread of the block takes part.
__device__ void locate(const TileParams& p, Cut (&cuts)[2], long long (&scan)[kWarps + 1]) {
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, warp = tid / 32;
    auto length_of = [&](int s, int& before, int& tokens) -> long long {
        before = tokens = 0;
        if (s >= p.a.sequences) {
            return 0;
        }
        const Sequence q = sequence_at(p.a, s);
        before = q.keys - q.count;
        tokens = q.count;
        return head_length(before, tokens, p.log_tokens);
    };
    int before = 0, tokens = 0;
    long long length = length_of(tid, before, tokens);
    long long sum = length;
    for (int s = tid + kThreads; s < p.a.sequences; s += kThreads) {
        int b, t;
        sum += length_of(s, b, t);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        sum += __shfl_xor_sync(kFullMask, sum, off);
    }
    if (lane == 0) {
        scan[warp] = sum;
    }
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        total += scan[w];
    }
    total *= p.a.kv_heads;
    const int parts = part_count(total, static_cast<int>(gridDim.x), kLeastPart);
    const int cta = static_cast<int>(blockIdx.x);
    if (cta >= parts) {
        if (tid < 2) {
            cuts[tid] = Cut{0, 0, 0, 0, 0};
        }
        __syncthreads();
        return;
    }
    const long long place[2] = {cut_place(total, parts, cta), cut_place(total, parts, cta + 1)};
    const long long tolerance = cut_tolerance(total, parts);
    if (tid < 2 && place[tid] == total) {
        cuts[tid] = Cut{total, p.a.sequences, 0, 0, 0};
    }
    long long running = 0;
    for (int first = 0; first < p.a.sequences; first += kThreads) {
        if (first != 0) {
            length = length_of(first + tid, before, tokens);
        }
        const long long mine = length * p.a.kv_heads;
        long long upto = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long other = __shfl_up_sync(kFullMask, upto, off);
            upto += lane >= off ? other : 0;
        }
        __syncthreads();
        if (lane == 31) {
            scan[warp] = upto;
        }
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            upto += w < warp ? scan[w] : 0;
            all += scan[w];
        }
        const long long begins = running + upto - mine;
        for (int c = 0; c < 2; ++c) {
            if (place[c] >= begins && place[c] < begins + mine) {
                cuts[c] = cut_at(place[c], place[c] - begins, first + tid, before, tokens, p.log_tokens, length,
                                 tolerance);
            }
        }
        running += all;
    }
    __syncthreads();
}

// A role's place in the CTA's sequence of key tiles.
struct Steps {
    Walk walk;
    Piece piece;
    int j, round;
    bool valid;
    __device__ __forceinline__ void begin(const TileParams& p, const Cut& lo, long long end) {
        walk.begin(SequenceOf{p.a}, lo, end);
        round = 0;
        valid = walk.next(SequenceOf{p.a}, p.a.sequences, p.a.kv_heads, p.log_tokens, piece);
        j = valid ? piece.from : 0;
    }
    __device__ __forceinline__ void advance(const TileParams& p) {
        if (++j == piece.to) {
            ++round;
            valid = walk.next(SequenceOf{p.a}, p.a.sequences, p.a.kv_heads, p.log_tokens, piece);
            j = valid ? piece.from : 0;
        }
    }
};

template <bool kPaged>
__global__ void __launch_bounds__(kThreads, 2) fb_packed_forward_tiles(const __grid_constant__ TileParams p) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (sm100::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_tiles = base;
    const uint32_t ring = base + 2 * kTileBytes;
    const Barriers bar{ring + kSlots * kTileBytes};
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ Cut cuts[2];
    __shared__ long long scan[kWarps + 1];

    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x / 32), 0);
    const int lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int b = 0; b < 2; ++b) {
            sm100::mbar_init(bar.q_full(b), 1);
            sm100::mbar_init(bar.q_empty(b), 1);
        }
        sm100::mbar_init(bar.s_full(), 1);
        sm100::mbar_init(bar.s_free(), 4);     // one arrival per softmax warp
        sm100::mbar_init(bar.p_ready(), 4);
        sm100::mbar_init(bar.pv_done(), 1);
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
    locate(p, cuts, scan);
    sm100::tc_fence_before_sync();
    __syncthreads();
    sm100::tc_fence_after_sync();
    const uint32_t tmem_s = tmem_slot, tmem_o = tmem_slot + 128, tmem_p = tmem_slot + 192;
    volatile int* abort = &abort_flag;
    const Cut lo = cuts[0];
    const long long end = cuts[1].at;

    if (warp == 0) {
        Steps keys, values;     // the next K tile to fetch; the next V tile, one step behind
        keys.begin(p, lo, end);
        values.begin(p, lo, end);
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        auto load = [&](const CUtensorMap* map, const Steps& at) {
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
                    // A page that is not there is read from outside the cache, as zeros.
                    const int key = at.j * kKeyTile + lane * p.box_rows;
                    const long long page = key < at.piece.sequence.keys ? page_of(p.a, at.piece.index, key) : -1;
                    const long long row = page < 0 ? p.a.pages * p.a.kv_heads * p.a.page_size
                                                   : (page * p.a.kv_heads + at.piece.head) * p.a.page_size +
                                                         key % p.a.page_size;
                    sm100::tma_load_2d(dst + lane * p.box_rows * (kHead * 2), map, full, 0, static_cast<int>(row));
                }
            } else if (lane == 0) {
                sm100::tma_load_3d(dst, map, full, 0, at.piece.head, at.piece.sequence.first + at.j * kKeyTile);
            }
            __syncwarp();
            if (++slot == kSlots) {
                slot = 0;
                phase ^= 1u;
            }
        };
        auto load_keys = [&]() {
            if (keys.j == keys.piece.from) {
                // A new piece: its queries go into the buffer of its parity, free once the piece two
                // rounds back has issued its last scores.
                const int b = keys.round & 1;
                if (keys.round >= 2 &&
                    !sm100::mbar_wait_warp(bar.q_empty(b), ((keys.round >> 1) - 1) & 1, abort)) {
                    ok = false;
                    return;
                }
                if (lane == 0) {
                    sm100::mbar_expect_tx(bar.q_full(b), static_cast<uint32_t>(p.group << p.log_tokens) * (kHead * 2));
                    sm100::tma_load_3d(q_tiles + b * kTileBytes, &p.map_q, bar.q_full(b), 0,
                                       keys.piece.head * p.group, keys.piece.sequence.first + keys.piece.first_token);
                }
            }
            load(&p.map_k, keys);
            keys.advance(p);
        };
        if (keys.valid) {
            load_keys();
        }
        while (ok && values.valid) {
            if (keys.valid) {
                load_keys();
            }
            if (ok) {
                load(&p.map_v, values);
                values.advance(p);
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
        Steps ahead, now;
        ahead.begin(p, lo, end);
        now.begin(p, lo, end);
        uint32_t issued = 0;
        auto issue_scores = [&]() {
            if (!ok || !ahead.valid) {
                return;
            }
            const int b = ahead.round & 1;
            if (ahead.j == ahead.piece.from &&
                !sm100::mbar_wait_warp(bar.q_full(b), (ahead.round >> 1) & 1, abort)) {
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
            const bool last = ahead.j + 1 == ahead.piece.to;
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
            ahead.advance(p);
        };
        issue_scores();
        for (uint32_t n = 0; ok && now.valid; ++n) {
            issue_scores();    // of the next step, as soon as this step's have been read
            if (!ok || !sm100::mbar_wait_warp(bar.p_ready(), n & 1, abort)) {
                break;
            }
            const uint32_t v_tile = next_tile();
            if (v_tile == 0) {
                break;
            }
            const int present = now.piece.sequence.keys - now.j * kKeyTile;
            if (present < kKeyTile) {
                // Rows behind the sequence's last key hold anything, and 0 times that need not be 0.
                const int from = max(present, 0) * (kHead * 2);
                for (int at = from + lane * 16; at < kTileBytes; at += 512) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_tile + at), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            const uint64_t v_desc = desc_mnmajor(v_tile, 0, 16);
            if (sm100::elect_one()) {
                sm100::mma_f16_ts_at<-1>(tmem_o, tmem_p, v_desc, 0, kIdescPV, now.j > now.piece.from);
#pragma unroll
                for (int ks = 1; ks < 8; ++ks) {
                    sm100::mma_f16_ts_at<1>(tmem_o, tmem_p + ks * 8, v_desc, ks * 128, kIdescPV);
                }
                sm100::mma_commit(bar.pv_done());
                sm100::mma_commit(bar.slot_empty(slot));
            }
            __syncwarp();
            step_ring();
            now.advance(p);
        }
    } else {
        const int quadrant = warp % 4;
        const int row = quadrant * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quadrant * 32) << 16;
        const int token = row / p.group;
        const float scale2 = p.a.scale * kLog2e;
        const F2 scale_pair = f2_pack(scale2, scale2);
        if (row == 0) {
            p.records[blockIdx.x] = make_record(SequenceOf{p.a}, p.log_tokens, lo, cuts[1]);
        }
        Walk walk;
        Piece piece;
        walk.begin(SequenceOf{p.a}, lo, end);
        uint32_t n = 0;
        bool ok = true;
        while (ok && walk.next(SequenceOf{p.a}, p.a.sequences, p.a.kv_heads, p.log_tokens, piece)) {
            const bool valid = token < piece.tokens;
            const bool active = __any_sync(kFullMask, valid);
            const int position = valid ? piece.position() + token : -1;
            float m = kNoKey;     // reference exponent of the row (base 2)
            F2 l = 0;             // the row sum, in two partial sums
            for (int j = piece.from; j < piece.to; ++j, ++n) {
                if (!sm100::mbar_wait_warp(bar.s_full(), n & 1, abort)) {
                    ok = false;
                    break;
                }
                sm100::tc_fence_after_sync();
                // The scores are read twice, 32 columns at a time and the next 32 on their way: a row's
                // 128 at once left no registers (the kernel spilled 950 bytes and took three times as long).
                uint32_t raw[2][32];
                const int visible = position - j * kKeyTile;     // columns up to this one are seen
                const bool masked = j * kKeyTile + kKeyTile - 1 > piece.position();
                float alpha = 1.0f;
                bool moved = false;
                if (active) {
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    sm100::tmem_ld_32x32(tmem_s + lane_base, raw[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        sm100::tmem_ld_wait();
                        sm100::tmem_ld_32x32(tmem_s + lane_base + 32 * ((c + 1) % 4), raw[(c + 1) & 1]);
                        uint32_t (&now)[32] = raw[c & 1];
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                now[i] = 32 * c + i <= visible ? now[i] : 0xff800000u;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                top[t] = max3_nan(top[t], __uint_as_float(now[i + t]), __uint_as_float(now[i + 4 + t]));
                            }
                        }
                    }
                    // The scale is positive, so the maximum may be scaled after it is taken.
                    const float local = max3_nan(top[0], top[1], max3_nan(top[2], top[3], top[3])) * scale2;
                    const float mx = max3_nan(m, local, local);
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
                    if (j > piece.from && __any_sync(kFullMask, moved)) {
                        const F2 a2 = f2_pack(alpha, alpha);
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t acc[16];
                            sm100::tmem_ld_32x16(tmem_o + lane_base + c * 16, acc);
                            sm100::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                float x, y;
                                f2_unpack(f2_mul(f2_pack(__uint_as_float(acc[i]), __uint_as_float(acc[i + 1])), a2), x, y);
                                acc[i] = __float_as_uint(x);
                                acc[i + 1] = __float_as_uint(y);
                            }
                            sm100::tmem_st_32x16(tmem_o + lane_base + c * 16, acc);
                        }
                    }
                    const F2 shift = f2_pack(-m, -m);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        sm100::tmem_ld_wait();
                        if (c < 3) {
                            sm100::tmem_ld_32x32(tmem_s + lane_base + 32 * (c + 1), raw[(c + 1) & 1]);
                        } else {
                            // All scores are read: the next step's may come.
                            sm100::tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0) {
                                sm100::mbar_arrive(bar.s_free());
                            }
                        }
                        uint32_t (&now)[32] = raw[c & 1];
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                now[i] = 32 * c + i <= visible ? now[i] : 0xff800000u;
                            }
                        }
                        uint32_t packed[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float x, y;
                            const F2 t = f2_fma(f2_pack(__uint_as_float(now[2 * i]), __uint_as_float(now[2 * i + 1])),
                                                scale_pair, shift);
                            if ((i & 3) == 0) {
                                exp2_pair_fma(t, x, y);
                            } else {
                                f2_unpack(t, x, y);
                                x = fast_exp2(x);
                                y = fast_exp2(y);
                            }
                            l = f2_add(l, f2_pack(x, y));
                            packed[i] = pack2(x, y);
                        }
                        sm100::tmem_st_32x16(tmem_p + lane_base + c * 16, packed);
                    }
                    sm100::tmem_st_wait();
                } else {
                    __syncwarp();
                    if (lane == 0) {
                        sm100::mbar_arrive(bar.s_free());
                    }
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
            float total = sum_x + sum_y;
            if (m == kNoKey) {
                total = 0.0f;    // (the polynomial's least power of two is not 0)
            }
            const int head = piece.head * p.group + row - token * p.group;
            const long long at_row = piece.sequence.first + piece.first_token + token;
            const bool whole = piece.whole();
            float* part = p.parts + (2 * size_t{blockIdx.x} + (piece.from == 0 ? 1 : 0)) * kPartFloats;
            const float inv = position < 0 ? 0.0f : 1.0f / total;   // no key at all gives zeros
            __half* out = p.a.o + at_row * p.a.o_stride + head * kHead;
            uint32_t acc[64];
            if (active) {
                sm100::tmem_ld_32x32(tmem_o + lane_base, reinterpret_cast<uint32_t(&)[32]>(acc[0]));
                sm100::tmem_ld_32x32(tmem_o + lane_base + 32, reinterpret_cast<uint32_t(&)[32]>(acc[32]));
                sm100::tmem_ld_wait();
            }
            if (valid && whole) {
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[i] = position < 0 ? 0.0f : __uint_as_float(acc[b * 8 + i]) * inv;
                    }
                    *reinterpret_cast<uint4*>(out + 8 * b) = pack8(v);
                }
            }
            if (valid && !whole) {
#pragma unroll
                for (int b = 0; b < 16; ++b) {
                    reinterpret_cast<uint4*>(part)[b * kRows + row] =
                        make_uint4(acc[4 * b], acc[4 * b + 1], acc[4 * b + 2], acc[4 * b + 3]);
                }
            }
            sm100::tc_fence_before_sync();
            if (valid && whole && p.a.lse != nullptr) {
                p.a.lse[static_cast<long long>(head) * p.a.rows + at_row] =
                    position < 0 ? -INFINITY : (m + log2f(total)) * kLn2;
            }
            if (valid && !whole) {
                part[kRows * kHead + row] = m;
                part[kRows * kHead + kRows + row] = total;
            }
        }
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

// Block (k, y) joins rows 32 y .. of the tile that CTA k began and did not end, if there is one: eight threads
// per row, eight columns each.
__global__ void __launch_bounds__(256) fb_packed_join(const JoinParams p) {
    dependency_wait();
    dependency_release();
    const int k = static_cast<int>(blockIdx.x);
    const Record mine = p.records[k];
    if (mine.tail_part == 0) {
        return;
    }
    const int row = static_cast<int>(blockIdx.y) * 32 + threadIdx.x / 8;
    const int piece = threadIdx.x % 8;
    const int token = row / p.group;
    if (token >= mine.tokens) {
        return;
    }
    int last = k + 1;
    while (last < p.ctas - 1 && p.records[last].head_part == 2) {
        ++last;
    }
    auto part_of = [&](int cta) { return p.parts + (2 * static_cast<size_t>(cta) + (cta == k ? 1 : 0)) * kPartFloats; };
    float top = kNoKey;
    for (int cta = k; cta <= last; ++cta) {
        top = max3_nan(top, part_of(cta)[kRows * kHead + row], kNoKey);
    }
    float total = 0.0f;
    float acc[8] = {};
#pragma unroll 4
    for (int cta = k; cta <= last; ++cta) {
        const float* part = part_of(cta);
        const float m = part[kRows * kHead + row];
        const float weight = m == kNoKey ? 0.0f : fast_exp2(m - top);
        const float4 x = reinterpret_cast<const float4*>(part)[(2 * piece) * kRows + row];
        const float4 y = reinterpret_cast<const float4*>(part)[(2 * piece + 1) * kRows + row];
        const float sum = part[kRows * kHead + kRows + row];
        if (m != kNoKey) {    // (a part of no key may hold 0 times anything)
            total = fmaf(sum, weight, total);
            acc[0] = fmaf(x.x, weight, acc[0]);
            acc[1] = fmaf(x.y, weight, acc[1]);
            acc[2] = fmaf(x.z, weight, acc[2]);
            acc[3] = fmaf(x.w, weight, acc[3]);
            acc[4] = fmaf(y.x, weight, acc[4]);
            acc[5] = fmaf(y.y, weight, acc[5]);
            acc[6] = fmaf(y.z, weight, acc[6]);
            acc[7] = fmaf(y.w, weight, acc[7]);
        }
    }
    const bool none = mine.position + token < 0;
    const int head = mine.kv_head * p.group + row - token * p.group;
    const long long at_row = mine.first_row + token;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        acc[i] = none ? 0.0f : acc[i] / total;
    }
    *reinterpret_cast<uint4*>(p.a.o + at_row * p.a.o_stride + head * kHead + 8 * piece) = pack8(acc);
    if (piece == 0 && p.a.lse != nullptr) {
        p.a.lse[static_cast<long long>(head) * p.a.rows + at_row] = none ? -INFINITY : (top + log2f(total)) * kLn2;
    }
}

// ---- host -------------------------------------------------------------------------------------------

size_t records_bytes(int ctas) { return (static_cast<size_t>(ctas) * sizeof(Record) + 255) / 256 * 256; }

}  // namespace

cudaError_t packed_forward_error_flag(int* value, bool reset) { return read_error_word(value, reset); }

cudaError_t packed_forward_workspace(size_t* bytes) {
    int sms = 148;
    const cudaError_t e = sm_count(&sms);
    *bytes = records_bytes(2 * sms) + 2 * static_cast<size_t>(2 * sms) * kPartFloats * sizeof(float);
    return e;
}

cudaError_t packed_forward(const PackedArgs& args, void* workspace, cudaStream_t stream) {
    TileParams p;
    std::memset(&p, 0, sizeof p);
    p.a = args;
    p.group = args.heads / args.kv_heads;
    while ((2 << p.log_tokens) * p.group <= kRows) {
        ++p.log_tokens;
    }
    int sms = 148;
    cudaError_t e = sm_count(&sms);
    const int ctas = 2 * sms;
    const bool paged = args.table != nullptr;
    if (e == cudaSuccess) {
        e = encode_rows(&p.map_q, args.q, args.heads, args.rows, args.q_stride, p.group, 1 << p.log_tokens);
    }
    if (paged) {
        p.box_rows = std::min(args.page_size, kKeyTile);
        p.boxes = kKeyTile / p.box_rows;
        const long long rows = args.pages * args.kv_heads * args.page_size;
        if (e == cudaSuccess) e = encode_pages(&p.map_k, args.k, rows, p.box_rows);
        if (e == cudaSuccess) e = encode_pages(&p.map_v, args.v, rows, p.box_rows);
    } else {
        if (e == cudaSuccess) e = encode_rows(&p.map_k, args.k, args.kv_heads, args.rows, args.kv_stride, 1, kKeyTile);
        if (e == cudaSuccess) e = encode_rows(&p.map_v, args.v, args.kv_heads, args.rows, args.kv_stride, 1, kKeyTile);
    }
    if (e != cudaSuccess) {
        return e;
    }
    p.records = static_cast<Record*>(workspace);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + records_bytes(ctas));
    const auto kernel = paged ? fb_packed_forward_tiles<true> : fb_packed_forward_tiles<false>;
    static std::atomic<bool> configured[2][64] = {};
    e = allow_shared_memory(kernel, kSmem, configured[paged]);
    if (e != cudaSuccess) {
        return e;
    }
    e = launch_dependent(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmem, stream, p);
    if (e != cudaSuccess) {
        return e;
    }
    JoinParams j = {args, p.records, p.parts, ctas, p.group};
    return launch_dependent(fb_packed_join, dim3(static_cast<unsigned>(ctas), kRows / 32), dim3(256), 0, stream, j);
}

}  // namespace fb
