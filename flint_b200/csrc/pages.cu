// Which sequence holds which pages of a paged cache: sharing, growing, cutting, renumbering, and copying the pages that this
// asks for (extensions: the reference has no cache).
//
// All but the copies are bound by latency: chains of dependent loads, barriers and launches. As parts of a graph a fork takes 2.4 us (8
// sequences of 22 entries) to 4.3 us (512 of 66), a reservation 3.4 to 4.8 us, a compaction of 4,000 pages 9.5 us. Copies are bound by
// HBM: 1,175 moves of 395 KB take 169 us, 5.5 TB/s. A truncation takes 1.2 us (8 sequences, within their last page) to 2.5 us (512 sequences
// that give back 66 pages each; 64 that give back 800 11 us).
// Counts of references change by integer atomics, whose order does not matter; where an order does matter (which free page
// goes to whom, which move stands where) places come from prefix sums, never from who came first. What needs those runs on one
// cluster of eight CTAs, which meet at the cluster's barrier instead of between launches.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <cstring>

#include "common.h"
#include "device_utils.cuh"
#include "flint/flint_b200.h"
#include "pages.h"
#include "sm100.cuh"

namespace {

constexpr int kMostArrays = 128;
constexpr int kChunkBytes = 8192;      // that a block copies at a time
// Up to which pools are small (their kernels' comments).
constexpr int kSmallPages = 32768;

__device__ int g_pages_error = 0;

struct Pool {
    int sequences, stride, pages, size, log_size;
};

// Numbers out of range are passed over and reported.
__device__ __forceinline__ void report() { atomicExch(&g_pages_error, 1); }

__device__ __forceinline__ int in_range(const Pool& pool, int given) {
    const int length = min(max(given, 0), pool.stride << pool.log_size);
    if (length != given) {
        report();
    }
    return length;
}
__device__ __forceinline__ int length_of(const Pool& pool, const int* lengths, int s) { return in_range(pool, lengths[s]); }
__device__ __forceinline__ int entries_of(const Pool& pool, int length) {
    return (length + pool.size - 1) >> pool.log_size;
}
__device__ __forceinline__ bool is_page(const Pool& pool, int page) {
    const bool is = page >= 0 && page < pool.pages;
    if (!is) {
        report();
    }
    return is;
}

// ---- one cluster's prefix sums ----------------------------------------------------------------------------

constexpr int kRanks = 8;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Everybody's earlier writes to global memory are visible behind it, too.
__device__ __forceinline__ void meet() {
    __threadfence();
    __syncwarp();
    sm100::cluster_sync_all();
}

template <typename T>
__device__ __forceinline__ T warp_prefix(T v, int lane) {      // inclusive
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const T other = __shfl_up_sync(fb::kFullMask, v, off);
        v += lane >= off ? other : 0;
    }
    return v;
}

// The sum of v over the threads before this one; `all` over the block. The last barrier leaves `scan` free.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T& all, long long (&scan)[kWarps]) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const T upto = warp_prefix(v, lane);
    if (lane == 31) {
        scan[warp] = upto;
    }
    __syncthreads();
    const T sums = warp_prefix(static_cast<T>(scan[lane]), lane);
    all = __shfl_sync(fb::kFullMask, sums, 31);
    const T before = __shfl_sync(fb::kFullMask, sums, max(warp - 1, 0));
    __syncthreads();
    return (warp > 0 ? before : 0) + upto - v;
}

// A CTA's share of `count` items, in order.
struct Slice {
    int begin, end;
    __device__ __forceinline__ Slice(int count, int rank) {
        const int each = (count + kRanks - 1) / kRanks;
        begin = min(count, rank * each);
        end = min(count, begin + each);
    }
};

// Puts a CTA's number where every CTA reads it behind the next meet().
__device__ __forceinline__ void publish(long long* shared_slots, int rank, long long value) {
    if (threadIdx.x < kRanks) {
        const uint32_t to = sm100::map_to_cta(sm100::smem_u32(shared_slots + rank), threadIdx.x);
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(value) : "memory");
    }
}
__device__ __forceinline__ long long sum_of(const long long* slots, int ranks) {
    long long sum = 0;
    for (int r = 0; r < ranks; ++r) {
        sum += slots[r];
    }
    return sum;
}

// ---- fork ---------------------------------------------------------------------------------------------

struct ForkArgs {
    Pool pool;
    int* next_table;
    int* next_lengths;
    int* next_references;
    const int* table;
    const int* lengths;
    const int* references;
    const int* parents;
};

// Tables, lengths, and the references to start from; a warp has a row, 32 entries at a time.
__global__ void __launch_bounds__(256) fb_pages_fork_tables(const ForkArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    const int lane = threadIdx.x % 32;
    const int warps = gridDim.x * 8, first = blockIdx.x * 8 + threadIdx.x / 32;
    for (int page = blockIdx.x * 256 + threadIdx.x; page < p.pool.pages; page += gridDim.x * 256) {
        p.next_references[page] = p.references[page];
    }
    for (int t = first; t < p.pool.sequences; t += warps) {
        const int parent = p.parents[t];
        const bool has = parent >= 0 && parent < p.pool.sequences;
        if (!has && parent != -1) {
            report();
        }
        const int length = has ? length_of(p.pool, p.lengths, parent) : 0;
        const int entries = entries_of(p.pool, length);
        for (int e = lane; e < p.pool.stride; e += 32) {
            p.next_table[static_cast<long long>(t) * p.pool.stride + e] =
                e < entries ? p.table[static_cast<long long>(parent) * p.pool.stride + e] : -1;
        }
        if (lane == 0) {
            p.next_lengths[t] = length;
        }
    }
}

// One reference less for what stood in the old tables, one more for what stands in the new ones.
__global__ void __launch_bounds__(256) fb_pages_fork_references(const ForkArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    const int lane = threadIdx.x % 32;
    const int warps = gridDim.x * 8, first = blockIdx.x * 8 + threadIdx.x / 32;
    for (int item = first; item < 2 * p.pool.sequences; item += warps) {
        const bool is_new = item >= p.pool.sequences;
        const int s = is_new ? item - p.pool.sequences : item;
        const int entries = entries_of(p.pool, length_of(p.pool, is_new ? p.next_lengths : p.lengths, s));
        const int* row = (is_new ? p.next_table : p.table) + static_cast<long long>(s) * p.pool.stride;
        for (int e = lane; e < entries; e += 32) {
            const int page = row[e];
            if (is_page(p.pool, page)) {
                atomicAdd(p.next_references + page, is_new ? 1 : -1);
            }
        }
    }
}

// The same in one launch, a thread of a cluster per entry: 8 sequences of 22 entries 15.9 us with what follows, 18.0 in two launches.
// (With several entries per thread the cluster is the slower one: 512 sequences of 66 entries 37.3 us, 35.4 in two launches.)
__global__ void __launch_bounds__(kThreads) fb_pages_fork_small(const ForkArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    const int i = static_cast<int>(sm100::cluster_cta_rank()) * kThreads + static_cast<int>(threadIdx.x);
    for (int page = i; page < p.pool.pages; page += kRanks * kThreads) {
        p.next_references[page] = p.references[page];
    }
    int had = -1, gets = -1;      // the page that the entry had, and the one that it gets; -1 for none
    if (i < p.pool.sequences * p.pool.stride) {
        const int t = static_cast<int>(static_cast<unsigned>(i) / static_cast<unsigned>(p.pool.stride)), e = i - t * p.pool.stride;
        const int parent = p.parents[t];
        const bool has = parent >= 0 && parent < p.pool.sequences;
        if (!has && parent != -1) {
            report();
        }
        const int before = length_of(p.pool, p.lengths, t), length = has ? length_of(p.pool, p.lengths, parent) : 0;
        const bool old = e < entries_of(p.pool, before), now = e < entries_of(p.pool, length);
        had = old ? p.table[i] : -1;
        gets = now ? p.table[parent * p.pool.stride + e] : -1;
        p.next_table[i] = gets;
        if (e == 0) {
            p.next_lengths[t] = length;
        }
        had = old && is_page(p.pool, had) ? had : -1;
        gets = now && is_page(p.pool, gets) ? gets : -1;
    }
    meet();
    if (had != gets) {
        if (gets >= 0) {
            atomicAdd(p.next_references + gets, 1);
        }
        if (had >= 0) {
            atomicAdd(p.next_references + had, -1);
        }
    }
}

// ---- truncate -------------------------------------------------------------------------------------------

struct TruncateArgs {
    Pool pool;
    int* table;
    int* lengths;
    int* references;
    const int* keep;
};

__global__ void __launch_bounds__(256) fb_pages_truncate(const TruncateArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    const int lane = threadIdx.x % 32;
    const int warps = gridDim.x * 8, first = blockIdx.x * 8 + threadIdx.x / 32;
    for (int s = first; s < p.pool.sequences; s += warps) {
        const int length = length_of(p.pool, p.lengths, s), keep = p.keep[s];
        if (keep < 0) {
            report();
        }
        const int kept = min(length, max(keep, 0));
        int* row = p.table + static_cast<long long>(s) * p.pool.stride;
        for (int e = entries_of(p.pool, kept) + lane; e < entries_of(p.pool, length); e += 32) {
            const int page = row[e];
            if (is_page(p.pool, page)) {
                atomicSub(p.references + page, 1);
            }
            row[e] = -1;
        }
        __syncwarp();      // (everybody has the length)
        if (lane == 0) {
            p.lengths[s] = kept;
        }
    }
}

// ---- reserve --------------------------------------------------------------------------------------------

struct ReserveArgs {
    Pool pool;
    int* table;
    int* lengths;
    int* references;
    int* moves;
    int* counts;
    const int* added;
    int* growers;      // [pages]: sequences that write into a page that they share, and
    int* lowest;       // [pages]: the first of them (both of pages with such sequences only)
    int* fresh;        // [pages]: free pages in order, as many as are needed
    int* needs;        // [sequences][2]: where a sequence's pages stand in that list, its move's place or -1
};

// (ReserveArgs' lists are used where shared memory has no room.)
struct Growth {
    int length, entries, fresh, last;     // last: the partly filled page that it writes into, or -1
};
__device__ __forceinline__ Growth growth_of(const ReserveArgs& p, int s) {
    Growth g;
    g.length = length_of(p.pool, p.lengths, s);
    const int given = p.added[s], added = min(max(given, 0), (p.pool.stride << p.pool.log_size) - g.length);
    if (added != given) {
        report();
    }
    g.entries = entries_of(p.pool, g.length);
    g.fresh = entries_of(p.pool, g.length + added) - g.entries;
    g.last = -1;
    if (added > 0 && (g.length & (p.pool.size - 1)) != 0) {
        const int page = p.table[static_cast<long long>(s) * p.pool.stride + g.entries - 1];
        g.last = is_page(p.pool, page) ? page : -1;
    }
    g.length += added;
    return g;
}

__global__ void __launch_bounds__(kThreads) fb_pages_reserve(const ReserveArgs p) {
    __shared__ long long scan[kWarps];
    __shared__ long long need_of[kRanks], copies_of[kRanks], free_of[kRanks];
    fb::dependency_wait();
    fb::dependency_release();
    sm100::cluster_sync_all();      // every CTA of the cluster runs before any writes to another one's memory
    const int rank = static_cast<int>(sm100::cluster_cta_rank()), tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const Slice mine(p.pool.sequences, rank), pages(p.pool.pages, rank);
    // How many sequences write into each partly filled page, and the first of them.
    for (int s = mine.begin + tid; s < mine.end; s += kThreads) {
        const Growth g = growth_of(p, s);
        if (g.last >= 0) {
            p.growers[g.last] = 0;
            p.lowest[g.last] = INT_MAX;
        }
    }
    // Meanwhile: free pages in this CTA's share.
    int frees = 0;
    for (int page = pages.begin + tid; page < pages.end; page += kThreads) {
        frees += p.references[page] == 0 ? 1 : 0;
    }
    block_prefix(frees, frees, scan);
    publish(free_of, rank, frees);
    meet();
    for (int s = mine.begin + tid; s < mine.end; s += kThreads) {
        const Growth g = growth_of(p, s);
        if (g.last >= 0) {
            atomicAdd(p.growers + g.last, 1);
            atomicMin(p.lowest + g.last, s);
        }
    }
    meet();
    auto copies = [&](const Growth& g, int s) {
        return g.last >= 0 && !(p.growers[g.last] >= p.references[g.last] && p.lowest[g.last] == s);
    };
    long long need = 0;      // (sequences can ask for more than 2^31 pages together)
    int moved = 0;
    for (int s = mine.begin + tid; s < mine.end; s += kThreads) {
        const Growth g = growth_of(p, s);
        const int copy = copies(g, s) ? 1 : 0;
        need += g.fresh + copy;
        moved += copy;
    }
    block_prefix(need, need, scan);
    block_prefix(moved, moved, scan);
    publish(need_of, rank, need);
    publish(copies_of, rank, moved);
    meet();
    const long long all_need = sum_of(need_of, kRanks), all_free = sum_of(free_of, kRanks);
    const int all_moves = all_need <= all_free ? static_cast<int>(sum_of(copies_of, kRanks)) : 0;
    if (rank == 0 && tid == 0) {
        p.counts[0] = all_moves;
        p.counts[1] = static_cast<int>(min(max(all_need - all_free, 0LL), static_cast<long long>(INT_MAX)));
    }
    for (int i = all_moves + rank * kThreads + tid; i < p.pool.sequences; i += kRanks * kThreads) {
        p.moves[2 * i] = p.moves[2 * i + 1] = -1;
    }
    if (all_need <= all_free) {      // (one outcome for the whole cluster)
        // The free pages in order, and every sequence's place among those who need some.
        int at = static_cast<int>(sum_of(free_of, rank));
        for (int from = pages.begin; from < pages.end && at < all_need; from += kThreads) {
            const int page = from + tid;
            const bool is = page < pages.end && p.references[page] == 0;
            int here = 0;
            const int place = at + block_prefix(is ? 1 : 0, here, scan);
            if (is && place < all_need) {
                p.fresh[place] = page;
            }
            at += here;
        }
        int place = static_cast<int>(sum_of(need_of, rank)), move = static_cast<int>(sum_of(copies_of, rank));
        for (int from = mine.begin; from < mine.end; from += kThreads) {
            const int s = from + tid;
            int its = 0, copy = 0;
            if (s < mine.end) {
                const Growth g = growth_of(p, s);
                copy = copies(g, s) ? 1 : 0;
                its = g.fresh + copy;
            }
            int here = 0, moves = 0;
            const int before = place + block_prefix(its, here, scan), move_before = move + block_prefix(copy, moves, scan);
            if (s < mine.end) {
                p.needs[2 * s] = before;
                p.needs[2 * s + 1] = copy != 0 ? move_before : -1;
            }
            place += here;
            move += moves;
        }
    }
    meet();      // (references and who copies are read, by everybody)
    if (all_need > all_free) {
        return;
    }
    for (int s = mine.begin + warp; s < mine.end; s += kWarps) {
        const Growth g = growth_of(p, s);
        int place = p.needs[2 * s];
        const int move = p.needs[2 * s + 1];
        int* row = p.table + static_cast<long long>(s) * p.pool.stride;
        if (move >= 0) {
            const int page = p.fresh[place++];
            if (lane == 0) {
                p.moves[2 * move] = g.last;
                p.moves[2 * move + 1] = page;
                atomicSub(p.references + g.last, 1);
                p.references[page] = 1;
                row[g.entries - 1] = page;
            }
        }
        for (int e = lane; e < g.fresh; e += 32) {
            const int page = p.fresh[place + e];
            p.references[page] = 1;
            row[g.entries + e] = page;
        }
        __syncwarp();      // (everybody has the length)
        if (lane == 0) {
            p.lengths[s] = g.length;
        }
    }
}

// The same for up to a thread per sequence and pools that are read soon: one block, whose barriers take a tenth of a cluster's (512
// sequences on 3,500 pages 37.3 us with what else a step does, 47.9 with the cluster; 8 sequences 15.9 and 19.3).
// Sequences that write into the same page meet in a table of pages in shared memory.
constexpr int kSlots = 2048;
constexpr int kListed = 4096;      // free pages that shared memory holds

__global__ void __launch_bounds__(kThreads) fb_pages_reserve_small(const ReserveArgs p) {
    __shared__ long long scan[kWarps];
    __shared__ int page_of_slot[kSlots], growers[kSlots], lowest[kSlots];
    __shared__ int listed[kListed];
    fb::dependency_wait();
    fb::dependency_release();
    const int tid = static_cast<int>(threadIdx.x), lane = tid % 32, s = tid;
    const bool is = s < p.pool.sequences;
    Growth g = {0, 0, 0, -1};
    if (is) {
        g = growth_of(p, s);
    }
    const int references = g.last >= 0 ? p.references[g.last] : 0;
    // Free pages among the first 4,096, four per thread.
    auto free_of = [&](int at) {      // a bit for each of four pages
        unsigned free = 0;
        if (at + 4 <= p.pool.pages) {
            const int4 four = *reinterpret_cast<const int4*>(p.references + at);
            free = (four.x == 0 ? 1u : 0u) | (four.y == 0 ? 2u : 0u) | (four.z == 0 ? 4u : 0u) | (four.w == 0 ? 8u : 0u);
        } else {
            for (int i = 0; at + i < p.pool.pages; ++i) {
                free |= p.references[at + i] == 0 ? 1u << i : 0u;
            }
        }
        return free;
    };
    unsigned free = free_of(4 * tid);
    for (int i = tid; i < kSlots; i += kThreads) {
        page_of_slot[i] = -1;
        growers[i] = 0;
        lowest[i] = INT_MAX;
    }
    __syncthreads();
    int slot = 0;
    if (g.last >= 0) {
        slot = static_cast<int>((static_cast<unsigned>(g.last) * 2654435761u) >> 21);
        static_assert(kSlots == 1 << (32 - 21) && kSlots > kThreads, "the table is never full");
        for (;;) {
            const int before = atomicCAS(&page_of_slot[slot], -1, g.last);
            if (before == -1 || before == g.last) {
                break;
            }
            slot = (slot + 1) % kSlots;
        }
        atomicAdd(&growers[slot], 1);
        atomicMin(&lowest[slot], s);
    }
    __syncthreads();
    const bool copies = g.last >= 0 && !(growers[slot] >= references && lowest[slot] == s);
    // Pages that are needed, and in the upper bits copies.
    constexpr int kShift = 44;
    const long long mine = static_cast<long long>(g.fresh) + (copies ? 1 + (1LL << kShift) : 0);
    long long all = 0;
    const long long before = block_prefix(mine, all, scan);
    const long long all_need = all & ((1LL << kShift) - 1);
    int place = 0;
    long long found = 0;
    for (int from = 0; from < p.pool.pages && found < all_need; from += 4 * kThreads) {
        if (from > 0) {
            free = free_of(from + 4 * tid);
        }
        int here = 0;
        long long at = found + block_prefix(__popc(free), here, scan);
        for (; free != 0 && at < all_need; free &= free - 1, ++at) {
            const int page = from + 4 * tid + __ffs(free) - 1;
            if (at < kListed) {
                listed[at] = page;
            } else {
                p.fresh[at] = page;
            }
        }
        found += here;
    }
    const bool enough = found >= all_need;
    const int all_moves = enough ? static_cast<int>(all >> kShift) : 0;
    if (tid == 0) {
        p.counts[0] = all_moves;
        p.counts[1] = static_cast<int>(min(max(all_need - found, 0LL), static_cast<long long>(INT_MAX)));
    }
    if (s >= all_moves && is) {
        p.moves[2 * s] = p.moves[2 * s + 1] = -1;
    }
    __syncthreads();      // the list is written, and references are read
    if (!enough) {
        return;
    }
    auto page_at = [&](int i) { return i < kListed ? listed[i] : p.fresh[i]; };
    place = static_cast<int>(before & ((1LL << kShift) - 1));
    int* row = p.table + static_cast<long long>(s) * p.pool.stride;
    if (copies) {
        const int page = page_at(place++), move = static_cast<int>(before >> kShift);
        p.moves[2 * move] = g.last;
        p.moves[2 * move + 1] = page;
        atomicSub(p.references + g.last, 1);
        p.references[page] = 1;
        row[g.entries - 1] = page;
    }
    if (is) {
        p.lengths[s] = g.length;
    }
    // A warp's sequences one by one where one has many pages, else all at once.
    if (__any_sync(fb::kFullMask, g.fresh > 4)) {
        for (int l = 0; l < 32; ++l) {
            const int count = __shfl_sync(fb::kFullMask, g.fresh, l), at = __shfl_sync(fb::kFullMask, place, l);
            const int entries = __shfl_sync(fb::kFullMask, g.entries, l);
            int* its = p.table + static_cast<long long>(s - lane + l) * p.pool.stride + entries;
            for (int e = lane; e < count; e += 32) {
                const int page = page_at(at + e);
                p.references[page] = 1;
                its[e] = page;
            }
        }
    } else {
        for (int e = 0; e < g.fresh; ++e) {
            const int page = page_at(place + e);
            p.references[page] = 1;
            row[g.entries + e] = page;
        }
    }
}

// ---- compact --------------------------------------------------------------------------------------------

struct CompactArgs {
    Pool pool;
    int* next_table;
    int* next_references;
    int* moves;
    int* counts;
    const int* table;
    const int* lengths;
    const int* references;
    int* number;       // [pages]: a used page's new number
    int* sources;      // [pages / 2] used pages behind the place of the last one, in order
    int* holes;        // [pages / 2] free pages before it
};

__global__ void __launch_bounds__(kThreads) fb_pages_compact(const CompactArgs p) {
    __shared__ long long scan[kWarps];
    __shared__ long long used_of[kRanks], below_of[kRanks];
    fb::dependency_wait();
    fb::dependency_release();
    sm100::cluster_sync_all();      // every CTA of the cluster runs before any writes to another one's memory
    const int rank = static_cast<int>(sm100::cluster_cta_rank()), tid = threadIdx.x;
    const Slice pages(p.pool.pages, rank);
    int used = 0;
    for (int page = pages.begin + tid; page < pages.end; page += kThreads) {
        used += p.references[page] > 0 ? 1 : 0;
    }
    block_prefix(used, used, scan);
    publish(used_of, rank, used);
    meet();
    const int count = static_cast<int>(sum_of(used_of, kRanks));
    int below = 0;      // used pages before the place of the last one
    for (int page = pages.begin + tid; page < min(pages.end, count); page += kThreads) {
        below += p.references[page] > 0 ? 1 : 0;
    }
    block_prefix(below, below, scan);
    publish(below_of, rank, below);
    meet();
    const int staying = static_cast<int>(sum_of(below_of, kRanks)), moved = count - staying;
    if (rank == 0 && tid == 0) {
        p.counts[0] = moved;
        p.counts[1] = count;
    }
    int before = static_cast<int>(sum_of(used_of, rank));
    for (int from = pages.begin; from < pages.end; from += kThreads) {
        const int page = from + tid;
        const bool is = page < pages.end && p.references[page] > 0;
        int here = 0;
        const int place = before + block_prefix(is ? 1 : 0, here, scan);     // used pages before this one
        if (page < pages.end) {
            if (is && page >= count) {
                p.sources[place - staying] = page;
            } else if (!is && page < count) {
                p.holes[page - place] = page;
            }
            if (is && page < count) {
                p.number[page] = page;
                p.next_references[page] = p.references[page];
            } else if (page >= count) {
                p.next_references[page] = 0;
            }
        }
        before += here;
    }
    meet();
    for (int i = rank * kThreads + tid; i < p.pool.pages / 2; i += kRanks * kThreads) {
        const int from = i < moved ? p.sources[i] : -1, to = i < moved ? p.holes[i] : -1;
        p.moves[2 * i] = from;
        p.moves[2 * i + 1] = to;
        if (i < moved) {
            p.number[from] = to;
            p.next_references[to] = p.references[from];
        }
    }
    // (The cluster's writes are complete for the launch behind this one, which waits for it.)
}

__global__ void __launch_bounds__(256) fb_pages_renumber(const CompactArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    const int lane = threadIdx.x % 32;
    const int warps = gridDim.x * 8, first = blockIdx.x * 8 + threadIdx.x / 32;
    for (int s = first; s < p.pool.sequences; s += warps) {
        const int entries = entries_of(p.pool, length_of(p.pool, p.lengths, s));
        const long long row = static_cast<long long>(s) * p.pool.stride;
        for (int e = lane; e < p.pool.stride; e += 32) {
            int number = -1;
            if (e < entries) {
                const int page = p.table[row + e];
                // (A page that stands in a table and has no reference has no number.)
                if (is_page(p.pool, page)) {
                    if (p.references[page] > 0) {
                        number = p.number[page];
                    } else {
                        report();
                    }
                }
            }
            p.next_table[row + e] = number;
        }
    }
}

// ---- copying pages -----------------------------------------------------------------------------------------

struct CopyArgs {
    const int* moves;
    const int* counts;
    long long most_moves;
    int pages, arrays, chunks;             // chunks: of all arrays, per move
    int first_chunk[kMostArrays + 1];
    unsigned bytes[kMostArrays];           // of a page
    unsigned char* base[kMostArrays];
};

// Blocks take chunks of 8 KB, of one array and move each: bound by HBM. Neither end is read again soon, which the loads and stores
// say (1,175 moves of 395 KB 189 us with the compaction, 179 so; chunks of 16 KB 181).
__global__ void __launch_bounds__(256) fb_pages_copy(const __grid_constant__ CopyArgs p) {
    fb::dependency_wait();
    fb::dependency_release();
    const long long moves = min(static_cast<long long>(max(p.counts[0], 0)), p.most_moves);
    // Items blockIdx + k gridDim, in moves and chunks of them (one division where every item would take a long one).
    const int more_moves = static_cast<int>(gridDim.x) / p.chunks, more_chunks = static_cast<int>(gridDim.x) - more_moves * p.chunks;
    long long move = static_cast<int>(blockIdx.x) / p.chunks;
    int chunk = static_cast<int>(blockIdx.x) - static_cast<int>(move) * p.chunks;
    for (; move < moves; move += more_moves, chunk += more_chunks, move += chunk >= p.chunks ? 1 : 0,
                         chunk -= chunk >= p.chunks ? p.chunks : 0) {
        const int from = p.moves[2 * move], to = p.moves[2 * move + 1];
        if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
            if (from != -1 || to != -1) {
                report();
            }
            continue;
        }
        int low = 0, high = p.arrays - 1;       // the last array that begins at or before the chunk
        while (low < high) {
            const int middle = (low + high + 1) / 2;
            if (p.first_chunk[middle] <= chunk) {
                low = middle;
            } else {
                high = middle - 1;
            }
        }
        const unsigned bytes = p.bytes[low], begin = static_cast<unsigned>(chunk - p.first_chunk[low]) * kChunkBytes;
        const unsigned here = min(bytes - begin, static_cast<unsigned>(kChunkBytes));
        const unsigned char* source = p.base[low] + static_cast<size_t>(from) * bytes + begin;
        unsigned char* target = p.base[low] + static_cast<size_t>(to) * bytes + begin;
        if (bytes % 16 == 0) {      // (then the array begins on such a boundary: layer_alignment)
            constexpr int kWords = kChunkBytes / (256 * 16);
            uint4 held[kWords];
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const unsigned at = (i * 256 + threadIdx.x) * 16;
                if (at < here) {
                    held[i] = __ldcs(reinterpret_cast<const uint4*>(source + at));
                }
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const unsigned at = (i * 256 + threadIdx.x) * 16;
                if (at < here) {
                    __stcs(reinterpret_cast<uint4*>(target + at), held[i]);
                }
            }
        } else {
            for (unsigned at = threadIdx.x * 4; at < here; at += 1024) {
                *reinterpret_cast<unsigned*>(target + at) = *reinterpret_cast<const unsigned*>(source + at);
            }
        }
    }
}

// ---- entry points --------------------------------------------------------------------------------------------

constexpr flint_status kBad = FLINT_ERROR_INVALID_ARGUMENT;
constexpr size_t kMostSequences = 65535;
constexpr size_t kMostPages = size_t{1} << 24;

flint_status check_pool(const char* name, const flint_b200_page_pool* pool, Pool* out) {
    if (pool == nullptr) {
        return fb::fail(kBad, "%s: pool is null", name);
    }
    if (pool->sequences > kMostSequences) {
        return fb::fail(kBad, "%s: sequences (%zu) can be up to %zu", name, pool->sequences, kMostSequences);
    }
    if (pool->pages == 0 || pool->pages > kMostPages) {
        return fb::fail(kBad, "%s: pages (%zu) must be from 1 to %zu", name, pool->pages, kMostPages);
    }
    const size_t size = pool->page_size;
    if (size < 16 || size > 1024 || (size & (size - 1)) != 0) {
        return fb::fail(kBad, "%s: page_size (%zu) must be a power of two from 16 to 1024", name, size);
    }
    if (pool->table_stride == 0 || pool->table_stride > (size_t{1} << 26) / size) {
        return fb::fail(kBad, "%s: table_stride (%zu) must be from 1 to %zu", name, pool->table_stride,
                        (size_t{1} << 26) / size);
    }
    out->sequences = static_cast<int>(pool->sequences);
    out->stride = static_cast<int>(pool->table_stride);
    out->pages = static_cast<int>(pool->pages);
    out->size = static_cast<int>(size);
    out->log_size = 0;
    while ((1 << out->log_size) < out->size) {
        ++out->log_size;
    }
    return FLINT_OK;
}

// Three lists of pages and two numbers per sequence.
size_t workspace_bytes_of(const Pool& pool) {
    return (3 * static_cast<size_t>(pool.pages) + 2 * static_cast<size_t>(pool.sequences)) * 4 + 16;
}

flint_status check_workspace(const char* name, const Pool& pool, size_t given) {
    if (given < workspace_bytes_of(pool)) {
        return fb::fail(kBad, "%s: needs %zu bytes of workspace, given %zu", name, workspace_bytes_of(pool), given);
    }
    return FLINT_OK;
}

size_t table_bytes(const Pool& pool) { return static_cast<size_t>(pool.sequences) * pool.stride * 4; }
size_t row_bytes(const Pool& pool) { return static_cast<size_t>(pool.sequences) * 4; }
size_t page_numbers(const Pool& pool) { return static_cast<size_t>(pool.pages) * 4; }

// No sequences, or one page, leave nothing in some of the lists: those may be null, and stand as something that overlaps
// nothing.
fb::Span list(const char* what, const void* pointer, size_t bytes, const void* instead) {
    return bytes != 0 ? fb::Span{what, pointer, bytes} : fb::Span{what, instead, 0};
}

// A warp per sequence, or a thread per page, up to eight blocks on every SM.
cudaError_t row_grid(long long warps, long long threads, dim3* grid) {
    int sms = 148;
    const cudaError_t e = fb::sm_count(&sms);
    const long long blocks = std::max((warps + 7) / 8, (threads + 255) / 256);
    *grid = dim3(static_cast<unsigned>(std::min<long long>(std::max<long long>(blocks, 1), 8LL * sms)));
    return e;
}

}  // namespace

namespace fb {

cudaError_t pages_error_flag(int* value, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(value, g_pages_error, sizeof(int));
    if (e == cudaSuccess && reset && *value != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_pages_error, &zero, sizeof(int));
    }
    return e;
}

}  // namespace fb

extern "C" {

flint_status flint_b200_pages_workspace(const flint_b200_page_pool* shape, size_t* bytes) {
    constexpr const char* name = "flint_b200_pages_workspace";
    Pool pool;
    FB_TRY(check_pool(name, shape, &pool));
    if (bytes == nullptr) {
        return fb::fail(kBad, "%s: bytes is null", name);
    }
    *bytes = workspace_bytes_of(pool);
    return FLINT_OK;
}

flint_status flint_b200_pages_fork(void* next_table, void* next_lengths, void* next_references,
                                   const void* page_table, const void* lengths, const void* references,
                                   const void* parents, const flint_b200_page_pool* shape, flint_stream stream) {
    constexpr const char* name = "flint_b200_pages_fork";
    Pool pool;
    FB_TRY(check_pool(name, shape, &pool));
    const fb::Span spans[] = {
        list("next_table", next_table, table_bytes(pool), references),
        list("next_lengths", next_lengths, row_bytes(pool), references),
        {"next_references", next_references, page_numbers(pool)},
        list("page_table", page_table, table_bytes(pool), references),
        list("lengths", lengths, row_bytes(pool), references),
        {"references", references, page_numbers(pool)},
        list("parents", parents, row_bytes(pool), references),
    };
    FB_TRY(fb::check_spans(name, spans, 3));
    const ForkArgs p = {pool,
                        static_cast<int*>(next_table),
                        static_cast<int*>(next_lengths),
                        static_cast<int*>(next_references),
                        static_cast<const int*>(page_table),
                        static_cast<const int*>(lengths),
                        static_cast<const int*>(references),
                        static_cast<const int*>(parents)};
    if (static_cast<long long>(pool.sequences) * pool.stride <= kRanks * kThreads && pool.pages <= kSmallPages) {
        FB_CUDA(fb::launch_dependent_cluster(fb_pages_fork_small, dim3(kRanks), dim3(kThreads), kRanks, 0, stream, p));
        return FLINT_OK;
    }
    dim3 grid;
    FB_CUDA(row_grid(pool.sequences, pool.pages, &grid));
    FB_CUDA(fb::launch_dependent(fb_pages_fork_tables, grid, dim3(256), 0, stream, p));
    if (pool.sequences > 0) {
        FB_CUDA(row_grid(2LL * pool.sequences, 0, &grid));
        FB_CUDA(fb::launch_dependent(fb_pages_fork_references, grid, dim3(256), 0, stream, p));
    }
    return FLINT_OK;
}

flint_status flint_b200_pages_reserve(void* page_table, void* lengths, void* references, void* moves, void* counts,
                                      const void* added, const flint_b200_page_pool* shape, void* workspace,
                                      size_t workspace_bytes, flint_stream stream) {
    constexpr const char* name = "flint_b200_pages_reserve";
    Pool pool;
    FB_TRY(check_pool(name, shape, &pool));
    FB_TRY(check_workspace(name, pool, workspace_bytes));
    const fb::Span spans[] = {
        list("page_table", page_table, table_bytes(pool), references),
        list("lengths", lengths, row_bytes(pool), references),
        {"references", references, page_numbers(pool)},
        list("moves", moves, 2 * row_bytes(pool), references),
        {"counts", counts, 8},
        {"workspace", workspace, workspace_bytes_of(pool)},
        list("added", added, row_bytes(pool), references),
    };
    FB_TRY(fb::check_spans(name, spans, 6));
    int* space = static_cast<int*>(workspace);
    const size_t pages = static_cast<size_t>(pool.pages);
    const ReserveArgs p = {pool,
                           static_cast<int*>(page_table),
                           static_cast<int*>(lengths),
                           static_cast<int*>(references),
                           static_cast<int*>(moves),
                           static_cast<int*>(counts),
                           static_cast<const int*>(added),
                           space,
                           space + pages,
                           space + 2 * pages,
                           space + 3 * pages};
    if (pool.sequences <= kThreads && pool.pages <= kSmallPages) {
        FB_CUDA(fb::launch_dependent(fb_pages_reserve_small, dim3(1), dim3(kThreads), 0, stream, p));
        return FLINT_OK;
    }
    FB_CUDA(fb::launch_dependent_cluster(fb_pages_reserve, dim3(kRanks), dim3(kThreads), kRanks, 0, stream, p));
    return FLINT_OK;
}

flint_status flint_b200_pages_truncate(void* page_table, void* lengths, void* references, const void* keep,
                                       const flint_b200_page_pool* shape, flint_stream stream) {
    constexpr const char* name = "flint_b200_pages_truncate";
    Pool pool;
    FB_TRY(check_pool(name, shape, &pool));
    if (pool.sequences == 0) {
        return FLINT_OK;
    }
    const fb::Span spans[] = {
        {"page_table", page_table, table_bytes(pool)},
        {"lengths", lengths, row_bytes(pool)},
        {"references", references, page_numbers(pool)},
        {"keep", keep, row_bytes(pool)},
    };
    FB_TRY(fb::check_spans(name, spans, 3));
    const TruncateArgs p = {pool, static_cast<int*>(page_table), static_cast<int*>(lengths),
                            static_cast<int*>(references), static_cast<const int*>(keep)};
    dim3 grid;
    FB_CUDA(row_grid(pool.sequences, 0, &grid));
    FB_CUDA(fb::launch_dependent(fb_pages_truncate, grid, dim3(256), 0, stream, p));
    return FLINT_OK;
}

flint_status flint_b200_pages_compact(void* next_table, void* next_references, void* moves, void* counts,
                                      const void* page_table, const void* lengths, const void* references,
                                      const flint_b200_page_pool* shape, void* workspace, size_t workspace_bytes,
                                      flint_stream stream) {
    constexpr const char* name = "flint_b200_pages_compact";
    Pool pool;
    FB_TRY(check_pool(name, shape, &pool));
    FB_TRY(check_workspace(name, pool, workspace_bytes));
    const fb::Span spans[] = {
        list("next_table", next_table, table_bytes(pool), references),
        {"next_references", next_references, page_numbers(pool)},
        list("moves", moves, static_cast<size_t>(pool.pages / 2) * 8, references),
        {"counts", counts, 8},
        {"workspace", workspace, workspace_bytes_of(pool)},
        list("page_table", page_table, table_bytes(pool), references),
        list("lengths", lengths, row_bytes(pool), references),
        {"references", references, page_numbers(pool)},
    };
    FB_TRY(fb::check_spans(name, spans, 5));
    int* space = static_cast<int*>(workspace);
    const size_t pages = static_cast<size_t>(pool.pages);
    const CompactArgs p = {pool,
                           static_cast<int*>(next_table),
                           static_cast<int*>(next_references),
                           static_cast<int*>(moves),
                           static_cast<int*>(counts),
                           static_cast<const int*>(page_table),
                           static_cast<const int*>(lengths),
                           static_cast<const int*>(references),
                           space,
                           space + pages,
                           space + 2 * pages};
    FB_CUDA(fb::launch_dependent_cluster(fb_pages_compact, dim3(kRanks), dim3(kThreads), kRanks, 0, stream, p));
    if (pool.sequences > 0) {
        dim3 grid;
        FB_CUDA(row_grid(pool.sequences, 0, &grid));
        FB_CUDA(fb::launch_dependent(fb_pages_renumber, grid, dim3(256), 0, stream, p));
    }
    return FLINT_OK;
}

flint_status flint_b200_pages_copy(void* const* arrays, const size_t* page_bytes, size_t count, size_t pages,
                                   const void* moves, const void* counts, size_t most_moves, flint_stream stream) {
    constexpr const char* name = "flint_b200_pages_copy";
    if (count > static_cast<size_t>(kMostArrays)) {
        return fb::fail(kBad, "%s: count (%zu) can be up to %d", name, count, kMostArrays);
    }
    if (pages > kMostPages || most_moves > kMostPages) {
        return fb::fail(kBad, "%s: pages (%zu) and most_moves (%zu) can be up to %zu", name, pages, most_moves,
                        kMostPages);
    }
    if (count == 0 || pages == 0 || most_moves == 0) {
        return FLINT_OK;
    }
    if (arrays == nullptr || page_bytes == nullptr) {
        return fb::fail(kBad, "%s: %s is null", name, arrays == nullptr ? "arrays" : "page_bytes");
    }
    CopyArgs p;
    std::memset(&p, 0, sizeof p);
    fb::Span spans[kMostArrays + 2];
    constexpr size_t kMostBytes = size_t{1} << 28;
    long long chunks = 0;
    for (size_t i = 0; i < count; ++i) {
        if (page_bytes[i] == 0 || page_bytes[i] % 4 != 0 || page_bytes[i] > kMostBytes) {
            return fb::fail(kBad, "%s: page_bytes[%zu] (%zu) must be a multiple of 4 from 4 to %zu", name, i,
                            page_bytes[i], kMostBytes);
        }
        p.first_chunk[i] = static_cast<int>(chunks);
        p.bytes[i] = static_cast<unsigned>(page_bytes[i]);
        p.base[i] = static_cast<unsigned char*>(arrays[i]);
        chunks += static_cast<long long>((page_bytes[i] + kChunkBytes - 1) / kChunkBytes);
        spans[i] = fb::Span{"an array", arrays[i], pages * page_bytes[i], fb::layer_alignment(pages * page_bytes[i])};
    }
    p.first_chunk[count] = static_cast<int>(chunks);
    spans[count] = fb::Span{"moves", moves, most_moves * 8};
    spans[count + 1] = fb::Span{"counts", counts, 8};
    FB_TRY(fb::check_spans(name, spans, count + 2, count));
    p.moves = static_cast<const int*>(moves);
    p.counts = static_cast<const int*>(counts);
    p.most_moves = static_cast<long long>(most_moves);
    p.pages = static_cast<int>(pages);
    p.arrays = static_cast<int>(count);
    p.chunks = static_cast<int>(chunks);
    int sms = 148;
    FB_CUDA(fb::sm_count(&sms));
    const long long blocks = std::min<long long>(p.most_moves * chunks, 8LL * sms);
    FB_CUDA(fb::launch_dependent(fb_pages_copy, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p));
    return FLINT_OK;
}

}  // extern "C"
