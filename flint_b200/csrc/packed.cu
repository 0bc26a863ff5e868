// Attention over sequences of different lengths, packed one behind the other or in the pages of a
// cache, and the entry points of both (extensions: the reference has equal lengths only,
// src/api/gpt2.cpp:495-530).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "common.h"
#include "device_utils.cuh"
#include "flint/flint_b200.h"
#include "packed.cuh"
#include "packed_maps.h"

namespace fb {
namespace {

constexpr int kHead = 64;

// Copies the new tokens' keys and values into their pages: eight lanes per row of 64 values.
__global__ void __launch_bounds__(256)
    fb_paged_store(const PackedArgs p, __half* k_pages, __half* v_pages) {
    fb::dependency_wait();
    fb::dependency_release();
    const int piece = threadIdx.x % 8;
    const long long first = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / 8;
    const long long stride = static_cast<long long>(gridDim.x) * 32;
    for (int s = blockIdx.y; s < p.sequences; s += gridDim.y) {
        const Sequence q = sequence_at(p, s);
        for (long long item = first; item < static_cast<long long>(q.count) * p.kv_heads * 2; item += stride) {
            const int which = static_cast<int>(item % 2);
            const int head = static_cast<int>(item / 2 % p.kv_heads);
            const int i = static_cast<int>(item / 2 / p.kv_heads);
            const int key = q.keys - q.count + i;
            if (key < 0) {
                continue;
            }
            const long long page = page_of(p, s, key);
            if (page < 0) {
                continue;
            }
            const __half* from = (which == 0 ? p.k : p.v) + (q.first + static_cast<long long>(i)) * p.kv_stride +
                                 head * kHead;
            __half* to = (which == 0 ? k_pages : v_pages) +
                         ((page * p.kv_heads + head) * p.page_size + key % p.page_size) * kHead;
            reinterpret_cast<uint4*>(to)[piece] = reinterpret_cast<const uint4*>(from)[piece];
        }
    }
}

dim3 sequence_grid(const PackedArgs& p, int items_per_block, long long items, int sms) {
    const long long per_sequence = (items / std::max(1, p.sequences) + items_per_block) / items_per_block;
    const unsigned y = static_cast<unsigned>(std::min(p.sequences, 65535));
    const long long most = std::max<long long>(1, 16LL * sms / y + 1);
    return dim3(static_cast<unsigned>(std::min(std::max<long long>(1, 2 * per_sequence), most)), y);
}

}  // namespace

namespace {

constexpr unsigned kHeadWidth = 64;

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encode_fn(EncodeTiled* out) {
    static std::atomic<EncodeTiled> cached{nullptr};
    EncodeTiled found = cached.load(std::memory_order_relaxed);
    if (found == nullptr) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult status;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &status);
        if (e != cudaSuccess) {
            return e;
        }
        if (status != cudaDriverEntryPointSuccess || fn == nullptr) {
            return cudaErrorNotSupported;
        }
        found = reinterpret_cast<EncodeTiled>(fn);
        cached.store(found, std::memory_order_relaxed);
    }
    *out = found;
    return cudaSuccess;
}

cudaError_t encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                   const cuuint32_t* box) {
    EncodeTiled fn = nullptr;
    const cudaError_t e = encode_fn(&fn);
    if (e != cudaSuccess) {
        return e;
    }
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank), const_cast<void*>(base),
                          dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace

cudaError_t encode_rows(CUtensorMap* map, const __half* base, int heads, int rows, long long stride, int box_heads,
                        int box_rows) {
    const cuuint64_t dims[3] = {kHeadWidth, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[2] = {kHeadWidth * 2, static_cast<cuuint64_t>(stride) * 2};
    const cuuint32_t box[3] = {kHeadWidth, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
    return encode(map, base, 3, dims, strides, box);
}

cudaError_t encode_pages(CUtensorMap* map, const __half* base, long long rows, int box_rows) {
    const cuuint64_t dims[2] = {kHeadWidth, static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {kHeadWidth * 2};
    const cuuint32_t box[2] = {kHeadWidth, static_cast<cuuint32_t>(box_rows)};
    return encode(map, base, 2, dims, strides, box);
}

cudaError_t packed_error_flag(int* value, bool reset) {
    int here = 0, forward = 0, backward = 0;
    cudaError_t e = read_error_word(&here, reset);
    if (e == cudaSuccess) e = packed_forward_error_flag(&forward, reset);
    if (e == cudaSuccess) e = packed_backward_error_flag(&backward, reset);
    *value = here != 0 || forward != 0 || backward != 0 ? 1 : 0;
    return e;
}

}  // namespace fb

// ---- entry points ------------------------------------------------------------------------------

namespace {

constexpr flint_status kBad = FLINT_ERROR_INVALID_ARGUMENT;
constexpr size_t kMostSequences = 65535;
constexpr size_t kMostRows = size_t{1} << 24;
constexpr size_t kMostHeads = 1024;
constexpr size_t kMostGroup = 128;
constexpr size_t kMostStride = size_t{1} << 24;

flint_status check_rows(const char* name, size_t sequences, size_t rows, size_t heads, size_t kv_heads,
                        size_t head_width, size_t q_stride, size_t kv_stride, size_t o_stride) {
    if (sequences > kMostSequences || rows > kMostRows) {
        return fb::fail(kBad, "%s: sequences (%zu) can be up to %zu, and rows (%zu) up to %zu", name, sequences,
                        kMostSequences, rows, kMostRows);
    }
    if (kv_heads == 0 || heads == 0 || heads > kMostHeads || heads % kv_heads != 0 || heads / kv_heads > kMostGroup) {
        return fb::fail(kBad,
                        "%s: heads (%zu) must be from 1 to %zu and a multiple of kv_heads (%zu), up to %zu times it",
                        name, heads, kMostHeads, kv_heads, kMostGroup);
    }
    if (head_width != 64) {
        return fb::fail(kBad, "%s: head_width (%zu) must be 64", name, head_width);
    }
    const struct {
        const char* name;
        size_t value, least;
    } strides[] = {{"q_stride", q_stride, heads * 64}, {"kv_stride", kv_stride, kv_heads * 64},
                   {"o_stride", o_stride, heads * 64}};
    for (const auto& s : strides) {
        if (s.value % 8 != 0 || s.value < s.least || s.value > kMostStride) {
            return fb::fail(kBad, "%s: %s (%zu) must be a multiple of 8 from %zu to %zu", name, s.name, s.value,
                            s.least, kMostStride);
        }
    }
    return FLINT_OK;
}

flint_status check_scale(const char* name, float scale) {
    if (!std::isfinite(scale) || scale <= 0.0f) {
        return fb::fail(kBad, "%s: scale (%g) must be finite and positive", name, static_cast<double>(scale));
    }
    return FLINT_OK;
}

// A matrix of `rows` rows of `width` bytes, `stride` bytes apart; a contiguous array is one row.
struct Rows {
    const char* name;
    const void* pointer;
    size_t rows, width, stride;
    size_t bytes() const { return rows == 0 ? 0 : (rows - 1) * stride + width; }
};

bool rows_overlap(const Rows& a, const Rows& b) {
    if (!fb::overlap(a.pointer, a.bytes(), b.pointer, b.bytes())) {
        return false;
    }
    if (a.rows < 2 || b.rows < 2 || a.stride != b.stride) {
        return true;
    }
    // Columns of one matrix of rows do not touch each other although their ranges interleave.
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.pointer), y = reinterpret_cast<uintptr_t>(b.pointer);
    const size_t gap = y >= x ? (y - x) % a.stride : (a.stride - (x - y) % a.stride) % a.stride;
    return gap < a.width || gap + b.width > a.stride;
}

// As fb::check_spans, for rows with gaps between them.
template <size_t N>
flint_status check_all(const char* name, const Rows (&list)[N], size_t outputs) {
    fb::Span spans[N];
    for (size_t i = 0; i < N; ++i) {
        spans[i] = fb::Span{list[i].name, list[i].pointer, list[i].bytes()};
    }
    FB_TRY(fb::check_spans(name, spans, N, 0));
    for (size_t i = 0; i < outputs; ++i) {
        for (size_t j = i + 1; j < N; ++j) {
            if (rows_overlap(list[i], list[j])) {
                return fb::fail(kBad, "%s: %s and %s overlap", name, list[i].name, list[j].name);
            }
        }
    }
    return FLINT_OK;
}

Rows flat(const char* name, const void* pointer, size_t bytes) { return Rows{name, pointer, 1, bytes, bytes}; }

Rows token_rows(const char* name, const void* pointer, size_t rows, size_t heads, size_t stride) {
    return Rows{name, pointer, rows, heads * 128, stride * 2};
}

// An array that may be left out stands in the list as something that overlaps nothing.
Rows optional(const char* name, const void* pointer, size_t bytes, const void* instead) {
    return pointer != nullptr ? flat(name, pointer, bytes) : flat(name, instead, 0);
}

flint_status check_workspace(const char* name, size_t needed, size_t given) {
    if (given < needed) {
        return fb::fail(kBad, "%s: needs %zu bytes of workspace, given %zu", name, needed, given);
    }
    return FLINT_OK;
}

flint_status check_shape(const char* name, const flint_b200_packed_shape* shape) {
    if (shape == nullptr) {
        return fb::fail(kBad, "%s: shape is null", name);
    }
    return check_rows(name, shape->sequences, shape->rows, shape->heads, shape->kv_heads, shape->head_width,
                      shape->q_stride, shape->kv_stride, shape->o_stride);
}

flint_status check_shape(const char* name, const flint_b200_paged_shape* shape) {
    if (shape == nullptr) {
        return fb::fail(kBad, "%s: shape is null", name);
    }
    FB_TRY(check_rows(name, shape->sequences, shape->rows, shape->heads, shape->kv_heads, shape->head_width,
                      shape->q_stride, shape->kv_stride, shape->o_stride));
    const size_t size = shape->page_size;
    if (size < 16 || size > 1024 || (size & (size - 1)) != 0) {
        return fb::fail(kBad, "%s: page_size (%zu) must be a power of two from 16 to 1024", name, size);
    }
    constexpr size_t kMost = (size_t{1} << 31) - 1;
    if (shape->pages == 0 || shape->pages > kMost / size / shape->kv_heads) {
        return fb::fail(kBad, "%s: pages (%zu) must be from 1 to %zu", name, shape->pages,
                        kMost / size / shape->kv_heads);
    }
    if (shape->table_stride == 0 || shape->table_stride > (size_t{1} << 26) / size) {
        return fb::fail(kBad, "%s: table_stride (%zu) must be from 1 to %zu", name, shape->table_stride,
                        (size_t{1} << 26) / size);
    }
    if (shape->longest == 0 || shape->longest > kMostRows) {
        return fb::fail(kBad, "%s: longest (%zu) must be from 1 to %zu", name, shape->longest, kMostRows);
    }
    return FLINT_OK;
}

template <typename Shape>
fb::PackedArgs base_args(const Shape& s, float scale) {
    fb::PackedArgs p = {};
    p.sequences = static_cast<int>(s.sequences);
    p.rows = static_cast<int>(s.rows);
    p.heads = static_cast<int>(s.heads);
    p.kv_heads = static_cast<int>(s.kv_heads);
    p.q_stride = static_cast<long long>(s.q_stride);
    p.kv_stride = static_cast<long long>(s.kv_stride);
    p.o_stride = static_cast<long long>(s.o_stride);
    p.scale = scale;
    return p;
}

fb::PackedArgs paged_args(const flint_b200_paged_shape& s, float scale) {
    fb::PackedArgs p = base_args(s, scale);
    p.pages = static_cast<long long>(s.pages);
    p.page_size = static_cast<int>(s.page_size);
    p.table_stride = static_cast<int>(s.table_stride);
    return p;
}

template <typename Shape>
bool nothing(const Shape& s) {
    return s.sequences == 0 || s.rows == 0;
}

size_t cache_bytes(const flint_b200_paged_shape& s) { return s.pages * s.kv_heads * s.page_size * 128; }

}  // namespace

extern "C" {

flint_status flint_b200_packed_attention_workspace(const flint_b200_packed_shape* shape, size_t* bytes) {
    constexpr const char* name = "flint_b200_packed_attention_workspace";
    FB_TRY(check_shape(name, shape));
    if (bytes == nullptr) {
        return fb::fail(kBad, "%s: bytes is null", name);
    }
    FB_CUDA(fb::packed_forward_workspace(bytes));
    return FLINT_OK;
}

flint_status flint_b200_packed_attention_forward(void* o, void* lse, const void* q, const void* k, const void* v,
                                                 const void* starts, const flint_b200_packed_shape* shape,
                                                 float scale, void* workspace, size_t workspace_bytes,
                                                 flint_stream stream) {
    constexpr const char* name = "flint_b200_packed_attention_forward";
    FB_TRY(check_shape(name, shape));
    FB_TRY(check_scale(name, scale));
    if (nothing(*shape)) {
        return FLINT_OK;
    }
    size_t needed = 0;
    FB_TRY(flint_b200_packed_attention_workspace(shape, &needed));
    FB_TRY(check_workspace(name, needed, workspace_bytes));
    const size_t rows = shape->rows;
    const Rows list[] = {
        token_rows("o", o, rows, shape->heads, shape->o_stride),
        optional("lse", lse, shape->heads * rows * 4, o),
        flat("workspace", workspace, needed),
        token_rows("q", q, rows, shape->heads, shape->q_stride),
        token_rows("k", k, rows, shape->kv_heads, shape->kv_stride),
        token_rows("v", v, rows, shape->kv_heads, shape->kv_stride),
        flat("starts", starts, (shape->sequences + 1) * 4),
    };
    FB_TRY(check_all(name, list, 3));
    fb::PackedArgs p = base_args(*shape, scale);
    p.q = static_cast<const __half*>(q);
    p.k = static_cast<const __half*>(k);
    p.v = static_cast<const __half*>(v);
    p.o = static_cast<__half*>(o);
    p.lse = static_cast<float*>(lse);
    p.starts = static_cast<const int*>(starts);
    FB_CUDA(fb::packed_forward(p, p.rows, workspace, stream));
    return FLINT_OK;
}

flint_status flint_b200_packed_attention_backward_workspace(const flint_b200_packed_shape* shape, size_t* bytes) {
    constexpr const char* name = "flint_b200_packed_attention_backward_workspace";
    FB_TRY(check_shape(name, shape));
    if (bytes == nullptr) {
        return fb::fail(kBad, "%s: bytes is null", name);
    }
    FB_CUDA(fb::packed_backward_workspace(shape->sequences, shape->rows, shape->heads, shape->kv_heads, bytes));
    return FLINT_OK;
}

flint_status flint_b200_packed_attention_backward(void* dq, void* dk, void* dv, const void* d_o, const void* o,
                                                  const void* lse, const void* q, const void* k, const void* v,
                                                  const void* starts, const flint_b200_packed_shape* shape,
                                                  float scale, void* workspace, size_t workspace_bytes,
                                                  flint_stream stream) {
    constexpr const char* name = "flint_b200_packed_attention_backward";
    FB_TRY(check_shape(name, shape));
    FB_TRY(check_scale(name, scale));
    if (nothing(*shape)) {
        return FLINT_OK;
    }
    size_t needed = 0;
    FB_TRY(flint_b200_packed_attention_backward_workspace(shape, &needed));
    FB_TRY(check_workspace(name, needed, workspace_bytes));
    const size_t rows = shape->rows;
    const Rows list[] = {
        token_rows("dq", dq, rows, shape->heads, shape->q_stride),
        token_rows("dk", dk, rows, shape->kv_heads, shape->kv_stride),
        token_rows("dv", dv, rows, shape->kv_heads, shape->kv_stride),
        flat("workspace", workspace, needed),
        token_rows("d_o", d_o, rows, shape->heads, shape->o_stride),
        token_rows("o", o, rows, shape->heads, shape->o_stride),
        flat("lse", lse, shape->heads * rows * 4),
        token_rows("q", q, rows, shape->heads, shape->q_stride),
        token_rows("k", k, rows, shape->kv_heads, shape->kv_stride),
        token_rows("v", v, rows, shape->kv_heads, shape->kv_stride),
        flat("starts", starts, (shape->sequences + 1) * 4),
    };
    FB_TRY(check_all(name, list, 4));
    fb::PackedArgs p = base_args(*shape, scale);
    p.q = static_cast<const __half*>(q);
    p.k = static_cast<const __half*>(k);
    p.v = static_cast<const __half*>(v);
    p.o = static_cast<__half*>(const_cast<void*>(o));
    p.lse = static_cast<float*>(const_cast<void*>(lse));
    p.starts = static_cast<const int*>(starts);
    const fb::PackedGradients g{static_cast<__half*>(dq), static_cast<__half*>(dk), static_cast<__half*>(dv),
                                static_cast<const __half*>(d_o)};
    FB_CUDA(fb::packed_backward(p, g, workspace, stream));
    return FLINT_OK;
}

flint_status flint_b200_paged_store(void* k_pages, void* v_pages, const void* k, const void* v, const void* starts,
                                    const void* lengths, const void* page_table, const flint_b200_paged_shape* shape,
                                    flint_stream stream) {
    constexpr const char* name = "flint_b200_paged_store";
    FB_TRY(check_shape(name, shape));
    if (nothing(*shape)) {
        return FLINT_OK;
    }
    const Rows list[] = {
        flat("k_pages", k_pages, cache_bytes(*shape)),
        flat("v_pages", v_pages, cache_bytes(*shape)),
        token_rows("k", k, shape->rows, shape->kv_heads, shape->kv_stride),
        token_rows("v", v, shape->rows, shape->kv_heads, shape->kv_stride),
        flat("starts", starts, (shape->sequences + 1) * 4),
        flat("lengths", lengths, shape->sequences * 4),
        flat("page_table", page_table, shape->sequences * shape->table_stride * 4),
    };
    FB_TRY(check_all(name, list, 2));
    fb::PackedArgs p = paged_args(*shape, 1.0f);
    p.k = static_cast<const __half*>(k);
    p.v = static_cast<const __half*>(v);
    p.starts = static_cast<const int*>(starts);
    p.lengths = static_cast<const int*>(lengths);
    p.table = static_cast<const int*>(page_table);
    int sms = 148;
    FB_CUDA(fb::sm_count(&sms));
    FB_CUDA(fb::launch_dependent(fb::fb_paged_store,
                                 fb::sequence_grid(p, 32, static_cast<long long>(p.rows) * p.kv_heads * 2, sms),
                                 dim3(256), 0, stream, p, static_cast<__half*>(k_pages),
                                 static_cast<__half*>(v_pages)));
    return FLINT_OK;
}

flint_status flint_b200_paged_attention_workspace(const flint_b200_paged_shape* shape, size_t* bytes) {
    constexpr const char* name = "flint_b200_paged_attention_workspace";
    FB_TRY(check_shape(name, shape));
    if (bytes == nullptr) {
        return fb::fail(kBad, "%s: bytes is null", name);
    }
    FB_CUDA(fb::packed_forward_workspace(bytes));
    return FLINT_OK;
}

flint_status flint_b200_paged_attention(void* o, void* lse, const void* q, const void* k_pages, const void* v_pages,
                                        const void* starts, const void* lengths, const void* page_table,
                                        const flint_b200_paged_shape* shape, float scale, void* workspace,
                                        size_t workspace_bytes, flint_stream stream) {
    constexpr const char* name = "flint_b200_paged_attention";
    FB_TRY(check_shape(name, shape));
    FB_TRY(check_scale(name, scale));
    if (nothing(*shape)) {
        return FLINT_OK;
    }
    size_t needed = 0;
    FB_TRY(flint_b200_paged_attention_workspace(shape, &needed));
    FB_TRY(check_workspace(name, needed, workspace_bytes));
    const Rows list[] = {
        token_rows("o", o, shape->rows, shape->heads, shape->o_stride),
        optional("lse", lse, shape->heads * shape->rows * 4, o),
        flat("workspace", workspace, needed),
        token_rows("q", q, shape->rows, shape->heads, shape->q_stride),
        flat("k_pages", k_pages, cache_bytes(*shape)),
        flat("v_pages", v_pages, cache_bytes(*shape)),
        flat("starts", starts, (shape->sequences + 1) * 4),
        flat("lengths", lengths, shape->sequences * 4),
        flat("page_table", page_table, shape->sequences * shape->table_stride * 4),
    };
    FB_TRY(check_all(name, list, 3));
    fb::PackedArgs p = paged_args(*shape, scale);
    p.q = static_cast<const __half*>(q);
    p.k = static_cast<const __half*>(k_pages);
    p.v = static_cast<const __half*>(v_pages);
    p.o = static_cast<__half*>(o);
    p.lse = static_cast<float*>(lse);
    p.starts = static_cast<const int*>(starts);
    p.lengths = static_cast<const int*>(lengths);
    p.table = static_cast<const int*>(page_table);
    FB_CUDA(fb::packed_forward(p, static_cast<int>(shape->longest), workspace, stream));
    return FLINT_OK;
}

}  // extern "C"
