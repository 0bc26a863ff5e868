// Attention over sequences of different lengths: what the entry points (packed.cu) hand to the
// kernels. A batch is `rows` rows of tokens; sequence s has rows starts[s] .. starts[s + 1] - 1,
// and heads lie side by side in a row (64 values each).
#pragma once

#include <cstddef>

#include <cuda_fp16.h>
#include <cuda_runtime_api.h>

namespace fb {

struct PackedArgs {
    const __half* q;        // [rows, q_stride]
    const __half* k;        // packed: [rows, kv_stride]; paged: [pages, kv_heads, page_size, 64]
    const __half* v;
    __half* o;              // [rows, o_stride]
    float* lse;             // [heads, rows], may be null
    const int* starts;      // [sequences + 1]
    const int* lengths;     // paged: keys of each sequence, the new ones among them; packed: null
    const int* table;       // paged: [sequences, table_stride] page numbers
    long long q_stride, kv_stride, o_stride;   // elements between rows
    long long pages;
    int page_size, table_stride;
    int sequences, rows, heads, kv_heads;
    float scale;
};

struct PackedGradients {
    __half* dq;             // rows as q's
    __half* dk;             // rows as k's
    __half* dv;
    const __half* d_o;      // rows as o's
};

// Forward, over packed or paged keys; the workspace's size depends on the GPU only. `longest` is about how many new
// tokens a sequence has at most (paged keys; it chooses the kernel's form).
cudaError_t packed_forward(const PackedArgs& args, int longest, void* workspace, cudaStream_t stream);
cudaError_t packed_forward_workspace(size_t* bytes);
cudaError_t packed_forward_error_flag(int* value, bool reset);

// Backward, of packed keys: args.o and args.lse are the forward's results.
cudaError_t packed_backward(const PackedArgs& args, const PackedGradients& gradients, void* workspace,
                            cudaStream_t stream);
cudaError_t packed_backward_workspace(size_t sequences, size_t rows, size_t heads, size_t kv_heads, size_t* bytes);
cudaError_t packed_backward_error_flag(int* value, bool reset);

// Device error words of these kernels: a wait that gave up, or starts, lengths or page
// numbers outside their ranges (which are clamped, so that nothing outside is touched).
cudaError_t packed_error_flag(int* value, bool reset);

}  // namespace fb
