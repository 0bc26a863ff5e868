/* Extensions of the Blackwell build that the reference library does not have:
 * fused (flash) causal attention, the optimizer and loss-scaling kernels, a
 * model variant that uses them, and hooks for data-parallel training. None of
 * these has a counterpart in the reference's include/flint/flint.h; they follow
 * the same conventions (device pointers, caller's stream, flint_status,
 * flint_last_error). The PyTorch oracle they are checked against is the
 * reference's scripts/gpt2_torch.py (attention: :52-60, AdamW groups: :161-175,
 * train_step: :178-192). */
#ifndef FLINT_FLINT_B200_H
#define FLINT_FLINT_B200_H

#include "flint/flint.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 1 if a kernel (GEMM, attention, column sums, cross-entropy, log-probabilities) gave up on a
 * bounded barrier wait since the last call, or one that reads starts, lengths or page numbers
 * met one out of range (the flag is cleared), 0 otherwise.
 * Synchronises the device; meant for tests. */
FLINT_API flint_status flint_b200_kernel_fault(int* raised);

/* Kernels this library has launched in this process so far (host counter). */
FLINT_API flint_status flint_b200_launch_count(unsigned long long* launches);

/* Diagnostic (no counterpart in the reference): the rate of the tensor pipe for
 * the small MMAs that attention with head width 64 is made of. One CTA on an
 * otherwise idle GPU issues `count` (1 to 4,096) tcgen05.mma of kind::f16 with
 * M = 128, K = 16 and N = `n` (64 or 128) back to back from one elected thread,
 * the A operand read from shared memory or, when a_in_tmem is not 0, from tensor
 * memory; operands are zeros. *issue_clocks receives the SM clocks until the last
 * one was accepted, *complete_clocks until all had completed. Waits for the
 * stream; meant for `python -m flint_b200.kernel_bench --group mma`. */
FLINT_API flint_status flint_b200_mma_clocks(int n, int a_in_tmem, int count,
                                             long long* issue_clocks, long long* complete_clocks,
                                             flint_stream stream);

/* Causal attention without materialising scores or probabilities:
 * o[b] = softmax(scale * q[b] k[b]^T + causal mask) v[b] for `batches`
 * (sequence, head) pairs, all FP16 [batches, length, head_width] contiguous;
 * lse[batches, length] FP32 receives log-sum-exp of the scaled scores (natural
 * log), which the backward pass needs. head_width must be 64, length a
 * multiple of 8 up to 1,024, scale finite and positive. */
FLINT_API flint_status flint_b200_attention_forward(void* o, void* lse, const void* q,
                                                    const void* k, const void* v, size_t batches,
                                                    size_t length, size_t head_width, float scale,
                                                    flint_stream stream);

/* Gradients of the above: dq, dk, dv from d_o, o, lse and q, k, v (layouts as
 * above). delta is an FP32 scratch [batches, length] the call overwrites. */
FLINT_API flint_status flint_b200_attention_backward(void* dq, void* dk, void* dv, const void* d_o,
                                                     const void* o, const void* lse, void* delta,
                                                     const void* q, const void* k, const void* v,
                                                     size_t batches, size_t length,
                                                     size_t head_width, float scale,
                                                     flint_stream stream);

/* flint_gpt2_create with a choice of attention: flash_attention non-zero builds
 * the model on the fused kernels above (no T x T buffers, so far less memory);
 * zero is flint_gpt2_create. */
FLINT_API flint_status flint_b200_gpt2_create(const flint_gpt2_config* config, int flash_attention,
                                              flint_gpt2** model);

/* Called on the launching host thread from inside
 * flint_b200_gpt2_backward_buckets each time every kernel that writes one
 * contiguous range of the gradient arena has been enqueued: bucket 0 is ln_f,
 * buckets 1..layers are the blocks from last to first, and the final bucket is
 * wte + wpe. A data-parallel trainer records an event there and starts that
 * range's all-reduce on another stream. */
typedef void (*flint_b200_bucket_callback)(void* user, int bucket, void* gradients, size_t bytes);

/* flint_gpt2_backward plus the callback above (which may be null). */
FLINT_API flint_status flint_b200_gpt2_backward_buckets(flint_gpt2* model, const void* tokens,
                                                        int accumulate, flint_stream stream,
                                                        flint_b200_bucket_callback callback,
                                                        void* user);

/* Called on the launching host thread from inside flint_b200_gpt2_forward_stages
 * before the kernels of each stage are enqueued: stage 0 is the embedding,
 * stages 1..layers the transformer blocks in order, stage layers + 1 the final
 * LayerNorm with the output layer and the loss. A trainer whose weights arrive
 * bucket by bucket (a sharded optimizer's all-gather) makes the stream wait
 * there for that stage's weights only. */
typedef void (*flint_b200_stage_callback)(void* user, int stage);

/* flint_gpt2_forward plus the callback above (which may be null). */
FLINT_API flint_status flint_b200_gpt2_forward_stages(flint_gpt2* model, const void* tokens,
                                                      const void* targets, float scale,
                                                      flint_stream stream,
                                                      flint_b200_stage_callback callback,
                                                      void* user);

/* The contiguous FP32 range that holds every gradient, in parameter order. */
FLINT_API flint_status flint_b200_gpt2_gradient_arena(const flint_gpt2* model, void** base,
                                                      size_t* bytes);

/* The FP16 compute copy of the index-th master weight (what the GEMMs read), or
 * null for biases and LayerNorm parameters, which have none. An optimizer that
 * writes it together with the master weight saves flint_gpt2_sync_weights. */
FLINT_API flint_status flint_b200_gpt2_compute_copy(const flint_gpt2* model, size_t index,
                                                    void** address);

/* Fused AdamW over `count` FP32 values (PyTorch semantics, decoupled decay):
 *   g = grad * grad_scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
 *   p = p - lr * (weight_decay * p + (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps))
 * and, when half_copy is not null, half_copy = half(p). When *skip (a device
 * int, may be null) is non-zero the call changes nothing: a step whose
 * gradients overflowed is dropped. */
FLINT_API flint_status flint_b200_adamw(void* param, void* m, void* v, const void* grad,
                                        void* half_copy, size_t count, float lr, float beta1,
                                        float beta2, float eps, float weight_decay,
                                        float grad_scale, int step, const int* skip,
                                        flint_stream stream);

/* One tensor of a multi-tensor AdamW plan; half_copy may be null. */
typedef struct {
    void* param;
    void* m;
    void* v;
    const void* grad;
    void* half_copy;
    size_t count;
    float weight_decay;
} flint_b200_adamw_tensor;

/* A plan lets one launch update every tensor of a model. tensors is a host
 * array; *bytes is the device memory the plan needs; *items is what
 * flint_b200_adamw_run takes. */
FLINT_API flint_status flint_b200_adamw_plan_bytes(const flint_b200_adamw_tensor* tensors,
                                                   size_t count, size_t* bytes);
FLINT_API flint_status flint_b200_adamw_plan_items(const flint_b200_adamw_tensor* tensors,
                                                   size_t count, size_t* items);

/* Writes the plan into device memory `plan` (16-byte aligned, plan_bytes long)
 * and waits for the copy, so tensors may be freed on return. */
FLINT_API flint_status flint_b200_adamw_plan(void* plan, size_t plan_bytes,
                                             const flint_b200_adamw_tensor* tensors, size_t count,
                                             flint_stream stream);

/* flint_b200_adamw over every tensor of the plan, each with its own weight
 * decay, in one launch. */
FLINT_API flint_status flint_b200_adamw_run(const void* plan, size_t items, float lr, float beta1,
                                            float beta2, float eps, float grad_scale, int step,
                                            const int* skip, flint_stream stream);

/* flint_bias_gradient for callers that cannot supply a workspace. It has no
 * counterpart in the reference. The result is flint_bias_gradient's bit for bit;
 * the partial sums live in a 4 MiB array built into the library instead of a
 * caller buffer, and the call allocates nothing (no cudaMalloc, no cudaFree).
 * It exists for hosts that may not allocate device memory once they are running:
 * a plug-in inside an application that owns the whole memory budget, or a loop
 * that cannot afford the device-wide synchronisation cudaMalloc implies.
 *
 * Limit: ceil(rows / 256) * cols * 8 bytes must fit in 4 MiB (for example 16,384
 * rows x 3,072 cols needs 1.5 MiB); larger shapes fail with
 * FLINT_ERROR_INVALID_ARGUMENT and should use flint_bias_gradient. Every GPU
 * that loads the library holds the 4 MiB until the process exits.
 *
 * The first call on each device looks up the array's device address; make that
 * call before starting any stream capture. All calls share the one array, so two
 * calls that can overlap on the GPU (different streams, no ordering between
 * them) race on it; calls ordered on one stream are fine, and nothing has to be
 * cleared between them. */
FLINT_API flint_status flint_b200_bias_gradient_static(void* dbias, const void* dy, size_t rows,
                                                       size_t cols, int accumulate,
                                                       flint_stream stream);

/* ---- decoding with a KV cache (the reference's inference milestone, README.md:148; it has
 * no code for it, so nothing here has a counterpart in its header) ----
 *
 * A generator decodes with the weights of `model` (whose FP16 copies must be in
 * sync): `sequences` sequences (1..64) side by side, each up to `max_length`
 * positions (a multiple of 8, at most min(block_size, 1024)). It owns the cache
 * [layer][K|V][sequence][head][position][64] in FP16 and its scratch; with
 * int8_weights it also owns an int8 copy of every matrix with one FP32 scale per
 * output row (w[n, :] ~ q[n, :] * scale[n], q = round(w / scale), scale = max|w| / 127),
 * halving the bytes a decode step reads. Heads must be 64 wide. */
typedef struct flint_b200_generator flint_b200_generator;

FLINT_API flint_status flint_b200_generator_create(const flint_gpt2* model, size_t sequences,
                                                   size_t max_length, int int8_weights,
                                                   flint_b200_generator** generator);
FLINT_API void flint_b200_generator_destroy(flint_b200_generator* generator);

/* Re-derives the int8 copies after the model's weights changed. */
FLINT_API flint_status flint_b200_generator_refresh(flint_b200_generator* generator,
                                                    flint_stream stream);

/* Starts over: tokens is uint16 [sequences, length], length a multiple of 8 up
 * to max_length. Runs the prompt through the tensor-core GEMMs and the fused
 * causal attention kernel, stores every position's keys and values in the
 * cache and leaves the logits of each sequence's last position. */
FLINT_API flint_status flint_b200_generator_prefill(flint_b200_generator* generator,
                                                    const void* tokens, size_t length,
                                                    flint_stream stream);

/* Appends one token per sequence (uint16 [sequences]) at the next position:
 * leaves its logits and writes each sequence's most likely next token (lowest
 * index among equals, padded columns excluded) to next_tokens (uint16
 * [sequences] on the device; null keeps it internal). With use_graph non-zero
 * the step's launches are captured into a CUDA graph on the first call and
 * replayed afterwards (the position lives in device memory); tokens and
 * next_tokens must then be the same buffers on every call. */
FLINT_API flint_status flint_b200_generator_step(flint_b200_generator* generator,
                                                 const void* tokens, void* next_tokens,
                                                 int use_graph, flint_stream stream);

/* FP32 logits [sequences, padded_vocab] of the last position processed, and how
 * many positions each sequence holds. */
FLINT_API flint_status flint_b200_generator_logits(const flint_b200_generator* generator,
                                                   const void** logits, size_t* position);

/* Bytes the next decode step must read from HBM: the weights (each matrix once)
 * and the cache. */
FLINT_API flint_status flint_b200_generator_bytes_per_step(const flint_b200_generator* generator,
                                                           size_t* weight_bytes,
                                                           size_t* cache_bytes);

/* ---- sequences of different lengths --------------------------------------------------------
 *
 * A batch is `rows` rows, one per token, in which the sequences lie one behind the other:
 * `starts` (int32 [sequences + 1] on the device, non-decreasing, 0 .. rows) says where, sequence s
 * having rows starts[s] .. starts[s + 1] - 1, which may be none; rows outside all sequences are
 * left as they are. Heads of 64 FP16 values lie side by side in a row; rows of q (and dq) are q_stride
 * elements apart, those of k, v (dk, dv) kv_stride, those of o (d_o) o_stride, so that the parts of
 * a product's [q | k | v] rows can be given as they lie. Query head h reads head
 * h / (heads / kv_heads) of k and v. lse is FP32 [heads, rows].
 *
 * Limits: sequences up to 65,535, rows up to 2^24, heads up to 1,024 and up to 128 times kv_heads,
 * strides multiples of 8 up to 2^24, scale finite and positive. Pointers are 16-byte aligned and
 * outputs overlap neither each other nor inputs (columns of one matrix do not overlap).
 * What lies in device memory (starts, lengths, page numbers) is not known to the host: values
 * outside their ranges are clamped by the kernels, which touch nothing outside the arrays, and
 * reported by flint_b200_kernel_fault; the results are then undefined.
 *
 * A workspace is overwritten by every call and keeps nothing from one to the next; calls that can
 * run at the same time need one each. Its size depends on the shape and on the GPU's SM count. */
typedef struct {
    size_t sequences;
    size_t rows;
    size_t heads;
    size_t kv_heads;
    size_t head_width;
    size_t q_stride;
    size_t kv_stride;
    size_t o_stride;
} flint_b200_packed_shape;

FLINT_API flint_status flint_b200_packed_attention_workspace(const flint_b200_packed_shape* shape,
                                                             size_t* bytes);

/* Causal attention within each sequence: o_i = sum over j <= i of p_ij v_j with p the softmax of
 * scale * q_i . k_j, and lse_i (may be null) the natural log of the scores' sum of exponentials. Keys whose
 * score is minus infinity weigh nothing (a row of nothing else is NaN). Values of a sequence
 * reach only that sequence, whatever they are; within it a value of v that is not finite may reach
 * rows up to 127 before its own. */
FLINT_API flint_status flint_b200_packed_attention_forward(
    void* o, void* lse, const void* q, const void* k, const void* v, const void* starts,
    const flint_b200_packed_shape* shape, float scale, void* workspace, size_t workspace_bytes,
    flint_stream stream);

FLINT_API flint_status flint_b200_packed_attention_backward_workspace(
    const flint_b200_packed_shape* shape, size_t* bytes);

/* Gradients of the above from d_o and the forward call's o and lse. dk and dv are sums over the
 * query heads that share a head, taken in one fixed order: results repeat bit for bit. A row that is NaN makes its
 * dq NaN, and dk and dv of the keys that it sees. Within a sequence a value that is not finite may also reach rows
 * of its block of 128 that have no part in it: dq of up to 127 rows before one of k, and dk and dv of up
 * to 127 rows behind one of q or d_o.
 * The scores' gradients p (d_o . v - d_o . o) are rounded to FP16 before they meet scale: beyond 65,504 they are
 * infinite, and so are dq and dk, and below 2^-25 they are lost. d_o of up to some thousands for inputs of size
 * one stays clear of the first. */
FLINT_API flint_status flint_b200_packed_attention_backward(
    void* dq, void* dk, void* dv, const void* d_o, const void* o, const void* lse, const void* q,
    const void* k, const void* v, const void* starts, const flint_b200_packed_shape* shape,
    float scale, void* workspace, size_t workspace_bytes, flint_stream stream);

/* A cache of keys and values in pages, FP16 [pages, kv_heads, page_size, 64] each: page_size is a
 * power of two from 16 to 1,024, pages * kv_heads * page_size below 2^31. Position t of sequence s
 * is slot t % page_size of page page_table[s * table_stride + t / page_size] (int32 on the device,
 * 0 .. pages - 1 where a position is used, anything elsewhere). `lengths` (int32 [sequences] on the
 * device, up to table_stride * page_size) counts each sequence's positions, this call's new tokens
 * among them: those are the last starts[s + 1] - starts[s] ones. `longest` says how many new tokens a
 * sequence has at most; it chooses the kernel and bounds nothing. The other fields and limits are
 * flint_b200_packed_shape's; kv_stride is that of the new tokens' k and v. */
typedef struct {
    size_t sequences;
    size_t rows;
    size_t heads;
    size_t kv_heads;
    size_t head_width;
    size_t q_stride;
    size_t kv_stride;
    size_t o_stride;
    size_t pages;
    size_t page_size;
    size_t table_stride;
    size_t longest;
} flint_b200_paged_shape;

/* Copies the new tokens' keys and values into their positions of the cache. Two sequences that
 * store into one page's same slot race; sequences may share pages that they only read. */
FLINT_API flint_status flint_b200_paged_store(void* k_pages, void* v_pages, const void* k,
                                              const void* v, const void* starts,
                                              const void* lengths, const void* page_table,
                                              const flint_b200_paged_shape* shape,
                                              flint_stream stream);

FLINT_API flint_status flint_b200_paged_attention_workspace(const flint_b200_paged_shape* shape,
                                                            size_t* bytes);

/* Attention of the new tokens over the cache, in which their own keys and values are already:
 * each sees the positions up to its own. lse may be null. A token without any position
 * (a sequence whose length is below its number of new tokens) gets zeros and an lse of minus infinity.
 * Slots behind a sequence's last position may hold anything. */
FLINT_API flint_status flint_b200_paged_attention(void* o, void* lse, const void* q,
                                                  const void* k_pages, const void* v_pages,
                                                  const void* starts, const void* lengths,
                                                  const void* page_table,
                                                  const flint_b200_paged_shape* shape, float scale,
                                                  void* workspace, size_t workspace_bytes,
                                                  flint_stream stream);

/* ---- probabilities of tokens ----------------------------------------------------------------
 *
 * Over the first vocab columns of each row x of logits [rows, cols], FP16 or (fp32_logits not 0)
 * FP32:  lse = log sum exp x,  log_probs = x[target] - lse,  entropy = -sum p log p with
 * p = exp(x - lse), all FP32 [rows];  top_tokens (uint16 [rows, top]) the columns of the `top`
 * largest logits in descending order, equal ones by ascending column, and top_log_probs (FP32
 * [rows, top]) theirs. targets are uint16; one that is not below vocab marks a row that does not count: its
 * log-probability is 0. log_probs (with targets), entropy and lse may be null, and with top 0 the top's arrays.
 * A logit of minus infinity is a token that cannot come; a row of nothing else has an entropy of 0 and
 * log-probabilities and an lse of minus infinity. A row with a NaN or plus infinity has NaNs
 * (NaN sorts above all numbers). cols is a multiple of 8 from 8 to 65,536, top up to 32 and vocab, rows up to 2^31. */
FLINT_API flint_status flint_b200_token_log_probs(void* log_probs, void* entropy, void* lse,
                                                  void* top_log_probs, void* top_tokens,
                                                  const void* logits, const void* targets,
                                                  int fp32_logits, size_t rows, size_t vocab,
                                                  size_t cols, size_t top, flint_stream stream);

/* The logits' gradient for the gradients d_log_probs and d_entropy (FP32 [rows], one may be null) of
 * the above's outputs, from its lse and entropy:
 *   dlogits_c = d_log_probs ([c == target] - p_c) - d_entropy p_c (log p_c + entropy)
 * in the logits' type, +0 in columns from vocab on; targets not below vocab count as
 * d_log_probs = 0. A column of minus infinity gets 0 (but for its own d_log_probs as a target), and so does a row of
 * nothing else. dlogits may be logits itself. lse has no gradient. p is exp(x - lse) with lse in FP32, off by up to
 * |lse| 2^-24 of itself: 2^-9 for FP16 rows near -65,504; FP32 rows that lie farther from 0 as a whole are better shifted
 * first, which changes no output but lse. */
FLINT_API flint_status flint_b200_token_log_probs_backward(
    void* dlogits, const void* logits, const void* targets, const void* lse, const void* entropy,
    const void* d_log_probs, const void* d_entropy, int fp32_logits, size_t rows, size_t vocab,
    size_t cols, flint_stream stream);

/* Sets *found_nonfinite (device int) to 1 if any of the count FP32 values is
 * inf or NaN; leaves it unchanged otherwise, so several calls can share it.
 * When sum_squares (device double, may be null) is given, adds the sum of
 * squares of the values times scale^2 to it (for gradient-norm clipping). */
FLINT_API flint_status flint_b200_check_gradients(const void* grad, size_t count, float scale,
                                                  int* found_nonfinite, double* sum_squares,
                                                  flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_B200_H */
