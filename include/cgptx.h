/*
 * cgptx.h — C-ABI of the MI355X (gfx950) training hot path.
 *
 * Every entry point takes plain device pointers, sizes, a dtype code and a
 * hipStream_t (passed as void*), enqueues work on that stream and returns a
 * status code. Nothing here throws, synchronises (unless stated) or owns a
 * caller tensor. Citations name the interface of B4rtekk1/CGPT that an entry
 * point stands in for (paths relative to the reference checkout).
 *
 * Scratch memory (row statistics, split-K partials, sort buffers) comes from
 * a per-(device, stream) arena that grows on the first eager call with a given
 * problem size. While a stream is being captured into a hipGraph the arena
 * cannot grow: a call that would need more scratch than an earlier eager call
 * reserved returns CGPTX_CAPTURE_ALLOC, or is recorded in a slower form where
 * scratch only makes it faster (padded copies of ragged operands, split-K
 * partials of contractions other than whole, long ones, shared key blocks).
 * Run each op once eagerly before capture, exactly as the reference warms up
 * before cudaStreamBeginCapture (train/train.cpp:545-548). A recorded call keeps
 * the scratch of the stream it was captured on: replays, on whatever stream, have
 * to be ordered with the library's other work on that stream and with other graphs
 * captured there, or their results and that work's are undefined (later calls are
 * not touched). An arena that grows later leaves the block that a recorded call
 * works in until cgptx_release_scratch, which ends the use of such graphs.
 *
 * Threading: one host thread per stream, as in the reference.
 */
#ifndef CGPTX_H
#define CGPTX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Storage dtypes; numeric values follow enum class Dtype (include/core/dtype.h:12-21). */
enum { CGPTX_F16 = 0, CGPTX_BF16 = 1, CGPTX_F32 = 2 };

/* Status codes. The C++ layer maps INVALID_ARGUMENT to std::invalid_argument,
 * OVERFLOW to std::overflow_error and RUNTIME to the fatal path of
 * include/core/cuda_check.h:19-38. */
enum {
    CGPTX_OK = 0,
    CGPTX_INVALID_ARGUMENT = 1,
    CGPTX_OVERFLOW = 2,
    CGPTX_RUNTIME = 3,
    CGPTX_CAPTURE_ALLOC = 4
};

typedef void* cgptx_stream; /* hipStream_t */

/* Message of the last failing call on this host thread ("" if none). */
const char* cgptx_last_error(void);
/* Library version string. */
const char* cgptx_version(void);
/* Releases every scratch arena of the current device (synchronises the device). Graphs of calls that work in one, recorded before, must
 * not be replayed any more; the composed step (cgptx_train.h) records its own anew. */
int cgptx_release_scratch(void);
/* Bytes of the scratch arena bound to (current device, stream): the largest request any operator has made on
 * that stream so far, rounded up to 1 MiB; 0 when the stream has none. For a train step it is dominated by the
 * logits chunk of the cut cross-entropy (rows x vocabulary in the storage dtype, up to 2 GiB - 1 MiB). */
size_t cgptx_scratch_bytes(cgptx_stream stream);

/* ------------------------------------------------------------------ backward */

/* rmsnorm_backward — include/ops/backward/rmsnorm_backward.h:21-29.
 * x, dy, dx: [rows, hidden]; weight, grad_weight: [hidden]; all of `dtype`.
 * dx = dy*w*r - x*(sum_j dy_j w_j x_j)*r^3/hidden, r = rsqrt(mean(x^2)+eps);
 * grad_weight_j = sum_rows dy*x*r. Both outputs are overwritten. */
int cgptx_rmsnorm_backward(void* grad_input, void* grad_weight,
                           const void* grad_output, const void* input,
                           const void* weight, size_t rows, size_t hidden,
                           float epsilon, int dtype, cgptx_stream stream);

/* rmsnorm_backward that allocates nothing. No counterpart in the reference: it is for callers that cannot
 * allocate device memory — code under hipGraph capture that has not run eagerly first, tight serving loops,
 * harnesses that forbid hipMalloc. Same arguments, kernels and results (bit for bit) as cgptx_rmsnorm_backward;
 * the partial sums of the weight gradient go to a 16 MiB block built into the library's device image (each GPU
 * the library runs on holds one until the process ends) instead of the per-stream arena. A shape that needs
 * more (4 bytes x hidden x the blocks resident on the device, at most a few thousand, for hidden sizes the row
 * kernel takes: multiples of 8 up to 2048 in 16-bit storage; else 4 bytes x rows + 1 KiB x hidden) returns
 * CGPTX_INVALID_ARGUMENT with both sizes in the message, before anything is launched. Calls no hipMalloc / hipFree. Every call on a GPU
 * shares that GPU's block: calls that overlap on one GPU (different streams or threads) race; calls on one
 * stream are ordered. */
int cgptx_rmsnorm_backward_static(void* grad_input, void* grad_weight,
                                  const void* grad_output, const void* input,
                                  const void* weight, size_t rows, size_t hidden,
                                  float epsilon, int dtype, cgptx_stream stream);

/* rope_backward — include/ops/backward/rope_backward.h:22-31.
 * q grads [batch, sequence, query_heads, head_dim], k grads [.., kv_heads, ..],
 * caches [cache_positions, rotary_dim/2]; adjacent pairs (2p, 2p+1) rotate by
 * the inverse angle; the tail past rotary_dim is copied. rotary_dim 0 = head_dim. */
int cgptx_rope_backward(void* grad_query, void* grad_key,
                        const void* grad_rotated_query,
                        const void* grad_rotated_key, const void* cos_cache,
                        const void* sin_cache, size_t batch, size_t sequence,
                        size_t query_heads, size_t kv_heads, size_t head_dim,
                        size_t rotary_dim, size_t position_offset,
                        size_t cache_positions, int dtype, cgptx_stream stream);

/* swiglu_backward (separate gate/up) — include/ops/backward/swiglu_backward.h:30-38. */
int cgptx_swiglu_backward(void* grad_gate, void* grad_up,
                          const void* grad_output, const void* gate,
                          const void* up, size_t count, int accumulate_gate,
                          int accumulate_up, int dtype, cgptx_stream stream);

/* swiglu_backward (packed [rows, 2*hidden] = [gate | up]) —
 * src/ops/backward/swiglu_backward.cu:830-883. */
int cgptx_swiglu_backward_packed(void* grad_gate_up, const void* grad_output,
                                 const void* gate_up, size_t rows,
                                 size_t hidden, int accumulate_gate_up,
                                 int dtype, cgptx_stream stream);

/* linear_backward — include/ops/backward/linear_backward.h:36-46.
 * dX[rows,in] = dY[rows,out]·W[out,in]; dW[out,in] = dYᵀ·X; db[out] = Σ_rows dY.
 * fp32 accumulation; each accumulate_* flag adds into the existing output.
 * Any of grad_input / grad_weight / grad_bias may be NULL to skip that product
 * (the reference always computes all three). */
int cgptx_linear_backward(void* grad_input, void* grad_weight, void* grad_bias,
                          const void* grad_output, const void* input,
                          const void* weight, size_t rows, size_t in_features,
                          size_t out_features, int accumulate_input,
                          int accumulate_weight, int accumulate_bias, int dtype,
                          cgptx_stream stream);

/* embedding_backward — include/ops/backward/embedding_backward.h:35-42.
 * dW[id_t,:] += dY[t,:]. Rows are summed in ascending token order with a
 * rounding to `dtype` after every add, which is the arithmetic of
 * src/ops/cpu/backward/embedding_backward_cpu.cpp:99-112, so the result is
 * deterministic. ids >= vocab are skipped (always; the reference leaves that
 * case undefined without bounds_check). */
int cgptx_embedding_backward(void* grad_weight, const void* grad_output,
                             const uint32_t* token_ids, size_t token_count,
                             size_t vocab, size_t hidden, int bounds_check,
                             int accumulate_weight, int dtype,
                             cgptx_stream stream);

/* cross_entropy_forward_backward — include/ops/cross_entropy.h:25-32.
 * loss[1] (fp32) = mean_r (logsumexp z_r − z_{r,y_r}) over rows with y_r < vocab;
 * gradient = (softmax − onehot)·gradient_scale/rows in `dtype`. */
int cgptx_cross_entropy_forward_backward(float* loss, void* gradient,
                                         const void* logits,
                                         const uint32_t* targets, size_t rows,
                                         size_t vocab, float gradient_scale,
                                         int dtype, cgptx_stream stream);

/* cross_entropy_forward — include/ops/cross_entropy.h:37-42. */
int cgptx_cross_entropy_forward(float* loss, const void* logits,
                                const uint32_t* targets, size_t rows,
                                size_t vocab, int dtype, cgptx_stream stream);

/* cut_cross_entropy_forward_backward — include/ops/cut_cross_entropy.h:25-33.
 * z = X·Cᵀ is never stored in full. The reference is F32-only with no gradient
 * scale; here any dtype is accepted, gradient_scale multiplies both gradients
 * (1.0 reproduces the reference) and accumulate_classifier adds into dC (needed
 * for tied embeddings). */
int cgptx_cut_cross_entropy_forward_backward(
    float* loss, void* input_gradient, void* classifier_gradient,
    const void* input, const void* classifier, const uint32_t* targets,
    size_t rows, size_t hidden, size_t vocab, float gradient_scale,
    int accumulate_classifier, int dtype, cgptx_stream stream);

/* flash_gqa_attention_backward_with_lse — include/ops/backward/attention_backward.h:57-70.
 * q, o, dO, dQ: [batch, query_sequence, query_heads, head_dim];
 * k, v, dK, dV: [batch, kv_sequence, kv_heads, head_dim];
 * logsumexp fp32 [batch, query_sequence, query_heads] = ln Σ exp(scale·q·k).
 * attention_scale <= 0 selects 1/sqrt(head_dim). Causal: key j visible to query
 * i iff j <= query_position_offset + i. */
int cgptx_flash_gqa_attention_backward_with_lse(
    void* grad_query, void* grad_key, void* grad_value, const void* grad_output,
    const void* output, const float* logsumexp, const void* query,
    const void* key, const void* value, size_t batch, size_t query_sequence,
    size_t kv_sequence, size_t query_heads, size_t kv_heads, size_t head_dim,
    float attention_scale, int causal, size_t query_position_offset,
    int accumulate_grads, int dtype, cgptx_stream stream);

/* flash_gqa_attention_backward — include/ops/backward/attention_backward.h:24-35.
 * Same without saved output/LSE: both are recomputed first. */
int cgptx_flash_gqa_attention_backward(
    void* grad_query, void* grad_key, void* grad_value, const void* grad_output,
    const void* query, const void* key, const void* value, size_t batch,
    size_t query_sequence, size_t kv_sequence, size_t query_heads,
    size_t kv_heads, size_t head_dim, float attention_scale, int causal,
    size_t query_position_offset, int accumulate_grads, int dtype,
    cgptx_stream stream);

/* Layer norm's gradient (no counterpart in the reference, whose models have RMS norms only; the manner is
 * rmsnorm_backward's). x, dy, dx, residual: [rows, hidden]; weight, grad_weight, grad_bias: [hidden]; all of `dtype`.
 * With xh = (x - mean)/sqrt(mean((x - mean)^2) + eps) and g = dy*w:
 * dx = (g - mean(g) - xh*mean(g*xh))/sqrt(...) + residual, grad_weight = sum_rows dy*xh, grad_bias = sum_rows dy.
 * residual is the gradient that reaches x past the norm; it may be NULL and may be grad_input. grad_bias may be NULL.
 * Outputs are overwritten. */
int cgptx_layernorm_backward(void* grad_input, void* grad_weight, void* grad_bias,
                             const void* grad_output, const void* input,
                             const void* weight, const void* residual, size_t rows,
                             size_t hidden, float epsilon, int dtype,
                             cgptx_stream stream);

/* Dropout's gradient with the mask of the forward call of the same probability, seed, offset, counter and count (see
 * cgptx_dropout_forward): grad_input = grad_output*mask, added to what grad_input holds with `accumulate`.
 * grad_input may be grad_output (without accumulate). */
int cgptx_dropout_backward(void* grad_input, const void* grad_output, size_t count,
                           float probability, uint64_t seed, uint64_t offset,
                           const uint64_t* counter, int accumulate, int dtype,
                           cgptx_stream stream);

/* Gradients of differential attention (see cgptx_differential_attention_forward, which leaves output, second and
 * logsumexp). grad_lambda: fp32 [query_heads]. accumulate_grads adds to all four. The workgroups' parts of every sum meet
 * in a fixed order: results do not depend on scheduling. How many parts there are goes by the sizes and, where the scratch
 * arena cannot grow (a call that is recorded on a stream where no eager call of its sizes ran), by what it has room for:
 * such a call adds in another order than an eager one, and its results may differ from that one's by rounding. In 16-bit
 * storage P1 - lambda P2 and the score gradients are rounded to it once before their products, as in plain attention, and
 * row sums come from output and second as they are stored; in half precision the former are enlarged by a power of two
 * first where output gradients are small. Keys that no query sees get gradients of 0 whatever they hold. */
int cgptx_differential_attention_backward(
    void* grad_query, void* grad_key, void* grad_value, float* grad_lambda,
    const void* grad_output, const void* output, const void* second,
    const float* logsumexp, const void* query, const void* key, const void* value,
    const float* lambda, size_t batch, size_t query_sequence, size_t kv_sequence,
    size_t query_heads, size_t kv_heads, size_t head_dim, float attention_scale,
    int causal, size_t query_position_offset, int accumulate_grads, int dtype,
    cgptx_stream stream);

/* Gradients of differential_lambda's vectors from grad_lambda (fp32 [heads]), in their shapes and dtype; one set for all
 * heads gets the sum over the heads. */
int cgptx_differential_lambda_backward(void* grad_query1, void* grad_key1,
                                       void* grad_query2, void* grad_key2,
                                       const float* grad_lambda, const void* query1,
                                       const void* key1, const void* query2,
                                       const void* key2, size_t sets, size_t heads,
                                       size_t width, int dtype, cgptx_stream stream);

/* Gradients of linear attention (see cgptx_linear_attention_forward). grad_final_state: the gradient that reaches the final state, NULL
 * for none; grad_initial_state: the one that reaches the initial state, NULL where it is not wanted, else no other tensor of the call;
 * both fp32 like the states. accumulate_grads adds to grad_query, grad_key and grad_value; grad_initial_state is overwritten. The decays get
 * no gradient: they are constants of a model. How sums are cut and rounded is as in the forward call. */
int cgptx_linear_attention_backward(
    void* grad_query, void* grad_key, void* grad_value, float* grad_initial_state,
    const void* grad_output, const float* grad_final_state, const void* query,
    const void* key, const void* value, const float* log_decay,
    const float* initial_state, size_t batch, size_t sequence, size_t query_heads,
    size_t kv_heads, size_t head_dim, float attention_scale, int accumulate_grads,
    int dtype, cgptx_stream stream);

/* Gradients of the norms between two branches (see cgptx_sandwich_norm_forward). stream_output is the forward's; grad_stream_output is the
 * gradient that reaches it past the norm (NULL for none), grad_normed the one of normed. With G = grad_stream_output + that norm's gradient:
 * grad_stream_input = residual_scale*G, grad_branch the branch norm's gradient of gate*G, grad_gate = sum G*rmsnorm(branch)*branch_weight
 * over the rows of a gate. grad_gate may be NULL (and is, without a gate); grad_stream_input may be grad_stream_output. Outputs are
 * overwritten. */
int cgptx_sandwich_norm_backward(
    void* grad_stream_input, void* grad_branch, void* grad_branch_weight,
    void* grad_gate, void* grad_norm_weight, const void* grad_stream_output,
    const void* grad_normed, const void* stream_output, const void* branch,
    const void* branch_weight, const void* gate, const void* norm_weight,
    size_t rows, size_t hidden, size_t gate_rows, float residual_scale,
    float epsilon, int dtype, cgptx_stream stream);

/* ------------------------------------------------------------------- AdamW */

/* AdamWOptions — include/optim/adamw.h:12-27. */
typedef struct cgptx_adamw_options {
    float learning_rate;
    float beta1;
    float beta2;
    float epsilon;
    float weight_decay;
    float loss_scale;
    float max_grad_norm; /* +inf disables clipping */
} cgptx_adamw_options;

/* One parameter tensor of a batched update (AdamWBatchEntry + AdamWState,
 * include/optim/adamw.h:33-57). parameter/gradient are `dtype`; the three state
 * buffers are fp32. */
typedef struct cgptx_adamw_entry {
    void* parameter;
    const void* gradient;
    float* master_parameter;
    float* first_moment;
    float* second_moment;
    size_t count;
    int dtype;
} cgptx_adamw_entry;

typedef struct cgptx_adamw_workspace cgptx_adamw_workspace; /* AdamWWorkspace, adamw.h:60-84 */

int cgptx_adamw_workspace_create(cgptx_adamw_workspace** workspace);
int cgptx_adamw_workspace_destroy(cgptx_adamw_workspace* workspace);

/* adamw_step_many_async — include/optim/adamw.h:103-107 → src/optim/adamw.cu:276-346.
 * One global-norm AdamW update over all entries, fully on the device: gradient
 * statistics, non-finite check (skip everything, latch a sticky flag, do not
 * advance the step), bias correction, clipping, update. The first call binds the
 * workspace to this entry list and uploads initial_step; later calls must pass
 * the same list. Never synchronises. */
int cgptx_adamw_step_many_async(cgptx_adamw_workspace* workspace,
                                const cgptx_adamw_entry* entries,
                                size_t entry_count,
                                const cgptx_adamw_options* options,
                                uint64_t initial_step, cgptx_stream stream);

/* adamw_check — include/optim/adamw.h:114-115 → adamw.cu:348-359. Synchronises
 * the stream; *all_finite = 0 if any step since the last check saw NaN/Inf;
 * *step = device step counter; clears the sticky flag. */
int cgptx_adamw_check(cgptx_adamw_workspace* workspace, int* all_finite,
                      uint64_t* step, cgptx_stream stream);

/* adamw_step (single tensor, host-synchronous) — include/optim/adamw.h:131-136 →
 * adamw.cu:396-435. bias corrections come from the host in double as there;
 * *updated = 0 if the gradient held NaN/Inf (nothing is changed then). */
int cgptx_adamw_step(void* parameter, const void* gradient,
                     float* master_parameter, float* first_moment,
                     float* second_moment, size_t count, int dtype,
                     const cgptx_adamw_options* options, uint64_t next_step,
                     int* updated, cgptx_stream stream);

/* ------------------------------------------------------------------ forward */

/* rmsnorm_forward — include/ops/rmsnorm.h. y = x·rsqrt(mean x²+eps)·w. */
int cgptx_rmsnorm_forward(void* output, const void* input, const void* weight,
                          size_t rows, size_t hidden, float epsilon, int dtype,
                          cgptx_stream stream);

/* rope_forward (in place on q and k) — include/ops/rope.h:32-39. */
int cgptx_rope_forward(void* query, void* key, const void* cos_cache,
                       const void* sin_cache, size_t batch, size_t sequence,
                       size_t query_heads, size_t kv_heads, size_t head_dim,
                       size_t rotary_dim, size_t position_offset,
                       size_t cache_positions, int dtype, cgptx_stream stream);

/* swiglu_forward — include/ops/swiglu.h. out = silu(gate)·up. */
int cgptx_swiglu_forward(void* output, const void* gate, const void* up,
                         size_t count, int dtype, cgptx_stream stream);

/* swiglu_forward (packed input [rows, 2*hidden] = [gate | up]) — include/ops/swiglu.h:33-37,
 * src/ops/swiglu.cu:152-170. output is [rows, hidden]. */
int cgptx_swiglu_forward_packed(void* output, const void* gate_up, size_t rows,
                                size_t hidden, int dtype, cgptx_stream stream);

/* linear_forward — include/ops/linear.h. Y[rows,out] = X[rows,in]·W[out,in]ᵀ (+ bias[out]).
 * bias may be NULL. */
int cgptx_linear_forward(void* output, const void* input, const void* weight,
                         const void* bias, size_t rows, size_t in_features,
                         size_t out_features, int dtype, cgptx_stream stream);

/* The feed-forward's gate and up projections and its SwiGLU in one call — the sequence
 * linear_forward(gate), linear_forward(up), swiglu_forward(activated, gate, up) of
 * src/core/transformer_block.cu:586-590 with the concatenated layouts of include/ops/swiglu.h:33-37:
 * weight = [gate_proj; up_proj] ([2*hidden, in]), gate_up = [rows, 2*hidden] = [gate | up] (kept for the
 * backward pass), activated[rows, hidden] = silu(gate)·up from the rounded gate and up values. Large
 * aligned shapes run as one contraction whose epilogue writes all three; the rest as the two operators. */
int cgptx_linear_swiglu_forward(void* gate_up, void* activated, const void* input,
                                const void* weight, size_t rows, size_t in_features,
                                size_t hidden, int dtype, cgptx_stream stream);

/* The input gradient of the feed-forward's down projection and the SwiGLU gradient in one call — the
 * sequence linear_backward(down) (input gradient only), swiglu_backward of
 * src/core/transformer_block.cu:663-666 with the concatenated layouts of
 * src/ops/backward/swiglu_backward.cu:830-883: weight = down_proj ([out, hidden]), gate_up = the forward's
 * [rows, 2*hidden] = [gate | up], grad_gate_up = [rows, 2*hidden] = [dgate | dup], computed from
 * grad_output·weight rounded to the storage dtype. grad_activated ([rows, hidden]) is working memory: the
 * two-operator path writes the intermediate gradient there, the fused contraction (large aligned shapes)
 * leaves it untouched. */
int cgptx_linear_swiglu_backward(void* grad_gate_up, void* grad_activated, const void* grad_output,
                                 const void* weight, const void* gate_up, size_t rows,
                                 size_t hidden, size_t out_features, int dtype, cgptx_stream stream);

/* The weight gradients of `count` layers of one shape in one launch — `count` calls of linear_backward
 * (include/ops/backward/linear_backward.h:36-46) that ask for the weight gradient only, as
 * src/core/transformer_block.cu:660-745 makes them for every block of a model: layer j reads grad_output +
 * j * grad_output_stride ([rows, out_features]) and input + j * input_stride ([rows, in_features]), strides in
 * elements, and writes rows j * out_features .. of grad_weight ([count * out_features, in_features]). One launch
 * over all layers' tiles fills the chip without splitting the row sum of each product into partial tiles; shapes it
 * does not take (fp32 storage, out_features not a multiple of 256, unaligned tensors) run as `count` separate
 * weight gradients. */
int cgptx_linear_backward_weights_stacked(void* grad_weight, const void* grad_output, const void* input,
                                          size_t rows, size_t in_features, size_t out_features, size_t count,
                                          size_t grad_output_stride, size_t input_stride, int dtype,
                                          cgptx_stream stream);

/* embedding_forward — include/ops/embedding.h. out[t,:] = W[id_t,:]; ids >= vocab give a zero row. */
int cgptx_embedding_forward(void* output, const uint32_t* token_ids,
                            size_t token_count, const void* weight,
                            size_t vocab, size_t hidden, int dtype,
                            cgptx_stream stream);

/* flash_gqa_attention_forward_with_lse — include/ops/attention.h:70-78.
 * logsumexp may be NULL (flash_gqa_attention_forward, attention.h:47-54). */
int cgptx_flash_gqa_attention_forward(
    void* output, float* logsumexp, const void* query, const void* key,
    const void* value, size_t batch, size_t query_sequence, size_t kv_sequence,
    size_t query_heads, size_t kv_heads, size_t head_dim, float attention_scale,
    int causal, size_t query_position_offset, int dtype, cgptx_stream stream);

/* Layer norm: y = (x - mean(x))/sqrt(mean((x - mean)^2) + eps)*w + b over rows of `hidden` values; bias may be NULL.
 * No counterpart in the reference (RMS norms only). */
int cgptx_layernorm_forward(void* output, const void* input, const void* weight,
                            const void* bias, size_t rows, size_t hidden,
                            float epsilon, int dtype, cgptx_stream stream);

/* Dropout onto a residual stream: output = residual + input*mask, mask = 0 with the given probability and the inverse of
 * the share kept otherwise. No counterpart in the reference. residual may be NULL; output may be input or residual.
 * The mask is never stored. Elements 8j .. 8j + 7 take the eight 16-bit numbers (low halves first) of Philox 4x32-10
 * with key `seed` at counter offset + j (+ *counter, read on the device when the call runs, where counter is not NULL: a
 * replayed graph draws new masks as a program moves it on); an element is dropped where its number is below
 * round(65536*probability). A call uses up (count + 7)/8 counter values: the next one's offset starts behind them.
 * 0 <= probability <= 1, in steps of 2^-16; count 0 does nothing. */
int cgptx_dropout_forward(void* output, const void* input, const void* residual,
                          size_t count, float probability, uint64_t seed,
                          uint64_t offset, const uint64_t* counter, int dtype,
                          cgptx_stream stream);

/* Differential attention (no counterpart in the reference; tensors, options and checks are flash_gqa_attention's). A head's
 * query and key are two halves of head_dim/2, values are head_dim wide:
 *   output = softmax(s q1 k1') v - lambda[head] softmax(s q2 k2') v.
 * head_dim: even, at most 128; attention_scale <= 0 selects s = 1/sqrt(head_dim/2); lambda: fp32 [query_heads], on the
 * device. For the backward pass: second [batch, query_sequence, query_heads, head_dim] = softmax(s q2 k2') v, logsumexp
 * fp32 [2, batch, query_sequence, query_heads] of both maps; either may be NULL. Few queries of many keys: workgroups share
 * the keys, as many as the scratch arena has room for; recorded where it cannot grow, the call adds in another order. In 16-bit
 * storage a map's probabilities are rounded to it once before their product with v. */
int cgptx_differential_attention_forward(
    void* output, void* second, float* logsumexp, const void* query,
    const void* key, const void* value, const float* lambda, size_t batch,
    size_t query_sequence, size_t kv_sequence, size_t query_heads,
    size_t kv_heads, size_t head_dim, float attention_scale, int causal,
    size_t query_position_offset, int dtype, cgptx_stream stream);

/* The weights of differential attention's second maps: lambda[h] = exp(q1.k1) - exp(q2.k2) + initial, fp32 [heads], from
 * learned vectors [sets, width] of `dtype`; sets = heads, or 1: one set for all heads. */
int cgptx_differential_lambda_forward(float* lambda, const void* query1,
                                      const void* key1, const void* query2,
                                      const void* key2, float initial, size_t sets,
                                      size_t heads, size_t width, int dtype,
                                      cgptx_stream stream);

/* Linear attention with a decay for each key/value head (no counterpart in the reference; tensors, heads and scale are
 * flash_gqa_attention's, one sequence length for all). A kv head keeps a matrix S [head_dim, head_dim] that the query heads of its group read:
 *   S_t = exp(log_decay) S_{t-1} + k_t v_t',  output_t = s S_t' q_t.
 * log_decay: fp32 [kv_heads] on the device, at most 0 (larger values count as 0; -inf forgets all but the token itself). States are fp32
 * [batch, kv_heads, head_dim (k), head_dim (v)]; initial_state NULL: zeros; final_state, the matrix behind the last token, may be
 * NULL and must not be initial_state. head_dim up to 128, batch up to 65535, batch*query_heads up to 2^20, sequence up to 2^30; attention_scale <= 0
 * selects 1/sqrt(head_dim).
 * What a token adds to the final state n tokens further on is exact to 2^-22, and to 2^-21 (1 + |n log_decay|) for its weight, of itself. For the
 * output of 16-bit inputs, scores and states are rounded to 16 bits once where they enter a product and decayed values kept to 2^-16. Half
 * precision brings scores, states and decayed values into its range by a power of two for all of a tile's: each of them may also be off by 2^-22
 * (scores, states) or 2^-39 (decayed values, also of the final state) of the tile's largest.
 * A token that is not finite reaches itself and the tokens behind it. Long sequences are walked in parts side by side, as many as the scratch
 * arena has room for: recorded where it cannot grow, the call adds in another order. */
int cgptx_linear_attention_forward(
    void* output, float* final_state, const void* query, const void* key,
    const void* value, const float* log_decay, const float* initial_state,
    size_t batch, size_t sequence, size_t query_heads, size_t kv_heads,
    size_t head_dim, float attention_scale, int dtype, cgptx_stream stream);

/* One token of linear attention for every sequence: query, output [batch, query_heads, head_dim], key, value [batch, kv_heads, head_dim];
 * next_state = exp(log_decay) state + k v', output from next_state, which may be state itself. All sums are fp32. */
int cgptx_linear_attention_step(
    void* output, float* next_state, const float* state, const void* query,
    const void* key, const void* value, const float* log_decay, size_t batch,
    size_t query_heads, size_t kv_heads, size_t head_dim, float attention_scale,
    int dtype, cgptx_stream stream);

/* The norm behind a branch with its gate, the scale of the residual stream and the norm in front of the next branch (no counterpart in the
 * reference):
 *   stream_output = residual_scale*stream_input + gate*rmsnorm(branch)*branch_weight,  normed = rmsnorm(stream_output)*norm_weight,
 * rows of `hidden` values, rmsnorm(x) = x/sqrt(mean(x^2) + eps); the second norm reads stream_output as it is stored. gate
 * [gate_rows, hidden]: one row for all rows (a learned vector), one for each, or one for every rows/gate_rows rows in turn (a sequence's);
 * NULL with gate_rows 0: no gate. stream_output may be stream_input. At most 2^30 rows and 2^25 columns. */
int cgptx_sandwich_norm_forward(
    void* stream_output, void* normed, const void* stream_input,
    const void* branch, const void* branch_weight, const void* gate,
    const void* norm_weight, size_t rows, size_t hidden, size_t gate_rows,
    float residual_scale, float epsilon, int dtype, cgptx_stream stream);

/* Residual helpers used by the block (src/core/transformer_block.cu:134-144, 242-248):
 * out = a + b, and out += b, elementwise over `count` values. */
int cgptx_add(void* output, const void* a, const void* b, size_t count,
              int dtype, cgptx_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* CGPTX_H */
