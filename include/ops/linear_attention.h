// linear_attention_forward and linear_attention_step over the entry points of the same names (include/cgptx.h). No counterparts in the reference;
// tensors and options are those of flash_gqa_attention_forward, causal and of one sequence. log_decay is F32 [kv heads], states are F32
// [batch, kv heads, head_dim, head_dim]; a null initial state is zeros, a null final state is not wanted.
#pragma once

#include "ops/attention.h"

namespace cgptx_detail {
inline AttentionShape linear_shape(const char* op, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& log_decay,
                                   std::initializer_list<const Tensor*> states, const FlashAttentionOptions& o) {
    const AttentionShape s = attention_shape(op, query, key, value, o);
    if (!o.causal || o.query_position_offset != 0 || s.kv_sequence != s.query_sequence)
        throw std::invalid_argument(std::string(op) + ": queries and keys must be of the same tokens, the mask causal and its offset 0");
    require_device(op, {&log_decay});
    if (log_decay.dtype() != Dtype::F32 || log_decay.dim() != 1 || log_decay.size(0) != o.num_kv_heads)
        throw std::invalid_argument(std::string(op) + ": log_decay must be F32 [kv heads]");
    const std::vector<std::size_t> shape{s.batch, o.num_kv_heads, o.head_dim, o.head_dim};
    for (const Tensor* state : states) {
        if (state == nullptr) continue;
        require_device(op, {state});
        if (state->dtype() != Dtype::F32 || state->shape() != shape)
            throw std::invalid_argument(std::string(op) + ": states must be F32 [batch, kv heads, head_dim, head_dim]");
    }
    return s;
}
inline float* state_data(Tensor* state) { return state != nullptr ? static_cast<float*>(state->raw_data()) : nullptr; }
inline const float* state_data(const Tensor* state) { return state != nullptr ? static_cast<const float*>(state->raw_data()) : nullptr; }
}  // namespace cgptx_detail

inline void linear_attention_forward(Tensor& output, Tensor* final_state, const Tensor& query, const Tensor& key, const Tensor& value,
                                     const Tensor& log_decay, const Tensor* initial_state = nullptr, hipStream_t stream = nullptr,
                                     const FlashAttentionOptions& options = {}) {
    using namespace cgptx_detail;
    const char* op = "linear_attention_forward";
    require_device(op, {&output, &query, &key, &value});
    require_same_dtype(op, query, {&output, &key, &value});
    require_same_shape(op, query, {&output});
    const AttentionShape s = linear_shape(op, query, key, value, log_decay, {final_state, initial_state}, options);
    check(cgptx_linear_attention_forward(output.raw_data(), state_data(final_state), query.raw_data(), key.raw_data(), value.raw_data(),
                                         static_cast<const float*>(log_decay.raw_data()), state_data(initial_state), s.batch, s.query_sequence,
                                         options.num_query_heads, options.num_kv_heads, options.head_dim, options.attention_scale,
                                         dtype_code(query.dtype()), stream));
}

// One token of every sequence; next_state may be state.
inline void linear_attention_step(Tensor& output, Tensor& next_state, const Tensor& state, const Tensor& query, const Tensor& key,
                                  const Tensor& value, const Tensor& log_decay, hipStream_t stream = nullptr,
                                  const FlashAttentionOptions& options = {}) {
    using namespace cgptx_detail;
    const char* op = "linear_attention_step";
    require_device(op, {&output, &query, &key, &value});
    require_same_dtype(op, query, {&output, &key, &value});
    require_same_shape(op, query, {&output});
    const AttentionShape s = linear_shape(op, query, key, value, log_decay, {&next_state, &state}, options);
    if (s.query_sequence != 1) throw std::invalid_argument("linear_attention_step: query must be one token of every sequence");
    check(cgptx_linear_attention_step(output.raw_data(), state_data(&next_state), state_data(&state), query.raw_data(), key.raw_data(),
                                      value.raw_data(), static_cast<const float*>(log_decay.raw_data()), s.batch, options.num_query_heads,
                                      options.num_kv_heads, options.head_dim, options.attention_scale, dtype_code(query.dtype()), stream));
}
