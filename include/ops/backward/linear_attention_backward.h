// linear_attention_backward over the entry point of the same name (include/cgptx.h). A null grad_final_state: nothing reaches the final state; a
// null grad_initial_state: not wanted.
#pragma once

#include "ops/linear_attention.h"

inline void linear_attention_backward(Tensor& grad_query, Tensor& grad_key, Tensor& grad_value, Tensor* grad_initial_state,
                                      const Tensor& grad_output, const Tensor* grad_final_state, const Tensor& query, const Tensor& key,
                                      const Tensor& value, const Tensor& log_decay, const Tensor* initial_state = nullptr,
                                      hipStream_t stream = nullptr, const FlashAttentionOptions& options = {}, bool accumulate_grads = false) {
    using namespace cgptx_detail;
    const char* op = "linear_attention_backward";
    require_device(op, {&grad_query, &grad_key, &grad_value, &grad_output, &query, &key, &value});
    require_same_dtype(op, query, {&grad_query, &grad_key, &grad_value, &grad_output, &key, &value});
    require_same_shape(op, query, {&grad_query, &grad_output});
    require_same_shape(op, key, {&grad_key, &grad_value});
    const AttentionShape s = linear_shape(op, query, key, value, log_decay, {grad_initial_state, grad_final_state, initial_state}, options);
    check(cgptx_linear_attention_backward(grad_query.raw_data(), grad_key.raw_data(), grad_value.raw_data(), state_data(grad_initial_state),
                                          grad_output.raw_data(), state_data(grad_final_state), query.raw_data(), key.raw_data(),
                                          value.raw_data(), static_cast<const float*>(log_decay.raw_data()), state_data(initial_state), s.batch,
                                          s.query_sequence, options.num_query_heads, options.num_kv_heads, options.head_dim,
                                          options.attention_scale, accumulate_grads, dtype_code(query.dtype()), stream));
}
