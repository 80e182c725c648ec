// differential_attention_backward and differential_lambda_backward over the entry points of the same names (include/cgptx.h).
#pragma once

#include "ops/differential_attention.h"

inline void differential_attention_backward(Tensor& grad_query, Tensor& grad_key, Tensor& grad_value, Tensor& grad_lambda,
                                            const Tensor& grad_output, const Tensor& output, const Tensor& second, const Tensor& logsumexp,
                                            const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& lambda,
                                            hipStream_t stream = nullptr, const FlashAttentionOptions& options = {},
                                            bool accumulate_grads = false) {
    using namespace cgptx_detail;
    const char* op = "differential_attention_backward";
    require_device(op, {&grad_query, &grad_key, &grad_value, &grad_lambda, &grad_output, &output, &second, &logsumexp, &query, &key, &value,
                        &lambda});
    require_same_dtype(op, query, {&grad_query, &grad_key, &grad_value, &grad_output, &output, &second, &key, &value});
    require_same_shape(op, query, {&grad_query, &grad_output, &output, &second});
    require_same_shape(op, key, {&grad_key, &grad_value});
    require_same_dtype(op, lambda, {&grad_lambda});
    require_same_shape(op, lambda, {&grad_lambda});
    const AttentionShape s = differential_shape(op, query, key, value, lambda, &logsumexp, options);
    check(cgptx_differential_attention_backward(
        grad_query.raw_data(), grad_key.raw_data(), grad_value.raw_data(), static_cast<float*>(grad_lambda.raw_data()),
        grad_output.raw_data(), output.raw_data(), second.raw_data(), static_cast<const float*>(logsumexp.raw_data()), query.raw_data(),
        key.raw_data(), value.raw_data(), static_cast<const float*>(lambda.raw_data()), s.batch, s.query_sequence, s.kv_sequence,
        options.num_query_heads, options.num_kv_heads, options.head_dim, options.attention_scale, options.causal,
        options.query_position_offset, accumulate_grads, dtype_code(query.dtype()), stream));
}

inline void differential_lambda_backward(Tensor& grad_query1, Tensor& grad_key1, Tensor& grad_query2, Tensor& grad_key2,
                                         const Tensor& grad_lambda, const Tensor& query1, const Tensor& key1, const Tensor& query2,
                                         const Tensor& key2, hipStream_t stream = nullptr) {
    using namespace cgptx_detail;
    differential_vectors("differential_lambda_backward", grad_lambda,
                         {&query1, &key1, &query2, &key2, &grad_query1, &grad_key1, &grad_query2, &grad_key2});
    check(cgptx_differential_lambda_backward(grad_query1.raw_data(), grad_key1.raw_data(), grad_query2.raw_data(), grad_key2.raw_data(),
                                             static_cast<const float*>(grad_lambda.raw_data()), query1.raw_data(), key1.raw_data(),
                                             query2.raw_data(), key2.raw_data(), query1.size(0), grad_lambda.size(0), query1.size(1),
                                             dtype_code(query1.dtype()), stream));
}
