// differential_attention_forward and differential_lambda_forward over the entry points of the same names (include/cgptx.h). No
// counterparts in the reference; tensors and options are those of flash_gqa_attention_forward_with_lse. A head's query and key hold
// both maps' halves side by side; lambda and both logsumexps ([2, batch, sequence, heads]) are F32.
#pragma once

#include "ops/attention.h"

namespace cgptx_detail {
inline AttentionShape differential_shape(const char* op, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& lambda,
                                         const Tensor* logsumexp, const FlashAttentionOptions& o) {
    const AttentionShape s = attention_shape(op, query, key, value, o);
    if (o.head_dim % 2 != 0) throw std::invalid_argument(std::string(op) + ": head_dim must be even");
    if (lambda.dtype() != Dtype::F32 || lambda.numel() != o.num_query_heads)
        throw std::invalid_argument(std::string(op) + ": lambda must be F32 [query heads]");
    if (logsumexp != nullptr &&
        (logsumexp->dtype() != Dtype::F32 || logsumexp->numel() != 2 * s.batch * s.query_sequence * o.num_query_heads))
        throw std::invalid_argument(std::string(op) + ": logsumexp must be F32 [2, batch, sequence, heads]");
    return s;
}
inline void differential_attention(Tensor& output, Tensor* second, Tensor* logsumexp, const Tensor& query, const Tensor& key,
                                   const Tensor& value, const Tensor& lambda, hipStream_t stream, const FlashAttentionOptions& options) {
    const char* op = "differential_attention_forward";
    require_device(op, {&output, &query, &key, &value, &lambda});
    require_same_dtype(op, query, {&output, &key, &value});
    require_same_shape(op, query, {&output});
    if (second != nullptr) {
        require_device(op, {second, logsumexp});
        require_same_dtype(op, query, {second});
        require_same_shape(op, query, {second});
    }
    const AttentionShape s = differential_shape(op, query, key, value, lambda, logsumexp, options);
    check(cgptx_differential_attention_forward(
        output.raw_data(), second != nullptr ? second->raw_data() : nullptr,
        logsumexp != nullptr ? static_cast<float*>(logsumexp->raw_data()) : nullptr, query.raw_data(), key.raw_data(), value.raw_data(),
        static_cast<const float*>(lambda.raw_data()), s.batch, s.query_sequence, s.kv_sequence, options.num_query_heads,
        options.num_kv_heads, options.head_dim, options.attention_scale, options.causal, options.query_position_offset,
        dtype_code(query.dtype()), stream));
}
// Vectors [sets, width] of lambda [heads].
inline void differential_vectors(const char* op, const Tensor& lambda, std::initializer_list<const Tensor*> vectors) {
    const Tensor& first = **vectors.begin();
    for (const Tensor* v : vectors) {
        require_device(op, {v});
        require_same_dtype(op, first, {v});
        require_same_shape(op, first, {v});
    }
    require_device(op, {&lambda});
    if (lambda.dtype() != Dtype::F32 || lambda.dim() != 1 || first.dim() != 2 || (first.size(0) != 1 && first.size(0) != lambda.size(0)))
        throw std::invalid_argument(std::string(op) + ": lambda must be F32 [heads], the vectors one set for all heads or one for each");
}
}  // namespace cgptx_detail

// With what differential_attention_backward needs.
inline void differential_attention_forward(Tensor& output, Tensor& second, Tensor& logsumexp, const Tensor& query, const Tensor& key,
                                           const Tensor& value, const Tensor& lambda, hipStream_t stream = nullptr,
                                           const FlashAttentionOptions& options = {}) {
    cgptx_detail::differential_attention(output, &second, &logsumexp, query, key, value, lambda, stream, options);
}
inline void differential_attention_forward(Tensor& output, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& lambda,
                                           hipStream_t stream = nullptr, const FlashAttentionOptions& options = {}) {
    cgptx_detail::differential_attention(output, nullptr, nullptr, query, key, value, lambda, stream, options);
}

inline void differential_lambda_forward(Tensor& lambda, const Tensor& query1, const Tensor& key1, const Tensor& query2, const Tensor& key2,
                                        float initial, hipStream_t stream = nullptr) {
    using namespace cgptx_detail;
    differential_vectors("differential_lambda_forward", lambda, {&query1, &key1, &query2, &key2});
    check(cgptx_differential_lambda_forward(static_cast<float*>(lambda.raw_data()), query1.raw_data(), key1.raw_data(), query2.raw_data(),
                                            key2.raw_data(), initial, query1.size(0), lambda.size(0), query1.size(1),
                                            dtype_code(query1.dtype()), stream));
}
