// layernorm_backward over cgptx_layernorm_backward. The bias's gradient and the gradient that reaches the input past the norm
// (which may be grad_input itself) are optional: null for none.
#pragma once

#include "core/status.h"
#include "core/tensor.h"

inline void layernorm_backward(Tensor& grad_input, Tensor& grad_weight, Tensor* grad_bias, const Tensor& grad_output, const Tensor& input,
                               const Tensor& weight, float epsilon, hipStream_t stream = nullptr, const Tensor* residual = nullptr) {
    using namespace cgptx_detail;
    const char* op = "layernorm_backward";
    require_device(op, {&grad_input, &grad_weight, &grad_output, &input, &weight});
    require_same_dtype(op, input, {&grad_input, &grad_weight, &grad_output, &weight});
    if (input.dim() == 0 || weight.dim() != 1 || weight.size(0) != input.shape().back() || grad_weight.shape() != weight.shape())
        throw std::invalid_argument("layernorm_backward: incompatible shapes");
    require_same_shape(op, input, {&grad_input, &grad_output});
    if (grad_bias != nullptr) {
        require_device(op, {grad_bias});
        require_same_dtype(op, input, {grad_bias});
        require_same_shape(op, weight, {grad_bias});
    }
    if (residual != nullptr) {
        require_device(op, {residual});
        require_same_dtype(op, input, {residual});
        require_same_shape(op, input, {residual});
    }
    const std::size_t hidden = input.shape().back();
    check(cgptx_layernorm_backward(grad_input.raw_data(), grad_weight.raw_data(), grad_bias != nullptr ? grad_bias->raw_data() : nullptr,
                                   grad_output.raw_data(), input.raw_data(), weight.raw_data(),
                                   residual != nullptr ? residual->raw_data() : nullptr, input.numel() / hidden, hidden, epsilon,
                                   dtype_code(input.dtype()), stream));
}
