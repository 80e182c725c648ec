// layernorm_forward over cgptx_layernorm_forward. No counterpart in the reference (RMS norms only); the manner is that of
// include/ops/rmsnorm.h. Without a bias: the overload that takes none.
#pragma once

#include "core/status.h"
#include "core/tensor.h"

namespace cgptx_detail {
inline void layernorm(Tensor& output, const Tensor& input, const Tensor& weight, const Tensor* bias, const float epsilon,
                      hipStream_t stream) {
    const char* op = "layernorm_forward";
    require_device(op, {&output, &input, &weight});
    require_same_dtype(op, input, {&output, &weight});
    if (input.dim() == 0 || weight.dim() != 1 || weight.size(0) != input.shape().back())
        throw std::invalid_argument("layernorm_forward: incompatible shapes");
    require_same_shape(op, input, {&output});
    if (bias != nullptr) {
        require_device(op, {bias});
        require_same_dtype(op, input, {bias});
        require_same_shape(op, weight, {bias});
    }
    const std::size_t hidden = input.shape().back();
    check(cgptx_layernorm_forward(output.raw_data(), input.raw_data(), weight.raw_data(), bias != nullptr ? bias->raw_data() : nullptr,
                                  input.numel() / hidden, hidden, epsilon, dtype_code(input.dtype()), stream));
}
}  // namespace cgptx_detail

inline void layernorm_forward(Tensor& output, const Tensor& input, const Tensor& weight, const Tensor& bias, float epsilon,
                              hipStream_t stream = nullptr) {
    cgptx_detail::layernorm(output, input, weight, &bias, epsilon, stream);
}
inline void layernorm_forward(Tensor& output, const Tensor& input, const Tensor& weight, float epsilon, hipStream_t stream = nullptr) {
    cgptx_detail::layernorm(output, input, weight, nullptr, epsilon, stream);
}
