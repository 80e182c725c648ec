// sandwich_norm_backward over the entry point of the same name (include/cgptx.h). A null grad_stream_output: nothing reaches the stream past the
// norm; grad_gate may be null, and is without a gate.
#pragma once

#include "ops/sandwich_norm.h"

inline void sandwich_norm_backward(Tensor& grad_stream_input, Tensor& grad_branch, Tensor& grad_branch_weight, Tensor* grad_gate,
                                   Tensor& grad_norm_weight, const Tensor* grad_stream_output, const Tensor& grad_normed,
                                   const Tensor& stream_output, const Tensor& branch, const Tensor& branch_weight, const Tensor* gate,
                                   const Tensor& norm_weight, float residual_scale, float epsilon, hipStream_t stream = nullptr) {
    using namespace cgptx_detail;
    const char* op = "sandwich_norm_backward";
    sandwich_shapes(op, stream_output, {&grad_stream_input, &grad_branch, grad_stream_output, &grad_normed, &branch},
                    {&grad_branch_weight, &grad_norm_weight, &branch_weight, &norm_weight}, gate);
    if (grad_gate != nullptr) {
        if (gate == nullptr) throw std::invalid_argument("sandwich_norm_backward: no gate whose gradient could be asked for");
        require_device(op, {grad_gate});
        require_same_dtype(op, *gate, {grad_gate});
        require_same_shape(op, *gate, {grad_gate});
    }
    check(cgptx_sandwich_norm_backward(
        grad_stream_input.raw_data(), grad_branch.raw_data(), grad_branch_weight.raw_data(), grad_gate != nullptr ? grad_gate->raw_data() : nullptr,
        grad_norm_weight.raw_data(), grad_stream_output != nullptr ? grad_stream_output->raw_data() : nullptr, grad_normed.raw_data(),
        stream_output.raw_data(), branch.raw_data(), branch_weight.raw_data(), gate != nullptr ? gate->raw_data() : nullptr,
        norm_weight.raw_data(), stream_output.size(0), stream_output.size(1), gate != nullptr ? gate->size(0) : 0, residual_scale, epsilon,
        dtype_code(stream_output.dtype()), stream));
}
