// dropout_backward over cgptx_dropout_backward: the gradient under the mask that dropout_forward had of the same options.
#pragma once

#include "ops/dropout.h"

inline void dropout_backward(Tensor& grad_input, const Tensor& grad_output, hipStream_t stream = nullptr,
                             const DropoutOptions& options = {}, bool accumulate = false) {
    using namespace cgptx_detail;
    const char* op = "dropout_backward";
    require_device(op, {&grad_input, &grad_output});
    require_same_dtype(op, grad_output, {&grad_input});
    require_same_shape(op, grad_output, {&grad_input});
    check(cgptx_dropout_backward(grad_input.raw_data(), grad_output.raw_data(), grad_output.numel(), options.probability, options.seed,
                                 options.offset, options.counter, accumulate, dtype_code(grad_output.dtype()), stream));
}
