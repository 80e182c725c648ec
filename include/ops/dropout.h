// dropout_forward over cgptx_dropout_forward, which says how a mask follows from the options. No counterpart in the reference.
#pragma once

#include "core/status.h"
#include "core/tensor.h"

// The defaults are one mask like any other: calls that are to have masks of their own need a seed or an offset of their own.
struct DropoutOptions {
    float probability = 0.1F;
    std::uint64_t seed = 0;
    std::uint64_t offset = 0;                  // a call uses up (elements + 7) / 8 counter values from here on
    const std::uint64_t* counter = nullptr;    // on the device, added to the offset when the call runs
};

// output = residual + input under the mask; output may be input or residual.
inline void dropout_forward(Tensor& output, const Tensor& input, const Tensor& residual, hipStream_t stream = nullptr,
                            const DropoutOptions& options = {}) {
    using namespace cgptx_detail;
    const char* op = "dropout_forward";
    require_device(op, {&output, &input, &residual});
    require_same_dtype(op, input, {&output, &residual});
    require_same_shape(op, input, {&output, &residual});
    check(cgptx_dropout_forward(output.raw_data(), input.raw_data(), residual.raw_data(), input.numel(), options.probability, options.seed,
                                options.offset, options.counter, dtype_code(input.dtype()), stream));
}
inline void dropout_forward(Tensor& output, const Tensor& input, hipStream_t stream = nullptr, const DropoutOptions& options = {}) {
    using namespace cgptx_detail;
    const char* op = "dropout_forward";
    require_device(op, {&output, &input});
    require_same_dtype(op, input, {&output});
    require_same_shape(op, input, {&output});
    check(cgptx_dropout_forward(output.raw_data(), input.raw_data(), nullptr, input.numel(), options.probability, options.seed,
                                options.offset, options.counter, dtype_code(input.dtype()), stream));
}
