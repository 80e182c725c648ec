// sandwich_norm_forward over the entry point of the same name (include/cgptx.h). No counterpart in the reference, whose blocks have one norm in
// front of each branch; the manner is that of include/ops/rmsnorm.h. Rows [rows, hidden]; a gate [gate rows, hidden] or none (null).
#pragma once

#include "core/status.h"
#include "core/tensor.h"

namespace cgptx_detail {
inline void sandwich_shapes(const char* op, const Tensor& first, std::initializer_list<const Tensor*> rows,
                            std::initializer_list<const Tensor*> weights, const Tensor* gate) {
    if (first.dim() != 2) throw std::invalid_argument(std::string(op) + ": rows must be [rows, hidden]");
    require_device(op, {&first});
    for (const Tensor* t : rows) {
        if (t == nullptr) continue;
        require_device(op, {t});
        require_same_dtype(op, first, {t});
        require_same_shape(op, first, {t});
    }
    for (const Tensor* t : weights) {
        require_device(op, {t});
        require_same_dtype(op, first, {t});
        if (t->dim() != 1 || t->size(0) != first.size(1)) throw std::invalid_argument(std::string(op) + ": incompatible shapes");
    }
    if (gate == nullptr) return;
    require_device(op, {gate});
    require_same_dtype(op, first, {gate});
    if (gate->dim() != 2 || gate->size(1) != first.size(1) || gate->size(0) == 0 || first.size(0) % gate->size(0) != 0)
        throw std::invalid_argument(std::string(op) + ": the gate must have one row for every equal number of rows");
}
}  // namespace cgptx_detail

inline void sandwich_norm_forward(Tensor& stream_output, Tensor& normed, const Tensor& stream_input, const Tensor& branch,
                                  const Tensor& branch_weight, const Tensor* gate, const Tensor& norm_weight, float residual_scale, float epsilon,
                                  hipStream_t stream = nullptr) {
    using namespace cgptx_detail;
    sandwich_shapes("sandwich_norm_forward", stream_input, {&stream_output, &normed, &branch}, {&branch_weight, &norm_weight}, gate);
    check(cgptx_sandwich_norm_forward(stream_output.raw_data(), normed.raw_data(), stream_input.raw_data(), branch.raw_data(),
                                      branch_weight.raw_data(), gate != nullptr ? gate->raw_data() : nullptr, norm_weight.raw_data(),
                                      stream_input.size(0), stream_input.size(1), gate != nullptr ? gate->size(0) : 0, residual_scale, epsilon,
                                      dtype_code(stream_input.dtype()), stream));
}
