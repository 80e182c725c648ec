// Layer norm forward and backward for gfx950.
//
//   xh = (x - mean(x)) r,  r = 1/sqrt(mean((x - mean(x))^2) + eps),  y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)) [+ residual],  dw = sum_rows dy xh,  db = sum_rows dy
//
// The mean is taken off before squares are summed: in a row far from zero the difference of mean(x^2) and mean(x)^2
// would be rounding. Nothing is saved between the passes; the backward pass has the row at hand and takes its statistics
// anew. All sums are fp32.
//
// One workgroup takes a row at a time and walks it as often as a sum needs (the row comes from the caches behind the
// first walk); a second kernel walks columns for dw and db.
#include "common.hpp"
#include "reduce.hpp"

#include <cmath>
#include <limits>

namespace cgptx {
namespace {

constexpr int kThreads = 256;
constexpr int kWavesPerBlock = kThreads / kWave;

// Sum over the workgroup, the same bits in every thread. `stage` may be used again behind the next call's first barrier.
__device__ __forceinline__ float block_sum(float v, float* stage) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) stage[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int s = 0; s < kWavesPerBlock; ++s) v += stage[s];
    return v;
}

template <typename T, bool Backward>
__global__ __launch_bounds__(kThreads) void layernorm_row_kernel(T* out, float* __restrict__ statistics /* [rows][mean, r] */,
                                                                 const T* __restrict__ dy, const T* residual, const T* x,
                                                                 const T* __restrict__ w, const T* __restrict__ bias, int rows,
                                                                 int hidden, float inv_hidden, float eps) {
    __shared__ float stage[kWavesPerBlock];
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const std::size_t base = static_cast<std::size_t>(row) * hidden;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < hidden; c += kThreads) sum += to_f32(x[base + c]);
        const float mean = block_sum(sum, stage) * inv_hidden;
        float squares = 0.0f;
        for (int c = threadIdx.x; c < hidden; c += kThreads) {
            const float d = to_f32(x[base + c]) - mean;
            squares = fmaf(d, d, squares);
        }
        const float r = 1.0f / sqrtf(block_sum(squares, stage) * inv_hidden + eps);
        if constexpr (Backward) {
            float g_sum = 0.0f, gx_sum = 0.0f;
            for (int c = threadIdx.x; c < hidden; c += kThreads) {
                const float g = to_f32(dy[base + c]) * to_f32(w[c]);
                g_sum += g;
                gx_sum = fmaf(g, (to_f32(x[base + c]) - mean) * r, gx_sum);
            }
            const float g_mean = block_sum(g_sum, stage) * inv_hidden;
            const float gx_mean = block_sum(gx_sum, stage) * inv_hidden;
            if (threadIdx.x == 0) {
                statistics[2 * static_cast<std::size_t>(row)] = mean;
                statistics[2 * static_cast<std::size_t>(row) + 1] = r;
            }
            for (int c = threadIdx.x; c < hidden; c += kThreads) {
                const float xh = (to_f32(x[base + c]) - mean) * r;
                float v = r * (to_f32(dy[base + c]) * to_f32(w[c]) - g_mean - xh * gx_mean);
                if (residual != nullptr) v += to_f32(residual[base + c]);
                out[base + c] = from_f32<T>(v);
            }
        } else {
            for (int c = threadIdx.x; c < hidden; c += kThreads) {
                float v = (to_f32(x[base + c]) - mean) * r * to_f32(w[c]);
                if (bias != nullptr) v += to_f32(bias[c]);
                out[base + c] = from_f32<T>(v);
            }
        }
    }
}

// Partial sums [slices][hidden] of dw and, behind them, of db: 64 columns and a slice of the rows per workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void layernorm_column_kernel(float* __restrict__ partial, const T* __restrict__ dy,
                                                                    const T* __restrict__ x, const float* __restrict__ statistics,
                                                                    int rows, int hidden, int rows_per_slice) {
    __shared__ float stage[2][kWavesPerBlock][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int col = blockIdx.x * kWave + lane;
    const int row_begin = blockIdx.y * rows_per_slice, row_end = min(rows, row_begin + rows_per_slice);
    float dw = 0.0f, db = 0.0f;
    if (col < hidden) {
        for (int row = row_begin + wave; row < row_end; row += kWavesPerBlock) {
            const std::size_t index = static_cast<std::size_t>(row) * hidden + col;
            const float mean = statistics[2 * static_cast<std::size_t>(row)], r = statistics[2 * static_cast<std::size_t>(row) + 1];
            const float g = to_f32(dy[index]);
            dw = fmaf(g, (to_f32(x[index]) - mean) * r, dw);
            db += g;
        }
    }
    stage[0][wave][lane] = dw;
    stage[1][wave][lane] = db;
    __syncthreads();
    if (wave < 2 && col < hidden) {
        float total = 0.0f;
#pragma unroll
        for (int s = 0; s < kWavesPerBlock; ++s) total += stage[wave][s][lane];
        partial[(static_cast<std::size_t>(wave) * gridDim.y + blockIdx.y) * hidden + col] = total;
    }
}

int validate(const char* name, std::size_t rows, std::size_t hidden, float eps, int dtype) {
    const std::string n(name);
    if (!valid_dtype(dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (!std::isfinite(eps) || eps <= 0.0f) return fail(CGPTX_INVALID_ARGUMENT, n + ": epsilon must be finite and positive");
    if (rows == 0 || hidden == 0) return fail(CGPTX_INVALID_ARGUMENT, n + ": empty shape");
    constexpr std::size_t limit = std::size_t{1} << 30;
    if (rows > limit || hidden > limit) return fail(CGPTX_INVALID_ARGUMENT, n + ": dimensions exceed supported range");
    return CGPTX_OK;
}

int row_blocks(int rows) { return rows < compute_units() * 8 ? rows : compute_units() * 8; }

}  // namespace
}  // namespace cgptx

extern "C" int cgptx_layernorm_forward(void* output, const void* input, const void* weight, const void* bias, size_t rows,
                                       size_t hidden, float epsilon, int dtype, cgptx_stream stream_) {
    using namespace cgptx;
    if (int s = validate("layernorm_forward", rows, hidden, epsilon, dtype)) return s;
    if (output == nullptr || input == nullptr || weight == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, "layernorm_forward: null tensor");
    auto stream = static_cast<hipStream_t>(stream_);
    const int r = static_cast<int>(rows), h = static_cast<int>(hidden);
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        hipLaunchKernelGGL((layernorm_row_kernel<T, false>), dim3(row_blocks(r)), dim3(kThreads), 0, stream, static_cast<T*>(output),
                           nullptr, nullptr, nullptr, static_cast<const T*>(input), static_cast<const T*>(weight),
                           static_cast<const T*>(bias), r, h, 1.0f / static_cast<float>(h), epsilon);
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}

extern "C" int cgptx_layernorm_backward(void* grad_input, void* grad_weight, void* grad_bias, const void* grad_output,
                                        const void* input, const void* weight, const void* residual, size_t rows, size_t hidden,
                                        float epsilon, int dtype, cgptx_stream stream_) {
    using namespace cgptx;
    if (int s = validate("layernorm_backward", rows, hidden, epsilon, dtype)) return s;
    if (grad_input == nullptr || grad_weight == nullptr || grad_output == nullptr || input == nullptr || weight == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, "layernorm_backward: null tensor");
    auto stream = static_cast<hipStream_t>(stream_);
    const int r = static_cast<int>(rows), h = static_cast<int>(hidden);
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        auto* dy = static_cast<const T*>(grad_output);
        auto* x = static_cast<const T*>(input);
        const int slices = r < 256 ? 1 : (r < 65536 ? 64 : 256);
        const int rows_per_slice = (r + slices - 1) / slices;
        const std::size_t statistics_bytes = (2 * rows * sizeof(float) + 255) & ~std::size_t{255};
        void* mem = nullptr;
        if (int s = scratch(stream, statistics_bytes + 2 * static_cast<std::size_t>(slices) * hidden * sizeof(float), &mem)) return s;
        auto* statistics = static_cast<float*>(mem);
        auto* partial = reinterpret_cast<float*>(static_cast<char*>(mem) + statistics_bytes);
        hipLaunchKernelGGL((layernorm_row_kernel<T, true>), dim3(row_blocks(r)), dim3(kThreads), 0, stream, static_cast<T*>(grad_input),
                           statistics, dy, static_cast<const T*>(residual), x, static_cast<const T*>(weight), nullptr, r, h,
                           1.0f / static_cast<float>(h), epsilon);
        CGPTX_LAUNCH_CHECK();
        hipLaunchKernelGGL((layernorm_column_kernel<T>), dim3((h + kWave - 1) / kWave, slices), dim3(kThreads), 0, stream, partial, dy,
                           x, statistics, r, h, rows_per_slice);
        CGPTX_LAUNCH_CHECK();
        launch_column_partial_reduce<T>(static_cast<T*>(grad_weight), partial, slices, h, 0, stream);
        CGPTX_LAUNCH_CHECK();
        if (grad_bias != nullptr) {
            launch_column_partial_reduce<T>(static_cast<T*>(grad_bias), partial + static_cast<std::size_t>(slices) * hidden, slices, h,
                                            0, stream);
            CGPTX_LAUNCH_CHECK();
        }
        return CGPTX_OK;
    });
}
