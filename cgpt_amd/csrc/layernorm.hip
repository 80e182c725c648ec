// Layer norm forward and backward for gfx950.
//
//   xh = (x - mean(x)) r,  r = 1/sqrt(mean((x - mean(x))^2) + eps),  y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)) [+ residual],  dw = sum_rows dy xh,  db = sum_rows dy
//
// The mean is taken off before squares are summed: in a row far from zero the difference of mean(x^2) and mean(x)^2
// would be rounding. Nothing is saved between the passes; the backward pass has the row at hand and takes its statistics
// anew. All sums are fp32.
//
// What bounds it is memory: x (and dy, residual) read once, y or dx written once. Rows of up to 16384 values stay in registers between
// the sums and the store (layernorm_rows): a wavefront owns one or several rows, or several wavefronts one, the next row's
// loads are in flight while a row is summed, and dw and db gather in the registers of the lanes that own their columns. Per-workgroup
// partial sums of them go to scratch and a second launch adds them in a fixed order. Longer rows are walked as often as a sum
// needs by a workgroup, and columns by a kernel of their own.
//
// 32768 x 1024 in bf16: forward 24.5 us (5.5 TB/s), backward with the residual gradient 57 (4.7 TB/s: the row pass 45, the column
// sums' launch 5.5). 5005 x 1001 in fp32, backward: 17.7 (13.4 and 4). 16 x 768 in fp16, forward: 3.1 on the device. Backward rows of
// more than 8192 values in fp32 are in registers by name only: sixteen wavefronts leave 128 a lane, and 150 values are spilled (1024 x
// 16384: 87 us, 2.3 TB/s). 16384 x 2048 in bf16, 288 registers and so one wavefront a SIMD: 40 us, 5.0 TB/s.
#include "common.hpp"
#include "reduce.hpp"
#include "row_vectors.hpp"

#include <cmath>
#include <limits>

namespace cgptx {
namespace {

constexpr int kThreads = kRowThreads;
constexpr int kWavesPerBlock = kRowWaves;

// ------------------------------------------------------------------------------------------------ rows of any length
template <typename T, bool Backward>
__global__ __launch_bounds__(kLongThreads) void layernorm_row_kernel(T* out, float* __restrict__ statistics /* [rows][mean, r] */,
                                                                     const T* __restrict__ dy, const T* residual, const T* x,
                                                                     const T* __restrict__ w, const T* __restrict__ bias, int rows,
                                                                     int hidden, float inv_hidden, float eps) {
    constexpr int VEC = kVec128<T>;
    using F = vec_t<float, VEC>;
    __shared__ float stage[kLongThreads / kWave];
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const std::size_t base = static_cast<std::size_t>(row) * hidden;
        float sum = 0.0f;
        walk_row(x + base, hidden, [&](int, int, const F& v) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += v[e];
        });
        const float mean = block_sum(sum, stage) * inv_hidden;
        float squares = 0.0f;
        walk_row(x + base, hidden, [&](int, int count, const F& v) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = e < count ? v[e] - mean : 0.0f;
                squares = fmaf(d, d, squares);
            }
        });
        const float r = 1.0f / sqrtf(block_sum(squares, stage) * inv_hidden + eps);
        if constexpr (Backward) {
            float g_sum = 0.0f, gx_sum = 0.0f;
            walk_row(x + base, hidden, [&](int col, int count, const F& v) {
                const F grad = vec_to_f32<T, VEC>(load_some<T>(dy + base + col, count)), weight = vec_to_f32<T, VEC>(load_some<T>(w + col, count));
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float g = grad[e] * weight[e];
                    g_sum += g;
                    gx_sum = fmaf(g, (v[e] - mean) * r, gx_sum);
                }
            });
            const float g_mean = block_sum(g_sum, stage) * inv_hidden;
            const float gx_mean = block_sum(gx_sum, stage) * inv_hidden;
            if (threadIdx.x == 0) {
                statistics[2 * static_cast<std::size_t>(row)] = mean;
                statistics[2 * static_cast<std::size_t>(row) + 1] = r;
            }
            walk_row(x + base, hidden, [&](int col, int count, const F& v) {
                const F grad = vec_to_f32<T, VEC>(load_some<T>(dy + base + col, count)), weight = vec_to_f32<T, VEC>(load_some<T>(w + col, count));
                F dx;
#pragma unroll
                for (int e = 0; e < VEC; ++e) dx[e] = r * (grad[e] * weight[e] - g_mean - (v[e] - mean) * r * gx_mean);
                if (residual != nullptr) dx += vec_to_f32<T, VEC>(load_some<T>(residual + base + col, count));
                store_some<T>(out + base + col, vec_from_f32<T, VEC>(dx), count);
            });
        } else {
            walk_row(x + base, hidden, [&](int col, int count, const F& v) {
                const F weight = vec_to_f32<T, VEC>(load_some<T>(w + col, count));
                F y = bias != nullptr ? vec_to_f32<T, VEC>(load_some<T>(bias + col, count)) : F(0.0f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) y[e] = fmaf((v[e] - mean) * r, weight[e], y[e]);
                store_some<T>(out + base + col, vec_from_f32<T, VEC>(y), count);
            });
        }
    }
}

// Partial sums [slices][hidden] of dw and, behind them, of db: a vector of columns per lane and a slice of the rows per workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void layernorm_column_kernel(float* __restrict__ partial, const T* __restrict__ dy,
                                                                    const T* __restrict__ x, const float* __restrict__ statistics,
                                                                    int rows, int hidden, int rows_per_slice) {
    constexpr int VEC = kVec128<T>;
    using F = vec_t<float, VEC>;
    __shared__ F stage[2][kWavesPerBlock][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int col = (blockIdx.x * kWave + lane) * VEC, count = hidden - col;
    const int row_begin = blockIdx.y * rows_per_slice, row_end = min(rows, row_begin + rows_per_slice);
    F dw(0.0f), db(0.0f);
    if (count > 0) {
        for (int row = row_begin + wave; row < row_end; row += kWavesPerBlock) {
            const std::size_t index = static_cast<std::size_t>(row) * hidden + col;
            const float mean = statistics[2 * static_cast<std::size_t>(row)], r = statistics[2 * static_cast<std::size_t>(row) + 1];
            const F g = vec_to_f32<T, VEC>(load_some<T>(dy + index, count)), v = vec_to_f32<T, VEC>(load_some<T>(x + index, count));
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                dw[e] = fmaf(g[e], (v[e] - mean) * r, dw[e]);
                db[e] += g[e];
            }
        }
    }
    stage[0][wave][lane] = dw;
    stage[1][wave][lane] = db;
    __syncthreads();
    if (wave < 2 && count > 0) {
        F total(0.0f);
#pragma unroll
        for (int s = 0; s < kWavesPerBlock; ++s) total += stage[wave][s][lane];
        float* to = partial + (static_cast<std::size_t>(wave) * gridDim.y + blockIdx.y) * hidden + col;
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
            store_some<float>(to + e, vec_t<float, 4>{total[e], total[e + 1], total[e + 2], total[e + 3]}, count - e);
    }
}

// ------------------------------------------------------------------------------------------------ rows in registers
// Makes the compiler forget what it has computed from a vector, so that it is computed again and not kept in registers.
template <bool FORGET, typename V>
__device__ __forceinline__ void forget(V& v) {
    if constexpr (FORGET) {
        auto words = __builtin_bit_cast(vec_t<unsigned int, 4>, v);
        asm volatile("" : "+v"(words));
        v = __builtin_bit_cast(V, words);
    }
}

// LPR lanes of a wavefront (WAVES = 1), or WAVES wavefronts, share a row; a lane holds K vectors of it.
template <typename T, int LPR, int WAVES, int K, bool Backward>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * kWave : kThreads) void layernorm_rows_kernel(
    T* out, float* __restrict__ partial /* [2][blocks][hidden]: dw, db */, const T* __restrict__ dy, const T* residual, const T* x,
    const T* __restrict__ w, const T* __restrict__ bias, int rows, int hidden, float inv_hidden, float eps) {
    constexpr int VEC = kVec128<T>;
    constexpr int kBlockWaves = WAVES > 4 ? WAVES : kWavesPerBlock;
    constexpr int kRowsPerWave = kWave / LPR;                                     // of WAVES = 1
    constexpr int kRowsPerBlock = WAVES > 1 ? kBlockWaves / WAVES : kBlockWaves * kRowsPerWave;
    static_assert(WAVES == 1 || kRowsPerBlock == 1, "the wavefronts of a row meet at the workgroup's barriers");
    using F = vec_t<float, VEC>;
    using V = vec_t<T, VEC>;
    // Sixteen wavefronts of a workgroup leave 128 registers: what a row's vectors give is computed again for every use.
    constexpr bool LEAN = WAVES > 4, AHEAD = !(Backward && LEAN && K * VEC > 8);  // AHEAD: the next row is requested before this one is used
    __shared__ float stage[4][WAVES];  // mean | variance | both means of the gradient
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int sub = WAVES > 1 ? static_cast<int>(threadIdx.x) : lane % LPR;
    const int slot = WAVES > 1 ? 0 : wave * kRowsPerWave + lane / LPR;  // which of the workgroup's rows

    int count[K];  // elements of the row that a lane's vectors hold
    V wv[K], bv[K];
    F acc_w[K], acc_b[K];
#pragma unroll
    for (int c = 0; c < K; ++c) {
        const int col = (c * LPR * WAVES + sub) * VEC;
        count[c] = hidden - col;
        wv[c] = load_some<T>(w + col, count[c]);
        acc_w[c] = acc_b[c] = F(0.0f);
        if constexpr (!Backward) bv[c] = bias != nullptr ? load_some<T>(bias + col, count[c]) : V(static_cast<T>(0.0f));
    }
    struct Row {
        V x[K], dy[K], residual[K];
    };
    auto fetch = [&](long row, Row& r) __attribute__((always_inline)) {
        const std::size_t base = static_cast<std::size_t>(row) * hidden;
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const int col = (c * LPR * WAVES + sub) * VEC, n = row < rows ? count[c] : 0;
            r.x[c] = load_some<T>(x + base + col, n);
            if constexpr (Backward) {
                r.dy[c] = load_some<T>(dy + base + col, n);
                if (residual != nullptr) r.residual[c] = load_some<T>(residual + base + col, n);
            }
        }
    };
    const long stride = static_cast<long>(gridDim.x) * kRowsPerBlock;
    Row now, next;
    fetch(static_cast<long>(blockIdx.x) * kRowsPerBlock + slot, now);
    for (long first = static_cast<long>(blockIdx.x) * kRowsPerBlock; first < rows; first += stride) {
        const long row = first + slot;
        if (AHEAD && first + stride < rows) fetch(row + stride, next);
        const std::size_t base = static_cast<std::size_t>(row) * hidden;
        float sum[1] = {0.0f}, squares[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F xv = vec_to_f32<T, VEC>(now.x[c]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[0] += xv[e];
            forget<LEAN>(now.x[c]);
        }
        row_sums<LPR, WAVES>(sum, stage);
        const float mean = sum[0] * inv_hidden;
        auto centred = [&](int c) __attribute__((always_inline)) {
            F xc = vec_to_f32<T, VEC>(now.x[c]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) xc[e] = e < count[c] ? xc[e] - mean : 0.0f;
            return xc;
        };
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F xc = centred(c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) squares[0] = fmaf(xc[e], xc[e], squares[0]);
            forget<LEAN>(now.x[c]);
        }
        row_sums<LPR, WAVES>(squares, stage + 1);
        const float r = 1.0f / sqrtf(squares[0] * inv_hidden + eps);
        if constexpr (Backward) {
            auto scaled = [&](int c) __attribute__((always_inline)) {
                F g = vec_to_f32<T, VEC>(now.dy[c]);
                const F weight = vec_to_f32<T, VEC>(wv[c]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] *= weight[e];
                return g;
            };
            float g_sums[2] = {0.0f, 0.0f};  // of g and of g xh
#pragma unroll
            for (int c = 0; c < K; ++c) {
                const F xc = centred(c), g = scaled(c), grad = vec_to_f32<T, VEC>(now.dy[c]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float xh = xc[e] * r;
                    acc_w[c][e] = fmaf(grad[e], xh, acc_w[c][e]);
                    acc_b[c][e] += grad[e];
                    g_sums[0] += g[e];
                    g_sums[1] = fmaf(g[e], xh, g_sums[1]);
                }
                forget<LEAN>(now.x[c]);
                forget<LEAN>(now.dy[c]);
            }
            row_sums<LPR, WAVES>(g_sums, stage + 2);
            const float g_mean = g_sums[0] * inv_hidden, gx_mean = g_sums[1] * inv_hidden;
#pragma unroll
            for (int c = 0; c < K; ++c) {
                const F xc = centred(c), g = scaled(c);
                F v;
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = r * (g[e] - g_mean - xc[e] * r * gx_mean);
                if (residual != nullptr) v += vec_to_f32<T, VEC>(now.residual[c]);
                if (row < rows) store_some<T>(out + base + (c * LPR * WAVES + sub) * VEC, vec_from_f32<T, VEC>(v), count[c]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < K; ++c) {
                const F xc = centred(c), weight = vec_to_f32<T, VEC>(wv[c]), shift = vec_to_f32<T, VEC>(bv[c]);
                F v;
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = fmaf(xc[e] * r, weight[e], shift[e]);
                if (row < rows) store_some<T>(out + base + (c * LPR * WAVES + sub) * VEC, vec_from_f32<T, VEC>(v), count[c]);
            }
        }
        if constexpr (AHEAD) now = next;
        else if (first + stride < rows) fetch(row + stride, now);
    }
    if constexpr (Backward) {
        float* const mine[2] = {partial + static_cast<std::size_t>(blockIdx.x) * hidden,
                                partial + (static_cast<std::size_t>(gridDim.x) + blockIdx.x) * hidden};
        if constexpr (WAVES > 1) {
#pragma unroll
            for (int c = 0; c < K; ++c) {
                const int col = (c * LPR * WAVES + sub) * VEC;
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    store_some<float>(mine[0] + col + e, vec_t<float, 4>{acc_w[c][e], acc_w[c][e + 1], acc_w[c][e + 2], acc_w[c][e + 3]}, count[c] - e);
                    store_some<float>(mine[1] + col + e, vec_t<float, 4>{acc_b[c][e], acc_b[c][e + 1], acc_b[c][e + 2], acc_b[c][e + 3]}, count[c] - e);
                }
            }
        } else {
            // The row slots of a wavefront, then the workgroup's wavefronts.
            __shared__ float fold[kBlockWaves][LPR * K * VEC];
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int c = 0; c < K; ++c)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        float v = which == 0 ? acc_w[c][e] : acc_b[c][e];
#pragma unroll
                        for (int offset = LPR; offset < kWave; offset <<= 1) v += __shfl_xor(v, offset, kWave);
                        if (lane < LPR) fold[wave][(c * LPR + sub) * VEC + e] = v;
                    }
                __syncthreads();
                for (int col = threadIdx.x; col < hidden; col += kThreads) {
                    float v = 0.0f;
#pragma unroll
                    for (int s = 0; s < kBlockWaves; ++s) v += fold[s][col];
                    mine[which][col] = v;
                }
            }
        }
    }
}

// dw and, of a second row of workgroups, db from the workgroups' partial sums.
template <typename T, int COLUMNS>
__global__ __launch_bounds__(kFinishThreads) void layernorm_finish_kernel(T* __restrict__ dw, T* __restrict__ db,
                                                                          const float* __restrict__ partial, int parts, int hidden, int units) {
    __shared__ float folded[kFolded], stage[4 * COLUMNS];
    column_partial_reduce_body<T, COLUMNS>(blockIdx.y == 0 ? dw : db, partial + blockIdx.y * static_cast<std::size_t>(parts) * hidden, parts,
                                           hidden, 0, static_cast<int>(blockIdx.x), units, folded, stage);
}

// Kernel for rows of `hidden` values; rows of a workgroup; threads of one.
template <typename T, bool Backward>
struct RowPlan {
    void (*kernel)(T*, float*, const T*, const T*, const T*, const T*, const T*, int, int, float, float) = nullptr;
    int rows_per_block = 0, threads = 0;

    template <int LPR, int WAVES, int K>
    void take() {
        kernel = layernorm_rows_kernel<T, LPR, WAVES, K, Backward>;
        rows_per_block = WAVES > 1 ? 1 : kWavesPerBlock * kWave / LPR;
        threads = WAVES > 4 ? WAVES * kWave : kThreads;
    }
    // Up to 32 values of a row in a lane where one wavefront has it, 16 where several do: the backward pass holds five of each.
    explicit RowPlan(int hidden) {
        const int vectors = (hidden + kVec128<T> - 1) / kVec128<T>;
        constexpr bool kHalf = sizeof(T) == 2;
        if (vectors <= 16) take<16, 1, 1>();
        else if (vectors <= 32) take<32, 1, 1>();
        else if (vectors <= 64) take<64, 1, 1>();
        else if (vectors <= 128) take<64, 1, 2>();
        else if (vectors <= 256) take<64, 1, 4>();
        else if (vectors <= 512) take<64, 4, 2>();
        else if (vectors <= 1024) take<64, kHalf ? 16 : 4, kHalf ? 1 : 4>();
        else if (vectors <= 2048) take<64, 16, 2>();
        else if (vectors <= 4096 && !kHalf) take<64, 16, kHalf ? 1 : 4>();
    }
    int blocks(int rows) const {
        const int wanted = (rows + rows_per_block - 1) / rows_per_block, resident = resident_blocks(reinterpret_cast<const void*>(kernel), threads);
        return wanted < resident ? wanted : resident;
    }
};

int validate(const char* name, std::size_t rows, std::size_t hidden, float eps, int dtype) {
    const std::string n(name);
    if (!valid_dtype(dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (!std::isfinite(eps) || eps <= 0.0f) return fail(CGPTX_INVALID_ARGUMENT, n + ": epsilon must be finite and positive");
    if (rows == 0 || hidden == 0) return fail(CGPTX_INVALID_ARGUMENT, n + ": empty shape");
    constexpr std::size_t limit = std::size_t{1} << 30;
    if (rows > limit || hidden > limit) return fail(CGPTX_INVALID_ARGUMENT, n + ": dimensions exceed supported range");
    return CGPTX_OK;
}

int row_blocks(int rows) { return rows < compute_units() * 2 ? rows : compute_units() * 2; }

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
        if (const RowPlan<T, false> plan(h); plan.kernel != nullptr) {
            hipLaunchKernelGGL(plan.kernel, dim3(plan.blocks(r)), dim3(plan.threads), 0, stream, static_cast<T*>(output), nullptr, nullptr,
                               nullptr, static_cast<const T*>(input), static_cast<const T*>(weight), static_cast<const T*>(bias), r, h,
                               1.0f / static_cast<float>(h), epsilon);
            CGPTX_LAUNCH_CHECK();
            return CGPTX_OK;
        }
        hipLaunchKernelGGL((layernorm_row_kernel<T, false>), dim3(row_blocks(r)), dim3(kLongThreads), 0, stream, static_cast<T*>(output),
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
        if (const RowPlan<T, true> plan(h); plan.kernel != nullptr) {
            const int blocks = plan.blocks(r);
            void* mem = nullptr;
            if (int s = scratch(stream, 2 * static_cast<std::size_t>(blocks) * hidden * sizeof(float), &mem)) return s;
            auto* partial = static_cast<float*>(mem);
            hipLaunchKernelGGL(plan.kernel, dim3(blocks), dim3(plan.threads), 0, stream, static_cast<T*>(grad_input), partial, dy,
                               static_cast<const T*>(residual), x, static_cast<const T*>(weight), nullptr, r, h, 1.0f / static_cast<float>(h),
                               epsilon);
            CGPTX_LAUNCH_CHECK();
            const int columns = finish_columns(h);
            auto finish = columns == 16 ? layernorm_finish_kernel<T, 16> : layernorm_finish_kernel<T, 32>;
            hipLaunchKernelGGL(finish, dim3((h + columns - 1) / columns, grad_bias != nullptr ? 2 : 1), dim3(kFinishThreads), 0, stream,
                               static_cast<T*>(grad_weight), static_cast<T*>(grad_bias), partial, blocks, h, compute_units());
            CGPTX_LAUNCH_CHECK();
            return CGPTX_OK;
        }
        const int slices = r < 256 ? 1 : (r < 65536 ? 64 : 256);
        const int rows_per_slice = (r + slices - 1) / slices;
        const std::size_t statistics_bytes = (2 * rows * sizeof(float) + 255) & ~std::size_t{255};
        void* mem = nullptr;
        if (int s = scratch(stream, statistics_bytes + 2 * static_cast<std::size_t>(slices) * hidden * sizeof(float), &mem)) return s;
        auto* statistics = static_cast<float*>(mem);
        auto* partial = reinterpret_cast<float*>(static_cast<char*>(mem) + statistics_bytes);
        hipLaunchKernelGGL((layernorm_row_kernel<T, true>), dim3(row_blocks(r)), dim3(kLongThreads), 0, stream, static_cast<T*>(grad_input),
                           statistics, dy, static_cast<const T*>(residual), x, static_cast<const T*>(weight), nullptr, r, h,
                           1.0f / static_cast<float>(h), epsilon);
        CGPTX_LAUNCH_CHECK();
        hipLaunchKernelGGL((layernorm_column_kernel<T>), dim3((h + kWave * kVec128<T> - 1) / (kWave * kVec128<T>), slices), dim3(kThreads), 0, stream, partial, dy,
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
