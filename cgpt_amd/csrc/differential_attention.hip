// Differential attention for gfx950: causal grouped-query attention whose map is the difference of two softmax maps (T. Ye and
// others, "Differential Transformer", 2024), forward and backward, and the learned weights of the second maps.
//
// A head of width D has two maps of width D/2: q = [q1 | q2], k = [k1 | k2], v of width D, a weight lambda per query head:
//   P1 = softmax(s q1 k1'), P2 = softmax(s q2 k2'),  O = P1 v - lambda P2 v        (s = 1/sqrt(D/2) unless given)
// The forward pass leaves the logarithms of both maps' sums and, beside O, the second map's own output O2 = P2 v. With G = dO v',
// delta1 = rowsum(P1 G) = dO.(O + lambda O2) and delta2 = rowsum(P2 G) = dO.O2 the gradients are
//   dS1 = P1 (G - delta1), dS2 = -lambda P2 (G - delta2),  dq_i = s dS_i k_i, dk_i = s dS_i' q_i,
//   dv = (P1 - lambda P2)' dO,  dlambda = -sum over the head's rows of delta2.
// G and the product with dO are shared by the maps: a backward pass multiplies as much as one of plain attention with heads of D,
// where two calls with heads of D/2 and values of D would multiply two thirds more.
// dlambda cancels over rows and keys, and it is fp32: the dQ pass corrects the delta2 that it takes from the rounded O2 by
// rowsum(dS2), which is what that rounding left (the rows of P2 sum to one).
//
// This file holds the entries and the kernels that take every call: head widths that are not multiples of 16 (fp32: of 8), tensors off
// 16-byte boundaries (differential_attention_mfma.hip and differential_attention_f32.hip have the others). One wavefront per output
// row, fp32 arithmetic, lane l holding elements l and l + 64 of the head. No atomics: every row has one owner that adds its terms in
// a fixed order. What bounds them is the reduction over the lanes for every score: 32 x 1024 tokens of 8:2 heads of 128, bf16, take
// 21 ms forward and 46 backward where the matrix kernels take 0.16 and 0.36.
#include "differential_attention.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace cgptx {
namespace {

constexpr int kScalarWaves = kThreads / kWave;

using Params = DifferentialArgs;

template <typename T>
struct RowPair {
    float a, b;  // elements lane and lane + 64 of a row (0 past the end)
    __device__ __forceinline__ static RowPair load(const T* row, int d) {
        const int lane = threadIdx.x & (kWave - 1);
        return {lane < d ? to_f32(row[lane]) : 0.0f, lane + kWave < d ? to_f32(row[lane + kWave]) : 0.0f};
    }
    __device__ __forceinline__ void store(T* row, int d, bool accumulate) const {
        const int lane = threadIdx.x & (kWave - 1);
        if (lane < d) row[lane] = from_f32<T>(accumulate ? a + to_f32(row[lane]) : a);
        if (lane + kWave < d) row[lane + kWave] = from_f32<T>(accumulate ? b + to_f32(row[lane + kWave]) : b);
    }
};
template <typename T>
__device__ __forceinline__ float row_dot(const RowPair<T>& x, const RowPair<T>& y) {
    return wave_sum(fmaf(x.a, y.a, x.b * y.b));
}
// The scores of both maps: products of the elements below and from `half` on.
template <typename T>
__device__ __forceinline__ vec_t<float, 2> row_scores(const RowPair<T>& x, const RowPair<T>& y, int half) {
    const int lane = threadIdx.x & (kWave - 1);
    const float a = x.a * y.a, b = x.b * y.b;
    return {wave_sum((lane < half ? a : 0.0f) + (lane + kWave < half ? b : 0.0f)),
            wave_sum((lane < half ? 0.0f : a) + (lane + kWave < half ? 0.0f : b))};
}
// By the map that a lane's elements belong to.
template <typename T>
__device__ __forceinline__ RowPair<T> of_maps(float first, float second, int half) {
    const int lane = threadIdx.x & (kWave - 1);
    return {lane < half ? first : second, lane + kWave < half ? first : second};
}

// A wavefront's row. The workgroups fill a second axis of the grid where there are more than a launch has along one.
__device__ __forceinline__ long scalar_row() {
    return (blockIdx.x + static_cast<long>(gridDim.x) * blockIdx.y) * kScalarWaves + threadIdx.x / kWave;
}

struct QueryRow {
    int b, q, h, kvh;
    __device__ __forceinline__ QueryRow(long row, const Params& p) {
        h = static_cast<int>(row % p.hq);
        q = static_cast<int>((row / p.hq) % p.qs);
        b = static_cast<int>(row / (static_cast<long>(p.hq) * p.qs));
        kvh = h / (p.hq / p.hkv);
    }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void differential_forward_scalar_kernel(Params p) {
    const long row = scalar_row();
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq;
    if (row >= rows) return;
    const QueryRow at(row, p);
    const int half = p.d / 2;
    const RowPair<T> q = RowPair<T>::load(static_cast<const T*>(p.q) + row * p.d, p.d);
    const long base = (static_cast<long>(at.b) * p.ks * p.hkv + at.kvh) * p.d, stride = static_cast<long>(p.hkv) * p.d;
    const T *k = static_cast<const T*>(p.k) + base, *v = static_cast<const T*>(p.v) + base;
    const int end = p.causal ? min(p.ks, p.offset + at.q + 1) : p.ks;
    // The maxima start at the least finite number: behind keys whose scores are -Inf there is still something to subtract from one.
    constexpr float kLeast = -3.402823466e38f;
    float m[2] = {kLeast, kLeast}, l[2] = {0.0f, 0.0f};
    RowPair<T> o[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    for (int j = 0; j < end; ++j) {
        const vec_t<float, 2> s = row_scores(q, RowPair<T>::load(k + j * stride, p.d), half);
        const RowPair<T> vr = RowPair<T>::load(v + j * stride, p.d);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float score = s[i] * p.scale, top = fmaxf(m[i], score);
            const float alpha = expf(m[i] - top), e = expf(score - top);
            l[i] = l[i] * alpha + e;
            o[i].a = fmaf(e, vr.a, o[i].a * alpha);
            o[i].b = fmaf(e, vr.b, o[i].b * alpha);
            m[i] = top;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float inverse = 1.0f / l[i];
        o[i].a *= inverse;
        o[i].b *= inverse;
        if (p.lse_out != nullptr && (threadIdx.x & (kWave - 1)) == 0) p.lse_out[i * rows + row] = m[i] + logf(l[i]);
    }
    if (p.second != nullptr) o[1].store(static_cast<T*>(p.second) + row * p.d, p.d, false);
    const float lambda = p.lambda[at.h];
    RowPair<T>{fmaf(-lambda, o[1].a, o[0].a), fmaf(-lambda, o[1].b, o[0].b)}.store(static_cast<T*>(p.out) + row * p.d, p.d, false);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void differential_dq_scalar_kernel(Params p) {
    const long row = scalar_row();
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq;
    if (row >= rows) return;
    const QueryRow at(row, p);
    const int half = p.d / 2;
    const float lambda = p.lambda[at.h];
    const RowPair<T> q = RowPair<T>::load(static_cast<const T*>(p.q) + row * p.d, p.d);
    const RowPair<T> dout = RowPair<T>::load(static_cast<const T*>(p.dout) + row * p.d, p.d);
    const float delta2 = row_dot(dout, RowPair<T>::load(static_cast<const T*>(p.o2) + row * p.d, p.d));
    const float delta1 = fmaf(lambda, delta2, row_dot(dout, RowPair<T>::load(static_cast<const T*>(p.o) + row * p.d, p.d)));
    const float lse1 = p.lse[row], lse2 = p.lse[rows + row];
    const long base = (static_cast<long>(at.b) * p.ks * p.hkv + at.kvh) * p.d, stride = static_cast<long>(p.hkv) * p.d;
    const T *k = static_cast<const T*>(p.k) + base, *v = static_cast<const T*>(p.v) + base;
    const int end = p.causal ? min(p.ks, p.offset + at.q + 1) : p.ks;
    RowPair<T> dq{0.0f, 0.0f};
    float rest = 0.0f;  // rowsum(P2 (G - delta2))
    for (int j = 0; j < end; ++j) {
        const RowPair<T> kr = RowPair<T>::load(k + j * stride, p.d);
        const vec_t<float, 2> s = row_scores(q, kr, half);
        const float g = row_dot(dout, RowPair<T>::load(v + j * stride, p.d));
        const float ds1 = expf(s[0] * p.scale - lse1) * (g - delta1), ds2 = expf(s[1] * p.scale - lse2) * (g - delta2);
        rest += ds2;
        const RowPair<T> ds = of_maps<T>(ds1, -lambda * ds2, half);
        dq.a = fmaf(ds.a, kr.a, dq.a);
        dq.b = fmaf(ds.b, kr.b, dq.b);
    }
    dq.a *= p.gradient_scale;
    dq.b *= p.gradient_scale;
    dq.store(static_cast<T*>(p.dq) + row * p.d, p.d, p.accumulate != 0);
    if ((threadIdx.x & (kWave - 1)) == 0) {
        p.delta[row] = delta1;
        p.delta[rows + row] = delta2;
        p.lambda_partial[(static_cast<long>(at.h) * p.batch + at.b) * p.qs + at.q] = -(delta2 + rest);
    }
}

// dK and dV of one (batch, key, kv-head) row per wavefront: the heads of the group in ascending order, each over the queries that
// see the key in ascending order.
template <typename T>
__global__ __launch_bounds__(kThreads) void differential_dkv_scalar_kernel(Params p) {
    __shared__ double stage[kScalarWaves];
    add_lambda_parts<kThreads>(p, stage);
    const long row = scalar_row();
    if (row >= static_cast<long>(p.batch) * p.ks * p.hkv) return;
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq;
    const int kvh = static_cast<int>(row % p.hkv), j = static_cast<int>((row / p.hkv) % p.ks);
    const int b = static_cast<int>(row / (static_cast<long>(p.hkv) * p.ks));
    const int half = p.d / 2, group = p.hq / p.hkv;
    const RowPair<T> k = RowPair<T>::load(static_cast<const T*>(p.k) + row * p.d, p.d);
    const RowPair<T> v = RowPair<T>::load(static_cast<const T*>(p.v) + row * p.d, p.d);
    RowPair<T> dk{0.0f, 0.0f}, dv{0.0f, 0.0f};
    for (int g = 0; g < group; ++g) {
        const int h = kvh * group + g;
        const float lambda = p.lambda[h];
        for (int query = p.causal ? max(0, j - p.offset) : 0; query < p.qs; ++query) {
            const long at = (static_cast<long>(b) * p.qs + query) * p.hq + h;
            const RowPair<T> q = RowPair<T>::load(static_cast<const T*>(p.q) + at * p.d, p.d);
            const RowPair<T> dout = RowPair<T>::load(static_cast<const T*>(p.dout) + at * p.d, p.d);
            const vec_t<float, 2> s = row_scores(q, k, half);
            const float grad = row_dot(dout, v);
            const float p1 = expf(s[0] * p.scale - p.lse[at]), p2 = expf(s[1] * p.scale - p.lse[rows + at]);
            const float map = fmaf(-lambda, p2, p1);
            const RowPair<T> ds = of_maps<T>(p1 * (grad - p.delta[at]), -lambda * (p2 * (grad - p.delta[rows + at])), half);
            dv.a = fmaf(map, dout.a, dv.a);
            dv.b = fmaf(map, dout.b, dv.b);
            dk.a = fmaf(ds.a, q.a, dk.a);
            dk.b = fmaf(ds.b, q.b, dk.b);
        }
    }
    dk.a *= p.gradient_scale;
    dk.b *= p.gradient_scale;
    dk.store(static_cast<T*>(p.dk) + row * p.d, p.d, p.accumulate != 0);
    dv.store(static_cast<T*>(p.dv) + row * p.d, p.d, p.accumulate != 0);
}

// ------------------------------------------------------------------------------------------------ lambda
// lambda of a head = exp(q1.k1) - exp(q2.k2) + initial, from vectors of its own or one set for all heads; a wavefront per set.
// What bounds it is the launch: 8 sets of 64 in fp32 take 2.2 us forward and 2.7 backward.
struct LambdaVectors {
    const void* vector[4];  // q1, k1, q2, k2: [sets, width]
};
template <typename T>
__device__ __forceinline__ vec_t<float, 2> lambda_terms(const LambdaVectors& in, long set, int width) {
    const T *q1 = static_cast<const T*>(in.vector[0]) + set * width, *k1 = static_cast<const T*>(in.vector[1]) + set * width;
    const T *q2 = static_cast<const T*>(in.vector[2]) + set * width, *k2 = static_cast<const T*>(in.vector[3]) + set * width;
    float first = 0.0f, second = 0.0f;
    for (int i = threadIdx.x & (kWave - 1); i < width; i += kWave) {
        first = fmaf(to_f32(q1[i]), to_f32(k1[i]), first);
        second = fmaf(to_f32(q2[i]), to_f32(k2[i]), second);
    }
    return {expf(wave_sum(first)), expf(wave_sum(second))};
}
template <typename T>
__global__ __launch_bounds__(kWave) void lambda_forward_kernel(float* lambda, LambdaVectors in, int sets, int heads, int width,
                                                               float initial) {
    const vec_t<float, 2> e = lambda_terms<T>(in, blockIdx.x, width);
    const float value = e[0] - e[1] + initial;
    if (sets > 1) {
        if (threadIdx.x == 0) lambda[blockIdx.x] = value;
    } else {
        for (int h = threadIdx.x; h < heads; h += kWave) lambda[h] = value;
    }
}
struct LambdaGradients {
    void* vector[4];
};
template <typename T>
__global__ __launch_bounds__(kWave) void lambda_backward_kernel(LambdaGradients out, const float* __restrict__ dlambda, LambdaVectors in,
                                                                int sets, int heads, int width) {
    const vec_t<float, 2> e = lambda_terms<T>(in, blockIdx.x, width);
    float grad = 0.0f;
    if (sets > 1) {
        grad = dlambda[blockIdx.x];
    } else {
        for (int h = threadIdx.x; h < heads; h += kWave) grad += dlambda[h];
        grad = wave_sum(grad);
    }
    const float first = grad * e[0], second = -grad * e[1];
    const long base = static_cast<long>(blockIdx.x) * width;
    for (int i = threadIdx.x; i < width; i += kWave) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
            static_cast<T*>(out.vector[n])[base + i] =
                from_f32<T>((n < 2 ? first : second) * to_f32(static_cast<const T*>(in.vector[n ^ 1])[base + i]));
    }
}

// ------------------------------------------------------------------------------------------------ host
struct Shape {
    std::size_t batch, qs, ks, hq, hkv, d;
    float scale;
    int causal;
    std::size_t offset;
    int dtype;
};

int validate(const char* name, const Shape& s) {
    const std::string n(name);
    if (!valid_dtype(s.dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (s.batch == 0 || s.qs == 0 || s.ks == 0 || s.hq == 0 || s.hkv == 0 || s.d == 0 || s.hq % s.hkv != 0)
        return fail(CGPTX_INVALID_ARGUMENT, n + ": invalid tensors or options");
    if (!std::isfinite(s.scale)) return fail(CGPTX_INVALID_ARGUMENT, n + ": attention scale must be finite");
    if (s.causal && (s.offset > s.ks || s.qs > s.ks - s.offset))
        return fail(CGPTX_INVALID_ARGUMENT, n + ": causal range exceeds the key sequence");
    if (s.d % 2 != 0 || s.d > 128) return fail(CGPTX_INVALID_ARGUMENT, n + ": head_dim must be even and not exceed 128");
    constexpr std::size_t limit = 1u << 30;
    if (s.batch > 65535 || s.qs > limit || s.ks > limit || s.hq > 65535 || (s.causal && s.offset > limit) || s.hq * s.d > limit)
        return fail(CGPTX_OVERFLOW, n + ": dimension exceeds the supported range");
    const std::size_t rows = std::max(s.batch * s.qs * s.hq, s.batch * s.ks * s.hkv);
    if (rows / kScalarWaves >= (std::size_t{1} << 31)) return fail(CGPTX_OVERFLOW, n + ": too many rows");
    return CGPTX_OK;
}

Params make_params(const Shape& s, const void* q, const void* k, const void* v, const float* lambda) {
    Params p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.lambda = lambda;
    p.batch = static_cast<int>(s.batch);
    p.qs = static_cast<int>(s.qs);
    p.ks = static_cast<int>(s.ks);
    p.hq = static_cast<int>(s.hq);
    p.hkv = static_cast<int>(s.hkv);
    p.d = static_cast<int>(s.d);
    p.scale = s.scale > 0.0f ? s.scale : 1.0f / std::sqrt(static_cast<float>(s.d / 2));
    p.gradient_scale = s.ks > 1 ? p.scale : 0.0f;
    p.causal = s.causal ? 1 : 0;
    p.offset = s.causal ? static_cast<int>(s.offset) : 0;
    p.dtype = s.dtype;
    return p;
}

dim3 scalar_grid(std::size_t rows) {
    const std::size_t blocks = (rows + kScalarWaves - 1) / kScalarWaves, axis = std::min(blocks, kLaunchThreads / kThreads);
    return dim3(static_cast<unsigned int>(axis), static_cast<unsigned int>((blocks + axis - 1) / axis));
}

bool aligned(std::initializer_list<const void*> tensors) {
    for (const void* t : tensors)
        if (!is_aligned16(t)) return false;  // an absent one is
    return true;
}

int validate_lambda(const char* name, std::size_t sets, std::size_t heads, std::size_t width, int dtype) {
    const std::string n(name);
    if (!valid_dtype(dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (heads == 0 || width == 0 || (sets != 1 && sets != heads))
        return fail(CGPTX_INVALID_ARGUMENT, n + ": vectors must be one set for all heads or one for each");
    constexpr std::size_t limit = std::size_t{1} << 30;
    if (heads > 65535 || width > limit) return fail(CGPTX_OVERFLOW, n + ": dimension exceeds the supported range");
    return CGPTX_OK;
}

}  // namespace

KeyWalk key_walk(const DifferentialArgs& a) {
    KeyWalk walk{};
    walk.batch = a.batch;
    walk.qs = a.qs;
    walk.ks = a.ks;
    walk.hkv = a.hkv;
    walk.group = a.hq / a.hkv;
    walk.d = a.d;
    walk.causal = a.causal;
    walk.offset = a.offset;
    return walk;
}

int launchable_parts(const KeyWalk& walk, int threads) {
    const long key_blocks = (walk.ks + walk.block_rows - 1) / walk.block_rows;
    return static_cast<int>(std::min<long>(key_block_parts(walk), std::max<long>(static_cast<long>(kLaunchThreads) / threads / key_blocks, 1)));
}

int differential_backward_scratch(DifferentialArgs& a, int statistics, long lambda_parts, int splits, hipStream_t stream) {
    auto rounded = [](std::size_t bytes) { return (bytes + 255) & ~std::size_t{255}; };
    const std::size_t first = rounded(static_cast<std::size_t>(statistics) * a.batch * a.qs * a.hq * sizeof(float));
    const std::size_t by_row_block = rounded(static_cast<std::size_t>(lambda_parts) * a.hq * sizeof(float)), fixed = first + 2 * by_row_block;
    const std::size_t part = 2 * static_cast<std::size_t>(a.batch) * a.ks * a.hkv * a.d * sizeof(float);
    a.lambda_parts = lambda_parts;
    a.splits = splits;
    auto wanted = [&] { return fixed + (a.splits > 1 ? a.splits * part : 0); };
    void* memory = nullptr;
    std::size_t held = 0;
    if (int st = scratch_up_to(stream, wanted(), &memory, &held)) return st;
    while (a.splits > 1 && held < wanted()) --a.splits;
    if (int st = scratch(stream, wanted(), &memory)) return st;
    a.delta = static_cast<float*>(memory);
    a.lambda_partial = reinterpret_cast<float*>(static_cast<char*>(memory) + first);
    a.largest = reinterpret_cast<float*>(static_cast<char*>(memory) + first + by_row_block);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(memory) + fixed);
    return CGPTX_OK;
}

}  // namespace cgptx

extern "C" int cgptx_differential_lambda_forward(float* lambda, const void* query1, const void* key1, const void* query2,
                                                 const void* key2, float initial, size_t sets, size_t heads, size_t width, int dtype,
                                                 cgptx_stream stream) {
    using namespace cgptx;
    const char* name = "differential_lambda_forward";
    if (int st = validate_lambda(name, sets, heads, width, dtype)) return st;
    if (!std::isfinite(initial)) return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": the initial value must be finite");
    const LambdaVectors in{{query1, key1, query2, key2}};
    for (const void* v : in.vector)
        if (v == nullptr) return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    if (lambda == nullptr) return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        hipLaunchKernelGGL((lambda_forward_kernel<T>), dim3(static_cast<unsigned int>(sets)), dim3(kWave), 0,
                           static_cast<hipStream_t>(stream), lambda, in, static_cast<int>(sets), static_cast<int>(heads),
                           static_cast<int>(width), initial);
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}

extern "C" int cgptx_differential_lambda_backward(void* grad_query1, void* grad_key1, void* grad_query2, void* grad_key2,
                                                  const float* grad_lambda, const void* query1, const void* key1, const void* query2,
                                                  const void* key2, size_t sets, size_t heads, size_t width, int dtype,
                                                  cgptx_stream stream) {
    using namespace cgptx;
    const char* name = "differential_lambda_backward";
    if (int st = validate_lambda(name, sets, heads, width, dtype)) return st;
    const LambdaVectors in{{query1, key1, query2, key2}};
    const LambdaGradients out{{grad_query1, grad_key1, grad_query2, grad_key2}};
    for (int n = 0; n < 4; ++n)
        if (in.vector[n] == nullptr || out.vector[n] == nullptr || grad_lambda == nullptr)
            return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        hipLaunchKernelGGL((lambda_backward_kernel<T>), dim3(static_cast<unsigned int>(sets)), dim3(kWave), 0,
                           static_cast<hipStream_t>(stream), out, grad_lambda, in, static_cast<int>(sets), static_cast<int>(heads),
                           static_cast<int>(width));
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}

extern "C" int cgptx_differential_attention_forward(void* output, void* second, float* logsumexp, const void* query, const void* key,
                                                    const void* value, const float* lambda, size_t batch, size_t query_sequence,
                                                    size_t kv_sequence, size_t query_heads, size_t kv_heads, size_t head_dim,
                                                    float attention_scale, int causal, size_t query_position_offset, int dtype,
                                                    cgptx_stream stream) {
    using namespace cgptx;
    const char* name = "differential_attention_forward";
    const Shape s{batch, query_sequence, kv_sequence, query_heads, kv_heads, head_dim, attention_scale, causal, query_position_offset,
                  dtype};
    if (int st = validate(name, s)) return st;
    if (output == nullptr || query == nullptr || key == nullptr || value == nullptr || lambda == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    Params p = make_params(s, query, key, value, lambda);
    p.out = output;
    p.second = second;
    p.lse_out = logsumexp;
    if (aligned({output, second, query, key, value})) {
        if (differential_mfma_takes(p)) return differential_mfma_forward(p, static_cast<hipStream_t>(stream));
        if (differential_f32_takes(p)) return differential_f32_forward(p, static_cast<hipStream_t>(stream));
    }
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        hipLaunchKernelGGL((differential_forward_scalar_kernel<T>), scalar_grid(batch * query_sequence * query_heads), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), p);
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}

extern "C" int cgptx_differential_attention_backward(void* grad_query, void* grad_key, void* grad_value, float* grad_lambda,
                                                     const void* grad_output, const void* output, const void* second,
                                                     const float* logsumexp, const void* query, const void* key, const void* value,
                                                     const float* lambda, size_t batch, size_t query_sequence, size_t kv_sequence,
                                                     size_t query_heads, size_t kv_heads, size_t head_dim, float attention_scale,
                                                     int causal, size_t query_position_offset, int accumulate_grads, int dtype,
                                                     cgptx_stream stream_) {
    using namespace cgptx;
    const char* name = "differential_attention_backward";
    const Shape s{batch, query_sequence, kv_sequence, query_heads, kv_heads, head_dim, attention_scale, causal, query_position_offset,
                  dtype};
    if (int st = validate(name, s)) return st;
    if (grad_query == nullptr || grad_key == nullptr || grad_value == nullptr || grad_lambda == nullptr || grad_output == nullptr ||
        output == nullptr || second == nullptr || logsumexp == nullptr || query == nullptr || key == nullptr || value == nullptr ||
        lambda == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    auto stream = static_cast<hipStream_t>(stream_);
    Params p = make_params(s, query, key, value, lambda);
    p.dout = grad_output;
    p.o = output;
    p.o2 = second;
    p.lse = logsumexp;
    p.dq = grad_query;
    p.dk = grad_key;
    p.dv = grad_value;
    p.dlambda = grad_lambda;
    p.accumulate = accumulate_grads != 0;
    if (aligned({grad_query, grad_key, grad_value, grad_output, output, second, query, key, value})) {
        if (differential_mfma_takes(p)) return differential_mfma_backward(p, stream);
        if (differential_f32_takes(p)) return differential_f32_backward(p, stream);
    }
    const std::size_t rows = batch * query_sequence * query_heads;
    const long lambda_parts = static_cast<long>(batch * query_sequence);
    if (int st = differential_backward_scratch(p, 2, lambda_parts, 1, stream)) return st;
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        hipLaunchKernelGGL((differential_dq_scalar_kernel<T>), scalar_grid(rows), dim3(kThreads), 0, stream, p);
        CGPTX_LAUNCH_CHECK();
        hipLaunchKernelGGL((differential_dkv_scalar_kernel<T>), scalar_grid(batch * kv_sequence * kv_heads), dim3(kThreads), 0,
                           stream, p);
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}
