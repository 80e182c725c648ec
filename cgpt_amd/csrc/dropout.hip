// Dropout with a mask that is never stored, forward (onto a residual stream) and backward, for gfx950.
//
// The mask comes from a counter-based generator: Philox 4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011). Its key is the seed; the value n of its counter gives four words
// of 32 bits, eight numbers of 16 bits (low half first), one for each of the elements 8 (n - offset) .. + 7. An element is
// kept where its number is not below round(65536 p), and is multiplied by the inverse of the share kept. So a mask is a
// function of (seed, offset, element) alone, whatever the type, the alignment and the launch, and the backward pass makes it
// again. 16 bits: the probability is a multiple of 2^-16, at half of the generator's work per element of 32.
//
// A thread takes the eight elements of a counter value. What bounds it is memory: the generator's ten rounds run while the values
// are on their way. 33554432 bf16 values, forward onto a residual and backward (335 MB): 56 us, 6.0 TB/s. A thread to
// every eight elements instead of a few to each takes 225 us for 134217728 of them where 16 workgroups a CU in a loop took 257.
#include "common.hpp"

namespace cgptx {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;  // elements of a counter value

struct DropoutArgs {
    unsigned int threshold;  // of 65536: numbers below it drop their element
    float scale;             // of what is kept
    std::uint64_t seed, offset;
    const std::uint64_t* counter;  // added to the offset, or null
    std::size_t count;
};

__device__ __forceinline__ vec_t<std::uint32_t, 4> philox(std::uint64_t counter, std::uint64_t seed) {
    std::uint32_t c0 = static_cast<std::uint32_t>(counter), c1 = static_cast<std::uint32_t>(counter >> 32), c2 = 0, c3 = 0;
    std::uint32_t k0 = static_cast<std::uint32_t>(seed), k1 = static_cast<std::uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const std::uint64_t a = static_cast<std::uint64_t>(0xD2511F53u) * c0, b = static_cast<std::uint64_t>(0xCD9E8D57u) * c2;
        c0 = static_cast<std::uint32_t>(b >> 32) ^ c1 ^ k0;
        c2 = static_cast<std::uint32_t>(a >> 32) ^ c3 ^ k1;
        c1 = static_cast<std::uint32_t>(b);
        c3 = static_cast<std::uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {c0, c1, c2, c3};
}

// Eight elements on a 16-byte boundary.
template <bool ONCE, typename T>
__device__ __forceinline__ vec_t<T, kGroup> load_group(const T* p) {
    if constexpr (sizeof(T) == 2) {
        return load_vec_once<ONCE, T, kGroup>(p);
    } else {
        const vec_t<T, 4> a = load_vec_once<ONCE, T, 4>(p), b = load_vec_once<ONCE, T, 4>(p + 4);
        return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
}
template <bool ONCE, typename T>
__device__ __forceinline__ void store_group(T* p, vec_t<T, kGroup> v) {
    if constexpr (sizeof(T) == 2) {
        store_vec_once<ONCE, T, kGroup>(p, v);
    } else {
        store_vec_once<ONCE, T, 4>(p, vec_t<T, 4>{v[0], v[1], v[2], v[3]});
        store_vec_once<ONCE, T, 4>(p + 4, vec_t<T, 4>{v[4], v[5], v[6], v[7]});
    }
}

// output = dropout(input) + added, rounded once; `added` (or null) and input may be the output.
template <typename T, bool ONCE>
__global__ __launch_bounds__(kThreads) void dropout_kernel(T* output, const T* input, const T* added, DropoutArgs args, bool vector_ok) {
    using Values = vec_t<T, kGroup>;
    const std::uint64_t first = args.offset + (args.counter != nullptr ? *args.counter : 0);
    const std::size_t groups = (args.count + kGroup - 1) / kGroup;
    for (std::size_t g = static_cast<std::size_t>(blockIdx.x) * kThreads + threadIdx.x; g < groups;
         g += static_cast<std::size_t>(gridDim.x) * kThreads) {
        const std::size_t at = g * kGroup;
        const bool whole = vector_ok && at + kGroup <= args.count;
        Values x, y;
        if (whole) {
            x = load_group<ONCE, T>(input + at);
            if (added != nullptr) y = load_group<ONCE, T>(added + at);
        } else {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) {
                const bool live = at + e < args.count;
                x[e] = live ? input[at + e] : static_cast<T>(0.0f);
                y[e] = live && added != nullptr ? added[at + e] : static_cast<T>(0.0f);
            }
        }
        const vec_t<std::uint32_t, 4> words = philox(first + g, args.seed);
        Values out;
#pragma unroll
        for (int e = 0; e < kGroup; ++e) {
            const unsigned int number = e % 2 == 0 ? words[e / 2] & 0xFFFFu : words[e / 2] >> 16;
            // Not a product with zero: what is dropped is zero whatever stood there.
            const float beside = added != nullptr ? to_f32(static_cast<T>(y[e])) : 0.0f;
            out[e] = from_f32<T>(number >= args.threshold ? fmaf(to_f32(static_cast<T>(x[e])), args.scale, beside) : beside);
        }
        if (whole) {
            store_group<ONCE, T>(output + at, out);
        } else {
#pragma unroll
            for (int e = 0; e < kGroup; ++e)
                if (at + e < args.count) output[at + e] = out[e];
        }
    }
}

int launch(const char* name, void* output, const void* input, const void* added, std::size_t count, float probability,
           std::uint64_t seed, std::uint64_t offset, const std::uint64_t* counter, int dtype, cgptx_stream stream) {
    const std::string n(name);
    if (!valid_dtype(dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (!(probability >= 0.0f && probability <= 1.0f))
        return fail(CGPTX_INVALID_ARGUMENT, n + ": the probability must be between 0 and 1");
    if (reinterpret_cast<std::uintptr_t>(counter) % sizeof(std::uint64_t) != 0)
        return fail(CGPTX_INVALID_ARGUMENT, n + ": the counter must be aligned to 8 bytes");
    if (count == 0) return CGPTX_OK;
    if (output == nullptr || input == nullptr) return fail(CGPTX_INVALID_ARGUMENT, n + ": null tensor");
    DropoutArgs args{};
    args.threshold = static_cast<unsigned int>(static_cast<double>(probability) * 65536.0 + 0.5);
    args.scale = args.threshold == 65536u ? 0.0f : 65536.0f / static_cast<float>(65536u - args.threshold);
    args.seed = seed;
    args.offset = offset;
    args.counter = counter;
    args.count = count;
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        const std::size_t blocks = ((count + kGroup - 1) / kGroup + kThreads - 1) / kThreads;
        const std::size_t cap = kLaunchThreads / kThreads;
        const bool vector_ok = is_aligned16(output) && is_aligned16(input) && is_aligned16(added);
        // A call that moves more than half of what the memory-side cache holds leaves it to its neighbours: the pair of calls above
        // 62.7 -> 55.9 us; of two calls that move half of it each (without the residual) 42.7 us, 46.8 if they did.
        const bool once = count * sizeof(T) * (added != nullptr && added != output ? 3 : 2) > kMemoryCacheBytes / 2;
        auto kernel = once ? dropout_kernel<T, true> : dropout_kernel<T, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned int>(blocks < cap ? blocks : cap)), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), static_cast<T*>(output), static_cast<const T*>(input),
                           static_cast<const T*>(added), args, vector_ok);
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}

}  // namespace
}  // namespace cgptx

extern "C" int cgptx_dropout_forward(void* output, const void* input, const void* residual, size_t count, float probability,
                                     uint64_t seed, uint64_t offset, const uint64_t* counter, int dtype, cgptx_stream stream) {
    return cgptx::launch("dropout_forward", output, input, residual, count, probability, seed, offset, counter, dtype, stream);
}

extern "C" int cgptx_dropout_backward(void* grad_input, const void* grad_output, size_t count, float probability, uint64_t seed,
                                      uint64_t offset, const uint64_t* counter, int accumulate, int dtype, cgptx_stream stream) {
    return cgptx::launch("dropout_backward", grad_input, grad_output, accumulate ? grad_input : nullptr, count, probability, seed, offset,
                         counter, dtype, stream);
}
