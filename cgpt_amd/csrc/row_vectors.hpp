// What the norms that keep rows in registers share: rows in vectors of 16 bytes at any address, sums over a row's lanes or wavefronts, and
// walks of a workgroup over rows that are longer.
#pragma once

#include "common.hpp"

namespace cgptx {

constexpr int kRowThreads = 256;
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kLongThreads = 1024;  // of the kernels for rows of any length

// Sum over kLongThreads, the same bits in every thread. `stage` may be used again behind the next call's first barrier.
__device__ __forceinline__ float block_sum(float v, float* stage) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) stage[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int s = 0; s < kLongThreads / kWave; ++s) v += stage[s];
    return v;
}

// 16 bytes of a row, at any element's address: a row's start is aligned as its width allows (the vector memory instructions
// take any address).
template <typename T>
struct Unaligned {
    typedef vec_t<T, kVec128<T>> type __attribute__((aligned(sizeof(T))));
};
// The first `count` elements from p on, zeros behind them.
template <typename T>
__device__ __forceinline__ vec_t<T, kVec128<T>> load_some(const T* p, int count) {
    if (count >= kVec128<T>) return *reinterpret_cast<const typename Unaligned<T>::type*>(p);
    vec_t<T, kVec128<T>> v(static_cast<T>(0.0f));
#pragma unroll
    for (int e = 0; e < kVec128<T> - 1; ++e)
        if (e < count) v[e] = p[e];
    return v;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, vec_t<T, kVec128<T>> v, int count) {
    if (count >= kVec128<T>) {
        *reinterpret_cast<typename Unaligned<T>::type*>(p) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < kVec128<T> - 1; ++e)
        if (e < count) p[e] = v[e];
}

// A row in walks of a workgroup: use(first column, elements of it, its values as fp32).
template <typename T, typename Use>
__device__ __forceinline__ void walk_row(const T* row, int hidden, Use&& use) {
    constexpr int VEC = kVec128<T>;
    for (int col = threadIdx.x * VEC; col < hidden; col += kLongThreads * VEC)
        use(col, hidden - col, vec_to_f32<T, VEC>(load_some<T>(row + col, hidden - col)));
}

// Sums over the LPR lanes, or the WAVES wavefronts, of a row; the same bits in all of its lanes. `stage` is not used for another sum
// before the workgroup has met twice more: one barrier a sum is enough.
template <int LPR, int WAVES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*stage)[WAVES]) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = wave_sum<LPR>(v[n]);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & (kWave - 1)) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) stage[n][threadIdx.x / kWave] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = 0.0f;
#pragma unroll
            for (int s = 0; s < WAVES; ++s) v[n] += stage[n][s];
        }
    }
}

}  // namespace cgptx
