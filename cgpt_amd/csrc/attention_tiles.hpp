// What the matrix-core kernels of attention share: operand fragments of v_mfma_f32_32x32x16, the mapping of workgroups to query
// blocks, and the LDS-direct streaming of 64-row tiles (the schemes are described in attention.hip).
#pragma once

#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace cgptx {

constexpr int kThreads = 256;
constexpr int kBlockRows = 128;  // stationary rows per block (32 per wave)
constexpr int kStream = 64;      // streamed rows per LDS tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

using acc_t = vec_t<float, 16>;
using s16x4 = vec_t<short, 4>;

template <typename T>
struct Mma;
// The compiler places result and addend (this file is built with MFMA results in vector registers, where the
// softmax arithmetic reads them without a copy).
template <>
struct Mma<bf16_t> {
    using frag = vec_t<bf16_t, 8>;
    __device__ static __forceinline__ acc_t run(frag a, frag b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<f16_t> {
    using frag = vec_t<f16_t, 8>;
    __device__ static __forceinline__ acc_t run(frag a, frag b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// Fragment with the head dimension as contraction index taken from global memory (for the operand that stays in registers):
// lane -> row lane%32, elements d = 16*step + 8*(lane/32) .. +7.
template <typename T>
__device__ __forceinline__ typename Mma<T>::frag global_frag(const T* row_ptr, bool live, int step, int d) {
    const int lane = threadIdx.x & 63;
    const int col = step * 16 + (lane >> 5) * 8;
    using frag = typename Mma<T>::frag;
    if (live && col < d) return *reinterpret_cast<const frag*>(row_ptr + col);
    return frag(static_cast<T>(0.0f));
}

// Accumulator registers 8*step .. 8*step+7 as a 16-bit k-operand.
template <typename T>
__device__ __forceinline__ typename Mma<T>::frag acc_frag(const acc_t& acc, int step) {
    vec_t<float, 8> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = acc[8 * step + e];
    return vec_from_f32<T, 8>(f);
}

// Streamed index of accumulator register i: 8*(i/4) + 4*(lane/32) + i%4.
__device__ __forceinline__ int acc_row(int i) { return 8 * (i >> 2) + 4 * ((threadIdx.x & 63) >> 5) + (i & 3); }

// Query block, head and batch entry of a workgroup of the forward and dQ kernels (grid: query blocks
// x heads x batch). Workgroups start in the order of their linear id, as slots become free, and go
// to the 8 XCDs round-robin. Under a causal mask a query block's work grows with its position, so
// the linear id is read position-major with the last (longest) query blocks first: the work that
// is handed out last is the shortest, which keeps the tail of the launch short, and every XCD
// receives the same mix of lengths.
// Each XCD has its own L2, and the workgroups that stream the same K and V are the heads of one GQA group
// at every query position: when the (batch, kv-head) pairs divide evenly over the 8 XCDs, XCD x (linear id
// mod 8) takes pairs x, x + 8, ... and walks positions (longest first) x its pairs x the heads of the group,
// so that the workgroups resident on an XCD at any time share a few K/V streams instead of each bringing
// its own from memory.
struct BlockCoordinates {
    int q_block;  // first query row
    int h, b;
};
template <int ROWS = kBlockRows>
__device__ __forceinline__ BlockCoordinates block_coordinates(int hkv) {
    constexpr unsigned int kXcds = 8;
    const unsigned int linear = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
    const unsigned int heads = gridDim.y, batch = gridDim.z, positions = gridDim.x;
    const unsigned int pairs = batch * static_cast<unsigned int>(hkv), group = heads / static_cast<unsigned int>(hkv);
    BlockCoordinates c;
    if (pairs % kXcds == 0) {
        const unsigned int xcd = linear % kXcds, local = linear / kXcds;
        const unsigned int per_position = (pairs / kXcds) * group;
        const unsigned int position = local / per_position, rest = local - position * per_position;
        const unsigned int pair = xcd + kXcds * (rest / group), head_in_group = rest % group;
        c.q_block = static_cast<int>(positions - 1 - position) * ROWS;
        c.b = static_cast<int>(pair / static_cast<unsigned int>(hkv));
        c.h = static_cast<int>((pair % static_cast<unsigned int>(hkv)) * group + head_in_group);
        return c;
    }
    const unsigned int per_position = heads * batch;
    const unsigned int position = linear / per_position, rest = linear - position * per_position;
    c.q_block = static_cast<int>(positions - 1 - position) * ROWS;
    c.h = static_cast<int>(rest % heads);
    c.b = static_cast<int>(rest / heads);
    return c;
}

// delta = Σ_d dO·O of the rows whose dO fragments a wavefront holds, in all lanes of a row, left in memory (with LSE·log2 e
// beside it) for the dK/dV pass. A pass of its own read dO once more and was one launch more: backward in a graph, batch x length
// x heads x width, 3 x 100 x 4:2 x 64 16.2 -> 15.3 us, 1 x 512 x 32:8 x 128 42.8 -> 42.4, 8 x 4096 x 12:4 x 64 748 -> 736,
// 32 x 1024 x 8:2 x 128 the same. The order of additions is that of a butterfly over the row's groups of eight columns.
template <typename T, int STEPS>
__device__ __forceinline__ float row_delta(const typename Mma<T>::frag (&dof)[STEPS], const typename Mma<T>::frag (&of)[STEPS]) {
    float sum[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const auto o = vec_to_f32<T, 8>(of[s]), dout = vec_to_f32<T, 8>(dof[s]);
        sum[s] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[s] = fmaf(dout[e], o[e], sum[s]);
    }
#pragma unroll
    for (int w = STEPS / 2; w > 0; w /= 2)
#pragma unroll
        for (int s = 0; s < w; ++s) sum[s] += sum[s + w];
    return sum[0] + __shfl_xor(sum[0], 32, kWave);
}
template <typename T, int STEPS>
__device__ __forceinline__ float row_delta(const typename Mma<T>::frag (&dof)[STEPS], const T* o_row, bool live, int d) {
    typename Mma<T>::frag of[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) of[s] = global_frag<T>(o_row, live, s, d);
    return row_delta<T, STEPS>(dof, of);
}

template <int W>
constexpr int kWideTile = kStream * W;  // elements of one 64 x W tile

constexpr int kSchedMfma = 0x008, kSchedDsRead = 0x100;
template <int CLASS, int COUNT>
__device__ __forceinline__ void sched_group() {
    if constexpr (COUNT > 0) __builtin_amdgcn_sched_group_barrier(CLASS, COUNT, 0);
}
// LEAD LDS reads up front, then MFMAS matrix instructions with the remaining READS - LEAD reads
// spread between the first ones of them.
template <int MFMAS, int READS, int LEAD, int I = 0>
__device__ __forceinline__ void sched_reads_under_mfmas() {
    if constexpr (I == 0) sched_group<kSchedDsRead, LEAD>();
    if constexpr (I < MFMAS) {
        constexpr int kRest = READS - LEAD;
        constexpr int kSpan = MFMAS - 2;  // the last two MFMAs need no further reads
        constexpr int kDone = I < kSpan ? (I * kRest) / kSpan : kRest;
        constexpr int kNext = I + 1 < kSpan ? ((I + 1) * kRest) / kSpan : kRest;
        sched_group<kSchedMfma, 1>();
        sched_group<kSchedDsRead, kNext - kDone>();
        sched_reads_under_mfmas<MFMAS, READS, LEAD, I + 1>();
    }
}

// MFMAS matrix instructions with READS LDS reads, VALU vector and TRANS transcendental instructions of
// independent work dealt out evenly between them (reads lead by a few so that operands arrive in time).
constexpr int kSchedValu = 0x002, kSchedTrans = 0x400;
template <int MFMAS, int READS, int VALU, int TRANS, int I = 0>
__device__ __forceinline__ void sched_pipeline() {
    if constexpr (I == 0) sched_group<kSchedDsRead, (READS < 6 ? READS : 6)>();
    if constexpr (I < MFMAS) {
        constexpr int kLead = READS < 6 ? READS : 6;
        constexpr int kRest = READS - kLead;
        sched_group<kSchedMfma, 1>();
        sched_group<kSchedDsRead, ((I + 1) * kRest) / MFMAS - (I * kRest) / MFMAS>();
        sched_group<kSchedValu, ((I + 1) * VALU) / MFMAS - (I * VALU) / MFMAS>();
        sched_group<kSchedTrans, ((I + 1) * TRANS) / MFMAS - (I * TRANS) / MFMAS>();
        sched_pipeline<MFMAS, READS, VALU, TRANS, I + 1>();
    }
}

template <int W>
__device__ __forceinline__ int swizzle(int row) {
    static_assert(W == 64 || W == 128, "padded widths of the LDS-direct kernels");
    if constexpr (W == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

using lds_void_ptr = __attribute__((address_space(3))) void*;

// Where a lane's 16 bytes of a streamed tile come from. One load instruction fills 1 KiB = R rows
// (R = 4 for W = 128, 8 for W = 64); load i of wavefront w covers tile rows 4 R i + R w .. + R - 1,
// lane l owning LDS slot (row R w + l / chunks per row, chunk l % chunks per row).
struct TileSource {
    __amdgpu_buffer_rsrc_t rsrc;
    int voffset;    // bytes, loop-invariant
    int row_bytes;  // bytes between consecutive sequence positions
};

// last_row: elements of the last row that belong to the buffer (head_dim when base points at one
// head, the whole row when the head is chosen by the scalar offset of each load).
template <typename T, int W>
__device__ __forceinline__ TileSource make_source(const T* base, long row_stride, int rows, int d, int wave,
                                                  long last_row) {
    constexpr int kChunks = W / 8, kRowsPerLoad = 64 / kChunks;
    const int lane = threadIdx.x & 63;
    TileSource s;
    s.row_bytes = static_cast<int>(row_stride * sizeof(T));
    const int bytes = static_cast<int>(((rows - 1) * row_stride + last_row) * sizeof(T));
    s.rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, bytes, 0x00020000);
    const int r = wave * kRowsPerLoad + lane / kChunks;
    const int chunk = (lane % kChunks) ^ swizzle<W>(r);
    // Chunks beyond head_dim get an offset past every valid byte: the load then returns zeros.
    s.voffset = chunk * 8 < d ? r * s.row_bytes + chunk * 16 : (1 << 30);
    return s;
}

template <typename T, int W>
__device__ __forceinline__ void stream_tile(const TileSource& s, int row0, T* tile, int wave) {
    constexpr int kRowsPerLoad = 64 / (W / 8), kLoads = kStream / (4 * kRowsPerLoad);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(s.rsrc, (lds_void_ptr)(tile + (i * 4 + wave) * kRowsPerLoad * W), 16,
                                                 s.voffset, (row0 + i * 4 * kRowsPerLoad) * s.row_bytes, 0, 0);
}

// Element offset (within a 32-row block of a swizzled tile) of the lane's ds_read_b128 fragment:
// row lane%32, head-dim elements 16*step + 8*(lane/32) .. +7.
template <int W>
__device__ __forceinline__ int wide_direct_offset(int lane, int step) {
    const int row = lane & 31;
    return row * W + (((2 * step + (lane >> 5)) ^ swizzle<W>(row)) * 8);
}
// Element offset (within a 16-row block) of the lane's ds_read_b64_tr_b16 address for head-dim
// columns 32t .. 32t+31: rows {0-3 | 4-7} (+8 for the second read), see transposed_frag.
template <int W>
__device__ __forceinline__ int wide_transposed_offset(int lane, int t, int second) {
    const int row = (lane >> 5) * 4 + ((lane & 15) >> 2) + second * 8;
    const int chunk = t * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    return row * W + ((chunk ^ swizzle<W>(row)) * 8) + (lane & 1) * 4;
}
template <typename T>
__device__ __forceinline__ typename Mma<T>::frag wide_transposed_frag(const T* block, int first, int second) {
    using lds_ptr = __attribute__((address_space(3))) s16x4*;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(block + first));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(block + second));
    vec_t<short, 8> both;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        both[e] = lo[e];
        both[4 + e] = hi[e];
    }
    return __builtin_bit_cast(typename Mma<T>::frag, both);
}

// max(a, b, c) in one instruction; the operands are never NaN here.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

constexpr float kRescaleThreshold = 8.0f;  // log2 of the factor by which probabilities may exceed 1

// Exchange between lane l and lane l^32.
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Forward and dQ in two parts (PARTS = 2): a workgroup takes 64 query rows instead of 128 and two of its four wavefronts
// each walk the even and the odd key tiles; their sums meet in LDS. For calls whose blocks of 128 rows leave compute units
// idle: twice the workgroups, half the tiles one after the other, at twice the LDS (128 KiB with heads of 128: one
// workgroup per CU). One sequence of 512, 32 heads of 128: forward 15.2 -> 12.5 us, dQ 18.2 -> 15.1.
template <typename T, int W, int PARTS>
__device__ __forceinline__ T* wide_stages() {
    if constexpr (PARTS == 1) {
        __shared__ __align__(1024) T lds[4 * kWideTile<W>];
        return lds;
    } else {
        extern __shared__ __align__(1024) unsigned char wide_smem[];
        return reinterpret_cast<T*>(wide_smem);
    }
}
// A wavefront's accumulators in LDS, 16 bytes per lane side by side.
template <int DT>
__device__ __forceinline__ void deposit_sums(vec_t<float, 4>* to, const acc_t (&sums)[DT]) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            to[(4 * t + q) * kWave] = vec_t<float, 4>{sums[t][4 * q], sums[t][4 * q + 1], sums[t][4 * q + 2], sums[t][4 * q + 3]};
}
// Which of the two products is rounded is written out, here and where the parts' sums of probabilities meet: left to the compiler it
// may change with the code around it, and two kernels that promise each other's bits would differ.
template <int DT>
__device__ __forceinline__ void add_sums(const vec_t<float, 4>* from, acc_t (&sums)[DT], float mine, float other) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const vec_t<float, 4> v = from[(4 * t + q) * kWave];
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[t][4 * q + e] = fmaf(sums[t][4 * q + e], mine, v[e] * other);
        }
}

// dK and dV from the parts of shared key blocks, added in the order of the parts; four elements per thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_dkv_reduce_kernel(T* __restrict__ dk, T* __restrict__ dv,
                                                                       const float* __restrict__ partial, long count,
                                                                       int splits, int accumulate) {
    const long stride = static_cast<long>(gridDim.x) * kThreads;
#pragma unroll 1
    for (long quad = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x; quad < count / 2; quad += stride) {  // count elements of dK, then of dV
        const bool second = quad >= count / 4;
        const long at = (second ? quad - count / 4 : quad) * 4;
        const float* source = partial + (second ? count : 0) + at;
        vec_t<float, 4> sum = load_vec<float, 4>(source);
        int s = 1;
        for (; s + 3 < splits; s += 4) {
            vec_t<float, 4> v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = load_vec<float, 4>(source + 2 * (s + i) * count);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += v[i];
        }
        for (; s < splits; ++s) sum += load_vec<float, 4>(source + 2 * s * count);
        T* out = (second ? dv : dk) + at;
        if (accumulate) sum += vec_to_f32<T, 4>(load_vec<T, 4>(out));
        store_vec<T, 4>(out, vec_from_f32<T, 4>(sum));
    }
}

template <typename T>
int launch_dkv_reduce(long count, void* dk, void* dv, const float* partial, int splits, int accumulate, hipStream_t stream) {
    const long blocks = std::min<long>((count / 2 + kThreads - 1) / kThreads, kLaunchThreads / kThreads);
    hipLaunchKernelGGL((attention_dkv_reduce_kernel<T>), dim3(static_cast<unsigned int>(blocks)), dim3(kThreads), 0, stream,
                       static_cast<T*>(dk), static_cast<T*>(dv), partial, count, splits, accumulate);
    CGPTX_LAUNCH_CHECK();
    return CGPTX_OK;
}

// What decides how many workgroups share a key block in a dK/dV pass whose workgroups hold `block_rows` keys of one kv head, of which
// `waves` wavefronts walk tiles of `stream_rows` queries of their own, `tile_us` each.
struct KeyWalk {
    long batch, qs, ks, hkv, group, d;
    int causal;
    long offset, block_rows, stream_rows, waves;
    double tile_us;
};
inline int key_block_parts(const KeyWalk& k) {
    const long units = compute_units(), key_blocks = (k.ks + k.block_rows - 1) / k.block_rows, pairs = k.hkv * k.batch;
    long longest = 0, total = 0;
    for (long i = 0; i < key_blocks; ++i) {
        const long begin = k.causal ? std::max<long>(0, i * k.block_rows - k.offset) / k.stream_rows * k.stream_rows : 0;
        const long walked = begin < k.qs ? (k.qs - begin + k.stream_rows - 1) / k.stream_rows * k.group : 0;
        const long tiles = (walked + k.waves - 1) / k.waves;
        longest = std::max(longest, tiles);
        total += tiles * pairs;
        if (total > 16 * units * std::max<long>(longest, 1)) return 1;  // a full chip many times over
    }
    const double megabytes = static_cast<double>(k.batch * k.ks * k.hkv * k.d) * 8e-6;
    int best = 1;
    double best_us = 0.0;
    for (int parts = 1; parts <= 16 && parts <= std::max<long>(longest, 1); ++parts) {
        const double busiest = std::max<double>(std::ceil(static_cast<double>(longest) / parts), static_cast<double>(total) / static_cast<double>(units));
        const double us = busiest * k.tile_us + (parts > 1 ? 5.0 + 0.4 * megabytes * parts : 0.0);
        if (parts == 1 || us < best_us) {
            best = parts;
            best_us = us;
        }
    }
    return best;
}

}  // namespace cgptx
