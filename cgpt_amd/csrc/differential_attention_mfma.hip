// Differential attention on the matrix cores, 16-bit storage (formulas: differential_attention.hip; operand layouts and the
// streaming of tiles: attention.hip, attention_tiles.hpp).
//
// A head's row of q or k is kept in LDS and registers as two halves of W/2 columns, each padded with zeros from D/2: the score
// tile of a map is the product over its half, and both maps' score gradients meet the other operand's halves in one accumulator
// of width W. So the tiles, fragments and register counts are those of plain attention with heads of W, and what the maps add
// is a second set of exponentials and, in the forward pass, a second product with v (the maps' sums are known only at its end).
//
//   forward : block = 128 queries of one (batch, q-head), wave = 32 queries; streams 64-key K/V tiles; per tile and map Sᵀ = K·Qᵀ
//             and its softmax, then Oᵀ_i += Vᵀ·Pᵀ_i for both maps from the same fragments of V.
//   dQ      : same shape; Sᵀ_i = K_i·Qᵀ_i, Gᵀ = V·dOᵀ, dQᵀ_i += Kᵀ_i·dSᵀ_i. Leaves both maps' statistics for the dK/dV pass, and
//             dlambda's parts.
//   dK/dV   : block = 128 keys of one (batch, kv-head), wave = 32 keys; streams 64-query Q/dO tiles of every q-head of the group.
//
// Probabilities and score gradients are rounded to 16 bits once, half a step relative to the value, to be operands: results have some
// sqrt(2) of the error that rounding exact ones leaves. In two parts each they would take a third more products in dQ, half as many
// more in dK/dV and two thirds forward. All sums are fp32.
//
// 32 x 1024 tokens of 8:2 heads of 128, bf16, causal: forward 156 to 162 us (103 GFLOP, 640 TFLOP/s), dQ 166 to 180, dK/dV 190 to
// 230, the higher ones when the clock has come down from 2.14 to 1.9 GHz. 5 x 1001 tokens of 12:4 heads of 64, fp16: dQ 34 to 38, dK/dV
// 45 to 51 and 7 for the sum of its parts. Matrix instructions take a third of the cycles and vector instructions, half of them the
// maps' exponentials with what stands around them, 40 to 45 per cent.
#include "attention_tiles.hpp"
#include "differential_attention.hpp"

#include <algorithm>
#include <utility>

namespace cgptx {
namespace {

// Rows of a [.., sequence, heads, d] tensor from one (batch, head) on, streamed in 64-row tiles. A tile's buffer starts at its first
// row, so that 32 bits hold every offset in it however long the sequence is; rows past the end and padding columns are zeros.
struct RowStream {
    const char* base;
    long bytes;     // from base to the end of the last row's part that belongs to it
    int row_bytes;  // between consecutive sequence positions
    int voffset;    // of a lane's 16 bytes in the first load of a tile
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int row0) const {
        const long skipped = static_cast<long>(row0) * row_bytes;
        const long left = min(bytes - skipped, 1l << 30);
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + skipped), 0, static_cast<int>(left), 0x00020000);
    }
};
// Column of the tensor's row that padded column `c` (a multiple of 8) of a tile holds, or -1. HALVES: two halves of W/2 (q, k).
template <int W, bool HALVES>
__device__ __forceinline__ int source_column(int c, int d) {
    if constexpr (HALVES) {
        const int half = c / (W / 2), within = c % (W / 2);
        return within < d / 2 ? half * (d / 2) + within : -1;
    } else {
        return c < d ? c : -1;
    }
}
template <typename T, int W, bool HALVES>
__device__ __forceinline__ RowStream make_stream(const void* tensor, long offset, long row_stride, int rows, int d, int wave, long last_row) {
    constexpr int kChunks = W / 8, kRowsPerLoad = 64 / kChunks;
    const int lane = threadIdx.x & 63;
    RowStream s;
    s.base = static_cast<const char*>(tensor) + offset * static_cast<long>(sizeof(T));
    s.row_bytes = static_cast<int>(row_stride * sizeof(T));
    s.bytes = ((rows - 1) * row_stride + last_row) * static_cast<long>(sizeof(T));
    const int r = wave * kRowsPerLoad + lane / kChunks;
    const int column = source_column<W, HALVES>(((lane % kChunks) ^ swizzle<W>(r)) * 8, d);
    s.voffset = column >= 0 ? r * s.row_bytes + column * static_cast<int>(sizeof(T)) : (1 << 30);
    return s;
}
__device__ __forceinline__ vec_t<unsigned int, 4> load_words(__amdgpu_buffer_rsrc_t rsrc, int voffset) {
    return __builtin_bit_cast(vec_t<unsigned int, 4>, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voffset, 0, 0));
}
// 16 bytes per lane, 1 KiB in all, straight into LDS.
__device__ __forceinline__ void load_chunks(__amdgpu_buffer_rsrc_t rsrc, void* to, int voffset, int soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr)(to), 16, voffset, soffset, 0, 0);
}
template <typename T, int W>
__device__ __forceinline__ void stream_rows(const RowStream& s, int row0, T* tile, int wave) {
    constexpr int kRowsPerLoad = 64 / (W / 8), kLoads = kStream / (4 * kRowsPerLoad);
    const __amdgpu_buffer_rsrc_t rsrc = s.at(row0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        load_chunks(rsrc, tile + (i * 4 + wave) * kRowsPerLoad * W, s.voffset, i * 4 * kRowsPerLoad * s.row_bytes);
}

// Element offsets in LDS of a lane's fragments of a tile that starts at element `tile` (a multiple of 512). The offsets of a tile differ by
// bits that the swizzle only flips, so one register per kind of read stands for all of them: row-wise ones of step s, and
// transposed ones of column block t, whose second read (see wide_transposed_offset) lies eight rows further with bit 4 flipped.
template <int W>
struct TileOffsets {
    int direct, transposed;
    __device__ __forceinline__ TileOffsets(int lane) : direct(wide_direct_offset<W>(lane, 0)), transposed(wide_transposed_offset<W>(lane, 0, 0)) {}
    __device__ __forceinline__ TileOffsets at(int tile) const {
        TileOffsets o = *this;
        o.direct += tile;
        o.transposed += tile;
        asm volatile("" : "+v"(o.direct), "+v"(o.transposed));  // derived anew for each tile: no registers for all of them
        return o;
    }
    template <typename T>
    __device__ __forceinline__ typename Mma<T>::frag row(const T* lds, int block, int step) const {
        return *reinterpret_cast<const typename Mma<T>::frag*>(lds + block * W + (direct ^ (16 * step)));
    }
    template <typename T>
    __device__ __forceinline__ typename Mma<T>::frag columns(const T* lds, int block, int t) const {
        return wide_transposed_frag<T>(lds + block * W, transposed ^ (32 * t), (transposed ^ (32 * t) ^ 16) + 8 * W);
    }
};

// The operand that stays in registers, from global memory: lane -> its row (lane%32), padded columns 16*step + 8*(lane/32) .. + 7; zeros for
// a row that is not live. The row lies `row_bytes` behind element `offset` of the tensor, whose part that the wavefront's rows
// are in has `bytes` from there on.
template <typename T, int W, bool HALVES>
__device__ __forceinline__ void load_rows(typename Mma<T>::frag (&rows)[W / 16], const void* tensor, long offset, long bytes, int row_bytes,
                                          bool live, int d) {
    using frag = typename Mma<T>::frag;
    const int half = (threadIdx.x & 63) >> 5;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(static_cast<const T*>(tensor) + offset), 0,
                                                                          static_cast<int>(min(bytes, 1l << 30)), 0x00020000);
#pragma unroll
    for (int i = 0; i < W / 16; ++i) {
        const int column = source_column<W, HALVES>(i * 16 + half * 8, d);
        rows[i] = __builtin_bit_cast(frag, load_words(rsrc, live && column >= 0 ? row_bytes + column * static_cast<int>(sizeof(T)) : 1 << 30));
    }
}

// Stores a wavefront's transposed accumulators (lane = row, registers = padded columns) times a factor, four elements at a time.
// value(t, r) is register r of column block t. (fp32: parts, stored without adding.)
template <typename T, int W, bool HALVES, typename Value>
__device__ __forceinline__ void store_columns(T* row, int d, bool accumulate, Value&& value) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < W / 32; ++t) {
        if constexpr (sizeof(T) == 2) {
            // A lane has quads of its row's columns, its partner in the other half of the wavefront the quads between: swapped, a lane has
            // eight in a row of every other group.
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                const int column = source_column<W, HALVES>(t * 32 + (g + (lane >> 5)) * 8, d);
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(value(t, 4 * g + e)), __float_as_uint(value(t, 4 * g + 4 + e)),
                                                                          false, false);
                    v[e] = __uint_as_float(swapped[0]);
                    v[4 + e] = __uint_as_float(swapped[1]);
                }
                if (column < 0) continue;
                vec_t<float, 8> sum{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
                if (accumulate) sum += vec_to_f32<T, 8>(load_vec<T, 8>(row + column));
                store_vec<T, 8>(row + column, vec_from_f32<T, 8>(sum));
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int column = source_column<W, HALVES>(t * 32 + g * 8, d);
                if (column < 0) continue;
                T* to = row + column + (lane >> 5) * 4;
                vec_t<float, 4> v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = value(t, 4 * g + e);
                store_vec<T, 4>(to, v);
            }
        }
    }
}

// Whether rows `from` .. 63 of a tile hold an Inf or a NaN (the same answer in all lanes): their products with 0 are not 0. Looked at in
// halves of 32 rows.
template <typename T, int W>
__device__ __forceinline__ bool not_finite(const T* tile, int from) {
    using pair = vec_t<T, 2>;
    float sum = 0.0f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (half == 0 && from >= 32) continue;
#pragma unroll
        for (int i = 0; i < W / 16; ++i) {
            const auto words = *reinterpret_cast<const vec_t<unsigned int, 4>*>(tile + ((half * (W / 16) + i) * kWave + (threadIdx.x & 63)) * 8);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const pair x = __builtin_bit_cast(pair, words[w]), zeros(static_cast<T>(0.0f));
                if constexpr (__is_same(T, f16_t)) sum = __builtin_amdgcn_fdot2(x, zeros, sum, false);
                else sum = __builtin_amdgcn_fdot2_f32_bf16(x, zeros, sum, false);
            }
        }
    }
    return __any(!(sum == 0.0f));
}
// A hidden key's probability is 0, but 0 x Inf is NaN in the matrix instruction: a tile on the causal diagonal (at most two of a
// wavefront's) that is not finite is left out of the products and added key by key behind the walk, by the lanes that see the key.
struct LeftOut {
    int hidden, first, tiles = 0;  // first key that a row of the wavefront does not see, its tile; bits of the tiles from there on
    __device__ __forceinline__ LeftOut(const DifferentialArgs& p, int wave_first_q)
        : hidden(p.offset + wave_first_q + 1), first(p.causal ? hidden / kStream : 1 << 30) {}
    // Whether tile j is one of them (the wavefront's causal mask allows it and the tile's values are not finite).
    template <typename T, int W>
    __device__ __forceinline__ bool out(int j, const T* tile) {
        if (j < first || !not_finite<T, W>(tile, hidden - j * kStream)) return false;
        tiles |= 1 << (j - first);
        return true;
    }
    template <typename Use>
    __device__ __forceinline__ void each_key(int ks, Use&& use) const {
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            if ((tiles >> i & 1) == 0) continue;
#pragma unroll 1
            for (int key = (first + i) * kStream; key < min(ks, (first + i + 1) * kStream); ++key) use(key);
        }
    }
};
// The accumulators in the lane's own memory, where code that runs once in a blue moon takes no registers from the walk.
template <int COUNT>
struct Parked {
    volatile float values[COUNT * 16];
    __device__ __forceinline__ void put(int t, const acc_t& sums) {
#pragma unroll
        for (int e = 0; e < 16; ++e) values[t * 16 + e] = sums[e];
    }
    __device__ __forceinline__ void get(int t, acc_t& sums) const {
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[e] = values[t * 16 + e];
    }
};
// Product of columns from .. from + count - 1 of two rows.
template <typename T>
__device__ __noinline__ float row_product(const T* a, const T* b, int count) {
    float sum = 0.0f;
    for (int c = 0; c < count; ++c) sum = fmaf(to_f32(a[c]), to_f32(b[c]), sum);
    return sum;
}
// Column of a row that register `index` of a lane's accumulators (16 to a block of 32 columns) stands for, or -1.
template <int W, bool HALVES>
__device__ __forceinline__ int register_column(int index, int d) {
    const int block = source_column<W, HALVES>(index / 16 * 32 + (index % 16 >> 2) * 8, d);
    return block < 0 ? -1 : block + ((threadIdx.x & 63) >> 5) * 4 + (index & 3);
}

struct RowTiles {
    int b, h, kvh, row, row_wave, part;  // row: of the workgroup's first, of a head's queries
    int first_q, last_q;                 // tokens of the wavefront's first and last row
    int q;                               // token of this lane's row
    int beside;                          // heads from h to this lane's row's
    bool live, wave_live;
    template <int PARTS, bool SPLIT = false>
    __device__ __forceinline__ static RowTiles of(const DifferentialArgs& p, int wave) {
        constexpr int kRows = kBlockRows / PARTS;
        RowTiles r;
        const int pack = SPLIT ? p.pack : 1;
        if constexpr (SPLIT) {  // workgroups that share a query block next to each other
            r.b = blockIdx.z;
            r.h = blockIdx.y * pack;
            r.row = static_cast<int>(blockIdx.x) / p.splits * kRows;
        } else {
            const BlockCoordinates where = block_coordinates<kRows>(p.hkv);
            r.b = where.b;
            r.h = where.h;
            r.row = where.q_block;
        }
        r.kvh = r.h / (p.hq / p.hkv);
        r.row_wave = wave % (4 / PARTS);
        r.part = wave / (4 / PARTS);
        const int first = r.row + r.row_wave * 32, mine = first + static_cast<int>(threadIdx.x & 31);
        r.first_q = first / pack;
        r.last_q = min((first + 31) / pack, p.qs - 1);
        r.q = mine / pack;
        r.beside = mine - r.q * pack;
        r.live = r.q < p.qs;
        r.wave_live = r.first_q < p.qs;
        return r;
    }
    // Elements from the start of a tensor like q to this lane's row.
    __device__ __forceinline__ long offset(const DifferentialArgs& p) const {
        return ((static_cast<long>(b) * p.qs + q) * p.hq + h + beside) * p.d;
    }
};

// SPLIT: p.splits workgroups share a query block's keys, and a block has the rows of p.pack heads of a group, which read the same keys;
// each workgroup leaves its sums, and the maxima that they stand to, in p.partial, and
// differential_combine_kernel brings them together.
template <typename T, int W, int PARTS, bool SPLIT>
__global__ __launch_bounds__(kThreads, 2) void differential_forward_kernel(DifferentialArgs p) {
    using frag = typename Mma<T>::frag;
    constexpr int STEPS = W / 16, HALF = STEPS / 2, DT = W / 32;
    T* const lds = wide_stages<T, W, PARTS>();  // [stage][part][K | V]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const RowTiles at = RowTiles::of<PARTS, SPLIT>(p, wave);
    const long q_stride = static_cast<long>(p.hq) * p.d, kv_stride = static_cast<long>(p.hkv) * p.d;
    const long q_offset = at.offset(p), first_row = at.wave_live ? ((static_cast<long>(at.b) * p.qs + at.first_q) * p.hq + at.h) * p.d : 0;
    const int row_bytes = ((at.q - at.first_q) * p.hq + at.beside) * p.d * static_cast<int>(sizeof(T));
    const long wave_bytes = at.wave_live ? ((at.last_q - at.first_q + 1) * q_stride - at.h * p.d) * static_cast<long>(sizeof(T)) : 0;
    const long kv_offset = static_cast<long>(at.b) * p.ks * kv_stride + at.kvh * p.d;
    const RowStream k_src = make_stream<T, W, true>(p.k, kv_offset, kv_stride, p.ks, p.d, wave, p.d);
    const RowStream v_src = make_stream<T, W, false>(p.v, kv_offset, kv_stride, p.ks, p.d, wave, p.d);

    const int last_q_block = min((at.row + kBlockRows / PARTS - 1) / (SPLIT ? p.pack : 1), p.qs - 1);
    const int k_end = p.causal ? min(p.ks, p.offset + last_q_block + 1) : p.ks;
    const int all_tiles = (k_end + kStream - 1) / kStream, split = SPLIT ? static_cast<int>(blockIdx.x) % p.splits : 0;
    const int begin = SPLIT ? static_cast<int>(static_cast<long>(split) * all_tiles / p.splits) : 0;
    const int tiles = SPLIT ? static_cast<int>(static_cast<long>(split + 1) * all_tiles / p.splits) : all_tiles;  // end of this workgroup's
    auto request = [&](int j, T* stage) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < PARTS; ++g) {
            if (j + g >= tiles) break;
            stream_rows<T, W>(k_src, (j + g) * kStream, stage + 2 * g * kWideTile<W>, wave);
            stream_rows<T, W>(v_src, (j + g) * kStream, stage + (2 * g + 1) * kWideTile<W>, wave);
        }
    };
    request(begin, lds);

    frag qf[STEPS];
    load_rows<T, W, true>(qf, p.q, first_row, wave_bytes, row_bytes, at.live, p.d);
    const TileOffsets<W> offsets(lane);

    // Both maps' sums, and their running maxima m of the raw scores (the scale is positive) as in attention.hip: mb = m * scale2, 0 while
    // m is -inf; it follows the maximum only when that has moved by more than 2^8 in probability.
    acc_t o[2][DT];
    float m[2], mb[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int t = 0; t < DT; ++t) o[i][t] = acc_t(0.0f);
        m[i] = -INFINITY;
        mb[i] = 0.0f;
        l[i] = 0.0f;
    }
    const float scale2 = p.scale * kLog2e;
    const int wave_first_q = at.first_q, wave_last_q = at.last_q;
    const bool wave_live = at.wave_live;
    const int q_limit = p.causal ? p.offset + at.q : p.ks;  // largest visible key of this lane's query
    const int clear_limit = p.causal ? min(p.ks - 1, p.offset + wave_first_q) : p.ks - 1;  // tiles up to here need no mask

    LeftOut left(p, wave_first_q);
    for (int first = begin; first < tiles; first += PARTS) {
        const int j = first + at.part, k0 = j * kStream, stage = ((first - begin) / PARTS) & 1;
        const int tile = (stage * PARTS + at.part) * 2 * kWideTile<W>;  // K's; V's is the next
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's part of the tiles is in LDS
        __syncthreads();                     // ... and everybody else's; the other stage is free
        request(first + PARTS, lds + (stage ^ 1) * PARTS * 2 * kWideTile<W>);
        if (PARTS > 1 && j >= tiles) continue;
        if (!wave_live || (p.causal && k0 > p.offset + wave_last_q) || left.out<T, W>(j, lds + tile + kWideTile<W>)) continue;
        const bool masked = k0 + kStream - 1 > clear_limit;
        const int bound = min(q_limit, p.ks - 1) - k0 - 4 * (lane >> 5);  // of the tile's keys, what this lane's query sees

        const TileOffsets<W> here = offsets.at(tile);
        frag pf[2][2][2];  // [map][32 keys][16 keys]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            acc_t st[2] = {acc_t(0.0f), acc_t(0.0f)};
            {
                frag ka[2][HALF];
#pragma unroll
                for (int s = 0; s < HALF; ++s) {
                    ka[0][s] = here.row(lds, 0, i * HALF + s);
                    ka[1][s] = here.row(lds, 32, i * HALF + s);
                }
#pragma unroll
                for (int s = 0; s < HALF; ++s) {
                    st[0] = Mma<T>::run(ka[0][s], qf[i * HALF + s], st[0]);
                    st[1] = Mma<T>::run(ka[1][s], qf[i * HALF + s], st[1]);
                }
                sched_reads_under_mfmas<2 * HALF, 2 * HALF, 4>();
            }
            __builtin_amdgcn_sched_barrier(0);
            if (masked) {
                asm volatile("" ::: "memory");  // keeps the masking out of the common path (no if-conversion)
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        st[sub][e] = (sub * 32 + 8 * (e >> 2) + (e & 3) <= bound) ? st[sub][e] : -INFINITY;
            }
            float top = max3(st[0][0], st[1][0], st[0][1]);
            top = max3(top, st[1][1], st[0][2]);
#pragma unroll
            for (int e = 2; e < 16; ++e) top = max3(top, st[1][e], e + 1 < 16 ? st[0][e + 1] : st[1][e]);
            top = fmaxf(top, other_half(top));
            if (__any(top > m[i] && (top - m[i]) * scale2 > kRescaleThreshold)) {
                const float next = fmaxf(m[i], top);
                const float next_b = next == -INFINITY ? 0.0f : next * scale2;
                const float alpha = __builtin_amdgcn_exp2f(m[i] == -INFINITY ? -INFINITY : m[i] * scale2 - next_b);
                l[i] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t) o[i][t] *= alpha;
                m[i] = next;
                mb[i] = next_b;
            }
            float sum = 0.0f;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float prob = __builtin_amdgcn_exp2f(fmaf(st[sub][e], scale2, -mb[i]));
                    st[sub][e] = prob;
                    sum += prob;
                }
            l[i] += sum;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int s = 0; s < 2; ++s) pf[i][sub][s] = acc_frag<T>(st[sub], s);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                frag vt[DT];
#pragma unroll
                for (int t = 0; t < DT; ++t) vt[t] = here.columns(lds, kStream + sub * 32 + s * 16, t);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    o[0][t] = Mma<T>::run(vt[t], pf[0][sub][s], o[0][t]);
                    o[1][t] = Mma<T>::run(vt[t], pf[1][sub][s], o[1][t]);
                }
            }
        sched_reads_under_mfmas<8 * DT, 8 * DT, 8>();
        __builtin_amdgcn_sched_barrier(0);
    }
    if (left.tiles != 0) {
        Parked<2 * DT> sums;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            sums.put(t, o[0][t]);
            sums.put(DT + t, o[1][t]);
        }
        const T* q_row = static_cast<const T*>(p.q) + q_offset;
        left.each_key(p.ks, [&](int key) {
            if (!at.live || key > q_limit) return;
            const T* k_row = static_cast<const T*>(p.k) + kv_offset + key * kv_stride;
            const T* v_row = static_cast<const T*>(p.v) + kv_offset + key * kv_stride;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float score = row_product(q_row + i * (p.d / 2), k_row + i * (p.d / 2), p.d / 2);
                const float next = fmaxf(m[i], score), next_b = next == -INFINITY ? 0.0f : next * scale2;
                const float alpha = __builtin_amdgcn_exp2f(m[i] == -INFINITY ? -INFINITY : mb[i] - next_b);
                const float e = __builtin_amdgcn_exp2f(fmaf(score, scale2, -next_b));
                l[i] = fmaf(l[i], alpha, lane < 32 ? e : 0.0f);  // a row's sum is that of its two lanes'
                m[i] = next;
                mb[i] = next_b;
#pragma unroll 1
                for (int r = 0; r < DT * 16; ++r) {
                    const int column = register_column<W, false>(r, p.d);
                    if (column >= 0) sums.values[i * DT * 16 + r] = fmaf(e, to_f32(v_row[column]), sums.values[i * DT * 16 + r] * alpha);
                }
            }
        });
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            sums.get(t, o[0][t]);
            sums.get(DT + t, o[1][t]);
        }
    }
    if constexpr (PARTS > 1) {
        // The second part's sums are brought to the common maximum and added to the first's.
        constexpr int kWords = 2 * (4 * DT + 1);
        auto* meet = reinterpret_cast<vec_t<float, 4>*>(lds) + at.row_wave * kWords * kWave + lane;
        __syncthreads();
        if (at.part != 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                deposit_sums<DT>(meet + i * (4 * DT + 1) * kWave, o[i]);
                meet[(i * (4 * DT + 1) + 4 * DT) * kWave] = vec_t<float, 4>{m[i], l[i], 0.0f, 0.0f};
            }
        }
        __syncthreads();
        if (at.part != 0) return;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const vec_t<float, 4> theirs = meet[(i * (4 * DT + 1) + 4 * DT) * kWave];
            const float top = fmaxf(m[i], theirs[0]);
            const float top_b = top == -INFINITY ? 0.0f : top * scale2;
            const float mine = m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mb[i] - top_b);
            const float other = theirs[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(theirs[0] * scale2 - top_b);
            l[i] = fmaf(l[i], mine, theirs[1] * other);
            add_sums<DT>(meet + i * (4 * DT + 1) * kWave, o[i], mine, other);
            mb[i] = top_b;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) l[i] += other_half(l[i]);
    if (!at.live) return;
    if constexpr (SPLIT) {
        const long rows = static_cast<long>(p.batch) * p.qs * p.hq, row = (static_cast<long>(at.b) * p.qs + at.q) * p.hq + at.h + at.beside;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long to = (static_cast<long>(split) * 2 + i) * rows + row;
            store_columns<float, W, false>(p.partial + to * p.d, p.d, false, [&](int t, int e) { return o[i][t][e]; });
            if (lane < 32) {
                p.delta[2 * to] = l[i] > 0.0f || l[i] != l[i] ? mb[i] : -INFINITY;  // no key that the row sees: no part of it
                p.delta[2 * to + 1] = l[i];
            }
        }
        return;
    }
    const float lambda = p.lambda[at.h];
    const float inverse1 = 1.0f / l[0], inverse2 = 1.0f / l[1];
    store_columns<T, W, false>(static_cast<T*>(p.out) + q_offset, p.d, false,
                               [&](int t, int e) { return fmaf(-lambda, o[1][t][e] * inverse2, o[0][t][e] * inverse1); });
    if (p.second != nullptr)
        store_columns<T, W, false>(static_cast<T*>(p.second) + q_offset, p.d, false, [&](int t, int e) { return o[1][t][e] * inverse2; });
    if (p.lse_out != nullptr) {  // one map from either half of the wavefront
        const long rows = static_cast<long>(p.batch) * p.qs * p.hq, row = (static_cast<long>(at.b) * p.qs + at.q) * p.hq + at.h + at.beside;
        const bool second = lane >= 32;
        p.lse_out[(second ? rows : 0) + row] = ((second ? mb[1] : mb[0]) + log2f(second ? l[1] : l[0])) * kLn2;
    }
}

// A row of a forward pass whose keys were shared, from what the workgroups left: both maps' sums brought to their common maxima. What
// bounds it is the way to memory, where the other XCDs' workgroups have left their parts: a workgroup has a row, a wavefront a map's even or odd
// parts, and all of its loads are on their way before the first is used (one after the other, a wavefront to a row: 17 us for 32
// parts).
constexpr int kMostSplits = 64;
template <typename T, int MOST>
__global__ __launch_bounds__(kThreads) void differential_combine_kernel(DifferentialArgs p) {
    __shared__ vec_t<float, 2> stage[4][kWave];
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq, row = blockIdx.x;
    const int lane = threadIdx.x & (kWave - 1), at = 2 * lane, wave = threadIdx.x / kWave, map = wave & 1, odd = wave >> 1;
    vec_t<float, 2> part[MOST / 2];
#pragma unroll
    for (int u = 0; u < MOST / 2; ++u)
        if (2 * u + odd < p.splits) part[u] = load_vec<float, 2>(p.partial + ((2l * (2 * u + odd) + map) * rows + row) * p.d + min(at, p.d - 2));
    // A part per lane: all their maxima and sums at once.
    const long mine = 2 * ((2l * min(lane, p.splits - 1) + map) * rows + row);
    const float part_top = lane < p.splits ? p.delta[mine] : -INFINITY, part_sum = lane < p.splits ? p.delta[mine + 1] : 0.0f;
    const float top = wave_max(part_top), weight = part_top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(part_top - top);
    const float sum = wave_sum(part_sum * weight);
    vec_t<float, 2> o(0.0f);
#pragma unroll
    for (int u = 0; u < MOST / 2; ++u) {
        if (2 * u + odd >= p.splits) break;
        const float factor = __shfl(weight, 2 * u + odd, kWave);
        o[0] = fmaf(part[u][0], factor, o[0]);
        o[1] = fmaf(part[u][1], factor, o[1]);
    }
    stage[wave][lane] = o * (1.0f / sum);
    if (p.lse_out != nullptr && odd == 0 && lane == 0) p.lse_out[map * rows + row] = (top + log2f(sum)) * kLn2;
    __syncthreads();
    if (wave != 0 || at >= p.d) return;
    const float lambda = p.lambda[row % p.hq];
    const vec_t<float, 2> first = stage[0][lane] + stage[2][lane], second = stage[1][lane] + stage[3][lane];
    const vec_t<float, 2> out{fmaf(-lambda, second[0], first[0]), fmaf(-lambda, second[1], first[1])};
    store_vec<T, 2>(static_cast<T*>(p.out) + row * p.d + at, vec_from_f32<T, 2>(out));
    if (p.second != nullptr) store_vec<T, 2>(static_cast<T*>(p.second) + row * p.d + at, vec_from_f32<T, 2>(second));
}

// Half precision's smallest normal number is 2^-14. Score gradients P (G - delta) are rounded to storage before their products, and where
// output gradients are small (P is some 1/n beside a dO of any size) they are below it and lose their digits. So they are enlarged by a power of
// two, which costs nothing inside P's exponent, and the sums are made smaller by it: by what brings the largest |dO| (of the row for
// dq, of the (batch entry, kv head) for dk and dv) to between 4 and 8, where dO of deviation 1 has it. P v has to be some thousands there
// before a score gradient of 128 columns passes 65504; sums that are not finite then are taken again in fp32 (dq_of_row, dk_of_row), some
// hundred times slower.
template <typename T>
constexpr bool kEnlarged = __is_same(T, f16_t);
// The power that brings `largest` to between 4 and 8: 0 from 4 on and for what is no number, at most `most`.
__device__ __forceinline__ int enlarging_power(float largest, int most) {
    return max(min(127 + 2 - static_cast<int>(__float_as_uint(largest) >> 23), most), 0);
}
// The largest of the absolute values of a row in half precision, in all lanes of the row.
template <int STEPS>
__device__ __forceinline__ float largest_of_row(const Mma<f16_t>::frag (&row)[STEPS]) {
    using words = vec_t<unsigned int, 4>;
    using pair = vec_t<unsigned short, 2>;
    pair top(static_cast<unsigned short>(0));
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) top = __builtin_elementwise_max(top, __builtin_bit_cast(pair, __builtin_bit_cast(words, row[s])[w] & 0x7FFF7FFFu));
    const unsigned short mine = top[0] > top[1] ? top[0] : top[1];
    const float value = to_f32(__builtin_bit_cast(f16_t, mine));
    return __uint_as_float(max(__float_as_uint(value), __float_as_uint(other_half(value))));  // as bits: a NaN is the largest
}
// Whether any of the sums is not finite.
template <int DT>
__device__ __forceinline__ bool any_not_finite(const acc_t (&sums)[DT]) {
    float zero = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) zero = fmaf(sums[t][e], 0.0f, zero);
    return !(zero == 0.0f);
}
// The sign of -lambda.
__device__ __forceinline__ float sign_of_second(float lambda) { return lambda > 0.0f ? -1.0f : 1.0f; }

// A row of d elements in a wavefront, lane l with elements l and l + 64, those of the second map apart from those of the first.
struct WaveRow {
    float x[2];
    template <typename T>
    __device__ __forceinline__ static WaveRow load(const T* row, int d) {
        const int lane = threadIdx.x & 63;
        return {{lane < d ? to_f32(row[lane]) : 0.0f, lane + kWave < d ? to_f32(row[lane + kWave]) : 0.0f}};
    }
    __device__ __forceinline__ float dot(const WaveRow& y) const { return wave_sum(fmaf(x[0], y.x[0], x[1] * y.x[1])); }
    __device__ __forceinline__ bool finite() const { return !__any(!(fmaf(x[0], 0.0f, x[1] * 0.0f) == 0.0f)); }
    // The product's elements of the first map or the second.
    __device__ __forceinline__ float dot(const WaveRow& y, bool second, int d) const {
        const int lane = threadIdx.x & 63;
        const float a = (lane >= d / 2) == second ? x[0] * y.x[0] : 0.0f, b = (lane + kWave >= d / 2) == second ? x[1] * y.x[1] : 0.0f;
        return wave_sum(a + b);
    }
    __device__ __forceinline__ void add(const WaveRow& y, float first, float second, int d) {
        const int lane = threadIdx.x & 63;
        x[0] = fmaf(lane < d / 2 ? first : second, y.x[0], x[0]);
        x[1] = fmaf(lane + kWave < d / 2 ? first : second, y.x[1], x[1]);
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, int d, float factor, bool accumulate) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            T* to = row + lane + i * kWave;
            if (lane + i * kWave < d) *to = from_f32<T>(fmaf(x[i], factor, accumulate ? to_f32(*to) : 0.0f));
        }
    }
};
// A row of dq by a wavefront, its products in fp32: of `keys` keys from k and v on, its probabilities exp(score * scale - lse).
template <typename T>
__device__ __noinline__ WaveRow dq_of_row(const T* q, const T* d_o, const T* k, const T* v, long kv_stride, int keys, int d, float scale, float lse1,
                                          float lse2, float delta1, float delta2, float lambda) {
    const WaveRow query = WaveRow::load(q, d), dout = WaveRow::load(d_o, d);
    WaveRow sum{};
    for (int j = 0; j < keys; ++j) {
        const WaveRow key = WaveRow::load(k + j * kv_stride, d);
        const float g = dout.dot(WaveRow::load(v + j * kv_stride, d));
        const float ds1 = expf(query.dot(key, false, d) * scale - lse1) * (g - delta1), ds2 = expf(query.dot(key, true, d) * scale - lse2) * (g - delta2);
        sum.add(key, ds1, -lambda * ds2, d);
    }
    return sum;
}
// Adds to a row of dk by a wavefront, its products in fp32, what `queries` queries give, `stride` heads apart from q and d_o on, with their four
// statistics `rows` apart.
template <typename T>
__device__ __noinline__ WaveRow dk_of_row(WaveRow sum, WaveRow k, WaveRow v, const T* q, const T* d_o, const float* statistics, long rows, int queries,
                                          int stride, int d, float scale2, float sign) {
    for (int i = 0; i < queries; ++i) {
        const long head = static_cast<long>(i) * stride;
        const float* of_row = statistics + head;
        const WaveRow query = WaveRow::load(q + head * d, d);
        const float g = WaveRow::load(d_o + head * d, d).dot(v) + of_row[2 * rows];  // G - delta1
        const float p1 = __builtin_amdgcn_exp2f(fmaf(query.dot(k, false, d), scale2, -of_row[0]));
        const float p2 = __builtin_amdgcn_exp2f(fmaf(query.dot(k, true, d), scale2, -of_row[rows]));
        sum.add(query, p1 * g, p2 * fmaf(sign, g, of_row[3 * rows]), d);
    }
    return sum;
}

template <typename T, int W, int PARTS>
__global__ __launch_bounds__(kThreads, W == 64 ? 3 : 2) void differential_dq_kernel(DifferentialArgs p) {
    using frag = typename Mma<T>::frag;
    constexpr int STEPS = W / 16, HALF = STEPS / 2, DT = W / 32;
    T* const lds = wide_stages<T, W, PARTS>();  // [stage][part][K | V]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const RowTiles at = RowTiles::of<PARTS>(p, wave);
    const long q_stride = static_cast<long>(p.hq) * p.d, kv_stride = static_cast<long>(p.hkv) * p.d;
    const long q_offset = at.offset(p), first_row = at.wave_live ? ((static_cast<long>(at.b) * p.qs + at.first_q) * p.hq + at.h) * p.d : 0;
    const int row_bytes = ((at.q - at.first_q) * p.hq + at.beside) * p.d * static_cast<int>(sizeof(T));
    const long wave_bytes = at.wave_live ? ((at.last_q - at.first_q + 1) * q_stride - at.h * p.d) * static_cast<long>(sizeof(T)) : 0;
    const long kv_offset = static_cast<long>(at.b) * p.ks * kv_stride + at.kvh * p.d;
    const RowStream k_src = make_stream<T, W, true>(p.k, kv_offset, kv_stride, p.ks, p.d, wave, p.d);
    const RowStream v_src = make_stream<T, W, false>(p.v, kv_offset, kv_stride, p.ks, p.d, wave, p.d);

    const int last_q_block = min(at.row + kBlockRows / PARTS, p.qs) - 1;
    const int k_end = p.causal ? min(p.ks, p.offset + last_q_block + 1) : p.ks;
    const int tiles = (k_end + kStream - 1) / kStream;
    auto request = [&](int j, T* stage) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < PARTS; ++g) {
            if (j + g >= tiles) break;
            stream_rows<T, W>(k_src, (j + g) * kStream, stage + 2 * g * kWideTile<W>, wave);
            stream_rows<T, W>(v_src, (j + g) * kStream, stage + (2 * g + 1) * kWideTile<W>, wave);
        }
    };
    request(0, lds);

    frag qf[STEPS], dof[STEPS];
    load_rows<T, W, true>(qf, p.q, first_row, wave_bytes, row_bytes, at.live, p.d);
    load_rows<T, W, false>(dof, p.dout, first_row, wave_bytes, row_bytes, at.live, p.d);
    const float lambda = p.lambda[at.h];
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq, row = (static_cast<long>(at.b) * p.qs + at.q) * p.hq + at.h;
    float delta1, delta2;
    {
        frag of[STEPS], o2f[STEPS];
        load_rows<T, W, false>(of, p.o, first_row, wave_bytes, row_bytes, at.live, p.d);
        load_rows<T, W, false>(o2f, p.o2, first_row, wave_bytes, row_bytes, at.live, p.d);
        delta2 = row_delta<T, STEPS>(dof, o2f);
        delta1 = fmaf(lambda, delta2, row_delta<T, STEPS>(dof, of));
    }
    float lse1 = at.live ? p.lse[row] * kLog2e : 0.0f, lse2 = at.live ? p.lse[rows + row] * kLog2e : 0.0f;
    int k_off[STEPS], kt_off[DT][2];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) k_off[s] = wide_direct_offset<W>(lane, s);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        kt_off[t][0] = wide_transposed_offset<W>(lane, t, 0);
        kt_off[t][1] = wide_transposed_offset<W>(lane, t, 1);
    }

    acc_t dq[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = acc_t(0.0f);
    float rest = 0.0f;  // rowsum(P2 (G - delta2)): what the rounding of O2 left in delta2
    const long row_part = (static_cast<long>(at.b) * gridDim.x + at.row / (kBlockRows / PARTS)) * (4 / PARTS) + at.row_wave;
    const float scale2 = p.scale * kLog2e;
    const int wave_first_q = at.first_q, wave_last_q = at.last_q;
    const bool wave_live = at.wave_live;
    const int q_limit = p.causal ? p.offset + at.q : p.ks;
    const int clear_limit = p.causal ? min(p.ks - 1, p.offset + wave_first_q) : p.ks - 1;

    // Rows that see few keys: their score gradients are small beside the deltas that they are differences of, so that the rounding of O and
    // O2 in these shows (4 queries of 4 keys, bf16: dQ off by 0.0037 of its norm, 0.0024 with what follows; the first 64 rows of 1001 tokens, more
    // than a third of dQ's norm, fp16: 1.58 times as far off as the rounded exact dQ, 1.43 with it). Where all keys that a wavefront's rows see
    // are in the first tile: rowsum(P (G - delta)) first, which is what delta lacks, then the walk.
    auto few_keys = [&](int last_q) { return tiles == 1 || (p.causal && p.offset + last_q < kStream); };
    if (few_keys(min(at.row + 31, p.qs - 1))) {  // of the workgroup's first wavefront
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's part of the tile is in LDS
        __syncthreads();
    }
    if (few_keys(wave_last_q)) {
        float lack1 = 0.0f, lack2 = 0.0f;
#pragma unroll 1
        for (int first_key = 0; first_key < kStream; first_key += 32) {
            const T* k_rows = lds + first_key * W;
            acc_t st[2] = {acc_t(0.0f), acc_t(0.0f)}, g(0.0f);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                st[s / HALF] = Mma<T>::run(*reinterpret_cast<const frag*>(k_rows + k_off[s]), qf[s], st[s / HALF]);
                g = Mma<T>::run(*reinterpret_cast<const frag*>(k_rows + kWideTile<W> + k_off[s]), dof[s], g);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (first_key + 4 * (lane >> 5) + 8 * (e >> 2) + (e & 3) > min(q_limit, p.ks - 1)) continue;
                lack1 = fmaf(__builtin_amdgcn_exp2f(fmaf(st[0][e], scale2, -lse1)), g[e] - delta1, lack1);
                lack2 = fmaf(__builtin_amdgcn_exp2f(fmaf(st[1][e], scale2, -lse2)), g[e] - delta2, lack2);
            }
        }
        delta1 += lack1 + __shfl_xor(lack1, 32);
        delta2 += lack2 + __shfl_xor(lack2, 32);
    }
    if (at.live && at.part == 0 && lane < 32) {
        // In the form that the dK/dV pass needs fewest instructions for: |lambda| inside the second map's exponent, and its sign, as
        // that of -lambda, on what is left of its score gradient, whose G already has delta1 taken off.
        p.delta[row] = lse1;
        p.delta[rows + row] = lse2 - log2f(fabsf(lambda));
        p.delta[2 * rows + row] = -delta1;
        p.delta[3 * rows + row] = sign_of_second(lambda) * (delta1 - delta2);
    }
    if constexpr (kEnlarged<T>) {
        const float largest = largest_of_row<STEPS>(dof), power = static_cast<float>(enlarging_power(largest, 24));
        const bool finite = (delta1 + delta2 + lse1 + lse2) * 0.0f == 0.0f;  // if not, no sum that the row is in will be: nothing to save
        const float of_wave = wave_max(finite ? largest : INFINITY);
        lse1 -= power;
        lse2 -= power;
        if (lane == 0 && at.part == 0) p.largest[at.h * p.lambda_parts + row_part] = of_wave;
    }
    LeftOut left(p, wave_first_q);
    for (int first = 0; first < tiles; first += PARTS) {
        const int j = first + at.part, k0 = j * kStream, stage = (first / PARTS) & 1;
        const T* k_tile = lds + (stage * PARTS + at.part) * 2 * kWideTile<W>;
        const T* v_tile = k_tile + kWideTile<W>;
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's part of the tiles is in LDS
        __syncthreads();                     // ... and everybody else's; the other stage is free
        request(first + PARTS, lds + (stage ^ 1) * PARTS * 2 * kWideTile<W>);
        if (PARTS > 1 && j >= tiles) continue;
        if (!wave_live || (p.causal && k0 > p.offset + wave_last_q) || left.out<T, W>(j, k_tile)) continue;
        const bool masked = k0 + kStream - 1 > clear_limit;
        const int bound = min(q_limit, p.ks - 1) - k0 - 4 * (lane >> 5);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            acc_t st[2] = {acc_t(0.0f), acc_t(0.0f)}, g(0.0f);
            {
                frag ka[STEPS], va[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    ka[s] = *reinterpret_cast<const frag*>(k_tile + sub * 32 * W + k_off[s]);
                    va[s] = *reinterpret_cast<const frag*>(v_tile + sub * 32 * W + k_off[s]);
                }
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    st[s / HALF] = Mma<T>::run(ka[s], qf[s], st[s / HALF]);
                    g = Mma<T>::run(va[s], dof[s], g);
                }
                sched_reads_under_mfmas<2 * STEPS, 2 * STEPS, 4>();
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                st[0][e] = __builtin_amdgcn_exp2f(fmaf(st[0][e], scale2, -lse1)) * (g[e] - delta1);
                st[1][e] = __builtin_amdgcn_exp2f(fmaf(st[1][e], scale2, -lse2)) * (g[e] - delta2);
            }
            if (masked) {
                asm volatile("" ::: "memory");  // keeps the masking out of the common path (no if-conversion)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool visible = sub * 32 + 8 * (e >> 2) + (e & 3) <= bound;
                    st[0][e] = visible ? st[0][e] : 0.0f;
                    st[1][e] = visible ? st[1][e] : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) rest += st[1][e];
            __builtin_amdgcn_sched_barrier(0);
            {
                frag dsf[2][2], kt[2][DT];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    dsf[0][s] = acc_frag<T>(st[0], s);
                    dsf[1][s] = acc_frag<T>(st[1], s);
                    const T* block = k_tile + (sub * 32 + s * 16) * W;
#pragma unroll
                    for (int t = 0; t < DT; ++t) kt[s][t] = wide_transposed_frag<T>(block, kt_off[t][0], kt_off[t][1]);
                }
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int t = 0; t < DT; ++t) dq[t] = Mma<T>::run(kt[s][t], dsf[t / (DT / 2)][s], dq[t]);
                sched_reads_under_mfmas<2 * DT, 4 * DT, 6>();
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (left.tiles != 0) {
        Parked<DT> sums;
#pragma unroll
        for (int t = 0; t < DT; ++t) sums.put(t, dq[t]);
        const T *q_row = static_cast<const T*>(p.q) + q_offset, *do_row = static_cast<const T*>(p.dout) + q_offset;
        left.each_key(p.ks, [&](int key) {
            if (!at.live || key > q_limit) return;
            const T* k_row = static_cast<const T*>(p.k) + kv_offset + key * kv_stride;
            const float g = row_product(do_row, static_cast<const T*>(p.v) + kv_offset + key * kv_stride, p.d);
            const float s1 = row_product(q_row, k_row, p.d / 2), s2 = row_product(q_row + p.d / 2, k_row + p.d / 2, p.d / 2);
            const float ds1 = __builtin_amdgcn_exp2f(fmaf(s1, scale2, -lse1)) * (g - delta1);
            const float ds2 = __builtin_amdgcn_exp2f(fmaf(s2, scale2, -lse2)) * (g - delta2);
            if (lane < 32) rest += ds2;  // a row's rest is the sum of its two lanes'
#pragma unroll 1
            for (int r = 0; r < DT * 16; ++r) {
                const int column = register_column<W, true>(r, p.d);
                if (column >= 0) sums.values[r] = fmaf(r < DT * 8 ? ds1 : ds2, to_f32(k_row[column]), sums.values[r]);
            }
        });
#pragma unroll
        for (int t = 0; t < DT; ++t) sums.get(t, dq[t]);
    }
    if constexpr (PARTS > 1) {
        auto* meet = reinterpret_cast<vec_t<float, 4>*>(lds) + at.row_wave * (4 * DT + 1) * kWave + lane;
        __syncthreads();
        if (at.part != 0) {
            deposit_sums<DT>(meet, dq);
            meet[4 * DT * kWave] = vec_t<float, 4>{rest, 0.0f, 0.0f, 0.0f};
        }
        __syncthreads();
        if (at.part != 0) return;
        add_sums<DT>(meet, dq, 1.0f, 1.0f);
        rest += meet[4 * DT * kWave][0];
    }
    float smaller = 1.0f;
    bool stored = false;
    if constexpr (kEnlarged<T>) {
        using words = vec_t<unsigned int, 4>;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {  // the power again: it takes no register through the walk
            auto w = __builtin_bit_cast(words, dof[s]);
            asm volatile("" : "+v"(w));
            dof[s] = __builtin_bit_cast(frag, w);
        }
        const int power = enlarging_power(largest_of_row<STEPS>(dof), 24);
        smaller = ldexpf(1.0f, -power);
        rest *= smaller;
        const bool finite = (delta1 + delta2 + lse1 + lse2) * 0.0f == 0.0f;
        const unsigned long long half = __ballot(at.live && power > 0 && finite && any_not_finite(dq));
        for (unsigned int lost = static_cast<unsigned int>(half | half >> 32); lost != 0; lost &= lost - 1) {
            const int from = __builtin_ctz(lost), q = __shfl(at.q, from);
            const long of_row = (static_cast<long>(at.b) * p.qs + q) * p.hq + at.h;
            const WaveRow exact = dq_of_row<T>(static_cast<const T*>(p.q) + of_row * p.d, static_cast<const T*>(p.dout) + of_row * p.d,
                                               static_cast<const T*>(p.k) + kv_offset, static_cast<const T*>(p.v) + kv_offset, kv_stride,
                                               p.causal ? min(p.ks, p.offset + q + 1) : p.ks, p.d, p.scale, p.lse[of_row], p.lse[rows + of_row],
                                               __shfl(delta1, from), __shfl(delta2, from), lambda);
            exact.store(static_cast<T*>(p.dq) + of_row * p.d, p.d, p.gradient_scale, p.accumulate != 0);
            stored = stored || (lane & 31) == from;
        }
    }
    {
        // -(delta2 + rest) of the wavefront's rows.
        const float mine = at.live ? rest + (lane < 32 ? delta2 : 0.0f) : 0.0f;
        const float sum = wave_sum(mine);
        if (lane == 0) p.lambda_partial[at.h * p.lambda_parts + row_part] = -sum;
    }
    if (!at.live || stored) return;
    const float factor[2] = {p.gradient_scale * smaller, -lambda * p.gradient_scale * smaller};
    store_columns<T, W, true>(static_cast<T*>(p.dq) + q_offset, p.d, p.accumulate != 0,
                              [&](int t, int e) { return dq[t][e] * factor[t / (DT / 2)]; });
}

// dK/dV: keys are stationary, 32 per wavefront with their K and V fragments and accumulators in registers; 64-query Q/dO tiles of
// every q-head of the group pass through two LDS stages with their statistics. A tile is 4 N matrix instructions (N = W/8), in slots
// of one with a scheduling fence after each: what else a tile has to do runs in the shadow of instructions that it does not depend
// on, if it stands between them. With H = N/2, halves of 32 queries in brackets:
//   Sᵀ(0) H | Gᵀ(0), Sᵀ(1) by turns 2H | Gᵀ(1), dV(0) by turns 2H | dV(1) H | dK(0) H | dK(1) H
// The exponentials and the packed P1 - lambda P2 of a half run from the end of its scores to its dV, its score gradients from there
// to its dK: two maps' worth take about as long as the matrix instructions (plain attention's half of that), so they are dealt out
// over all slots between.
template <int W>
constexpr int kDkvSmem = 4 * kWideTile<W> * 2 + 8 * kStream * static_cast<int>(sizeof(float));

// Where a 64-query tile comes from and goes to.
template <typename T>
struct QueryTile {
    bool live;
    __amdgpu_buffer_rsrc_t q, dout, stat;
    T* stage;
    float* stat_stage;
};

enum class Product { scores, grads, values, keys };
struct Slot {
    Product product;
    int half, index;
};
constexpr Slot dkv_slot(int k, int h) {
    if (k < h) return {Product::scores, 0, k};
    if (k < 3 * h) return (k - h) % 2 == 0 ? Slot{Product::grads, 0, (k - h) / 2} : Slot{Product::scores, 1, (k - h) / 2};
    if (k < 5 * h) return (k - h) % 2 == 0 ? Slot{Product::grads, 1, (k - 3 * h) / 2} : Slot{Product::values, 0, (k - 3 * h) / 2};
    if (k < 6 * h) return {Product::values, 1, k - 5 * h};
    if (k < 7 * h) return {Product::keys, 0, k - 6 * h};
    return {Product::keys, 1, k - 7 * h};
}
// Slot in which step n of 8 of a half's exponentials (or score gradients) runs.
constexpr int exponential_slot(int half, int n, int h) { return (half == 0 ? h + 2 : 3 * h + 2) + n * (2 * h - 2) / 8; }
constexpr int gradient_slot(int half, int n, int h) { return (half == 0 ? 4 * h + h / 2 : 6 * h - h / 4) + n * (half == 0 ? 3 * h / 2 : 5 * h / 4) / 8; }

// The power for dk of a (batch entry, kv head): by the largest |dO| that the dQ pass found, and so that P1 + |lambda| P2 stays in range.
// Every wavefront works it out by itself.
__device__ __forceinline__ int enlargement(const DifferentialArgs& p, int b, int kvh, float scale2) {
    const int lane = threadIdx.x & 63, group = p.hq / p.hkv, per_head = static_cast<int>(p.lambda_parts / p.batch);
    const float* from = p.largest + static_cast<long>(kvh) * group * p.lambda_parts + static_cast<long>(b) * per_head;
    float largest = 0.0f, weight = 0.0f;
    for (int i = lane; i < group * per_head; i += kWave) {
        const int head = i / per_head;
        largest = fmaxf(largest, from[head * p.lambda_parts + (i - head * per_head)]);
    }
    for (int head = lane; head < group; head += kWave) weight = fmaxf(weight, fabsf(p.lambda[kvh * group + head]));
    const int most = 14 - (static_cast<int>(__float_as_uint(1.0f + wave_max(weight)) >> 23) - 127);
    const int power = scale2 > 0x1p-60f ? enlarging_power(wave_max(largest), most) : 0;
    return __builtin_amdgcn_readfirstlane(power);
}

template <typename T, int W>
__global__ __launch_bounds__(kThreads, 1) void differential_dkv_kernel(DifferentialArgs p) {
    using frag = typename Mma<T>::frag;
    constexpr int STEPS = W / 16, HALF = STEPS / 2, DT = W / 32;
    extern __shared__ __align__(1024) unsigned char wide_smem[];
    T* lds = reinterpret_cast<T*>(wide_smem);                                           // [stage][Q | dO]
    float* stats = reinterpret_cast<float*>(wide_smem + 4 * kWideTile<W> * sizeof(T));  // [stage][the dQ pass's four][64]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroup -> (key block or pair of them, kv head, batch entry), as in attention.hip's dK/dV: the owners of an XCD's workgroups
    // stream the same Q and dO.
    int block = static_cast<int>(blockIdx.x), b = static_cast<int>(blockIdx.z), kvh = static_cast<int>(blockIdx.y);
    {
        constexpr unsigned int kXcds = 8;
        const unsigned int linear = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
        const unsigned int owners = gridDim.y * gridDim.z;
        const unsigned int xcds = owners % kXcds == 0 ? kXcds : 1;
        if (xcds > 1 || p.by_block) {
            const unsigned int xcd = linear % xcds, local = linear / xcds, mine = owners / xcds;
            const unsigned int owner = xcd + xcds * (p.by_block ? local % mine : local / gridDim.x);
            block = static_cast<int>(p.by_block ? local / mine : local % gridDim.x);
            kvh = static_cast<int>(owner % gridDim.y);
            b = static_cast<int>(owner / gridDim.y);
        }
    }
    const int group = p.hq / p.hkv;
    const long q_stride = static_cast<long>(p.hq) * p.d, kv_stride = static_cast<long>(p.hkv) * p.d;
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq;
    const float scale2 = p.scale * kLog2e;
    const long q_batch = static_cast<long>(b) * p.qs * q_stride + kvh * group * p.d;
    const RowStream q_src = make_stream<T, W, true>(p.q, q_batch, q_stride, p.qs, p.d, wave, p.d);
    const RowStream do_src = make_stream<T, W, false>(p.dout, q_batch, q_stride, p.qs, p.d, wave, p.d);
    const TileOffsets<W> offsets(lane);

    const int key_blocks = (p.ks + kBlockRows - 1) / kBlockRows;
    const int part = p.splits > 1 ? block % p.splits : 0;
    if (p.splits > 1) block /= p.splits;
    int power = 0;  // score gradients and probabilities are 2^power as large
    if constexpr (kEnlarged<T>) power = enlargement(p, b, kvh, scale2);
    const float score0 = static_cast<float>(power) / scale2;  // where scores start
    const float smaller = ldexpf(1.0f, -power), k_factor = p.gradient_scale * smaller;
    for (int turn = 0; turn < (p.paired ? 2 : 1); ++turn) {
        const int block_index = turn == 0 ? block : key_blocks - 1 - block;
        if (turn == 1 && block_index <= block) break;
        const int k_block = block_index * kBlockRows;
        const int k_row = k_block + wave * 32 + (lane & 31);
        // A key that no query sees is zeros here, whatever its rows hold: its hidden probabilities are factors of G, and the zeros of
        // queries past the end factors of both.
        const bool k_live = k_row < p.ks, k_seen = k_live && (!p.causal || k_row - p.offset < p.qs);
        const long k_head = static_cast<long>(b) * p.ks * kv_stride + kvh * p.d, k_offset = k_head + k_row * kv_stride;
        frag kf[STEPS], vf[STEPS];
        const int first_key = k_block + wave * 32, key_bytes = (lane & 31) * static_cast<int>(kv_stride * sizeof(T));
        const long wave_bytes = first_key < p.ks ? ((min(p.ks - first_key, 32) - 1) * kv_stride + p.d) * static_cast<long>(sizeof(T)) : 0;
        const long first_row = first_key < p.ks ? k_head + first_key * kv_stride : 0;
        load_rows<T, W, true>(kf, p.k, first_row, wave_bytes, key_bytes, k_seen, p.d);
        load_rows<T, W, false>(vf, p.v, first_row, wave_bytes, key_bytes, k_seen, p.d);
        acc_t dk[DT], dv[DT];
#pragma unroll
        for (int t = 0; t < DT; ++t) dk[t] = dv[t] = acc_t(0.0f);
        // First query tile that sees a key of this block; the (head of the group, query tile) pairs form one sequence.
        const int q_begin = p.causal ? max(0, k_block - p.offset) / kStream * kStream : 0;
        const int tiles_per_head = q_begin < p.qs ? (p.qs - q_begin + kStream - 1) / kStream : 0;
        const long all_tiles = static_cast<long>(tiles_per_head) * group;
        const int first_index = p.splits > 1 ? static_cast<int>(part * all_tiles / p.splits) : 0;
        const int total_tiles = static_cast<int>(p.splits > 1 ? (part + 1) * all_tiles / p.splits : all_tiles);  // end of the part
        const int wave_last_key = k_block + wave * 32 + 31;

        constexpr int kRowsPerLoad = 64 / (W / 8), kLoads = kStream / (4 * kRowsPerLoad);
        using NextTile = QueryTile<T>;
        auto next_tile = [&](int tile) {
            NextTile n;
            n.live = tile < total_tiles;
            const int head = min(tile / max(tiles_per_head, 1), group - 1);
            const int q0 = q_begin + (tile - head * tiles_per_head) * kStream;
            RowStream of_head = q_src;
            of_head.base += head * p.d * static_cast<int>(sizeof(T));
            n.q = of_head.at(n.live ? q0 : 0);
            of_head = do_src;
            of_head.base += head * p.d * static_cast<int>(sizeof(T));
            n.dout = of_head.at(n.live ? q0 : 0);
            // One float per query and statistic: wavefront w brings statistic w.
            const float* from = p.delta + wave * rows + (static_cast<long>(b) * p.qs + q0) * p.hq + kvh * group + head;
            const long left = ((static_cast<long>(p.qs) - 1 - q0) * p.hq + 1) * static_cast<long>(sizeof(float));
            n.stat = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), 0, static_cast<int>(min(left, 1l << 30)), 0x00020000);
            n.stage = lds + (tile & 1) * 2 * kWideTile<W>;
            n.stat_stage = stats + ((tile & 1) * 4 + wave) * kStream;
            return n;
        };
        const int stat_voffset = lane * p.hq * static_cast<int>(sizeof(float));
        auto request_part = [&](const NextTile& n, int i) {
            if (!n.live) return;
            if (i < kLoads) {
                const int soffset = i * 4 * kRowsPerLoad * q_src.row_bytes;
                T* to = n.stage + (i * 4 + wave) * kRowsPerLoad * W;
                load_chunks(n.q, to, q_src.voffset, soffset);
                load_chunks(n.dout, to + kWideTile<W>, do_src.voffset, soffset);
            } else if (i == kLoads) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(n.stat, (lds_void_ptr)(n.stat_stage), 4, stat_voffset, 0, 0, 0);
            }
        };

        // MASKED: some (query, key) pairs of this wavefront are hidden (causal mask, keys past the end); first = first visible register
        // coordinate for this lane's key. Queries past the end need nothing: their dO rows, delta and lse are zeros.
        auto tile_body = [&]<bool MASKED>(int stage, float sign, int first, const NextTile& next) {
            constexpr int H = W / 16, kSlots = 8 * H, kLookAhead = W == 64 ? 2 : 6;
            if constexpr (W == 128) {
                using words = vec_t<unsigned int, 4>;
                // K and V are operands only: in the accumulation registers, where the matrix instructions read them as they are. Left to
                // the compiler they were copied out in every tile, some 60 of its 860 instructions.
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    auto k_words = __builtin_bit_cast(words, kf[i]), v_words = __builtin_bit_cast(words, vf[i]);
                    asm volatile("" : "+a"(k_words), "+a"(v_words));
                    kf[i] = __builtin_bit_cast(frag, k_words);
                    vf[i] = __builtin_bit_cast(frag, v_words);
                }
            }
            const TileOffsets<W> here = offsets.at(stage * 2 * kWideTile<W>);
            const float* stat = stats + stage * 4 * kStream + 4 * (lane >> 5);
            acc_t s_acc[2][2], g_acc[2];                              // [half][map]
            vec_t<unsigned int, 4> p_words[2][2], ds_words[2][2][2];  // [half][16-query step], [half][map][step]: k-operands of dV, dK
            vec_t<float, 4> lse_q[2][4][2], delta_q[2][4];
            frag operand[kSlots];
            auto read_operand = [&]<int K>() {
                constexpr Slot at = dkv_slot(K, H);
                if constexpr (at.product == Product::scores) operand[K] = here.row(lds, at.half * 32, at.index % 2 * HALF + at.index / 2);
                else if constexpr (at.product == Product::grads) operand[K] = here.row(lds, kStream + at.half * 32, at.index);
                else operand[K] = here.columns(lds, (at.product == Product::values ? kStream : 0) + at.half * 32 + at.index / DT * 16, at.index % DT);
            };
            auto multiply = [&]<int K>() {
                constexpr Slot at = dkv_slot(K, H);
                if constexpr (at.product == Product::scores) {
                    constexpr int map = at.index % 2, s = at.index / 2;
                    s_acc[at.half][map] = Mma<T>::run(operand[K], kf[map * HALF + s], s == 0 ? acc_t(kEnlarged<T> ? score0 : 0.0f) : s_acc[at.half][map]);
                } else if constexpr (at.product == Product::grads) {
                    g_acc[at.half] = Mma<T>::run(operand[K], vf[at.index], g_acc[at.half]);  // from -delta1 on
                } else {
                    constexpr int s = at.index / DT, t = at.index % DT;
                    if constexpr (at.product == Product::values) dv[t] = Mma<T>::run(operand[K], __builtin_bit_cast(frag, p_words[at.half][s]), dv[t]);
                    else dk[t] = Mma<T>::run(operand[K], __builtin_bit_cast(frag, ds_words[at.half][t / (DT / 2)][s]), dk[t]);
                }
            };
            // Statistics of steps N and N + 1 (N even), read a few slots ahead of them: KIND 0 both lse, 1 -delta1 (where G's sums
            // start), 2 what the second map's score gradient differs by.
            auto read_statistics = [&]<int HALF_TILE, int N, int KIND>() {
                auto read = [&](int which) { return *reinterpret_cast<const vec_t<float, 4>*>(stat + which * kStream + HALF_TILE * 32 + 4 * N); };
                if constexpr (KIND == 0) {
                    lse_q[HALF_TILE][N / 2][0] = read(0);
                    lse_q[HALF_TILE][N / 2][1] = read(1);
                } else if constexpr (KIND == 1) {
                    const vec_t<float, 4> v = read(2);
#pragma unroll
                    for (int e = 0; e < 4; ++e) g_acc[HALF_TILE][2 * N + e] = v[e];
                } else {
                    delta_q[HALF_TILE][N / 2] = read(3);
                }
            };
            // Step N of 8 of a half: scores 2 N and 2 N + 1.
            auto exponentials = [&]<int HALF_TILE, int N>() {
                vec_t<float, 2> map;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    constexpr int i0 = 2 * N;
                    float p1 = __builtin_amdgcn_exp2f(fmaf(s_acc[HALF_TILE][0][i0 + e], scale2, -lse_q[HALF_TILE][N / 2][0][(i0 & 3) + e]));
                    float p2 = __builtin_amdgcn_exp2f(fmaf(s_acc[HALF_TILE][1][i0 + e], scale2, -lse_q[HALF_TILE][N / 2][1][(i0 & 3) + e]));
                    if constexpr (MASKED) {
                        const bool visible = HALF_TILE * 32 + 8 * (i0 >> 2) + (i0 & 3) + e >= first;
                        p1 = visible ? p1 : 0.0f;
                        p2 = visible ? p2 : 0.0f;
                    }
                    s_acc[HALF_TILE][0][i0 + e] = p1;
                    s_acc[HALF_TILE][1][i0 + e] = p2;
                    map[e] = fmaf(sign, p2, p1);
                }
                p_words[HALF_TILE][N / 4][N % 4] = __builtin_bit_cast(unsigned int, vec_from_f32<T, 2>(map));
            };
            auto gradients = [&]<int HALF_TILE, int N>() {
                vec_t<float, 2> first_map, second_map;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float g = g_acc[HALF_TILE][2 * N + e];  // G - delta1
                    first_map[e] = s_acc[HALF_TILE][0][2 * N + e] * g;
                    second_map[e] = s_acc[HALF_TILE][1][2 * N + e] * fmaf(sign, g, delta_q[HALF_TILE][N / 2][(2 * N & 3) + e]);
                }
                ds_words[HALF_TILE][0][N / 4][N % 4] = __builtin_bit_cast(unsigned int, vec_from_f32<T, 2>(first_map));
                ds_words[HALF_TILE][1][N / 4][N % 4] = __builtin_bit_cast(unsigned int, vec_from_f32<T, 2>(second_map));
            };
            auto beside = [&]<int K, int N>() {
                if constexpr (N % 2 == 0) {
                    constexpr int kAhead = W == 64 ? 1 : 3;
                    if constexpr (exponential_slot(0, N, H) - kAhead == K) read_statistics.template operator()<0, N, 0>();
                    if constexpr (exponential_slot(1, N, H) - kAhead == K) read_statistics.template operator()<1, N, 0>();
                    if constexpr (H - kAhead == K) read_statistics.template operator()<0, N, 1>();
                    if constexpr (3 * H - kAhead == K) read_statistics.template operator()<1, N, 1>();
                    if constexpr (gradient_slot(0, N, H) - kAhead == K) read_statistics.template operator()<0, N, 2>();
                    if constexpr (gradient_slot(1, N, H) - kAhead == K) read_statistics.template operator()<1, N, 2>();
                }
                if constexpr (exponential_slot(0, N, H) == K) exponentials.template operator()<0, N>();
                if constexpr (exponential_slot(1, N, H) == K) exponentials.template operator()<1, N>();
                if constexpr (gradient_slot(0, N, H) == K) gradients.template operator()<0, N>();
                if constexpr (gradient_slot(1, N, H) == K) gradients.template operator()<1, N>();
            };
            auto slot = [&]<int K>() {
                if constexpr (K + kLookAhead < kSlots) read_operand.template operator()<K + kLookAhead>();
                multiply.template operator()<K>();
                if constexpr (K <= kLoads) request_part(next, K);
                [&]<int... N>(std::integer_sequence<int, N...>) { (beside.template operator()<K, N>(), ...); }(std::make_integer_sequence<int, 8>{});
                __builtin_amdgcn_sched_barrier(0);
            };
            [&]<int... K>(std::integer_sequence<int, K...>) {
                (read_operand.template operator()<K>(), ...);
            }(std::make_integer_sequence<int, kLookAhead>{});
            __builtin_amdgcn_sched_barrier(0);
            [&]<int... K>(std::integer_sequence<int, K...>) { (slot.template operator()<K>(), ...); }(std::make_integer_sequence<int, kSlots>{});
        };

        // Every wavefront runs every tile; per head the tiles that need the mask come first: two loops with one straight-line body each.
        int masked_per_head = 0;
        if (wave_last_key >= p.ks) masked_per_head = tiles_per_head;
        else if (p.causal) masked_per_head = min(tiles_per_head, max(0, (wave_last_key - p.offset - q_begin + kStream - 1) / kStream));
        auto arrive = [&]() {
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's part of the tile is in LDS
            __syncthreads();                     // ... and everybody else's; the other stage is free
        };
        {
            const NextTile first_tile = next_tile(first_index);
#pragma unroll
            for (int i = 0; i <= kLoads; ++i) request_part(first_tile, i);
        }
        for (int head = 0; head < group; ++head) {
            const int tile0 = head * tiles_per_head;
            const int begin = max(0, first_index - tile0), end = min(tiles_per_head, total_tiles - tile0);
            if (begin >= end) continue;
            const float sign = sign_of_second(p.lambda[kvh * group + head]);
            for (int t = begin; t < min(masked_per_head, end); ++t) {
                const int tile = tile0 + t, q0 = q_begin + t * kStream;
                arrive();
                const int causal_first = p.causal ? k_row - p.offset - q0 - 4 * (lane >> 5) : -(1 << 30);
                tile_body.template operator()<true>(tile & 1, sign, k_live ? causal_first : (1 << 30), next_tile(tile + 1));
            }
            for (int t = max(masked_per_head, begin); t < end; ++t) {
                arrive();
                tile_body.template operator()<false>((tile0 + t) & 1, sign, 0, next_tile(tile0 + t + 1));
            }
        }
        __syncthreads();  // the next key block's first loads overwrite stage 0
        const long count = static_cast<long>(p.batch) * p.ks * kv_stride;
        float* const part_dk = p.splits > 1 ? p.partial + 2 * part * count : nullptr;
        bool stored = false;  // dk
        if constexpr (kEnlarged<T>) {
            const unsigned long long half = __ballot(k_seen && power > 0 && any_not_finite(dk));
            for (unsigned int lost = static_cast<unsigned int>(half | half >> 32); lost != 0; lost &= lost - 1) {
                const int from = __builtin_ctz(lost), key = k_block + wave * 32 + from;
                const long of_key = k_head + key * kv_stride;
                const WaveRow k = WaveRow::load(static_cast<const T*>(p.k) + of_key, p.d), v = WaveRow::load(static_cast<const T*>(p.v) + of_key, p.d);
                if (!k.finite() || !v.finite()) continue;
                WaveRow exact{};
                for (int tile = first_index; tile < total_tiles; ++tile) {
                    const int head = kvh * group + tile / tiles_per_head, q0 = q_begin + tile % tiles_per_head * kStream;
                    const int first = p.causal ? max(q0, key - p.offset) : q0, end = min(q0 + kStream, p.qs);
                    const long row = (static_cast<long>(b) * p.qs + first) * p.hq + head;
                    exact = dk_of_row<T>(exact, k, v, static_cast<const T*>(p.q) + row * p.d, static_cast<const T*>(p.dout) + row * p.d, p.delta + row,
                                         rows, end - first, p.hq, p.d, scale2, sign_of_second(p.lambda[head]));
                }
                if (part_dk != nullptr) exact.store(part_dk + of_key, p.d, p.gradient_scale, false);
                else exact.store(static_cast<T*>(p.dk) + of_key, p.d, p.gradient_scale, p.accumulate != 0);
                stored = stored || (lane & 31) == from;
            }
        }
        if (!k_live) continue;
        if (p.splits > 1) {
            float* to = part_dk + k_offset;
            if (!stored) store_columns<float, W, true>(to, p.d, false, [&](int t, int e) { return dk[t][e] * k_factor; });
            store_columns<float, W, false>(to + count, p.d, false, [&](int t, int e) { return dv[t][e] * smaller; });
        } else {
            if (!stored) store_columns<T, W, true>(static_cast<T*>(p.dk) + k_offset, p.d, p.accumulate != 0, [&](int t, int e) { return dk[t][e] * k_factor; });
            store_columns<T, W, false>(static_cast<T*>(p.dv) + k_offset, p.d, p.accumulate != 0, [&](int t, int e) { return dv[t][e] * smaller; });
        }
    }
    add_lambda_parts<kThreads>(p, reinterpret_cast<double*>(wide_smem));
}

template <typename Fn>
int dispatch(const DifferentialArgs& a, Fn&& fn) {
    const bool narrow = a.d <= 64;
    if (a.dtype == CGPTX_F16) return narrow ? fn.template operator()<f16_t, 64>() : fn.template operator()<f16_t, 128>();
    return narrow ? fn.template operator()<bf16_t, 64>() : fn.template operator()<bf16_t, 128>();
}

// Whether forward and dQ run in two parts: blocks of 64 rows that all find a place on the chip at once (two per CU with heads of 64),
// and more than one key tile. Where the longest block of 128 rows walks many tiles while others are done early (a causal mask), or
// blocks of 64 rows find places beside each other, twice as many: 2 x 2048 tokens of 8 heads of 128, causal, forward 80 -> 61 us, backward 134
// -> 123; 1 x 4096 of 12 heads of 64 88 -> 71 and 197 -> 177. Blocks of equal length on 128-wide heads lose by it (78 -> 100), as do walks of up
// to 16 tiles (8 x 512 tokens of 12 heads of 64 19 -> 21) and, nearly always, more blocks (4 x 2048 of 8 heads of 128 84 -> 116).
bool two_parts(const DifferentialArgs& a) {
    const long blocks = (static_cast<long>(a.qs) + kBlockRows / 2 - 1) / (kBlockRows / 2) * a.hq * a.batch;
    const bool narrow = a.d <= 64, uneven = a.causal && a.offset <= a.qs, long_walk = a.ks >= 24 * kStream;
    return a.ks > kStream && blocks <= static_cast<long>(compute_units()) * (narrow ? 2 : 1) * (long_walk && (uneven || narrow) ? 2 : 1);
}
template <auto Kernel, int W, int PARTS, bool SPLIT = false>
int launch_rows(const DifferentialArgs& a, hipStream_t stream) {
    constexpr int smem = PARTS == 1 ? 0 : 8 * kWideTile<W> * 2;  // [stage][part][K | V] of 16-bit elements
    if constexpr (PARTS > 1) {
        static const hipError_t status =
            hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
        CGPTX_HIP(status);
    }
    const long rows = static_cast<long>(a.qs) * (SPLIT ? a.pack : 1);
    const dim3 grid(static_cast<unsigned int>((rows + kBlockRows / PARTS - 1) / (kBlockRows / PARTS) * (SPLIT ? a.splits : 1)),
                    static_cast<unsigned int>(a.hq / (SPLIT ? a.pack : 1)), static_cast<unsigned int>(a.batch));
    hipLaunchKernelGGL(Kernel, grid, dim3(kThreads), smem, stream, a);
    CGPTX_LAUNCH_CHECK();
    return CGPTX_OK;
}

long key_values(const DifferentialArgs& a) { return static_cast<long>(a.batch) * a.ks * a.hkv * a.d; }

template <typename T, int W>
int launch_dkv(DifferentialArgs a, hipStream_t stream) {
    const auto kernel = differential_dkv_kernel<T, W>;
    static const hipError_t status =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kDkvSmem<W>);
    CGPTX_HIP(status);
    const unsigned int key_blocks = static_cast<unsigned int>((a.ks + kBlockRows - 1) / kBlockRows);
    const std::size_t blocks = static_cast<std::size_t>(key_blocks) * a.hkv * a.batch;
    // Under a causal mask key blocks (i, last - i) together are as long as any other two; where the single blocks do not fill the chip
    // their longest is shorter than a pair.
    a.paired = a.splits == 1 && a.causal && blocks > static_cast<std::size_t>(compute_units());
    a.by_block = a.splits > 1 && key_blocks * static_cast<unsigned int>(a.splits) < static_cast<unsigned int>(compute_units());
    const dim3 grid(a.paired ? (key_blocks + 1) / 2 : key_blocks * static_cast<unsigned int>(a.splits), static_cast<unsigned int>(a.hkv),
                    static_cast<unsigned int>(a.batch));
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), kDkvSmem<W>, stream, a);
    CGPTX_LAUNCH_CHECK();
    return a.splits > 1 ? launch_dkv_reduce<T>(key_values(a), a.dk, a.dv, a.partial, a.splits, a.accumulate, stream) : CGPTX_OK;
}

// Row wavefronts of a dQ launch per head: the parts of a head's dlambda.
long lambda_parts(const DifferentialArgs& a) {
    const int block = two_parts(a) ? kBlockRows / 2 : kBlockRows;
    return (static_cast<long>(a.qs) + block - 1) / block * (block / 32) * a.batch;
}

}  // namespace

bool differential_mfma_takes(const DifferentialArgs& a) { return a.dtype != CGPTX_F32 && a.d % 16 == 0; }

// Workgroups that share a query block's keys in the forward pass: as many as find a place on the chip beside each other, of four tiles
// or more, if that is predicted to take less time: sharing costs a launch and the sums' way to memory and back. Few queries of many keys
// (a token at a time against a long sequence) leave most of the chip idle otherwise: one query of 8:2 heads of 128, bf16, on 8192 keys
// 164 -> 16 us, on 131072 2694 -> 54.
int forward_splits(const DifferentialArgs& a) {
    if (!two_parts(a)) return 1;
    const long blocks = (static_cast<long>(a.qs) * a.pack + kBlockRows / 2 - 1) / (kBlockRows / 2) * (a.hq / a.pack) * a.batch;
    const long keys = a.causal ? std::min<long>(a.ks, static_cast<long>(a.offset) + a.qs) : a.ks, tiles = (keys + kStream - 1) / kStream;
    const long most = std::min<long>({static_cast<long>(compute_units()) * (a.d <= 64 ? 2 : 1) / blocks, tiles / 4, kMostSplits});
    const double pair_us = a.d <= 64 ? 1.4 : 2.2;  // two tiles, one in either part of a workgroup
    const double megabytes = static_cast<double>(a.batch) * a.qs * a.hq * a.d * 16e-6;  // both maps' sums of a part, there and back
    long best = 1;
    double best_us = 0.0;
    for (long splits = 1; splits <= most; ++splits) {
        const double us = static_cast<double>((tiles + 2 * splits - 1) / (2 * splits)) * pair_us + (splits > 1 ? 5.0 + 0.4 * megabytes * splits : 0.0);
        if (splits == 1 || us < best_us) {
            best = splits;
            best_us = us;
        }
    }
    return static_cast<int>(best);
}

int differential_mfma_forward(DifferentialArgs a, hipStream_t stream) {
    const std::size_t rows = static_cast<std::size_t>(a.batch) * a.qs * a.hq, part = 2 * rows * (a.d + 2) * sizeof(float);
    const int group = a.hq / a.hkv;
    a.pack = static_cast<long>(a.qs) * group <= kBlockRows / 2 ? group : 1;  // one block has a whole group's rows
    a.splits = forward_splits(a);
    if (a.splits > 1) {  // an arena that cannot grow has room for fewer
        void* memory = nullptr;
        std::size_t held = 0;
        if (int st = scratch_up_to(stream, a.splits * part, &memory, &held)) return st;
        a.splits = static_cast<int>(std::min<std::size_t>(a.splits, held / part));
        a.partial = static_cast<float*>(memory);
        a.delta = a.partial + 2 * rows * a.d * static_cast<std::size_t>(std::max(a.splits, 0));
    }
    return dispatch(a, [&]<typename T, int W>() -> int {
        if (a.splits > 1) {
            if (int st = launch_rows<differential_forward_kernel<T, W, 2, true>, W, 2, true>(a, stream)) return st;
            auto combine = a.splits <= 8 ? differential_combine_kernel<T, 8> : differential_combine_kernel<T, kMostSplits>;
            hipLaunchKernelGGL(combine, dim3(static_cast<unsigned int>(rows)), dim3(kThreads), 0, stream, a);
            CGPTX_LAUNCH_CHECK();
            return CGPTX_OK;
        }
        return two_parts(a) ? launch_rows<differential_forward_kernel<T, W, 2, false>, W, 2>(a, stream)
                            : launch_rows<differential_forward_kernel<T, W, 1, false>, W, 1>(a, stream);
    });
}

int differential_mfma_backward(DifferentialArgs a, hipStream_t stream) {
    KeyWalk walk = key_walk(a);
    walk.block_rows = kBlockRows;
    walk.stream_rows = kStream;
    walk.waves = 1;
    walk.tile_us = a.d <= 64 ? 1.2 : 2.0;
    if (int st = differential_backward_scratch(a, 4, lambda_parts(a), launchable_parts(walk, kThreads), stream)) return st;
    return dispatch(a, [&]<typename T, int W>() -> int {
        if (int st = two_parts(a) ? launch_rows<differential_dq_kernel<T, W, 2>, W, 2>(a, stream)
                                  : launch_rows<differential_dq_kernel<T, W, 1>, W, 1>(a, stream))
            return st;
        return launch_dkv<T, W>(a, stream);
    });
}

}  // namespace cgptx
