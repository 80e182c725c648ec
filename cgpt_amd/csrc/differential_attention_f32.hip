// Differential attention, fp32 storage and arithmetic, on v_mfma_f32_16x16x4_f32 (formulas: differential_attention.hip; the scheme is
// that of attention_f32.hip: 16 stationary rows per workgroup, the streamed tiles of 16 split between its eight wavefronts, score
// registers that are the second product's operand as they are, partial results that meet in LDS in wavefront order).
//
// 4 x 512 tokens of 8:2 heads of 128: forward 102 us (3.2 GFLOP, 32 TFLOP/s of 154), backward 232. A tile comes from the caches once
// for 16 stationary rows, and that it is waited for bounds it; read with a branch around each load, and with the columns of the rows behind the
// walk held in registers through it, the same took 112 and 317.
//
// Rows of q and k are kept as two halves of D/2 columns, padded with zeros from d/2, so that a map's scores are the product over its
// chunks, and a result block of dq or dk belongs to one map. V, dO and their products are shared by the maps. A row touches no row
// that the causal mask hides from it: see left_out.
#include "attention_tiles.hpp"
#include "differential_attention.hpp"

#include <algorithm>

namespace cgptx {
namespace {

constexpr int kWaves = 8;
constexpr int kF32Threads = kWaves * kWave;
constexpr int kTile = 16;  // stationary rows of a workgroup, streamed rows of a step

using quad = vec_t<float, 4>;
using pair = vec_t<float, 2>;

__device__ __forceinline__ quad mfma(float a, float b, quad c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Column of the tensor's row that padded column c holds, or -1. HALVES: two halves of D/2 (q, k), else one row (v, o).
template <int D, bool HALVES>
__device__ __forceinline__ int source(int c, int d) {
    if constexpr (HALVES) {
        const int half = c / (D / 2), within = c % (D / 2);
        return within < d / 2 ? half * (d / 2) + within : -1;
    } else {
        return c < d ? c : -1;
    }
}

// Rows row0 .. row0 + 15 of a head, of which those below `limit` exist, as a buffer: what lies outside it, like kNowhere, is read as
// zero, without a branch around each load. The arguments are the same in all lanes.
struct TileRows {
    __amdgpu_buffer_rsrc_t rsrc;
    int row_bytes;
    static constexpr int kNowhere = 1 << 30;  // 16 rows of 65535 heads of 128 end before it
    __device__ __forceinline__ TileRows(const float* head, long row_stride, int row0, int limit, int d) {
        const int rows = min(limit - row0, kTile);
        const float* first = head + (rows > 0 ? row0 * row_stride : 0);
        row_bytes = static_cast<int>(row_stride) * 4;
        rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(first), 0, rows > 0 ? (rows - 1) * row_bytes + d * 4 : 0, 0x00020000);
    }
    __device__ __forceinline__ quad four(int row, int column) const {
        const int at = column >= 0 ? row * row_bytes + column * 4 : kNowhere;
        return __builtin_bit_cast(quad, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
    }
    __device__ __forceinline__ pair two(int row, int column) const {
        const int at = column >= 0 ? row * row_bytes + column * 4 : kNowhere;
        return __builtin_bit_cast(pair, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, 0));
    }
};

// A tile as an operand that is contracted over the head dimension: lane l holds row l % 16's padded columns 16 c + 4 (l / 16) .. + 3
// of chunk c. Rows that do not exist are zeros.
template <int D, bool HALVES>
struct RowOperand {
    quad chunk[D / 16];
    __device__ __forceinline__ void load(const TileRows& tile, int d) {
        const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) chunk[c] = tile.four(lane & 15, source<D, HALVES>(16 * c + (lane >> 4) * 4, d));
    }
};
template <int FROM, int TO, int D, bool HALVES>
__device__ __forceinline__ quad product(const RowOperand<D, HALVES>& a, const RowOperand<D, HALVES>& b) {
    quad sum[2] = {quad(0.0f), quad(0.0f)};  // two chains: consecutive MFMAs do not wait for each other
#pragma unroll
    for (int c = FROM; c < TO; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e & 1] = mfma(a.chunk[c][e], b.chunk[c][e], sum[e & 1]);
    return sum[0] + sum[1];
}

// Element of a padded row that result block (b, e), row m of 16, holds, and the map that it belongs to with HALVES. Blocks of 64
// columns; where both halves share one, a lane's four are two of either.
template <int D, bool HALVES>
__device__ __forceinline__ constexpr int padded_column(int b, int e, int m) {
    return HALVES && D == 64 ? (e >> 1) * 32 + 2 * m + (e & 1) : 64 * b + 4 * m + e;
}
template <int D>
__device__ __forceinline__ constexpr int map_of(int b, int e) {
    return D == 64 ? e >> 1 : b;
}

// Rows of a tile as the operand of a product over the rows: lane l holds, for each r, the columns (b, 0 .. 3, l % 16) of row
// 4 (l / 16) + r.
template <int D, bool HALVES>
struct ColumnOperand {
    quad part[4][D / 64];
    __device__ __forceinline__ void load(const TileRows& tile, int d) {
        const int lane = threadIdx.x & (kWave - 1), m = lane & 15;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
                const int row = 4 * (lane >> 4) + r, first = source<D, HALVES>(padded_column<D, HALVES>(b, 0, m), d);
                if constexpr (HALVES && D == 64) {
                    const pair x = tile.two(row, first), y = tile.two(row, source<D, HALVES>(padded_column<D, HALVES>(b, 2, m), d));
                    part[r][b] = quad{x[0], x[1], y[0], y[1]};
                } else {
                    part[r][b] = tile.four(row, first);
                }
            }
    }
};
template <int D>
using Result = quad[D / 64][4];
// result += rows^T x values, by the map of a result's block with HALVES (else values[0] for all).
template <int D, bool HALVES>
__device__ __forceinline__ void accumulate(Result<D>& result, const ColumnOperand<D, HALVES>& rows, const quad& first, const quad& second) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                result[b][e] = mfma(rows.part[r][b][e], HALVES && map_of<D>(b, e) == 1 ? second[r] : first[r], result[b][e]);
}
// Whether the tile holds an Inf or a NaN (the same answer in all lanes): 0 x is 0 for every other x. A tile on the causal diagonal has
// rows that some stationary rows do not see; their values are 0, and 0 x Inf is NaN. Such a tile with such a row is left out of the
// walk and added row by row behind it.
template <int D, bool HALVES>
__device__ __forceinline__ bool non_finite(const ColumnOperand<D, HALVES>& rows) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fmaf(rows.part[r][b][e], 0.0f, sum);
    return __ballot(!(sum == 0.0f)) != 0;
}
// accumulate() over the rows row0 + i, below `limit`, that this lane's stationary row sees; no other row is multiplied.
template <int D, bool HALVES, typename Visible>
__device__ __forceinline__ void accumulate_visible(Result<D>& result, const float* base, long row_stride, int row0, int limit, int d,
                                                   const quad& first, const quad& second, Visible&& visible) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll 1
    for (int i = 0; i < kTile; ++i) {
        const int r = i & 3, from = (lane & 15) + 16 * (i >> 2);
        const float value[2] = {__shfl(r == 0 ? first[0] : r == 1 ? first[1] : r == 2 ? first[2] : first[3], from, kWave),
                                __shfl(r == 0 ? second[0] : r == 1 ? second[1] : r == 2 ? second[2] : second[3], from, kWave)};
        if (row0 + i >= limit || !visible(i)) continue;
        const float* row = base + (row0 + i) * row_stride;
        int group = lane >> 4;
        asm volatile("" : "+v"(group));  // the columns are worked out here, not kept in registers through the walk
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int column = source<D, HALVES>(padded_column<D, HALVES>(b, e, 4 * group + c), d);
                    if (column >= 0) result[b][e][c] = fmaf(row[column], value[HALVES ? map_of<D>(b, e) : 0], result[b][e][c]);
                }
    }
}

// Sum over the four lane groups of a stationary row.
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}

// The wavefronts' partial results [kWaves][16 rows][D padded columns] in LDS; rows are padded by one 16-byte chunk.
template <int D>
constexpr int kPitch = D + 4;
template <int D>
constexpr int kSmemBytes = kWaves * kTile * kPitch<D> * 4;
template <int D, bool HALVES>
__device__ __forceinline__ void deposit(float* lds, int wave, const Result<D>& result, float factor) {
    const int lane = threadIdx.x & (kWave - 1);
    float* row = lds + (wave * kTile + (lane & 15)) * kPitch<D>;
#pragma unroll
    for (int b = 0; b < D / 64; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) row[padded_column<D, HALVES>(b, e, 4 * (lane >> 4) + c)] = result[b][e][c] * factor;
}
// Thread t's four consecutive padded columns of a row, added up in wavefront order.
template <int D>
struct Share {
    int row, at;
    __device__ __forceinline__ Share() : row(threadIdx.x / (D / 4)), at((threadIdx.x % (D / 4)) * 4) {}
    __device__ __forceinline__ quad collect(const float* lds) const {
        if (row >= kTile) return quad(0.0f);
        quad sum = *reinterpret_cast<const quad*>(lds + row * kPitch<D> + at);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += *reinterpret_cast<const quad*>(lds + (w * kTile + row) * kPitch<D> + at);
        return sum;
    }
};

template <int D>
__device__ __forceinline__ void clear(Result<D>& result) {
#pragma unroll
    for (int b = 0; b < D / 64; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) result[b][e] = quad(0.0f);
}

template <int D>
__global__ __launch_bounds__(kF32Threads, D == 64 ? 4 : 2) void differential_f32_forward_kernel(DifferentialArgs p) {
    extern __shared__ __align__(16) float lds[];
    __shared__ float wave_max[2][kWaves][kTile], wave_total[2][kWaves][kTile];
    constexpr int HALF = D / 32;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), g = lane >> 4;
    const int q0 = (gridDim.x - 1 - blockIdx.x) * kTile, h = blockIdx.y, b = blockIdx.z, kvh = h / (p.hq / p.hkv);  // longest first
    const int query = q0 + (lane & 15);
    const long q_stride = static_cast<long>(p.hq) * p.d, kv_stride = static_cast<long>(p.hkv) * p.d;
    const float* k_base = static_cast<const float*>(p.k) + static_cast<long>(b) * p.ks * kv_stride + static_cast<long>(kvh) * p.d;
    const float* v_base = static_cast<const float*>(p.v) + static_cast<long>(b) * p.ks * kv_stride + static_cast<long>(kvh) * p.d;
    RowOperand<D, true> q;
    q.load(TileRows(static_cast<const float*>(p.q) + static_cast<long>(b) * p.qs * q_stride + static_cast<long>(h) * p.d, q_stride, q0, p.qs, p.d), p.d);
    const int last_key = p.causal ? min(p.ks - 1, p.offset + min(q0 + kTile, p.qs) - 1) : p.ks - 1;
    const int tiles = last_key / kTile + 1;
    const int my_last = p.causal ? min(p.ks - 1, p.offset + query) : p.ks - 1;
    const int first_masked = p.causal ? (p.offset + q0 + 1) / kTile : tiles;  // tile with a key that a query of the block does not see

    float m[2] = {-INFINITY, -INFINITY}, total[2] = {0.0f, 0.0f};
    Result<D> o[2];
    clear<D>(o[0]);
    clear<D>(o[1]);
    auto key_rows = [&](RowOperand<D, true>& k, int t) {
        k.load(TileRows(k_base, kv_stride, t * kTile, t < tiles ? p.ks : 0, p.d), p.d);
    };
    bool left_out = false;
    RowOperand<D, true> k, ahead;
    key_rows(k, wave);
    for (int t = wave; t < tiles; t += kWaves) {
        ColumnOperand<D, false> v;
        v.load(TileRows(v_base, kv_stride, t * kTile, p.ks, p.d), p.d);
        key_rows(ahead, t + kWaves);
        quad s[2] = {product<0, HALF>(k, q), product<HALF, 2 * HALF>(k, q)};  // lane: query l % 16, keys 4 g + r
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float peak = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[i][r] = t * kTile + 4 * g + r <= my_last ? s[i][r] * p.scale : -INFINITY;
                peak = fmaxf(peak, s[i][r]);
            }
            const float next = fmaxf(m[i], group_max(peak));
            const float base = next == -INFINITY ? 0.0f : next;  // no key visible so far: all terms below are 0
            const float alpha = expf(m[i] - base);
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[i][r] = expf(s[i][r] - base);
                sum += s[i][r];
            }
            total[i] = total[i] * alpha + group_sum(sum);
            m[i] = next;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][c][e] *= alpha;
        }
        if (t >= first_masked && non_finite(v)) {
            left_out = true;
        } else {
            accumulate<D, false>(o[0], v, s[0], s[0]);
            accumulate<D, false>(o[1], v, s[1], s[1]);
        }
        k = ahead;
    }
    if (left_out) {
        for (int t = wave; t < tiles; t += kWaves) {
            ColumnOperand<D, false> v;
            v.load(TileRows(v_base, kv_stride, t * kTile, p.ks, p.d), p.d);
            if (t < first_masked || !non_finite(v)) continue;
            key_rows(k, t);
            quad s[2] = {product<0, HALF>(k, q), product<HALF, 2 * HALF>(k, q)};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][r] = expf(s[i][r] * p.scale - (m[i] == -INFINITY ? 0.0f : m[i]));
                accumulate_visible<D, false>(o[i], v_base, kv_stride, t * kTile, p.ks, p.d, s[i], s[i],
                                             [&](int row) { return t * kTile + row <= my_last; });
            }
        }
    }
    if (lane < kTile) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            wave_max[i][wave][lane] = m[i];
            wave_total[i][wave][lane] = total[i];
        }
    }
    __syncthreads();
    // Common maximum over the wavefronts, then the weighted sums, one map after the other through the same memory.
    const Share<D> share;
    const long row = static_cast<long>(b) * p.qs + q0 + share.row;
    const bool mine = share.row < kTile && q0 + share.row < p.qs && share.at < p.d;
    quad of_map[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float peak = wave_max[i][0][lane & 15];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) peak = fmaxf(peak, wave_max[i][w][lane & 15]);
        if (i > 0) __syncthreads();
        deposit<D, false>(lds, wave, o[i], expf(m[i] - (peak == -INFINITY ? 0.0f : peak)));
        __syncthreads();
        of_map[i] = share.collect(lds);
        if (!mine) continue;
        float top = wave_max[i][0][share.row];
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wave_max[i][w][share.row]);
        float sum = 0.0f;  // every query sees a key: where the maximum is -Inf all its scores are -Inf or NaN
        for (int w = 0; w < kWaves; ++w) sum += wave_total[i][w][share.row] * expf(wave_max[i][w][share.row] - top);
        of_map[i] *= 1.0f / sum;
        if (share.at == 0 && p.lse_out != nullptr)
            p.lse_out[(static_cast<long>(i) * p.batch * p.qs + row) * p.hq + h] = top + logf(sum);
    }
    if (!mine) return;
    const float lambda = p.lambda[h];
    const long to = row * q_stride + static_cast<long>(h) * p.d + share.at;
    quad out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = fmaf(-lambda, of_map[1][e], of_map[0][e]);
    store_vec<float, 4>(static_cast<float*>(p.out) + to, out);
    if (p.second != nullptr) store_vec<float, 4>(static_cast<float*>(p.second) + to, of_map[1]);
}

template <int D>
__device__ __forceinline__ float row_delta(const RowOperand<D, false>& dout, const TileRows& rows, int d) {
    RowOperand<D, false> o;
    o.load(rows, d);
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fmaf(dout.chunk[c][e], o.chunk[c][e], sum);
    return group_sum(sum);
}

template <int D>
__global__ __launch_bounds__(kF32Threads, D == 64 ? 4 : 2) void differential_f32_dq_kernel(DifferentialArgs p) {
    extern __shared__ __align__(16) float lds[];
    __shared__ float wave_rest[kWaves][kTile];
    constexpr int HALF = D / 32;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), g = lane >> 4;
    const int q0 = (gridDim.x - 1 - blockIdx.x) * kTile, h = blockIdx.y, b = blockIdx.z, kvh = h / (p.hq / p.hkv);
    const int query = q0 + (lane & 15);
    const bool live = query < p.qs;
    const long q_stride = static_cast<long>(p.hq) * p.d, kv_stride = static_cast<long>(p.hkv) * p.d;
    const float* k_base = static_cast<const float*>(p.k) + static_cast<long>(b) * p.ks * kv_stride + static_cast<long>(kvh) * p.d;
    const float* v_base = static_cast<const float*>(p.v) + static_cast<long>(b) * p.ks * kv_stride + static_cast<long>(kvh) * p.d;
    const long q_head = static_cast<long>(b) * p.qs * q_stride + static_cast<long>(h) * p.d;
    auto rows_of = [&](const void* tensor) { return TileRows(static_cast<const float*>(tensor) + q_head, q_stride, q0, p.qs, p.d); };
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq, stat = (static_cast<long>(b) * p.qs + query) * p.hq + h;
    const float lambda = p.lambda[h];
    RowOperand<D, true> q;
    RowOperand<D, false> dout;
    q.load(rows_of(p.q), p.d);
    dout.load(rows_of(p.dout), p.d);
    const float delta2 = row_delta<D>(dout, rows_of(p.o2), p.d);
    const float delta1 = fmaf(lambda, delta2, row_delta<D>(dout, rows_of(p.o), p.d));
    if (wave == 0 && lane < kTile && live) {
        p.delta[stat] = delta1;
        p.delta[rows + stat] = delta2;
    }
    const float lse1 = live ? p.lse[stat] : 0.0f, lse2 = live ? p.lse[rows + stat] : 0.0f;
    const int last_key = p.causal ? min(p.ks - 1, p.offset + min(q0 + kTile, p.qs) - 1) : p.ks - 1;
    const int my_last = p.causal ? min(p.ks - 1, p.offset + query) : p.ks - 1;
    const int first_masked = p.causal ? (p.offset + q0 + 1) / kTile : last_key / kTile + 1;

    Result<D> dq;
    clear<D>(dq);
    float rest = 0.0f;  // of rowsum(P2 (G - delta2))
    bool left_out = false;
    struct Gradients {
        quad first, second;
    };
    auto score_gradients = [&](int t) {  // lane: query l % 16, keys 4 g + r
        RowOperand<D, true> k;
        RowOperand<D, false> v;
        k.load(TileRows(k_base, kv_stride, t * kTile, p.ks, p.d), p.d);
        v.load(TileRows(v_base, kv_stride, t * kTile, p.ks, p.d), p.d);
        const quad s1 = product<0, HALF>(k, q), s2 = product<HALF, 2 * HALF>(k, q), grad = product<0, 2 * HALF>(v, dout);
        Gradients ds;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool seen = t * kTile + 4 * g + r <= my_last;
            ds.first[r] = seen ? expf(s1[r] * p.scale - lse1) * (grad[r] - delta1) : 0.0f;
            ds.second[r] = seen ? expf(s2[r] * p.scale - lse2) * (grad[r] - delta2) : 0.0f;
        }
        return ds;
    };
    for (int t = wave; t <= last_key / kTile; t += kWaves) {
        ColumnOperand<D, true> columns;
        columns.load(TileRows(k_base, kv_stride, t * kTile, p.ks, p.d), p.d);
        Gradients ds = score_gradients(t);
        rest += (ds.second[0] + ds.second[1]) + (ds.second[2] + ds.second[3]);
        if (t >= first_masked && non_finite(columns)) left_out = true;
        else accumulate<D, true>(dq, columns, ds.first, ds.second * -lambda);
    }
    if (left_out) {
        for (int t = wave; t <= last_key / kTile; t += kWaves) {
            ColumnOperand<D, true> columns;
            columns.load(TileRows(k_base, kv_stride, t * kTile, p.ks, p.d), p.d);
            if (t < first_masked || !non_finite(columns)) continue;
            const Gradients ds = score_gradients(t);
            accumulate_visible<D, true>(dq, k_base, kv_stride, t * kTile, p.ks, p.d, ds.first, ds.second * -lambda,
                                        [&](int row) { return t * kTile + row <= my_last; });
        }
    }
    rest = group_sum(rest);
    if (lane < kTile) wave_rest[wave][lane] = live ? (wave == 0 ? rest + delta2 : rest) : 0.0f;
    deposit<D, true>(lds, wave, dq, p.gradient_scale);
    __syncthreads();
    if (threadIdx.x < kTile) {
        float sum = wave_rest[0][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += wave_rest[w][lane];
        sum = wave_sum<kTile>(sum);
        if (lane == 0) p.lambda_partial[h * p.lambda_parts + static_cast<long>(b) * gridDim.x + q0 / kTile] = -sum;
    }
    const Share<D> share;
    quad sum = share.collect(lds);
    const int column = source<D, true>(share.at, p.d);
    if (share.row >= kTile || q0 + share.row >= p.qs || column < 0) return;
    float* to = static_cast<float*>(p.dq) + (static_cast<long>(b) * p.qs + q0 + share.row) * q_stride + static_cast<long>(h) * p.d + column;
    if (p.accumulate) sum += load_vec<float, 4>(to);
    store_vec<float, 4>(to, sum);
}

template <int D>
__global__ __launch_bounds__(kF32Threads, D == 64 ? 4 : 2) void differential_f32_dkv_kernel(DifferentialArgs p) {
    extern __shared__ __align__(16) float lds[];
    constexpr int HALF = D / 32;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), g = lane >> 4;
    const int part = blockIdx.x % p.splits, k0 = blockIdx.x / p.splits * kTile;  // the first keys have most queries
    const int kvh = blockIdx.y, b = blockIdx.z, group = p.hq / p.hkv;
    const int key = k0 + (lane & 15);
    const long q_stride = static_cast<long>(p.hq) * p.d, kv_stride = static_cast<long>(p.hkv) * p.d;
    const long kv_head = static_cast<long>(b) * p.ks * kv_stride + static_cast<long>(kvh) * p.d;
    const long rows = static_cast<long>(p.batch) * p.qs * p.hq;
    RowOperand<D, true> k;
    RowOperand<D, false> v;
    k.load(TileRows(static_cast<const float*>(p.k) + kv_head, kv_stride, k0, p.ks, p.d), p.d);
    v.load(TileRows(static_cast<const float*>(p.v) + kv_head, kv_stride, k0, p.ks, p.d), p.d);
    const int first_query = p.causal ? max(0, key - p.offset) : 0;  // that sees this lane's key
    const int first_tile = p.causal ? max(0, k0 - p.offset) / kTile : 0;
    const int tiles = max(0, (p.qs + kTile - 1) / kTile - first_tile);

    Result<D> dk, dv;
    clear<D>(dk);
    clear<D>(dv);
    const long items = static_cast<long>(tiles) * group;
    const int begin = static_cast<int>(part * items / p.splits) + wave, end = static_cast<int>((part + 1) * items / p.splits);
    bool left_out = false;
    // Item i is (head of the group, query tile): step(its head's Q and dO, first query, the map and both score gradients of
    // queries 4 g + r).
    auto walk = [&](auto&& step) __attribute__((always_inline)) {
        for (int i = begin; i < end; i += kWaves) {
            const int head = i / tiles, row0 = (first_tile + i - head * tiles) * kTile, h = kvh * group + head;
            const float* q_base = static_cast<const float*>(p.q) + static_cast<long>(b) * p.qs * q_stride + static_cast<long>(h) * p.d;
            const float* do_base = static_cast<const float*>(p.dout) + static_cast<long>(b) * p.qs * q_stride + static_cast<long>(h) * p.d;
            const float lambda = p.lambda[h];
            quad s1, s2, grad;
            {
                RowOperand<D, true> q;
                RowOperand<D, false> dout;
                q.load(TileRows(q_base, q_stride, row0, p.qs, p.d), p.d);
                dout.load(TileRows(do_base, q_stride, row0, p.qs, p.d), p.d);
                s1 = product<0, HALF>(q, k);  // lane: key l % 16, queries 4 g + r
                s2 = product<HALF, 2 * HALF>(q, k);
                grad = product<0, 2 * HALF>(dout, v);
            }
            quad map, ds1, ds2;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = row0 + 4 * g + r;
                const bool seen = row >= first_query && row < p.qs && key < p.ks;
                const long stat = (static_cast<long>(b) * p.qs + min(row, p.qs - 1)) * p.hq + h;
                const float p1 = seen ? expf(s1[r] * p.scale - p.lse[stat]) : 0.0f;
                const float p2 = seen ? -lambda * expf(s2[r] * p.scale - p.lse[rows + stat]) : 0.0f;
                map[r] = p1 + p2;
                ds1[r] = seen ? p1 * (grad[r] - p.delta[stat]) : 0.0f;
                ds2[r] = seen ? p2 * (grad[r] - p.delta[rows + stat]) : 0.0f;
            }
            step(q_base, do_base, row0, map, ds1, ds2);
        }
    };
    auto masked = [&](int row0) { return p.causal && row0 < k0 + kTile - 1 - p.offset; };  // a query that does not see a key of the block
    walk([&](const float* q_base, const float* do_base, int row0, const quad& map, const quad& ds1, const quad& ds2)
             __attribute__((always_inline)) {
        {
            ColumnOperand<D, false> columns;
            columns.load(TileRows(do_base, q_stride, row0, p.qs, p.d), p.d);
            if (masked(row0) && non_finite(columns)) left_out = true;
            else accumulate<D, false>(dv, columns, map, map);
        }
        ColumnOperand<D, true> columns;
        columns.load(TileRows(q_base, q_stride, row0, p.qs, p.d), p.d);
        if (masked(row0) && non_finite(columns)) left_out = true;
        else accumulate<D, true>(dk, columns, ds1, ds2);
    });
    if (left_out) {
        walk([&](const float* q_base, const float* do_base, int row0, const quad& map, const quad& ds1, const quad& ds2)
                 __attribute__((always_inline)) {
            if (!masked(row0)) return;
            auto visible = [&](int i) { return row0 + i >= first_query; };
            {
                ColumnOperand<D, false> columns;
                columns.load(TileRows(do_base, q_stride, row0, p.qs, p.d), p.d);
                if (non_finite(columns)) accumulate_visible<D, false>(dv, do_base, q_stride, row0, p.qs, p.d, map, map, visible);
            }
            ColumnOperand<D, true> columns;
            columns.load(TileRows(q_base, q_stride, row0, p.qs, p.d), p.d);
            if (non_finite(columns)) accumulate_visible<D, true>(dk, q_base, q_stride, row0, p.qs, p.d, ds1, ds2, visible);
        });
    }
    const long count = static_cast<long>(p.batch) * p.ks * kv_stride;
    const Share<D> share;
    auto store = [&](float* whole, float* in_part, quad sum, int column) {
        if (share.row >= kTile || k0 + share.row >= p.ks || column < 0) return;
        float* to = (p.splits == 1 ? whole : in_part) + (static_cast<long>(b) * p.ks + k0 + share.row) * kv_stride +
                    static_cast<long>(kvh) * p.d + column;
        if (p.accumulate && p.splits == 1) sum += load_vec<float, 4>(to);
        store_vec<float, 4>(to, sum);
    };
    deposit<D, true>(lds, wave, dk, p.gradient_scale);
    __syncthreads();
    store(static_cast<float*>(p.dk), p.partial + 2 * part * count, share.collect(lds), source<D, true>(share.at, p.d));
    __syncthreads();
    deposit<D, false>(lds, wave, dv, 1.0f);
    __syncthreads();
    store(static_cast<float*>(p.dv), p.partial + (2 * part + 1) * count, share.collect(lds), source<D, false>(share.at, p.d));
    __syncthreads();
    add_lambda_parts<kF32Threads>(p, reinterpret_cast<double*>(lds));
}

template <auto Kernel, int SMEM>
int launch(long blocks, int heads, const DifferentialArgs& args, hipStream_t stream) {
    static const hipError_t status =
        hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    CGPTX_HIP(status);
    hipLaunchKernelGGL(Kernel, dim3(static_cast<unsigned int>(blocks), static_cast<unsigned int>(heads), static_cast<unsigned int>(args.batch)),
                       dim3(kF32Threads), SMEM, stream, args);
    CGPTX_LAUNCH_CHECK();
    return CGPTX_OK;
}
long row_tiles(int rows) { return (static_cast<long>(rows) + kTile - 1) / kTile; }

}  // namespace

bool differential_f32_takes(const DifferentialArgs& a) {
    return a.dtype == CGPTX_F32 && a.d % 8 == 0 && row_tiles(std::max(a.qs, a.ks)) <= static_cast<long>(kLaunchThreads / kF32Threads);
}

int differential_f32_forward(const DifferentialArgs& a, hipStream_t stream) {
    return a.d <= 64 ? launch<differential_f32_forward_kernel<64>, kSmemBytes<64>>(row_tiles(a.qs), a.hq, a, stream)
                     : launch<differential_f32_forward_kernel<128>, kSmemBytes<128>>(row_tiles(a.qs), a.hq, a, stream);
}

int differential_f32_backward(DifferentialArgs a, hipStream_t stream) {
    KeyWalk walk = key_walk(a);
    walk.block_rows = walk.stream_rows = kTile;
    walk.waves = kWaves;
    walk.tile_us = 10.0;
    if (int st = differential_backward_scratch(a, 2, row_tiles(a.qs) * a.batch, launchable_parts(walk, kF32Threads), stream)) return st;
    if (int st = a.d <= 64 ? launch<differential_f32_dq_kernel<64>, kSmemBytes<64>>(row_tiles(a.qs), a.hq, a, stream)
                           : launch<differential_f32_dq_kernel<128>, kSmemBytes<128>>(row_tiles(a.qs), a.hq, a, stream))
        return st;
    if (int st = a.d <= 64 ? launch<differential_f32_dkv_kernel<64>, kSmemBytes<64>>(row_tiles(a.ks) * a.splits, a.hkv, a, stream)
                           : launch<differential_f32_dkv_kernel<128>, kSmemBytes<128>>(row_tiles(a.ks) * a.splits, a.hkv, a, stream))
        return st;
    if (a.splits > 1) {
        const long count = static_cast<long>(a.batch) * a.ks * a.hkv * a.d;
        if (int st = launch_dkv_reduce<float>(count, a.dk, a.dv, a.partial, a.splits, a.accumulate, stream)) return st;
    }
    return CGPTX_OK;
}

}  // namespace cgptx
