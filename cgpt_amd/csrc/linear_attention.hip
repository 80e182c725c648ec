// Linear attention with a decay for gfx950: every key/value head keeps a matrix of head_dim x head_dim that forgets a fixed share of itself
// at each token, and a query reads it. Forward, backward, and the step of a single token.
//
//   S_t = g S_{t-1} + k_t v_t',  o_t = s S_t' q_t = s sum_{r <= t} g^(t-r) (q_t.k_r) v_r + s g^(t+1) S' q_t    (g = exp(log_decay), S before token 0)
//
// All that a forward and a backward pass compute is one sum over pairs of tokens in either direction of time,
//   out_t = sum_r g^|t-r| (x_t.y_r) z_r + g^.. C' x_t,     C the matrix that the tokens before (behind) leave:
//   o = (q, k, v; S),  dq = (dO, v, k; S') forward,  dv = (k, q, dO; dS),  dk = (v, dO, q; dS') backward in time,
// and the matrices: S_T = sum_r g^(T-1-r) k_r v_r' + g^T S, dS = s sum_t g^(t+1) q_t dO_t' + g^T dS_T. The heads of a group share k and v and
// so the matrix: for dk and dv a token counts once for every head of the group.
//
// A workgroup walks chunks of 64 tokens: in a chunk the pairs are a masked product of tiles, Z'P' with P = (X Y') g^|t-r|, and what came before
// it is C' X'. The matrix stays in the accumulation registers from chunk to chunk, 32 of its columns a wavefront, and goes as an operand into its
// product as it lies (the columns of Y are read in the order that makes it so). Long sequences are cut into segments that
// workgroups walk side by side: one launch leaves each segment's own matrix, one adds them up along the sequence, and the third starts each
// segment from there.
//
// 16-bit storage: P, C and the decayed Z are rounded to it once where they become operands, sums are fp32. In half precision a power of two
// brings them into its range where they leave it. Matrices that the caller gets (fp32) come from Z in two parts, high and low.
// An Inf or NaN reaches the tokens that see it and no others: chunks that hold one are added up token by token.
#include "attention_tiles.hpp"

#include <cmath>
#include <string>

namespace cgptx {
namespace {

constexpr int kChunk = 64;

template <typename T>
using frag_t = vec_t<T, 8>;

template <typename T>
__device__ __forceinline__ acc_t multiply(const frag_t<T>& a, const frag_t<T>& b, acc_t c) {
    if constexpr (sizeof(T) == 2) {
        return Mma<T>::run(a, b, c);
    } else {  // element e of both operands: the pair of columns e and 8 + e of sixteen
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
}

// A tile of 64 rows in LDS: swizzled for 16-bit storage (attention_tiles.hpp), rows four words apart in banks for fp32.
template <typename T, int W>
constexpr int kPitch = sizeof(T) == 2 ? W : W + 4;
template <typename T, int W>
constexpr int kTile = kChunk * kPitch<T, W>;
template <typename T>
constexpr int kPairsPitch = sizeof(T) == 2 ? kChunk : kChunk + 4;

// Row block + lane%32 of a tile, columns 16 step + 8 (lane/32) .. + 7.
template <typename T, int W>
__device__ __forceinline__ frag_t<T> row_frag(const T* tile, int block, int step) {
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const frag_t<T>*>(tile + block * W + wide_direct_offset<W>(lane, step));
    } else {
        const T* from = tile + (block + (lane & 31)) * kPitch<T, W> + 16 * step + 8 * (lane >> 5);
        const auto lo = load_vec<T, 4>(from), hi = load_vec<T, 4>(from + 4);
        return frag_t<T>{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
}
// Column 32 t + lane%32 of a tile, rows block + {0-3 | 4-7} and eight further. SWAPPED: the columns of a group of sixteen in the order 0-3, 8-11,
// 4-7, 12-15, so that a product's registers 8 s .. 8 s + 7 hold rows 16 s + 8 (lane/32) .. + 7: those of row_frag.
template <typename T, int W, bool SWAPPED>
__device__ __forceinline__ frag_t<T> column_frag(const T* tile, int block, int t) {
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 2) {
        if constexpr (!SWAPPED) {
            return wide_transposed_frag<T>(tile + block * W, wide_transposed_offset<W>(lane, t, 0), wide_transposed_offset<W>(lane, t, 1));
        } else {
            auto offset = [&](int second) {
                const int row = (lane >> 5) * 4 + ((lane & 15) >> 2) + second * 8, chunk = t * 4 + ((lane >> 4) & 1) * 2 + (lane & 1);
                return row * W + ((chunk ^ swizzle<W>(row)) * 8) + ((lane >> 1) & 1) * 4;
            };
            return wide_transposed_frag<T>(tile + block * W, offset(0), offset(1));
        }
    } else {
        const int m = lane & 31, column = 32 * t + (SWAPPED ? (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1) : m);
        frag_t<T> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = tile[(block + (e & 4) * 2 + 4 * (lane >> 5) + (e & 3)) * kPitch<T, W> + column];
        return f;
    }
}
// Registers 8 step .. 8 step + 7 of an accumulator as an operand.
template <typename T>
__device__ __forceinline__ frag_t<T> operand_of(const acc_t& acc, int step) {
    vec_t<float, 8> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = acc[8 * step + e];
    return vec_from_f32<T, 8>(f);
}
// Row of the matrix that register i of its accumulator k holds, less 32 k.
__device__ __forceinline__ int matrix_row(int i) { return 16 * (i >> 3) + 8 * ((threadIdx.x & 63) >> 5) + (i & 7); }

// The 64 x 64 pairs of a chunk: row t, eight of the other tokens side by side as an operand takes them (c of eight).
template <typename T>
__device__ __forceinline__ T* pairs_at(T* pairs, int t, int c) {
    if constexpr (sizeof(T) == 2) return pairs + t * kPairsPitch<T> + (c ^ (t & 7)) * 8;
    else return pairs + t * kPairsPitch<T> + c * 8;
}

// One head of a [.., tokens, heads, d] tensor.
template <typename T>
struct Rows {
    const T* base;  // of the batch entry's head
    long stride;    // elements between tokens
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* from, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, bytes, 0x00020000);
}
// 16 bytes a lane, 1 KiB in all, straight into LDS.
__device__ __forceinline__ void load_chunks(__amdgpu_buffer_rsrc_t rsrc, void* to, int voffset, int soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr)(to), 16, voffset, soffset, 0, 0);
}
// Rows row0 .. row0 + 63 of a head, zeros behind the last token and behind column d. DIRECT (16-bit storage, 16-byte boundaries): straight into
// LDS; the tile is there behind s_waitcnt vmcnt(0) and a barrier.
template <typename T, int W, bool DIRECT>
__device__ __forceinline__ void load_tile(T* tile, const Rows<T>& rows, int row0, int tokens, int d, bool vectors) {
    constexpr int kThreadsHere = W * 2;  // W/32 wavefronts
    const T* first = rows.base + static_cast<long>(row0) * rows.stride;
    const int left = min(kChunk, tokens - row0);
    if constexpr (DIRECT) {
        constexpr int kChunks = W / 8, kRowsPerLoad = 64 / kChunks, kWaves = W / 32;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int row_bytes = static_cast<int>(rows.stride) * 2;
        const __amdgpu_buffer_rsrc_t rsrc = buffer_of(first, (left - 1) * row_bytes + d * 2);
        const int r = wave * kRowsPerLoad + lane / kChunks, chunk = (lane % kChunks) ^ swizzle<W>(r);
        const int voffset = chunk * 8 < d ? r * row_bytes + chunk * 16 : 1 << 30;
#pragma unroll
        for (int i = 0; i < kChunk / (kWaves * kRowsPerLoad); ++i)
            load_chunks(rsrc, tile + (i * kWaves + wave) * kRowsPerLoad * W, voffset, i * kWaves * kRowsPerLoad * row_bytes);
    } else {
        constexpr int VEC = kVec128<T>, kPieces = W / VEC;
        for (int n = threadIdx.x; n < kChunk * kPieces; n += kThreadsHere) {
            const int r = n / kPieces, piece = n % kPieces, column = piece * VEC;
            vec_t<T, VEC> v(static_cast<T>(0.0f));
            if (r < left && column < d) {
                const T* from = first + static_cast<long>(r) * rows.stride + column;
                if (vectors) {
                    v = load_vec<T, VEC>(from);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (column + e < d) v[e] = from[e];
                }
            }
            if constexpr (sizeof(T) == 2) store_vec<T, VEC>(tile + r * W + ((piece ^ swizzle<W>(r)) * 8), v);
            else store_vec<T, VEC>(tile + r * kPitch<T, W> + column, v);
        }
    }
}
// The tiles that load_tile asked for are there, for every wavefront.
__device__ __forceinline__ void tiles_there() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
}

// log2 of the decay. No growth: what is above 1 counts as 1. A head that forgets everything (-inf) has 0^0 = 1.
__device__ __forceinline__ float log2_decay(float log_decay) {
    const float l = log_decay * kLog2e;
    return l > 0.0f ? 0.0f : l < -1.0e4f ? -1.0e4f : l;  // a NaN stays one
}
__device__ __forceinline__ float power(float l, int n) { return exp2f(l * static_cast<float>(n)); }

template <typename V>
__device__ __forceinline__ float finite_test(const V& f, float sum) {  // stays 0 while all is finite
    if constexpr (sizeof(f[0]) == 2) {
        using T = std::remove_cv_t<std::remove_reference_t<decltype(f[0])>>;
        const auto words = __builtin_bit_cast(vec_t<unsigned int, 4>, f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (__is_same(T, f16_t)) sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(vec_t<f16_t, 2>, words[w]), vec_t<f16_t, 2>(static_cast<f16_t>(0.0f)), sum, false);
            else sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(vec_t<bf16_t, 2>, words[w]), vec_t<bf16_t, 2>(static_cast<bf16_t>(0.0f)), sum, false);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(f[e], 0.0f, sum);
    }
    return sum;
}

// Half precision: the power of two that brings a largest magnitude into 2^low .. 2^high, 1 where it is there already (or zero, or not finite).
__device__ __forceinline__ float range_scale(float largest, int low, int high) {
    const int e = static_cast<int>((__float_as_uint(largest) >> 23) & 0xFF) - 127;
    if (e >= 128 || e <= -127 || (e >= low && e < high)) return 1.0f;
    const int target = e < low ? low : high - 1;
    return __uint_as_float(static_cast<unsigned int>(min(max(target - e, -126), 126) + 127) << 23);
}
template <typename T>
constexpr bool kNarrow = __is_same(T, f16_t);  // a range that sums leave

// Z of a wavefront's 32 columns: four operands of sixteen rows.
template <typename T>
struct Values {
    frag_t<T> z[4];
    template <int W>
    __device__ __forceinline__ void load(const T* tile, int column_block) {
#pragma unroll
        for (int s = 0; s < 4; ++s) z[s] = column_frag<T, W, false>(tile, 16 * s, column_block);
    }
    __device__ __forceinline__ bool finite() const {
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s) sum = finite_test(z[s], sum);
        return !__any(!(sum == 0.0f));
    }
    __device__ __forceinline__ float largest() const {
        float most = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const auto f = vec_to_f32<T, 8>(z[s]);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]));
        }
        return wave_max(most);
    }
};

// Weights of a chunk's tokens as what follows the chunk sees them (forward in time: 1 for token `end`, else g^(end - token); backward: g^(token
// + 1)), for the rows that a lane's operands hold.
struct Weights {
    float base[8];  // of the rows of sixteen
    float l, scale;
    bool reverse;
    __device__ __forceinline__ static int row(int e) { return 4 * ((threadIdx.x & 63) >> 5) + (e & 3) + 2 * (e & 4); }
    __device__ __forceinline__ Weights(float l_, float scale_, bool reverse_) : l(l_), scale(scale_), reverse(reverse_) {
#pragma unroll
        for (int e = 0; e < 8; ++e) base[e] = scale * power(l, reverse ? row(e) + 1 : 16 - row(e));
    }
    // Of block s of sixteen rows; `end` is kChunk but for a sequence's last chunk.
    __device__ __forceinline__ vec_t<float, 8> of(int s, int end) const {
        vec_t<float, 8> w;
        if (reverse || end == kChunk) {
            const float f = power(l, reverse ? 16 * s : 48 - 16 * s);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = base[e] * f;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = scale * power(l, max(end - 16 * s - row(e), 0));
        }
        return w;
    }
};

// matrix += Y' (w Z) over a chunk, the matrix decayed by `factor` first. EXACT: w Z in two parts.
template <typename T, int W, bool EXACT>
__device__ __forceinline__ void update_matrix(acc_t (&matrix)[W / 32], float factor, const T* y_tile, const Values<T>& values, const Weights& weights,
                                              int end) {
    float up = 1.0f;
    if constexpr (kNarrow<T>) {
        up = range_scale(values.largest(), -3, 15);
        up = up < 1.0f ? 1.0f : up;  // only what is small loses digits
        factor *= up;
    }
    if (factor != 1.0f)
#pragma unroll
        for (int k = 0; k < W / 32; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) matrix[k][i] *= factor;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        auto w = weights.of(s, end);
        if constexpr (kNarrow<T>) w *= up;
        const vec_t<float, 8> product = vec_to_f32<T, 8>(values.z[s]) * w;
        const frag_t<T> high = vec_from_f32<T, 8>(product);
        frag_t<T> low;
        if constexpr (EXACT && sizeof(T) == 2) low = vec_from_f32<T, 8>(product - vec_to_f32<T, 8>(high));
#pragma unroll
        for (int k = 0; k < W / 32; ++k) {
            const frag_t<T> y = column_frag<T, W, true>(y_tile, 16 * s, k);
            matrix[k] = multiply<T>(y, high, matrix[k]);
            if constexpr (EXACT && sizeof(T) == 2) matrix[k] = multiply<T>(y, low, matrix[k]);
        }
    }
    if constexpr (kNarrow<T>)
        if (up != 1.0f) {
            const float down = 1.0f / up;
#pragma unroll
            for (int k = 0; k < W / 32; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) matrix[k][i] *= down;
        }
}

struct LinearArgs {
    const void *q, *k, *v, *dout;
    void *out, *dq, *dk, *dv;
    const float *log_decay, *before, *d_after;
    float *after, *d_before;
    float *ahead, *behind;  // [batch x kv_heads][segments][d][d]: what comes before a segment, and the gradient from behind it
    int batch, tokens, hq, hkv, d;
    int segments, segment_chunks;
    float scale;
    int accumulate, vectors;
};

// One sum over pairs (see above): its tensors, heads and weights.
template <typename T>
struct Task {
    const T *x, *y, *z;
    T* out;
    int x_heads, y_heads;
    const float* carry;  // of the pair (batch entry, kv head) and segment; null: zero
    float carry_factor;  // of the matrix as it is loaded
    bool transposed;
    float pair_scale, matrix_scale, out_scale;  // of P, of what is added to the matrix, of the matrix's part of the output
};

// The output of one head in one segment.
template <typename T, int W, bool REVERSE, bool DIRECT>
__device__ __forceinline__ void walk_segment(const LinearArgs& a, const Task<T>& task, int b, int head, int segment, T* lds) {
    constexpr int K = W / 32, kTables = W == 128 ? 1 : 2;
    T *x_tile = lds, *y_tile = lds + kTile<T, W>, *z_tile = lds + 2 * kTile<T, W>, *pairs = lds + 3 * kTile<T, W>;
    __shared__ float pair_scales[3];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int d = a.d, tokens = a.tokens;
    const int heads_each = task.y_heads > task.x_heads ? task.y_heads / task.x_heads : 1;
    const int y_first = static_cast<int>(static_cast<long>(head) * task.y_heads / task.x_heads);
    const int kv = REVERSE ? head : y_first;
    const float l = log2_decay(a.log_decay[kv]);

    const long x_stride = static_cast<long>(task.x_heads) * d, y_stride = static_cast<long>(task.y_heads) * d;
    const Rows<T> x{task.x + static_cast<long>(b) * tokens * x_stride + static_cast<long>(head) * d, x_stride};
    const long y_offset = static_cast<long>(b) * tokens * y_stride + static_cast<long>(y_first) * d;

    // Which 32 x 32 tiles of pairs a wavefront makes: 0 and 1 on the diagonal, 2 the one beside it. W = 64: wavefront 0 makes 0 and 2.
    float table[kTables][16];
    auto tile_t = [](int tile) { return tile == 2 ? (REVERSE ? 0 : 1) : tile; };
    auto tile_r = [](int tile) { return tile == 2 ? (REVERSE ? 1 : 0) : tile; };
    auto my_tile = [&](int n) { return n == 0 ? wave : 2; };
    auto apart = [&](int tile, int i) {
        const int t = tile_t(tile) * 32 + (lane & 31), r = tile_r(tile) * 32 + acc_row(i);
        return REVERSE ? r - t : t - r;
    };
#pragma unroll
    for (int n = 0; n < kTables; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) table[n][i] = task.pair_scale * power(l, max(apart(my_tile(n), i), 0));
    const Weights weights(l, task.matrix_scale, REVERSE);

    acc_t matrix[K];
    const int column = wave * 32 + (lane & 31);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 32 * k + matrix_row(i);
            matrix[k][i] = task.carry != nullptr && row < d && column < d ? task.carry[task.transposed ? column * d + row : row * d + column] * task.carry_factor : 0.0f;
        }
    bool empty = task.carry == nullptr;

    const int chunks_in_all = (tokens + kChunk - 1) / kChunk;
    const int first_chunk = segment * a.segment_chunks, last_chunk = min(first_chunk + a.segment_chunks, chunks_in_all) - 1;
    const int steps = last_chunk - first_chunk + 1;
    for (int step = 0; step < steps; ++step) {
        const int row0 = (REVERSE ? last_chunk - step : first_chunk + step) * kChunk;
        const int length = min(kChunk, tokens - row0);
        acc_t o[2];
        for (int each = 0; each < heads_each; ++each) {
            __syncthreads();  // everybody has read the last tiles
            const Rows<T> y{task.y + y_offset + static_cast<long>(each) * d, y_stride}, z{task.z + y_offset + static_cast<long>(each) * d, y_stride};
            if (each == 0) load_tile<T, W, DIRECT>(x_tile, x, row0, tokens, d, a.vectors);
            load_tile<T, W, DIRECT>(y_tile, y, row0, tokens, d, a.vectors);
            load_tile<T, W, DIRECT>(z_tile, z, row0, tokens, d, a.vectors);
            tiles_there();
            // P' = (Y X') g^.., tile by tile.
#pragma unroll
            for (int n = 0; n < kTables; ++n) {
                const int tile = my_tile(n);
                if (tile > 2 || (n > 0 && wave > 0)) continue;
                const int tt = tile_t(tile), tr = tile_r(tile);
                acc_t p(0.0f);
#pragma unroll
                for (int s = 0; s < W / 16; ++s) p = multiply<T>(row_frag<T, W>(y_tile, tr * 32, s), row_frag<T, W>(x_tile, tt * 32, s), p);
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = apart(tile, i) >= 0 ? p[i] * table[n][i] : 0.0f;
                if constexpr (kNarrow<T>) {
                    float most = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(p[i]));
                    const float scale = range_scale(wave_max(most), -3, 15);
                    if (scale != 1.0f)
#pragma unroll
                        for (int i = 0; i < 16; ++i) p[i] *= scale;
                    if (lane == 0) pair_scales[tile] = scale;
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) *reinterpret_cast<frag_t<T>*>(pairs_at<T>(pairs, tt * 32 + (lane & 31), 4 * tr + 2 * s + half)) = operand_of<T>(p, s);
            }
            // What came before the chunk.
            if (each == 0) {
                o[0] = o[1] = acc_t(0.0f);
                if (!empty) {
                    float scale = 1.0f;
                    if constexpr (kNarrow<T>) {
                        float most = 0.0f;
#pragma unroll
                        for (int k = 0; k < K; ++k)
#pragma unroll
                            for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(matrix[k][i]));
                        scale = range_scale(wave_max(most), -3, 15);
                    }
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            frag_t<T> m;
                            if constexpr (kNarrow<T>) {
                                acc_t scaled = matrix[k];
                                if (scale != 1.0f) scaled *= scale;
                                m = operand_of<T>(scaled, s);
                            } else {
                                m = operand_of<T>(matrix[k], s);
                            }
#pragma unroll
                            for (int t = 0; t < 2; ++t) o[t] = multiply<T>(m, row_frag<T, W>(x_tile, 32 * t, 2 * k + s), o[t]);
                        }
                    const float factor = task.out_scale / scale;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int place = t * 32 + (lane & 31);
                        const float f = factor * power(l, max(REVERSE ? length - 1 - place : place, 0));
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[t][i] *= f;
                    }
                }
            }
            __syncthreads();  // all pairs are there
            Values<T> values;
            values.template load<W>(z_tile, wave);
            if (values.finite()) {
#pragma unroll
                for (int tile = 0; tile < 3; ++tile) {
                    const int tt = tile_t(tile), tr = tile_r(tile);
                    float scale = 1.0f;
                    if constexpr (kNarrow<T>) {
                        scale = pair_scales[tile];
                        if (scale != 1.0f) o[tt] *= scale;
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        o[tt] = multiply<T>(values.z[2 * tr + s], *reinterpret_cast<const frag_t<T>*>(pairs_at<T>(pairs, tt * 32 + (lane & 31), 4 * tr + 2 * s + half)), o[tt]);
                    if constexpr (kNarrow<T>)
                        if (scale != 1.0f) o[tt] *= 1.0f / scale;
                }
            } else {
                // A pair that the mask hides is 0, but 0 x Inf is NaN in a product of tiles.
                for (int r = 0; r < kChunk; ++r)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int place = t * 32 + (lane & 31), in_block = r & 15;
                        const bool seen = REVERSE ? r >= place : r <= place;
                        if (!seen) continue;
                        const int c = 2 * (r >> 4) + ((in_block >> 2) & 1), e = (in_block & 3) + 4 * (in_block >> 3);
                        float p = to_f32(pairs_at<T>(pairs, place, c)[e]);
                        if constexpr (kNarrow<T>) p *= 1.0f / pair_scales[(r >> 5) == t ? t : 2];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int at = wave * 32 + acc_row(i);
                            T value;
                            if constexpr (sizeof(T) == 2) value = z_tile[r * W + (((at >> 3) ^ swizzle<W>(r)) * 8) + (at & 7)];
                            else value = z_tile[r * kPitch<T, W> + at];
                            o[t][i] = fmaf(p, to_f32(value), o[t][i]);
                        }
                    }
            }
            if (step + 1 < steps) update_matrix<T, W, false>(matrix, each == 0 ? power(l, length) : 1.0f, y_tile, values, weights, kChunk);
        }
        empty = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int place = t * 32 + (lane & 31);
            if (place >= length) continue;
            T* to = task.out + static_cast<long>(b) * tokens * x_stride + static_cast<long>(row0 + place) * x_stride + static_cast<long>(head) * d;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = wave * 32 + 8 * g + 4 * half;
                vec_t<float, 4> v{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]};
                if (a.vectors) {
                    if (at < d) {
                        if (a.accumulate) v += vec_to_f32<T, 4>(load_vec<T, 4>(to + at));
                        store_vec<T, 4>(to + at, vec_from_f32<T, 4>(v));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e < d) to[at + e] = from_f32<T>(a.accumulate ? v[e] + to_f32(to[at + e]) : v[e]);
                }
            }
        }
    }
}

// A workgroup's unit (batch entry, kv head, segment) and which of the unit's `members` it is. The workgroups of a unit read the same rows: where
// the units divide evenly over the 8 XCDs, whose workgroups are dealt out in turn, a unit's stay on one.
struct Unit {
    int pair, segment, member;
};
__device__ __forceinline__ Unit unit_of(unsigned int id, unsigned int members, unsigned int units, int segments) {
    unsigned int unit, member;
    if (units % 8 == 0) {
        const unsigned int local = id / 8;
        unit = id % 8 + 8 * (local / members);
        member = local % members;
    } else {
        unit = id / members;
        member = id % members;
    }
    return {static_cast<int>(unit / static_cast<unsigned int>(segments)), static_cast<int>(unit % static_cast<unsigned int>(segments)), static_cast<int>(member)};
}

template <typename T>
__device__ __forceinline__ T* shared_memory() {
    extern __shared__ __align__(1024) unsigned char linear_smem[];
    return reinterpret_cast<T*>(linear_smem);
}

__device__ __forceinline__ const float* carry_of(const float* stored, const float* given, const LinearArgs& a, int pair, int segment) {
    const long matrix = static_cast<long>(a.d) * a.d;
    if (a.segments > 1) return stored + (static_cast<long>(pair) * a.segments + segment) * matrix;
    return given != nullptr ? given + pair * matrix : nullptr;
}

template <typename T, int W, bool DIRECT>
__global__ __launch_bounds__(W * 2, 2) void linear_forward_kernel(LinearArgs a) {
    const int group = a.hq / a.hkv;
    const Unit u = unit_of(blockIdx.x, group, gridDim.x / group, a.segments);
    const int b = u.pair / a.hkv, kv = u.pair % a.hkv;
    Task<T> task;
    task.x = static_cast<const T*>(a.q);
    task.y = static_cast<const T*>(a.k);
    task.z = static_cast<const T*>(a.v);
    task.out = static_cast<T*>(a.out);
    task.x_heads = a.hq;
    task.y_heads = a.hkv;
    task.carry = carry_of(a.ahead, a.before, a, u.pair, u.segment);
    task.carry_factor = a.segments > 1 ? 1.0f : power(log2_decay(a.log_decay[kv]), 1);
    task.transposed = false;
    task.pair_scale = a.scale;
    task.matrix_scale = 1.0f;
    task.out_scale = a.scale;
    walk_segment<T, W, false, DIRECT>(a, task, b, kv * group + u.member, u.segment, shared_memory<T>());
}

// dk and dv of all units first, whose walks are as many times longer as a group has heads, then dq.
template <typename T, int W, bool DIRECT>
__global__ __launch_bounds__(W * 2, 2) void linear_backward_kernel(LinearArgs a) {
    const unsigned int group = a.hq / a.hkv, units = gridDim.x / (group + 2);
    Task<T> task;
    const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v), *dout = static_cast<const T*>(a.dout);
    if (blockIdx.x < 2 * units) {
        const Unit u = unit_of(blockIdx.x, 2, units, a.segments);
        const bool dk = u.member == 0;
        task.x = dk ? v : k;
        task.y = dk ? dout : q;
        task.z = dk ? q : dout;
        task.out = static_cast<T*>(dk ? a.dk : a.dv);
        task.x_heads = a.hkv;
        task.y_heads = a.hq;
        task.carry = carry_of(a.behind, a.d_after, a, u.pair, u.segment);
        task.carry_factor = 1.0f;
        task.transposed = dk;
        task.pair_scale = task.matrix_scale = a.scale;
        task.out_scale = 1.0f;
        walk_segment<T, W, true, DIRECT>(a, task, u.pair / a.hkv, u.pair % a.hkv, u.segment, shared_memory<T>());
    } else {
        const Unit u = unit_of(blockIdx.x - 2 * units, group, units, a.segments);
        const int kv = u.pair % a.hkv;
        task.x = dout;
        task.y = v;
        task.z = k;
        task.out = static_cast<T*>(a.dq);
        task.x_heads = a.hq;
        task.y_heads = a.hkv;
        task.carry = carry_of(a.ahead, a.before, a, u.pair, u.segment);
        task.carry_factor = a.segments > 1 ? 1.0f : power(log2_decay(a.log_decay[kv]), 1);
        task.transposed = true;
        task.pair_scale = a.scale;
        task.matrix_scale = 1.0f;
        task.out_scale = a.scale;
        walk_segment<T, W, false, DIRECT>(a, task, u.pair / a.hkv, kv * static_cast<int>(group) + u.member, u.segment, shared_memory<T>());
    }
}

// Every segment's own matrix: what its tokens leave to those behind it (blockIdx.y = 0: k v') or before it (1: q dO' of the group's heads). The
// last one's goes to `after` as its last token sees it, the first one's to d_before; each where the caller asked for it.
template <typename T, int W, bool DIRECT>
__global__ __launch_bounds__(W * 2, 2) void linear_segments_kernel(LinearArgs a, int first_part) {
    constexpr int K = W / 32;
    T* lds = shared_memory<T>();
    T *y_tile = lds, *z_tile = lds + kTile<T, W>;
    const bool reverse = first_part + blockIdx.y == 1;
    const int pair = static_cast<int>(blockIdx.x / a.segments), segment = static_cast<int>(blockIdx.x % a.segments);
    const int b = pair / a.hkv, kv = pair % a.hkv, d = a.d, tokens = a.tokens;
    const bool outermost = segment == (reverse ? 0 : a.segments - 1);
    const long matrix_size = static_cast<long>(d) * d;
    float* to = reverse ? a.behind : a.ahead;
    if (outermost) {
        to = reverse ? a.d_before : a.after;
        if (to == nullptr) return;
        to += pair * matrix_size;
    } else {
        to += (static_cast<long>(pair) * a.segments + segment) * matrix_size;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float l = log2_decay(a.log_decay[kv]);
    const Weights weights(l, reverse ? a.scale : 1.0f, reverse);
    const int heads = reverse ? a.hq : a.hkv, heads_each = reverse ? a.hq / a.hkv : 1;
    const long stride = static_cast<long>(heads) * d;
    const T* y_base = static_cast<const T*>(reverse ? a.q : a.k) + static_cast<long>(b) * tokens * stride + static_cast<long>(kv) * heads_each * d;
    const T* z_base = static_cast<const T*>(reverse ? a.dout : a.v) + static_cast<long>(b) * tokens * stride + static_cast<long>(kv) * heads_each * d;

    acc_t matrix[K];
#pragma unroll
    for (int k = 0; k < K; ++k) matrix[k] = acc_t(0.0f);
    const int first_chunk = segment * a.segment_chunks, last_chunk = min(first_chunk + a.segment_chunks, (tokens + kChunk - 1) / kChunk) - 1;
    for (int step = 0; step <= last_chunk - first_chunk; ++step) {
        const int row0 = (reverse ? last_chunk - step : first_chunk + step) * kChunk;
        const int length = min(kChunk, tokens - row0);
        const int end = outermost && !reverse && row0 + kChunk >= tokens ? length - 1 : length;  // the token that sees weight 1
        for (int each = 0; each < heads_each; ++each) {
            __syncthreads();
            load_tile<T, W, DIRECT>(y_tile, Rows<T>{y_base + static_cast<long>(each) * d, stride}, row0, tokens, d, a.vectors);
            load_tile<T, W, DIRECT>(z_tile, Rows<T>{z_base + static_cast<long>(each) * d, stride}, row0, tokens, d, a.vectors);
            tiles_there();
            Values<T> values;
            values.template load<W>(z_tile, wave);
            update_matrix<T, W, true>(matrix, each == 0 ? power(l, end) : 1.0f, y_tile, values, weights, end);
        }
    }
    const int column = wave * 32 + (lane & 31);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 32 * k + matrix_row(i);
            if (row < d && column < d) to[row * d + column] = matrix[k][i];
        }
}

// The segments' matrices become what comes before each (blockIdx.y = 0) or behind it (1), in order along the sequence, a thread an element.
constexpr int kAhead = 8;  // loads in flight
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a, int first_part) {
    const bool reverse = first_part + blockIdx.y == 1;
    const long matrix = static_cast<long>(a.d) * a.d, at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= matrix * a.batch * a.hkv) return;
    const long pair = at / matrix, element = at - pair * matrix;
    const float l = log2_decay(a.log_decay[pair % a.hkv]);
    const float* given = reverse ? a.d_after : a.before;
    float* result = reverse ? a.d_before : a.after;
    float running = given != nullptr ? given[at] * (reverse ? 1.0f : power(l, 1)) : 0.0f;
    const int n = a.segments, whole = a.segment_chunks * kChunk, last = a.tokens - (n - 1) * whole;  // tokens of the last segment
    if (n > 1) {
        float* slots = (reverse ? a.behind : a.ahead) + pair * n * matrix + element;
        for (int j0 = 0; j0 < n; j0 += kAhead) {
            float own[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int place = j0 + j;
                own[j] = place < n - 1 ? slots[static_cast<long>(reverse ? n - 1 - place : place) * matrix] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int place = j0 + j;
                if (place >= n) break;
                const int segment = reverse ? n - 1 - place : place;
                slots[static_cast<long>(segment) * matrix] = running;
                if (place < n - 1) running = fmaf(running, power(l, segment == n - 1 ? last : whole), own[j]);
            }
        }
    }
    if (result != nullptr) result[at] = fmaf(running, power(l, reverse ? (n == 1 ? last : whole) : last - 1), result[at]);
}

// ------------------------------------------------------------------------------------------------ one token
// S' = g S + k v', o = s S'' q. A workgroup has 32 columns of a kv head's matrix, a thread 4 columns of every 32nd row; heads of the group one after
// the other from registers.
constexpr int kStepThreads = 256, kStepColumns = 32;
template <typename T, bool VECTORS>
__global__ __launch_bounds__(kStepThreads) void linear_step_kernel(T* __restrict__ out, float* next, const float* state, const T* __restrict__ q,
                                                                   const T* __restrict__ k, const T* __restrict__ v,
                                                                   const float* __restrict__ log_decay, int hq, int hkv, int d, float scale) {
    constexpr int kRows = kStepThreads / (kStepColumns / 4), kOwn = 128 / kRows;
    __shared__ vec_t<float, 4> stage[kStepThreads / kWave][kStepColumns / 4];
    const int blocks = (d + kStepColumns - 1) / kStepColumns;
    const long pair = blockIdx.x / blocks;
    const int block = static_cast<int>(blockIdx.x % blocks), b = static_cast<int>(pair / hkv), kv = static_cast<int>(pair % hkv), group = hq / hkv;
    const int sub = threadIdx.x % (kStepColumns / 4), row0 = threadIdx.x / (kStepColumns / 4);
    const int column = block * kStepColumns + sub * 4;
    const float* from = state + pair * d * d;
    float* to = next + pair * d * d;
    vec_t<float, 4> s[kOwn];
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
        const int row = row0 + n * kRows;
        s[n] = vec_t<float, 4>(0.0f);
        if (row < d) {
            if constexpr (VECTORS) {
                if (column < d) s[n] = load_vec<float, 4>(from + row * d + column);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (column + e < d) s[n][e] = from[row * d + column + e];
            }
        }
    }
    const float g = power(log2_decay(log_decay[kv]), 1);
    vec_t<float, 4> value(0.0f);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (column + e < d) value[e] = to_f32(v[pair * d + column + e]);
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
        const int row = row0 + n * kRows;
        if (row >= d) continue;
        const float key = to_f32(k[pair * d + row]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], g, key * value[e]);
        if constexpr (VECTORS) {
            if (column < d) store_vec<float, 4>(to + row * d + column, s[n]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (column + e < d) to[row * d + column + e] = s[n][e];
        }
    }
    for (int h = 0; h < group; ++h) {
        const long head = static_cast<long>(b) * hq + static_cast<long>(kv) * group + h;
        vec_t<float, 4> sum(0.0f);
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            const int row = row0 + n * kRows;
            const float query = row < d ? to_f32(q[head * d + row]) : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = row < d ? fmaf(query, s[n][e], sum[e]) : sum[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int offset = 32; offset >= 8; offset /= 2) sum[e] += __shfl_xor(sum[e], offset, kWave);
        if (h > 0) __syncthreads();
        if ((threadIdx.x & 63) < kStepColumns / 4) stage[threadIdx.x / kWave][sub] = sum;
        __syncthreads();
        if (threadIdx.x < kStepColumns) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kStepThreads / kWave; ++w) total += stage[w][threadIdx.x / 4][threadIdx.x % 4];
            const int at = block * kStepColumns + static_cast<int>(threadIdx.x);
            if (at < d) out[head * d + at] = from_f32<T>(total * scale);
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
struct Shape {
    std::size_t batch, tokens, hq, hkv, d;
    float scale;
    int dtype;
};

int validate(const char* name, const Shape& s) {
    const std::string n(name);
    if (!valid_dtype(s.dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (s.batch == 0 || s.tokens == 0 || s.hq == 0 || s.hkv == 0 || s.d == 0 || s.hq % s.hkv != 0)
        return fail(CGPTX_INVALID_ARGUMENT, n + ": invalid tensors or options");
    if (!std::isfinite(s.scale)) return fail(CGPTX_INVALID_ARGUMENT, n + ": attention scale must be finite");
    if (s.d > 128) return fail(CGPTX_INVALID_ARGUMENT, n + ": head_dim must not exceed 128");
    // A chunk of 64 tokens and a launch's workgroups are counted in 32 bits.
    if (s.batch > 65535 || s.tokens > (std::size_t{1} << 30) || s.hq > 65535 || s.batch * s.hq > (std::size_t{1} << 20))
        return fail(CGPTX_OVERFLOW, n + ": dimension exceeds the supported range");
    return CGPTX_OK;
}
float chosen_scale(const Shape& s) { return s.scale > 0.0f ? s.scale : 1.0f / std::sqrt(static_cast<float>(s.d)); }

bool aligned(std::initializer_list<const void*> tensors) {
    for (const void* t : tensors)
        if (!is_aligned16(t)) return false;  // an absent one is
    return true;
}

LinearArgs make_args(const Shape& s, const void* q, const void* k, const void* v, const float* log_decay, const float* before) {
    LinearArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.log_decay = log_decay;
    a.before = before;
    a.batch = static_cast<int>(s.batch);
    a.tokens = static_cast<int>(s.tokens);
    a.hq = static_cast<int>(s.hq);
    a.hkv = static_cast<int>(s.hkv);
    a.d = static_cast<int>(s.d);
    a.scale = chosen_scale(s);
    return a;
}

// Segments for `walks` workgroups in each, of whole chunks: as many as keep every compute unit busy twice over.
void cut(LinearArgs& a, long walks, int most) {
    const int chunks = (a.tokens + kChunk - 1) / kChunk;
    const long wanted = std::max<long>(1, (2L * compute_units() + walks - 1) / walks);
    const int segments = static_cast<int>(std::min<long>({wanted, static_cast<long>((chunks + 3) / 4), static_cast<long>(most)}));
    a.segment_chunks = (chunks + segments - 1) / segments;
    a.segments = (chunks + a.segment_chunks - 1) / a.segment_chunks;
}

template <typename T, int W>
constexpr int kWalkBytes = (3 * kTile<T, W> + kChunk * kPairsPitch<T>) * static_cast<int>(sizeof(T));
template <typename T, int W>
constexpr int kSegmentBytes = 2 * kTile<T, W> * static_cast<int>(sizeof(T));

template <auto Kernel>
int allow_shared(int bytes) {
    if (bytes <= 64 * 1024) return CGPTX_OK;
    static const hipError_t once = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return check_hip(once, "hipFuncSetAttribute");
}

template <typename T, int W, bool DIRECT>
int run(LinearArgs& a, bool backward, hipStream_t stream) {
    const long pairs = static_cast<long>(a.batch) * a.hkv;
    const int group = a.hq / a.hkv, parts = backward ? 2 : 1;
    const std::size_t slots = static_cast<std::size_t>(pairs) * a.d * a.d;
    cut(a, pairs * group, 1 << 20);
    // Segments need scratch; a call that cannot have it all takes fewer, one sequence a walk with none.
    if (a.segments > 1) {
        void* memory = nullptr;
        std::size_t held = 0;
        auto wanted = [&] { return static_cast<std::size_t>(parts) * a.segments * slots * sizeof(float); };
        if (int st = scratch_up_to(stream, wanted(), &memory, &held)) return st;
        while (a.segments > 1 && held < wanted()) cut(a, pairs * group, a.segments - 1);
        a.ahead = static_cast<float*>(memory);
        a.behind = a.ahead + a.segments * slots;
    }
    const bool first = a.segments > 1 || a.after != nullptr, second = backward && (a.segments > 1 || a.d_before != nullptr);
    const int first_part = first ? 0 : 1, count = (first ? 1 : 0) + (second ? 1 : 0);
    if (count > 0) {
        if (int st = allow_shared<linear_segments_kernel<T, W, DIRECT>>(kSegmentBytes<T, W>)) return st;
        hipLaunchKernelGGL((linear_segments_kernel<T, W, DIRECT>), dim3(static_cast<unsigned int>(pairs * a.segments), count), dim3(W * 2), (kSegmentBytes<T, W>), stream, a, first_part);
        CGPTX_LAUNCH_CHECK();
        hipLaunchKernelGGL(linear_join_kernel, dim3(static_cast<unsigned int>((slots + 255) / 256), count), dim3(256), 0, stream, a, first_part);
        CGPTX_LAUNCH_CHECK();
    }
    const long units = pairs * a.segments;
    if (backward) {
        if (int st = allow_shared<linear_backward_kernel<T, W, DIRECT>>(kWalkBytes<T, W>)) return st;
        hipLaunchKernelGGL((linear_backward_kernel<T, W, DIRECT>), dim3(static_cast<unsigned int>(units * (group + 2))), dim3(W * 2), (kWalkBytes<T, W>), stream, a);
    } else {
        if (int st = allow_shared<linear_forward_kernel<T, W, DIRECT>>(kWalkBytes<T, W>)) return st;
        hipLaunchKernelGGL((linear_forward_kernel<T, W, DIRECT>), dim3(static_cast<unsigned int>(units * group)), dim3(W * 2), (kWalkBytes<T, W>), stream, a);
    }
    CGPTX_LAUNCH_CHECK();
    return CGPTX_OK;
}

int run_any(LinearArgs& a, bool backward, bool on_boundaries, int dtype, hipStream_t stream) {
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        a.vectors = on_boundaries && a.d % kVec128<T> == 0;
        if constexpr (sizeof(T) == 2) {
            // 32 bits hold every offset in a chunk.
            if (a.vectors && static_cast<long>(a.hq) * a.d * kChunk * 2 < (1L << 30))
                return a.d <= 64 ? run<T, 64, true>(a, backward, stream) : run<T, 128, true>(a, backward, stream);
        }
        return a.d <= 64 ? run<T, 64, false>(a, backward, stream) : run<T, 128, false>(a, backward, stream);
    });
}

}  // namespace
}  // namespace cgptx

extern "C" int cgptx_linear_attention_forward(void* output, float* final_state, const void* query, const void* key, const void* value,
                                              const float* log_decay, const float* initial_state, size_t batch, size_t sequence,
                                              size_t query_heads, size_t kv_heads, size_t head_dim, float attention_scale, int dtype,
                                              cgptx_stream stream) {
    using namespace cgptx;
    const char* name = "linear_attention_forward";
    const Shape s{batch, sequence, query_heads, kv_heads, head_dim, attention_scale, dtype};
    if (int st = validate(name, s)) return st;
    if (output == nullptr || query == nullptr || key == nullptr || value == nullptr || log_decay == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    if (final_state != nullptr && final_state == initial_state)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": the final state must not be the initial one");
    LinearArgs a = make_args(s, query, key, value, log_decay, initial_state);
    a.out = output;
    a.after = final_state;
    return run_any(a, false, aligned({output, query, key, value}), dtype, static_cast<hipStream_t>(stream));
}

extern "C" int cgptx_linear_attention_backward(void* grad_query, void* grad_key, void* grad_value, float* grad_initial_state,
                                               const void* grad_output, const float* grad_final_state, const void* query, const void* key,
                                               const void* value, const float* log_decay, const float* initial_state, size_t batch,
                                               size_t sequence, size_t query_heads, size_t kv_heads, size_t head_dim,
                                               float attention_scale, int accumulate_grads, int dtype, cgptx_stream stream) {
    using namespace cgptx;
    const char* name = "linear_attention_backward";
    const Shape s{batch, sequence, query_heads, kv_heads, head_dim, attention_scale, dtype};
    if (int st = validate(name, s)) return st;
    if (grad_query == nullptr || grad_key == nullptr || grad_value == nullptr || grad_output == nullptr || query == nullptr || key == nullptr ||
        value == nullptr || log_decay == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    if (grad_initial_state != nullptr && (grad_initial_state == grad_final_state || grad_initial_state == initial_state))
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": the initial state's gradient must be a tensor of its own");
    LinearArgs a = make_args(s, query, key, value, log_decay, initial_state);
    a.dout = grad_output;
    a.dq = grad_query;
    a.dk = grad_key;
    a.dv = grad_value;
    a.d_after = grad_final_state;
    a.d_before = grad_initial_state;
    a.accumulate = accumulate_grads != 0;
    return run_any(a, true, aligned({grad_query, grad_key, grad_value, grad_output, query, key, value}), dtype, static_cast<hipStream_t>(stream));
}

extern "C" int cgptx_linear_attention_step(void* output, float* next_state, const float* state, const void* query, const void* key,
                                           const void* value, const float* log_decay, size_t batch, size_t query_heads, size_t kv_heads,
                                           size_t head_dim, float attention_scale, int dtype, cgptx_stream stream) {
    using namespace cgptx;
    const char* name = "linear_attention_step";
    const Shape s{batch, 1, query_heads, kv_heads, head_dim, attention_scale, dtype};
    if (int st = validate(name, s)) return st;
    if (output == nullptr || next_state == nullptr || state == nullptr || query == nullptr || key == nullptr || value == nullptr ||
        log_decay == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    const int hq = static_cast<int>(query_heads), hkv = static_cast<int>(kv_heads), d = static_cast<int>(head_dim);
    const unsigned int grid = static_cast<unsigned int>(batch * kv_heads) * static_cast<unsigned int>((d + kStepColumns - 1) / kStepColumns);
    const bool vectors = d % 4 == 0 && aligned({next_state, state});
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        auto kernel = vectors ? linear_step_kernel<T, true> : linear_step_kernel<T, false>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(kStepThreads), 0, static_cast<hipStream_t>(stream), static_cast<T*>(output), next_state, state,
                           static_cast<const T*>(query), static_cast<const T*>(key), static_cast<const T*>(value), log_decay, hq, hkv, d,
                           chosen_scale(s));
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}
