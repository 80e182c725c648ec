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
// it is C' X'. The matrix stays in registers from chunk to chunk, 32 of its columns a wavefront, and goes as an operand into its
// product as it lies (the columns of Y are read in the order that makes it so). Where there are fewer sequences than compute units, they are cut into
// segments that workgroups walk side by side: one launch leaves each segment's own matrix, one adds them up along the sequence, and the third starts
// each segment from there.
//
// 16-bit storage: P, C and the decayed Z are rounded to it once where they become operands, sums are fp32. In half precision a power of two
// brings them into its range where they leave it. The matrix in a walk is fed with the decayed Z in two parts, high and low,
// and the matrices that are stored (fp32) with three in bfloat16.
// An Inf or NaN reaches the tokens that see it and no others: chunks that hold one are added up token by token.
// Times in the comments are medians of passes in a row over three sets of inputs, the variants in turn on one card.
#include "attention_tiles.hpp"

#include <cmath>
#include <string>
#include <type_traits>

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

// A lane's offset in a tile, one register for all of a kind of reads: the swizzle only flips bits of it (16-bit storage). `anew` keeps the
// compiler from holding the sums with every step's constant in registers of their own.
__device__ __forceinline__ int anew(int offset) {
    asm volatile("" : "+v"(offset));
    return offset;
}
template <typename T, int W>
__device__ __forceinline__ int row_offset() {
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 2) return wide_direct_offset<W>(lane, 0);
    else return (lane & 31) * kPitch<T, W> + 8 * (lane >> 5);
}
// Row block + lane%32 of a tile, columns 16 step + 8 (lane/32) .. + 7.
template <typename T, int W>
__device__ __forceinline__ frag_t<T> row_frag(const T* tile, int offset, int block, int step) {
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const frag_t<T>*>(tile + block * W + (offset ^ (16 * step)));
    } else {
        const T* from = tile + block * kPitch<T, W> + offset + 16 * step;
        const auto lo = load_vec<T, 4>(from), hi = load_vec<T, 4>(from + 4);
        return frag_t<T>{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
}
// Column 32 t + lane%32 of a tile, rows block + {0-3 | 4-7} and eight further.
template <typename T, int W>
__device__ __forceinline__ frag_t<T> column_frag(const T* tile, int block, int t) {
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 2) {
        return wide_transposed_frag<T>(tile + block * W, wide_transposed_offset<W>(lane, t, 0), wide_transposed_offset<W>(lane, t, 1));
    } else {
        frag_t<T> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = tile[(block + (e & 4) * 2 + 4 * (lane >> 5) + (e & 3)) * kPitch<T, W> + 32 * t + (lane & 31)];
        return f;
    }
}
// The same with the columns of a group of sixteen in the order 0-3, 8-11, 4-7, 12-15, so that a product's registers 8 s .. 8 s + 7 hold rows
// 16 s + 8 (lane/32) .. + 7: those of row_frag.
template <typename T, int W>
__device__ __forceinline__ int swapped_offset() {
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 2) {
        const int row = (lane >> 5) * 4 + ((lane & 15) >> 2), chunk = ((lane >> 4) & 1) * 2 + (lane & 1);
        return row * W + ((chunk ^ swizzle<W>(row)) * 8) + ((lane >> 1) & 1) * 4;
    } else {
        const int m = lane & 31;
        return 4 * (lane >> 5) * kPitch<T, W> + ((m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1));
    }
}
template <typename T, int W>
__device__ __forceinline__ frag_t<T> swapped_frag(const T* tile, int offset, int block, int t) {
    if constexpr (sizeof(T) == 2) {  // eight rows further bit 4 of the offset is flipped
        return wide_transposed_frag<T>(tile + block * W, offset ^ (32 * t), (offset ^ (32 * t) ^ 16) + 8 * W);
    } else {
        frag_t<T> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = tile[(block + (e & 4) * 2 + (e & 3)) * kPitch<T, W> + offset + 32 * t];
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
__device__ __forceinline__ vec_t<unsigned int, 4> load_words(__amdgpu_buffer_rsrc_t rsrc, int voffset, int soffset) {
    return __builtin_bit_cast(vec_t<unsigned int, 4>, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voffset, soffset, 0));
}
__device__ __forceinline__ void store_words(vec_t<unsigned int, 4> words, __amdgpu_buffer_rsrc_t rsrc, int voffset) {
    __builtin_amdgcn_raw_buffer_store_b128(words, rsrc, voffset, 0, 0);
}
// Rows row0 .. row0 + 63 of a head on their way to a tile, zeros behind the last token and behind column d. STAGED (16-bit storage on 16-byte
// boundaries): fetch asks for them, and they wait in registers until store. (Loads straight into LDS would save the registers, but every
// transposing read of another tile waits for them.)
template <typename T, int W, bool STAGED, int THREADS>
struct Incoming {
    static constexpr int kChunks = W / 8;  // of a row
    static constexpr int kRows = THREADS / kChunks, kPieces = kChunk / kRows;
    Rows<T> rows;
    int row0;
    __amdgpu_buffer_rsrc_t rsrc;
    int voffset, further;  // a lane's first piece; bytes to its next one, kRows on
    vec_t<unsigned int, 4> piece[STAGED ? kPieces : 1];

    __device__ __forceinline__ Incoming(long stride, int d) {
        if constexpr (STAGED) {
            const int row_bytes = static_cast<int>(stride) * 2, r = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks;
            voffset = chunk * 8 < d ? r * row_bytes + chunk * 16 : 1 << 30;
            further = kRows * row_bytes;
        }
    }
    // Says which rows; the pieces of STAGED are asked for, and stored, one by one.
    __device__ __forceinline__ void set(const Rows<T>& from, int first, int tokens, int d) {
        rows = from;
        row0 = first;
        if constexpr (STAGED)
            rsrc = buffer_of(rows.base + static_cast<long>(row0) * rows.stride, (min(kChunk, tokens - row0) - 1) * static_cast<int>(rows.stride) * 2 + d * 2);
    }
    __device__ __forceinline__ void fetch(int i) {
        if constexpr (STAGED) piece[i] = load_words(rsrc, voffset, i * further);
    }
    __device__ __forceinline__ void store(int i, T* tile, int tokens, int d, bool vectors) const {
        if constexpr (STAGED) {
            const int r = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks;
            *reinterpret_cast<vec_t<unsigned int, 4>*>(tile + (r + i * kRows) * W + ((chunk ^ swizzle<W>(r)) * 8)) = piece[i];
        } else if (i == 0) {
            const T* first = rows.base + static_cast<long>(row0) * rows.stride;
            const int left = min(kChunk, tokens - row0);
            constexpr int VEC = kVec128<T>, kVectors = W / VEC;
#pragma unroll 4
            for (int n = threadIdx.x; n < kChunk * kVectors; n += THREADS) {
                const int r = n / kVectors, p = n % kVectors, column = p * VEC;
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
                if constexpr (sizeof(T) == 2) store_vec<T, VEC>(tile + r * W + ((p ^ swizzle<W>(r)) * 8), v);
                else store_vec<T, VEC>(tile + r * kPitch<T, W> + column, v);
            }
        }
    }
};

// log2 of the decay. No growth: what is above 1 counts as 1. A head that forgets everything (-inf) has 0^0 = 1.
__device__ __forceinline__ float log2_decay(float log_decay) {
    const float l = log_decay * kLog2e;
    return l > 0.0f ? 0.0f : l < -1.0e4f ? -1.0e4f : l;  // a NaN stays one
}
__device__ __forceinline__ float power(float l, int n) { return __builtin_amdgcn_exp2f(l * static_cast<float>(n)); }

// Half precision: the power of two that brings a largest magnitude into 2^low .. 2^high, 1 where it is there already (or zero, or not finite).
__device__ __forceinline__ float range_scale(float largest, int low, int high) {
    const int e = static_cast<int>((__float_as_uint(largest) >> 23) & 0xFF) - 127;
    if (e >= 128 || e <= -127 || (e >= low && e < high)) return 1.0f;
    const int target = e < low ? low : high - 1;
    return __uint_as_float(static_cast<unsigned int>(min(max(target - e, -126), 126) + 127) << 23);
}
// The largest finite magnitude that walk(use) hands out in a wavefront.
template <typename Walk>
__device__ __forceinline__ float largest_finite(Walk&& walk) {
    float most = 0.0f;
    walk([&](float value) __attribute__((always_inline)) { most = fmaxf(most, fabsf(value)); });
    most = wave_max(most);
    if (most == __builtin_inff()) {
        most = 0.0f;
        walk([&](float value) __attribute__((always_inline)) { most = fabsf(value) < __builtin_inff() ? fmaxf(most, fabsf(value)) : most; });
        most = wave_max(most);
    }
    return most;
}
template <typename T>
constexpr bool kNarrow = __is_same(T, f16_t);  // a range that sums leave

// Z of a wavefront's 32 columns: four operands of sixteen rows.
template <typename T>
struct Values {
    frag_t<T> z[4];
    template <int W>
    __device__ __forceinline__ void load(const T* tile, int column_block, int first = 0, int count = 4) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s >= first && s < first + count) z[s] = column_frag<T, W>(tile, 16 * s, column_block);
    }
    // 16-bit storage: the largest magnitude's bits in each half of a word.
    __device__ __forceinline__ unsigned int largest_bits() const {
        using Halves = vec_t<unsigned short, 2>;
        Halves most(static_cast<unsigned short>(0));
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const auto words = __builtin_bit_cast(vec_t<unsigned int, 2 * sizeof(T)>, z[s]);
#pragma unroll
            for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(Halves, words[w] & 0x7FFF7FFFu));
        }
        return __builtin_bit_cast(unsigned int, most);
    }
    __device__ __forceinline__ bool finite() const {
        if constexpr (sizeof(T) == 4) {
            float sum = 0.0f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(z[s][e], 0.0f, sum);
            return sum == 0.0f;
        } else {
            constexpr unsigned int kInf = kNarrow<T> ? 0x7C00u : 0x7F80u;
            const unsigned int most = largest_bits();
            return (most & 0xFFFFu) < kInf && (most >> 16) < kInf;
        }
    }
    // Half precision: the largest finite magnitude in the wavefront.
    __device__ __forceinline__ float largest() const {
        unsigned int bits = largest_bits();
        bits = max(bits & 0xFFFFu, bits >> 16);
        if (__any(bits >= 0x7C00u))
            return largest_finite([&](auto&& use) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) use(to_f32(z[s][e]));
            });
        return wave_max(to_f32(__builtin_bit_cast(f16_t, static_cast<unsigned short>(bits))));
    }
};

// Weights of a chunk's tokens as what follows the chunk sees them (forward in time: 1 for token `end`, else g^(end - token); backward: g^(token
// + 1)), for the rows that a lane's operands hold in COUNT steps of sixteen from `first` on.
template <int COUNT>
struct Weights {
    vec_t<float, 8> w[COUNT];
    __device__ __forceinline__ static int row(int e) { return 4 * ((threadIdx.x & 63) >> 5) + (e & 3) + 2 * (e & 4); }
    __device__ __forceinline__ Weights(float l, float scale, bool reverse, int end, int first = 0) {
#pragma unroll
        for (int s = 0; s < COUNT; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = 16 * (first + s) + row(e);
                w[s][e] = scale * power(l, reverse ? at + 1 : max(end - at, 0));
            }
    }
};

// w Z of sixteen rows as operands, made in eight steps. 16-bit storage: two parts leave 2^-16 of it in bfloat16 and 2^-22 in half precision, a
// third one 2^-24.
template <typename T, int PARTS>
struct Weighted {
    static constexpr int kParts = sizeof(T) == 4 ? 1 : kNarrow<T> ? 2 : PARTS;
    vec_t<T, 2> part[kParts][4];
    vec_t<float, 2> rest[4];
    __device__ __forceinline__ void step(int i, const frag_t<T>& z, const vec_t<float, 8>& w, float up) {
        const int j = i / 2;
        if (i % 2 == 0) {
            rest[j] = vec_t<float, 2>{to_f32(z[2 * j]) * w[2 * j], to_f32(z[2 * j + 1]) * w[2 * j + 1]};
            if constexpr (kNarrow<T>) rest[j] *= up;
            part[0][j] = vec_from_f32<T, 2>(rest[j]);
        } else {
#pragma unroll
            for (int n = 1; n < kParts; ++n) {
                rest[j] -= vec_to_f32<T, 2>(part[n - 1][j]);
                part[n][j] = vec_from_f32<T, 2>(rest[j]);
            }
        }
    }
    __device__ __forceinline__ frag_t<T> operand(int n) const {
        return frag_t<T>{part[n][0][0], part[n][0][1], part[n][1][0], part[n][1][1], part[n][2][0], part[n][2][1], part[n][3][0], part[n][3][1]};
    }
};
template <typename T, int W, int K>
__device__ __forceinline__ void read_rows_of(frag_t<T> (&y)[K], const T* tile, int offset, int s) {
#pragma unroll
    for (int k = 0; k < K; ++k) y[k] = swapped_frag<T, W>(tile, offset, 16 * s, k);
}
// matrix += Y' (w Z) for sixteen rows, operand(n) one of kParts parts of w Z; between(i, count) follows the i-th matrix instruction of `count`.
template <typename T, int K, int PARTS, typename Operand, typename Between>
__device__ __forceinline__ void add_rows(acc_t (&matrix)[K], const frag_t<T> (&y)[K], Operand&& operand, Between&& between) {
    constexpr int kParts = Weighted<T, PARTS>::kParts;
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
        const frag_t<T> part = operand(n);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            matrix[k] = multiply<T>(y[k], part, matrix[k]);
            between(n * K + k, kParts * K);
        }
    }
}
// The steps of `all` that come behind instruction i of `count`.
template <typename Step>
__device__ __forceinline__ void share_of(int all, int i, int count, Step&& step) {
#pragma unroll
    for (int n = 0; n < all; ++n)
        if (n * count / all == i) step(n);
}
// Half precision: values are weighted at the upper end of its range (the two parts of one that is 2^-17 of the largest still leave 2^-22 of it), the
// matrix along with them until it is brought back.
template <typename T, int K>
__device__ __forceinline__ void enlarge(acc_t (&matrix)[K], float up) {
    if (kNarrow<T> && up != 1.0f)
#pragma unroll
        for (int k = 0; k < K; ++k) matrix[k] *= up;
}
// For outputs in half precision: by the largest value times the largest weight, and not by more than 2^30, or than a state at the end of fp32's
// range leaves: matrix_scale has brought the matrix below 2^15, and a group's heads add less than 2^92 where they are enlarged at all.
template <typename T, int K>
__device__ __forceinline__ float enlarge_by_values(acc_t (&matrix)[K], float matrix_scale, const Values<T>& values, float largest_weight) {
    if constexpr (!kNarrow<T>) return 1.0f;
    const float up = fminf(range_scale(values.largest() * largest_weight, 14, 15), fminf(0x1p110f * matrix_scale, 0x1p30f));
    enlarge<T, K>(matrix, up);
    return up;
}
// For matrices that are stored: by the largest weighted value, however small (a chunk whose last values are zeros, weights that begin below 2^-30).
// `size`, what the matrix cannot exceed, leaves it room: 64 values of less than 2^16 each add 2^22 times the largest weighted one at most.
template <typename T, int K>
__device__ __forceinline__ float enlarge_by_products(acc_t (&matrix)[K], float& size, const Values<T>& values, const Weights<4>& weights) {
    if constexpr (!kNarrow<T>) return 1.0f;
    const float largest = largest_finite([&](auto&& use) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) use(to_f32(values.z[s][e]) * weights.w[s][e]);
    });
    const float room = __uint_as_float(__float_as_uint(0x1p120f / size) & 0x7F800000u);  // a power of two, 2^-6 or more
    const float up = fminf(range_scale(largest, 14, 15), room);
    size = fminf(fmaf(largest, 0x1p22f, size), 0x1p126f);
    enlarge<T, K>(matrix, up);
    return up;
}
template <typename T, int K>
__device__ __forceinline__ void bring_back(acc_t (&matrix)[K], float up) {
    if (kNarrow<T> && up != 1.0f)
#pragma unroll
        for (int k = 0; k < K; ++k) matrix[k] *= 1.0f / up;
}

template <int K>
__device__ __forceinline__ float largest_of(const acc_t (&matrix)[K]) {
    return largest_finite([&](auto&& use) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) use(matrix[k][i]);
    });
}
// The matrix that a walk starts from: `factor` times the stored one, zeros for none. A wavefront has 32 columns and rows
// from first_row on.
template <int K>
__device__ __forceinline__ void load_matrix(acc_t (&matrix)[K], const float* from, float factor, bool transposed, int d, int column_block, int first_row) {
    const int column = column_block * 32 + (threadIdx.x & 31), row0 = first_row + matrix_row(0);
    const __amdgpu_buffer_rsrc_t rsrc = buffer_of(from, from != nullptr ? d * d * 4 : 0);  // reads behind its end give zeros
    const int row_step = (transposed ? 1 : d) * 4, first = (transposed ? column * d + row0 : row0 * d + column) * 4;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int further = 32 * k + 16 * (i >> 3) + (i & 7);  // rows
            const int at = column < d && row0 + further < d ? first + further * row_step : 1 << 30;
            matrix[k][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, 0)) * factor;
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
    int heads_each;  // query heads that a workgroup takes one after the other, of a group
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

template <int W>
__device__ __forceinline__ int column_block_of() {
    return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % (W / 32);
}
// A lane's offset further by `columns`, a power of two that no read adds by itself.
template <typename T>
__device__ __forceinline__ int along(int offset, int columns) {
    return sizeof(T) == 2 ? offset ^ columns : offset + columns;
}

// The output of one head in one segment. Two wavefronts have the same 32 columns of Z, the matrix and the output, each half of the matrix's rows and
// half of a chunk's tokens: W/2 x 32 and 32 x 32 in registers (fp32, whose operands are twice as large, spills 16 to 55 registers of 256). In a
// chunk: scores of the pairs, by three wavefronts, and what came before it, where each has half of both sums and leaves the other's to it | all is
// there, X and Z have been read, the next chunk's are on their way (Y has two buffers in 16-bit storage) | products with Z, the matrix, the output |
// the next chunk is there. What bounds it is how long these steps wait for each other (32 sequences of 1024 tokens, 8 and 2 heads of 128: the matrix
// cores are busy for 23 per cent of the launch, forward and backward). With a wavefront for both halves a chunk has half the instructions in all and
// takes as long where 16 chunks follow each other (that case: 61 us forward, 148 backward; with two 62 and 143), and longer where there are few (77
// tokens of half precision: 11.1 us, with two 9.1; fp32, 2 x 333 tokens, backward: 37, with two 31).
template <typename T, int W>
constexpr int kWalkThreads = W * 4;
template <typename T>
constexpr int kYTiles = sizeof(T) == 2 ? 2 : 1;
template <typename T>
constexpr bool kShares = sizeof(T) == 2;  // the weighted Z of the wavefronts of a column block: two steps of sixteen rows each, by the LDS
template <typename T, int W, bool REVERSE, bool STAGED>
__device__ __forceinline__ void walk_segment(const LinearArgs& a, const Task<T>& task, int b, int head, int segment, T* lds) {
    constexpr int kBlocks = W / 32, K = kBlocks / 2, kSeesBoth = REVERSE ? 0 : 1;  // the half of the tokens that sees both
    using In = Incoming<T, W, STAGED, kWalkThreads<T, W>>;
    constexpr int kPieces = In::kPieces;
    T *x_tile = lds, *z_tile = lds + kTile<T, W>, *y_tiles = lds + 2 * kTile<T, W>, *pairs = y_tiles + kYTiles<T> * kTile<T, W>;
    float* halves = reinterpret_cast<float*>(pairs + kChunk * kPairsPitch<T>);
    T* weighted_z = reinterpret_cast<T*>(halves + kWalkThreads<T, W> * 16) + column_block_of<W>() * 8 * 512;
    __shared__ float pair_scales[3];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int column_block = column_block_of<W>(), mine = wave / kBlocks, place = mine * 32 + (lane & 31);
    const int d = a.d, tokens = a.tokens;
    const int group = a.hq / a.hkv, heads_each = REVERSE ? group : a.heads_each;
    const int kv = REVERSE ? head : head / group, y_first = REVERSE ? head * group : kv;
    const float l = log2_decay(a.log_decay[kv]);

    const long x_stride = static_cast<long>(task.x_heads) * d, y_stride = static_cast<long>(task.y_heads) * d;
    const Rows<T> x{task.x + static_cast<long>(b) * tokens * x_stride + static_cast<long>(head) * d, x_stride};
    const long y_offset = static_cast<long>(b) * tokens * y_stride + static_cast<long>(y_first) * d;
    const Rows<T> y{task.y + y_offset, y_stride}, z{task.z + y_offset, y_stride};

    const int chunks_in_all = (tokens + kChunk - 1) / kChunk;
    const int first_chunk = segment * a.segment_chunks, last_chunk = min(first_chunk + a.segment_chunks, chunks_in_all) - 1;
    const int steps = last_chunk - first_chunk + 1;
    auto row_of = [&](int step) { return (REVERSE ? last_chunk - step : first_chunk + step) * kChunk; };
    In in_x(x_stride, d), in_y(y_stride, d), in_z(y_stride, d);
    // Forward in time the heads of a group share Y and Z, backward X and the output.
    auto turn_to = [&](int step, int each) __attribute__((always_inline)) {
        const int row0 = row_of(step);
        const long further = static_cast<long>(each) * d, x_further = REVERSE ? 0 : further, y_further = REVERSE ? further : 0;
        in_x.set(Rows<T>{x.base + x_further, x.stride}, row0, tokens, d);
        in_y.set(Rows<T>{y.base + y_further, y.stride}, row0, tokens, d);
        in_z.set(Rows<T>{z.base + y_further, z.stride}, row0, tokens, d);
    };
    int buffer = 0;
    turn_to(0, 0);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
        in_x.fetch(n);
        in_y.fetch(n);
        in_z.fetch(n);
    }

    // The 32 x 32 tile of pairs that a wavefront makes: 0 and 1 on the diagonal, 2 the one beside it.
    const bool makes_pairs = wave < 3;
    const int tile = min(wave, 2), tile_t = tile == 2 ? kSeesBoth : tile, tile_r = tile == 2 ? 1 - kSeesBoth : tile;
    acc_t table;
    unsigned int seen[8];  // bfloat16: masks of two elements each
    constexpr float kHidden = __is_same(T, bf16_t) ? 0.0f : -1.0f;  // a weight that is seen may round to 0, but is never below it
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int t = tile_t * 32 + (lane & 31), r = tile_r * 32 + acc_row(i), far = REVERSE ? r - t : t - r;
        table[i] = far >= 0 ? task.pair_scale * power(l, far) : kHidden;
        if (i % 2 == 0) seen[i / 2] = 0;
        if (far >= 0) seen[i / 2] |= i % 2 == 0 ? 0xFFFFu : 0xFFFF0000u;
    }
    const Weights<kShares<T> ? 2 : 4> weights(l, task.matrix_scale, REVERSE, kChunk, kShares<T> ? 2 * mine : 0);
    const float largest_weight = REVERSE ? task.matrix_scale * power(l, 1) : 1.0f;

    acc_t matrix[K];
    load_matrix<K>(matrix, task.carry, task.carry_factor, task.transposed, d, column_block, mine * 32 * K);
    const int row_at = row_offset<T, W>(), swapped_at = along<T>(swapped_offset<T, W>(), mine * 32 * K);
    T* const out = task.out + static_cast<long>(b) * tokens * x_stride + static_cast<long>(head) * d;
    // Eight columns of four of a chunk's output, twice (quarter 0, 1). Rows and columns that are not there lie behind the end of a buffer, where
    // stores are dropped.
    auto store_output = [&](int quarter, const acc_t& o, const acc_t& within, float since, T* out, int row0, int length) __attribute__((always_inline)) {
        const int g = quarter * 2;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(o[4 * g + e], since, within[4 * g + e]);
        T* first = out + row0 * x_stride;
        if constexpr (STAGED) {
            const __amdgpu_buffer_rsrc_t rsrc = buffer_of(first, static_cast<int>(((length - 1) * x_stride + d) * static_cast<long>(sizeof(T))));
            // A lane has quads of its row's columns, its partner in the other half of the wavefront the quads between: swapped, each has eight in a
            // row.
            const int at = column_block * 32 + 8 * (g + half), row = place * static_cast<int>(x_stride * sizeof(T));
            vec_t<float, 8> all;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[e]), __float_as_uint(v[4 + e]), false, false);
                all[e] = __uint_as_float(swapped[0]);
                all[4 + e] = __uint_as_float(swapped[1]);
            }
            store_words(__builtin_bit_cast(vec_t<unsigned int, 4>, vec_from_f32<T, 8>(all)), rsrc, place < length && at < d ? row + at * 2 : 1 << 30);
        } else {
            if (place >= length) return;
            T* to = first + place * x_stride;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int at = column_block * 32 + 8 * (g + q) + 4 * half;
                if (a.vectors) {
                    if (at < d) store_vec<T, 4>(to + at, vec_from_f32<T, 4>(vec_t<float, 4>{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]}));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e < d) to[at + e] = from_f32<T>(v[4 * q + e]);
                }
            }
        }
    };
    auto store_x = [&](int n) __attribute__((always_inline)) { in_x.store(n, x_tile, tokens, d, a.vectors); };
    auto store_y = [&](int n) __attribute__((always_inline)) { in_y.store(n, y_tiles + buffer * kTile<T, W>, tokens, d, a.vectors); };
    auto store_z = [&](int n) __attribute__((always_inline)) { in_z.store(n, z_tile, tokens, d, a.vectors); };
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
        store_x(n);
        store_y(n);
        store_z(n);
    }
    for (int step = 0; step < steps; ++step) {
        const int row0 = row_of(step), length = min(kChunk, tokens - row0);
        acc_t o, within;  // by what came before the chunk, and by its own tokens
        float since, matrix_scale = 1.0f;
        for (int each = 0; each < heads_each; ++each) {
            const T* y_tile = y_tiles + buffer * kTile<T, W>;
            const bool last_each = each + 1 == heads_each, update = REVERSE || last_each, before = !REVERSE || each == 0;
            T* const out_each = REVERSE ? out : out + static_cast<long>(each) * d;
            __syncthreads();  // the tiles are there

            // The next tiles are asked for (behind the last ones, those once more), X alone where the next head shares Y and Z.
            turn_to(last_each ? min(step + 1, steps - 1) : step, last_each ? 0 : each + 1);
            auto fetch = [&](int n) __attribute__((always_inline)) {
                if (n < kPieces) in_x.fetch(n);
                else if (n < 2 * kPieces) in_y.fetch(n - kPieces);
                else in_z.fetch(n - 2 * kPieces);
            };
            constexpr int AHEAD = 2;
            const int at = anew(row_at);
            // P' = (Y X') g^..
            if (makes_pairs) {
                constexpr int STEPS = W / 16;
                frag_t<T> xs[AHEAD + 1], ys[AHEAD + 1];
                auto read = [&](int s) __attribute__((always_inline)) {
                    xs[s % (AHEAD + 1)] = row_frag<T, W>(x_tile, at, 32 * tile_t, s);
                    ys[s % (AHEAD + 1)] = row_frag<T, W>(y_tile, at, 32 * tile_r, s);
                };
#pragma unroll
                for (int s = 0; s < AHEAD; ++s) read(s);
                acc_t p(0.0f);
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    if (s + AHEAD < STEPS) read(s + AHEAD);
                    p = multiply<T>(ys[s % (AHEAD + 1)], xs[s % (AHEAD + 1)], p);
                }
                // What the mask hides is 0 whatever the scores are; what has decayed to 0 is not where they are not finite.
                if constexpr (__is_same(T, bf16_t)) {
                    p *= table;
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float weight = table[i];
                        asm volatile("" : "+v"(weight));  // compared anew: no registers for sixteen masks
                        p[i] = weight < 0.0f ? 0.0f : p[i] * weight;
                    }
                }
                if constexpr (kNarrow<T>) {
                    const float scale = range_scale(largest_finite([&](auto&& use) __attribute__((always_inline)) {
#pragma unroll
                                                        for (int i = 0; i < 16; ++i) use(p[i]);
                                                    }),
                                                    -3, 15);
                    p *= scale;
                    pair_scales[tile] = scale;
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    frag_t<T> part = operand_of<T>(p, s);
                    if constexpr (__is_same(T, bf16_t)) {
                        auto words = __builtin_bit_cast(vec_t<unsigned int, 4>, part);
#pragma unroll
                        for (int w = 0; w < 4; ++w) words[w] &= seen[4 * s + w];
                        part = __builtin_bit_cast(frag_t<T>, words);
                    }
                    *reinterpret_cast<frag_t<T>*>(pairs_at<T>(pairs, tile_t * 32 + (lane & 31), 4 * tile_r + 2 * s + half)) = part;
                }
            }
            // C' X' of the wavefront's rows of C, for its own tokens and for the other half's. Once the matrix has been read it decays.
            Values<T> values;
            if (before) {
                constexpr int STEPS = W / 32;
                const int rows_at = along<T>(at, mine * 16 * STEPS);
                if constexpr (kNarrow<T>) matrix_scale = range_scale(largest_of(matrix), -3, 15);
                const float passed = update ? power(l, length) : 1.0f;
                frag_t<T> xs[AHEAD + 1][2], m[2];
                auto fetch_some = [&](int i, int count) __attribute__((always_inline)) {
                    share_of(kPieces, i, count, fetch);
                    if (update) share_of(2 * kPieces, i, count, [&](int n) __attribute__((always_inline)) { fetch(kPieces + n); });
                };
                auto read = [&](int s) __attribute__((always_inline)) {
                    xs[s % (AHEAD + 1)][0] = row_frag<T, W>(x_tile, rows_at, 32 * mine, s);
                    xs[s % (AHEAD + 1)][1] = row_frag<T, W>(x_tile, rows_at, 32 - 32 * mine, s);
                };
                auto operand = [&](int s) __attribute__((always_inline)) {
                    acc_t from = matrix[s / 2];
                    if constexpr (kNarrow<T>) from *= matrix_scale;
                    m[s % 2] = operand_of<T>(from, s % 2);
                };
#pragma unroll
                for (int s = 0; s < AHEAD; ++s) read(s);
                operand(0);
                acc_t other(0.0f);
                o = acc_t(0.0f);
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    if (s + AHEAD < STEPS) read(s + AHEAD);
                    else values.template load<W>(z_tile, column_block, 2 * (s + AHEAD - STEPS), 2);
                    other = multiply<T>(m[s % 2], xs[s % (AHEAD + 1)][1], other);
                    if (s + 1 < STEPS) operand(s + 1);
                    fetch_some(2 * s, 2 * STEPS);
                    o = multiply<T>(m[s % 2], xs[s % (AHEAD + 1)][0], o);
#pragma unroll
                    for (int e = 0; e < 8; ++e) matrix[s / 2][8 * (s % 2) + e] *= passed;
                    fetch_some(2 * s + 1, 2 * STEPS);
                }
                if constexpr (kNarrow<T>) {
                    o *= 1.0f / matrix_scale;
                    other *= 1.0f / matrix_scale;
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    store_vec<float, 4>(halves + ((wave * 4 + n) * 64 + lane) * 4, vec_t<float, 4>{other[4 * n], other[4 * n + 1], other[4 * n + 2], other[4 * n + 3]});
                since = task.out_scale * power(l, max(REVERSE ? length - 1 - place : place, 0));
                within = acc_t(0.0f);
                if (a.accumulate && place < length) {
                    const T* from = out_each + (row0 + place) * x_stride;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int column = column_block * 32 + acc_row(i);
                        if (column < d) within[i] += to_f32(from[column]);
                    }
                }
            } else {
                values.template load<W>(z_tile, column_block);
#pragma unroll
                for (int n = 0; n < 3 * kPieces; ++n) fetch(n);
            }
            const bool finite = !__any(!values.finite());
            const float up = update ? enlarge_by_values<T, K>(matrix, matrix_scale, values, largest_weight) : 1.0f;
            if (kShares<T> && update)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    Weighted<T, 2> weighted;
                    const frag_t<T> z = mine != 0 ? values.z[2 + s] : values.z[s];
#pragma unroll
                    for (int i = 0; i < 8; ++i) weighted.step(i, z, weights.w[s], up);
#pragma unroll
                    for (int n = 0; n < 2; ++n) *reinterpret_cast<frag_t<T>*>(weighted_z + ((4 * mine + 2 * s + n) * 64 + lane) * 8) = weighted.operand(n);
                }
            __syncthreads();  // all pairs, halves and weighted Z are there, X and Z have been read
            if (before)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const auto v = load_vec<float, 4>(halves + (((wave ^ kBlocks) * 4 + n) * 64 + lane) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * n + e] += v[e];
                }
            auto pair_frag = [&](int r, int s) { return *reinterpret_cast<const frag_t<T>*>(pairs_at<T>(pairs, place, 4 * r + 2 * s + half)); };
            Values<T> shown = values;
            if (!finite) {
                // A pair that the mask hides is 0, but 0 x Inf is NaN in a product of tiles: token by token, for those that see it.
#pragma unroll 1
                for (int r = 0; r < kChunk; ++r) {
                    const int tr = r >> 5;
                    if (tr != mine && mine != kSeesBoth) continue;
                    float scale = 1.0f;
                    if constexpr (kNarrow<T>) scale = 1.0f / pair_scales[tr == mine ? tr : 2];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        if ((r >> 4) != n) continue;
                        frag_t<T> one = values.z[n];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (Weights<1>::row(e) != (r & 15)) one[e] = static_cast<T>(0.0f);
                        const acc_t term = multiply<T>(one, pair_frag(n / 2, n % 2), acc_t(0.0f));
#pragma unroll
                        for (int i = 0; i < 16; ++i) within[i] = (REVERSE ? r >= place : r <= place) ? fmaf(term[i], scale, within[i]) : within[i];
                    }
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) shown.z[s] = frag_t<T>(static_cast<T>(0.0f));
            }
            frag_t<T> seen_pairs[2][2], own[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                own[s] = mine != 0 ? shown.z[2 + s] : shown.z[s];
                seen_pairs[0][s] = pair_frag(mine, s);
                seen_pairs[1][s] = pair_frag(1 - kSeesBoth, s);
            }
            // between(i) follows the i-th of two products. Half precision: a tile's products, whose scale may be anything up to 2^123 where all its pairs
            // have decayed, are added up apart; `within` itself keeps its range.
            auto add_pairs = [&](auto&& between) __attribute__((always_inline)) {
                auto scaled = [&](int tile, auto&& add) __attribute__((always_inline)) {
                    if constexpr (kNarrow<T>) {
                        acc_t sum(0.0f);
                        add(sum);
                        const float back = 1.0f / pair_scales[tile];
#pragma unroll
                        for (int i = 0; i < 16; ++i) within[i] = fmaf(sum[i], back, within[i]);
                    } else {
                        add(within);
                    }
                };
                scaled(mine, [&](acc_t& sum) __attribute__((always_inline)) {
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        sum = multiply<T>(own[s], seen_pairs[0][s], sum);
                        between(s);
                    }
                });
                if (mine == kSeesBoth)
                    scaled(2, [&](acc_t& sum) __attribute__((always_inline)) {
#pragma unroll
                        for (int s = 0; s < 2; ++s) sum = multiply<T>(shown.z[2 * (1 - kSeesBoth) + s], seen_pairs[1][s], sum);
                    });
            };
            if (!update) {
                add_pairs([&](int i) __attribute__((always_inline)) { share_of(kPieces, i, 2, store_x); });
#pragma unroll
                for (int g = 0; g < 2; ++g) store_output(g, o, within, since, out_each, row0, length);
                continue;
            }
            Weighted<T, 2> weighted[kShares<T> ? 1 : 2];
            frag_t<T> rows[2][K], shared[2][2];
            const int swapped = anew(swapped_at);
            // Step s of what the matrix gets: Y's columns and, where it is shared, the weighted Z.
            auto read = [&](int s) __attribute__((always_inline)) {
                read_rows_of<T, W>(rows[s % 2], y_tile, swapped, s);
                if constexpr (kShares<T>)
#pragma unroll
                    for (int n = 0; n < 2; ++n) shared[s % 2][n] = *reinterpret_cast<const frag_t<T>*>(weighted_z + ((2 * s + n) * 64 + lane) * 8);
            };
            read(0);
            add_pairs([&](int i) __attribute__((always_inline)) {
                if constexpr (!kShares<T>)
                    share_of(8, i, 2, [&](int n) __attribute__((always_inline)) { weighted[0].step(n, values.z[0], weights.w[0], up); });
            });
            if constexpr (kYTiles<T> == 2) buffer ^= 1;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (s < 3) read(s + 1);
                auto operand = [&](int n) __attribute__((always_inline)) {
                    if constexpr (kShares<T>) return shared[s % 2][n];
                    else return weighted[s % 2].operand(n);
                };
                add_rows<T, K, 2>(matrix, rows[s % 2], operand, [&](int i, int count) __attribute__((always_inline)) {
                    if constexpr (!kShares<T>)
                        if (s < 3)
                            share_of(8, i, count, [&](int n) __attribute__((always_inline)) { weighted[(s + 1) % 2].step(n, values.z[s + 1], weights.w[s + 1], up); });
                    if (s >= 1)
                        share_of(kPieces, (s - 1) * count + i, 3 * count, [&](int n) __attribute__((always_inline)) {
                            store_x(n);
                            store_z(n);
                            if constexpr (kYTiles<T> == 2) store_y(n);
                        });
                    if constexpr (!REVERSE)
                        if (s == 3)
                            share_of(2, i, count, [&](int n) __attribute__((always_inline)) { store_output(n, o, within, since, out_each, row0, length); });
                });
            }
            bring_back<T, K>(matrix, up);
            if constexpr (kYTiles<T> == 1) {
                __syncthreads();  // Y has been read
#pragma unroll
                for (int n = 0; n < kPieces; ++n) store_y(n);
            }
        }
        if constexpr (REVERSE)
#pragma unroll
            for (int g = 0; g < 2; ++g) store_output(g, o, within, since, out, row0, length);
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

// A segment's own matrix: what its tokens leave to those behind it (k v') or, reverse, before it (q dO' of the group's heads). The last one's goes
// to `after` as its last token sees it, the first one's to d_before, each where the caller asked for it; a sequence's only one with what is passed
// on through it.
template <typename T, int W, bool STAGED, int HALVES>
__device__ __forceinline__ void sum_segment(const LinearArgs& a, bool reverse, int pair, int segment, T* lds) {
    constexpr int kBlocks = W / 32, K = kBlocks / HALVES;
    using In = Incoming<T, W, STAGED, W * 2 * HALVES>;
    constexpr int kPieces = In::kPieces;
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
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), column_block = wave % kBlocks, first_row = wave / kBlocks * 32 * K;
    const float l = log2_decay(a.log_decay[kv]);
    Weights<4> weights(l, reverse ? a.scale : 1.0f, reverse, kChunk);
    float size = 0.0f;
    const int heads = reverse ? a.hq : a.hkv, heads_each = reverse ? a.hq / a.hkv : 1;
    const long stride = static_cast<long>(heads) * d;
    const T* y_base = static_cast<const T*>(reverse ? a.q : a.k) + static_cast<long>(b) * tokens * stride + static_cast<long>(kv) * heads_each * d;
    const T* z_base = static_cast<const T*>(reverse ? a.dout : a.v) + static_cast<long>(b) * tokens * stride + static_cast<long>(kv) * heads_each * d;

    acc_t matrix[K];
#pragma unroll
    for (int k = 0; k < K; ++k) matrix[k] = acc_t(0.0f);
    const int first_chunk = segment * a.segment_chunks, last_chunk = min(first_chunk + a.segment_chunks, (tokens + kChunk - 1) / kChunk) - 1;
    const int steps = (last_chunk - first_chunk + 1) * heads_each;  // a chunk's heads one after the other
    auto row_of = [&](int step) { return (reverse ? last_chunk - step / heads_each : first_chunk + step / heads_each) * kChunk; };
    In in_y(stride, d), in_z(stride, d);
    auto turn_to = [&](int step) __attribute__((always_inline)) {
        const long further = static_cast<long>(step % heads_each) * d;
        in_y.set(Rows<T>{y_base + further, stride}, row_of(step), tokens, d);
        in_z.set(Rows<T>{z_base + further, stride}, row_of(step), tokens, d);
    };
    auto fetch = [&](int i) __attribute__((always_inline)) {
        in_y.fetch(i);
        in_z.fetch(i);
    };
    auto store_tiles = [&](int i, int step) __attribute__((always_inline)) {
        T* tiles = lds + (step & 1) * 2 * kTile<T, W>;
        in_y.store(i, tiles, tokens, d, a.vectors);
        in_z.store(i, tiles + kTile<T, W>, tokens, d, a.vectors);
    };
    const int swapped_at = along<T>(swapped_offset<T, W>(), first_row);
    turn_to(0);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) fetch(i);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) store_tiles(i, 0);
    for (int step = 0; step < steps; ++step) {
        const T* tiles = lds + (step & 1) * 2 * kTile<T, W>;
        const int row0 = row_of(step), length = min(kChunk, tokens - row0);
        const int end = outermost && !reverse && row0 + kChunk >= tokens ? length - 1 : length;  // the token that sees weight 1
        __syncthreads();  // the tiles are there
        turn_to(min(step + 1, steps - 1));  // (behind the last ones, those once more)
        Values<T> values;
        frag_t<T> rows[2][K];
        Weighted<T, 3> weighted[2];
        const int swapped = anew(swapped_at);
        values.template load<W>(tiles + kTile<T, W>, column_block);
        read_rows_of<T, W>(rows[0], tiles, swapped, 0);
        if (step % heads_each == 0) {
            const float passed = power(l, end);
            size *= passed;
#pragma unroll
            for (int k = 0; k < K; ++k) matrix[k] *= passed;
        }
        if (!reverse && end != kChunk) weights = Weights<4>(l, 1.0f, false, end);
        const float up = enlarge_by_products<T, K>(matrix, size, values, weights);
#pragma unroll
        for (int i = 0; i < 8; ++i) weighted[0].step(i, values.z[0], weights.w[0], up);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s < 3) read_rows_of<T, W>(rows[(s + 1) % 2], tiles, swapped, s + 1);
            add_rows<T, K, 3>(matrix, rows[s % 2], [&](int n) { return weighted[s % 2].operand(n); }, [&](int i, int count) __attribute__((always_inline)) {
                if (s == 0) share_of(kPieces, i, count, fetch);
                if (s < 3) share_of(8, i, count, [&](int n) __attribute__((always_inline)) { weighted[(s + 1) % 2].step(n, values.z[s + 1], weights.w[s + 1], up); });
                if (s == 3) share_of(kPieces, i, count, [&](int n) __attribute__((always_inline)) { store_tiles(n, step + 1); });
            });
        }
        bring_back<T, K>(matrix, up);
    }
    const int column = column_block * 32 + (lane & 31);
    const float* given = a.segments > 1 ? nullptr : reverse ? a.d_after : a.before;
    if (given != nullptr) given += pair * matrix_size;
    const float passed = power(l, tokens);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = first_row + 32 * k + matrix_row(i);
            if (row < d && column < d) to[row * d + column] = given != nullptr ? fmaf(given[row * d + column], passed, matrix[k][i]) : matrix[k][i];
        }
}

// The outputs; behind them, where a sequence is one segment, the last states.
template <typename T, int W, bool STAGED>
__global__ __launch_bounds__((kWalkThreads<T, W>), (W == 64 ? 2 : 1)) void linear_forward_kernel(LinearArgs a) {
    const unsigned int group = a.hq / a.hkv, members = group / a.heads_each, units = a.batch * a.hkv * a.segments;
    if (blockIdx.x >= units * members) return sum_segment<T, W, STAGED, 2>(a, false, static_cast<int>(blockIdx.x - units * members), 0, shared_memory<T>());
    const Unit u = unit_of(blockIdx.x, members, units, a.segments);
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
    walk_segment<T, W, false, STAGED>(a, task, b, kv * static_cast<int>(group) + u.member * a.heads_each, u.segment, shared_memory<T>());
}

// dk and dv of all units first, whose walks are as many times longer as a group has heads, then dq; behind them, where a sequence is one segment, the
// gradients of the first states.
template <typename T, int W, bool STAGED>
__global__ __launch_bounds__((kWalkThreads<T, W>), (W == 64 ? 2 : 1)) void linear_backward_kernel(LinearArgs a) {
    const unsigned int group = a.hq / a.hkv, members = group / a.heads_each, units = a.batch * a.hkv * a.segments;
    if (blockIdx.x >= units * (members + 2)) return sum_segment<T, W, STAGED, 2>(a, true, static_cast<int>(blockIdx.x - units * (members + 2)), 0, shared_memory<T>());
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
        walk_segment<T, W, true, STAGED>(a, task, u.pair / a.hkv, u.pair % a.hkv, u.segment, shared_memory<T>());
    } else {
        const Unit u = unit_of(blockIdx.x - 2 * units, members, units, a.segments);
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
        walk_segment<T, W, false, STAGED>(a, task, u.pair / a.hkv, kv * static_cast<int>(group) + u.member * a.heads_each, u.segment, shared_memory<T>());
    }
}

// Every segment's own matrix; blockIdx.y = 1: reverse.
template <typename T, int W, bool STAGED>
__global__ __launch_bounds__(W * 2, 2) void linear_segments_kernel(LinearArgs a) {
    sum_segment<T, W, STAGED, 1>(a, blockIdx.y == 1, static_cast<int>(blockIdx.x / a.segments), static_cast<int>(blockIdx.x % a.segments), shared_memory<T>());
}

// The segments' matrices become what comes before each (blockIdx.y = 0) or behind it (1), in order along the sequence, a thread an element.
// What it waits for is the loads: 32 at a time in workgroups of one wavefront (128 segments of 4 matrices of 64 x 64: the call takes 66 us, with
// 8 at a time in workgroups of four 71, with 64 at a time 117).
constexpr int kAhead = 32, kJoinThreads = 64;
__global__ __launch_bounds__(kJoinThreads) void linear_join_kernel(LinearArgs a) {
    const bool reverse = blockIdx.y == 1;
    const long matrix = static_cast<long>(a.d) * a.d, at = static_cast<long>(blockIdx.x) * kJoinThreads + threadIdx.x;
    if (at >= matrix * a.batch * a.hkv) return;
    const long pair = at / matrix, element = at - pair * matrix;
    const float l = log2_decay(a.log_decay[pair % a.hkv]);
    const float* given = reverse ? a.d_after : a.before;
    float* result = reverse ? a.d_before : a.after;
    float running = given != nullptr ? given[at] * (reverse ? 1.0f : power(l, 1)) : 0.0f;
    const int n = a.segments, whole = a.segment_chunks * kChunk, last = a.tokens - (n - 1) * whole;  // tokens of the last segment
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
    if (result != nullptr) result[at] = fmaf(running, power(l, reverse ? whole : last - 1), result[at]);
}

// ------------------------------------------------------------------------------------------------ one token
// S' = g S + k v', o = s S'' q. Bound by the states, which are read and written once. A workgroup has 32 columns of a kv head's matrix, a thread four
// columns of every 32nd row, all of them on their way at once; what the rows share (k, q) comes by the LDS. Query heads are summed over the rows
// from registers, kStepHeads between two barriers. 512 sequences, 2 matrices of 128 x 128: 134 MB in 25.8 us, 5.2 TB/s; with 16 columns a
// workgroup 41 us, with 64 columns 48, with 128 27, and with stores that stay in the caches 34. One sequence: 4.4 us.
constexpr int kStepThreads = 256, kStepColumns = 32, kStepHeads = 4;
template <typename T, bool VECTORS>
__global__ __launch_bounds__(kStepThreads) void linear_step_kernel(T* __restrict__ out, float* next, const float* state, const T* __restrict__ q,
                                                                   const T* __restrict__ k, const T* __restrict__ v,
                                                                   const float* __restrict__ log_decay, int hq, int hkv, int d, float scale) {
    constexpr int kAcross = kStepColumns / 4, kRows = kStepThreads / kAcross, kOwn = 128 / kRows, kWaves = kStepThreads / kWave;
    __shared__ __align__(16) float keys[128], queries[kStepHeads][128];  // a thread's rows one after the other
    __shared__ __align__(16) float stage[kStepHeads][kWaves][kStepColumns];
    const int blocks = (d + kStepColumns - 1) / kStepColumns;
    const long pair = blockIdx.x / blocks;
    const int first = static_cast<int>(blockIdx.x % blocks) * kStepColumns, b = static_cast<int>(pair / hkv), kv = static_cast<int>(pair % hkv), group = hq / hkv;
    const int sub = threadIdx.x % kAcross, row0 = threadIdx.x / kAcross, wave = threadIdx.x / kWave;
    const int column = first + sub * 4;
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
    const T* heads = q + (static_cast<long>(b) * hq + static_cast<long>(kv) * group) * d;
    auto place = [](int row) { return row % kRows * kOwn + row / kRows; };
    if (threadIdx.x < 128) keys[place(threadIdx.x)] = threadIdx.x < d ? to_f32(k[pair * d + threadIdx.x]) : 0.0f;
    for (int h0 = 0; h0 < group; h0 += kStepHeads) {
#pragma unroll
        for (int n = 0; n < kStepHeads * 128; n += kStepThreads) {
            const int h = (n + static_cast<int>(threadIdx.x)) / 128, row = (n + threadIdx.x) % 128;
            queries[h][place(row)] = h0 + h < group && row < d ? to_f32(heads[(h0 + h) * d + row]) : 0.0f;
        }
        __syncthreads();
        if (h0 == 0)
#pragma unroll
            for (int n = 0; n < kOwn; ++n) {
                const int row = row0 + n * kRows;
                const float key = keys[row0 * kOwn + n];
                if (row >= d) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], g, key * value[e]);
                if constexpr (VECTORS) {
                    if (column < d) __builtin_nontemporal_store(s[n], reinterpret_cast<vec_t<float, 4>*>(to + row * d + column));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (column + e < d) to[row * d + column + e] = s[n][e];
                }
            }
#pragma unroll
        for (int h = 0; h < kStepHeads; ++h) {
            if (h0 + h >= group) break;
            vec_t<float, 4> sum(0.0f);
#pragma unroll
            for (int n = 0; n < kOwn; ++n) {
                const float query = queries[h][row0 * kOwn + n];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(query, s[n][e], sum[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int offset = 32; offset >= kAcross; offset /= 2) sum[e] += __shfl_xor(sum[e], offset, kWave);
            if ((threadIdx.x & 63) < kAcross) store_vec<float, 4>(&stage[h][wave][4 * sub], sum);
        }
        __syncthreads();
        for (int n = threadIdx.x; n < kStepHeads * kStepColumns; n += kStepThreads) {
            const int h = n / kStepColumns, at = n % kStepColumns;
            if (h0 + h >= group || first + at >= d) continue;
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) total += stage[h][w][at];
            out[(static_cast<long>(b) * hq + static_cast<long>(kv) * group + h0 + h) * d + first + at] = from_f32<T>(total * scale);
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

// Cuts the sequences into at most `most` segments of whole chunks, and says how many of a group's query heads a workgroup takes one after the other.
// Walks that give three compute units of four work are not cut: two segments each would need their matrices first (32 sequences of 1024 tokens,
// 8 query and 2 kv heads of 128: 62 us forward and 143 backward, cut in two 94 and 228). Then every query head has a workgroup of its own;
// where sequences have to be cut, a group's heads share what is done for k and v, unless that leaves units without work (backward has three
// walks a segment then: 5 sequences of 1001 half precision tokens, 12 and 4 heads of 64: 45 us, heads apart 51). Segments are two chunks or
// longer in 16-bit storage (of one chunk: 77 tokens 15.6 us instead of 9.1); in fp32, whose products take longer than what a segment costs, one
// (2 sequences of 333 tokens, 4 heads of 40, backward: 31 us, two chunks or longer 44). Two a unit where the tokens allow it (32768 tokens, 12 and 4
// heads of 64, forward: 66 us, one a unit 71).
// Backward the rule goes by dq's walks. Those of dk and dv are as many times fewer and longer as a group has heads, and are not cut for that: 256 query heads
// of 1024 tokens and 128 columns in all take 143 us in groups of four, 250 of eight, 477 of sixteen, 940 of 32.
void cut(LinearArgs& a, int most, bool backward, bool fp32) {
    const int chunks = (a.tokens + kChunk - 1) / kChunk, group = a.hq / a.hkv;
    const long pairs = static_cast<long>(a.batch) * a.hkv, units = compute_units();
    auto fills = [&](long walks) { return walks * 4 >= units * 3; };
    auto segments_for = [&](long walks) {
        if (fills(walks)) return 1;
        return static_cast<int>(std::min<long>({(2 * units + walks - 1) / walks, static_cast<long>(fp32 ? chunks : (chunks + 1) / 2), static_cast<long>(most)}));
    };
    a.heads_each = !fills(pairs * group) && fills(pairs * segments_for(pairs) * (backward ? 3 : 1)) ? group : 1;
    const int segments = segments_for(pairs * (group / a.heads_each));
    a.segment_chunks = (chunks + segments - 1) / segments;
    a.segments = (chunks + a.segment_chunks - 1) / a.segment_chunks;
}

template <typename T, int W>
constexpr int kWalkBytes = ((2 + kYTiles<T>) * kTile<T, W> + kChunk * kPairsPitch<T>) * static_cast<int>(sizeof(T)) + kWalkThreads<T, W> * 16 * 4 + (kShares<T> ? W / 32 * 8192 : 0);
template <typename T, int W>
constexpr int kSegmentBytes = 4 * kTile<T, W> * static_cast<int>(sizeof(T));

template <auto Kernel>
int allow_shared(int bytes) {
    if (bytes <= 64 * 1024) return CGPTX_OK;
    static const hipError_t once = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return check_hip(once, "hipFuncSetAttribute");
}

template <typename T, int W, bool STAGED>
int run(LinearArgs& a, bool backward, hipStream_t stream) {
    const long pairs = static_cast<long>(a.batch) * a.hkv;
    const int parts = backward ? 2 : 1;
    const std::size_t slots = static_cast<std::size_t>(pairs) * a.d * a.d;
    cut(a, 1 << 20, backward, sizeof(T) == 4);
    // Segments need scratch; a call that cannot have it all takes fewer, one sequence a walk with none.
    if (a.segments > 1) {
        void* memory = nullptr;
        std::size_t held = 0;
        auto wanted = [&] { return static_cast<std::size_t>(parts) * a.segments * slots * sizeof(float); };
        if (int st = scratch_up_to(stream, wanted(), &memory, &held)) return st;
        while (a.segments > 1 && held < wanted()) cut(a, a.segments - 1, backward, sizeof(T) == 4);
        a.ahead = static_cast<float*>(memory);
        a.behind = a.ahead + a.segments * slots;
    }
    if (a.segments > 1) {
        if (int st = allow_shared<linear_segments_kernel<T, W, STAGED>>(kSegmentBytes<T, W>)) return st;
        hipLaunchKernelGGL((linear_segments_kernel<T, W, STAGED>), dim3(static_cast<unsigned int>(pairs * a.segments), parts), dim3(W * 2), (kSegmentBytes<T, W>), stream, a);
        CGPTX_LAUNCH_CHECK();
        hipLaunchKernelGGL(linear_join_kernel, dim3(static_cast<unsigned int>((slots + kJoinThreads - 1) / kJoinThreads), parts), dim3(kJoinThreads), 0, stream, a);
        CGPTX_LAUNCH_CHECK();
    }
    const bool state_too = a.segments == 1 && (backward ? a.d_before : a.after) != nullptr;
    const long units = pairs * a.segments, members = a.hq / a.hkv / a.heads_each, states = state_too ? pairs : 0;
    if (backward) {
        if (int st = allow_shared<linear_backward_kernel<T, W, STAGED>>(kWalkBytes<T, W>)) return st;
        hipLaunchKernelGGL((linear_backward_kernel<T, W, STAGED>), dim3(static_cast<unsigned int>(units * (members + 2) + states)), dim3((kWalkThreads<T, W>)), (kWalkBytes<T, W>), stream, a);
    } else {
        if (int st = allow_shared<linear_forward_kernel<T, W, STAGED>>(kWalkBytes<T, W>)) return st;
        hipLaunchKernelGGL((linear_forward_kernel<T, W, STAGED>), dim3(static_cast<unsigned int>(units * members + states)), dim3((kWalkThreads<T, W>)), (kWalkBytes<T, W>), stream, a);
    }
    CGPTX_LAUNCH_CHECK();
    return CGPTX_OK;
}

int run_any(LinearArgs& a, bool backward, bool on_boundaries, int dtype, hipStream_t stream) {
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        // 32 bits hold every offset in a chunk.
        a.vectors = on_boundaries && a.d % kVec128<T> == 0 && static_cast<std::size_t>(a.hq) * a.d * kChunk * sizeof(T) < (std::size_t{1} << 30);
        if constexpr (sizeof(T) == 2)
            if (a.vectors) return a.d <= 64 ? run<T, 64, true>(a, backward, stream) : run<T, 128, true>(a, backward, stream);
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
