// The norms between two branches of a block for gfx950, forward and backward: the norm behind the first branch with its gate, the scaled residual
// stream, and the norm in front of the next branch.
//
//   xs = a x + gate (f rf) u,  rf = 1/sqrt(mean(f^2) + eps);   y = (xs rs) w,  rs = 1/sqrt(mean(xs^2) + eps)
//   G = dxs + rs (dy w - xs rs^2 mean(dy w xs)),   dx = a G,   h = gate u G,   df = rf (h - f rf^2 mean(h f)),
//   dw = sum_rows dy xs rs,  du = sum_rows gate G f rf,  dgate = u sum_rows G f rf (over the rows of a gate)
//
// What bounds it is memory: two rows read and two written forward, four and two backward, where the operators one by one would read the stream and
// the branch again for every norm, gate and sum. A row stays in registers between its sums and its stores (row_vectors.hpp), backward with a part of
// it in scratch memory where it is wide (see RowPlan); forward the second norm's sum is taken from the stream as it is stored, backward both norms'
// first sums in one go and the branch norm's second one when G is known. All sums are fp32; G is not rounded before either gradient.
// u and gate are constant over the rows of a gate, so one sum of G f rf stands for both their gradients. Workgroups have rows of one gate as
// a rule (BY_BLOCK); where there are so many gates that most would have few rows, a row's lanes take whole gates one after the other
// (BY_SLOT), and write the gate's gradient themselves. Per-workgroup partial sums go to scratch and a second launch adds them in a fixed order.
// 32768 bfloat16 rows of 1024: forward 268 MB in 49 us (5.5 TB/s), backward with 32 gates 403 MB in 84 (4.8 TB/s), of which the second launch 5.
#include "common.hpp"
#include "reduce.hpp"
#include "row_vectors.hpp"

#include <algorithm>
#include <cmath>
#include <string>

namespace cgptx {
namespace {

// Rows are stored past the caches, which keep what other workgroups are about to read (bfloat16, 2048 rows of 4096: backward 30 -> 25 us; fp32, 5005
// rows of 1001: forward 21 -> 16, backward 43 -> 41).
template <typename T>
__device__ __forceinline__ void store_past(T* p, vec_t<T, kVec128<T>> v, int count) {
    if (count >= kVec128<T>) __builtin_nontemporal_store(v, reinterpret_cast<typename Unaligned<T>::type*>(p));
    else store_some<T>(p, v, count);
}

struct Sizes {
    int rows, hidden;
    int gates, per_gate;  // gate rows (at least one), rows of each
    int parts;            // workgroups of a gate (BY_BLOCK)
    float scale, inv_hidden, eps;
};
struct Inputs {
    const void *x, *f, *u, *gate, *w;        // backward: x is the stream behind the branch
    const void *d_stream, *dy;
};

// The rows of one of a workgroup's slots in turn: gate and row within it.
template <int SLOTS, bool BY_SLOT>
struct RowWalk {
    int gate, within, first;  // first: the same for the workgroup's slots, what ends the walk
    __device__ __forceinline__ RowWalk(const Sizes& s, int slot) {
        if constexpr (BY_SLOT) {
            first = static_cast<int>(blockIdx.x) * SLOTS;
            gate = first + slot;
            within = 0;
        } else {
            gate = static_cast<int>(blockIdx.x) / s.parts;
            first = static_cast<int>(blockIdx.x) % s.parts * SLOTS;
            within = first + slot;
        }
    }
    __device__ __forceinline__ void advance(const Sizes& s) {
        if constexpr (BY_SLOT) {
            if (++within < s.per_gate) return;
            within = 0;
            first += static_cast<int>(gridDim.x) * SLOTS;
            gate += static_cast<int>(gridDim.x) * SLOTS;
        } else {
            first += s.parts * SLOTS;
            within += s.parts * SLOTS;
        }
    }
    __device__ __forceinline__ bool done(const Sizes& s) const { return first >= (BY_SLOT ? s.gates : s.per_gate); }
    __device__ __forceinline__ bool live(const Sizes& s) const { return BY_SLOT ? gate < s.gates : within < s.per_gate; }
    __device__ __forceinline__ std::size_t row(const Sizes& s) const { return static_cast<std::size_t>(gate) * s.per_gate + within; }
};

template <int WAVES>
constexpr int kThreadsOf = (WAVES > 4 ? WAVES : kRowWaves) * kWave;
// LPR lanes of a wavefront (WAVES = 1), or WAVES wavefronts, share a row; a lane holds K vectors of it.
template <typename T, int LPR, int WAVES, int K>
struct Layout {
    static constexpr int VEC = kVec128<T>, kThreadsHere = kThreadsOf<WAVES>, kBlockWaves = kThreadsHere / kWave;
    static constexpr int kSlots = WAVES > 1 ? 1 : kBlockWaves * kWave / LPR;
    static_assert(WAVES == 1 || kBlockWaves == WAVES, "the wavefronts of a row meet at the workgroup's barriers");
    int sub, slot;
    __device__ __forceinline__ Layout()
        : sub(WAVES > 1 ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % LPR), slot(WAVES > 1 ? 0 : static_cast<int>(threadIdx.x) / LPR) {}
    __device__ __forceinline__ int column(int c) const { return (c * LPR * WAVES + sub) * VEC; }
};

template <typename T, int LPR, int WAVES, int K, bool BY_SLOT>
__global__ __launch_bounds__(kThreadsOf<WAVES>) void sandwich_forward_kernel(T* stream, T* __restrict__ normed, Inputs in,
                                                                                              Sizes s) {
    using L = Layout<T, LPR, WAVES, K>;
    constexpr int VEC = L::VEC;
    using F = vec_t<float, VEC>;
    using V = vec_t<T, VEC>;
    constexpr bool AHEAD = WAVES <= 4;  // the next row is requested before this one is used
    __shared__ float stage[2][WAVES];
    const L at;
    const T *x = static_cast<const T*>(in.x), *f = static_cast<const T*>(in.f), *gate = static_cast<const T*>(in.gate);
    RowWalk<L::kSlots, BY_SLOT> walk(s, at.slot);
    int count[K];
    V uv[K], wv[K], gv[K];
#pragma unroll
    for (int c = 0; c < K; ++c) {
        count[c] = s.hidden - at.column(c);
        uv[c] = load_some<T>(static_cast<const T*>(in.u) + at.column(c), count[c]);
        wv[c] = load_some<T>(static_cast<const T*>(in.w) + at.column(c), count[c]);
        gv[c] = V(static_cast<T>(1.0f));
        if (!BY_SLOT && gate != nullptr) gv[c] = load_some<T>(gate + static_cast<std::size_t>(walk.gate) * s.hidden + at.column(c), count[c]);
    }
    struct Row {
        V x[K], f[K];
    };
    auto fetch = [&](const RowWalk<L::kSlots, BY_SLOT>& from, Row& r) __attribute__((always_inline)) {
        const bool live = from.live(s);
        const std::size_t base = live ? from.row(s) * s.hidden : 0;
#pragma unroll
        for (int c = 0; c < K; ++c) {
            r.x[c] = load_some<T>(x + base + at.column(c), live ? count[c] : 0);
            r.f[c] = load_some<T>(f + base + at.column(c), live ? count[c] : 0);
        }
    };
    Row now, next;
    fetch(walk, now);
    while (!walk.done(s)) {
        auto following = walk;
        following.advance(s);
        if (AHEAD && !following.done(s)) fetch(following, next);
        const bool live = walk.live(s);
        if (BY_SLOT && live && walk.within == 0)
#pragma unroll
            for (int c = 0; c < K; ++c) gv[c] = load_some<T>(gate + static_cast<std::size_t>(walk.gate) * s.hidden + at.column(c), count[c]);
        const std::size_t base = live ? walk.row(s) * s.hidden : 0;
        float squares[1] = {0.0f}, stream_squares[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F fv = vec_to_f32<T, VEC>(now.f[c]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) squares[0] = fmaf(fv[e], fv[e], squares[0]);
        }
        row_sums<LPR, WAVES>(squares, stage);
        const float rf = 1.0f / sqrtf(squares[0] * s.inv_hidden + s.eps);
        V out[K];
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F xv = vec_to_f32<T, VEC>(now.x[c]), fv = vec_to_f32<T, VEC>(now.f[c]), u = vec_to_f32<T, VEC>(uv[c]), g = vec_to_f32<T, VEC>(gv[c]);
            F v;
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = fmaf(s.scale, xv[e], g[e] * (fv[e] * rf * u[e]));
            out[c] = vec_from_f32<T, VEC>(v);
            const F stored = vec_to_f32<T, VEC>(out[c]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) stream_squares[0] = fmaf(stored[e], stored[e], stream_squares[0]);
            if (live) store_past<T>(stream + base + at.column(c), out[c], count[c]);
        }
        row_sums<LPR, WAVES>(stream_squares, stage + 1);
        const float rs = 1.0f / sqrtf(stream_squares[0] * s.inv_hidden + s.eps);
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F stored = vec_to_f32<T, VEC>(out[c]), w = vec_to_f32<T, VEC>(wv[c]);
            F v;
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = stored[e] * rs * w[e];
            if (live) store_past<T>(normed + base + at.column(c), vec_from_f32<T, VEC>(v), count[c]);
        }
        walk = following;
        if constexpr (AHEAD) now = next;
        else if (!walk.done(s)) fetch(walk, now);
    }
}

struct Outputs {
    void *dx, *df, *dgate;
    float* partial;  // [3][workgroups][hidden]: dw, du and (BY_BLOCK) dgate
};

template <typename T, int LPR, int WAVES, int K, bool BY_SLOT>
__global__ __launch_bounds__(kThreadsOf<WAVES>) void sandwich_backward_kernel(Outputs out, Inputs in, Sizes s) {
    using L = Layout<T, LPR, WAVES, K>;
    constexpr int VEC = L::VEC;
    using F = vec_t<float, VEC>;
    using V = vec_t<T, VEC>;
    constexpr bool AHEAD = WAVES <= 4;
    __shared__ float stage[4][WAVES];
    const L at;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const T *stream = static_cast<const T*>(in.x), *f = static_cast<const T*>(in.f), *gate = static_cast<const T*>(in.gate);
    const T *d_stream = static_cast<const T*>(in.d_stream), *dy = static_cast<const T*>(in.dy);
    T *dx = static_cast<T*>(out.dx), *df = static_cast<T*>(out.df), *dgate = static_cast<T*>(out.dgate);
    RowWalk<L::kSlots, BY_SLOT> walk(s, at.slot);
    int count[K];
    V uv[K], wv[K], gv[K];
    F sum_w[K], sum_a[K], sum_u[BY_SLOT ? K : 1];  // dy xs rs; G f rf of a gate; BY_SLOT: gate G f rf of all
#pragma unroll
    for (int c = 0; c < K; ++c) {
        count[c] = s.hidden - at.column(c);
        uv[c] = load_some<T>(static_cast<const T*>(in.u) + at.column(c), count[c]);
        wv[c] = load_some<T>(static_cast<const T*>(in.w) + at.column(c), count[c]);
        gv[c] = V(static_cast<T>(1.0f));
        if (!BY_SLOT && gate != nullptr) gv[c] = load_some<T>(gate + static_cast<std::size_t>(walk.gate) * s.hidden + at.column(c), count[c]);
        sum_w[c] = sum_a[c] = F(0.0f);
        if constexpr (BY_SLOT) sum_u[c] = F(0.0f);
    }
    struct Row {
        V stream[K], f[K], d_stream[K], dy[K];
    };
    auto fetch = [&](const RowWalk<L::kSlots, BY_SLOT>& from, Row& r) __attribute__((always_inline)) {
        const bool live = from.live(s);
        const std::size_t base = live ? from.row(s) * s.hidden : 0;
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const int n = live ? count[c] : 0;
            r.stream[c] = load_some<T>(stream + base + at.column(c), n);
            r.dy[c] = load_some<T>(dy + base + at.column(c), n);
            r.f[c] = load_some<T>(f + base + at.column(c), n);
            r.d_stream[c] = load_some<T>(d_stream != nullptr ? d_stream + base + at.column(c) : dy, d_stream != nullptr ? n : 0);
        }
    };
    Row now, next;
    fetch(walk, now);
    while (!walk.done(s)) {
        auto following = walk;
        following.advance(s);
        if (AHEAD && !following.done(s)) fetch(following, next);
        const bool live = walk.live(s);
        if (BY_SLOT && live && walk.within == 0)
#pragma unroll
            for (int c = 0; c < K; ++c) gv[c] = load_some<T>(gate + static_cast<std::size_t>(walk.gate) * s.hidden + at.column(c), count[c]);
        const std::size_t base = live ? walk.row(s) * s.hidden : 0;
        float sums[3] = {0.0f, 0.0f, 0.0f};  // xs^2, dy w xs, f^2
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F xs = vec_to_f32<T, VEC>(now.stream[c]), d = vec_to_f32<T, VEC>(now.dy[c]), w = vec_to_f32<T, VEC>(wv[c]), fv = vec_to_f32<T, VEC>(now.f[c]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sums[0] = fmaf(xs[e], xs[e], sums[0]);
                sums[1] = fmaf(d[e] * w[e], xs[e], sums[1]);
                sums[2] = fmaf(fv[e], fv[e], sums[2]);
            }
        }
        row_sums<LPR, WAVES>(sums, stage);
        const float rs = 1.0f / sqrtf(sums[0] * s.inv_hidden + s.eps), rf = 1.0f / sqrtf(sums[2] * s.inv_hidden + s.eps);
        const float mean = sums[1] * rs * s.inv_hidden;  // of dy w (xs rs)
        float branch[1] = {0.0f};                        // h f
        F g[K];
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F xs = vec_to_f32<T, VEC>(now.stream[c]), d = vec_to_f32<T, VEC>(now.dy[c]), w = vec_to_f32<T, VEC>(wv[c]), fv = vec_to_f32<T, VEC>(now.f[c]);
            const F u = vec_to_f32<T, VEC>(uv[c]), by = vec_to_f32<T, VEC>(gv[c]), past = vec_to_f32<T, VEC>(now.d_stream[c]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xh = xs[e] * rs, fh = fv[e] * rf;
                g[c][e] = fmaf(rs, fmaf(-xh, mean, d[e] * w[e]), past[e]);
                sum_w[c][e] = fmaf(d[e], xh, sum_w[c][e]);
                sum_a[c][e] = fmaf(g[c][e], fh, sum_a[c][e]);
                branch[0] = fmaf(by[e] * u[e] * g[c][e], fh, branch[0]);
            }
        }
        row_sums<LPR, WAVES>(branch, stage + 3);
        const float branch_mean = branch[0] * s.inv_hidden;
#pragma unroll
        for (int c = 0; c < K; ++c) {
            const F fv = vec_to_f32<T, VEC>(now.f[c]), u = vec_to_f32<T, VEC>(uv[c]), by = vec_to_f32<T, VEC>(gv[c]);
            F of_x, of_f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                of_x[e] = s.scale * g[c][e];
                of_f[e] = rf * fmaf(-fv[e] * rf, branch_mean, by[e] * u[e] * g[c][e]);
            }
            if (live) {
                store_past<T>(dx + base + at.column(c), vec_from_f32<T, VEC>(of_x), count[c]);
                store_past<T>(df + base + at.column(c), vec_from_f32<T, VEC>(of_f), count[c]);
            }
        }
        if constexpr (BY_SLOT) {
            if (live && walk.within + 1 == s.per_gate) {
#pragma unroll
                for (int c = 0; c < K; ++c) {
                    const F by = vec_to_f32<T, VEC>(gv[c]), u = vec_to_f32<T, VEC>(uv[c]);
                    F v;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        sum_u[c][e] = fmaf(by[e], sum_a[c][e], sum_u[c][e]);
                        v[e] = u[e] * sum_a[c][e];
                    }
                    if (dgate != nullptr)
                        store_some<T>(dgate + static_cast<std::size_t>(walk.gate) * s.hidden + at.column(c), vec_from_f32<T, VEC>(v), count[c]);
                    sum_a[c] = F(0.0f);
                }
            }
        }
        walk = following;
        if constexpr (AHEAD) now = next;
        else if (!walk.done(s)) fetch(walk, now);
    }
    // Partial sums: dw, du and, of a workgroup's own gate, dgate.
    auto part = [&](int which, int c, int e) __attribute__((always_inline)) {
        if (which == 0) return sum_w[c][e];
        if constexpr (BY_SLOT) return sum_u[c][e];
        else return sum_a[c][e] * to_f32(which == 1 ? gv[c][e] : uv[c][e]);
    };
    constexpr int kParts = BY_SLOT ? 2 : 3;
#pragma unroll
    for (int which = 0; which < kParts; ++which) {
        if (which == 2 && dgate == nullptr) break;
        float* mine = out.partial + (static_cast<std::size_t>(which) * gridDim.x + blockIdx.x) * s.hidden;
        if constexpr (WAVES > 1) {
#pragma unroll
            for (int c = 0; c < K; ++c)
#pragma unroll
                for (int e = 0; e < VEC; e += 4)
                    store_some<float>(mine + at.column(c) + e, vec_t<float, 4>{part(which, c, e), part(which, c, e + 1), part(which, c, e + 2), part(which, c, e + 3)},
                                      count[c] - e);
        } else {
            // The row slots of a wavefront, then the workgroup's wavefronts.
            __shared__ float fold[L::kBlockWaves][LPR * K * VEC];
            __syncthreads();
#pragma unroll
            for (int c = 0; c < K; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float v = part(which, c, e);
#pragma unroll
                    for (int offset = LPR; offset < kWave; offset <<= 1) v += __shfl_xor(v, offset, kWave);
                    if (lane < LPR) fold[wave][(c * LPR + at.sub) * VEC + e] = v;
                }
            __syncthreads();
            for (int col = threadIdx.x; col < s.hidden; col += L::kThreadsHere) {
                float v = 0.0f;
#pragma unroll
                for (int n = 0; n < L::kBlockWaves; ++n) v += fold[n][col];
                mine[col] = v;
            }
        }
    }
}

// dw (blockIdx.y = 0) and du (1) from all workgroups' partial sums, the gradient of gate y - 2 from those of its own.
template <typename T, int COLUMNS>
__global__ __launch_bounds__(kFinishThreads) void sandwich_finish_kernel(T* __restrict__ dw, T* __restrict__ du, T* __restrict__ dgate,
                                                                         const float* __restrict__ partial, int blocks, int parts, int hidden,
                                                                         int units) {
    __shared__ float folded[kFolded], stage[4 * COLUMNS];
    const int which = static_cast<int>(blockIdx.y);
    const std::size_t pitch = static_cast<std::size_t>(hidden);
    if (which < 2)
        column_partial_reduce_body<T, COLUMNS>(which == 0 ? dw : du, partial + which * blocks * pitch, blocks, hidden, 0, static_cast<int>(blockIdx.x), units,
                                               folded, stage);
    else
        column_partial_reduce_body<T, COLUMNS>(dgate + (which - 2) * pitch, partial + (2 * static_cast<std::size_t>(blocks) + static_cast<std::size_t>(which - 2) * parts) * pitch,
                                               parts, hidden, 0, static_cast<int>(blockIdx.x), units, folded, stage);
}

// ------------------------------------------------------------------------------------------------ rows of any length
__device__ __forceinline__ std::size_t gate_base(const Sizes& s, int row) { return static_cast<std::size_t>(row / s.per_gate) * s.hidden; }
template <typename T>
__device__ __forceinline__ vec_t<float, kVec128<T>> gate_values(const T* gate, std::size_t base, int col, int count) {
    if (gate == nullptr) return vec_t<float, kVec128<T>>(1.0f);
    return vec_to_f32<T, kVec128<T>>(load_some<T>(gate + base + col, count));
}

template <typename T>
__global__ __launch_bounds__(kLongThreads) void sandwich_long_forward_kernel(T* stream, T* normed, Inputs in, Sizes s) {
    constexpr int VEC = kVec128<T>;
    using F = vec_t<float, VEC>;
    __shared__ float stage[kLongThreads / kWave];
    const T *x = static_cast<const T*>(in.x), *f = static_cast<const T*>(in.f), *gate = static_cast<const T*>(in.gate), *u = static_cast<const T*>(in.u),
            *w = static_cast<const T*>(in.w);
    for (int row = blockIdx.x; row < s.rows; row += gridDim.x) {
        const std::size_t base = static_cast<std::size_t>(row) * s.hidden, gates = gate_base(s, row);
        float sum = 0.0f;
        walk_row(f + base, s.hidden, [&](int, int, const F& v) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum = fmaf(v[e], v[e], sum);
        });
        const float rf = 1.0f / sqrtf(block_sum(sum, stage) * s.inv_hidden + s.eps);
        sum = 0.0f;
        walk_row(f + base, s.hidden, [&](int col, int count, const F& v) {
            const F xv = vec_to_f32<T, VEC>(load_some<T>(x + base + col, count)), uv = vec_to_f32<T, VEC>(load_some<T>(u + col, count)),
                    g = gate_values<T>(gate, gates, col, count);
            F o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = fmaf(s.scale, xv[e], g[e] * (v[e] * rf * uv[e]));
            const vec_t<T, VEC> stored = vec_from_f32<T, VEC>(o);
            store_some<T>(stream + base + col, stored, count);
            const F seen = vec_to_f32<T, VEC>(stored);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum = fmaf(e < count ? seen[e] : 0.0f, e < count ? seen[e] : 0.0f, sum);
        });
        const float rs = 1.0f / sqrtf(block_sum(sum, stage) * s.inv_hidden + s.eps);
        // A thread reads what it wrote itself.
        walk_row(static_cast<const T*>(stream) + base, s.hidden, [&](int col, int count, const F& v) {
            const F wv = vec_to_f32<T, VEC>(load_some<T>(w + col, count));
            F o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = v[e] * rs * wv[e];
            store_some<T>(normed + base + col, vec_from_f32<T, VEC>(o), count);
        });
    }
}

// What the gradients' columns need of a row: rs, rs^2 mean(dy w xs) and rf.
struct RowStatistics {
    float rs, pull, rf;
};
template <typename T>
__global__ __launch_bounds__(kLongThreads) void sandwich_long_backward_kernel(Outputs out, RowStatistics* __restrict__ statistics, Inputs in, Sizes s) {
    constexpr int VEC = kVec128<T>;
    using F = vec_t<float, VEC>;
    __shared__ float stage[kLongThreads / kWave];
    const T *stream = static_cast<const T*>(in.x), *f = static_cast<const T*>(in.f), *gate = static_cast<const T*>(in.gate), *u = static_cast<const T*>(in.u),
            *w = static_cast<const T*>(in.w), *d_stream = static_cast<const T*>(in.d_stream), *dy = static_cast<const T*>(in.dy);
    T* df = static_cast<T*>(out.df);
    for (int row = blockIdx.x; row < s.rows; row += gridDim.x) {
        const std::size_t base = static_cast<std::size_t>(row) * s.hidden, gates = gate_base(s, row);
        float squares = 0.0f, product = 0.0f, branch_squares = 0.0f;
        walk_row(stream + base, s.hidden, [&](int col, int count, const F& v) {
            const F d = vec_to_f32<T, VEC>(load_some<T>(dy + base + col, count)), wv = vec_to_f32<T, VEC>(load_some<T>(w + col, count)),
                    fv = vec_to_f32<T, VEC>(load_some<T>(f + base + col, count));
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                squares = fmaf(v[e], v[e], squares);
                product = fmaf(d[e] * wv[e], v[e], product);
                branch_squares = fmaf(fv[e], fv[e], branch_squares);
            }
        });
        const float rs = 1.0f / sqrtf(block_sum(squares, stage) * s.inv_hidden + s.eps);
        const float mean = block_sum(product, stage) * rs * s.inv_hidden;
        const float rf = 1.0f / sqrtf(block_sum(branch_squares, stage) * s.inv_hidden + s.eps);
        auto gradient = [&](int col, int count, const F& v) {
            const F d = vec_to_f32<T, VEC>(load_some<T>(dy + base + col, count)), wv = vec_to_f32<T, VEC>(load_some<T>(w + col, count));
            F g(0.0f);
            if (d_stream != nullptr) g = vec_to_f32<T, VEC>(load_some<T>(d_stream + base + col, count));
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[e] = fmaf(rs, fmaf(-v[e] * rs, mean, d[e] * wv[e]), g[e]);
            return g;
        };
        float branch = 0.0f;
        walk_row(stream + base, s.hidden, [&](int col, int count, const F& v) {
            const F g = gradient(col, count, v), by = gate_values<T>(gate, gates, col, count), uv = vec_to_f32<T, VEC>(load_some<T>(u + col, count)),
                    fv = vec_to_f32<T, VEC>(load_some<T>(f + base + col, count));
#pragma unroll
            for (int e = 0; e < VEC; ++e) branch = fmaf(by[e] * uv[e] * g[e], fv[e] * rf, branch);
        });
        const float branch_mean = block_sum(branch, stage) * s.inv_hidden;
        if (threadIdx.x == 0) statistics[row] = {rs, mean * rs, rf};
        walk_row(stream + base, s.hidden, [&](int col, int count, const F& v) {
            const F g = gradient(col, count, v), by = gate_values<T>(gate, gates, col, count), uv = vec_to_f32<T, VEC>(load_some<T>(u + col, count)),
                    fv = vec_to_f32<T, VEC>(load_some<T>(f + base + col, count));
            F of_f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) of_f[e] = rf * fmaf(-fv[e] * rf, branch_mean, by[e] * uv[e] * g[e]);
            store_some<T>(df + base + col, vec_from_f32<T, VEC>(of_f), count);
        });
    }
}

// G of a vector of a row.
template <typename T>
__device__ __forceinline__ vec_t<float, kVec128<T>> stream_gradient(const Inputs& in, const RowStatistics& r, std::size_t at, int col, int count) {
    constexpr int VEC = kVec128<T>;
    using F = vec_t<float, VEC>;
    const F xs = vec_to_f32<T, VEC>(load_some<T>(static_cast<const T*>(in.x) + at, count)), d = vec_to_f32<T, VEC>(load_some<T>(static_cast<const T*>(in.dy) + at, count)),
            w = vec_to_f32<T, VEC>(load_some<T>(static_cast<const T*>(in.w) + col, count));
    F g(0.0f);
    if (in.d_stream != nullptr) g = vec_to_f32<T, VEC>(load_some<T>(static_cast<const T*>(in.d_stream) + at, count));
#pragma unroll
    for (int e = 0; e < VEC; ++e) g[e] = fmaf(r.rs, fmaf(-xs[e], r.pull, d[e] * w[e]), g[e]);
    return g;
}

// Columns: a vector of them a lane, rows dealt out to a workgroup's wavefronts; a workgroup takes `span` gates one after the other (parts = 1),
// or one of the parts of a gate's rows. Runs before dx is written, which may lie where d_stream does.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void sandwich_column_kernel(Outputs out, const RowStatistics* __restrict__ statistics, Inputs in, Sizes s,
                                                                      int span) {
    constexpr int VEC = kVec128<T>;
    using F = vec_t<float, VEC>;
    __shared__ F stage[kRowWaves][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int col = static_cast<int>(blockIdx.x * kWave + lane) * VEC, count = s.hidden - col;
    const int first = static_cast<int>(blockIdx.y) / s.parts * span, part = static_cast<int>(blockIdx.y) % s.parts;
    const T *f = static_cast<const T*>(in.f), *dy = static_cast<const T*>(in.dy), *stream = static_cast<const T*>(in.x), *gate = static_cast<const T*>(in.gate);
    auto total = [&](const F& mine) {  // of the wavefronts, in the first one
        __syncthreads();
        stage[wave][lane] = mine;
        __syncthreads();
        F sum(0.0f);
#pragma unroll
        for (int n = 0; n < kRowWaves; ++n) sum += stage[n][lane];
        return sum;
    };
    auto leave = [&](int which, const F& v) {
        float* to = out.partial + (static_cast<std::size_t>(which) * gridDim.y + blockIdx.y) * s.hidden + col;
#pragma unroll
        for (int e = 0; e < VEC; e += 4) store_some<float>(to + e, vec_t<float, 4>{v[e], v[e + 1], v[e + 2], v[e + 3]}, count - e);
    };
    F u(0.0f), sum_w(0.0f), sum_u(0.0f);
    if (count > 0) u = vec_to_f32<T, VEC>(load_some<T>(static_cast<const T*>(in.u) + col, count));
    for (int g = first; g < min(first + span, s.gates); ++g) {
        F sum_a(0.0f);
        if (count > 0) {
            for (int within = part * kRowWaves + wave; within < s.per_gate; within += s.parts * kRowWaves) {
                const std::size_t row = static_cast<std::size_t>(g) * s.per_gate + within, at = row * s.hidden + col;
                const RowStatistics r = statistics[row];
                const F grad = stream_gradient<T>(in, r, at, col, count), fv = vec_to_f32<T, VEC>(load_some<T>(f + at, count)),
                        d = vec_to_f32<T, VEC>(load_some<T>(dy + at, count)), xs = vec_to_f32<T, VEC>(load_some<T>(stream + at, count));
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    sum_w[e] = fmaf(d[e], xs[e] * r.rs, sum_w[e]);
                    sum_a[e] = fmaf(grad[e], fv[e] * r.rf, sum_a[e]);
                }
            }
        }
        sum_a = total(sum_a);
        if (wave == 0 && count > 0) {
            const F by = gate_values<T>(gate, static_cast<std::size_t>(g) * s.hidden, col, count);
            sum_u += by * sum_a;
            if (out.dgate != nullptr) {
                if (s.parts > 1) leave(2, u * sum_a);
                else store_some<T>(static_cast<T*>(out.dgate) + static_cast<std::size_t>(g) * s.hidden + col, vec_from_f32<T, VEC>(u * sum_a), count);
            }
        }
    }
    sum_w = total(sum_w);
    if (wave == 0 && count > 0) {
        leave(0, sum_w);
        leave(1, sum_u);
    }
}

template <typename T>
__global__ __launch_bounds__(kLongThreads) void sandwich_long_stream_kernel(T* dx, const RowStatistics* __restrict__ statistics, Inputs in, Sizes s) {
    constexpr int VEC = kVec128<T>;
    for (int row = blockIdx.x; row < s.rows; row += gridDim.x) {
        const RowStatistics r = statistics[row];
        const std::size_t base = static_cast<std::size_t>(row) * s.hidden;
        for (int col = threadIdx.x * VEC; col < s.hidden; col += kLongThreads * VEC) {
            const int count = s.hidden - col;
            store_some<T>(dx + base + col, vec_from_f32<T, VEC>(stream_gradient<T>(in, r, base + col, col, count) * s.scale), count);
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
template <typename T>
struct RowPlan {
    using Forward = void (*)(T*, T*, Inputs, Sizes);
    using Backward = void (*)(Outputs, Inputs, Sizes);
    Forward forward[2] = {};  // BY_BLOCK, BY_SLOT
    Backward backward[2] = {};
    int slots = 0, threads = 0;

    template <int LPR, int WAVES, int K>
    void take() {
        using L = Layout<T, LPR, WAVES, K>;
        forward[0] = sandwich_forward_kernel<T, LPR, WAVES, K, false>;
        forward[1] = sandwich_forward_kernel<T, LPR, WAVES, K, true>;
        backward[0] = sandwich_backward_kernel<T, LPR, WAVES, K, false>;
        backward[1] = sandwich_backward_kernel<T, LPR, WAVES, K, true>;
        slots = L::kSlots;
        threads = L::kThreadsHere;
    }
    // Up to 16 values of a row in a lane. Backward holds eleven of each: 250 registers at 16 values, two wavefronts a SIMD. With eight wavefronts a
    // row (4097 to 8192 columns) up to 13 registers are spilled, with sixteen (8193 to 16384 in 16-bit storage), which leave a lane 128, 127 to 188:
    // backward in bfloat16 with one gate, in TB/s of what is read and written, 5.0 at 32768 x 1024, 4.7 at 8192 x 4096, 4.1 at 4096 x 8192, 0.9 at
    // 2730 x 12288, 1.1 at 2048 x 16384, and 1.7 with the kernels for rows of any length at 1638 x 20480; forward, which spills nothing, 5.4, 5.3,
    // 5.7, 4.8, 5.1 and 3.8.
    explicit RowPlan(int hidden) {
        const int vectors = (hidden + kVec128<T> - 1) / kVec128<T>;
        if (vectors <= 16) take<16, 1, 1>();
        else if (vectors <= 32) take<32, 1, 1>();
        else if (vectors <= 64) take<64, 1, 1>();
        else if (vectors <= 128) take<64, 1, 2>();
        else if (vectors <= 256) take<64, 4, 1>();
        else if (vectors <= 512) take<64, 4, 2>();
        else if (vectors <= 1024) take<64, 8, 2>();
        else if (vectors <= 2048) take<64, sizeof(T) == 2 ? 16 : 8, sizeof(T) == 2 ? 2 : 4>();
    }
    // How a launch deals its rows out: its workgroups, and which kernel takes them. Lanes take whole gates where there are at least twice as many as
    // the chip holds workgroups, or where a gate has fewer rows than a workgroup has slots. Else a workgroup leaves three rows of partial sums,
    // however few rows its gate has: many gates of few wide rows pay for that backward (bfloat16: 1000 rows of 4096 in 264 us with a gate each, in 21
    // with one for all; 32768 of 1024 in 116 with 512 gates, in 84 with 32).
    int deal(Sizes& s, const void* by_block, const void* by_slot, bool* slot) const {
        *slot = s.gates > 1 && (s.per_gate < slots || s.gates >= 2 * resident_blocks(by_block, threads));
        if (*slot) return std::min((s.gates + slots - 1) / slots, resident_blocks(by_slot, threads));
        s.parts = std::min((s.per_gate + slots - 1) / slots, std::max(1, resident_blocks(by_block, threads) / s.gates));
        return s.gates * s.parts;
    }
};

int validate(const char* name, std::size_t rows, std::size_t hidden, std::size_t gate_rows, const void* gate, float scale, float eps, int dtype) {
    const std::string n(name);
    if (!valid_dtype(dtype)) return fail(CGPTX_INVALID_ARGUMENT, n + ": unsupported dtype");
    if (!std::isfinite(eps) || eps <= 0.0f) return fail(CGPTX_INVALID_ARGUMENT, n + ": epsilon must be finite and positive");
    if (!std::isfinite(scale)) return fail(CGPTX_INVALID_ARGUMENT, n + ": the residual scale must be finite");
    if (rows == 0 || hidden == 0) return fail(CGPTX_INVALID_ARGUMENT, n + ": empty shape");
    if ((gate == nullptr) != (gate_rows == 0) || (gate_rows != 0 && rows % gate_rows != 0))
        return fail(CGPTX_INVALID_ARGUMENT, n + ": the gate must have one row for every equal number of rows, or none");
    // The second launch has 1024 threads for sixteen columns: 2^31 along an axis, which may have fewer than 2^32.
    if (rows > std::size_t{1} << 30 || hidden > std::size_t{1} << 25) return fail(CGPTX_INVALID_ARGUMENT, n + ": dimensions exceed supported range");
    return CGPTX_OK;
}

Sizes sizes_of(std::size_t rows, std::size_t hidden, std::size_t gate_rows, float scale, float eps) {
    Sizes s{};
    s.rows = static_cast<int>(rows);
    s.hidden = static_cast<int>(hidden);
    s.gates = gate_rows == 0 ? 1 : static_cast<int>(gate_rows);
    s.per_gate = s.rows / s.gates;
    s.parts = 1;
    s.scale = scale;
    s.inv_hidden = 1.0f / static_cast<float>(hidden);
    s.eps = eps;
    return s;
}

int row_blocks(int rows) { return std::min(rows, compute_units() * 2); }

template <typename T>
int launch_finish(const Outputs& out, void* dw, void* du, int blocks, int parts, int gates, int hidden, hipStream_t stream) {
    const int columns = finish_columns(hidden);
    auto finish = columns == 16 ? sandwich_finish_kernel<T, 16> : sandwich_finish_kernel<T, 32>;
    hipLaunchKernelGGL(finish, dim3((hidden + columns - 1) / columns, 2 + gates), dim3(kFinishThreads), 0, stream, static_cast<T*>(dw),
                       static_cast<T*>(du), static_cast<T*>(out.dgate), out.partial, blocks, parts, hidden, compute_units());
    CGPTX_LAUNCH_CHECK();
    return CGPTX_OK;
}

}  // namespace
}  // namespace cgptx

extern "C" int cgptx_sandwich_norm_forward(void* stream_output, void* normed, const void* stream_input, const void* branch,
                                           const void* branch_weight, const void* gate, const void* norm_weight, size_t rows, size_t hidden,
                                           size_t gate_rows, float residual_scale, float epsilon, int dtype, cgptx_stream stream_) {
    using namespace cgptx;
    const char* name = "sandwich_norm_forward";
    if (int st = validate(name, rows, hidden, gate_rows, gate, residual_scale, epsilon, dtype)) return st;
    if (stream_output == nullptr || normed == nullptr || stream_input == nullptr || branch == nullptr || branch_weight == nullptr ||
        norm_weight == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    auto stream = static_cast<hipStream_t>(stream_);
    Sizes s = sizes_of(rows, hidden, gate_rows, residual_scale, epsilon);
    const Inputs in{stream_input, branch, branch_weight, gate, norm_weight, nullptr, nullptr};
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        if (const RowPlan<T> plan(s.hidden); plan.slots != 0) {
            bool slot = false;
            const int blocks = plan.deal(s, reinterpret_cast<const void*>(plan.forward[0]), reinterpret_cast<const void*>(plan.forward[1]), &slot);
            hipLaunchKernelGGL(plan.forward[slot], dim3(blocks), dim3(plan.threads), 0, stream, static_cast<T*>(stream_output), static_cast<T*>(normed),
                               in, s);
        } else {
            hipLaunchKernelGGL((sandwich_long_forward_kernel<T>), dim3(row_blocks(s.rows)), dim3(kLongThreads), 0, stream,
                               static_cast<T*>(stream_output), static_cast<T*>(normed), in, s);
        }
        CGPTX_LAUNCH_CHECK();
        return CGPTX_OK;
    });
}

extern "C" int cgptx_sandwich_norm_backward(void* grad_stream_input, void* grad_branch, void* grad_branch_weight, void* grad_gate,
                                            void* grad_norm_weight, const void* grad_stream_output, const void* grad_normed,
                                            const void* stream_output, const void* branch, const void* branch_weight, const void* gate,
                                            const void* norm_weight, size_t rows, size_t hidden, size_t gate_rows, float residual_scale,
                                            float epsilon, int dtype, cgptx_stream stream_) {
    using namespace cgptx;
    const char* name = "sandwich_norm_backward";
    if (int st = validate(name, rows, hidden, gate_rows, gate, residual_scale, epsilon, dtype)) return st;
    if (grad_stream_input == nullptr || grad_branch == nullptr || grad_branch_weight == nullptr || grad_norm_weight == nullptr ||
        grad_normed == nullptr || stream_output == nullptr || branch == nullptr || branch_weight == nullptr || norm_weight == nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": null tensor");
    if (gate == nullptr && grad_gate != nullptr)
        return fail(CGPTX_INVALID_ARGUMENT, std::string(name) + ": no gate whose gradient could be asked for");
    auto stream = static_cast<hipStream_t>(stream_);
    Sizes s = sizes_of(rows, hidden, gate_rows, residual_scale, epsilon);
    const Inputs in{stream_output, branch, branch_weight, gate, norm_weight, grad_stream_output, grad_normed};
    Outputs out{grad_stream_input, grad_branch, grad_gate, nullptr};
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        void* memory = nullptr;
        const std::size_t row_bytes = hidden * sizeof(float);
        if (const RowPlan<T> plan(s.hidden); plan.slots != 0) {
            bool slot = false;
            const int blocks = plan.deal(s, reinterpret_cast<const void*>(plan.backward[0]), reinterpret_cast<const void*>(plan.backward[1]), &slot);
            const bool sum_gates = grad_gate != nullptr && !slot;
            if (int st = scratch(stream, (sum_gates ? 3 : 2) * static_cast<std::size_t>(blocks) * row_bytes, &memory)) return st;
            out.partial = static_cast<float*>(memory);
            hipLaunchKernelGGL(plan.backward[slot], dim3(blocks), dim3(plan.threads), 0, stream, out, in, s);
            CGPTX_LAUNCH_CHECK();
            return launch_finish<T>(out, grad_norm_weight, grad_branch_weight, blocks, s.parts, sum_gates ? s.gates : 0, s.hidden, stream);
        }
        constexpr int kSlices = 64;
        const int span = (s.gates + kSlices - 1) / kSlices;
        s.parts = s.gates < kSlices ? std::min(kSlices / s.gates, (s.per_gate + kRowWaves - 1) / kRowWaves) : 1;
        const int blocks = (s.gates + span - 1) / span * s.parts;
        const bool sum_gates = grad_gate != nullptr && s.parts > 1;
        const std::size_t statistics_bytes = (rows * sizeof(RowStatistics) + 255) & ~std::size_t{255};
        if (int st = scratch(stream, statistics_bytes + (sum_gates ? 3 : 2) * static_cast<std::size_t>(blocks) * row_bytes, &memory)) return st;
        auto* statistics = static_cast<RowStatistics*>(memory);
        out.partial = reinterpret_cast<float*>(static_cast<char*>(memory) + statistics_bytes);
        hipLaunchKernelGGL((sandwich_long_backward_kernel<T>), dim3(row_blocks(s.rows)), dim3(kLongThreads), 0, stream, out, statistics, in, s);
        CGPTX_LAUNCH_CHECK();
        const int per_block = kWave * kVec128<T>;
        hipLaunchKernelGGL((sandwich_column_kernel<T>), dim3((s.hidden + per_block - 1) / per_block, blocks), dim3(kRowThreads), 0, stream, out, statistics,
                           in, s, span);
        CGPTX_LAUNCH_CHECK();
        hipLaunchKernelGGL((sandwich_long_stream_kernel<T>), dim3(row_blocks(s.rows)), dim3(kLongThreads), 0, stream,
                           static_cast<T*>(grad_stream_input), statistics, in, s);
        CGPTX_LAUNCH_CHECK();
        return launch_finish<T>(out, grad_norm_weight, grad_branch_weight, blocks, s.parts, sum_gates ? s.gates : 0, s.hidden, stream);
    });
}
