// What the kernels of differential attention share: the call, and the entries of the 16-bit matrix-core kernels.
#pragma once

#include "attention_tiles.hpp"

namespace cgptx {

struct DifferentialArgs {
    void *out, *second;  // O and O2 (which may be null)
    float* lse_out;      // [2][batch, qs, hq], or null
    void *dq, *dk, *dv;
    float* dlambda;
    const void *q, *k, *v, *dout, *o, *o2;
    const float *lambda, *lse;
    // Statistics of the rows, [n][batch, qs, hq]. Backward: delta1, delta2 of the scalar and fp32 kernels; of the 16-bit ones, four in
    // the form that their dK/dV takes (lse1·log2 e, lse2·log2 e - log2|lambda|, -delta1, sign(-lambda)(delta1 - delta2)). Forward
    // with shared keys: [splits][2][batch, qs, hq] pairs of a map's largest score and the sum that stands to it.
    float* delta;
    float* lambda_partial;  // [hq][lambda_parts]: what a head's dlambda is the sum of
    float* largest;         // [hq][lambda_parts], half precision on the matrix cores: the largest |dO| of the same rows
    long lambda_parts;
    int batch, qs, ks, hq, hkv, d;
    float scale;           // of the scores
    float gradient_scale;  // of their gradients: the same, and 0 where there is one key, whose share is 1 whatever the score
    int causal, offset, accumulate;
    int dtype;
    // dK/dV on the matrix cores, set by its launch (fp32: splits only); a forward pass whose keys are shared sets splits, partial, delta:
    int paired;      // a workgroup takes key blocks (i, last - i) instead of one
    int splits;      // workgroups that share a key block's query tiles (never with paired)
    int by_block;    // splits > 1: workgroups go out block by block over all (batch, kv-head) pairs
    int pack;        // forward pass whose keys are shared: heads of a group that have their rows in one block
    float* partial;  // splits > 1: [splits][dK | dV][key, kv head, d] sums of the parts
};

// Whether the 16-bit matrix kernels serve a call's types and sizes: halves of a head in multiples of 8 (128-bit chunks of a row). 64
// rows of at most 65535 heads of 128 are less than 1 GiB, which their 32-bit offsets within a tile reach. Their tensors lie on 16-byte
// boundaries.
bool differential_mfma_takes(const DifferentialArgs& args);
int differential_mfma_forward(DifferentialArgs args, hipStream_t stream);  // takes scratch where few queries share many keys
int differential_mfma_backward(DifferentialArgs args, hipStream_t stream);  // takes its scratch itself

// The fp32 ones: halves of a head in multiples of 4, tensors on 16-byte boundaries, no more tiles of 16 rows than a launch has workgroups.
bool differential_f32_takes(const DifferentialArgs& args);
int differential_f32_forward(const DifferentialArgs& args, hipStream_t stream);
int differential_f32_backward(DifferentialArgs args, hipStream_t stream);

// A call's part of what key_block_parts goes by, and the parts for workgroups of `threads` each that one launch has room for.
KeyWalk key_walk(const DifferentialArgs& args);
int launchable_parts(const KeyWalk& walk, int threads);
// Takes a backward pass's scratch, [`statistics` floats per (batch, query, head) | dlambda's parts and the largest |dO| | parts of shared
// key blocks], and sets args' pointers and splits: at most `splits`, as many as an arena that cannot grow has room for.
int differential_backward_scratch(DifferentialArgs& args, int statistics, long lambda_parts, int splits, hipStream_t stream);
// dlambda from the parts that the dQ pass left, by the workgroups of the dK/dV pass that follows it, which has THREADS threads in each and
// none but this to add: a launch of its own took 3 to 5 us. From the last workgroup on, as the first ones have most to do. A
// head's sum has an order of its own, whatever the grid: every THREADS-th part in a thread, then a tree.
template <int THREADS>
__device__ __forceinline__ void add_lambda_parts(const DifferentialArgs& p, double* stage /* [THREADS / 64] */) {
    const unsigned int blocks = gridDim.x * gridDim.y * gridDim.z;
    const unsigned int linear = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
    for (unsigned int h = blocks - 1 - linear; h < static_cast<unsigned int>(p.hq); h += blocks) {
        const float* from = p.lambda_partial + h * p.lambda_parts;
        double sum = 0.0;
        for (long i = threadIdx.x; i < p.lambda_parts; i += THREADS) sum += from[i];
        sum = tree_sum_64(sum);
        __syncthreads();
        if (threadIdx.x % kWave == 0) stage[threadIdx.x / kWave] = sum;
        __syncthreads();
        if (threadIdx.x != 0) continue;
        for (int w = 1; w < THREADS / kWave; ++w) sum += stage[w];
        p.dlambda[h] = static_cast<float>(p.accumulate ? sum + p.dlambda[h] : sum);
    }
}

}  // namespace cgptx
