// What the two projection kernels' translation units share.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "common.cuh"
#include "glm53f_proj.h"

namespace kda {

// What a launch with an epilogue adds to a product y: residual + act(y + bias).
struct ProjEpilogue {
    const void* bias;  // [groups][n], or none
    const void* residual;  // of the results' type, or none
    long long bias_gstride, ldr, r_gstride;
    int bias_f32, act;
};

__device__ __forceinline__ float proj_bias(const ProjEpilogue& e, int group, int feature) {
    const long long at = group * e.bias_gstride + feature;
    return e.bias_f32 ? __ldg(static_cast<const float*>(e.bias) + at) : bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(e.bias) + at));
}

// In forms that lose nothing where the result is small (1 + erf, 1 + tanh would).
__device__ __forceinline__ float proj_act(int act, float y) {
    switch (act) {
        case GLM53F_PROJ_RELU: return y < 0.0f ? 0.0f : y;  // (a NaN stays one)
        case GLM53F_PROJ_SILU: return y / (1.0f + expf(-y));
        case GLM53F_PROJ_GELU: return 0.5f * y * erfcf(y * -0.70710678f);
        case GLM53F_PROJ_GELU_TANH: return y / (1.0f + expf(-1.5957691f * (y + 0.044715f * y * y * y)));
        case GLM53F_PROJ_SIGMOID: return 1.0f / (1.0f + expf(-y));
        default: return y;
    }
}

// One GEMM of a launch on SM pairs: tensor maps of the weight (boxes of 128 rows), the activations (boxes of row_tile / 2 rows)
// and, for bf16 results in aligned rows, of the output (boxes of 16 rows x 64 features); (k or feature, row, group), or
// (., group, row) when `swapped`.
struct PairProblem {
    CUtensorMap tm_w, tm_x, tm_out;
    void* out;
    long long ldo, o_gstride;
    int rows, n, kblocks, segments;  // k blocks of 64; k runs in `segments` equal parts
    int out_f32, tensor_out;
    int row_tile, n_tiles, r_tiles;
    int w_swapped, x_swapped, out_swapped;
    long long tiles;
    ProjEpilogue epi;  // a launch with an epilogue only
};

constexpr int kPairProblems = 2;
constexpr int kPairSplitRows = 192;  // rows per tile at most when k runs in segments
// proj_gemm_pair.cu: launches the tiles of n (1 or 2) problems.
int proj_gemm_pair_launch(const PairProblem* problems, int n, bool epilogue, int* status, cudaStream_t stream);

}  // namespace kda
