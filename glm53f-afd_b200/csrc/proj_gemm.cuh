// What the two projection kernels' translation units share.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include <type_traits>

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

// 1 / (1 + e^-y).  The exponential's argument is rounded, which costs 2 |y| half steps of the result, here and in the next.  A result below 2^-126 (y < -87.3), a subnormal
// number, is 0: keeping those takes two to four more instructions, 0.4 to 0.5 us of 18.2 at two groups of 333 rows x 8,192 f32 results of k = 128.
__device__ __forceinline__ float proj_sigmoid(float y) { return rcp_approx(1.0f + ex2_ftz(y * -kLog2e)); }
// y / (1 + e^-z), down to the smallest subnormal, by x = e^(-|z| / 2): y w w / (1 + x^2) with w = x where z < 0 and 1 elsewhere, so that no factor is a subnormal number
// where the result is none.  (y times the sigmoid is 0 from z = -87.3 on, where the result is near -1e-36: 2,048 rows x 8,192 results of k = 4,096
// 112.9 us, so 113.5.)
__device__ __forceinline__ float proj_times_sigmoid(float y, float z) {
    const float x = ex2_ftz(fabsf(z) * (-0.5f * kLog2e)), w = z < 0.0f ? x : 1.0f;
    return (y * w) * (rcp_approx(fmaf(x, x, 1.0f)) * w);
}
// gelu(y) = max(y, 0) - |y| erfc(z) / 2, z = |y| / sqrt 2, in 18 instructions where the library's erfc takes more than twice as many (two groups of 2,048 rows x 8,192
// results of k = 128: 71 us, 126 with it, 42 without an activation; in two-wide operations the constants take registers that then spill).  erfc(z) / 2 = t 2^(2 e),
// t = 1 / (1 + z / 2), 2 e = P(t) - z^2 log2 e - 1: P is a polynomial of degree nine that was fitted to log2(erfc(z) e^(z^2) / t) over 0 < t <= 1 so that its largest
// error is least (the form of the complementary error function in Press et al., Numerical Recipes, section 6.2; 1.6e-7 of erfc).  In f32 the exponent's rounding adds to that: 5e-7 of erfc
// down to y = -2, 1.5e-6 to -5, 8e-6 to -13, where the result ends.  Half the exponent twice, so that results down to the smallest subnormal stay; |y| is cut off where there is no
// result left, so that infinities do not meet zeros.
__device__ __forceinline__ float proj_gelu(float y) {
    const float a = fminf(fabsf(y), 64.0f), t = rcp_approx(fmaf(a, 0.35355339f, 1.0f));
    float e = fmaf(t, 0.122096911f, -0.588332713f);
    e = fmaf(t, e, 1.06586015f);
    e = fmaf(t, e, -0.811956286f);
    e = fmaf(t, e, 0.197740987f);
    e = fmaf(t, e, -0.133445442f);
    e = fmaf(t, e, 0.0696902201f);
    e = fmaf(t, e, 0.26985532f);
    e = fmaf(t, e, 0.721364856f);
    e = fmaf(t, e, -1.4128741f);
    e = fmaf(a * (-0.25f * kLog2e), a, e);
    const float x = ex2_ftz(e);
    return (y < 0.0f ? 0.0f : y) - a * t * x * x;  // (a NaN stays one)
}
// In forms whose relative error stays small where the result is (that of 1 + tanh would not); a sigmoid below 2^-126 is 0.
template <int ACT>
__device__ __forceinline__ float proj_act(float y) {
    if constexpr (ACT == GLM53F_PROJ_RELU) return y < 0.0f ? 0.0f : y;  // (a NaN stays one)
    if constexpr (ACT == GLM53F_PROJ_SILU) return proj_times_sigmoid(y, y);
    if constexpr (ACT == GLM53F_PROJ_GELU) return proj_gelu(y);
    if constexpr (ACT == GLM53F_PROJ_GELU_TANH) return proj_times_sigmoid(y, 1.5957691f * (y + 0.044715f * y * y * y));
    if constexpr (ACT == GLM53F_PROJ_SIGMOID) return proj_sigmoid(y);
    return y;
}
// N values at once: one branch for all of them (one each made the epilogue of 2,048 x 8,192 results 25 us longer without any activation).
template <int N, typename B>
__device__ __forceinline__ void proj_finish(int act, float (&v)[N], B&& bias, const float* res) {
    auto all = [&](auto a) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = proj_act<decltype(a)::value>(v[j] + bias(j));
    };
    switch (act) {
        case GLM53F_PROJ_RELU: all(std::integral_constant<int, GLM53F_PROJ_RELU>{}); break;
        case GLM53F_PROJ_SILU: all(std::integral_constant<int, GLM53F_PROJ_SILU>{}); break;
        case GLM53F_PROJ_GELU: all(std::integral_constant<int, GLM53F_PROJ_GELU>{}); break;
        case GLM53F_PROJ_GELU_TANH: all(std::integral_constant<int, GLM53F_PROJ_GELU_TANH>{}); break;
        case GLM53F_PROJ_SIGMOID: all(std::integral_constant<int, GLM53F_PROJ_SIGMOID>{}); break;
        default: all(std::integral_constant<int, GLM53F_PROJ_NONE>{});
    }
    if (res != nullptr)
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = res[j] + v[j];
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
    // A launch with an epilogue only: its fields, and whether the residual comes by tensor copies (boxes of 16 rows x 64 features, as the results leave).
    ProjEpilogue epi;
    CUtensorMap tm_res;
    int res_boxes, res_swapped;
};

constexpr int kPairProblems = 2;
constexpr int kPairSplitRows = 192;  // rows per tile at most when k runs in segments
// proj_gemm_pair.cu: launches the tiles of n (1 or 2) problems.
int proj_gemm_pair_launch(const PairProblem* problems, int n, bool epilogue, int* status, cudaStream_t stream);

}  // namespace kda
