// Linear attention with one decay a head: the prefill of packed sequences.

#include "common.cuh"
#include "kda_internal.h"

extern "C" int64_t glm53f_kda_lin_prefill_workspace_bytes(int32_t heads, int32_t batch, int32_t max_len) {
    if (heads < 1 || heads > 65535 || batch < 0 || max_len < 0) return 0;
    return 0;
}

extern "C" int glm53f_kda_lin_prefill_varlen(int32_t heads, int32_t qk_heads, int32_t batch, const int32_t* cu_rows, int32_t rows, int32_t max_len,
                                             const glm53f_bf16* q, int64_t q_stride, const glm53f_bf16* k, int64_t k_stride, const glm53f_bf16* v,
                                             int64_t v_stride, const float* g, int64_t g_stride, const void* state_in, void* state_out,
                                             const int64_t* state_off, int32_t state_bf16, float scale, glm53f_bf16* out, int64_t out_stride,
                                             void* workspace, int64_t workspace_bytes, glm53f_stream_t stream) {
    using namespace kda;
    if (rows < 0 || max_len < 0 || max_len > rows || workspace_bytes < 0 || (workspace == nullptr && workspace_bytes > 0)) return kInvalid;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return kInvalid;
    if (!lin_args_ok(heads, qk_heads, batch, cu_rows, q, q_stride, k, k_stride, v, v_stride, g, g_stride, state_in, state_off, out, out_stride)) return kInvalid;
    if (batch == 0) return 0;
    if (state_out == nullptr || out == nullptr) return kInvalid;
    return lin_rows_launch(heads, qk_heads, batch, cu_rows, nullptr, q, q_stride, k, k_stride, v, v_stride, g, g_stride, state_in, state_out, state_off,
                           state_bf16 != 0, false, scale, out, out_stride, reinterpret_cast<cudaStream_t>(stream));
}
