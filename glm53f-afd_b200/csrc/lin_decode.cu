// Linear attention with one decay a head, row by row: single tokens and windows of drafted ones.
//
//     S_t = e^g_t S_{t-1} + v_t k_t^T        y_t = scale S_t q_t        (S: [128 (v)][128 (k)] per request and head)
//
// Bound by HBM: a unit (request, head) reads and writes its state once, 64 or 32 KiB each way, beside 1 KiB a row.  The value rows of
// a state do not depend on one another, so a block of two warps takes a quarter of a unit and nothing is shared: a thread keeps four value rows x sixteen
// key channels in registers from the load to the store, all of its loads in flight at once, and walks the rows of the
// window.  Eight lanes make a value row's sum: the thread adds its sixteen products in order, then a halving exchange over the eight lanes adds the
// four rows' partial sums at once (four shuffles for four rows).  The arithmetic of a row does not depend on the call it
// comes in, and a bf16 state is rounded after every row: windows, commits and single rows leave the same bits.

#include "common.cuh"
#include "kda_internal.h"

namespace kda {
namespace {

constexpr int kLinThreads = 64, kLinSplit = 4;  // blocks a unit (of 128 threads, two a unit: 48 windows of 16 rows of f32 states 234 us, so 188; single rows the same)

struct LinStepParams {
    int heads, share;  // share: heads to a head of q and k
    const int32_t* cu;
    const int32_t* keep;
    const uint16_t *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    const float* g;
    long long g_stride;
    const void* state_in;
    void* state_out;
    const long long* state_off;
    float scale;
    uint16_t* out;
    long long out_stride;
};

// A row's inputs as a thread holds them: sixteen channels of q and k, four values, the log decay.
struct LinRow {
    uint4 q[2], k[2];
    uint2 v;
    float g;
};

__device__ __forceinline__ void widen8(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Two values rounded at once: one by one the conversions go through the unit of the transcendental functions, a quarter as fast (windows of 16 slots 36.6 us so, of which
// that unit was busy two thirds).
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A thread's four rows x (two runs of eight channels, 64 apart).  The vector forms need the state on 16 bytes.
template <bool BF16>
__device__ __forceinline__ void load_state(const void* base, long long at, bool vec, float (&s)[4][16]) {
    if constexpr (BF16) {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        if (vec) {
            uint4 r[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) r[i][j] = __ldcs(reinterpret_cast<const uint4*>(p + i * DK + 64 * j));
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) widen8(r[i][j], s[i] + 8 * j);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) s[i][j] = bf16_bits_to_f32(p[i * DK + 64 * (j >> 3) + (j & 7)]);
        }
    } else {
        const float* p = static_cast<const float*>(base) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* x = p + i * DK + 64 * (j >> 1) + 4 * (j & 1);
                if (vec) {
                    const float4 r = __ldcs(reinterpret_cast<const float4*>(x));
                    s[i][4 * j] = r.x, s[i][4 * j + 1] = r.y, s[i][4 * j + 2] = r.z, s[i][4 * j + 3] = r.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][4 * j + e] = x[e];
                }
            }
    }
}

template <bool BF16>
__device__ __forceinline__ void store_state(void* base, long long at, bool vec, const float (&s)[4][16]) {
    if constexpr (BF16) {
        uint16_t* p = static_cast<uint16_t*>(base) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float *x = &s[i][8 * j + 2 * e];
                    w[e] = bf16x2(x[0], x[1]);
                }
                if (vec) {
                    *reinterpret_cast<uint4*>(p + i * DK + 64 * j) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[i * DK + 64 * j + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                }
            }
    } else {
        float* p = static_cast<float*>(base) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float* x = p + i * DK + 64 * (j >> 1) + 4 * (j & 1);
                if (vec) {
                    *reinterpret_cast<float4*>(x) = make_float4(s[i][4 * j], s[i][4 * j + 1], s[i][4 * j + 2], s[i][4 * j + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = s[i][4 * j + e];
                }
            }
    }
}

__device__ __forceinline__ void to_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// ROUND: a bf16 state is rounded after every row (the prefill rounds once, when it stores).
template <bool BF16, bool ROUND>
__global__ void __launch_bounds__(kLinThreads, 8) lin_step_kernel(const __grid_constant__ LinStepParams p) {
    grid_ready();
    const long long unit = blockIdx.x / kLinSplit;
    const int b = (int)(unit / p.heads), h = (int)(unit % p.heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, oct = lane >> 3, l8 = lane & 7;
    const int row0 = ((int)(blockIdx.x % kLinSplit) * (kLinThreads / 32) + warp) * 16 + oct * 4;  // the thread's first value row
    const int first = p.cu[b];
    int n = p.cu[b + 1] - first;
    if (p.keep != nullptr) n = min(n, p.keep[b]);
    if (n <= 0 && (p.state_out == nullptr || p.state_out == p.state_in)) return;
    const long long off = p.state_off[b], at = off + ((long long)h * DV + row0) * DK + l8 * 8;
    const bool vec_in = ((reinterpret_cast<uintptr_t>(p.state_in) + (BF16 ? 2 : 4) * (uintptr_t)off) & 15) == 0;
    const bool vec_out = ((reinterpret_cast<uintptr_t>(p.state_out) + (BF16 ? 2 : 4) * (uintptr_t)off) & 15) == 0;

    const uint16_t* q = p.q + (long long)first * p.q_stride + (h / p.share) * DK + l8 * 8;
    const uint16_t* k = p.k + (long long)first * p.k_stride + (h / p.share) * DK + l8 * 8;
    const uint16_t* v = p.v + (long long)first * p.v_stride + h * DV + row0;
    const float* g = p.g + (long long)first * p.g_stride + h;
    auto fetch = [&](LinRow& x) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            x.q[j] = __ldg(reinterpret_cast<const uint4*>(q + 64 * j));
            x.k[j] = __ldg(reinterpret_cast<const uint4*>(k + 64 * j));
        }
        x.v = __ldg(reinterpret_cast<const uint2*>(v));
        x.g = __ldg(g);
        q += p.q_stride, k += p.k_stride, v += p.v_stride, g += p.g_stride;
    };
    LinRow next;
    if (n > 0) fetch(next);
    // A long window's other rows on their way to L2: loaded one row ahead, a row would take as long as memory does.  (48 windows of 16 rows of 64 heads 182 us, so 158,
    // of bf16 states 182 and 171; four windows of 8 rows of 8 heads 5.9 us, so 6.4: the copies come before the state's.)
    for (int t = 1 + (int)threadIdx.x; n > 8 && t < n; t += kLinThreads) {
        const uint16_t *qt = p.q + (long long)(first + t) * p.q_stride + (h / p.share) * DK, *kt = p.k + (long long)(first + t) * p.k_stride + (h / p.share) * DK;
        to_l2(qt), to_l2(qt + 64), to_l2(kt), to_l2(kt + 64);
        to_l2(p.v + (long long)(first + t) * p.v_stride + h * DV + (int)(blockIdx.x % kLinSplit) * (DV / kLinSplit));
        to_l2(p.g + (long long)(first + t) * p.g_stride + h);
    }
    float s[4][16];
    load_state<BF16>(p.state_in, at, vec_in, s);
    uint16_t* out = p.out == nullptr ? nullptr : p.out + (long long)first * p.out_stride + h * DV + row0;
    for (int t = 0; t < n; ++t) {
        const LinRow x = next;
        if (t + 1 < n) fetch(next);
        const float decay = expf(x.g);
        const float2 d2 = make_float2(decay, decay);
        const float val[4] = {__uint_as_float(x.v.x << 16), __uint_as_float(x.v.x & 0xffff0000u), __uint_as_float(x.v.y << 16),
                              __uint_as_float(x.v.y & 0xffff0000u)};
        float kk[16], qq[16];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            widen8(x.k[j], kk + 8 * j);
            widen8(x.q[j], qq + 8 * j);
        }
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v2 = make_float2(val[i], val[i]);
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float2 add = mul2(v2, make_float2(kk[j], kk[j + 1]));  // exact: two bf16 factors
                float2 z = fma2(make_float2(s[i][j], s[i][j + 1]), d2, add);
                if constexpr (BF16 && ROUND) {
                    const uint32_t two = bf16x2(z.x, z.y);
                    z = make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
                }
                s[i][j] = z.x, s[i][j + 1] = z.y;
                sum = fma2(z, make_float2(qq[j], qq[j + 1]), sum);
            }
            y[i] = sum.x + sum.y;
        }
        if (out != nullptr) {
            // Over the eight lanes of the four rows: lanes that differ in bit 2 take two rows each, in bit 1 one, in bit 0 add the halves.
            const bool up2 = l8 & 4, up1 = l8 & 2;
            float a = up2 ? y[2] : y[0], c = up2 ? y[3] : y[1];
            a += __shfl_xor_sync(0xffffffffu, up2 ? y[0] : y[2], 4);
            c += __shfl_xor_sync(0xffffffffu, up2 ? y[1] : y[3], 4);
            float e = up1 ? c : a;
            e += __shfl_xor_sync(0xffffffffu, up1 ? a : c, 2);
            e += __shfl_xor_sync(0xffffffffu, e, 1);
            if ((l8 & 1) == 0) out[l8 >> 1] = f32_to_bf16_bits(p.scale * e);
            out += p.out_stride;
        }
    }
    if (p.state_out != nullptr) store_state<BF16>(p.state_out, at, vec_out, s);
}

template <bool BF16, bool ROUND>
int step_launch(const LinStepParams& p, long long units, cudaStream_t stream) {
    return launch_early(lin_step_kernel<BF16, ROUND>, dim3((unsigned)(units * kLinSplit)), kLinThreads, 0, stream, p);
}

}  // namespace

bool lin_args_ok(int32_t heads, int32_t qk_heads, int32_t batch, const void* cu, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                 const void* v, int64_t v_stride, const void* g, int64_t g_stride, const void* state_in, const void* state_off, const void* out,
                 int64_t out_stride) {
    auto rows_ok = [](const void* x, int64_t stride, int32_t n) {
        return x != nullptr && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && stride % 8 == 0 && stride >= (int64_t)n * DK;
    };
    if (heads < 1 || heads > 65535 || qk_heads < 1 || heads % qk_heads || batch < 0) return false;
    if ((int64_t)heads * batch > 0x7fffffff / kLinSplit) return false;  // blocks of a launch
    if (batch == 0) return true;
    if (cu == nullptr || state_in == nullptr || state_off == nullptr || g == nullptr) return false;
    if (g_stride != 0 && g_stride < heads) return false;
    return rows_ok(q, q_stride, qk_heads) && rows_ok(k, k_stride, qk_heads) && rows_ok(v, v_stride, heads) && (out == nullptr || rows_ok(out, out_stride, heads));
}

int lin_rows_launch(int32_t heads, int32_t qk_heads, int32_t batch, const int32_t* cu, const int32_t* keep, const uint16_t* q, int64_t q_stride,
                    const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* g, int64_t g_stride, const void* state_in,
                    void* state_out, const int64_t* state_off, bool bf16_state, bool round_rows, float scale, uint16_t* out, int64_t out_stride,
                    cudaStream_t stream) {
    const LinStepParams p{heads, heads / qk_heads, cu, keep, q, k, v, q_stride, k_stride, v_stride, g, g_stride, state_in, state_out,
                          reinterpret_cast<const long long*>(state_off), scale, out, out_stride};
    const long long units = (long long)heads * batch;
    if (units == 0) return 0;
    if (!bf16_state) return step_launch<false, false>(p, units, stream);
    return round_rows ? step_launch<true, true>(p, units, stream) : step_launch<true, false>(p, units, stream);
}

}  // namespace kda

extern "C" int glm53f_kda_lin_decode_batch(int32_t heads, int32_t qk_heads, int32_t batch, const int32_t* cu_rows, const int32_t* keep,
                                           const glm53f_bf16* q, int64_t q_stride, const glm53f_bf16* k, int64_t k_stride, const glm53f_bf16* v,
                                           int64_t v_stride, const float* g, int64_t g_stride, const void* state_in, void* state_out,
                                           const int64_t* state_off, int32_t state_bf16, float scale, glm53f_bf16* out, int64_t out_stride,
                                           glm53f_stream_t stream) {
    using namespace kda;
    if (!lin_args_ok(heads, qk_heads, batch, cu_rows, q, q_stride, k, k_stride, v, v_stride, g, g_stride, state_in, state_off, out, out_stride)) return kInvalid;
    if (batch > 0 && state_out == nullptr && out == nullptr) return kInvalid;
    return lin_rows_launch(heads, qk_heads, batch, cu_rows, keep, q, q_stride, k, k_stride, v, v_stride, g, g_stride, state_in, state_out, state_off,
                           state_bf16 != 0, true, scale, out, out_stride, reinterpret_cast<cudaStream_t>(stream));
}
