// Verification of drafted tokens: how many rows of each window to keep, and the token behind them.
//
// Per request, with p_i the target's distribution behind row i and q_i the one that token i was drawn from, token i + 1 is
// kept while u_{i+1} q_{i+1}(token) < p_i(token); the next token is drawn by a running sum from max(p - q, 0) of the first refused
// token's row, or from p behind a whole window.
//
// Bound by HBM for many requests (logits are read once for a row's maximum and sum; the row that is drawn from comes from L2 the
// second time) and by latency for one.  A request is a thread-block cluster: each block takes a slice of the vocabulary, all rows of the
// window; the slices' maxima and sums meet in distributed shared memory, every block makes the same decision, and all of
// them draw together: a warp sums a run of consecutive weights, the one whose run holds the drawn point looks for it.  One launch,
// no scratch in global memory, no atomics: the same result every time.
//
// A draw decides between neighbours of a sum over the whole vocabulary, so weights and sums are formed in 64 bits there: in 32, the sums'
// rounding moves one draw in a few hundred to the next token.  The maxima and sums that judge a token are 32-bit ones (a relative 1e-7
// of a probability against u).

#include "common.cuh"
#include "kda_internal.h"

namespace kda {
namespace {

constexpr int kAccThreads = 512, kAccWarps = kAccThreads / 32, kAccBlocks = 8;  // blocks a request
constexpr int kAccRows = 8;  // rows judged at a time

struct AcceptParams {
    const int32_t* cu;
    long long vocab, ld, draft_ld;
    const void* target;
    const int32_t* tokens;
    const float* draft;
    const float* temperature;
    const float* u;
    int32_t *keep, *next;
};

struct AccShared {
    // What this block's slice gives, read by the other blocks of the cluster.
    float max[kAccRows], sum[kAccRows];
    int best[kAccRows];
    double part;      // the slice's weights
    int last;         // the slice's last index with a weight, or -1
    // Within the block.
    float wmax[kAccRows][kAccWarps], wsum[kAccRows][kAccWarps];
    int wbest[kAccRows][kAccWarps];
    double wpart[kAccWarps];
    int wlast[kAccWarps];
    float row_max[kAccRows], row_sum[kAccRows];
    int row_best[kAccRows];
    int kept;
};

__device__ __forceinline__ uint32_t cluster_block() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_block(const void* local, uint32_t block) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(block));
    return r;
}
__device__ __forceinline__ float peer_f32(const void* local, uint32_t block) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at_block(local, block)) : "memory");
    return v;
}
__device__ __forceinline__ int peer_i32(const void* local, uint32_t block) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at_block(local, block)) : "memory");
    return v;
}
__device__ __forceinline__ double peer_f64(const void* local, uint32_t block) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at_block(local, block)) : "memory");
    return v;
}

constexpr float kNoLogit = -INFINITY;
template <int KIND>
__device__ __forceinline__ float target_at(const void* row, long long i) {
    if constexpr (KIND == GLM53F_KDA_LOGITS_BF16) return bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(row) + i));
    else return __ldg(static_cast<const float*>(row) + i);
}
// Eight consecutive entries from i on, those at `end` and beyond as `fill`.
template <int KIND>
__device__ __forceinline__ void target_8(const void* row, long long i, long long end, bool vec, float fill, float (&x)[8]) {
    if (vec && i + 8 <= end) {
        if constexpr (KIND == GLM53F_KDA_LOGITS_BF16) {
            const uint4 r = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + i));
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = __uint_as_float(w[j] << 16);
                x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        } else {
            const float4* r = reinterpret_cast<const float4*>(static_cast<const float*>(row) + i);
            const float4 a = __ldg(r), b = __ldg(r + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = i + j < end ? target_at<KIND>(row, i + j) : fill;
    }
}

// e^((l - max) / t) with the largest logits at exactly 1 (an infinite one too) and NaN at 0.
__device__ __forceinline__ double logit_weight(float l, float max, double inv_t) {
    if (l == max) return 1.0;
    const double e = exp(((double)l - (double)max) * inv_t);
    return l < max ? e : 0.0;
}
__device__ __forceinline__ float finite_weight(float p) { return p > 0.0f && p < INFINITY ? p : 0.0f; }

// The larger of two (value, lowest index) pairs; an index of -1 is none.
__device__ __forceinline__ void take_best(float& m, int& i, float om, int oi) {
    if (oi >= 0 && (i < 0 || om > m || (om == m && oi < i))) m = om, i = oi;
}

// What a draw weighs: the row's distribution p, less the drafter's, or without the refused token.
enum : int { kWhole = 0, kLessDraft = 1, kWithout = 2 };

template <int KIND>
__global__ void __launch_bounds__(kAccThreads) accept_kernel(const __grid_constant__ AcceptParams p) {
    constexpr bool LOGITS = KIND != GLM53F_KDA_PROBABILITIES;
    constexpr int kSize = KIND == GLM53F_KDA_LOGITS_BF16 ? 2 : 4;
    __shared__ AccShared sh;
    grid_ready();
    const int b = blockIdx.x / kAccBlocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t block = cluster_block();
    const int first = p.cu[b], n = p.cu[b + 1] - first;
    if (n <= 0) {  // the same for the whole cluster
        if (block == 0 && tid == 0) p.keep[b] = 0, p.next[b] = -1;
        return;
    }
    const unsigned char* rows = static_cast<const unsigned char*>(p.target) + (long long)first * p.ld * kSize;
    auto row_at = [&](int i) { return static_cast<const void*>(rows + (long long)i * p.ld * kSize); };
    auto draft_at = [&](int i) { return p.draft + (long long)(first + i) * p.draft_ld; };
    const bool vec = (reinterpret_cast<uintptr_t>(p.target) & 15) == 0 && (p.ld * kSize) % 16 == 0;
    const bool vec_draft = (reinterpret_cast<uintptr_t>(p.draft) & 15) == 0 && p.draft_ld % 4 == 0;
    // (Capped: an infinite one would make 0 times infinity of a logit of -inf.)
    const float temperature = LOGITS && p.temperature != nullptr ? (p.temperature[b] < 1e30f ? p.temperature[b] : 1e30f) : 1.0f;
    const bool greedy = LOGITS && !(temperature > 0.0f);
    const float scale = greedy ? 0.0f : kLog2e / temperature;
    const double inv_t = greedy ? 0.0 : 1.0 / (double)temperature;
    // This block's slice, in runs of eight.
    const long long runs = (p.vocab + 7) / 8, run0 = runs * block / kAccBlocks, run1 = runs * (block + 1) / kAccBlocks;

    int kept = 1;  // rows kept so far
    float stop_max = 0.0f;
    int stop_best = -1;
    for (int g0 = 0;; g0 += kAccRows) {
        const int rows_here = min(n - g0, kAccRows);
        if constexpr (LOGITS) {
            for (int i = 0; i < rows_here; ++i) {
                const void* row = row_at(g0 + i);
                float m = kNoLogit, s = 0.0f;
                int best = -1;
                for (long long r = run0 + tid; r < run1; r += kAccThreads) {
                    float x[8];
                    target_8<KIND>(row, 8 * r, p.vocab, vec, kNoLogit, x);
                    if (greedy) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (x[j] > m || (best < 0 && x[j] == m && 8 * r + j < p.vocab)) m = x[j], best = (int)(8 * r + j);
                    } else {
                        float top = x[0];
#pragma unroll
                        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
                        if (top > m) {
                            s *= m == kNoLogit ? 0.0f : ex2_approx((m - top) * scale);
                            m = top;
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) s += x[j] == m ? (m == kNoLogit ? 0.0f : 1.0f) : x[j] < m ? ex2_approx((x[j] - m) * scale) : 0.0f;
                    }
                }
                // (Sums at a maximum of -inf are 0, and so are their factors.)
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d);
                    const int ob = __shfl_xor_sync(0xffffffffu, best, d);
                    if (greedy) {
                        take_best(m, best, om, ob);
                    } else {
                        const float top = fmaxf(m, om);
                        s = (m == top ? s : s * ex2_approx((m - top) * scale)) + (om == top ? os : os * ex2_approx((om - top) * scale));
                        m = top;
                    }
                }
                if (lane == 0) sh.wmax[i][warp] = m, sh.wsum[i][warp] = s, sh.wbest[i][warp] = best;
            }
            __syncthreads();
            if (tid < rows_here) {
                float m = sh.wmax[tid][0], s = sh.wsum[tid][0];
                int best = sh.wbest[tid][0];
                for (int w = 1; w < kAccWarps; ++w) {
                    const float om = sh.wmax[tid][w], os = sh.wsum[tid][w];
                    if (greedy) {
                        take_best(m, best, om, sh.wbest[tid][w]);
                    } else {
                        const float top = fmaxf(m, om);
                        s = (m == top ? s : s * ex2_approx((m - top) * scale)) + (om == top ? os : os * ex2_approx((om - top) * scale));
                        m = top;
                    }
                }
                sh.max[tid] = m, sh.sum[tid] = s, sh.best[tid] = best;
            }
            cluster_meet();
            if (tid < rows_here) {
                float m = peer_f32(&sh.max[tid], 0), s = peer_f32(&sh.sum[tid], 0);
                int best = peer_i32(&sh.best[tid], 0);
                for (uint32_t c = 1; c < kAccBlocks; ++c) {
                    const float om = peer_f32(&sh.max[tid], c), os = peer_f32(&sh.sum[tid], c);
                    if (greedy) {
                        take_best(m, best, om, peer_i32(&sh.best[tid], c));
                    } else {
                        const float top = fmaxf(m, om);
                        s = (m == top ? s : s * ex2_approx((m - top) * scale)) + (om == top ? os : os * ex2_approx((om - top) * scale));
                        m = top;
                    }
                }
                sh.row_max[tid] = m, sh.row_sum[tid] = s, sh.row_best[tid] = best;
            }
            __syncthreads();
        }
        // Each lane of the first warp judges one row's token.
        if (warp == 0) {
            bool keep = false;
            const int i = g0 + lane;
            if (lane < rows_here && i + 1 < n) {
                const int token = p.tokens[first + i + 1];
                if (token >= 0 && token < p.vocab) {
                    if (greedy) {
                        keep = token == sh.row_best[lane] && sh.row_max[lane] != kNoLogit;
                    } else {
                        const double q = p.draft == nullptr ? 1.0 : (double)finite_weight(draft_at(i + 1)[token]);
                        const float x = target_at<KIND>(row_at(i), token);
                        const double left = (double)p.u[first + i + 1] * q;
                        if constexpr (LOGITS) keep = left * (double)sh.row_sum[lane] < logit_weight(x, sh.row_max[lane], inv_t) && sh.row_max[lane] != kNoLogit;
                        else keep = left < (double)finite_weight(x);
                    }
                }
            }
            const unsigned all = __ballot_sync(0xffffffffu, keep);
            if (lane == 0) sh.kept = __ffs(~all) - 1;  // (lanes from rows_here on keep nothing)
        }
        __syncthreads();
        const int run = sh.kept;
        kept = g0 + run + 1;
        if (run < rows_here) {  // a refused token, or the window's last row
            if constexpr (LOGITS) stop_max = sh.row_max[run], stop_best = sh.row_best[run];
            break;
        }
        cluster_meet();  // nobody writes the next rows' maxima while a block still reads these
    }
    const int stop = kept - 1;
    const bool whole = kept == n;
    if (block == 0 && tid == 0) {
        p.keep[b] = kept;
        if (greedy) p.next[b] = stop_max == kNoLogit ? -1 : stop_best;
    }
    // ---- the draw ----
    if (!greedy) {
        const void* row = row_at(stop);
        const float* less = whole || p.draft == nullptr ? nullptr : draft_at(stop + 1);
        const int token = whole ? -1 : p.tokens[first + stop + 1];
        int mode = whole ? kWhole : less != nullptr ? kLessDraft : kWithout;
        const double x01 = fmax((double)p.u[first], 0.0);
        double norm = 1.0;  // the weights' sum, by which the drafter's probabilities are multiplied instead of dividing each of p's
        auto weights = [&](long long i, double (&w)[8]) {
            float x[8];
            target_8<KIND>(row, i, p.vocab, vec, LOGITS ? kNoLogit : 0.0f, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (LOGITS) w[j] = stop_max == kNoLogit ? 0.0 : logit_weight(x[j], stop_max, inv_t);
                else w[j] = (double)finite_weight(x[j]);
            }
            if (mode == kLessDraft) {
                float y[8];
                target_8<GLM53F_KDA_PROBABILITIES>(less, i, p.vocab, vec_draft, 0.0f, y);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double rest = w[j] - (double)finite_weight(y[j]) * norm;
                    w[j] = rest > 0.0 ? rest : 0.0;
                }
            } else if (mode == kWithout) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (i + j == token) w[j] = 0.0;
            }
        };
        // A warp's runs of the slice, consecutive ones.
        const long long mine0 = run0 + (run1 - run0) * warp / kAccWarps, mine1 = run0 + (run1 - run0) * (warp + 1) / kAccWarps;
        // The slice's sum into sh.part; returns all slices', and the sum before this block's.
        auto sum_up = [&](double& before, int& last_of_all) {
            double s = 0.0;
            int last = -1;
            for (long long r = mine0 + lane; r < mine1; r += 32) {
                double w[8];
                weights(8 * r, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    s += w[j];
                    if (w[j] > 0.0) last = (int)(8 * r + j);
                }
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, d);
                last = max(last, __shfl_xor_sync(0xffffffffu, last, d));
            }
            if (lane == 0) sh.wpart[warp] = s, sh.wlast[warp] = last;
            __syncthreads();
            if (tid == 0) {
                double t = 0.0;
                int l = -1;
                for (int w = 0; w < kAccWarps; ++w) t += sh.wpart[w], l = max(l, sh.wlast[w]);
                sh.part = t, sh.last = l;
            }
            cluster_meet();
            double all = 0.0;
            last_of_all = -1;
            for (uint32_t c = 0; c < kAccBlocks; ++c) {
                if (c == block) before = all;
                all += peer_f64(&sh.part, c);
                last_of_all = max(last_of_all, peer_i32(&sh.last, c));
            }
            cluster_meet();  // read everywhere before it is written again, and before a block leaves
            return all;
        };
        double before = 0.0;
        int last = -1;
        if (LOGITS && mode == kLessDraft) {
            mode = kWhole;
            norm = sum_up(before, last);
            mode = kLessDraft;
        }
        double total = sum_up(before, last);
        if (!(total > 0.0) && mode != kWhole) {
            mode = kWhole;
            total = sum_up(before, last);
        }
        const double point = x01 * total;
        if (!(total > 0.0)) {
            if (block == 0 && tid == 0) p.next[b] = -1;
        } else if (block == 0 && tid == 0 && !(point < total)) {
            p.next[b] = last;  // (u at its largest, rounded up to the whole)
        } else if (point < total) {
            // The warp whose run holds the point; the sums are those that made the total, added in the same order.
            double lo = before, own = 0.0;
            bool here = false;
            {
                double s = 0.0;
                for (int w = 0; w < kAccWarps; ++w) {
                    const double to = s + sh.wpart[w];
                    if (w == warp) lo = before + s, own = before + to;
                    s = to;
                }
                here = lo <= point && point < own;
            }
            if (here) {
                double sum = lo;
                int found = -1, seen = -1;
                for (long long r = mine0; r < mine1 && found < 0; r += 32) {
                    double w[8], s = 0.0;
                    if (r + lane < mine1) {
                        weights(8 * (r + lane), w);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = 0.0;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) s += w[j];
                    double upto = s;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const double o = __shfl_up_sync(0xffffffffu, upto, d);
                        if (lane >= d) upto += o;
                    }
                    double at = sum + (upto - s);
                    int hit = 0x7fffffff;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        at += w[j];
                        if (w[j] > 0.0) {
                            seen = (int)(8 * (r + lane) + j);
                            if (at > point && hit == 0x7fffffff) hit = seen;
                        }
                    }
                    hit = __reduce_min_sync(0xffffffffu, hit);
                    if (hit != 0x7fffffff) found = hit;
                    sum += __shfl_sync(0xffffffffu, upto, 31);
                }
                seen = __reduce_max_sync(0xffffffffu, seen);
                if (lane == 0) p.next[b] = found >= 0 ? found : seen;  // (seen: the last of the run, should the sums' order leave the point behind it)
            }
        }
    } else {
        cluster_meet();  // no block leaves while another may still read its sums
    }
}

template <int KIND>
int accept_launch(const AcceptParams& p, int batch, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)batch * kAccBlocks);
    cfg.blockDim = dim3(kAccThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kAccBlocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + early_attribute(attr[1]);
    return (int)cudaLaunchKernelEx(&cfg, accept_kernel<KIND>, p);
}

}  // namespace
}  // namespace kda

extern "C" int glm53f_kda_accept_batch(int32_t batch, const int32_t* cu_rows, int32_t vocab, const void* target, int32_t target_kind, int64_t ld,
                                       const int32_t* tokens, const float* draft, int64_t draft_ld, const float* temperature, const float* u,
                                       int32_t* keep, int32_t* next, glm53f_stream_t stream_) {
    using namespace kda;
    if (batch < 0 || batch > 0xfffffff || vocab < 1 || ld < vocab) return kInvalid;
    if (target_kind < GLM53F_KDA_PROBABILITIES || target_kind > GLM53F_KDA_LOGITS_BF16) return kInvalid;
    if (target_kind == GLM53F_KDA_PROBABILITIES && temperature != nullptr) return kInvalid;
    if (draft != nullptr && draft_ld < vocab) return kInvalid;
    if (batch == 0) return 0;
    if (!cu_rows || !target || !tokens || !u || !keep || !next) return kInvalid;
    if ((reinterpret_cast<uintptr_t>(target) & (target_kind == GLM53F_KDA_LOGITS_BF16 ? 1 : 3)) != 0 || (reinterpret_cast<uintptr_t>(draft) & 3) != 0) return kInvalid;
    const AcceptParams p{cu_rows, vocab, ld, draft_ld, target, tokens, draft, temperature, u, keep, next};
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (target_kind == GLM53F_KDA_LOGITS_F32) return accept_launch<GLM53F_KDA_LOGITS_F32>(p, batch, stream);
    if (target_kind == GLM53F_KDA_LOGITS_BF16) return accept_launch<GLM53F_KDA_LOGITS_BF16>(p, batch, stream);
    return accept_launch<GLM53F_KDA_PROBABILITIES>(p, batch, stream);
}
