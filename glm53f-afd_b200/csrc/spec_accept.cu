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

#include <type_traits>

#include "common.cuh"
#include "kda_internal.h"

namespace kda {
namespace {

constexpr int kAccMostWarps = 16;   // of a block: 8 or 16
constexpr int kAccMostBlocks = 16;  // blocks a request, 8 or 16
constexpr int kAccRows = 8;         // rows judged at a time

struct AcceptParams {
    const int32_t* cu;
    long long vocab, ld, draft_ld;
    const void* target;
    const int32_t* tokens;
    const float* draft;
    const float* temperature;
    const float* u;
    int32_t *keep, *next;
    int blocks;
};

struct AccShared {
    double power[32];  // 2^(j / 32)
    // What this block's slice gives, read by the other blocks of the cluster.
    float max[kAccRows], sum[kAccRows];
    int best[kAccRows];
    double part;      // the slice's weights
    // Within the block.
    float wmax[kAccRows][kAccMostWarps], wsum[kAccRows][kAccMostWarps];
    int wbest[kAccRows][kAccMostWarps];
    double wpart[kAccMostWarps];
    double slot[kAccMostWarps][32];  // a warp's weights, its places in 32 parts
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
// The two halves of it, for what need not be waited for at once.
__device__ __forceinline__ void cluster_said() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_heard() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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
// Eight consecutive entries from i on as they lie in memory (vector loads; or, where the row's end or its alignment rules those out, one at a
// time, those at `end` and beyond as `fill`), and as floats.  Apart, so that several loads are in flight before the first is looked at.
template <int KIND>
struct Eight {
    static constexpr int kWords = KIND == GLM53F_KDA_LOGITS_BF16 ? 4 : 8;
    uint32_t w[kWords];
    __device__ __forceinline__ void load_whole(const void* row, long long i) {
#pragma unroll
        for (int j = 0; j < kWords; j += 4) {
            const uint4 r = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(row) + i * (kWords / 2)) + j / 4);
            w[j] = r.x, w[j + 1] = r.y, w[j + 2] = r.z, w[j + 3] = r.w;
        }
    }
    __device__ __forceinline__ void load_some(const void* row, long long i, long long end, float fill) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = __float_as_uint(i + j < end ? target_at<KIND>(row, i + j) : fill);
            if constexpr (kWords == 8) w[j] = u;
            else w[j >> 1] = j & 1 ? w[j >> 1] | (u & 0xffff0000u) : u >> 16;
        }
    }
    __device__ __forceinline__ void load(const void* row, long long i, long long end, bool vec, float fill) {
        if (vec && i + 8 <= end) load_whole(row, i);
        else load_some(row, i, end, fill);
    }
    // The largest of them (NaN only where all are).
    __device__ __forceinline__ float top() const {
        if constexpr (kWords == 8) {
            const float* x = reinterpret_cast<const float*>(w);
            return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        } else {
            const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(w);
            const __nv_bfloat162 m = __hmax2(__hmax2(x[0], x[1]), __hmax2(x[2], x[3]));
            return fmaxf(__low2float(m), __high2float(m));
        }
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (kWords == 8) x[j] = __uint_as_float(w[j]);
            else x[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
        }
    }
};

// A row's weights in 64 bits: e^x of x = (l - max) / t <= 0.  x = (32 e + j) ln 2 / 32 + r, so e^x = 2^e 2^(j/32) e^r with |r| < 0.011, of which
// Taylor's series to the fourth power leaves 1.3e-12: a draw among 131,072 moves by it once in ten million.  (With the general exponential, and every
// special case looked at for every entry, a draw's pass took four times as many instructions.)  NaN and what is below e^-690 is 0.  Rows whose
// largest is infinite: see weights() in the kernel.
constexpr double kTurns = 46.166241308446828384;  // 32 / ln 2
struct RowScale {
    double max, inv_t, turns;  // turns: inv_t 32 / ln 2
};
__device__ __forceinline__ double logit_weight(float l, const RowScale& a, const double* power) {
    const double magic = 6755399441055744.0;  // 1.5 2^52: adding it rounds to an integer, which the low word then holds
    const double d = (double)l - a.max, x = d * a.inv_t, shifted = fma(d, a.turns, magic);
    const int n = __double2loint(shifted);
    const double whole = shifted - magic;
    double r = fma(whole, -0.021660849390173098, x);
    r = fma(whole, -2.325192846878874e-12, r);
    double y = fma(r, 1.0 / 24, 1.0 / 6);
    y = fma(r, y, 0.5);
    y = fma(r, y, 1.0);
    y = fma(r, y, 1.0);
    const double base = power[n & 31];
    return x > -690.0 ? y * __hiloint2double(__double2hiint(base) + ((n >> 5) << 20), __double2loint(base)) : 0.0;
}
__device__ __forceinline__ float finite_weight(float p) { return p > 0.0f && p < INFINITY ? p : 0.0f; }

// A row's statistics: its largest logit m, the sum of 2^((l - m) scale) over it, the lowest index of the largest (greedy).  A sum at a maximum of -inf is 0.
struct Stats {
    float m = kNoLogit, s = 0.0f;
    int best = -1;
};
template <bool GREEDY, int KIND>
__device__ __forceinline__ void take(Stats& a, const Eight<KIND>& in, int at, long long vocab, float scale) {
    const float top = in.top();
    float x[8];
    if constexpr (GREEDY) {
        if (top > a.m || a.best < 0) {
            in.get(x);
            a.m = fmaxf(top, a.m);
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (x[j] == top && at + j < vocab) a.best = at + j;
        }
    } else {
        if (top > a.m) {
            a.s *= a.m == kNoLogit ? 0.0f : ex2_approx((a.m - top) * scale);
            a.m = top;
        }
        in.get(x);
        float2 sum[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = mul2(fma2(make_float2(a.m, a.m), make_float2(-1.0f, -1.0f), make_float2(x[2 * j], x[2 * j + 1])), make_float2(scale, scale));
            sum[j] = make_float2(ex2_ftz(t.x), ex2_ftz(t.y));
        }
        float all = ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) + ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
        if (!(all < INFINITY)) {  // a NaN among them, or infinities: seldom, so one at a time
            all = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) all += x[j] == a.m ? (a.m == kNoLogit ? 0.0f : 1.0f) : x[j] < a.m ? ex2_ftz((x[j] - a.m) * scale) : 0.0f;
        }
        a.s += all;
    }
}
// Over the lanes of a warp.
template <bool GREEDY>
__device__ __forceinline__ void join_lanes(Stats& a, float scale) {
    float m = a.m;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if constexpr (GREEDY) {
        a.best = (int)__reduce_min_sync(0xffffffffu, a.best >= 0 && a.m == m ? (unsigned)a.best : 0xffffffffu);  // (none is -1)
    } else {
        float s = a.m == m ? a.s : a.s * ex2_ftz((a.m - m) * scale);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        a.s = s;
    }
    a.m = m;
}

// What a draw weighs: the row's distribution p, less the drafter's, or without the refused token.
enum : int { kWhole = 0, kLessDraft = 1, kWithout = 2 };

template <int KIND, int kAccWarps>
__global__ void __launch_bounds__(kAccWarps * 32, kAccWarps == 8 ? 3 : 1) accept_kernel(const __grid_constant__ AcceptParams p) {
    constexpr int kAccThreads = kAccWarps * 32, kAccDeep = KIND == GLM53F_KDA_LOGITS_BF16 ? 4 : 2;  // (rows read side by side)
    constexpr bool LOGITS = KIND != GLM53F_KDA_PROBABILITIES;
    constexpr int kSize = KIND == GLM53F_KDA_LOGITS_BF16 ? 2 : 4;
    __shared__ AccShared sh;
    if (threadIdx.x < 32) sh.power[threadIdx.x] = exp2((double)threadIdx.x / 32);
    grid_ready();
    const int blocks = p.blocks, b = blockIdx.x / blocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
    const long long runs = (p.vocab + 7) / 8, run0 = runs * block / blocks, run1 = runs * (block + 1) / blocks;

    __syncthreads();  // the powers
    int kept = 1;  // rows kept so far
    float stop_max = 0.0f;
    int stop_best = -1;
    for (int g0 = 0;; g0 += kAccRows) {
        const int rows_here = min(n - g0, kAccRows);
        // What the first warp's lanes judge, a row each, on its way meanwhile.
        int token = -1;
        float token_target = 0.0f;
        double token_left = 0.0;
        if (warp == 0 && lane < rows_here && g0 + lane + 1 < n) {
            const int i = g0 + lane;
            token = p.tokens[first + i + 1];
            if (token < 0 || token >= p.vocab) token = -1;
            if (token >= 0 && !greedy) {
                token_target = target_at<KIND>(row_at(i), token);
                token_left = (double)p.u[first + i + 1] * (p.draft == nullptr ? 1.0 : (double)fmaxf(draft_at(i + 1)[token], 0.0f));
            }
        }
        if constexpr (LOGITS) {
            auto read = [&](auto is_greedy) {
                constexpr bool GREEDY = decltype(is_greedy)::value;
                for (int i0 = 0; i0 < rows_here; i0 += kAccDeep) {
                    Stats st[kAccDeep];
                    const int deep = min(rows_here - i0, kAccDeep);
                    // All rows' entries at a place side by side, the next place's on their way while these are looked at.
                    Eight<KIND> now[kAccDeep], ahead[kAccDeep];
                    auto load = [&](long long r, Eight<KIND>(&to)[kAccDeep]) {
                        if (vec && 8 * r + 8 <= p.vocab) {
#pragma unroll
                            for (int d = 0; d < kAccDeep; ++d) to[d].load_whole(row_at(g0 + i0 + min(d, deep - 1)), 8 * r);
                        } else {
#pragma unroll
                            for (int d = 0; d < kAccDeep; ++d) to[d].load_some(row_at(g0 + i0 + min(d, deep - 1)), 8 * r, p.vocab, kNoLogit);
                        }
                    };
                    if (run0 + tid < run1) load(run0 + tid, now);
                    for (long long r = run0 + tid; r < run1; r += kAccThreads) {
                        if (r + kAccThreads < run1) load(r + kAccThreads, ahead);
#pragma unroll
                        for (int d = 0; d < kAccDeep; ++d) {
                            take<GREEDY>(st[d], now[d], (int)(8 * r), p.vocab, scale);
                            now[d] = ahead[d];
                        }
                    }
#pragma unroll
                    for (int d = 0; d < kAccDeep; ++d) {
                        join_lanes<GREEDY>(st[d], scale);
                        if (lane == 0 && d < deep) sh.wmax[i0 + d][warp] = st[d].m, sh.wsum[i0 + d][warp] = st[d].s, sh.wbest[i0 + d][warp] = st[d].best;
                    }
                }
                // A warp to a row: over the block's warps, then over the cluster's blocks.
                __syncthreads();
                if (warp < rows_here) {
                    Stats a;
                    if (lane < kAccWarps) a.m = sh.wmax[warp][lane], a.s = sh.wsum[warp][lane], a.best = sh.wbest[warp][lane];
                    join_lanes<GREEDY>(a, scale);
                    if (lane == 0) sh.max[warp] = a.m, sh.sum[warp] = a.s, sh.best[warp] = a.best;
                }
                cluster_meet();
                if (warp < rows_here) {
                    Stats a;
                    if (lane < blocks) {
                        a.m = peer_f32(&sh.max[warp], lane);
                        if constexpr (GREEDY) a.best = peer_i32(&sh.best[warp], lane);
                        else a.s = peer_f32(&sh.sum[warp], lane);
                    }
                    join_lanes<GREEDY>(a, scale);
                    if (lane == 0) sh.row_max[warp] = a.m, sh.row_sum[warp] = a.s, sh.row_best[warp] = a.best;
                }
                __syncthreads();
            };
            if (greedy) read(std::true_type{});
            else read(std::false_type{});
        }
        // Each lane of the first warp judges one row's token.
        if (warp == 0) {
            bool keep = false;
            if (token >= 0) {
                if (greedy) keep = token == sh.row_best[lane] && sh.row_max[lane] != kNoLogit;
                else if constexpr (LOGITS)
                {
                    const float m = sh.row_max[lane];
                    const double e = token_target == m ? 1.0 : m < INFINITY ? logit_weight(token_target, {(double)m, inv_t, inv_t * kTurns}, sh.power) : 0.0;
                    keep = token_left * (double)sh.row_sum[lane] < e && m != kNoLogit;
                }
                else keep = token_left < (double)finite_weight(token_target);
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
        // (Short of 1, whatever is given: the drawn point then lies before the whole.)
        const double x01 = fmin(fmax((double)p.u[first], 0.0), 1.0 - 0x1p-53);
        const RowScale row_scale{(double)stop_max, inv_t, inv_t * kTurns};
        double norm = 1.0;  // the weights' sum, by which the drafter's probabilities are multiplied instead of dividing each of p's
        struct Place {
            Eight<KIND> x;
            Eight<GLM53F_KDA_PROBABILITIES> y;
        };
        auto fetch = [&](long long i, Place& a) {
            a.x.load(row, i, p.vocab, vec, LOGITS ? kNoLogit : 0.0f);
            if (mode == kLessDraft) a.y.load(less, i, p.vocab, vec_draft, 0.0f);
        };
        auto weights = [&](long long i, const Place& a, double (&w)[8]) {
            float x[8];
            a.x.get(x);
            if constexpr (!LOGITS) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = (double)finite_weight(x[j]);
            } else if (fabsf(stop_max) < INFINITY) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = logit_weight(x[j], row_scale, sh.power);
            } else {  // infinite logits share everything; of -inf alone nothing is left
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = x[j] == INFINITY ? 1.0 : 0.0;
            }
            if (mode == kLessDraft) {
                float y[8];
                a.y.get(y);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double rest = fma((double)fmaxf(y[j], 0.0f), -norm, w[j]);
                    w[j] = rest > 0.0 ? rest : 0.0;
                }
            } else if (mode == kWithout && token >= i && token < i + 8) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (i + j == token) w[j] = 0.0;
            }
        };
        // A warp's runs of the slice, consecutive ones, in up to 32 slots of `group` steps of 32 runs.
        const long long mine0 = run0 + (run1 - run0) * warp / kAccWarps, mine1 = run0 + (run1 - run0) * (warp + 1) / kAccWarps;
        const int steps = (int)((mine1 - mine0 + 31) / 32), group = (steps + 31) / 32;
        double before = 0.0, total = 0.0;
        // Passes over the row, one body of code: of logits with the drafter's probabilities first the weights' sum, then what is drawn from, and
        // once more where that leaves nothing.
        const int drawn_from = mode;
        if (LOGITS && drawn_from == kLessDraft) mode = kWhole;
        for (bool said = false;; said = true) {
            int in_slot = 0, slot = 0;
            double part = 0.0, s = 0.0;
            Place now, ahead;
            if (mine0 + lane < mine1) fetch(8 * (mine0 + lane), now);
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
                const long long r = mine0 + 32 * k + lane;
                if (r + 32 < mine1) fetch(8 * (r + 32), ahead);
                if (r < mine1) {
                    double w[8];
                    weights(8 * r, now, w);
                    s += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                }
                now = ahead;
                if (++in_slot == group || k + 1 == steps) {
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
                    if (lane == 0) sh.slot[warp][slot] = s;
                    part += s;
                    s = 0.0;
                    in_slot = 0;
                    ++slot;
                }
            }
            if (lane == 0) sh.wpart[warp] = part;
            __syncthreads();
            if (said) cluster_heard();  // (the last pass's sums have been read everywhere)
            if (tid == 0) {
                double t = 0.0;
                for (int w = 0; w < kAccWarps; ++w) t += sh.wpart[w];
                sh.part = t;
            }
            cluster_meet();
            // Every warp adds the blocks' sums in the same order; each lane has fetched one.
            const double theirs = lane < blocks ? peer_f64(&sh.part, lane) : 0.0;
            total = 0.0;
            for (int c = 0; c < blocks; ++c) {
                if (c == (int)block) before = total;
                total += __shfl_sync(0xffffffffu, theirs, c);
            }
            cluster_said();
            if (mode == kWhole && drawn_from == kLessDraft && LOGITS && !said) {
                norm = total;
                mode = kLessDraft;
            } else if (!(total > 0.0) && mode != kWhole) {
                mode = kWhole;
            } else {
                break;
            }
        }
        const double point = x01 * total;
        if (!(total > 0.0)) {
            if (block == 0 && tid == 0) p.next[b] = -1;
        } else {
            // The warp whose runs hold the point, and the slot; the sums are those that made the total, added in the same order.
            double lo = before, s = 0.0;
            bool here = false;
            for (int w = 0; w < kAccWarps; ++w) {
                const double to = s + sh.wpart[w];
                if (w == warp) lo = before + s, here = before + s <= point && point < before + to;
                s = to;
            }
            if (here) {
                int slot = 0;
                double at_slot = 0.0;  // (lo + the slots before: the warp's sum was added up in this order)
                const int slots = (steps + group - 1) / group;
                while (slot + 1 < slots && !(point < lo + (at_slot + sh.slot[warp][slot]))) at_slot += sh.slot[warp][slot++];
                double sum = lo + at_slot;
                int found = -1, seen = -1;
                // (Through to the warp's last step: should the sums' rounding leave the point behind the slot, it is the first weight behind it.)
#pragma unroll 1
                for (int k = slot * group; k < steps && found < 0; ++k) {
                    const long long r = mine0 + 32 * k + lane;
                    double w[8], s8 = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = 0.0;
                    if (r < mine1) {
                        Place a;
                        fetch(8 * r, a);
                        weights(8 * r, a, w);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) s8 += w[j];
                    double upto = s8;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const double o = __shfl_up_sync(0xffffffffu, upto, d);
                        if (lane >= d) upto += o;
                    }
                    double at = sum + (upto - s8);
                    int hit = 0x7fffffff;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        at += w[j];
                        if (w[j] > 0.0) {
                            seen = (int)(8 * r + j);
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
        cluster_heard();  // no block leaves while another may still read its sums
    } else {
        cluster_meet();
    }
}

template <int KIND, int WARPS>
int accept_launch(AcceptParams p, int batch, int blocks, cudaStream_t stream) {
    p.blocks = blocks;
    static int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        const cudaError_t e = cudaFuncSetAttribute(accept_kernel<KIND, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
        configured_dev = dev;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)batch * p.blocks);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + early_attribute(attr[1]);
    return (int)cudaLaunchKernelEx(&cfg, accept_kernel<KIND, WARPS>, p);
}

// Few requests: as many threads each as a cluster can have, while every block has an SM.  Many: blocks of which an SM holds two.
template <int KIND>
int accept_launch(const AcceptParams& p, int batch, cudaStream_t stream) {
    const long long sms = sm_count();
    if (batch * (long long)kAccMostBlocks <= sms) return accept_launch<KIND, kAccMostWarps>(p, batch, kAccMostBlocks, stream);
    if (batch * 8ll <= sms) return accept_launch<KIND, kAccMostWarps>(p, batch, 8, stream);
    return accept_launch<KIND, 8>(p, batch, 8, stream);
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
    const AcceptParams p{cu_rows, vocab, ld, draft_ld, target, tokens, draft, temperature, u, keep, next, 8};
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (target_kind == GLM53F_KDA_LOGITS_F32) return accept_launch<GLM53F_KDA_LOGITS_F32>(p, batch, stream);
    if (target_kind == GLM53F_KDA_LOGITS_BF16) return accept_launch<GLM53F_KDA_LOGITS_BF16>(p, batch, stream);
    return accept_launch<GLM53F_KDA_PROBABILITIES>(p, batch, stream);
}
