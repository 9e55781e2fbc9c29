// Log probabilities of given tokens from rows of logits, with entropy and the best alternatives, and the logits' gradient.
//
// With t_j = (x_j - max x) / T and S = sum of e^t_j: log p_j = t_j - log S, entropy = log S - (sum of e^t_j t_j) / S.  Backwards, from the gradients
// l of the token's log probability and n of the entropy H: dx_j = (l ([j = token] - p_j) - n p_j (log p_j + H)) / T.
//
// Bound by HBM and the operations next to it: a row is read once (one exponential, 2/3 of what the units give at bf16 logits, and five or six instructions a value, in pairs).  Every warp keeps
// its running maximum, its lanes their sums against it, so that the maxima need no pass of their own; blocks of a cluster that share a row meet
// in distributed shared memory.  No scratch in global memory; the same bits every time.  336 rows of 131,072 bf16 logits take 25.9 us, 3.4 TB/s (1,000 rows
// 3.8), with five alternatives 30.6; one f32 row 4.6 us, with twenty 12.2: the rounds that find them, one after another.  Backwards 2,048 rows take 181 us, 5.9 TB/s.
//
// The alternatives need no second pass either.  Each thread knows the largest value it met; 128 groups of threads are 128 disjoint parts of the row, so the
// k-th largest of the groups' maxima is no larger than the row's k-th largest value.  Of the row's pieces of 32 x 16 bytes, whose
// maxima lie in shared memory, those that reach this bound (few more than k) are read again from L2, and the few values in them that reach it are
// ranked by counting.  Equal logits rank by index.  Rows of so many equal values that these do not fit take k rounds over the row instead.

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "kda_internal.h"

namespace kda {
namespace {

constexpr int kGroups = 128;
constexpr int kMostTop = 32;
constexpr int kPieces = 2048;     // of a block's part of a row
constexpr int kCandidates = 512;  // of a block's part; kMostBlocks * kMostTop at least
constexpr int kMostBlocks = 8;    // of a row
constexpr int kMostVocab = 2000000;  // (kMostBlocks * kPieces pieces hold 2,097,152 f32 logits)
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobParams {
    const void* logits;
    long long ld;
    int vocab, blocks, top;
    const int32_t* tokens;
    const float* temperature;
    float *logprob, *entropy, *lse;
    int32_t* top_ids;
    float* top_values;
    // backward
    const float *dlogprob, *dentropy;
    void* dlogits;
    long long dld;
};

struct Entry {
    float v;
    int id;
};
__device__ __forceinline__ bool before(const Entry& a, const Entry& b) { return a.v > b.v || (a.v == b.v && a.id < b.id); }

template <int WARPS>
struct Shared {
    float piece[kPieces];
    Entry candidate[kCandidates];
    int ahead[kCandidates];
    alignas(16) float group[32 * WARPS];
    Entry best[kMostTop];  // this block's, read by the row's first block
    float max, sum, sum_t;
    float wmax[WARPS], wsum[WARPS], wsum_t[WARPS];
    Entry wbest[WARPS];
    float bound;
    int candidates;
};

__device__ __forceinline__ float warp_max(float x) {  // NaN only where all are
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ __forceinline__ uint32_t cluster_place(const void* local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
    return r;
}
__device__ __forceinline__ float cluster_load(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// log2(e) / T.  A temperature of 0 or less (a row whose choice is greedy) and NaN: 1.
__device__ __forceinline__ float heat_of(const float* temperature, long long row) {
    const float t = temperature == nullptr ? 1.0f : __ldg(temperature + row);
    return t > 0.0f ? fminf(fmaxf(t, 1e-30f), 1e30f) : 1.0f;
}

// A row, counted from the 16-byte boundary at or below its start: values [skip, end) are the row's.
template <bool BF16>
struct Row {
    static constexpr int E = BF16 ? 8 : 4;
    const unsigned char* base;
    int skip;
    long long end;
    __device__ __forceinline__ Row(const void* logits, long long at, int vocab) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(logits) + at * (BF16 ? 2 : 4);
        base = reinterpret_cast<const unsigned char*>(a & ~(uintptr_t)15);
        skip = (int)((a & 15) / (BF16 ? 2 : 4));
        end = (long long)skip + vocab;
    }
    // The 16 bytes of values [E i, E i + E); what is not the row's -inf.
    __device__ __forceinline__ uint4 load(long long i) const {
        const long long at = i * E;
        if (at >= skip && at + E <= end) return *reinterpret_cast<const uint4*>(base + i * 16);
        uint4 r;
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = BF16 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (at + j < skip || at + j >= end) continue;
            if constexpr (BF16) {
                const uint32_t v = reinterpret_cast<const uint16_t*>(base)[at + j];
                w[j / 2] = j % 2 ? (w[j / 2] & 0xffffu) | v << 16 : (w[j / 2] & 0xffff0000u) | v;
            } else {
                w[j] = reinterpret_cast<const uint32_t*>(base)[at + j];
            }
        }
        return r;
    }
};
template <bool BF16>
__device__ __forceinline__ float value(const uint4& r, int j) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    if constexpr (BF16) return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    else return __uint_as_float(w[j]);
}
template <bool BF16>
__device__ __forceinline__ float largest(const uint4& r) {  // (of numbers; NaN where there is none)
    if constexpr (BF16) {
        const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&r);
        const __nv_bfloat162 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
        return fmaxf(__low2float(m), __high2float(m));
    } else {
        const float* w = reinterpret_cast<const float*>(&r);
        return fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
    }
}

// t = (x - m) log2(e) / T: the difference first, so that the largest logit's t is 0 itself, and no size of x or T does harm.
// Stands for -inf where maximum and temperature are ordinary (`plain`): finite times finite, so that no 0 meets an infinity.  (About -1e30, a bf16 value: for pairs of them kFloorPair.)
constexpr float kFloor = -0x1.92p99f;
constexpr uint32_t kFloorPair = 0xf149f149u;
__device__ __forceinline__ bool plain(float m, float c) { return c >= 1e-6f && c <= 1e6f && (m == -INFINITY || fabsf(m) <= 1e29f); }

// Sums of e^t and e^t t against the maximum m, in powers of two.
struct Sums {
    float m = -INFINITY, s = 0.0f, w = 0.0f;
    __device__ __forceinline__ void join(float om, float os, float ow, float c) {
        if (om > m) {
            const float keep_s = s, keep_w = w, keep_m = m;
            m = om, s = os, w = ow;
            om = keep_m, os = keep_s, ow = keep_w;
        }
        if (om == -INFINITY) {  // (a part of NaN and masked values has a sum without a maximum)
            s += os, w += ow;
            return;
        }
        const float d = (om - m) * c, f = ex2_ftz(d), dd = fmaxf(d, -1000.0f);
        s = fmaf(os, f, s), w = fmaf(f, fmaf(os, dd, ow), w);
    }
};
// A lane's, of values in pairs.
struct LaneSums {
    float m = -INFINITY;
    float2 s = {0.0f, 0.0f}, w = {0.0f, 0.0f};
    __device__ __forceinline__ void raise(float to, float c) {  // to > m
        if (m != -INFINITY) {
            const float d = (m - to) * c, f = ex2_ftz(d), dd = fmaxf(d, -1000.0f);
            w = mul2(make_float2(f, f), fma2(s, make_float2(dd, dd), w)), s = mul2(make_float2(f, f), s);
        }
        m = to;
    }
    template <bool BF16>
    __device__ __forceinline__ void add_plain(uint4 r, float c) {
        uint32_t* u = reinterpret_cast<uint32_t*>(&r);
        const float from = m == -INFINITY ? 0.0f : -m;
        const float2 c2 = make_float2(c, c), minus = make_float2(from, from);
#pragma unroll
        for (int j = 0; j < Row<BF16>::E / 2; ++j) {
            float2 x;
            if constexpr (BF16) {
                asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(u[j]) : "r"(kFloorPair));
                x = make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u));
            } else {
                x = make_float2(max_nan(__uint_as_float(u[2 * j]), kFloor), max_nan(__uint_as_float(u[2 * j + 1]), kFloor));
            }
            const float2 t = mul2(add2(x, minus), c2), e = make_float2(ex2_ftz(t.x), ex2_ftz(t.y));
            s = add2(s, e), w = fma2(e, t, w);
        }
    }
    template <bool BF16>
    __device__ __forceinline__ void add(const uint4& r, float c) {
        const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < Row<BF16>::E; ++j) {
            // (-inf: e^t is 0, and stays 0 times t; a NaN stays one)
            const float t = max_nan((value<BF16>(r, j) - from) * c, -1000.0f), e = ex2_ftz(t);
            s.x += e, w.x = fmaf(e, t, w.x);
        }
    }
};

// The sums of the first `lanes` (a power of two) lanes together, in pairs (a fixed order), in every lane.
__device__ __forceinline__ void join_lanes(Sums& x, int lanes, float c) {
    for (int d = 1; d < lanes; d *= 2) {
        const float m = __shfl_xor_sync(0xffffffffu, x.m, d), s = __shfl_xor_sync(0xffffffffu, x.s, d), w = __shfl_xor_sync(0xffffffffu, x.w, d);
        x.join(m, s, w, c);
    }
    x.m = __shfl_sync(0xffffffffu, x.m, 0), x.s = __shfl_sync(0xffffffffu, x.s, 0), x.w = __shfl_sync(0xffffffffu, x.w, 0);
}

// Among n entries, those that fewer than k come before, to their places.  By the whole block, several threads an entry, a part of the others each.
template <int WARPS>
__device__ __forceinline__ void rank(Shared<WARPS>& sh, int n, int k) {
    constexpr int kThreads = 32 * WARPS;
    int parts = 1;
    while (parts < 32 && 2 * parts * n <= kThreads) parts *= 2;
    for (int i = threadIdx.x; i < n; i += kThreads) sh.ahead[i] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < n * parts; e += kThreads) {
        const int i = e / parts, part = e % parts;
        const Entry mine = sh.candidate[i];
        int ahead = 0;
#pragma unroll 4
        for (int j = part; j < n; j += parts) ahead += before(sh.candidate[j], mine);
        if (parts == 1) sh.ahead[i] = ahead;
        else if (ahead != 0) atomicAdd(&sh.ahead[i], ahead);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (sh.ahead[i] < k) sh.best[sh.ahead[i]] = sh.candidate[i];
}

// Few rows: blocks of sixteen warps, a round of loads each.  Many: of eight, of which an SM holds three, so that no row waits for another's last step.  (Sixteen and eight, us: a row of 131,072 f32
// with twenty alternatives 12.2 and 16.0, 30 of them 15.3 and 19.8; of bf16 with five 30 rows 10.2 and 11.8, 40 rows 18.4 and 11.9, 336 rows 34.8 and 30.7.)
template <bool BF16, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 3 : 2) logprob_kernel(const LogprobParams p) {
    constexpr int E = Row<BF16>::E, kThreads = 32 * WARPS, kWarps = WARPS, kAtOnce = WARPS == 8 ? 8 : 4;  // pieces of a warp in flight
    __shared__ Shared<WARPS> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x % p.blocks;
    const long long row = blockIdx.x / p.blocks;
    grid_ready();
    const Row<BF16> x(p.logits, row * p.ld, p.vocab);
    const float heat = heat_of(p.temperature, row), c = kLog2e / heat;
    // The row's pieces (32 lanes of 16 bytes), in as many runs as blocks share it.
    const int pieces = (int)((x.end + 32 * E - 1) / (32 * E));
    const int first = (int)((long long)pieces * part / p.blocks), last = (int)((long long)pieces * (part + 1) / p.blocks);
    if (tid == 0) sh.candidates = 0;
    if (p.top > 0 && tid < kMostTop) sh.best[tid] = Entry{-INFINITY, -1};

    LaneSums mine;  // m: the warp's
    float most = -INFINITY;
    for (int i = first + warp; i < last; i += kWarps * kAtOnce) {
        uint4 r[kAtOnce];
        float top[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const long long at = i + u * kWarps < last ? (long long)(i + u * kWarps) * 32 + lane : x.end;  // (past the end: all -inf)
            r[u] = x.load(at);
        }
        float up = -INFINITY;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const float lane_top = largest<BF16>(r[u]);
            most = fmaxf(most, lane_top);
            top[u] = warp_max(lane_top);
            up = fmaxf(up, top[u]);
        }
        if (p.top > 0 && lane == 0)
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (i + u * kWarps < last) sh.piece[i + u * kWarps - first] = top[u];
        if (up > mine.m) mine.raise(up, c);
        if (plain(mine.m, c)) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) mine.add_plain<BF16>(r[u], c);
        } else {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) mine.add<BF16>(r[u], c);
        }
    }
    const float sum = warp_sum(mine.s.x + mine.s.y), sum_t = warp_sum(mine.w.x + mine.w.y);
    if (lane == 0) sh.wmax[warp] = mine.m, sh.wsum[warp] = sum, sh.wsum_t[warp] = sum_t;
    sh.group[tid] = most;
    __syncthreads();
    if (warp == kWarps - 1) {
        Sums all;
        if (lane < kWarps) all.m = sh.wmax[lane], all.s = sh.wsum[lane], all.w = sh.wsum_t[lane];
        join_lanes(all, kWarps, c);
        if (lane == 0) sh.max = all.m, sh.sum = all.s, sh.sum_t = all.w;
    }
    if (p.top > 0) {
        const int k = p.top;
        float g = -INFINITY;
        if (tid < kGroups) {
#pragma unroll
            for (int j = 0; j < kThreads / kGroups; ++j) g = fmaxf(g, sh.group[tid + j * kGroups]);
        }
        __syncthreads();
        if (tid < kGroups) sh.group[tid] = g;
        __syncthreads();
        if (tid < kGroups) {
            // (g is the k-th largest where fewer than k are larger and at least k no smaller)
            int larger = 0, no_smaller = 0;
#pragma unroll 8
            for (int j = 0; j < kGroups; j += 4) {
                const float4 o = *reinterpret_cast<const float4*>(sh.group + j);
                larger += (o.x > g) + (o.y > g) + (o.z > g) + (o.w > g);
                no_smaller += (o.x >= g) + (o.y >= g) + (o.z >= g) + (o.w >= g);
            }
            if (larger < k && no_smaller >= k) sh.bound = g;
        }
        __syncthreads();
        const float bound = sh.bound;
        // A warp looks at pieces warp, warp + kWarps, ..., as it read them: a lane a piece, then the lanes a piece together, two of them at a time.
        for (int i = warp; i < last - first; i += 32 * kWarps) {
            const int at = i + lane * kWarps;
            const float has = at < last - first ? sh.piece[at] : -INFINITY;
            uint32_t hits = __ballot_sync(0xffffffffu, has >= bound && has > -INFINITY);
            while (hits != 0) {
                long long piece[2];
                uint4 r[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    piece[u] = hits != 0 ? (long long)(first + i + (__ffs(hits) - 1) * kWarps) * 32 + lane : x.end;
                    hits &= hits - 1;
                    r[u] = x.load(piece[u]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (!(largest<BF16>(r[u]) >= bound)) continue;
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const float v = value<BF16>(r[u], j);
                        if (!(v >= bound && v > -INFINITY)) continue;
                        const int to = atomicAdd(&sh.candidates, 1);
                        if (to < kCandidates) sh.candidate[to] = Entry{v, (int)(piece[u] * E + j - x.skip)};
                    }
                }
            }
        }
        __syncthreads();
        if (sh.candidates <= kCandidates) {
            rank(sh, sh.candidates, k);
        } else {
            // The next entry of the order, k times over the part.
            Entry bar{INFINITY, -1};
            for (int n = 0; n < k; ++n) {
                Entry e{-INFINITY, 0x7fffffff};
                for (int i = first + warp; i < last; i += kWarps) {
                    const long long at = (long long)i * 32 + lane;
                    const uint4 r = x.load(at);
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const Entry o{value<BF16>(r, j), (int)(at * E + j - x.skip)};
                        if (o.v > -INFINITY && before(bar, o) && before(o, e)) e = o;
                    }
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    const Entry o{__shfl_xor_sync(0xffffffffu, e.v, d), __shfl_xor_sync(0xffffffffu, e.id, d)};
                    if (before(o, e)) e = o;
                }
                if (lane == 0) sh.wbest[warp] = e;
                __syncthreads();
                e = sh.wbest[0];
                for (int w = 1; w < kWarps; ++w)
                    if (before(sh.wbest[w], e)) e = sh.wbest[w];
                bar = e;
                if (tid == 0 && e.v > -INFINITY) sh.best[n] = e;
                __syncthreads();
            }
        }
    }
    if (p.blocks > 1) cluster_sync();
    else __syncthreads();
    if (part == 0) {
        if (p.blocks > 1 && p.top > 0) {  // the blocks' best together
            for (int i = tid; i < p.blocks * p.top; i += kThreads) {
                const uint32_t at = cluster_place(&sh.best[i % p.top], i / p.top);
                sh.candidate[i] = Entry{cluster_load(at), __float_as_int(cluster_load(at + 4))};
            }
            __syncthreads();
            if (tid < kMostTop) sh.best[tid] = Entry{-INFINITY, -1};
            __syncthreads();
            rank(sh, p.blocks * p.top, p.top);  // (empty places come behind; equal ones among them keep theirs)
            __syncthreads();
        }
        if (warp == 0) {
            const float inv = 1.0f / heat;
            Sums all;
            if (p.blocks == 1) {
                all.m = sh.max, all.s = sh.sum, all.w = sh.sum_t;
            } else {
                if (lane < p.blocks)
                    all.m = cluster_load(cluster_place(&sh.max, lane)), all.s = cluster_load(cluster_place(&sh.sum, lane)), all.w = cluster_load(cluster_place(&sh.sum_t, lane));
                join_lanes(all, p.blocks, c);
            }
            const bool none = all.m == -INFINITY && all.s == 0.0f;  // a row whose mask leaves nothing
            const float l2 = log2f(all.s), log_s = kLn2 * l2;
            if (lane == 0) {
                const int token = p.tokens == nullptr ? -1 : __ldg(p.tokens + row);
                if (p.logprob != nullptr) {
                    float lp = 0.0f;
                    if (token >= 0 && token < p.vocab) {
                        float v;
                        if constexpr (BF16) v = bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(p.logits) + row * p.ld + token));
                        else v = __ldg(static_cast<const float*>(p.logits) + row * p.ld + token);
                        lp = none ? -INFINITY : fmaf(v - all.m, inv, -log_s);  // (not in powers of two: a mask's lowest value would overflow)
                    }
                    p.logprob[row] = lp;
                }
                if (p.entropy != nullptr) p.entropy[row] = none ? 0.0f : kLn2 * (l2 - all.w / all.s);
                if (p.lse != nullptr) p.lse[row] = none ? -INFINITY : fmaf(kLn2, l2, all.m / heat);
            }
            if (lane < p.top) {
                const Entry e = sh.best[lane];
                p.top_ids[row * p.top + lane] = e.id;
                p.top_values[row * p.top + lane] = e.id < 0 ? -INFINITY : fmaf(e.v - all.m, inv, -log_s);
            }
        }
    }
    if (p.blocks > 1) cluster_sync();  // nobody leaves while its results may be read
}

// Backwards, log p = x / T - lse, whose parts are rounded at their size: p is off by at most 2 |lse| u of itself (u = 2^-24), 128 u for f32 logits up to kOrdinary, less than what a row's sum may be
// off by, and 512 u, a hundredth of the gradient's own rounding, for bf16.  Beyond it (low temperatures, logits far from 0, rows of nothing but a mask's lowest value) the row's maximum and sum are
// formed again and log p is (x - max) / T - log S as forwards: no size of x or T does harm, and lse may have overflowed.  Such a row is read twice, by its first block alone; the others leave.  Nothing is
// asked of other blocks, so the gradient may take the logits' place, each thread's pieces its own (plain loads).
constexpr int kBackThreads = 256, kBackAtOnce = 4, kBackWarps = kBackThreads / 32;
template <bool BF16>
constexpr float kOrdinary = BF16 ? 256.0f : 64.0f;

// A row's gradient by pieces of 16 bytes, as the gradient's row lies on them.
template <bool BF16>
struct Gradient {
    static constexpr int E = Row<BF16>::E;
    const Row<BF16> d, x;
    const LogprobParams& p;
    const long long row;
    float minus = 0.0f, from;  // log p = (x + minus) / T + from
    int token;                 // -1: none
    float inv, l, n, entropy;  // 1 / T, and the gradients / T
    __device__ __forceinline__ Gradient(const LogprobParams& q, long long r, float lse) : d(q.dlogits, r * q.dld, q.vocab), x(q.logits, r * q.ld, q.vocab), p(q), row(r), from(-lse) {
        token = __ldg(p.tokens + row);
        if (token < 0 || token >= p.vocab) token = -1;
        inv = 1.0f / heat_of(p.temperature, row);
        l = token >= 0 && p.dlogprob != nullptr ? __ldg(p.dlogprob + row) * inv : 0.0f;
        n = p.dentropy != nullptr ? __ldg(p.dentropy + row) * inv : 0.0f;
        entropy = n != 0.0f ? __ldg(p.entropy + row) : 0.0f;
    }
    __device__ __forceinline__ long long pieces() const { return (d.end + E - 1) / E; }
    __device__ __forceinline__ uint4 load(long long i) const {  // what is not the row's -inf
        if (d.skip == x.skip) return x.load(i);
        uint4 r;  // (rows that lie differently on their 16 bytes)
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = BF16 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const long long at = i * E + j - d.skip;
            if (at < 0 || at >= p.vocab) continue;
            if constexpr (BF16) {
                const uint32_t v = static_cast<const uint16_t*>(p.logits)[row * p.ld + at];
                w[j / 2] = j % 2 ? (w[j / 2] & 0xffffu) | v << 16 : (w[j / 2] & 0xffff0000u) | v;
            } else {
                w[j] = static_cast<const uint32_t*>(p.logits)[row * p.ld + at];
            }
        }
        return r;
    }
    // The pieces from `first` on that r holds, kBackThreads apart, up to `end` values.  SHIFT: `minus` is not 0.
    template <bool SHIFT, int N>
    __device__ __forceinline__ void store(const uint4 (&r)[N], long long first, long long end) const {
        // -p (n (log p + H) + l), in pairs; the token's value in its piece only.
        const float minus_l = -fmaf(n, entropy, l);
        const float2 inv2 = make_float2(inv, inv), from2 = make_float2(from, from), n2 = make_float2(-n, -n), l2 = make_float2(minus_l, minus_l), log2e2 = make_float2(kLog2e, kLog2e);
        const long long token_piece = token >= 0 ? ((long long)token + d.skip) / E : -1;
        const int token_at = token >= 0 ? (token + d.skip) % E : 0;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const long long i = first + u * kBackThreads;
            if (i * E >= end) continue;
            float y[E];
#pragma unroll
            for (int j = 0; j < E; j += 2) {
                float2 v = make_float2(value<BF16>(r[u], j), value<BF16>(r[u], j + 1));
                if constexpr (SHIFT) v = add2(v, make_float2(minus, minus));
                float2 lp = fma2(v, inv2, from2);
                lp = make_float2(max_nan(lp.x, -1000.0f), max_nan(lp.y, -1000.0f));
                const float2 t = mul2(lp, log2e2);
                v = mul2(make_float2(ex2_ftz(t.x), ex2_ftz(t.y)), fma2(n2, lp, l2));
                y[j] = v.x, y[j + 1] = v.y;
            }
            if (i == token_piece) {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (j == token_at) y[j] += l;
            }
            unsigned char* to = const_cast<unsigned char*>(d.base) + i * 16;
            if (i * E >= d.skip && i * E + E <= d.end) {
                uint4 o;
                uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (BF16) {
                        const __nv_bfloat162 two = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
                        w[j] = *reinterpret_cast<const uint32_t*>(&two);
                    } else {
                        w[j] = __float_as_uint(y[j]);
                    }
                }
                *reinterpret_cast<uint4*>(to) = o;
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (i * E + j < d.skip || i * E + j >= d.end) continue;
                    if constexpr (BF16) reinterpret_cast<uint16_t*>(to)[j] = f32_to_bf16_bits(y[j]);
                    else reinterpret_cast<float*>(to)[j] = y[j];
                }
            }
        }
    }
};

// A whole row by one block, N pieces of a thread in flight: its maximum and sum, then its gradient.
template <bool BF16, int N>
__device__ __forceinline__ void whole_row(const LogprobParams& p, long long row) {
    __shared__ float wmax[kBackWarps], wsum[kBackWarps];
    Gradient<BF16> g(p, row, 0.0f);
    const long long pieces = g.pieces();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float c = kLog2e / heat_of(p.temperature, row);
    uint4 r[N];
    LaneSums mine;  // m: the warp's
    for (long long i = warp * 32; i < pieces; i += kBackThreads * N) {
        float up = -INFINITY;
#pragma unroll
        for (int u = 0; u < N; ++u) r[u] = g.load(i + u * kBackThreads + lane);  // (past the end: all -inf)
#pragma unroll
        for (int u = 0; u < N; ++u) up = fmaxf(up, largest<BF16>(r[u]));
        up = warp_max(up);
        if (up > mine.m) mine.raise(up, c);
#pragma unroll
        for (int u = 0; u < N; ++u) mine.add<BF16>(r[u], c);
    }
    const float s = warp_sum(mine.s.x + mine.s.y);
    if (lane == 0) wmax[warp] = mine.m, wsum[warp] = s;
    __syncthreads();
    Sums all;
    if (lane < kBackWarps) all.m = wmax[lane], all.s = wsum[lane];
    join_lanes(all, kBackWarps, c);
    if (all.m == -INFINITY && all.s == 0.0f) g.l = g.n = g.entropy = 0.0f;  // a row that masks everything: no gradient
    else g.minus = -all.m, g.from = -kLn2 * log2f(all.s);
    for (long long i = threadIdx.x; i < pieces; i += kBackThreads * N) {
#pragma unroll
        for (int u = 0; u < N; ++u) r[u] = g.load(i + u * kBackThreads);
        g.template store<true>(r, i, g.d.end);
    }
}

template <bool BF16>
__device__ __noinline__ void whole_row_apart(const LogprobParams& p, long long row) { whole_row<BF16, 2>(p, row); }

// A block takes kBackThreads x kBackAtOnce pieces of the gradient's row.  ALL: rows that are read twice too, by a function, whose registers cost blocks beside one another; large calls leave these
// rows to the kernel behind this one.  (us, bf16 and f32 logits: one row of 131,072 2.4 and 2.4; 2,048 and 1,024 of them 191 and 178 so, 178 and 167 and a launch the other way.)
template <bool BF16, bool ALL>
__global__ void __launch_bounds__(kBackThreads, ALL ? (BF16 ? 5 : 6) : 0) logprob_backward_kernel(const __grid_constant__ LogprobParams p) {
    grid_ready();
    const long long row = blockIdx.x / p.blocks, first = (long long)(blockIdx.x % p.blocks) * kBackThreads * kBackAtOnce + threadIdx.x;
    const float lse = __ldg(p.lse + row);
    const Gradient<BF16> g(p, row, lse);
    uint4 r[kBackAtOnce];  // (asked for before anything is known of the row: a block lives for little more than a trip to memory)
#pragma unroll
    for (int u = 0; u < kBackAtOnce; ++u)
        if ((first + u * kBackThreads) * Row<BF16>::E < g.d.end) r[u] = g.load(first + u * kBackThreads);
    const bool ordinary = fabsf(lse) <= kOrdinary<BF16>;
    g.template store<false>(r, first, ordinary ? g.d.end : 0);
    if (ALL && !ordinary && blockIdx.x % p.blocks == 0) whole_row_apart<BF16>(p, row);
}
// A row a block.
template <bool BF16>
__global__ void __launch_bounds__(kBackThreads) logprob_backward_rest_kernel(const __grid_constant__ LogprobParams p) {
    grid_ready();
    if (!(fabsf(__ldg(p.lse + blockIdx.x)) <= kOrdinary<BF16>)) whole_row<BF16, kBackAtOnce>(p, blockIdx.x);
}

// Blocks that share a row: enough that a small call fills the GPU, while each still has a piece a warp.  (Up to two blocks an SM; 131,072 bf16 logits with five alternatives, us: 200 rows 21.5 with two
// blocks a row, 28.5 with one; 336 rows 30.6 with one, 35.2 with two; 250 rows, 32.5 with two and 30.1 with one, are the rule's loss.)
int row_blocks(long long rows, int vocab, bool bf16, int warps) {
    const int pieces = vocab / (bf16 ? 256 : 128) + 2;
    int n = 1;
    while (n < kMostBlocks && (pieces > n * kPieces || (rows * n < 2 * sm_count() && pieces >= 2 * n * warps))) n *= 2;
    return n;
}

bool logits_ok(const void* p, int32_t kind, int64_t ld, int32_t vocab) {
    if (kind != GLM53F_KDA_LOGITS_F32 && kind != GLM53F_KDA_LOGITS_BF16) return false;
    return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (kind == GLM53F_KDA_LOGITS_BF16 ? 1 : 3)) == 0 && ld >= vocab;
}
bool words(std::initializer_list<const void*> all) {
    for (const void* p : all)
        if (reinterpret_cast<uintptr_t>(p) & 3) return false;
    return true;
}

}  // namespace
}  // namespace kda

extern "C" int glm53f_kda_logprobs(int32_t rows, int32_t vocab, const void* logits, int32_t kind, int64_t ld, const int32_t* tokens, const float* temperature,
                                   float* logprob, float* entropy, float* lse, int32_t top, int32_t* top_ids, float* top_values, glm53f_stream_t stream) {
    using namespace kda;
    if (rows < 0 || vocab < 1 || vocab > kMostVocab || top < 0 || top > kMostTop) return kInvalid;
    if (rows == 0) return 0;
    if (!logits_ok(logits, kind, ld, vocab) || !words({tokens, temperature, logprob, entropy, lse, top_ids, top_values})) return kInvalid;
    if ((logprob != nullptr) != (tokens != nullptr) || (top > 0) != (top_ids != nullptr) || (top > 0) != (top_values != nullptr)) return kInvalid;
    if (logprob == nullptr && entropy == nullptr && lse == nullptr && top == 0) return kInvalid;
    const bool bf16 = kind == GLM53F_KDA_LOGITS_BF16;
    LogprobParams p{};
    p.logits = logits, p.ld = ld, p.vocab = vocab, p.top = top;
    const int warps = (long long)rows * kMostBlocks <= 2 * sm_count() ? 16 : 8;
    p.blocks = row_blocks(rows, vocab, bf16, warps);
    p.tokens = tokens, p.temperature = temperature, p.logprob = logprob, p.entropy = entropy, p.lse = lse, p.top_ids = top_ids, p.top_values = top_values;
    if ((long long)rows * p.blocks > 0x7fffffff) return kInvalid;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * p.blocks));
    cfg.blockDim = dim3(32 * warps);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    unsigned na = early_attribute(attr[0]);
    if (p.blocks > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)p.blocks;
        attr[na].val.clusterDim.y = 1;
        attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    if (warps == 16) return (int)(bf16 ? cudaLaunchKernelEx(&cfg, logprob_kernel<true, 16>, p) : cudaLaunchKernelEx(&cfg, logprob_kernel<false, 16>, p));
    return (int)(bf16 ? cudaLaunchKernelEx(&cfg, logprob_kernel<true, 8>, p) : cudaLaunchKernelEx(&cfg, logprob_kernel<false, 8>, p));
}

extern "C" int glm53f_kda_logprobs_backward(int32_t rows, int32_t vocab, const void* logits, int32_t kind, int64_t ld, const int32_t* tokens,
                                            const float* temperature, const float* lse, const float* entropy, const float* dlogprob, const float* dentropy,
                                            void* dlogits, int64_t dld, glm53f_stream_t stream) {
    using namespace kda;
    if (rows < 0 || vocab < 1 || vocab > kMostVocab) return kInvalid;
    if (rows == 0) return 0;
    if (!logits_ok(logits, kind, ld, vocab) || !logits_ok(dlogits, kind, dld, vocab) || !words({tokens, temperature, lse, entropy, dlogprob, dentropy})) return kInvalid;
    if (lse == nullptr || tokens == nullptr || (dlogprob == nullptr && dentropy == nullptr) || (dentropy != nullptr && entropy == nullptr)) return kInvalid;
    const bool bf16 = kind == GLM53F_KDA_LOGITS_BF16;
    const int per = kBackThreads * kBackAtOnce * (bf16 ? 8 : 4);
    LogprobParams p{};
    p.logits = logits, p.ld = ld, p.vocab = vocab;
    // (values before a row's start on its 16 bytes: at most these)
    const int size = bf16 ? 2 : 4, most = 16 / size - 1, skip = dld % (16 / size) == 0 ? (int)((reinterpret_cast<uintptr_t>(dlogits) & 15) / size) : most;
    p.blocks = (int)(((long long)vocab + skip + per - 1) / per);
    p.tokens = tokens, p.temperature = temperature, p.lse = const_cast<float*>(lse), p.entropy = const_cast<float*>(entropy);
    p.dlogprob = dlogprob, p.dentropy = dentropy, p.dlogits = dlogits, p.dld = dld;
    if ((long long)rows * p.blocks > 0x7fffffff) return kInvalid;
    const cudaStream_t on = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)(rows * p.blocks));
    if ((long long)rows * vocab * size < 128ll << 20)
        return bf16 ? launch_early(logprob_backward_kernel<true, true>, grid, kBackThreads, 0, on, p) : launch_early(logprob_backward_kernel<false, true>, grid, kBackThreads, 0, on, p);
    const int rc = bf16 ? launch_early(logprob_backward_kernel<true, false>, grid, kBackThreads, 0, on, p) : launch_early(logprob_backward_kernel<false, false>, grid, kBackThreads, 0, on, p);
    if (rc != 0) return rc;
    return bf16 ? launch_early(logprob_backward_rest_kernel<true>, dim3((unsigned)rows), kBackThreads, 0, on, p) : launch_early(logprob_backward_rest_kernel<false>, dim3((unsigned)rows), kBackThreads, 0, on, p);
}
