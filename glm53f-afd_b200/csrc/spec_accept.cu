// Verification of drafted tokens: how many rows of each window to keep, and the token behind them.
//
// Per request, with p_i the target's distribution behind row i and q_i the one that token i was drawn from, token i + 1 is
// kept while u_{i+1} q_{i+1}(token) < p_i(token); the next token is drawn by a running sum from max(p - q, 0) of the first refused
// token's row, or from p behind a whole window.
//
// Bound by HBM for many requests' windows, by the instructions of the draws next to it, and by latency for one.  A request is a thread-block cluster: each block
// takes a slice of the vocabulary, all rows of the window; the slices' maxima and sums meet in distributed shared memory, every block makes the same
// decision, and all of them draw together: a warp sums a run of consecutive weights, the one whose run holds the drawn point looks for it.  One launch, no
// scratch in global memory, no atomics: the same result every time.
//
// Rows are read between their 16-byte boundaries, wherever those lie, through a ring of asynchronous copies for each warp (48 greedy windows of eight rows of
// 131,072 bf16 logits, 101 MB: 27 us, 3.7 TB/s; with eight loads a lane in registers, which the compiler spills, 47, with two times four 39).  The row that is drawn
// from comes from L2 the second time; a draw of all 48 adds 16 us, another 16 with a drafter's distributions to read and a second pass.
//
// A draw decides between neighbours of a sum over the whole vocabulary, so weights and sums are formed in 64 bits there: in 32, the sums'
// rounding moves one draw in a few hundred to the next token.  The maxima and sums that judge a token are 32-bit ones (a relative 1e-7
// of a probability against u).

#include <type_traits>

#include "common.cuh"
#include "device_counts.h"
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

constexpr int kCopies = 16;  // of the table of powers
constexpr int kSlots = 4;

struct AccShared {
    double power[32][kCopies];  // 2^(j / 32)
    // What this block's slice gives, read by the other blocks of the cluster.
    float max[kAccRows], sum[kAccRows];
    int best[kAccRows];
    double part;      // the slice's weights
    // Within the block.
    float wmax[kAccRows][kAccMostWarps + 1], wsum[kAccRows][kAccMostWarps + 1];  // (the last place: the row's two ends)
    int wbest[kAccRows][kAccMostWarps + 1];
    double wpart[kAccMostWarps];
    double slot[kAccMostWarps][kSlots];  // a warp's weights, its places in so many parts
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

// Copies into a lane's own places of its warp's ring.
__device__ __forceinline__ void copy_16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>
__device__ __forceinline__ void copies_here() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }  // all but the last LATER groups

constexpr float kNoLogit = -INFINITY;
template <int KIND>
__device__ __forceinline__ float target_at(const void* row, long long i) {
    if constexpr (KIND == GLM53F_KDA_LOGITS_BF16) return bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(row) + i));
    else return __ldg(static_cast<const float*>(row) + i);
}
// Eight consecutive entries from i on as they lie in memory (vector loads; or, where a row's end rules those out, one at a time, those before the row and behind it as
// `fill`), and as floats.  Apart, so that several loads are in flight before the first is looked at.
template <int KIND>
struct Eight {
    static constexpr int kWords = KIND == GLM53F_KDA_LOGITS_BF16 ? 4 : 8;
    uint32_t w[kWords];
    // How many entries lie between a 16-byte boundary and the row: runs of eight begin that much before a multiple of eight.
    static __device__ __forceinline__ int shift(const void* row) { return (int)(reinterpret_cast<uintptr_t>(row) & 15) / (kWords / 2); }
    __device__ __forceinline__ void load_whole(const void* row, int i) {
#pragma unroll
        for (int j = 0; j < kWords; j += 4) {
            const uint4 r = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(row) + (long long)i * (kWords / 2)) + j / 4);
            w[j] = r.x, w[j + 1] = r.y, w[j + 2] = r.z, w[j + 3] = r.w;
        }
    }
    __device__ __forceinline__ void load_some(const void* row, int i, int end, float fill) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = __float_as_uint(i + j >= 0 && i + j < end ? target_at<KIND>(row, i + j) : fill);
            if constexpr (kWords == 8) w[j] = u;
            else w[j >> 1] = j & 1 ? w[j >> 1] | (u & 0xffff0000u) : u >> 16;
        }
    }
    __device__ __forceinline__ void load(const void* row, int i, int end, bool aligned, float fill) {
        if (aligned && i >= 0 && i <= end - 8) load_whole(row, i);
        else load_some(row, i, end, fill);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (kWords == 8) x[j] = __uint_as_float(w[j]);
            else x[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
        }
    }
};

// A row's weights in 64 bits: e^x of x = (l - max) / t <= 0.  With z = 32 x / ln 2 = 32 e + j + f, |f| <= 1/2: e^x = 2^e 2^(j/32) e^(f ln 2 / 32), of which
// Taylor's series to the fourth power leaves 1.3e-12: a draw among 131,072 moves by it once in ten million.  (With the general exponential, and every
// special case looked at for every entry, a draw's pass took four times as many instructions.)  NaN and what is below e^-690 is 0, by z itself: where
// f32 has few steps between max and max - 690 t, a logit at the rounded bound lies far below it, and the exponent's sum wraps there.  Rows whose
// largest is infinite: see weights() in the kernel.  The pass waits for instructions, of which this is 20 an entry; the table lies in sixteen copies, two banks each.
constexpr double kTurns = 46.166241308446828384;  // 32 / ln 2
struct RowScale {
    double max, turns;  // turns: 32 / (t ln 2)
};
__device__ __forceinline__ RowScale row_scale_of(float max, float t) { return {(double)max, kTurns / (double)t}; }
__device__ __forceinline__ double logit_weight(float l, const RowScale& a, const double* power) {  // power: the lane's copy
    constexpr double c = 1.0 / kTurns;
    const double magic = 6755399441055744.0;  // 1.5 2^52: adding it rounds to an integer, which the low word then holds
    const double z = ((double)l - a.max) * a.turns, shifted = z + magic;
    const int n = __double2loint(shifted);
    const double f = z - (shifted - magic);
    double y = fma(f, c * c * c * c / 24, c * c * c / 6);
    y = fma(f, y, c * c / 2);
    y = fma(f, y, c);
    y = fma(f, y, 1.0);
    const double base = power[(n & 31) * kCopies];
    y *= __hiloint2double(((n & ~31) << 15) + __double2hiint(base), __double2loint(base));
    return z >= -690.0 * kTurns ? y : 0.0;
}
__device__ __forceinline__ float finite_weight(float p) { return p > 0.0f && p < INFINITY ? p : 0.0f; }

// A row's statistics: its largest logit m, the sum of 2^((l - m) scale) over it, the lowest index of the largest (greedy).  A sum at a maximum of -inf is 0.
struct Stats {
    float m = kNoLogit, s = 0.0f;
    int best = -1;
};
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return fma2(a, make_float2(1.0f, 1.0f), b); }
// A chunk: four pieces of 16 bytes a lane, a piece's lanes next to one another; the lane's first entry is entry `at` of the row.
constexpr int kPieces = 4, kPiece = 512, kChunk = 32 * kPieces;  // (a chunk in pieces of one lane)
template <int KIND>
constexpr int kEach = KIND == GLM53F_KDA_LOGITS_BF16 ? 8 : 4;  // entries of a piece
template <int KIND>
__device__ __forceinline__ void entries(const uint4& piece, float (&x)[kEach<KIND>]) {
    const uint32_t w[4] = {piece.x, piece.y, piece.z, piece.w};
#pragma unroll
    for (int j = 0; j < kEach<KIND>; ++j) {
        if constexpr (kEach<KIND> == 4) x[j] = __uint_as_float(w[j]);
        else x[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    }
}
template <int KIND>
__device__ __forceinline__ float largest(const uint4 (&in)[kPieces]) {  // (NaN only where all are)
    const uint32_t* w = reinterpret_cast<const uint32_t*>(in);
    if constexpr (kEach<KIND> == 4) {
        float m = __uint_as_float(w[0]);
#pragma unroll
        for (int j = 1; j < 4 * kPieces; ++j) m = fmaxf(m, __uint_as_float(w[j]));
        return m;
    } else {
        const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(w);
        __nv_bfloat162 m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int j = 4; j < 4 * kPieces; ++j) m[j & 3] = __hmax2(m[j & 3], x[j]);
        m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
        return fmaxf(__low2float(m[0]), __high2float(m[0]));
    }
}
template <bool GREEDY, int KIND>
__device__ __forceinline__ void take(Stats& a, const uint4 (&in)[kPieces], int at, float scale) {
    const float top = largest<KIND>(in);
    float x[kEach<KIND>];
    if constexpr (GREEDY) {
        if (top > a.m) {
            a.m = top;
#pragma unroll
            for (int i = kPieces - 1; i >= 0; --i) {
                entries<KIND>(in[i], x);
#pragma unroll
                for (int j = kEach<KIND> - 1; j >= 0; --j)
                    if (x[j] == top) a.best = at + i * 32 * kEach<KIND> + j;
            }
        }
    } else {
        if (top > a.m) {
            a.s *= a.m == kNoLogit ? 0.0f : ex2_approx((a.m - top) * scale);
            a.m = top;
        }
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 less = make_float2(-a.m, -a.m), times = make_float2(scale, scale);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            entries<KIND>(in[i], x);
#pragma unroll
            for (int j = 0; j < kEach<KIND>; j += 2) {
                const float2 t = mul2(add2(make_float2(x[j], x[j + 1]), less), times);
                sum[j / 2 & 1] = add2(sum[j / 2 & 1], make_float2(ex2_ftz(t.x), ex2_ftz(t.y)));
            }
        }
        float all = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        if (!(all < INFINITY)) {  // a NaN among them, or infinities: seldom, so one at a time
            all = 0.0f;
#pragma unroll 1
            for (int i = 0; i < kPieces; ++i) {
                entries<KIND>(i == 0 ? in[0] : i == 1 ? in[1] : i == 2 ? in[2] : in[3], x);
#pragma unroll
                for (int j = 0; j < kEach<KIND>; ++j) all += x[j] == a.m ? (a.m == kNoLogit ? 0.0f : 1.0f) : x[j] < a.m ? ex2_ftz((x[j] - a.m) * scale) : 0.0f;
            }
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

// Chunks of a warp on their way.  (Four: 48 drawn windows 47 us, of which L1, that much smaller then, serves the row's second reading; two: 43.  One: 44.)
constexpr int kDeep = 2;

// What a draw weighs: the row's distribution p, less the drafter's, or without the refused token.
enum : int { kWhole = 0, kLessDraft = 1, kWithout = 2 };

template <int KIND, int kAccWarps>
__global__ void __launch_bounds__(kAccWarps * 32, kAccWarps == 8 ? 3 : 1) accept_kernel(const __grid_constant__ AcceptParams p) {
    extern __shared__ __align__(16) unsigned char rings[];
    constexpr bool LOGITS = KIND != GLM53F_KDA_PROBABILITIES;
    constexpr int kSize = KIND == GLM53F_KDA_LOGITS_BF16 ? 2 : 4;
    __shared__ AccShared sh;
    if (threadIdx.x < 32) {
        const double power = exp2((double)threadIdx.x / 32);
        for (int i = 0; i < kCopies; ++i) sh.power[threadIdx.x][i] = power;
    }
    grid_ready();
    const int blocks = p.blocks, b = blockIdx.x >> (__ffs(blocks) - 1), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t block = cluster_block();
    unsigned char* ring = rings + warp * (kDeep * kPieces * kPiece) + lane * 16;
    const int first = p.cu[b], n = p.cu[b + 1] - first;
    if (n <= 0) {  // the same for the whole cluster
        if (block == 0 && tid == 0) p.keep[b] = 0, p.next[b] = -1;
        return;
    }
    const unsigned char* rows = static_cast<const unsigned char*>(p.target) + (long long)first * p.ld * kSize;
    auto row_at = [&](int i) { return static_cast<const void*>(rows + (long long)i * p.ld * kSize); };
    auto draft_at = [&](int i) { return p.draft + (long long)(first + i) * p.draft_ld; };
    // (Capped, a NaN too: an infinite one would make 0 times infinity of a logit of -inf.)
    const float temperature = LOGITS && p.temperature != nullptr ? (p.temperature[b] < 1e30f ? p.temperature[b] : 1e30f) : 1.0f;
    const bool greedy = LOGITS && !(temperature > 0.0f);
    const float scale = greedy ? 0.0f : kLog2e / temperature;
    const double* power = &sh.power[0][lane % kCopies];
    const int block_bits = __ffs(blocks) - 1;  // (a power of two)
    // This block's slice [run0, run1) of `runs` runs of eight.
    auto slice = [&](long long runs, long long& run0, long long& run1) { run0 = runs * block >> block_bits, run1 = runs * (block + 1) >> block_bits; };

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
                // The pieces of the rows between their 16-byte boundaries, in lines of 32, all rows' one after the other; a warp takes consecutive lines, of one row or a few.
                // (An equal share of every row instead has a warp join its lanes for each: windows of eight rows 4 us longer.)
                constexpr int kWarpBits = kAccWarps == 16 ? 4 : 3;
                static_assert(1 << kWarpBits == kAccWarps, "warps");
                const int lines = (int)((p.vocab / kEach<KIND> + 31) / 32);
                const long long mine = (long long)block * kAccWarps + warp, all_lines = (long long)rows_here * lines;
                const int line0 = (int)(all_lines * mine >> (block_bits + kWarpBits)), line1 = (int)(all_lines * (mine + 1) >> (block_bits + kWarpBits));
                // The part of row i from line `line` of all on: address (of the lane's first piece), pieces, first entry.  Rows may have fewer pieces than lines make: then none.
                auto part_of = [&](int i, int line, const unsigned char*& from, int& pieces, int& at) {
                    const unsigned char* row = static_cast<const unsigned char*>(row_at(g0 + i));
                    const int lead = (int)(0 - reinterpret_cast<uintptr_t>(row) & 15);
                    const int inside = max((int)p.vocab - lead / kSize, 0) / kEach<KIND>, first_piece = (line - i * lines) * 32;
                    pieces = min(inside, (min(line1, (i + 1) * lines) - i * lines) * 32) - first_piece;
                    from = row + lead + (long long)(first_piece + lane) * 16;
                    at = lead / kSize + (first_piece + lane) * kEach<KIND>;
                };
                if (lane < kAccRows) sh.wmax[lane][warp] = kNoLogit, sh.wsum[lane][warp] = 0.0f, sh.wbest[lane][warp] = -1;  // (rows that this warp has nothing of)
                __syncwarp();
                const unsigned char* from = nullptr;
                int row = lines > 0 ? line0 / lines : 0, to_row = row, to_line = line0, left = 0, unused, to_slot = 0, slot = 0;
                auto send = [&] {  // the next chunk's copies; behind the last line, none
                    while (left <= 0 && to_line < line1) {
                        part_of(to_row, to_line, from, left, unused);
                        to_line = ++to_row * lines;
                    }
                    if (left > 0) {
                        unsigned char* to = ring + to_slot * (kPieces * kPiece);
                        if (left >= kChunk) {
#pragma unroll
                            for (int i = 0; i < kPieces; ++i) copy_16(to + i * kPiece, from + i * kPiece);
                        } else {
#pragma unroll
                            for (int i = 0; i < kPieces; ++i)
                                if (32 * i + lane < left) copy_16(to + i * kPiece, from + i * kPiece);
                        }
                        from += kPieces * kPiece;
                        left -= kChunk;
                    }
                    copies_sent();
                    to_slot = to_slot + 1 == kDeep ? 0 : to_slot + 1;
                };
#pragma unroll 1
                for (int j = 0; j < kDeep; ++j) send();
#pragma unroll 1
                for (int line = line0; line < line1; line = ++row * lines) {
                    Stats st;
                    const unsigned char* unread;
                    int pieces, at;
                    part_of(row, line, unread, pieces, at);
#pragma unroll 1
                    for (; pieces > 0; pieces -= kChunk, at += kChunk * kEach<KIND>) {
                        copies_here<kDeep - 1>();
                        const unsigned char* here = ring + slot * (kPieces * kPiece);
                        uint4 x[kPieces];
                        const uint32_t fill = KIND == GLM53F_KDA_LOGITS_BF16 ? 0xff80ff80u : 0xff800000u;  // -inf
#pragma unroll
                        for (int j = 0; j < kPieces; ++j) {
                            x[j] = make_uint4(fill, fill, fill, fill);
                            if (32 * j + lane < pieces) x[j] = *reinterpret_cast<const uint4*>(here + j * kPiece);
                        }
                        take<GREEDY, KIND>(st, x, at, scale);
                        slot = slot + 1 == kDeep ? 0 : slot + 1;
                        send();
                    }
                    join_lanes<GREEDY>(st, scale);
                    if (lane == 0) sh.wmax[row][warp] = st.m, sh.wsum[row][warp] = st.s, sh.wbest[row][warp] = st.best;
                }
                // What lies before the first boundary and behind the last, 14 entries at most: a row to a warp of the first block.
                if (warp < rows_here) {
                    const void* row = row_at(g0 + warp);
                    const int lead = (int)(0 - reinterpret_cast<uintptr_t>(row) & 15) / kSize;
                    const long long inside = max((p.vocab - lead) / kEach<KIND>, 0ll) * kEach<KIND>, at = lane < lead ? lane : inside + lane;
                    Stats a;
                    if (block == 0 && at < p.vocab && lane < 16) {
                        const float x = target_at<KIND>(row, at);
                        if (x > kNoLogit) a.m = x, a.s = 1.0f, a.best = (int)at;
                    }
                    join_lanes<GREEDY>(a, scale);
                    if (lane == 0) sh.wmax[warp][kAccWarps] = a.m, sh.wsum[warp][kAccWarps] = a.s, sh.wbest[warp][kAccWarps] = a.best;
                }
                __syncthreads();
                // A warp to a row: over the block's warps, then over the cluster's blocks.
                if (warp < rows_here) {
                    Stats a;
                    if (lane <= kAccWarps) a.m = sh.wmax[warp][lane], a.s = sh.wsum[warp][lane], a.best = sh.wbest[warp][lane];
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
                    const double e = token_target == m ? 1.0 : m < INFINITY ? logit_weight(token_target, row_scale_of(m, temperature), power) : 0.0;
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
        const RowScale row_scale = row_scale_of(stop_max, temperature);
        double norm = 1.0;  // the weights' sum, by which the drafter's probabilities are multiplied instead of dividing each of p's
        struct Place {
            Eight<KIND> x;
            Eight<GLM53F_KDA_PROBABILITIES> y;
        };
        const int shift = Eight<KIND>::shift(row), vocab = (int)p.vocab;
        const bool draft_too = less != nullptr && (Eight<GLM53F_KDA_PROBABILITIES>::shift(less) - shift) % 4 == 0;  // (16-byte boundaries at the same entries)
        auto fetch = [&](int i, Place& a) {
            a.x.load(row, i, vocab, true, LOGITS ? kNoLogit : 0.0f);
            if (mode == kLessDraft) a.y.load(less, i, vocab, draft_too, 0.0f);
        };
        auto weights = [&](int i, const Place& a, double (&w)[8]) {
            float x[8];
            a.x.get(x);
            if constexpr (!LOGITS) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = (double)finite_weight(x[j]);
            } else if (fabsf(stop_max) < INFINITY) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = logit_weight(x[j], row_scale, power);
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
                    const int hi = __double2hiint(rest), keep = ~(hi >> 31);  // (by the sign, beside the 64-bit pipe)
                    w[j] = __hiloint2double(hi & keep, __double2loint(rest) & keep);
                }
            } else if (mode == kWithout && (unsigned)(token - i) < 8u) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (i + j == token) w[j] = 0.0;
            }
        };
        long long run0, run1;
        slice((p.vocab + shift + 7) / 8, run0, run1);
        // A warp's runs of the slice, consecutive ones, in slots of `group` steps of 32 runs.
        const int mine0 = (int)(run0 + (run1 - run0) * warp / kAccWarps), mine1 = (int)(run0 + (run1 - run0) * (warp + 1) / kAccWarps);
        const int steps = (mine1 - mine0 + 31) / 32, group = (steps + kSlots - 1) / kSlots;
        double before = 0.0, total = 0.0;
        // Passes over the row, one body of code: of logits with the drafter's probabilities first the weights' sum, then what is drawn from, and
        // once more where that leaves nothing.
        const int drawn_from = mode;
        if (LOGITS && drawn_from == kLessDraft) mode = kWhole;
        for (bool said = false;; said = true) {
            int in_slot = 0, slot = 0;
            double part = 0.0, s = 0.0;
            Place now, ahead;
            if (mine0 + lane < mine1) fetch(8 * (mine0 + lane) - shift, now);
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
                const int r = mine0 + 32 * k + lane;
                if (r + 32 < mine1) fetch(8 * (r + 32) - shift, ahead);
                if (r < mine1) {
                    double w[8];
                    weights(8 * r - shift, now, w);
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
                    const int r = mine0 + 32 * k + lane;
                    double w[8], s8 = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = 0.0;
                    if (r < mine1) {
                        Place a;
                        fetch(8 * r - shift, a);
                        weights(8 * r - shift, a, w);
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
                            seen = 8 * r - shift + j;
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

// The launch of a configuration, and how many of its clusters the device holds at a time (asked of each device once; 0 where it cannot be told).
template <int KIND, int WARPS>
struct AcceptLaunch {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    AcceptLaunch(int batch, int blocks, cudaStream_t stream) {
        cfg.gridDim = dim3((unsigned)batch * blocks);
        cfg.blockDim = dim3(WARPS * 32);
        cfg.dynamicSmemBytes = KIND == GLM53F_KDA_PROBABILITIES ? 0 : WARPS * kDeep * kPieces * kPiece;  // (probabilities have no statistics)
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)blocks;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    cudaError_t configure() {
        static int configured_dev = -1;
        int dev = 0;
        cudaGetDevice(&dev);
        if (configured_dev == dev) return cudaSuccess;
        cudaError_t e = cudaFuncSetAttribute(accept_kernel<KIND, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(accept_kernel<KIND, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes);
        if (e == cudaSuccess) configured_dev = dev;
        return e;
    }
    int fit() {
        static DeviceCounts<2> counted;
        int dev = -1;
        cudaGetDevice(&dev);
        return counted.get(dev, attr[0].val.clusterDim.x == kAccMostBlocks, [&] {
            int n = 0;
            if (configure() == cudaSuccess && cudaOccupancyMaxActiveClusters(&n, accept_kernel<KIND, WARPS>, &cfg) == cudaSuccess) return n;
            cudaGetLastError();
            return -1;
        });
    }
    int run(AcceptParams p) {
        const cudaError_t e = configure();
        if (e != cudaSuccess) return (int)e;
        p.blocks = (int)attr[0].val.clusterDim.x;
        cfg.numAttrs = 1 + early_attribute(attr[1]);
        return (int)cudaLaunchKernelEx(&cfg, accept_kernel<KIND, WARPS>, p);
    }
};

// Few requests: as many threads each as a cluster can have, while all of them run at once.  (Eight windows of eight rows: 11 us in clusters of eight blocks of
// sixteen warps, which fit, 24 in clusters of sixteen, of which one would have to wait.)  Many: smaller blocks, of which an SM holds three.
template <int KIND>
int accept_launch(const AcceptParams& p, int batch, cudaStream_t stream) {
    AcceptLaunch<KIND, kAccMostWarps> most(batch, kAccMostBlocks, stream), many(batch, 8, stream);
    if (batch <= most.fit()) return most.run(p);
    if (batch <= many.fit()) return many.run(p);
    return AcceptLaunch<KIND, 8>(batch, 8, stream).run(p);
}

}  // namespace
}  // namespace kda

extern "C" int glm53f_kda_accept_batch(int32_t batch, const int32_t* cu_rows, int32_t vocab, const void* target, int32_t target_kind, int64_t ld,
                                       const int32_t* tokens, const float* draft, int64_t draft_ld, const float* temperature, const float* u,
                                       int32_t* keep, int32_t* next, glm53f_stream_t stream_) {
    using namespace kda;
    if (batch < 0 || batch > 0xfffffff || vocab < 1 || vocab > 0x7fffffc0 || ld < vocab) return kInvalid;
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
