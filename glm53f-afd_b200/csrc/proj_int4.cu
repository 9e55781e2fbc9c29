// Projections with 4-bit weights: out[r][o] = sum over k of x[r][k] s[o][k / G] (q[o][k] - z[o][k / G]), x bf16, q and z of 0 .. 15, s bf16, G of 32, 64 or 128.
//
// q - z is a whole number that bf16 holds, so the tensor cores' products are exact; a group's sum is formed in f32 and multiplied by its scale there.  No
// weight is rounded.
//
// The weight is laid out once (glm53f_kda_int4_pack) as the matrix instructions take it: tiles of 16 rows, in a tile pieces of 64 k, a piece 16 bytes for each
// lane of a warp, the four k steps' fragments a word each; in a word the pairs of neighbouring k lie 16 bits apart, so that a shift, a mask and one
// or put two of them into bf16s of 128 + q, from which 128 + z is taken.
//
// Few rows (this kernel): bound by HBM, the weights' bytes, and next to it by the eleven operations that a word of eight weights costs.  A block an SM; a warp copies tiles in bulk into a ring
// of shared memory, 58 KB (many long rows) to 200 KB ahead; the rows lie beside it; sixteen warps divide the k of a tile between them, two pieces at a time, and their sums meet in
// shared memory once a tile.  24,640 x 4,096 in groups of 128: 17.4 us a row (3.0 TB/s; 14.2 without widening and products), 18.7 for eight; 4,096 x 8,192: 7 and 8.6 us.
// (Loads into registers eight pieces ahead shared their scoreboards, so that each waited for all: 21.5 us.  One piece a stage, whose waiting and addresses cost as
// much as its products: 21.6 us.)  Eight rows are one instruction's columns and cost what one does; from nine on the other kernel takes them: eight
// rows take it 23.0, 11.4 and, of 500 x 512, 4.5 us, and this one 18.7, 8.5 and 2.6.  Rows of more than 150 KB together come with the weights, so that a row's bits depend on nothing but the row: 4,096
// outputs, eight rows of k = 9,600 10.5 us (38 by the other kernel), 12,288 12.3 (12.5), 16,384 in groups of 64 16.2 (19.1); 8,192 outputs, k = 28,672 46.9 (38.4) and 65,536 104 (81), of which
// the bits are the price.

#include <type_traits>

#include "common.cuh"
#include "glm53f_proj.h"
#include "kda_internal.h"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace kda {
namespace {

constexpr int kTile = 16;        // weight rows of a tile
constexpr int kPiece = 64;       // k of a piece
constexpr int kFewWarps = 16, kFewThreads = 32 * (kFewWarps + 1);  // the last warp loads
constexpr int kFewRows = 8;
constexpr int kFewX = 150 * 1024, kFewShared = 208 * 1024;  // bytes for the rows of x, and with the ring
constexpr int kFewStages = 12;   // of the ring, at most
constexpr int kRowPad = 8;       // bf16 between them: the eight rows that one load of fragments reads lie in different banks

struct Int4Layout {  // bytes from the packed weight's start
    long long tiles, pieces, groups, scales, zeros, bytes;
    Int4Layout(int64_t n, int64_t k, int group, bool has_zeros) {
        tiles = (n + kTile - 1) / kTile, pieces = k / kPiece, groups = k / group;
        auto up = [](long long x) { return (x + 255) / 256 * 256; };
        scales = up(tiles * pieces * 512);
        zeros = up(scales + tiles * groups * kTile * 2);
        bytes = has_zeros ? up(zeros + tiles * groups * kTile) : zeros;
    }
};

struct Int4Params {
    const uint16_t* x;
    long long ldx, ldo;
    const uint4* codes;
    const uint32_t* scales;   // [tile][group][8]: rows i and i + 8
    const uint16_t* zeros;    // the same in bytes
    void* out;
    int rows, n, k, out_f32;
    int tiles, pieces, split;  // warps that share a tile
    int x_bytes, stages;       // of shared memory for the rows of x; of the ring behind them
    int stage;                 // bytes of one
    int* status;
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_4(uint32_t at, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// The fragments of one k step: rows i (even registers) and i + 8, less lo and hi (128 + z in both halves).  The mask and the exponent come in registers: an
// instruction takes one constant, and with two the compiler makes two of it.
struct Widen {
    uint32_t mask, exponent;
    __device__ __forceinline__ Widen() {
        asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(mask));
        asm volatile("mov.b32 %0, 0x43004300;" : "=r"(exponent));
    }
    __device__ __forceinline__ void operator()(uint32_t w, uint32_t lo, uint32_t hi, uint32_t (&a)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t r;
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w >> (4 * j)), "r"(mask), "r"(exponent));  // (w & mask) | exponent
            a[j] = sub_bf16x2(r, j % 2 ? hi : lo);
        }
    }
};

enum : int { kStatusInt4FewEmpty = 178, kStatusInt4FewFull = 179 };

// A stage of the ring: two pieces (128 k) for each warp, the scales and zero points of their groups; LONG: and the rows of x over the same k.
template <int G, bool ZEROS>
struct Few {
    static constexpr int N = 2 * kPiece / G;                      // groups of a warp's pieces
    static constexpr int kScaleBytes = kPiece * 32 / G;           // of a piece (of 128: half of them, its pieces come in pairs)
    static constexpr int kZeroBytes = ZEROS ? kPiece * 16 / G : 0;
    static constexpr int oScales = kFewWarps * 1024, oZeros = oScales + 2 * kFewWarps * kScaleBytes, kStage = oZeros + 2 * kFewWarps * kZeroBytes;
    static constexpr int kLongPitch = 2 * kFewWarps * kPiece * 2 + 2 * kRowPad;  // between rows of x
};

// LONG: rows that do not all fit beside the ring.  They come with the weights, for every tile again (all warps share a tile then), and everything is summed in the same order: what up to eight
// rows hold, and how many there are, changes no bit of another.
template <int G, bool ZEROS, bool LONG>
__global__ void __launch_bounds__(kFewThreads, 1) int4_few_kernel(const Int4Params p) {
    using F = Few<G, ZEROS>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sums[2][kFewWarps][kTile * kFewRows];
    __shared__ __align__(16) uint4 nothing;  // what rows that are not there hold
    __shared__ __align__(8) uint64_t full[kFewStages], empty[kFewStages], x_full;
    __shared__ volatile uint32_t ctl[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int abreast = kFewWarps / p.split;                          // tiles at a time
    const int at_once = 2 * p.split, per = (p.pieces + at_once - 1) / at_once;  // pieces of a tile in a stage; stages of a tile
    const int groups = p.k / G, step = gridDim.x * abreast;
    const int pitch = LONG ? F::kLongPitch : (p.k + kRowPad) * 2, stage = LONG ? p.stage : F::kStage;
    unsigned char *ring = smem + p.x_bytes, *rows = LONG ? ring + F::kStage : smem;
    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], kFewWarps);
        mbar_init(&x_full, 1);
        ctl[0] = ctl[1] = 0u;
        nothing = make_uint4(0u, 0u, 0u, 0u);
        mbar_init_fence();
    }
    __syncthreads();
    const WaitCtx ctx{ctl, ctl + 1, p.status};
    grid_ready();
    int s = 0;
    uint32_t ph = 0;

    if (warp == kFewWarps) {
        // A lane a tile: its pieces of a stage lie together, their scales and zero points too.
        for (int tile = blockIdx.x * abreast; tile < p.tiles; tile += step) {
            const int tiles = min(abreast, p.tiles - tile);
            const long long t = tile + lane;
            for (int c = 0; c < per; ++c) {
                const int piece = c * at_once, pieces = min(at_once, p.pieces - piece);
                if (!tc::warp_all(mbar_wait(&empty[s], ph ^ 1u, ctx, kStatusInt4FewEmpty))) break;
                if (lane == 0) {
                    ctl[0] = ctl[0] + 1u;
                    mbar_arrive_expect_tx(&full[s], tiles * pieces * (512 + F::kScaleBytes + F::kZeroBytes) + (LONG ? p.rows * pieces * kPiece * 2 : 0));
                }
                __syncwarp();
                if (LONG && lane < p.rows) bulk_load(rows + s * stage + lane * pitch, p.x + lane * p.ldx + piece * kPiece, pieces * kPiece * 2, &full[s]);
                if (lane < tiles) {
                    unsigned char* to = ring + s * stage;
                    const long long group = t * groups + piece * kPiece / G;
                    bulk_load(to + lane * at_once * 512, p.codes + (t * p.pieces + piece) * 32, pieces * 512, &full[s]);
                    bulk_load(to + F::oScales + lane * at_once * F::kScaleBytes, p.scales + group * 8, pieces * F::kScaleBytes, &full[s]);
                    if constexpr (ZEROS) bulk_load(to + F::oZeros + lane * at_once * F::kZeroBytes, p.zeros + group * 8, pieces * F::kZeroBytes, &full[s]);
                }
                if (++s == p.stages) s = 0, ph ^= 1u;
            }
        }
    } else {
        if (!LONG && warp == 0) {
            if (lane == 0) mbar_arrive_expect_tx(&x_full, p.rows * p.k * 2);
            __syncwarp();
            if (lane < p.rows) bulk_load(smem + lane * pitch, p.x + lane * p.ldx, p.k * 2, &x_full);
        }
        const Widen widen;
        const int kw = warp % p.split, tw = warp / p.split, g = lane >> 2;  // this warp's part of k, its tile of those at a time
        const int xr = lane & 7;
        const bool there = xr < p.rows;
        const uint32_t xrow = there ? smem_u32(rows + xr * pitch + (lane >> 3) * 16) + kw * kPiece * 4 : smem_u32(&nothing), half = there ? 64u : 0u;
        const uint32_t xstep = !there ? 0u : LONG ? stage : at_once * kPiece * 2;  // from a stage to the next
        if (!LONG) mbar_wait(&x_full, 0u, ctx, kStatusInt4FewFull);
        int buf = 0;
        // Every warp takes part in each round, with or without a tile, as the barrier needs them.
        for (int tile = blockIdx.x * abreast; tile < p.tiles; tile += step, buf ^= 1) {
            float acc[4] = {};
            for (int c = 0; c < per; ++c) {
                mbar_wait(&full[s], ph, ctx, kStatusInt4FewFull);  // (after a wait that gave up all others do: the sums are lost, the status says so)
                const int mine = tile + tw < p.tiles ? p.pieces - c * at_once - 2 * kw : 0;  // pieces, of two
                const unsigned char* from = ring + s * stage;
                const uint32_t xat = xrow + (LONG ? s : c) * xstep;
                uint4 codes[2];
                uint32_t scale[F::N], zero[F::N];
                if (mine > 0) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) codes[u] = *reinterpret_cast<const uint4*>(from + warp * 1024 + u * 512 + lane * 16);
#pragma unroll
                    for (int j = 0; j < F::N; ++j) {
                        const int at = (warp * F::N + j) * 8 + g;
                        scale[j] = *(reinterpret_cast<const uint32_t*>(from + F::oScales) + at);
                        if constexpr (ZEROS) zero[j] = *(reinterpret_cast<const uint16_t*>(from + F::oZeros) + at);
                    }
                }
                auto taken = [&] {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[s]);
                    if (++s == p.stages) s = 0, ph ^= 1u;
                };
                if (!LONG) taken();
                constexpr int kSteps = G / 16;  // of a group
                float d[4] = {};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (u >= mine) break;
                    const uint32_t w[4] = {codes[u].x, codes[u].y, codes[u].z, codes[u].w};
                    uint32_t b[8];
                    ldmatrix_4(xat + u * 2 * half, b[0], b[1], b[2], b[3]);
                    ldmatrix_4(xat + u * 2 * half + half, b[4], b[5], b[6], b[7]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int step = 4 * u + q, j = step / kSteps;
                        uint32_t lo = 0x43084308u, hi = 0x43084308u;
                        if constexpr (ZEROS) lo = __byte_perm(zero[j], 0x43434343u, 0x4040), hi = __byte_perm(zero[j], 0x43434343u, 0x4141);
                        uint32_t a[4];
                        widen(w[q], lo, hi, a);
                        mma(d, a, b[2 * q], b[2 * q + 1]);
                        if (step % kSteps == kSteps - 1) {
                            const float s0 = __uint_as_float(scale[j] << 16), s1 = __uint_as_float(scale[j] & 0xffff0000u);
                            acc[0] = fmaf(s0, d[0], acc[0]), acc[1] = fmaf(s0, d[1], acc[1]);
                            acc[2] = fmaf(s1, d[2], acc[2]), acc[3] = fmaf(s1, d[3], acc[3]);
                            d[0] = d[1] = d[2] = d[3] = 0.0f;
                        }
                    }
                }
                if (LONG) taken();
            }
            float* to = sums[buf][warp];
            *reinterpret_cast<float2*>(to + g * kFewRows + 2 * (lane & 3)) = make_float2(acc[0], acc[1]);
            *reinterpret_cast<float2*>(to + (g + 8) * kFewRows + 2 * (lane & 3)) = make_float2(acc[2], acc[3]);
            named_bar_sync(1, 32 * kFewWarps);
            // (the next tile's sums go to the other buffer; this one is written again behind the next barrier)
            for (int e = tid; e < abreast * kTile * kFewRows; e += 32 * kFewWarps) {
                const int t = e / (kTile * kFewRows), in = e % (kTile * kFewRows), f = in % kTile, r = in / kTile;
                const int o = (tile + t) * kTile + f;
                if (r >= p.rows || o >= p.n) continue;
                float sum = 0.0f;
                for (int q = 0; q < p.split; ++q) sum += sums[buf][t * p.split + q][f * kFewRows + r];
                if (p.out_f32) static_cast<float*>(p.out)[r * p.ldo + o] = sum;
                else static_cast<uint16_t*>(p.out)[r * p.ldo + o] = f32_to_bf16_bits(sum);
            }
        }
    }
    if (ctl[1]) {  // after a wait that gave up, copies into this block's shared memory may still be in flight: a bounded time for them
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {
        }
    }
}

// ---- many rows ----------------------------------------------------------------------------------------------------------------
// From nine rows on, a tcgen05 product: a tile is 128 weight rows (the M operand) x N rows of x.  Warps that widen turn the packed words into bf16 fragments and store
// them into tensor memory, where a matrix instruction takes its first operand from: the packed layout is that of the fragments, so nothing is
// shuffled and shared memory holds x only.  A group's products go into one of two accumulators of their own; warps that sum fetch each, multiply it
// by the group's scales (a lane is a weight row) and add it to the f32 sums in their registers.  Roles of a block:
//   warp 0        tensor copies of x (64 k x N rows, 128-byte swizzle) into a ring
//   warps 1, 3    the matrix instructions (a stage each in turn, with groups of 128: the waits of a stage take one warp longer than its products the tensor cores)
//   warp 2        bulk copies of the packed words, 128 k at a time, into another
//   warps 4-      widen, 128 k at a time, two or four such stages in tensor memory
//   the others    sum: a warpgroup for each kSumCols columns
// Few tiles: the blocks of a cluster share a tile's k and add their sums, each for some rows, in rank order through distributed shared memory.
//
// N is the smallest that holds the rows, 128 at most (64 for more than 64 rows: 100 rows x 4,096 x 8,192 23.5 us against 20.8, 400 rows 76 against 58, 2,048 rows 202 against 145; only
// 500 x 512 is faster, 6.6 against 8.9).  Bound by the issue of widening and summing and by the chain from words to sums: 2,048 rows x 4,096 x 8,192 in groups of 128 take
// 141 to 159 us, 0.5 of the measured bf16 rate (their products alone 83); groups of 64 217, of 32 367, a fetch of the accumulator for each.  40 rows in groups of 64 with zero points 14.9 us.
// (Scales and zero points fetched a few groups ahead, without L2 asked before: 154 and 21.3 us.)

enum : int { kStatusInt4Empty = 170, kStatusInt4Full = 171, kStatusInt4AEmpty = 172, kStatusInt4AFull = 173, kStatusInt4AccEmpty = 174, kStatusInt4AccFull = 175, kStatusInt4Words = 176, kStatusInt4WordsFull = 177 };

struct ManyParams {
    CUtensorMap tm_x, tm_words, tm_scales, tm_zeros;  // (the last one with zero points only)
    const uint16_t* scales;
    void* out;
    long long ldo;
    int rows, n, k, out_f32, group;
    int tiles, pieces, groups;  // of 16 weight rows, of 64 k, of a row's scales
    int m_tiles, split;         // tiles of weight rows; blocks that share a tile's k
    int* status;
};

template <int N>
struct Many {
    static constexpr int kSumCols = N < 32 ? N : 32 * ((N + 63) / 64);  // (N = 128: 64)
    static constexpr int kSumGroups = N / kSumCols;
    // Warpgroups that widen, a stage each in turn.  Up to 32 rows one, two blocks an SM; more: two, one block.  (4,096 x 8,192, groups of 64, us, one and two: 16 rows 12.1 and 12.8, 40 rows 16.8 and
    // 14.9; 24,640 x 4,096 16 rows 23.3 and 28.0, 40 rows 32.4 and 33.8.)
    static constexpr int kWideners = N <= 32 ? 1 : 2;
    static constexpr int kSumWarp = 4 + 4 * kWideners;    // the first warp that sums
    static constexpr int kThreads = 32 * kSumWarp + 128 * kSumGroups;
    static constexpr int kBoxBytes = N * 128;             // 64 k of x
    static constexpr int kRing = N <= 32 ? 6 : 4;         // stages of 128 k: of x
    static constexpr int kStages = N <= 32 ? 2 : 4;      // ... in tensor memory (even, as the rings are: each of two warps that take turns then meets every phase of a place)
    static constexpr int kStageCols = 64;
    static constexpr int kAccs = 2;                       // accumulators, a group's products each
    static constexpr int kAccCols = kAccs * N;
    static constexpr int kUsed = kAccCols + kStages * kStageCols;
    static constexpr int kCols = kUsed <= 256 ? 256 : 512;
    static constexpr int kBlocks = kCols == 256 ? 2 : 1;  // an SM
    static constexpr int kWords = N <= 32 ? 6 : 4;        // stages of packed words in shared memory
    static constexpr int oZeros = 8 * 1024, kWordBytes = oZeros + 512;  // of a stage: two pieces of 8 tiles, and their zero points
    static constexpr int oWords = kRing * 2 * kBoxBytes;
    static constexpr int oBars = oWords + kWords * kWordBytes;
    static constexpr int oCtl = oBars + (2 * kRing + 2 * kWords + 2 * kStages + 2 * kAccs) * 8;
    static constexpr int kBytes = oCtl + 32 + 1024;
};

__device__ __forceinline__ void tensor_load_2d(void* to, const void* tm, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(to)),
                 "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void tensor_prefetch_2d(const void* tm, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer_load(const void* local, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// Where a block's tensor memory begins, known when it is compiled.
template <uint32_t AT>
struct Column {
    __device__ __forceinline__ constexpr operator uint32_t() const { return AT; }
};

// ZEROS: zero points are read; without them they are a constant (their forming takes a fifth of what widening does).
template <int N, bool ZEROS>
__global__ void __launch_bounds__(Many<N>::kThreads, Many<N>::kBlocks) int4_many_kernel(const __grid_constant__ ManyParams p) {
    using C = Many<N>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::oBars);
    uint64_t *empty = full + C::kRing, *w_full = empty + C::kRing, *w_empty = w_full + C::kWords, *a_full = w_empty + C::kWords, *a_empty = a_full + C::kStages, *acc_full = a_empty + C::kStages, *acc_empty = acc_full + C::kAccs;
    volatile uint32_t* ctl = reinterpret_cast<volatile uint32_t*>(smem + C::oCtl);
    uint32_t* tmem_slot = const_cast<uint32_t*>(ctl) + 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < C::kRing; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < C::kWords; ++i) mbar_init(&w_full[i], 1), mbar_init(&w_empty[i], 4);
        for (int i = 0; i < C::kStages; ++i) mbar_init(&a_full[i], 4), mbar_init(&a_empty[i], 1);
        for (int i = 0; i < C::kAccs; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], 4 * C::kSumGroups);
        ctl[0] = ctl[1] = 0u;
        mbar_init_fence();
    }
    if (warp == 1) tc::tmem_alloc(tmem_slot, C::kCols);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tm = *tmem_slot, stages0 = tm + C::kAccCols;
    const WaitCtx ctx{ctl, ctl + 1, p.status};
    const int split = p.split, part = split > 1 ? (int)cluster_rank() : 0, tile = (int)blockIdx.x / split;
    const int mt = tile % p.m_tiles, row0 = tile / p.m_tiles * N;       // this block's weight rows (in units of 128) and rows of x
    const int per = p.pieces / split, piece0 = part * per, stages = (per + 1) / 2;
    grid_ready();

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            for (int st = 0; st < stages; ++st) {
                const int pieces = min(per - 2 * st, 2);
                if (!mbar_wait(C::kRing != C::kStages ? &empty[s] : &a_empty[s], ph ^ 1u, ctx, kStatusInt4Empty)) break;
                ctl[0] = ctl[0] + 1u;
                mbar_arrive_expect_tx(&full[s], pieces * C::kBoxBytes);
                for (int i = 0; i < pieces; ++i)
                    tensor_load_2d(smem + (2 * s + i) * C::kBoxBytes, &p.tm_x, (piece0 + 2 * st + i) * kPiece, row0, &full[s]);
                if (++s == C::kRing) s = 0, ph ^= 1u;
            }
        }
    } else if (warp == 2) {
        // Eight tiles' words of two pieces, and their zero points, a box each; their scales, which the warps that sum fetch four groups ahead, into L2.
        if (lane == 0) {
            const int per_stage = 2 * kPiece / p.group, group0 = piece0 * kPiece / p.group;
            int c = 0;
            uint32_t ph = 0;
            for (int st = 0; st < stages; ++st) {
                if (!mbar_wait(&w_empty[c], ph ^ 1u, ctx, kStatusInt4Words)) break;
                unsigned char* words = smem + C::oWords + c * C::kWordBytes;
                mbar_arrive_expect_tx(&w_full[c], C::oZeros + (ZEROS ? 8 * per_stage * 16 : 0));
                tensor_load_2d(words, &p.tm_words, (piece0 + 2 * st) * 128, mt * 8, &w_full[c]);
                if constexpr (ZEROS) tensor_load_2d(words + C::oZeros, &p.tm_zeros, (group0 + st * per_stage) * 8, mt * 8, &w_full[c]);
                tensor_prefetch_2d(&p.tm_scales, (group0 + st * per_stage) * 8, mt * 8);
                if (++c == C::kWords) c = 0, ph ^= 1u;
            }
        }
    } else if (warp == 1 || warp == 3) {
        constexpr uint32_t idesc = tc::idesc_bf16(128, N, 0, 0, 0);
        const uint32_t leader = tc::elect_one();
        // The warp converged, one lane issuing, a stage's eight k steps unrolled for the group's size: little stands between two instructions (a loop that asks at each step
        // whether a group begins or ends took 190 cycles a step, three times the product's).  Of a descriptor only the low half changes, and where the tensor
        // memory begins is a constant wherever this kernel is alone on the SM, so that every operand is computed in uniform registers.
        auto products = [&](auto group_steps, auto begin) {
            constexpr int js = decltype(group_steps)::value;  // k steps of 16 of a group
            const uint32_t tm0 = begin, stage0 = tm0 + C::kAccCols;
            constexpr uint64_t high = (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61 | (uint64_t)(16 >> 4) << 16;
            const uint32_t ring0 = (smem_u32(smem) & 0x3FFFFu) >> 4;
            // With groups of 128 two warps take turns, each with an accumulator of its own; smaller groups use both within a stage, and a wait tells two of an accumulator's phases
            // apart, not three: one warp.
            constexpr int turns = js == 8 ? 2 : 1;
            for (int st = warp >> 1; st < stages && warp >> 1 < turns; st += turns) {
                const int a = st % C::kStages, s = st % C::kRing;
                const uint32_t w = stage0 + (uint32_t)(a * C::kStageCols);
                const bool whole = 2 * st + 1 < per;
                if (!tc::warp_all(mbar_wait(&full[s], st / C::kRing & 1, ctx, kStatusInt4Full))) return;
                if (!tc::warp_all(mbar_wait(&a_full[a], st / C::kStages & 1, ctx, kStatusInt4AFull))) return;
                const uint64_t x = high | (ring0 + (uint32_t)(s * 2 * (C::kBoxBytes >> 4)));
#pragma unroll
                for (int step = 0; step < 8; ++step) {
                    if (step == 4 && !whole) break;
                    const int job = st * (8 / js) + step / js, buf = job & 1;
                    if (step % js == 0) {
                        if (!tc::warp_all(mbar_wait(&acc_empty[buf], (job >> 1 & 1) ^ 1u, ctx, kStatusInt4AccEmpty))) return;
                        tc::fence_after_sync();
                    }
                    tc::mma_bf16_ts_if(leader, tm0 + (uint32_t)(buf * N), w + step * 8, x + (step / 4) * (C::kBoxBytes >> 4) + 2 * (step % 4), idesc, step % js != 0);
                    if (step % js == js - 1) tc::mma_commit_if(leader, &acc_full[buf]);
                }
                tc::mma_commit_if(leader, &a_empty[a]);
                if (C::kRing != C::kStages) tc::mma_commit_if(leader, &empty[s]);
            }
        };
        auto from = [&](auto begin) {
            if (p.group == 128) products(std::integral_constant<int, 8>{}, begin);
            else if (p.group == 64) products(std::integral_constant<int, 4>{}, begin);
            else products(std::integral_constant<int, 2>{}, begin);
        };
        // All 512 columns begin at 0; 256 at 0 or 256 beside another block of this kernel, and anywhere beside another kernel's smaller part.
        if (C::kCols == 512 || tm == 0) from(Column<0>{});
        else if (tm == 256) from(Column<256>{});
        else from(tm);
    } else if (warp >= 4 && warp < C::kSumWarp) {
        // Weight rows 32 q .. of each 128: two tiles of 16, the lanes' words of both pieces of a stage.
        const Widen widen;
        const int q = warp & 3, g = lane >> 2, turn = (warp - 4) >> 2;
        const int halves = 2 * kPiece / p.group, half_shift = p.group == 32 ? 0 : p.group == 64 ? 1 : 2;  // groups of a stage; which of them its halves of a piece (32 k) lie in
        for (int st = turn; st < stages; st += C::kWideners) {
            const int a = st % C::kStages, c = st % C::kWords, pieces = min(per - 2 * st, 2);
            if (!tc::warp_all(mbar_wait(&w_full[c], st / C::kWords & 1, ctx, kStatusInt4WordsFull))) break;
            const unsigned char* from = smem + C::oWords + c * C::kWordBytes;
            uint4 now[2][2];
            uint32_t zero[2][2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    now[i][t] = *reinterpret_cast<const uint4*>(from + (q * 2 + t) * 1024 + i * 512 + lane * 16);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if constexpr (ZEROS) zero[i][t][h] = reinterpret_cast<const uint16_t*>(from + C::oZeros)[((q * 2 + t) * halves + ((2 * i + h) >> half_shift)) * 8 + g];
                }
            if (!tc::warp_all(mbar_wait(&a_empty[a], (st / C::kStages & 1) ^ 1u, ctx, kStatusInt4AEmpty))) break;
            tc::fence_after_sync();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i >= pieces) break;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t words[4] = {now[i][t].x, now[i][t].y, now[i][t].z, now[i][t].w};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 32 k: their group's zero points
                        uint32_t lo = 0x43084308u, hi = 0x43084308u;
                        if constexpr (ZEROS) lo = __byte_perm(zero[i][t][h], 0x43434343u, 0x4040), hi = __byte_perm(zero[i][t][h], 0x43434343u, 0x4141);
                        uint32_t f[4], e[4];
                        widen(words[2 * h], lo, hi, f);
                        widen(words[2 * h + 1], lo, hi, e);
                        const uint32_t r[8] = {f[0], f[1], f[2], f[3], e[0], e[1], e[2], e[3]};
                        tc::tmem_st_pairs(stages0 + a * C::kStageCols + i * 32 + h * 16 + ((uint32_t)(q * 32 + t * 16) << 16), r);
                    }
                }
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&a_full[a]), mbar_arrive(&w_empty[c]);
        }
    } else if (warp >= C::kSumWarp) {
        const int sg = (warp - C::kSumWarp) >> 2, q = warp & 3, col0 = sg * C::kSumCols;
        const int w = mt * 8 + q * 2 + (lane >> 4);  // this lane's tile of 16 weight rows
        const int o = mt * 128 + q * 32 + lane;
        const bool there = w < p.tiles;
        const uint16_t* scale = p.scales + ((long long)(there ? w : 0) * p.groups * 8 + (lane & 7)) * 2 + (lane >> 3 & 1);
        const int group0 = piece0 * kPiece / p.group, jobs = per * kPiece / p.group;
        float sum[C::kSumCols];
#pragma unroll
        for (int c = 0; c < C::kSumCols; ++c) sum[c] = 0.0f;
        // Scales four groups ahead: a group of 32 k takes less time than a load.
        uint16_t ahead[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) ahead[u] = there && u < jobs ? __ldg(scale + (long long)(group0 + u) * 16) : 0;
        bool ok = true;
        for (int j = 0; j < jobs && ok; j += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (j + u >= jobs || !ok) continue;
                const int i = j + u, buf = i & 1;
                const float s = bf16_bits_to_f32(ahead[u]);
                ahead[u] = there && i + 4 < jobs ? __ldg(scale + (long long)(group0 + i + 4) * 16) : 0;
                if (!(ok = tc::warp_all(mbar_wait(&acc_full[buf], i >> 1 & 1, ctx, kStatusInt4AccFull)))) continue;
                tc::fence_after_sync();
                const float2 s2 = make_float2(s, s);
                constexpr int W = 16;
#pragma unroll
                for (int c0 = 0; c0 < C::kSumCols; c0 += W) {
                    uint32_t r[W];
                    tc::tmem_ld16(tc::tmem_addr(tm, q, buf * N + col0 + c0), r);
                    tc::tmem_ld_wait();
                    if (c0 + W == C::kSumCols) {  // the accumulator is free as soon as its last columns are in registers
                        tc::fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[buf]);
                    }
#pragma unroll
                    for (int c = 0; c < W; c += 2) {
                        const float2 v = fma2(s2, make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), make_float2(sum[c0 + c], sum[c0 + c + 1]));
                        sum[c0 + c] = v.x, sum[c0 + c + 1] = v.y;
                    }
                }
            }
        }
        auto store = [&](int c, float v) {
            const long long r = row0 + c;
            if (o < p.n && r < p.rows) {
                if (p.out_f32) static_cast<float*>(p.out)[r * p.ldo + o] = v;
                else static_cast<uint16_t*>(p.out)[r * p.ldo + o] = f32_to_bf16_bits(v);
            }
        };
        if (split == 1) {
            if (ok)
#pragma unroll
                for (int c = 0; c < C::kSumCols; ++c) store(col0 + c, sum[c]);
        } else {
            // x has been read; its ring takes the sums, [N][128].
            float* red = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int c = 0; c < C::kSumCols; ++c) red[(col0 + c) * 128 + q * 32 + lane] = sum[c];
        }
    }
    if (ctl[1]) {  // after a wait that gave up, copies into this block's shared memory may still be in flight: a bounded time for them
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) tc::tmem_dealloc(tm, C::kCols);
    if (split > 1) {
        cluster_meet();
        const float* red = reinterpret_cast<const float*>(smem);
        const int mine = N / split;
        for (int e = tid; e < mine * 128; e += C::kThreads) {
            const int c = part * mine + e / 128, f = e % 128, o = mt * 128 + f;
            const long long r = row0 + c;
            if (o >= p.n || r >= p.rows) continue;
            float v = 0.0f;
            for (int b = 0; b < split; ++b) v += peer_load(red + c * 128 + f, b);
            if (p.out_f32) static_cast<float*>(p.out)[r * p.ldo + o] = v;
            else static_cast<uint16_t*>(p.out)[r * p.ldo + o] = f32_to_bf16_bits(v);
        }
        cluster_meet();
    }
}

// A thread a word of the packed weight, or a group's pair of scales and zero points.  Once a weight: 24,640 x 4,096 99 us (15.9 for the bytes: the codes are read a byte at a time), 4,096 x 8,192 36.
__global__ void int4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int n, int k, int group, uint32_t* to, uint32_t* to_scales,
                                 uint16_t* to_zeros) {
    const long long tiles = (n + kTile - 1) / kTile, words = tiles * (k / kPiece) * 128, pairs = tiles * (k / group) * 8;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < words + pairs; i += (long long)gridDim.x * blockDim.x) {
        if (i < words) {
            const int s = (int)(i & 3), lane = (int)(i >> 2) & 31;
            const long long piece = i >> 7, tile = piece / (k / kPiece);
            const int k0 = (int)(piece % (k / kPiece)) * kPiece + 16 * s + 2 * (lane & 3), row = (int)tile * kTile + (lane >> 2);
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = row + 8 * (j & 1);
                const uint32_t two = r < n ? codes[((long long)r * k + k0 + 8 * (j >> 1)) / 2] : 0u;
                w |= (two & 15u) << (4 * j) | (two >> 4) << (16 + 4 * j);
            }
            to[i] = w;
        } else {
            const long long at = i - words, tile = at / (8ll * (k / group));
            const int gk = (int)(at / 8 % (k / group)), row = (int)tile * kTile + (int)(at & 7);
            uint32_t two = 0, z = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = row + 8 * h;
                if (r >= n) continue;
                two |= (uint32_t)scales[(long long)r * (k / group) + gk] << (16 * h);
                if (zeros != nullptr) z |= (uint32_t)(zeros[(long long)r * (k / group) + gk] & 15u) << (8 * h);
            }
            to_scales[at] = two;
            if (zeros != nullptr) to_zeros[at] = (uint16_t)z;
        }
    }
}

bool shape_ok(int32_t n, int32_t k, int32_t group) {
    return n >= 1 && n <= 1 << 30 && k >= kPiece && k % kPiece == 0 && k <= 65536 && (group == 32 || group == 64 || group == 128) && k % group == 0;
}
bool on16(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int G, bool ZEROS, bool LONG>
int few_launch(Int4Params& p, unsigned blocks, cudaStream_t stream) {
    using F = Few<G, ZEROS>;
    p.stage = LONG ? (F::kStage + p.rows * F::kLongPitch + 127) / 128 * 128 : F::kStage;
    static_assert(kFewShared / F::kStage <= kFewStages && (kFewShared - kFewX) / F::kStage >= 2 && kFewShared / (F::kStage + kFewRows * F::kLongPitch + 127) >= 2, "the ring's barriers, and two stages at least");
    p.stages = (kFewShared - p.x_bytes) / p.stage;
    const cudaError_t e = cudaFuncSetAttribute(int4_few_kernel<G, ZEROS, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared);
    if (e != cudaSuccess) return (int)e;
    return launch_early(int4_few_kernel<G, ZEROS, LONG>, dim3(blocks), kFewThreads, p.x_bytes + p.stages * p.stage, stream, p);
}

template <int N, bool ZEROS>
int many_launch(ManyParams& p, const uint16_t* x, long long ldx, const unsigned char* w, const Int4Layout& at, cudaStream_t stream) {
    using C = Many<N>;
    EncodeTiled enc = encode_tiled();
    if (enc == nullptr) return (int)cudaErrorNotSupported;
    auto map = [&](CUtensorMap* to, CUtensorMapDataType type, const void* from, long long inner, long long outer, long long pitch, int box_inner, int box_outer, CUtensorMapSwizzle swizzle) {
        const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer}, strides[1] = {(cuuint64_t)pitch};
        const cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer}, estr[2] = {1u, 1u};
        return enc(to, type, 2, const_cast<void*>(from), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    const int per_stage = 2 * kPiece / p.group;
    const long long groups = at.groups;
    if (!map(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, p.k, p.rows, ldx * 2, kPiece, N, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !map(&p.tm_words, CU_TENSOR_MAP_DATA_TYPE_UINT32, w, at.pieces * 128, at.tiles, at.pieces * 512, 256, 8, CU_TENSOR_MAP_SWIZZLE_NONE) ||
        !map(&p.tm_scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, w + at.scales, groups * 8, at.tiles, groups * 32, per_stage * 8, 8, CU_TENSOR_MAP_SWIZZLE_NONE) ||
        (ZEROS && !map(&p.tm_zeros, CU_TENSOR_MAP_DATA_TYPE_UINT16, w + at.zeros, groups * 8, at.tiles, groups * 16, per_stage * 8, 8, CU_TENSOR_MAP_SWIZZLE_NONE)))
        return (int)cudaErrorNotSupported;
    p.m_tiles = (p.n + 127) / 128;
    const long long tiles = (long long)p.m_tiles * ((p.rows - 1) / N + 1), room = (long long)sm_count() * C::kBlocks;
    p.split = 1;
    // Parts of k for the blocks of a cluster, of whole stages and groups, while all blocks run at once.
    for (int s = 8; s > 1 && p.split == 1; s /= 2)
        if (p.pieces % (2 * s) == 0 && p.pieces / s >= 4 && tiles * s <= room) p.split = s;
    if (tiles * p.split > 0x7fffffff) return kInvalid;
    cudaError_t e = cudaFuncSetAttribute(int4_many_kernel<N, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * p.split));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    unsigned na = early_attribute(attr[0]);
    if (p.split > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)p.split;
        attr[na].val.clusterDim.y = 1;
        attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    return (int)cudaLaunchKernelEx(&cfg, int4_many_kernel<N, ZEROS>, p);
}

}  // namespace
}  // namespace kda

extern "C" int64_t glm53f_kda_int4_bytes(int32_t n, int32_t k, int32_t group, int32_t zeros) {
    using namespace kda;
    return shape_ok(n, k, group) ? Int4Layout(n, k, group, zeros != 0).bytes : 0;
}

extern "C" int32_t glm53f_kda_int4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int32_t n, int32_t k, int32_t group, void* packed,
                                        glm53f_stream_t stream) {
    using namespace kda;
    if (!shape_ok(n, k, group) || codes == nullptr || scales == nullptr || (reinterpret_cast<uintptr_t>(scales) & 1) || !on16(packed)) return kInvalid;
    const Int4Layout at(n, k, group, zeros != nullptr);
    auto* to = static_cast<unsigned char*>(packed);
    const long long blocks = (at.tiles * at.pieces * 128 + at.tiles * at.groups * 8 + 255) / 256;
    int4_pack_kernel<<<(unsigned)(blocks < 65535 ? blocks : 65535), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        codes, scales, zeros, n, k, group, reinterpret_cast<uint32_t*>(to), reinterpret_cast<uint32_t*>(to + at.scales), reinterpret_cast<uint16_t*>(to + at.zeros));
    return (int)cudaGetLastError();
}

extern "C" int32_t glm53f_kda_proj_int4(const uint16_t* x, int64_t ldx, const void* packed, int32_t n, int32_t k, int32_t group, int32_t zeros, int32_t rows,
                                        void* out, int32_t out_f32, int64_t ldo, glm53f_stream_t stream) {
    using namespace kda;
    if (!shape_ok(n, k, group) || rows < 0 || ldx < k || ldx % 8 || ldo < n) return kInvalid;
    if (rows == 0) return 0;
    if (!on16(x) || !on16(packed) || out == nullptr || (reinterpret_cast<uintptr_t>(out) & (out_f32 ? 3 : 1))) return kInvalid;
    const Int4Layout at(n, k, group, zeros != 0);
    const auto* w = static_cast<const unsigned char*>(packed);
    int* status = status_word();
    if (status == nullptr) return (int)cudaErrorUnknown;
    const cudaStream_t on = reinterpret_cast<cudaStream_t>(stream);
    if (rows > kFewRows) {
        ManyParams m{};
        m.out = out, m.ldo = ldo, m.rows = rows, m.n = n, m.k = k, m.out_f32 = out_f32 != 0, m.group = group;
        m.scales = reinterpret_cast<const uint16_t*>(w + at.scales);
        m.tiles = (int)at.tiles, m.pieces = (int)at.pieces, m.groups = (int)at.groups;
        m.status = status;
        auto launch = [&](auto z) {
            constexpr bool Z = decltype(z)::value;
            if (rows <= 16) return many_launch<16, Z>(m, x, ldx, w, at, on);
            if (rows <= 32) return many_launch<32, Z>(m, x, ldx, w, at, on);
            if (rows <= 64) return many_launch<64, Z>(m, x, ldx, w, at, on);
            return many_launch<128, Z>(m, x, ldx, w, at, on);
        };
        return zeros ? launch(std::true_type{}) : launch(std::false_type{});
    }
    Int4Params p{};
    p.x = x, p.ldx = ldx, p.out = out, p.ldo = ldo, p.rows = rows, p.n = n, p.k = k, p.out_f32 = out_f32 != 0;
    p.codes = reinterpret_cast<const uint4*>(w), p.scales = reinterpret_cast<const uint32_t*>(w + at.scales), p.zeros = reinterpret_cast<const uint16_t*>(w + at.zeros);
    p.tiles = (int)at.tiles, p.pieces = (int)at.pieces, p.status = status;
    p.split = 1;
    while (p.split < kFewWarps && p.split * 4 <= p.pieces) p.split *= 2;
    const int x_bytes = (rows * (k + kRowPad) * 2 + 127) / 128 * 128;
    static_assert(kFewX / (2 * kFewRows) - kRowPad >= 2 * kFewWarps * kPiece, "rows that do not fit are long enough for all warps to share a tile");
    const bool longer = x_bytes > kFewX;
    p.x_bytes = longer ? 0 : x_bytes;
    const int abreast = kFewWarps / p.split, sms = sm_count();
    const long long want = (at.tiles + abreast - 1) / abreast;
    const unsigned blocks = (unsigned)(want < sms ? want : sms);
    auto launch = [&](auto g) {
        constexpr int G = decltype(g)::value;
        if (longer) return zeros ? few_launch<G, true, true>(p, blocks, on) : few_launch<G, false, true>(p, blocks, on);
        return zeros ? few_launch<G, true, false>(p, blocks, on) : few_launch<G, false, false>(p, blocks, on);
    };
    return group == 32   ? launch(std::integral_constant<int, 32>{})
           : group == 64 ? launch(std::integral_constant<int, 64>{})
                         : launch(std::integral_constant<int, 128>{});
}
