// Projections with 4-bit weights: out[r][o] = sum over k of x[r][k] s[o][k / G] (q[o][k] - z[o][k / G]), x bf16, q and z of 0 .. 15, s bf16, G of 32, 64 or 128.
//
// q - z is a whole number that bf16 holds, so the tensor cores' products are exact; a group's sum is formed in f32 and multiplied by its scale there.  No
// weight is rounded.
//
// The weight is laid out once (glm53f_kda_int4_pack) as the matrix instructions take it: tiles of 16 rows, in a tile pieces of 64 k, a piece 16 bytes for each
// lane of a warp, the four k steps' fragments a word each; in a word the pairs of neighbouring k lie 16 bits apart, so that a shift, a mask and one
// or put two of them into bf16s of 128 + q, from which 128 + z is taken.
//
// Few rows (this kernel): bound by HBM, the weights' bytes, and next to it by the seven operations that two words of weights cost.  A block an SM; the rows lie in its shared memory, its warps
// divide the k of a tile between them, pieces on their way in registers eight deep, across tiles; the warps' sums meet in shared memory once a tile.

#include <type_traits>

#include "common.cuh"
#include "glm53f_proj.h"
#include "kda_internal.h"

namespace kda {
namespace {

constexpr int kTile = 16;        // weight rows of a tile
constexpr int kPiece = 64;       // k of a piece
constexpr int kFewWarps = 16, kFewThreads = 32 * kFewWarps;
constexpr int kFewRows = 8;      // of x at a time
constexpr int kAhead = 8;        // pieces of a warp in flight
constexpr int kMostShared = 200 * 1024;  // for the rows of x
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
// The fragments of one k step: rows i (even registers) and i + 8, less lo and hi (128 + z in both halves).
__device__ __forceinline__ void widen(uint32_t w, uint32_t lo, uint32_t hi, uint32_t (&a)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = sub_bf16x2(((w >> (4 * j)) & 0x000f000fu) | 0x43004300u, j % 2 ? hi : lo);
}

// A piece on its way: its codes, the scales of its groups and their zero points.
template <int G, bool ZEROS>
struct Piece {
    static constexpr int N = G < kPiece ? kPiece / G : 1;
    uint4 codes;
    uint32_t scale[N];
    uint32_t zero[ZEROS ? N : 1];
};

template <int G, bool ZEROS>
__global__ void __launch_bounds__(kFewThreads, 1) int4_few_kernel(const Int4Params p) {
    using P = Piece<G, ZEROS>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float sums[2][kFewWarps][kTile * kFewRows];
    __shared__ __align__(16) uint4 nothing;  // what rows that are not there hold
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kw = warp % p.split, tw = warp / p.split, abreast = kFewWarps / p.split;  // this warp's part of k, its tile among those at a time
    const int per = (p.pieces + p.split - 1) / p.split;
    const int step = gridDim.x * abreast, tile0 = blockIdx.x * abreast + tw;
    const int groups = p.k / G, g = lane >> 2;
    grid_ready();

    // The next piece to load: its tile and place there.
    int ltile = tile0, li = 0;
    auto load = [&](P& x) {
        const int piece = kw + li * p.split;
        const bool ok = ltile < p.tiles && piece < p.pieces;
        if (ok) x.codes = __ldcs(p.codes + ((long long)ltile * p.pieces + piece) * 32 + lane);
        else x.codes = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int j = 0; j < P::N; ++j) {
            const long long at = ((long long)ltile * groups + (piece * kPiece + j * G) / G) * 8 + g;
            x.scale[j] = ok ? __ldg(p.scales + at) : 0u;
            if constexpr (ZEROS) x.zero[j] = ok ? (uint32_t)__ldg(p.zeros + at) : 0u;
        }
        if (++li == per) li = 0, ltile += step;
    };
    P ahead[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) load(ahead[u]);

    // The rows of x.
    const int pitch = (p.k + kRowPad) * 2;
    if (tid == 0) nothing = make_uint4(0u, 0u, 0u, 0u);
    for (int r = 0; r < p.rows; ++r)
        for (int i = tid; i < p.k / 8; i += kFewThreads)
            *reinterpret_cast<uint4*>(smem + r * pitch + i * 16) = __ldg(reinterpret_cast<const uint4*>(p.x + r * p.ldx) + i);
    __syncthreads();
    const int xr = lane & 7;
    const bool there = xr < p.rows;
    const uint32_t xrow = there ? smem_u32(smem + xr * pitch + (lane >> 3) * 16) : smem_u32(&nothing);

    float acc[4] = {};
    int i = 0, tile = tile0, buf = 0, round = 0;
    // Rounds: every warp of the block takes part in each, with or without a tile, as the barrier needs them.
    const int rounds = (p.tiles - (int)blockIdx.x * abreast + step - 1) / step;
    while (round < rounds) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (round < rounds) {
                const P x = ahead[u];
                load(ahead[u]);
                const int piece = kw + i * p.split;
                const uint32_t xat = there && piece < p.pieces ? xrow + piece * kPiece * 2 : smem_u32(&nothing), half = there && piece < p.pieces ? 64u : 0u;
                const uint32_t* w = reinterpret_cast<const uint32_t*>(&x.codes);
                constexpr int kSteps = 4 / P::N;  // of a group in the piece
                uint32_t b[4];
                float c[4] = {};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int j = s / kSteps;
                    uint32_t lo = 0x43084308u, hi = 0x43084308u;
                    if constexpr (ZEROS) {
                        lo = 0x43004300u | (x.zero[j] & 0xffu) * 0x00010001u;
                        hi = 0x43004300u | (x.zero[j] >> 8) * 0x00010001u;
                    }
                    uint32_t a[4];
                    widen(w[s], lo, hi, a);
                    if (s % 2 == 0) ldmatrix_4(xat + (s / 2) * half, b[0], b[1], b[2], b[3]);
                    mma(c, a, s % 2 ? b[2] : b[0], s % 2 ? b[3] : b[1]);
                    if (s % kSteps == kSteps - 1) {
                        const float s0 = __uint_as_float(x.scale[j] << 16), s1 = __uint_as_float(x.scale[j] & 0xffff0000u);
                        acc[0] = fmaf(s0, c[0], acc[0]), acc[1] = fmaf(s0, c[1], acc[1]);
                        acc[2] = fmaf(s1, c[2], acc[2]), acc[3] = fmaf(s1, c[3], acc[3]);
                        c[0] = c[1] = c[2] = c[3] = 0.0f;
                    }
                }
                if (++i == per) {
                    float* to = sums[buf][warp];
                    *reinterpret_cast<float2*>(to + g * kFewRows + 2 * (lane & 3)) = make_float2(acc[0], acc[1]);
                    *reinterpret_cast<float2*>(to + (g + 8) * kFewRows + 2 * (lane & 3)) = make_float2(acc[2], acc[3]);
                    acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
                    __syncthreads();
                    // (the next tile's sums go to the other buffer; this one is written again behind the next barrier)
                    for (int e = tid; e < abreast * kTile * kFewRows; e += kFewThreads) {
                        const int t = e / (kTile * kFewRows), in = e % (kTile * kFewRows), f = in % kTile, r = in / kTile;
                        const int o = (tile - tw + t) * kTile + f;
                        if (r >= p.rows || o >= p.n) continue;
                        float sum = 0.0f;
                        for (int q = 0; q < p.split; ++q) sum += sums[buf][t * p.split + q][f * kFewRows + r];
                        if (p.out_f32) static_cast<float*>(p.out)[r * p.ldo + o] = sum;
                        else static_cast<uint16_t*>(p.out)[r * p.ldo + o] = f32_to_bf16_bits(sum);
                    }
                    i = 0, tile += step, buf ^= 1, ++round;
                }
            }
        }
    }
}

// A thread a word of the packed weight, or a group's pair of scales and zero points.
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
    return n >= 1 && k >= kPiece && k % kPiece == 0 && k <= 65536 && (group == 32 || group == 64 || group == 128) && k % group == 0;
}
bool on16(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int G, bool ZEROS>
int few_launch(const Int4Params& p, unsigned blocks, int shared, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(int4_few_kernel<G, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e != cudaSuccess) return (int)e;
    return launch_early(int4_few_kernel<G, ZEROS>, dim3(blocks), kFewThreads, shared, stream, p);
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
    if (at.tiles > 0x3fffffff) return kInvalid;
    const auto* w = static_cast<const unsigned char*>(packed);
    Int4Params p{};
    p.ldx = ldx, p.ldo = ldo, p.n = n, p.k = k, p.out_f32 = out_f32 != 0;
    p.codes = reinterpret_cast<const uint4*>(w), p.scales = reinterpret_cast<const uint32_t*>(w + at.scales), p.zeros = reinterpret_cast<const uint16_t*>(w + at.zeros);
    p.tiles = (int)at.tiles, p.pieces = (int)at.pieces;
    p.split = 1;
    while (p.split < kFewWarps && p.split * 2 <= p.pieces) p.split *= 2;
    const int pitch = (k + kRowPad) * 2, fit = kMostShared / pitch, most = fit < kFewRows ? fit : kFewRows;  // rows of x that shared memory holds
    const int abreast = kFewWarps / p.split, sms = sm_count();
    const long long want = (at.tiles + abreast - 1) / abreast;
    const unsigned blocks = (unsigned)(want < sms ? want : sms);
    for (int r = 0; r < rows; r += most) {
        p.rows = rows - r < most ? rows - r : most;
        p.x = x + (long long)r * ldx;
        p.out = static_cast<unsigned char*>(out) + (long long)r * ldo * (out_f32 ? 4 : 2);
        auto launch = [&](auto g) {
            constexpr int G = decltype(g)::value;
            const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
            return zeros ? few_launch<G, true>(p, blocks, pitch * p.rows, s) : few_launch<G, false>(p, blocks, pitch * p.rows, s);
        };
        const int rc = group == 32   ? launch(std::integral_constant<int, 32>{})
                       : group == 64 ? launch(std::integral_constant<int, 64>{})
                                     : launch(std::integral_constant<int, 128>{});
        if (rc != 0) return rc;
    }
    return 0;
}
