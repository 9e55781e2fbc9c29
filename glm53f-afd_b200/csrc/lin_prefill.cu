// Linear attention with one decay a head: the prefill of packed sequences in chunks of 64 rows on the tensor cores.
//
//     S_t = e^g_t S_{t-1} + v_t k_t^T        y_t = scale S_t q_t
//
// With G_t the sum of a chunk's log decays up to and with row t, and S the state before the chunk (lane = value channel):
//     y_t  = scale (e^G_t S q_t + sum over s <= t of P_ts v_s),   P_ts = (q_t . k_s) e^(G_t - G_s)
//     S'   = e^G_63 S + sum over s of w_s v_s k_s^T,              w_s = e^(G_63 - G_s)
// so a chunk is four products: Q K^T, S Q^T, V^T P^T and (w V)^T K, all on operands as the tensor copies bring them (128-byte
// swizzle, K- or MN-major).  Bound by HBM where every SM has a chain (1 KiB a row and head); a chain's own pace is the tensor pipe's.
//
// Precision.  Sums are f32 in tensor memory, the state is f32 in registers.  What has to become a bf16 operand and is not one already goes
// as a sum of several: P and S as two (16 bits: beside an output's rounding to bf16 nothing is left of their errors; as one each
// they would add as much again), w V as three where the state is f32 (24 bits, all that f32 has) and as two where it is stored as
// bf16.  Differences of G are of sums in 64 bits, held as two f32: a row that forgets everything (-inf, taken as -104 a row, which
// is 0 in f32) must not blur those behind it.
//
// Roles of a block, one (chain, segment) each, all meeting at mbarriers:
//   warps 0-3    P of a chunk out of the accumulator into shared memory (hi and lo); the outputs of the one before: e^G_t and scale,
//                transposing matrix stores, rows of 256 bytes to global memory
//   warps 4-7    w V in parts, in V's own layout; the rows of a last, short chunk to zero (what lies there may be NaN)
//   warps 8-15   the state: 64 key channels of a value channel a thread; scaled, added to, split and given to the tensor core as an operand in
//                tensor memory
//   warp 16      tensor copies of q, k, v, two chunks ahead       warp 17  the products       warp 18  sums and factors of the decays
//
// Few chains: a sequence is cut into segments that are walked at the same time, each from the state that the segments before it
// leave.  That state comes from a pass over k and v alone (the state's product only), which writes what each segment adds from a zero
// state and how much of what was there it leaves; a small kernel runs along the segments.
//
// Every wait is bounded (codes 150-159 of the device status word); tensor memory is freed on every path.

#include <cuda.h>

#include "common.cuh"
#include "kda_internal.h"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace kda {
namespace {

constexpr int CH = 64;                                  // rows a chunk
constexpr int kTile = CH * DK * 2;                      // q, k or v of a chunk: two boxes of 64 rows x 128 bytes
constexpr int kBox = CH * 128;
constexpr int kStages = 2, kStage = 3 * kTile;
constexpr int oWV = kStages * kStage;                   // w V: three parts in V's layout
constexpr int oP = oWV + 3 * kTile;                     // P, two buffers of hi | lo
constexpr int oY = oP + 2 * 2 * kBox;                   // a chunk's outputs on their way out
constexpr int kDecays = 4;                              // chunks of decay factors in flight
struct Decays {
    float2 g[CH];     // G in powers of two: hi, lo
    float e[CH];      // scale e^G
    float w[CH];
    float all, pad[3];  // e^G of the whole chunk
};
constexpr int oDecays = oY + kTile;
constexpr int oBars = oDecays + kDecays * (int)sizeof(Decays);
enum : int { bFull = 0, bEmpty = bFull + kStages, bQK = bEmpty + kStages, bP = bQK + 2, bWV = bP + 2, bU, bUFree, bS, bO, bOFree, bDecay, bDecayFree = bDecay + kDecays, kBars = bDecayFree + kDecays };
constexpr int oCtl = oBars + kBars * 8;
constexpr int kSmem = oCtl + 16 + 1024;
static_assert(kSmem <= 232448 && sizeof(Decays) % 16 == 0, "shared memory");

constexpr int kPWarps = 4, kVWarps = 4, kSWarps = 8, kCopyWarp = 16, kMmaWarp = 17, kDecayWarp = 18, kThreads = 19 * 32;
constexpr int cQK = 0, cO1 = 128, cO2 = 192, cU = 256, cSHi = 384, cSLo = 448, kCols = 512;  // tensor memory columns

enum : int { kStatusLinFull = 150, kStatusLinEmpty, kStatusLinQK, kStatusLinP, kStatusLinWV, kStatusLinU, kStatusLinS, kStatusLinO, kStatusLinDecay, kStatusLinFree };

struct PrefillParams {
    alignas(64) CUtensorMap tm_q, tm_k, tm_v;  // (128, heads, rows), boxes of 64 rows x 64 channels
    int heads, share, batch;
    const int32_t* cu;
    const float* g;
    long long g_stride;
    const void* state_in;
    void* state_out;
    const long long* state_off;
    int state_bf16;
    float scale;
    uint16_t* out;
    long long out_stride;
    // Segments: `segments` of seg_chunks chunks a chain, one block each.  pass 0: a walk of the whole chain; 1: what a segment adds, for all but the last;
    // 2: with outputs, from the states that the segments before leave.
    int pass, segments, seg_chunks;
    float* states;  // [chain][segments][128 x 128]: pass 1 writes segment s's sum at s, lin_join_kernel makes it the state before segment s
    float* kept;    // [chain][segments]: how much of the state before it a segment leaves
    int* status;
};

__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, make_float2(-1.0f, -1.0f), a); }
__device__ __forceinline__ float2 lo_of(uint32_t hi, float2 x) {  // what a pair's hi parts leave
    return sub2(x, make_float2(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)));
}

// STATE: the pass that only sums up states.
template <bool STATE>
__global__ void __launch_bounds__(kThreads, 1) lin_prefill_kernel(const __grid_constant__ PrefillParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + oBars);
    Decays* decays = reinterpret_cast<Decays*>(smem + oDecays);
    volatile uint32_t* ctl = reinterpret_cast<volatile uint32_t*>(smem + oCtl);
    uint32_t* tmem_slot = const_cast<uint32_t*>(ctl) + 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&bar[bFull + i], 1), mbar_init(&bar[bEmpty + i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar[bQK + i], 1), mbar_init(&bar[bP + i], kPWarps);
        mbar_init(&bar[bWV], kVWarps);
        mbar_init(&bar[bU], 1);
        mbar_init(&bar[bUFree], kSWarps);
        mbar_init(&bar[bS], kSWarps);
        mbar_init(&bar[bO], 1);
        mbar_init(&bar[bOFree], kPWarps);
        for (int i = 0; i < kDecays; ++i) mbar_init(&bar[bDecay + i], 1), mbar_init(&bar[bDecayFree + i], kVWarps + kSWarps + (STATE ? 0 : kPWarps));
        ctl[0] = 0u;
        ctl[1] = 0u;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, kCols);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tm = *tmem_slot;
    const WaitCtx ctx{ctl, ctl + 1, p.status};
    grid_ready();

    // The block's chain and its chunks [c0, c0 + n).
    const int chain = (int)blockIdx.x / p.segments, seg = (int)blockIdx.x - chain * p.segments;
    const int b = chain / p.heads, h = chain - b * p.heads;
    const int first = p.cu[b], len = p.cu[b + 1] - first;
    const int chunks = (len + CH - 1) / CH, c0 = seg * p.seg_chunks;
    const int n = max(0, min(p.seg_chunks, chunks - c0));
    const bool last_seg = c0 + n >= chunks;
    const int row0 = first + c0 * CH, rows = min(len - c0 * CH, n * CH);  // this block's rows
    const bool idle = STATE ? last_seg : (n == 0 && seg > 0);
    auto arrive = [&](int i) {  // one arrival a warp, behind what its lanes have done
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[i]);
    };
    auto wait = [&](int i, uint32_t parity, int code) { return tc::warp_all(mbar_wait(&bar[i], parity & 1u, ctx, code)); };
    auto decay_wait = [&](int c) { return wait(bDecay + c % kDecays, c / kDecays, kStatusLinDecay); };

    if (idle) goto done;
    if (warp == kCopyWarp) {
        if (lane == 0) {
            for (int c = 0; c < n; ++c) {
                const int s = c % kStages, row = row0 + c * CH, hq = h / p.share;
                if (!mbar_wait(&bar[bEmpty + s], ((c / kStages) & 1) ^ 1u, ctx, kStatusLinEmpty)) goto done;
                unsigned char* st = smem + s * kStage;
                mbar_arrive_expect_tx(&bar[bFull + s], STATE ? 2 * kTile : 3 * kTile);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!STATE) tensor_load_3d(st + x * kBox, &p.tm_q, 64 * x, hq, row, &bar[bFull + s]);
                    tensor_load_3d(st + kTile + x * kBox, &p.tm_k, 64 * x, hq, row, &bar[bFull + s]);
                    tensor_load_3d(st + 2 * kTile + x * kBox, &p.tm_v, 64 * x, h, row, &bar[bFull + s]);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        constexpr uint32_t id_qk = tc::idesc_bf16(64, 64, 0, 0, 0), id_u = tc::idesc_bf16(128, 128, 1, 1, 0), id_s = tc::idesc_bf16(128, 64, 0, 0, 0),
                           id_pv = tc::idesc_bf16(128, 64, 1, 0, 0);
        const uint32_t leader = tc::elect_one();
        const int parts = p.state_bf16 ? 2 : 3;
        for (int c = 0; c < n; ++c) {
            const unsigned char *q = smem + (c % kStages) * kStage, *k = q + kTile, *v = k + kTile;
            if (!wait(bFull + c % kStages, c / kStages, kStatusLinFull)) goto done;
            tc::fence_after_sync();
            if (!STATE) {  // (its accumulator is free: P of the chunk two before was waited for)
#pragma unroll
                for (int i = 0; i < DK / 16; ++i)
                    tc::mma_bf16_if(leader, tm + cQK + 64 * (c & 1), tc::desc_sw128_kmajor(q, CH, 16 * i), tc::desc_sw128_kmajor(k, CH, 16 * i), id_qk, i > 0);
                tc::mma_commit_if(leader, &bar[bQK + (c & 1)]);
            }
            if (!wait(bWV, c, kStatusLinWV) || !wait(bUFree, c + 1, kStatusLinFree)) goto done;
            tc::fence_after_sync();
            for (int part = 0; part < parts; ++part)
#pragma unroll
                for (int i = 0; i < CH / 16; ++i)
                    tc::mma_bf16_if(leader, tm + cU, tc::desc_sw128_mnmajor(smem + oWV + part * kTile, CH, 16 * i), tc::desc_sw128_mnmajor(k, CH, 16 * i), id_u,
                                    part > 0 || i > 0);
            if (STATE) tc::mma_commit_if(leader, &bar[bEmpty + c % kStages]);
            tc::mma_commit_if(leader, &bar[bU]);
            if (!STATE) {
                if (!wait(bS, c, kStatusLinS) || !wait(bOFree, c + 1, kStatusLinFree)) goto done;
                tc::fence_after_sync();
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int i = 0; i < DK / 16; ++i)
                        tc::mma_bf16_ts_if(leader, tm + cO1, tm + (part ? cSLo : cSHi) + 8 * i, tc::desc_sw128_kmajor(q, CH, 16 * i), id_s, part > 0 || i > 0);
                if (!wait(bP + (c & 1), c / 2, kStatusLinP)) goto done;
                tc::fence_after_sync();
                const unsigned char* pt = smem + oP + (c & 1) * 2 * kBox;
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int i = 0; i < CH / 16; ++i)
                        tc::mma_bf16_if(leader, tm + cO2, tc::desc_sw128_mnmajor(v, CH, 16 * i), tc::desc_sw128_kmajor(pt + part * kBox, CH, 16 * i), id_pv, part > 0 || i > 0);
                tc::mma_commit_if(leader, &bar[bEmpty + c % kStages]);
                tc::mma_commit_if(leader, &bar[bO]);  // (the last one: whoever has seen it has seen the others)
            }
            if (leader) ctl[0] = ctl[0] + 1u;
        }
    } else if (warp == kDecayWarp) {
        const float* g = p.g + (long long)row0 * p.g_stride + h;
        float next[2];
        auto fetch = [&](int c) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = c * CH + 2 * lane + j;
                next[j] = r < rows ? __ldg(g + (long long)r * p.g_stride) : 0.0f;
            }
        };
        double total = 0.0;  // of the whole segment (pass 1)
        if (n > 0) fetch(0);
        for (int c = 0; c < n; ++c) {
            if (!wait(bDecayFree + c % kDecays, c / kDecays + 1, kStatusLinDecay)) goto done;
            double a[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) a[j] = (double)(next[j] < -104.0f ? -104.0f : next[j]) * 1.4426950408889634;
            if (c + 1 < n) fetch(c + 1);
            double upto = a[0] + a[1];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += o;
            }
            const double all = __shfl_sync(0xffffffffu, upto, 31), sum[2] = {upto - a[1], upto};
            Decays& x = decays[c % kDecays];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 2 * lane + j;
                const float hi = (float)sum[j];
                x.g[r] = make_float2(hi, (float)(sum[j] - (double)hi));
                x.e[r] = p.scale * exp2f(hi);
                x.w[r] = exp2f((float)(all - sum[j]));
            }
            if (lane == 0) x.all = exp2f((float)all);
            total += all;
            arrive(bDecay + c % kDecays);
        }
        if (STATE && lane == 0) p.kept[(long long)chain * p.segments + seg] = exp2f((float)total);
    } else if (warp < kPWarps) {
        if (!STATE) {
            const int w = warp;
            bool ok = true;
            // Chunk c's outputs: the accumulators' lanes are value channels, their columns rows.
            auto outputs = [&](int c) {
                ok = ok && wait(bO, c, kStatusLinO);
                if (!named_bar_all(1, kPWarps * 32, ok)) return false;  // (and the rows of the chunk before have left the staging)
                tc::fence_after_sync();
                const Decays& x = decays[c % kDecays];
                unsigned char* y = smem + oY;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int t0 = 0; t0 < CH; t0 += 16) {
                        uint32_t r1[8], r2[8];
                        const uint32_t at = tc::tmem_addr(tm, w, t0) + ((uint32_t)(16 * half) << 16);
                        tc::tmem_ld_frag(at + cO1, r1);
                        tc::tmem_ld_frag(at + cO2, r2);
                        tc::tmem_ld_wait();
                        uint32_t z[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {  // (two rows of a value channel: 8 (i / 2) + 2 (lane % 4) and the next)
                            const float2 e = *reinterpret_cast<const float2*>(&x.e[t0 + 8 * (i >> 1) + 2 * (lane & 3)]);
                            const float2 inner = mul2(make_float2(p.scale, p.scale), make_float2(__uint_as_float(r2[2 * i]), __uint_as_float(r2[2 * i + 1])));
                            const float2 v = fma2(e, make_float2(__uint_as_float(r1[2 * i]), __uint_as_float(r1[2 * i + 1])), inner);
                            z[i] = tc::bf16x2(v.x, v.y);
                        }
                        const int t = t0 + 8 * (lane >> 4) + (lane & 7), piece = 4 * w + 2 * half + ((lane >> 3) & 1);
                        tc::stmatrix_t4(y + t * 256 + ((piece ^ (t & 7)) << 4), z[0], z[1], z[2], z[3]);
                    }
                tc::fence_before_sync();
                arrive(bOFree);
                arrive(bDecayFree + c % kDecays);
                named_bar_sync(2, kPWarps * 32);
                uint16_t* out = p.out + (long long)(row0 + c * CH) * p.out_stride + h * DV;
#pragma unroll
                for (int i = 0; i < CH * 16 / (kPWarps * 32); ++i) {
                    const int t = i * (kPWarps * 2) + (tid >> 4), piece = tid & 15;
                    if (c * CH + t < rows)
                        *reinterpret_cast<uint4*>(out + (long long)t * p.out_stride + piece * 8) = *reinterpret_cast<const uint4*>(y + t * 256 + ((piece ^ (t & 7)) << 4));
                }
                return true;
            };
            for (int c = 0; c < n; ++c) {
                if (c > 0 && !outputs(c - 1)) goto done;
                ok = ok && wait(bQK + (c & 1), c / 2, kStatusLinQK) && decay_wait(c);
                if (!ok) continue;  // (the next vote ends it for all four warps)
                tc::fence_after_sync();
                const Decays& x = decays[c % kDecays];
                unsigned char* pt = smem + oP + (c & 1) * 2 * kBox;
                const int t_lo = 16 * w + (lane >> 2);
                const float2 g_lo = x.g[t_lo], g_hi = x.g[t_lo + 8];
                const int row = 16 * w + 8 * ((lane >> 3) & 1) + (lane & 7);  // the matrix row that this lane names
#pragma unroll
                for (int s0 = 0; s0 < CH; s0 += 16) {
                    uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
                    if (s0 <= 16 * w) {  // (columns behind the warp's rows are all above the diagonal)
                        uint32_t r[8];
                        tc::tmem_ld_frag(tc::tmem_addr(tm, w, cQK + 64 * (c & 1) + s0), r);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {  // columns 8 (i / 2) + 2 (lane % 4) and the next, rows t_lo + 8 (i % 2)
                            const int s = s0 + 8 * (i >> 1) + 2 * (lane & 3), t = t_lo + 8 * (i & 1);
                            const float4 gs = *reinterpret_cast<const float4*>(&x.g[s]);
                            const float2 gt = i & 1 ? g_hi : g_lo;
                            const float2 d0 = sub2(gt, make_float2(gs.x, gs.y)), d1 = sub2(gt, make_float2(gs.z, gs.w));
                            const float2 pv = mul2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), make_float2(ex2_ftz(d0.x + d0.y), ex2_ftz(d1.x + d1.y)));
                            const float2 z = make_float2(s <= t ? pv.x : 0.0f, s + 1 <= t ? pv.y : 0.0f);
                            hi[i] = tc::bf16x2(z.x, z.y);
                            const float2 rest = lo_of(hi[i], z);
                            lo[i] = tc::bf16x2(rest.x, rest.y);
                        }
                    }
                    unsigned char* at = pt + row * 128 + (((s0 / 8 + (lane >> 4)) ^ (row & 7)) << 4);
                    tc::stmatrix_4(at, hi[0], hi[1], hi[2], hi[3]);
                    tc::stmatrix_4(at + kBox, lo[0], lo[1], lo[2], lo[3]);
                }
                fence_proxy_async_smem();
                tc::fence_before_sync();
                arrive(bP + (c & 1));
            }
            if (n > 0 && !outputs(n - 1)) goto done;
        }
    } else if (warp < kPWarps + kVWarps) {
        const int vt = tid - kPWarps * 32;
        const bool three = !p.state_bf16;
        for (int c = 0; c < n; ++c) {
            if (!wait(bFull + c % kStages, c / kStages, kStatusLinFull) || !decay_wait(c)) goto done;
            if (c > 0 && !wait(bU, c - 1, kStatusLinU)) goto done;
            const Decays& x = decays[c % kDecays];
            unsigned char *k = smem + (c % kStages) * kStage + kTile, *v = k + kTile, *wv = smem + oWV;
            const int live = rows - c * CH;
#pragma unroll 2
            for (int i = 0; i < kTile / 16 / (kVWarps * 32); ++i) {
                const int at = (i * kVWarps * 32 + vt) * 16, r = (at >> 7) & (CH - 1);
                uint4 in = *reinterpret_cast<const uint4*>(v + at);
                if (r >= live) {  // behind the sequence: another one's rows, or none
                    in = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(v + at) = in;
                    *reinterpret_cast<uint4*>(k + at) = in;
                }
                const float w = x.w[r];
                const uint32_t pair[4] = {in.x, in.y, in.z, in.w};
                uint32_t part[3][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 z = mul2(make_float2(w, w), make_float2(__uint_as_float(pair[j] << 16), __uint_as_float(pair[j] & 0xffff0000u)));
                    part[0][j] = tc::bf16x2(z.x, z.y);
                    const float2 r1 = lo_of(part[0][j], z);
                    part[1][j] = tc::bf16x2(r1.x, r1.y);
                    const float2 r2 = lo_of(part[1][j], r1);
                    part[2][j] = tc::bf16x2(r2.x, r2.y);
                }
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (j < 2 || three) *reinterpret_cast<uint4*>(wv + j * kTile + at) = make_uint4(part[j][0], part[j][1], part[j][2], part[j][3]);
            }
            fence_proxy_async_smem();
            arrive(bWV);
            arrive(bDecayFree + c % kDecays);
        }
    } else {  // the state: thread = value channel 32 (warp % 4) + lane, key channels 64 half ..
        const int quad = warp & 3, half = (warp - kPWarps - kVWarps) >> 2, vc = 32 * quad + lane;
        const int in_state = vc * DK + 64 * half;
        float s[64];
        const bool from_segments = !STATE && p.pass == 2;
        float* mine = p.states + ((long long)chain * p.segments + seg) * (DK * DV) + in_state;
        const long long off = p.state_off[b] + (long long)h * DK * DV + in_state;
        if (STATE) {
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = 0.0f;
        } else if (from_segments || !p.state_bf16) {
            const float* src = from_segments ? mine : static_cast<const float*>(p.state_in) + off;
            if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(src + 4 * i);
                    s[4 * i] = x.x, s[4 * i + 1] = x.y, s[4 * i + 2] = x.z, s[4 * i + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] = src[i];
            }
        } else {
            const uint16_t* src = static_cast<const uint16_t*>(p.state_in) + off;
            if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * i);
                    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[8 * i + 2 * j] = __uint_as_float(u[j] << 16), s[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] = bf16_bits_to_f32(src[i]);
            }
        }
        auto give = [&]() {  // the state as an operand
#pragma unroll
            for (int i = 0; i < 64; i += 32) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float2 z = make_float2(s[i + 2 * j], s[i + 2 * j + 1]);
                    hi[j] = tc::bf16x2(z.x, z.y);
                    const float2 rest = lo_of(hi[j], z);
                    lo[j] = tc::bf16x2(rest.x, rest.y);
                }
                tc::tmem_st16(tc::tmem_addr(tm, quad, cSHi + 32 * half + i / 2), hi);
                tc::tmem_st16(tc::tmem_addr(tm, quad, cSLo + 32 * half + i / 2), lo);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            arrive(bS);
        };
        if (!STATE && n > 0) give();
        for (int c = 0; c < n; ++c) {
            if (!decay_wait(c) || !wait(bU, c, kStatusLinU)) goto done;
            tc::fence_after_sync();
            const float all = decays[c % kDecays].all;
#pragma unroll
            for (int i = 0; i < 64; i += 16) {
                uint32_t r[16];
                tc::tmem_ld16(tc::tmem_addr(tm, quad, cU + 64 * half + i), r);
                tc::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float2 z = fma2(make_float2(all, all), make_float2(s[i + j], s[i + j + 1]), make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])));
                    s[i + j] = z.x, s[i + j + 1] = z.y;
                }
            }
            tc::fence_before_sync();
            arrive(bUFree);
            arrive(bDecayFree + c % kDecays);
            if (!STATE && c + 1 < n) {
                if (!wait(bO, c, kStatusLinO)) goto done;  // the chunk's products have read the state before it
                tc::fence_after_sync();
                give();
            }
            if (warp == kPWarps + kVWarps && lane == 0) ctl[0] = ctl[0] + 1u;
        }
        if (STATE) {
#pragma unroll
            for (int i = 0; i < 16; ++i) *reinterpret_cast<float4*>(mine + 4 * i) = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
        } else if (last_seg && (n > 0 || seg == 0)) {
            if (!p.state_bf16) {
                float* dst = static_cast<float*>(p.state_out) + off;
                if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) dst[i] = s[i];
                }
            } else {
                uint16_t* dst = static_cast<uint16_t*>(p.state_out) + off;
                if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(tc::bf16x2(s[8 * i], s[8 * i + 1]), tc::bf16x2(s[8 * i + 2], s[8 * i + 3]),
                                                                           tc::bf16x2(s[8 * i + 4], s[8 * i + 5]), tc::bf16x2(s[8 * i + 6], s[8 * i + 7]));
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) dst[i] = f32_to_bf16_bits(s[i]);
                }
            }
        }
    }
done:
    // After an abort, copies into this block's shared memory may still be in flight: give them a bounded time.
    if (ctl[1]) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) tc::tmem_dealloc(tm, kCols);
}

// The state before each segment of a chain, from what the segments add: one thread for four entries of a state.  Segments that the sequence does not reach are
// left alone.
constexpr int kJoinThreads = 128, kJoinBlocks = DK * DV / 4 / kJoinThreads;
__global__ void __launch_bounds__(kJoinThreads) lin_join_kernel(const __grid_constant__ PrefillParams p) {
    grid_ready();
    const int chain = blockIdx.x / kJoinBlocks, b = chain / p.heads, h = chain - b * p.heads;
    const int at = ((int)(blockIdx.x % kJoinBlocks) * kJoinThreads + threadIdx.x) * 4;
    const int len = p.cu[b + 1] - p.cu[b], chunks = (len + CH - 1) / CH, used = max(1, (chunks + p.seg_chunks - 1) / p.seg_chunks);
    const long long off = p.state_off[b] + (long long)h * DK * DV + at;
    float4 s;
    if (p.state_bf16) {
        const uint16_t* src = static_cast<const uint16_t*>(p.state_in) + off;
        s = make_float4(bf16_bits_to_f32(src[0]), bf16_bits_to_f32(src[1]), bf16_bits_to_f32(src[2]), bf16_bits_to_f32(src[3]));
    } else {
        const float* src = static_cast<const float*>(p.state_in) + off;
        s = make_float4(src[0], src[1], src[2], src[3]);
    }
    float4* states = reinterpret_cast<float4*>(p.states + (long long)chain * p.segments * (DK * DV) + at);
    const float* kept = p.kept + (long long)chain * p.segments;
    for (int i = 0; i < used; ++i) {
        float4 add = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float d = i + 1 < used ? kept[i] : 0.0f;
        if (i + 1 < used) add = states[(long long)i * (DK * DV / 4)];
        states[(long long)i * (DK * DV / 4)] = s;
        s = make_float4(fmaf(d, s.x, add.x), fmaf(d, s.y, add.y), fmaf(d, s.z, add.z), fmaf(d, s.w, add.w));
    }
}

bool rows_map(CUtensorMap* tm, const void* base, int heads, long long rows, long long stride) {
    EncodeTiled enc = encode_tiled();
    if (enc == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)DK, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)DK * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)CH}, estr[3] = {1u, 1u, 1u};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool STATE>
int walk_launch(const PrefillParams& p, cudaStream_t stream) {
    static int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        const cudaError_t e = cudaFuncSetAttribute(lin_prefill_kernel<STATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return (int)e;
        configured_dev = dev;
    }
    return launch_early(lin_prefill_kernel<STATE>, dim3((unsigned)(p.heads * (long long)p.batch * p.segments)), kThreads, kSmem, stream, p);
}

// Segments of a chain: as many as give every SM a block, of eight chunks at least (a pass over fewer costs more than it saves).
int pick_segments(long long chains, int max_len) {
    const long long fit = sm_count() / (chains > 0 ? chains : 1), chunks = (max_len + CH - 1) / CH;
    long long n = chunks / 8 < fit ? chunks / 8 : fit;
    return n < 2 ? 1 : (int)n;
}
long long segment_bytes(long long chains, int segments) { return chains * segments * (4ll * DK * DV) + (chains * segments * 4 + 15) / 16 * 16; }

}  // namespace
}  // namespace kda

extern "C" int64_t glm53f_kda_lin_prefill_workspace_bytes(int32_t heads, int32_t batch, int32_t max_len) {
    using namespace kda;
    if (heads < 1 || heads > 65535 || batch < 1 || max_len < 1) return 0;
    const long long chains = (long long)heads * batch;
    const int n = pick_segments(chains, max_len);
    return n > 1 ? segment_bytes(chains, n) : 0;
}

extern "C" int glm53f_kda_lin_prefill_varlen(int32_t heads, int32_t qk_heads, int32_t batch, const int32_t* cu_rows, int32_t rows, int32_t max_len,
                                             const glm53f_bf16* q, int64_t q_stride, const glm53f_bf16* k, int64_t k_stride, const glm53f_bf16* v,
                                             int64_t v_stride, const float* g, int64_t g_stride, const void* state_in, void* state_out,
                                             const int64_t* state_off, int32_t state_bf16, float scale, glm53f_bf16* out, int64_t out_stride,
                                             void* workspace, int64_t workspace_bytes, glm53f_stream_t stream_) {
    using namespace kda;
    if (rows < 0 || max_len < 0 || max_len > rows || workspace_bytes < 0 || (workspace == nullptr && workspace_bytes > 0)) return kInvalid;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return kInvalid;
    if (!lin_args_ok(heads, qk_heads, batch, cu_rows, q, q_stride, k, k_stride, v, v_stride, g, g_stride, state_in, state_off, out, out_stride)) return kInvalid;
    if (batch == 0) return 0;
    if (state_out == nullptr || out == nullptr) return kInvalid;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (max_len <= 8)
        return lin_rows_launch(heads, qk_heads, batch, cu_rows, nullptr, q, q_stride, k, k_stride, v, v_stride, g, g_stride, state_in, state_out, state_off,
                               state_bf16 != 0, false, scale, out, out_stride, stream);
    PrefillParams p{};
    if (!rows_map(&p.tm_q, q, qk_heads, rows, q_stride) || !rows_map(&p.tm_k, k, qk_heads, rows, k_stride) || !rows_map(&p.tm_v, v, heads, rows, v_stride))
        return (int)cudaErrorNotSupported;
    p.heads = heads;
    p.share = heads / qk_heads;
    p.batch = batch;
    p.cu = cu_rows;
    p.g = g;
    p.g_stride = g_stride;
    p.state_in = state_in;
    p.state_out = state_out;
    p.state_off = reinterpret_cast<const long long*>(state_off);
    p.state_bf16 = state_bf16 != 0;
    p.scale = scale;
    p.out = out;
    p.out_stride = out_stride;
    p.status = status_word();
    if (p.status == nullptr) return (int)cudaErrorUnknown;
    const long long chains = (long long)heads * batch;
    const int chunks = (max_len + CH - 1) / CH;
    int n = pick_segments(chains, max_len);
    while (n > 1 && segment_bytes(chains, n) > workspace_bytes) --n;
    p.segments = n;
    p.seg_chunks = (chunks + n - 1) / n;
    p.segments = (chunks + p.seg_chunks - 1) / p.seg_chunks;
    if (p.segments <= 1) return walk_launch<false>(p, stream);
    p.states = static_cast<float*>(workspace);
    p.kept = p.states + chains * p.segments * (DK * DV);
    p.pass = 1;
    int rc = walk_launch<true>(p, stream);
    if (rc != 0) return rc;
    rc = launch_early(lin_join_kernel, dim3((unsigned)(chains * kJoinBlocks)), kJoinThreads, 0, stream, p);
    if (rc != 0) return rc;
    p.pass = 2;
    return walk_launch<false>(p, stream);
}
