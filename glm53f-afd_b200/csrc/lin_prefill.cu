// Linear attention with one decay a head: the prefill of packed sequences in chunks of 64 rows on the tensor cores.
//
//     S_t = e^g_t S_{t-1} + v_t k_t^T        y_t = scale S_t q_t
//
// With G_t the sum of a chunk's log decays up to and with row t, and S the state before the chunk (lane = value channel):
//     y_t  = scale (e^G_t S q_t + sum over s <= t of P_ts v_s),   P_ts = (q_t . k_s) e^(G_t - G_s)
//     S'   = e^G_63 S + sum over s of w_s v_s k_s^T,              w_s = e^(G_63 - G_s)
// so a chunk is four products: Q K^T, S Q^T, V^T P^T and (w V)^T K, all on operands as the tensor copies bring them (128-byte
// swizzle, K- or MN-major).  Bound by HBM where every SM has a chain, a sequence's head (1 KiB a row and head); a chain's own pace is the tensor pipe's.
//
// Precision.  Sums and the state are f32 in tensor memory, where the tensor core cuts each addition off: end states are 2e-7 to 1e-6 off, mostly too small, and 9e-6 after 4,000
// rows of hardly any decay.  What has to become an operand and is not bf16 already keeps more bits than that: w V
// goes as a sum of three bf16 parts where the state is f32 (24 bits, all that f32 has) and of two where it is stored as bf16, P as a sum of two (16 bits), S and
// scale e^G Q as f32 operands of which the tensor core takes 11 bits.  It cuts the rest off, always towards zero; the mean of both cuts is put back by q's factor (q_factor).  Outputs are then
// 1.67 to 1.69e-3 off 64 bits where their rounding to bf16 alone makes 1.66e-3, and 1e-5 too small on the mean (cut and left so 1.69 to 1.82e-3 and 1.6 to
// 6.6e-4; every value of q rounded to 11 bits instead the same, 64 heads x 8,192 rows 5 us longer; as single bf16 operands P and S would add as much as
// the rounding again).  Differences of G are of sums in 64 bits, held as two f32: a row that forgets everything (-inf, taken as
// -104, which is 0 in f32) must not blur those behind it.
//
// Roles of a block, one (sequence, head, segment) each, all meeting at mbarriers:
//   warps 0-3    P of a chunk out of the accumulator into shared memory (hi and lo)
//   warps 4-7    the outputs through transposing matrix stores to rows of 256 bytes
//   warps 8-11   scale e^G Q as f32
//   warps 12-19  the parts of w V^T into tensor memory; the rows of a last, short chunk to zero (what lies there may be NaN)
//   warps 20-27  the state, which is an operand of one product and the accumulator of the other: times e^G between the two
//   warp 28      tensor copies of q, k, v, three chunks ahead     warp 31  sums and factors of the decays
//   warp 29      the products with the state and to it            warp 30  the scores and their products with V
// A chunk's products take 1,920 cycles of the tensor pipe and, where every SM works, its rows 2,900 of a share of HBM; it takes 3,300 to 4,000.  What bounds it is what
// the other roles issue (2,200 instructions a scheduler) and the round of the state: its product with Q, its scaling, the sum of w V K, each of which waits
// for the one before.  So bodies are loops, waits sleep, and operands take the form that costs the fewest instructions.  148 heads x 4,096 rows take 145 us
// (69 of HBM's time), 64 heads x 8,192 rows in two segments 191 us (84), 8 heads x 65,536 in eighteen 202 us (82), by themselves over an evicted L2; call after call, inputs changing,
// the last two 210 and 227.  What was measured and is not here: w V^T through shared
// memory, the state's scaling in registers, registers moved between the roles, polling waits, a second buffer of q, half of q ahead, tiles brought to L2 before.
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
constexpr int kStages = 3, kStage = 3 * kTile;
constexpr int oQ = kStages * kStage;                    // scale e^G Q, f32: four boxes of 64 rows x 32 channels
constexpr int oP = oQ + 2 * kTile;                      // P: hi | lo, two buffers
constexpr int oY = oP + 4 * kBox;                       // half a chunk's outputs on their way out
struct Decays {
    float2 g[CH];     // G in powers of two: hi, lo
    float e[CH];      // scale e^G
    float w[CH];
    float all, pad[3];  // e^G of the whole chunk
};
constexpr int oDecays = oY + kTile / 2;
constexpr int oBars = oDecays + kStages * (int)sizeof(Decays);  // (a chunk's factors come and go with its rows)
enum : int {
    bFull = 0, bEmpty = bFull + kStages, bQK = bEmpty + kStages, bP, bReady, bState, bQS, bAdd = bQS + 2, bU = bAdd + 2, bO = bU + 2, bOFree = bO + 2, bClear = bOFree + 2, kBars
};
constexpr int oCtl = oBars + (kBars + 1) / 2 * 16;
constexpr int kSmem = oCtl + 16 + 1024;
static_assert(kSmem <= 232448 && sizeof(Decays) % 16 == 0, "shared memory");

constexpr int kOWarp = 4, kQWarp = 8, kVWarp = 12, kSWarp = 20, kCopyWarp = 28, kStateMmaWarp = 29, kScoreMmaWarp = 30, kDecayWarp = 31, kThreads = 32 * 32;
// Tensor memory columns: the state, the scores, two accumulators of outputs and two sets of w V^T in turn.
constexpr int cS = 0, cQK = 128, cO = 192, cWV = 320, kCols = 512;

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
    // Segments of seg_chunks chunks, one block each; in the pass that sums up states parts of part_chunks, one or two a segment.  What a part adds lies in a slot
    // of `states`, and how much of the state before it it leaves in `kept`; lin_join_kernel makes of a sequence's slots the states before its segments.
    int seg_chunks, part_chunks;
    int slots;  // of a head; 0: every sequence is one segment
    float *states, *kept;
    int* status;
};

// The block's work, r counting those of one head: (b, seg), found by each warp for itself.  Whole segments come first and then the sequences' rest, the longest
// first (within 32 sequences): blocks start in this order, and a long one that starts last would run alone.
template <bool STATE>
__device__ bool pick_work(const PrefillParams& p, int r, int lane, int& b, int& seg) {
    const int sub = p.seg_chunks / p.part_chunks;
    auto chunks_of = [&](int i) { return i < p.batch ? (p.cu[i + 1] - p.cu[i] + CH - 1) / CH : 0; };
    for (int g0 = 0; p.slots > 0 && g0 < p.batch; g0 += 32) {
        const int chunks = chunks_of(g0 + lane), mine = STATE ? max(chunks - 1, 0) / p.seg_chunks * sub : chunks / p.seg_chunks;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        const int all = __shfl_sync(0xffffffffu, upto, 31);
        if (r < all) {
            const int l = __ffs(__ballot_sync(0xffffffffu, upto > r)) - 1;
            b = g0 + l;
            seg = r - __shfl_sync(0xffffffffu, upto - mine, l);
            return true;
        }
        r -= all;
    }
    if (!STATE && p.slots == 0 && p.batch == 1) return true;
    for (int g0 = 0; !STATE && g0 < p.batch; g0 += 32) {
        const int chunks = chunks_of(g0 + lane), rest = chunks % p.seg_chunks;
        const int size = g0 + lane < p.batch && (rest > 0 || chunks == 0) ? rest : -1;  // (an empty sequence's state is handed on)
        const int all = __popc(__ballot_sync(0xffffffffu, size >= 0));
        if (r < all) {
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < 32; ++j) {
                const int other = __shfl_sync(0xffffffffu, size, j);
                rank += other > size || (other == size && j < lane);
            }
            const int l = __ffs(__ballot_sync(0xffffffffu, rank == r)) - 1;
            b = g0 + l;
            seg = __shfl_sync(0xffffffffu, chunks / p.seg_chunks, l);
            return true;
        }
        r -= all;
    }
    return false;
}
// A sequence's first slot: of a head's 2 (rows / segment's rows), enough for its segments' states and for two parts of each but the last.
__device__ __forceinline__ long long first_slot(const PrefillParams& p, int h, int first) {
    return (long long)h * p.slots + 2 * (first / (p.seg_chunks * CH));
}

__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, make_float2(-1.0f, -1.0f), a); }
__device__ __forceinline__ float2 lo_of(uint32_t hi, float2 x) {  // what a pair's hi parts leave
    return sub2(x, make_float2(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)));
}

// What the tensor core cuts off of an f32 operand's entries on the mean, of 11 bits taken: 2^-11 of an entry's power of two, so 2^-11 / (2 ln 2) of the entry where all mantissas are
// as likely on a logarithmic scale.
constexpr float kCutOff = 3.52e-4f;
// The factor of a row of q, scale e^G, with what makes up for the two cuts: of the state, unless it still is what came in as bf16 (`exact`), and of the products of factor and q, unless the
// factor has no more than the three bits that leave those in 11.
__device__ __forceinline__ float q_factor(float e, bool exact) {
    if (exact) return (__float_as_uint(e) & 0x1fffffu) == 0u ? e : e * (1.0f + kCutOff);
    return e * (1.0f + 2.0f * kCutOff);
}

// Shared-memory descriptors in the 128-byte swizzle (8-row groups 1,024 bytes apart): the low word from an address and the leading byte offset, which the
// products step through by adding to it.
__device__ __forceinline__ uint32_t desc_lo(uint32_t address, uint32_t leading) { return address >> 4 | leading >> 4 << 16; }
__device__ __forceinline__ uint64_t desc(uint32_t lo) {
    constexpr uint32_t hi = 1024 >> 4 | 1u << 14 | 2u << 29;
    return (uint64_t)hi << 32 | lo;
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
        for (int i = 0; i < kStages; ++i) mbar_init(&bar[bFull + i], 2), mbar_init(&bar[bEmpty + i], STATE ? 1 : 2);  // (full: the copies and the decays)
        mbar_init(&bar[bQK], 1);
        mbar_init(&bar[bP], 4);
        mbar_init(&bar[bReady], 5);  // q of a chunk (four warps), and the chunk before added to the state
        mbar_init(&bar[bState], 8);
        for (int i = 0; i < 2; ++i) mbar_init(&bar[bQS + i], 1), mbar_init(&bar[bAdd + i], STATE ? 8 : 16), mbar_init(&bar[bU + i], 1), mbar_init(&bar[bO + i], 1), mbar_init(&bar[bOFree + i], 4);
        mbar_init(&bar[bClear], 8);  // once, by the warps that clear a short last chunk's foreign rows
        ctl[0] = 0u;
        ctl[1] = 0u;
        mbar_init_fence();
    }
    if (warp == kStateMmaWarp) tc::tmem_alloc(tmem_slot, kCols);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tm = *tmem_slot;
    const WaitCtx ctx{ctl, ctl + 1, p.status};
    grid_ready();

    // The block's sequence and head and its chunks [c0, c0 + n).
    const int h = (int)blockIdx.x % p.heads;
    int b = 0, seg = 0;
    const bool idle = !pick_work<STATE>(p, (int)blockIdx.x / p.heads, lane, b, seg);
    b = (int)__reduce_max_sync(0xffffffffu, (unsigned)b);
    seg = (int)__reduce_max_sync(0xffffffffu, (unsigned)seg);
    const int first = p.cu[b], len = p.cu[b + 1] - first, seg_chunks = STATE ? p.part_chunks : p.seg_chunks;
    const int chunks = (len + CH - 1) / CH, c0 = seg * seg_chunks;
    const int n = max(0, min(seg_chunks, chunks - c0));
    const bool last_seg = c0 + n >= chunks;
    const int row0 = first + c0 * CH, rows = min(len - c0 * CH, n * CH);  // this block's rows
    auto arrive = [&](int i) {  // one arrival a warp, behind what its lanes have done
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[i]);
    };
    // A wait that sleeps in hardware first: the polling of mbar_wait by thirty warps is a third of what the block would issue.
    auto wait = [&](int i, uint32_t parity, int code) {
        return tc::warp_all(mbar_try_wait_hint(&bar[i], parity & 1u, 200000u) || mbar_wait(&bar[i], parity & 1u, ctx, code));
    };

    // The pass that only sums up states goes backwards: rows are then weighed by all that comes behind them in the segment, and nothing that has been
    // added is scaled again.  Its segments are whole ones.
    auto chunk_at = [&](int c) { return STATE ? n - 1 - c : c; };

    // The parts of w V^T, by eight warps: all chunks, or in the pass that only sums up states every other one (the warps that have no outputs to work on take the rest).
    auto weigh_values = [&](int vt, int first_chunk) {
        const int w = (vt >> 5) & 3, half = vt >> 7;
        const int parts = p.state_bf16 ? 2 : 3;
        for (int c = first_chunk; c < n; c += STATE ? 2 : 1) {
            // The products with these columns' last parts are through -- first, so that a chunk which this side skips is never the one the next barrier tells of.
            if (c > 1 && !wait(bU + (c & 1), c / 2 - 1, kStatusLinU)) return false;
            if (!wait(bFull + c % kStages, c / kStages, kStatusLinFull)) return false;
            const Decays& x = decays[c % kStages];
            unsigned char *k = smem + (c % kStages) * kStage + kTile, *v = k + kTile;
            const int live = rows - chunk_at(c) * CH;
            if (live < CH) {  // behind the sequence: another one's rows, or none
                for (int at = vt * 16; at < kTile; at += 256 * 16)
                    if (((at >> 7) & (CH - 1)) >= live) *reinterpret_cast<uint4*>(k + at) = *reinterpret_cast<uint4*>(v + at) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
                arrive(bClear);
            }
            tc::fence_after_sync();
#pragma unroll 1
            for (int sh = 0; sh < 2; ++sh) {
                uint32_t at = tc::tmem_addr(tm, w, cWV + 96 * (c & 1) + 16 * sh) + ((uint32_t)(16 * half) << 16), raw[8], part[8];
                float2 z[8];
                // V^T, value channels 32 w + 16 half + lane / 4 (+ 8): raw[2 i + 0 / 1] rows 32 sh + 8 i + 2 (lane % 4) and the next.
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 32 * sh + 16 * i + 8 * (lane >> 4) + (lane & 7), piece = 4 * w + 2 * half + ((lane >> 3) & 1);
                    tc::ldmatrix_t4(v + (piece >> 3) * kBox + r * 128 + (((piece & 7) ^ (r & 7)) << 4), raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]);
                }
                if (live < CH) {  // (whether or not the warp that clears these rows has been there; both products that read them wait: w V K for bAdd, V^T P^T for bClear)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 32 * sh + 8 * i + 2 * (lane & 3);
                        const uint32_t mask = (r < live ? 0xffffu : 0u) | (r + 1 < live ? 0xffff0000u : 0u);
                        raw[2 * i] &= mask, raw[2 * i + 1] &= mask;
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = *reinterpret_cast<const float2*>(&x.w[32 * sh + 8 * (i >> 1) + 2 * (lane & 3)]);
                    z[i] = mul2(f, make_float2(__uint_as_float(raw[i] << 16), __uint_as_float(raw[i] & 0xffff0000u)));
                }
#pragma unroll 1
                for (int j = 1; j < parts; ++j, at += 32) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        part[i] = tc::bf16x2(z[i].x, z[i].y);
                        z[i] = lo_of(part[i], z[i]);
                    }
                    tc::tmem_st_pairs(at, part);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) part[i] = tc::bf16x2(z[i].x, z[i].y);
                tc::tmem_st_pairs(at, part);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            arrive(bAdd + (c & 1));
        }
        return true;
    };

    if (idle) goto done;
    if (warp == kCopyWarp) {
        if (lane == 0) {
            for (int c = 0; c < n; ++c) {
                const int s = c % kStages, row = row0 + chunk_at(c) * CH, hq = h / p.share;
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
    } else if (warp == kStateMmaWarp) {
        constexpr uint32_t id_u = tc::idesc_bf16(128, 128, 0, 1, 0), id_s = tc::idesc_tf32(128, 64);
        const uint32_t leader = tc::elect_one();
        const int parts = p.state_bf16 ? 2 : 3;
        // As values that the compiler knows to be the same in all lanes: loops over them stay converged and the products' operands in uniform
        // registers.
        const int n_all = (int)__reduce_max_sync(0xffffffffu, (unsigned)n);
        const uint32_t tm_all = __reduce_max_sync(0xffffffffu, tm), base = __reduce_max_sync(0xffffffffu, smem_u32(smem));
        uint32_t stage = 0, phase = 0;
        for (int c = 0; c < n_all; ++c) {
            if (STATE && !wait(bFull + stage, phase, kStatusLinFull)) goto done;
            if (STATE && c == 0 && !wait(bState, 0, kStatusLinS)) goto done;  // (zeros)
            if (!STATE) {
                const uint32_t o = tm_all + cO + 64 * (c & 1);
                // (The state is there when its product with the chunk before has been waited for: one product's result as another's operand is not
                // in the order of their issue.)
                // (One barrier for all that this product waits for: each wait that is passed costs 200 cycles here.)
                if (c == 0) {
                    if (!wait(bState, 0, kStatusLinS)) goto done;
                    if (leader) mbar_arrive(&bar[bReady]);
                }
                if (!wait(bReady, c, kStatusLinQK)) goto done;
                tc::fence_after_sync();
                const uint32_t q32 = desc_lo(base + oQ, 16);
#pragma unroll
                for (int i = 0; i < DK / 8; ++i) tc::mma_tf32_ts_if(leader, o, tm_all + cS + 8 * i, desc(q32 + (i / 4) * (kBox >> 4) + 2 * (i % 4)), id_s, i > 0);
                tc::mma_commit_if(leader, &bar[bQS + (c & 1)]);  // (two in turn: their waiters may be a chunk apart)
            }
            if (!wait(bAdd + (c & 1), c / 2, kStatusLinWV)) goto done;
            tc::fence_after_sync();
            const uint32_t k = desc_lo(base + stage * kStage + kTile, kBox), wv = tm_all + cWV + 96 * (c & 1);
#pragma unroll 1
            for (int part = 0; part < parts; ++part)
#pragma unroll
                for (int i = 0; i < CH / 16; ++i) tc::mma_bf16_ts_if(leader, tm_all + cS, wv + 32 * part + 8 * i, desc(k + 128 * i), id_u, true);
            tc::mma_commit_if(leader, &bar[bEmpty + stage]);
            if (!STATE && c + 1 < n_all) tc::mma_commit_if(leader, &bar[bReady]);
            if (STATE && c + 1 == n_all) tc::mma_commit_if(leader, &bar[bQS]);  // (for the state's warps, which follow no chunk but the last)
            tc::mma_commit_if(leader, &bar[bU + (c & 1)]);  // (the last one: whoever has seen it has seen the others)
            if (++stage == kStages) stage = 0, phase ^= 1u;
            if (leader) ctl[0] = ctl[0] + 1u;
        }
    } else if (warp == kScoreMmaWarp) {
        constexpr uint32_t id_qk = tc::idesc_bf16(64, 64, 0, 0, 0), id_pv = tc::idesc_bf16(128, 64, 1, 0, 0);
        const uint32_t leader = tc::elect_one();
        const int n_all = STATE ? 0 : (int)__reduce_max_sync(0xffffffffu, (unsigned)n);
        const bool cut = __reduce_max_sync(0xffffffffu, (unsigned)(n * CH - rows)) != 0;  // the last chunk is a short one
        const uint32_t tm_all = __reduce_max_sync(0xffffffffu, tm), base = __reduce_max_sync(0xffffffffu, smem_u32(smem));
        uint32_t stage = 0, phase = 0, before = 0;  // of the scores; of the products with V, a chunk behind
        for (int c = 0; c <= n_all && n_all > 0; ++c) {
            if (c > 0 && !wait(bP, c - 1, kStatusLinP)) goto done;  // the scores have been read, and P is there
            if (c < n_all) {
                if (!wait(bFull + stage, phase, kStatusLinFull)) goto done;
                tc::fence_after_sync();
                const uint32_t q = desc_lo(base + stage * kStage, 16), k = q + (kTile >> 4);
#pragma unroll
                for (int i = 0; i < DK / 16; ++i) {
                    const uint32_t at = (i / 4) * (kBox >> 4) + 2 * (i % 4);
                    tc::mma_bf16_if(leader, tm_all + cQK, desc(q + at), desc(k + at), id_qk, i > 0);
                }
                tc::mma_commit_if(leader, &bar[bQK]);
            }
            if (c > 0) {
                if (!wait(bQS + ((c - 1) & 1), (c - 1) / 2, kStatusLinS)) goto done;  // which began the accumulator
                // P is 0 in the columns of foreign rows, but 0 times their NaN is not: they are cleared first.  (Nothing that arrives there waits for this product.)
                if (c == n_all && cut && !wait(bClear, 0, kStatusLinWV)) goto done;
                tc::fence_after_sync();
                const uint32_t v = desc_lo(base + before * kStage + 2 * kTile, kBox), o = tm_all + cO + 64 * ((c - 1) & 1);
                uint32_t pt = desc_lo(base + oP + ((c - 1) & 1) * 2 * kBox, 16);
#pragma unroll 1
                for (int part = 0; part < 2; ++part, pt += kBox >> 4)
#pragma unroll
                    for (int i = 0; i < CH / 16; ++i) tc::mma_bf16_if(leader, o, desc(v + 128 * i), desc(pt + 2 * i), id_pv, true);
                tc::mma_commit_if(leader, &bar[bEmpty + before]);
                tc::mma_commit_if(leader, &bar[bO + ((c - 1) & 1)]);
                before = before + 1 == kStages ? 0 : before + 1;
            }
            if (++stage == kStages) stage = 0, phase ^= 1u;
        }
    } else if (warp == kDecayWarp) {
        const float* g = p.g + (long long)row0 * p.g_stride + h;
        float next[2];
        auto fetch = [&](int c) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = chunk_at(c) * CH + 2 * lane + j;
                next[j] = r < rows ? __ldg(g + (long long)r * p.g_stride) : 0.0f;
            }
        };
        double total = 0.0;  // pass 1: of the segment's rows behind the chunk
        if (n > 0) fetch(0);
        for (int c = 0; c < n; ++c) {
            if (!wait(bEmpty + c % kStages, c / kStages + 1, kStatusLinDecay)) goto done;
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
            Decays& x = decays[c % kStages];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 2 * lane + j;
                const float hi = (float)sum[j];
                x.g[r] = make_float2(hi, (float)(sum[j] - (double)hi));
                x.e[r] = q_factor(p.scale * exp2f(hi), p.state_bf16 && c0 + c == 0);
                x.w[r] = exp2f((float)(STATE ? total + (all - sum[j]) : all - sum[j]));
            }
            if (lane == 0) x.all = exp2f((float)all);
            total += all;
            arrive(bFull + c % kStages);
        }
        if (STATE && lane == 0) p.kept[first_slot(p, h, first) + seg] = exp2f((float)total);
    } else if (STATE && warp < kQWarp) {
        if (!weigh_values(tid, 1)) goto done;
    } else if (warp < kOWarp) {
        if (!STATE) {
            const int w = warp, t_lo = 16 * w + (lane >> 2);
            const int row = 16 * w + 8 * ((lane >> 3) & 1) + (lane & 7);  // the matrix row that this lane names
            unsigned char* pt = smem + oP + row * 128;
            for (int j = w + 1; j < 4; ++j) {  // columns behind the warp's rows are all above the diagonal, in every chunk
                unsigned char* at = pt + (((2 * j + (lane >> 4)) ^ (row & 7)) << 4);
                for (int i = 0; i < 4; ++i) tc::stmatrix_4(at + i * kBox, 0u, 0u, 0u, 0u);
            }
            for (int c = 0; c < n; ++c) {
                if (!wait(bQK, c, kStatusLinQK)) goto done;  // (whoever issued the scores has seen the chunk's rows and decays arrive)
                tc::fence_after_sync();
                const Decays& x = decays[c % kStages];
                const float2 g_lo = x.g[t_lo], g_hi = x.g[t_lo + 8];
                unsigned char* mine = pt + (c & 1) * 2 * kBox;  // (the products that read this buffer last were issued before this chunk's scores: they are through)
#pragma unroll 2
                for (int j = 0; j <= w; ++j) {
                    uint32_t r[8], hi[4], lo[4];
                    tc::tmem_ld_frag(tc::tmem_addr(tm, w, cQK + 16 * j), r);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // columns 8 (i / 2) + 2 (lane % 4) and the next, rows t_lo + 8 (i % 2)
                        const int s = 16 * j + 8 * (i >> 1) + 2 * (lane & 3), t = t_lo + 8 * (i & 1);
                        const float4 gs = *reinterpret_cast<const float4*>(&x.g[s]);
                        const float2 gt = i & 1 ? g_hi : g_lo;
                        const float2 d0 = sub2(gt, make_float2(gs.x, gs.y)), d1 = sub2(gt, make_float2(gs.z, gs.w));
                        const float2 pv = mul2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), make_float2(ex2_ftz(d0.x + d0.y), ex2_ftz(d1.x + d1.y)));
                        const float2 z = mul2(make_float2(p.scale, p.scale), make_float2(s <= t ? pv.x : 0.0f, s + 1 <= t ? pv.y : 0.0f));
                        hi[i] = tc::bf16x2(z.x, z.y);
                        const float2 rest = lo_of(hi[i], z);
                        lo[i] = tc::bf16x2(rest.x, rest.y);
                    }
                    unsigned char* at = mine + (((2 * j + (lane >> 4)) ^ (row & 7)) << 4);
                    tc::stmatrix_4(at, hi[0], hi[1], hi[2], hi[3]);
                    tc::stmatrix_4(at + kBox, lo[0], lo[1], lo[2], lo[3]);
                }
                tc::fence_before_sync();
                fence_proxy_async_smem();
                arrive(bP);
            }
        }
    } else if (warp < kQWarp) {
        if (!STATE) {
            const int w = warp - kOWarp, ot = tid - 32 * kOWarp, t8 = ot >> 4, piece = ot & 15;
            unsigned char* y = smem + oY;
            const unsigned char* from = y + t8 * 256 + ((piece ^ t8) << 4);  // rows t8 + 8 i
            uint16_t* out = p.out + (long long)(row0 + t8) * p.out_stride + h * DV + piece * 8;
            const long long step = 8 * p.out_stride;
            for (int c = 0; c < n; ++c) {  // the accumulator's lanes are value channels, its columns rows
                bool ok = wait(bO + (c & 1), c / 2, kStatusLinO);
                tc::fence_after_sync();
#pragma unroll 1
                for (int rows32 = 0; rows32 < CH; rows32 += 32) {
                    if (!named_bar_all(1, 128, ok)) goto done;  // (and the rows before have left the staging)
#pragma unroll 2
                    for (int i = 0; i < 4; ++i) {
                        const int half = i >> 1, t0 = 16 * (i & 1);
                        uint32_t r[8];
                        tc::tmem_ld_frag(tc::tmem_addr(tm, w, cO + 64 * (c & 1) + rows32 + t0) + ((uint32_t)(16 * half) << 16), r);
                        tc::tmem_ld_wait();
                        uint32_t z[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = tc::bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                        const int t = t0 + 8 * (lane >> 4) + (lane & 7), to = 4 * w + 2 * half + ((lane >> 3) & 1);
                        tc::stmatrix_t4(y + t * 256 + ((to ^ (t & 7)) << 4), z[0], z[1], z[2], z[3]);
                    }
                    if (rows32) {
                        tc::fence_before_sync();
                        arrive(bOFree + (c & 1));
                    }
                    named_bar_sync(2, 128);
                    const int live = rows - c * CH - rows32 - t8;
#pragma unroll
                    for (int i = 0; i < 4; ++i, out += step)
                        if (8 * i < live) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(from + i * 2048);
                }
            }
        }
    } else if (warp < kVWarp) {
        if (!STATE) {
            // Chunk c's q, times scale e^G, as f32; a thread takes a piece of eight channels of every sixteenth row.
            // Eight lanes take four pieces each of two neighbouring rows, the halves crosswise, so that neither their loads nor their stores meet in a bank.
            const int qt = tid - 32 * kQWarp, l = qt & 7, r0 = 2 * (qt >> 4) + (l >> 2), sw = r0 & 7, piece = (l & 3) + 4 * ((l >> 2) ^ ((qt >> 3) & 1));
            unsigned char* to = smem + oQ + (piece >> 2) * kBox + r0 * 128;
            const int to0 = ((2 * (piece & 3)) ^ sw) << 4, to1 = ((2 * (piece & 3) + 1) ^ sw) << 4, from = r0 * 128 + ((piece ^ sw) << 4);
            for (int c = 0; c < n; ++c) {
                if (!wait(bFull + c % kStages, c / kStages, kStatusLinFull)) goto done;
                if (!wait(bOFree + (c & 1), c / 2 + 1, kStatusLinFree)) goto done;  // (the accumulator of the product that will wait for this)
                if (c > 0 && !wait(bQS + ((c - 1) & 1), (c - 1) / 2, kStatusLinQK)) goto done;
                const Decays& x = decays[c % kStages];
                const unsigned char* q = smem + (c % kStages) * kStage + from;
#pragma unroll 4
                for (int i = 0; i < 8; ++i) {
                    const uint4 in = *reinterpret_cast<const uint4*>(q + i * 2048);
                    const float f = x.e[16 * (i & 3) + r0];
                    const float2 e = make_float2(f, f);
                    unsigned char* at = to + 2 * (i >> 2) * kBox + (i & 3) * 2048;
                    const float2 a0 = mul2(e, make_float2(__uint_as_float(in.x << 16), __uint_as_float(in.x & 0xffff0000u)));
                    const float2 a1 = mul2(e, make_float2(__uint_as_float(in.y << 16), __uint_as_float(in.y & 0xffff0000u)));
                    const float2 a2 = mul2(e, make_float2(__uint_as_float(in.z << 16), __uint_as_float(in.z & 0xffff0000u)));
                    const float2 a3 = mul2(e, make_float2(__uint_as_float(in.w << 16), __uint_as_float(in.w & 0xffff0000u)));
                    *reinterpret_cast<float4*>(at + to0) = make_float4(a0.x, a0.y, a1.x, a1.y);
                    *reinterpret_cast<float4*>(at + to1) = make_float4(a2.x, a2.y, a3.x, a3.y);
                }
                fence_proxy_async_smem();
                arrive(bReady);
            }
        }
    } else if (warp < kSWarp) {
        if (!weigh_values(tid - 32 * kVWarp, 0)) goto done;
    } else if (warp < kCopyWarp) {  // the state: thread = value channel 32 (warp % 4) + lane, key channels 64 half ..
        const int quad = warp & 3, half = (warp - kSWarp) >> 2;
        const uint32_t at = tc::tmem_addr(tm, quad, cS + 64 * half);
        const int in_state = (32 * quad + lane) * DK + 64 * half;
        const bool from_segments = !STATE && p.slots > 0 && chunks > p.seg_chunks;
        float* mine = p.states + (first_slot(p, h, first) + seg) * (DK * DV) + in_state;
        const long long off = p.state_off[b] + (long long)h * DK * DV + in_state;
        const float* src32 = from_segments ? mine : static_cast<const float*>(p.state_in) + off;
        const uint16_t* src16 = static_cast<const uint16_t*>(p.state_in) + off;
        const bool wide = from_segments || !p.state_bf16, vec = ((wide ? reinterpret_cast<uintptr_t>(src32) : reinterpret_cast<uintptr_t>(src16)) & 15) == 0;
#pragma unroll 1
        for (int i = 0; i < 64; i += 16) {  // from memory
            uint32_t x[16];
            if (STATE) {
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = 0u;
            } else if (vec && wide) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 y = *reinterpret_cast<const uint4*>(src32 + i + 4 * j);
                    x[4 * j] = y.x, x[4 * j + 1] = y.y, x[4 * j + 2] = y.z, x[4 * j + 3] = y.w;
                }
            } else if (vec) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint4 y = *reinterpret_cast<const uint4*>(src16 + i + 8 * j);
                    const uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[8 * j + 2 * e] = u[e] << 16, x[8 * j + 2 * e + 1] = u[e] & 0xffff0000u;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = wide ? __float_as_uint(src32[i + j]) : (uint32_t)src16[i + j] << 16;
            }
            tc::tmem_st16(at + i, x);
        }
        tc::tmem_st_wait();
        tc::fence_before_sync();
        arrive(bState);
        for (int c = 0; c < n && !STATE; ++c) {
            // The chunk's outputs have read the state (and the chunk before has been added).
            if (!wait(bQS + (c & 1), c / 2, kStatusLinS)) goto done;
            const float all = decays[c % kStages].all;
            tc::fence_after_sync();
#pragma unroll 1
            for (int i = 0; i < 64; i += 32) {
                uint32_t x[32];
                tc::tmem_ld32(at + i, x);
                tc::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float2 z = mul2(make_float2(all, all), make_float2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
                    x[j] = __float_as_uint(z.x), x[j + 1] = __float_as_uint(z.y);
                }
                tc::tmem_st32(at + i, x);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            arrive(bAdd + (c & 1));
            if (warp == kSWarp && lane == 0) ctl[0] = ctl[0] + 1u;
        }
        if (n > 0 && !(STATE ? wait(bQS, 0, kStatusLinU) : wait(bU + ((n - 1) & 1), (n - 1) / 2, kStatusLinU))) goto done;  // (nobody leaves before the last product)
        tc::fence_after_sync();
        if (STATE || last_seg) {
            float* dst32 = STATE ? mine : static_cast<float*>(p.state_out) + off;
            uint16_t* dst16 = static_cast<uint16_t*>(p.state_out) + off;
            const bool wide_out = STATE || !p.state_bf16, vec_out = ((wide_out ? reinterpret_cast<uintptr_t>(dst32) : reinterpret_cast<uintptr_t>(dst16)) & 15) == 0;
#pragma unroll 1
            for (int i = 0; i < 64; i += 16) {
                uint32_t x[16];
                tc::tmem_ld16(at + i, x);
                tc::tmem_ld_wait();
                if (wide_out && vec_out) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) *reinterpret_cast<uint4*>(dst32 + i + j) = make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                } else if (wide_out) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) dst32[i + j] = __uint_as_float(x[j]);
                } else {
                    uint32_t y[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = tc::bf16x2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
                    if (vec_out) {
                        *reinterpret_cast<uint4*>(dst16 + i) = make_uint4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<uint4*>(dst16 + i + 8) = make_uint4(y[4], y[5], y[6], y[7]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) dst16[i + j] = (uint16_t)(y[j >> 1] >> (16 * (j & 1)));
                    }
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
    if (warp == kStateMmaWarp) tc::tmem_dealloc(tm, kCols);
}

// The state before each segment of the sequences that have more than one, from what their parts add: one thread for four entries of a state.
constexpr int kJoinThreads = 128, kJoinBlocks = DK * DV / 4 / kJoinThreads, kJoinAhead = 8;
__global__ void __launch_bounds__(kJoinThreads) lin_join_kernel(const __grid_constant__ PrefillParams p) {
    grid_ready();
    const int work = blockIdx.x / kJoinBlocks, h = work % p.heads, lane = threadIdx.x & 31;
    int r = work / p.heads, b = -1;
    for (int g0 = 0; g0 < p.batch; g0 += 32) {
        const int i = g0 + lane;
        const unsigned cut = __ballot_sync(0xffffffffu, i < p.batch && p.cu[i + 1] - p.cu[i] > p.seg_chunks * CH);
        const int all = __popc(cut);
        if (r < all) {
            b = g0 + (int)__fns(cut, 0, r + 1);
            break;
        }
        r -= all;
    }
    if (b < 0) return;
    const int at = ((int)(blockIdx.x % kJoinBlocks) * kJoinThreads + threadIdx.x) * 4;
    const int first = p.cu[b], chunks = (p.cu[b + 1] - first + CH - 1) / CH, sub = p.seg_chunks / p.part_chunks, parts = (chunks - 1) / p.seg_chunks * sub;
    const long long slot = first_slot(p, h, first);
    const long long off = p.state_off[b] + (long long)h * DK * DV + at;
    float4 s;
    if (p.state_bf16) {
        const uint16_t* src = static_cast<const uint16_t*>(p.state_in) + off;
        s = make_float4(bf16_bits_to_f32(src[0]), bf16_bits_to_f32(src[1]), bf16_bits_to_f32(src[2]), bf16_bits_to_f32(src[3]));
    } else {
        const float* src = static_cast<const float*>(p.state_in) + off;
        s = make_float4(src[0], src[1], src[2], src[3]);
    }
    float4* states = reinterpret_cast<float4*>(p.states + slot * (DK * DV) + at);
    const float* kept = p.kept + slot;
    // A segment's state takes a slot whose part has been read: segment i's comes behind the loads of parts up to i * sub at least.
    int seg = 0, in_seg = 0;
    for (int i = 0; i < parts; i += kJoinAhead) {
        float4 add[kJoinAhead];
        float d[kJoinAhead];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j)
            if (i + j < parts) add[j] = states[(long long)(i + j) * (DK * DV / 4)], d[j] = kept[i + j];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            if (i + j >= parts) break;
            if (in_seg == 0) states[(long long)seg * (DK * DV / 4)] = s, ++seg;
            if (++in_seg == sub) in_seg = 0;
            s = make_float4(fmaf(d[j], s.x, add[j].x), fmaf(d[j], s.y, add[j].y), fmaf(d[j], s.z, add[j].z), fmaf(d[j], s.w, add[j].w));
        }
    }
    states[(long long)seg * (DK * DV / 4)] = s;
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
int walk_launch(const PrefillParams& p, long long blocks, cudaStream_t stream) {
    static int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        const cudaError_t e = cudaFuncSetAttribute(lin_prefill_kernel<STATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return (int)e;
        configured_dev = dev;
    }
    return launch_early(lin_prefill_kernel<STATE>, dim3((unsigned)blocks), kThreads, kSmem, stream, p);
}

// Segments.  Were all sequences one block, the longest sequence's chunks would be the time where they are more than an SM's share of all chunks.  So the longest is
// cut into as many segments as there are SMs for it by that share, of kMinChunks chunks at least -- where that pays: a walk takes 2.0 us a chunk, the pass before it
// half that a chunk, and two more launches with the join as much as kExtraChunks chunks.  (Measured over an evicted L2: 8 heads x 1,024 rows 36 us in four segments
// and 41 whole; 8 x 512 rows 36 and 29, so whole; 64 x 1,024 rows 52 and 45, so whole; 8 x 2,048 rows 38 and 67.  Segments of two chunks
// take 4 us from 1,024 rows of one head and add 4 to 4,096 rows of four.)
constexpr int kMinChunks = 4, kExtraChunks = 7;
struct Segments {
    int seg_chunks, part_chunks;
    long long slots;  // of a head
};
Segments pick_segments(int heads, long long rows, int max_len, long long workspace_bytes) {
    const int chunks = (max_len + CH - 1) / CH;
    long long n = (long long)sm_count() * max_len / (heads * rows);
    n = n < chunks / kMinChunks ? n : chunks / kMinChunks;
    for (; n > 1; --n) {
        Segments x{};
        x.seg_chunks = (int)((chunks + n - 1) / n);
        const long long cuts = (rows - 1) / (x.seg_chunks * CH);  // segments that another one follows
        const int sub = cuts > 0 && heads * cuts * 2 <= sm_count() && x.seg_chunks >= 2 * kMinChunks ? 2 : 1;
        x.part_chunks = (x.seg_chunks + sub - 1) / sub;
        x.seg_chunks = x.part_chunks * sub;
        x.slots = 2 * (rows / (x.seg_chunks * CH));
        if (x.seg_chunks + x.part_chunks / 2 + kExtraChunks < chunks && heads * x.slots * (4ll * DK * DV + 4) <= workspace_bytes) return x;
    }
    return {(1 << 25) - 1, (1 << 25) - 1, 0};  // (every sequence whole, however long)
}

}  // namespace
}  // namespace kda

extern "C" int64_t glm53f_kda_lin_prefill_workspace_bytes(int32_t heads, int32_t batch, int32_t max_len) {
    using namespace kda;
    if (heads < 1 || heads > 65535 || batch < 1 || max_len < 1) return 0;
    // However many rows there are, a head's slots are twice the segments that SMs were counted for.
    const Segments x = pick_segments(heads, max_len, max_len, INT64_MAX);
    return x.slots > 0 ? 2ll * sm_count() * (4ll * DK * DV + 4) : 0;
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
    // A handful of rows a sequence: row by row, which is memory-bound over many chains and a row's latency over few.  (Measured over an evicted L2, rows against chunks:
    // 16 chains of 8 rows 14 and 16 us, of 16 rows 18 and 16; 512 chains of 32 rows 55 and 57 us, of 64 rows 117 and 59.)
    const long long waves = ((long long)heads * batch + sm_count() - 1) / sm_count();
    if (max_len <= 8 * (waves < 4 ? waves : 4))
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
    const Segments x = pick_segments(heads, rows, max_len, workspace_bytes);
    p.seg_chunks = x.seg_chunks;
    p.part_chunks = x.part_chunks;
    p.slots = (int)x.slots;
    if (x.slots == 0) return walk_launch<false>(p, (long long)heads * batch, stream);
    p.states = static_cast<float*>(workspace);
    p.kept = p.states + heads * x.slots * (DK * DV);
    const long long cuts = (rows - 1) / (x.seg_chunks * CH);
    int rc = walk_launch<true>(p, heads * cuts * (x.seg_chunks / x.part_chunks), stream);
    if (rc != 0) return rc;
    rc = launch_early(lin_join_kernel, dim3((unsigned)(heads * (cuts < batch ? cuts : batch) * kJoinBlocks)), kJoinThreads, 0, stream, p);
    if (rc != 0) return rc;
    return walk_launch<false>(p, heads * (cuts + batch), stream);
}
