// Gated linear recurrence, channel by channel: h_t = a_t h_{t-1} + c_t x_t, with a_t = e^g_t or the sigmoid of g_t, c_t = 1 or 1 - a_t.
//
// Row by row (decode), as a scan over packed sequences (prefill), and backwards: with e_t = a_{t+1} D_{t+1} the gradient that reaches row t from
// the rows behind it, D_t = dy_t + e_t, so e runs through the same recurrence from the other end; dx_t = c_t D_t and
// dg_t = D_t a'_t (h_{t-1} - [c = 1 - a] x_t), a' the gate's slope.
//
// Bound by HBM: a few operations a value, each value read once and written once.  Rows compose: over rows i..j the recurrence is
// h_j = A h_{i-1} + B with A the product of the a.  A tile is kRows rows of 64 channels; its values stay in registers (eight rows of two
// channels a thread, all loads in flight at once) while the warps' (A, B) meet in shared memory and the tile's in global memory, so a sequence is divided
// over the GPU and still read once: a tile says its (A, B), then looks back over those of the tiles before it to the nearest
// whose end state is known, and says its own.  Tiles are taken from a counter in their order, so whatever a tile waits for is with a block that
// runs already; the wait is bounded all the same (status 160, 161).
//
// The states between tiles come from one chain of h <- A h + B whatever a tile found ready: the same bits every time, with any workspace and beside any other request.

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "kda_internal.h"

namespace kda {
namespace {

constexpr int kChannels = 64;              // of a tile: two a lane
constexpr int kPer = 8;                    // rows of a thread
constexpr int kSave = 64;                  // rows between saved states
constexpr int kForwardWarps = 16, kBackwardWarps = 8;
constexpr int kForwardRows = kPer * kForwardWarps, kBackwardRows = kPer * kBackwardWarps;
static_assert(kForwardRows % kSave == 0 && kBackwardRows == kSave, "");

enum : int { kStatusScanBefore = 160, kStatusScanBehind = 161 };
enum : unsigned { kNothing = 0, kPart = 1, kWhole = 2 };  // what a tile has said

struct ScanParams {
    int channels, stripes, batch, rows, flags, vec;
    const int32_t* cu;
    const int32_t* keep;
    const void *g, *x, *dout;
    void *out, *dg, *dx;
    long long g_stride, x_stride, out_stride, dout_stride, dg_stride, dx_stride;
    const float* state_in;   // backward: the gradient of the end states, or none
    float* state_out;        // backward: the gradient of the start states, or none
    const long long* state_off;
    float* saves;
    // The workspace: [0] the counter, [1] whether somebody gave up, then what tiles said, their (A, B) and end states.
    unsigned* control;
    unsigned* said;
    float2* part;
    float* whole;
    long long tiles;
    int slots;
    int* status;
};

// Tile slots: sequence b's tiles of T rows lie at cu[b] / T + b and behind.  Every sequence has a slot at least, slots ascend with b, and rows / T + batch are enough.
__device__ __forceinline__ int slot_of(int first, int b, int tile_rows) { return first / tile_rows + b; }

// The sequence that slot lies in, by a converged warp: the last b with slot_of(cu[b], b) <= slot.
__device__ int sequence_of(const int32_t* cu, int batch, int slot, int tile_rows) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = batch;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const bool below = at < n && slot_of(__ldg(cu + lo + at), lo + at, tile_rows) <= slot;
        const int count = max(__popc(__ballot_sync(0xffffffffu, below)), 1);
        lo += (count - 1) * step;
        n = min(step, n - (count - 1) * step);
    }
    return lo;
}

__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void store_release(unsigned* p, unsigned v) { asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory"); }

// ---- values -------------------------------------------------------------------------------------------------------------------
// Two channels of a row, as loaded: bf16 pairs stay packed.
template <bool BF16>
struct Pair {
    float v[2];
    __device__ __forceinline__ float get(int i) const { return v[i]; }
};
template <>
struct Pair<true> {
    uint32_t v;
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i ? v & 0xffff0000u : v << 16); }
};
// Channels [at, at + valid) of a row; the others 0.
template <bool BF16>
__device__ __forceinline__ Pair<BF16> load_pair(const void* base, long long at, int valid, bool vec) {
    Pair<BF16> r;
    if constexpr (BF16) {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        if (vec) r.v = valid > 0 ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
        else r.v = (valid > 0 ? (uint32_t)__ldg(p) : 0u) | (valid > 1 ? (uint32_t)__ldg(p + 1) << 16 : 0u);
    } else {
        const float* p = static_cast<const float*>(base) + at;
        if (vec) {
            const float2 t = valid > 0 ? __ldg(reinterpret_cast<const float2*>(p)) : make_float2(0.0f, 0.0f);
            r.v[0] = t.x, r.v[1] = t.y;
        } else {
            r.v[0] = valid > 0 ? __ldg(p) : 0.0f, r.v[1] = valid > 1 ? __ldg(p + 1) : 0.0f;
        }
    }
    return r;
}
template <bool BF16>
__device__ __forceinline__ void store_pair(void* base, long long at, int valid, bool vec, float v0, float v1) {
    if (valid <= 0) return;
    if constexpr (BF16) {
        uint16_t* p = static_cast<uint16_t*>(base) + at;
        if (vec) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(v0, v1);
            *reinterpret_cast<__nv_bfloat162*>(p) = two;
        } else {
            p[0] = f32_to_bf16_bits(v0);
            if (valid > 1) p[1] = f32_to_bf16_bits(v1);
        }
    } else {
        float* p = static_cast<float*>(base) + at;
        if (vec) *reinterpret_cast<float2*>(p) = make_float2(v0, v1);
        else {
            p[0] = v0;
            if (valid > 1) p[1] = v1;
        }
    }
}

// a, and 1 - a without the cancellation where a is near one.  Of the sigmoid both from e^-|g|: no overflow, and the smaller one keeps its digits.
template <bool SIGMOID>
__device__ __forceinline__ void gate(float g, float& a, float& rest) {
    if constexpr (SIGMOID) {
        const float e = expf(-fabsf(g)), d = 1.0f + e;
        float r = rcp_approx(d);
        r = fmaf(r, fmaf(-d, r, 1.0f), r);  // (to half a step and a little)
        const float small = e * r;
        a = g < 0.0f ? small : r, rest = g < 0.0f ? r : small;
    } else {
        a = expf(g);
        rest = -expm1f(g);
    }
}

// ---- between tiles ------------------------------------------------------------------------------------------------------------
struct Link {  // a thread's channel of a tile: where its (A, B) and end state go
    const ScanParams& p;
    int half;  // which half of the stripe's channels: its two warps speak for themselves
    long long channel;

    __device__ __forceinline__ unsigned* said(int slot) const { return p.said + ((long long)slot * p.stripes * 2 + half); }
    __device__ __forceinline__ long long at(int slot) const { return (long long)slot * p.stripes * kChannels + channel; }
    __device__ __forceinline__ void say(int slot, unsigned what) const {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            __threadfence();
            store_release(said(slot), what);
        }
    }
};

// The state that reaches the tile in `slot` from the `count` > 0 tiles of its sequence before it (STEP -1) or behind it (STEP 1), by the converged warp of 32
// channels: the nearest known end state among the next 32 and the (A, B) from there on.
template <int STEP>
__device__ float look(const Link& k, int slot, int count) {
    const int lane = threadIdx.x & 31;
    const unsigned* mine = k.said(slot + STEP * (1 + min(lane, count - 1)));
    unsigned whole;
    uint64_t t0 = 0;
    for (int polls = 0;; ++polls) {
        const unsigned f = lane < count ? load_acquire(mine) : kNothing;
        whole = __ballot_sync(0xffffffffu, f == kWhole);
        const unsigned any = __ballot_sync(0xffffffffu, f != kNothing), nearer = whole ? (whole & -whole) - 1u : 0u;
        if (whole != 0 && (any & nearer) == nearer) break;
        if (polls % 64 == 63) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            const bool over = now - t0 > kWaitLimitNs, gone = load_acquire(k.p.control + 1) != 0;
            if (__any_sync(0xffffffffu, over || gone)) {
                if (lane == 0) {
                    atomicCAS(k.p.status, 0, STEP < 0 ? kStatusScanBefore : kStatusScanBehind);
                    store_release(k.p.control + 1, 1u);
                }
                return __int_as_float(0x7fc00000);
            }
        }
    }
    __syncwarp();
    const int from = __ffs(whole);
    float h = __ldcg(k.p.whole + k.at(slot + STEP * from));
#pragma unroll 4
    for (int i = from - 1; i > 0; --i) {
        const float2 ab = __ldcg(k.p.part + k.at(slot + STEP * i));
        h = fmaf(ab.x, h, ab.y);
    }
    return h;
}

// The tile's incoming state for this thread's channel, by the two warps of 64 channels: `first`: it starts its sequence's chain with `start`.  `more`: another tile waits for its end state.
template <int STEP>
__device__ float join(const Link& k, int slot, int count, float A, float B, float start, bool more) {
    if (count == 0) {
        if (more) {
            __stcg(k.p.whole + k.at(slot), fmaf(A, start, B));
            k.say(slot, kWhole);
        }
        return start;
    }
    if (more) {
        __stcg(k.p.part + k.at(slot), make_float2(A, B));
        k.say(slot, kPart);
    }
    const float h = look<STEP>(k, slot, count);
    if (more) {
        __stcg(k.p.whole + k.at(slot), fmaf(A, h, B));
        k.say(slot, kWhole);
    }
    return h;
}

__global__ void scan_clear_kernel(const ScanParams p) {
    grid_ready();
    const long long n = 4 + (long long)p.slots * p.stripes * 2;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) p.control[i] = 0u;
}

// Which tile a block is at.  LOOK: tiles come from the counter; otherwise the block walks its sequence's tiles, from the end that the pass starts at.
struct Place {
    int stripe, slot, b, first, n, tile, tiles;  // b < 0: no more
};
template <int T>
__device__ __forceinline__ void place_sequence(const ScanParams& p, Place& at) {
    at.first = min(max(__ldg(p.cu + at.b), 0), p.rows);
    at.n = max(min(__ldg(p.cu + at.b + 1), p.rows) - at.first, 0);
    at.tiles = max((at.n + T - 1) / T, 1);  // a sequence without rows has a tile all the same: its state passes through
}
// The counter's tile `ticket`, by a converged warp.  Sequences' tiles run forwards, or with REVERSE backwards, the stripes of channels fastest.
template <int T, bool REVERSE>
__device__ __forceinline__ void place_ticket(const ScanParams& p, unsigned ticket, Place& at) {
    at.b = -1;
    if (ticket >= p.tiles) return;
    at.stripe = (int)(ticket % p.stripes);
    const int i = (int)(ticket / p.stripes);
    at.slot = REVERSE ? p.slots - 1 - i : i;
    at.b = sequence_of(p.cu, p.batch, at.slot, T);
    place_sequence<T>(p, at);
    at.tile = at.slot - slot_of(at.first, at.b, T);
}
template <int T, bool REVERSE>
__device__ __forceinline__ void place_walk(const ScanParams& p, int walked, Place& at) {
    at.stripe = blockIdx.x % p.stripes;
    at.b = blockIdx.x / p.stripes;
    at.slot = 0;
    place_sequence<T>(p, at);
    at.tile = REVERSE ? at.tiles - 1 - walked : walked;
    if (walked >= at.tiles) at.b = -1;
}

// Calls f(sigmoid, complement) with the flags as compile-time constants.
template <typename F>
__device__ __forceinline__ void with_flags(int flags, F&& f) {
    using std::false_type, std::true_type;
    if (flags & GLM53F_KDA_SCAN_SIGMOID) {
        if (flags & GLM53F_KDA_SCAN_COMPLEMENT) f(true_type{}, true_type{});
        else f(true_type{}, false_type{});
    } else {
        if (flags & GLM53F_KDA_SCAN_COMPLEMENT) f(false_type{}, true_type{});
        else f(false_type{}, false_type{});
    }
}

// The blocks' loop over tiles: each(place, place_next) handles one and calls place_next between its loads and what needs them.
template <int T, int WARPS, bool LOOK, bool REVERSE, typename F>
__device__ __forceinline__ void for_tiles(const ScanParams& p, F&& each) {
    __shared__ Place place[2];
    const int lane = threadIdx.x & 31;
    const bool guide = threadIdx.x / 32 == WARPS - 1;
    unsigned ticket = 0;
    if (guide) {
        Place at;
        if constexpr (LOOK) {
            if (lane == 0) ticket = atomicAdd(p.control, 1u);
            const unsigned now = __shfl_sync(0xffffffffu, ticket, 0);
            if (lane == 0) ticket = atomicAdd(p.control, 1u);
            place_ticket<T, REVERSE>(p, now, at);
        } else {
            place_walk<T, REVERSE>(p, 0, at);
        }
        if (lane == 0) place[0] = at;
    }
    for (int i = 0;; ++i) {
        __syncthreads();
        const Place at = place[i & 1];
        if (at.b < 0) return;
        each(at, [&] {
            if (!guide) return;
            Place next;
            if constexpr (LOOK) {
                const unsigned now = __shfl_sync(0xffffffffu, ticket, 0);
                if (lane == 0) ticket = atomicAdd(p.control, 1u);
                place_ticket<T, REVERSE>(p, now, next);
            } else {
                place_walk<T, REVERSE>(p, i + 1, next);
            }
            if (lane == 0) place[(i + 1) & 1] = next;
        });
    }
}

template <bool LOOK, bool GB, bool XB>
__global__ void __launch_bounds__(kForwardWarps * 32, 2) scan_forward_kernel(const ScanParams p) {
    constexpr int T = kForwardRows;
    __shared__ float4 agg[kForwardWarps][32];
    __shared__ float carry[kChannels];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float walk = 0.0f;  // a walking block's state between its tiles, a channel a thread of the first two warps
    grid_ready();
    for_tiles<T, kForwardWarps, LOOK, false>(p, [&](const Place& at, auto&& place_next) {
        const int c0 = at.stripe * kChannels + 2 * lane, valid = min(p.channels - c0, 2), row0 = at.tile * T + warp * kPer;
        const int m = min(max(at.n - row0, 0), kPer);
        const long long row = (long long)at.first + row0;
        float a[kPer][2], b[kPer][2];
        {
            Pair<GB> g[kPer];
            Pair<XB> x[kPer];
#pragma unroll
            for (int r = 0; r < kPer; ++r) {
                const int v = r < m ? valid : 0;
                g[r] = load_pair<GB>(p.g, (row + r) * p.g_stride + c0, v, p.vec);
                x[r] = load_pair<XB>(p.x, (row + r) * p.x_stride + c0, v, p.vec);
            }
            place_next();
            if (at.tile >= at.tiles) return;  // a slot between two sequences
            with_flags(p.flags, [&](auto sigmoid, auto complement) {
#pragma unroll
                for (int r = 0; r < kPer; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float rest;
                        gate<decltype(sigmoid)::value>(g[r].get(i), a[r][i], rest);
                        b[r][i] = decltype(complement)::value ? rest * x[r].get(i) : x[r].get(i);
                        if (r >= m) a[r][i] = 1.0f, b[r][i] = 0.0f;  // rows past the end leave the state as it is
                    }
            });
        }
        float A[2] = {1.0f, 1.0f}, B[2] = {0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < kPer; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) A[i] *= a[r][i], B[i] = fmaf(a[r][i], B[i], b[r][i]);
        agg[warp][lane] = make_float4(A[0], B[0], A[1], B[1]);
        __syncthreads();
        if (warp < 2) {  // a channel a thread
            const int c = at.stripe * kChannels + tid;
            float TA = 1.0f, TB = 0.0f;
#pragma unroll
            for (int w = 0; w < kForwardWarps; ++w) {
                const float2 ab = reinterpret_cast<const float2*>(agg[w])[tid];
                TA *= ab.x, TB = fmaf(ab.x, TB, ab.y);
            }
            const long long off = p.state_off[at.b] + c;
            float h = at.tile == 0 && c < p.channels ? p.state_in[off] : walk;
            if constexpr (LOOK) h = join<-1>(Link{p, at.stripe * 2 + warp, c}, at.slot, at.tile, TA, TB, h, at.tile + 1 < at.tiles);
            else walk = fmaf(TA, h, TB);
            carry[tid] = h;
            if (at.n == 0 && c < p.channels) p.state_out[off] = h;
        }
        __syncthreads();
        float h[2] = {carry[2 * lane], carry[2 * lane + 1]};
        for (int w = 0; w < warp; ++w) {
            const float4 ab = agg[w][lane];
            h[0] = fmaf(ab.x, h[0], ab.y), h[1] = fmaf(ab.z, h[1], ab.w);
        }
        if (p.saves != nullptr && (warp * kPer) % kSave == 0 && (m > 0 || row0 == 0))
            store_pair<false>(p.saves, ((long long)slot_of(at.first, at.b, kSave) + row0 / kSave) * p.channels + c0, valid, p.channels % 2 == 0, h[0], h[1]);
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
            h[0] = fmaf(a[r][0], h[0], b[r][0]), h[1] = fmaf(a[r][1], h[1], b[r][1]);
            if (r < m && p.out != nullptr) store_pair<XB>(p.out, (row + r) * p.out_stride + c0, valid, p.vec, h[0], h[1]);
        }
        if (m > 0 && row0 + m == at.n) {
            float* s = p.state_out + p.state_off[at.b] + c0;
            if (valid > 0) s[0] = h[0];
            if (valid > 1) s[1] = h[1];
        }
    });
}

// As the forward pass from the other end, e in h's place: D_t = dy_t + e_t, e_{t-1} = a_t D_t.  The h of the tile's rows are formed again from the saved state at its start.
template <bool LOOK, bool GB, bool XB>
__global__ void __launch_bounds__(kBackwardWarps * 32, 2) scan_backward_kernel(const ScanParams p) {
    constexpr int T = kBackwardRows;
    __shared__ float4 agg[kBackwardWarps][32];  // as the forward pass
    __shared__ float2 back[kBackwardWarps][32];  // what the rows add to e
    __shared__ float carry[kChannels];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float walk = 0.0f;
    grid_ready();
    for_tiles<T, kBackwardWarps, LOOK, true>(p, [&](const Place& at, auto&& place_next) {
        const int c0 = at.stripe * kChannels + 2 * lane, valid = min(p.channels - c0, 2), row0 = at.tile * T + warp * kPer;
        const int m = min(max(at.n - row0, 0), kPer);
        const long long row = (long long)at.first + row0;
        Pair<GB> g[kPer];
        Pair<XB> x[kPer], dy[kPer];
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
            const int v = r < m ? valid : 0;
            g[r] = load_pair<GB>(p.g, (row + r) * p.g_stride + c0, v, p.vec);
            x[r] = load_pair<XB>(p.x, (row + r) * p.x_stride + c0, v, p.vec);
            dy[r] = load_pair<XB>(p.dout, (row + r) * p.dout_stride + c0, v, p.vec);
        }
        place_next();
        if (at.tile >= at.tiles) return;
        const long long save = ((long long)slot_of(at.first, at.b, kSave) + at.tile) * p.channels + c0;
        float before[2] = {valid > 0 ? __ldg(p.saves + save) : 0.0f, valid > 1 ? __ldg(p.saves + save + 1) : 0.0f};
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
            constexpr bool S = decltype(sigmoid)::value, C = decltype(complement)::value;
            float a[kPer][2], b[kPer][2];
            float A[2] = {1.0f, 1.0f}, B[2] = {0.0f, 0.0f}, F[2] = {0.0f, 0.0f};
#pragma unroll
            for (int r = 0; r < kPer; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float rest;
                    gate<S>(g[r].get(i), a[r][i], rest);
                    b[r][i] = C ? rest * x[r].get(i) : x[r].get(i);
                    if (r >= m) a[r][i] = 1.0f, b[r][i] = 0.0f;
                    A[i] *= a[r][i], B[i] = fmaf(a[r][i], B[i], b[r][i]);
                }
#pragma unroll
            for (int r = kPer - 1; r >= 0; --r)
#pragma unroll
                for (int i = 0; i < 2; ++i) F[i] = a[r][i] * (dy[r].get(i) + F[i]);
            agg[warp][lane] = make_float4(A[0], B[0], A[1], B[1]);
            back[warp][lane] = make_float2(F[0], F[1]);
            __syncthreads();
            if (warp < 2) {
                const int c = at.stripe * kChannels + tid;
                float TA = 1.0f, TF = 0.0f;
#pragma unroll
                for (int w = kBackwardWarps - 1; w >= 0; --w) {
                    const float wa = reinterpret_cast<const float2*>(agg[w])[tid].x;
                    TA *= wa, TF = fmaf(wa, TF, reinterpret_cast<const float*>(back[w])[tid]);
                }
                const long long off = p.state_off[at.b] + c;
                const bool last = at.tile + 1 == at.tiles, ok = c < p.channels;
                float e = last ? (ok && p.state_in != nullptr ? p.state_in[off] : 0.0f) : walk;
                if constexpr (LOOK) e = join<1>(Link{p, at.stripe * 2 + warp, c}, at.slot, at.tiles - 1 - at.tile, TA, TF, e, at.tile > 0);
                else walk = fmaf(TA, e, TF);
                carry[tid] = e;
                if (at.n == 0 && ok && p.state_out != nullptr) p.state_out[off] = e;
            }
            // Meanwhile: the states before this warp's rows, and before each of them.
            for (int w = 0; w < warp; ++w) {
                const float4 ab = agg[w][lane];
                before[0] = fmaf(ab.x, before[0], ab.y), before[1] = fmaf(ab.z, before[1], ab.w);
            }
#pragma unroll
            for (int r = 0; r < kPer; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float h = before[i];
                    before[i] = fmaf(a[r][i], h, b[r][i]);
                    b[r][i] = h;
                }
            __syncthreads();
            float e[2] = {carry[2 * lane], carry[2 * lane + 1]};
            for (int w = kBackwardWarps - 1; w > warp; --w) {
                const float4 ab = agg[w][lane];
                const float2 f = back[w][lane];
                e[0] = fmaf(ab.x, e[0], f.x), e[1] = fmaf(ab.z, e[1], f.y);
            }
#pragma unroll
            for (int r = kPer - 1; r >= 0; --r) {
                float dg[2], dx[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float d = dy[r].get(i) + e[i];
                    float rest = 1.0f, slope = a[r][i];
                    if constexpr (C || S) {
                        float again;
                        gate<S>(g[r].get(i), again, rest);
                    }
                    if constexpr (S) slope *= rest;
                    dx[i] = C ? rest * d : d;
                    dg[i] = d * slope * (C ? b[r][i] - x[r].get(i) : b[r][i]);
                    e[i] = a[r][i] * d;
                }
                if (r < m) {
                    store_pair<XB>(p.dx, (row + r) * p.dx_stride + c0, valid, p.vec, dx[0], dx[1]);
                    store_pair<GB>(p.dg, (row + r) * p.dg_stride + c0, valid, p.vec, dg[0], dg[1]);
                }
            }
            if (row0 == 0 && m > 0 && p.state_out != nullptr) {
                float* s = p.state_out + p.state_off[at.b] + c0;
                if (valid > 0) s[0] = e[0];
                if (valid > 1) s[1] = e[1];
            }
        });
    });
}

// Row by row, two channels a thread, eight rows' loads in flight.
constexpr int kStepThreads = 128;
template <bool GB, bool XB>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(const ScanParams p) {
    grid_ready();
    const int parts = (p.channels + 2 * kStepThreads - 1) / (2 * kStepThreads);
    const int b = blockIdx.x / parts, c0 = (int)(blockIdx.x % parts) * 2 * kStepThreads + 2 * (int)threadIdx.x, valid = min(p.channels - c0, 2);
    if (valid <= 0) return;
    const int first = __ldg(p.cu + b);
    int n = max(__ldg(p.cu + b + 1) - first, 0);
    if (p.keep != nullptr) n = min(n, max(__ldg(p.keep + b), 0));
    const long long off = p.state_off[b] + c0;
    float h[2] = {p.state_in[off], valid > 1 ? p.state_in[off + 1] : 0.0f};
    for (int t = 0; t < n; t += kPer) {
        Pair<GB> g[kPer];
        Pair<XB> x[kPer];
        const long long row = (long long)first + t;
        const int m = min(n - t, kPer);
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
            const int v = r < m ? valid : 0;
            g[r] = load_pair<GB>(p.g, (row + r) * p.g_stride + c0, v, p.vec);
            x[r] = load_pair<XB>(p.x, (row + r) * p.x_stride + c0, v, p.vec);
        }
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
#pragma unroll
            for (int r = 0; r < kPer; ++r) {
                if (r >= m) break;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float a, rest;
                    gate<decltype(sigmoid)::value>(g[r].get(i), a, rest);
                    h[i] = fmaf(a, h[i], decltype(complement)::value ? rest * x[r].get(i) : x[r].get(i));
                }
                if (p.out != nullptr) store_pair<XB>(p.out, (row + r) * p.out_stride + c0, valid, p.vec, h[0], h[1]);
            }
        });
    }
    if (p.state_out != nullptr) {
        p.state_out[off] = h[0];
        if (valid > 1) p.state_out[off + 1] = h[1];
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
constexpr int kAllFlags = GLM53F_KDA_SCAN_SIGMOID | GLM53F_KDA_SCAN_COMPLEMENT | GLM53F_KDA_SCAN_G_BF16 | GLM53F_KDA_SCAN_X_BF16;

struct Layout {  // of the workspace: bytes from its start
    long long slots, stripes, said, part, whole, bytes;
    Layout(int64_t channels, int64_t batch, int64_t rows, int tile_rows) {
        slots = rows / tile_rows + batch;
        stripes = (channels + kChannels - 1) / kChannels;
        auto up = [](long long x) { return (x + 255) / 256 * 256; };
        said = 16;
        part = up(said + slots * stripes * 2 * 4);
        whole = part + slots * stripes * kChannels * 8;
        bytes = whole + slots * stripes * kChannels * 4;
    }
};

bool even(const void* p, bool bf16) { return (reinterpret_cast<uintptr_t>(p) & (bf16 ? 3 : 7)) == 0; }
bool aligned(const void* p, bool bf16) { return (reinterpret_cast<uintptr_t>(p) & (bf16 ? 1 : 3)) == 0; }

// One matrix of rows: acceptable at all, and whether two channels of it are one access.
struct Matrix {
    const void* p;
    int64_t stride;
    bool bf16;
};
bool matrices_ok(const ScanParams& p, std::initializer_list<Matrix> all, int& vec) {
    vec = p.channels % 2 == 0;
    for (const Matrix& m : all) {
        if (m.p == nullptr || !aligned(m.p, m.bf16) || m.stride < p.channels) return false;
        vec = vec && m.stride % 2 == 0 && even(m.p, m.bf16);
    }
    return true;
}

// Starts LAUNCH(look, gb, xb) with the flags as constants.
template <typename F>
int with_types(int flags, bool look, F&& f) {
    using std::false_type, std::true_type;
    auto types = [&](auto l) {
        if (flags & GLM53F_KDA_SCAN_G_BF16) return flags & GLM53F_KDA_SCAN_X_BF16 ? f(l, true_type{}, true_type{}) : f(l, true_type{}, false_type{});
        return flags & GLM53F_KDA_SCAN_X_BF16 ? f(l, false_type{}, true_type{}) : f(l, false_type{}, false_type{});
    };
    return look ? types(true_type{}) : types(false_type{});
}

// The launch over tiles: with sequences of more than one tile and a workspace that holds what tiles say, taken from the counter; else a block walks each (sequence, stripe).
template <bool BACKWARD>
int tiles_launch(ScanParams& p, int max_len, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    constexpr int T = BACKWARD ? kBackwardRows : kForwardRows, threads = 32 * (BACKWARD ? kBackwardWarps : kForwardWarps);
    const Layout at(p.channels, p.batch, p.rows, T);
    p.stripes = (int)at.stripes;
    const bool look = max_len > T && workspace != nullptr && workspace_bytes >= at.bytes;
    if (at.stripes * p.batch > 0x7fffffff || at.slots * at.stripes > 0x7fffffff) return kInvalid;
    long long blocks = at.stripes * p.batch;
    if (look) {
        p.status = status_word();
        if (p.status == nullptr) return (int)cudaErrorUnknown;
        auto* w = static_cast<unsigned char*>(workspace);
        p.control = reinterpret_cast<unsigned*>(w);
        p.said = reinterpret_cast<unsigned*>(w + at.said);
        p.part = reinterpret_cast<float2*>(w + at.part);
        p.whole = reinterpret_cast<float*>(w + at.whole);
        p.slots = (int)at.slots;
        p.tiles = at.slots * at.stripes;
        const long long words = 4 + at.slots * at.stripes * 2, clear = (words + 255) / 256;
        const int rc = launch_early(scan_clear_kernel, dim3((unsigned)(clear < 512 ? clear : 512)), 256, 0, stream, p);
        if (rc != 0) return rc;
        const long long most = 2ll * sm_count();
        blocks = p.tiles < most ? p.tiles : most;
    }
    return with_types(p.flags, look, [&](auto l, auto gb, auto xb) {
        constexpr bool L = decltype(l)::value, G = decltype(gb)::value, X = decltype(xb)::value;
        if constexpr (BACKWARD) return launch_early(scan_backward_kernel<L, G, X>, dim3((unsigned)blocks), threads, 0, stream, p);
        else return launch_early(scan_forward_kernel<L, G, X>, dim3((unsigned)blocks), threads, 0, stream, p);
    });
}

// What every call needs; rows < 0: a call that does not say how many there are.
bool common_ok(int32_t channels, int32_t batch, const int32_t* cu, int32_t flags) {
    return channels >= 1 && batch >= 0 && (flags & ~kAllFlags) == 0 && (batch == 0 || cu != nullptr);
}
bool state_ok(const void* state) { return state != nullptr && (reinterpret_cast<uintptr_t>(state) & 3) == 0; }

}  // namespace
}  // namespace kda

extern "C" int64_t glm53f_kda_scan_workspace_bytes(int32_t channels, int32_t batch, int32_t rows) {
    using namespace kda;
    if (channels < 1 || batch < 1 || rows < 0) return 0;
    const Layout f(channels, batch, rows, kForwardRows), b(channels, batch, rows, kBackwardRows);
    return f.bytes > b.bytes ? f.bytes : b.bytes;
}

extern "C" int64_t glm53f_kda_scan_saves_rows(int32_t batch, int32_t rows) { return batch < 1 || rows < 0 ? 0 : (int64_t)rows / kda::kSave + batch; }

extern "C" int glm53f_kda_scan_decode_batch(int32_t channels, int32_t batch, const int32_t* cu_rows, const int32_t* keep, const void* g, int64_t g_stride,
                                            const void* x, int64_t x_stride, int32_t flags, const float* state_in, float* state_out, const int64_t* state_off,
                                            void* out, int64_t out_stride, glm53f_stream_t stream) {
    using namespace kda;
    if (!common_ok(channels, batch, cu_rows, flags)) return kInvalid;
    if (batch == 0) return 0;
    ScanParams p{};
    p.channels = channels, p.batch = batch, p.flags = flags, p.cu = cu_rows, p.keep = keep;
    p.g = g, p.g_stride = g_stride, p.x = x, p.x_stride = x_stride, p.out = out, p.out_stride = out_stride;
    p.state_in = state_in, p.state_out = state_out, p.state_off = reinterpret_cast<const long long*>(state_off);
    const bool gb = flags & GLM53F_KDA_SCAN_G_BF16, xb = flags & GLM53F_KDA_SCAN_X_BF16;
    const Matrix mg{g, g_stride, gb}, mx{x, x_stride, xb}, mo = out != nullptr ? Matrix{out, out_stride, xb} : mx;
    if (!matrices_ok(p, {mg, mx, mo}, p.vec) || !state_ok(state_in) || state_off == nullptr || (state_out == nullptr && out == nullptr)) return kInvalid;
    if (state_out != nullptr && !state_ok(state_out)) return kInvalid;
    const long long blocks = (long long)batch * ((channels + 2 * kStepThreads - 1) / (2 * kStepThreads));
    if (blocks > 0x7fffffff) return kInvalid;
    return with_types(flags, false, [&](auto, auto g_bf16, auto x_bf16) {
        return launch_early(scan_step_kernel<decltype(g_bf16)::value, decltype(x_bf16)::value>, dim3((unsigned)blocks), kStepThreads, 0,
                            reinterpret_cast<cudaStream_t>(stream), p);
    });
}

extern "C" int glm53f_kda_scan_prefill_varlen(int32_t channels, int32_t batch, const int32_t* cu_rows, int32_t rows, int32_t max_len, const void* g,
                                              int64_t g_stride, const void* x, int64_t x_stride, int32_t flags, const float* state_in, float* state_out,
                                              const int64_t* state_off, void* out, int64_t out_stride, float* saves, void* workspace, int64_t workspace_bytes,
                                              glm53f_stream_t stream) {
    using namespace kda;
    if (!common_ok(channels, batch, cu_rows, flags) || rows < 0 || max_len < 0 || max_len > rows || workspace_bytes < 0) return kInvalid;
    if (batch == 0) return 0;
    ScanParams p{};
    p.channels = channels, p.batch = batch, p.rows = rows, p.flags = flags, p.cu = cu_rows;
    p.g = g, p.g_stride = g_stride, p.x = x, p.x_stride = x_stride, p.out = out, p.out_stride = out_stride, p.saves = saves;
    p.state_in = state_in, p.state_out = state_out, p.state_off = reinterpret_cast<const long long*>(state_off);
    const bool gb = flags & GLM53F_KDA_SCAN_G_BF16, xb = flags & GLM53F_KDA_SCAN_X_BF16;
    const Matrix mg{g, g_stride, gb}, mx{x, x_stride, xb}, mo = out != nullptr ? Matrix{out, out_stride, xb} : mx;
    if (!matrices_ok(p, {mg, mx, mo}, p.vec) || !state_ok(state_in) || !state_ok(state_out) || state_off == nullptr) return kInvalid;
    if ((reinterpret_cast<uintptr_t>(saves) & 7) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return kInvalid;
    return tiles_launch<false>(p, max_len, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int glm53f_kda_scan_backward_varlen(int32_t channels, int32_t batch, const int32_t* cu_rows, int32_t rows, int32_t max_len, const void* g,
                                               int64_t g_stride, const void* x, int64_t x_stride, int32_t flags, const float* saves, const void* dout,
                                               int64_t dout_stride, const float* dstate, float* dstate_in, const int64_t* state_off, void* dg,
                                               int64_t dg_stride, void* dx, int64_t dx_stride, void* workspace, int64_t workspace_bytes,
                                               glm53f_stream_t stream) {
    using namespace kda;
    if (!common_ok(channels, batch, cu_rows, flags) || rows < 0 || max_len < 0 || max_len > rows || workspace_bytes < 0) return kInvalid;
    if (batch == 0) return 0;
    ScanParams p{};
    p.channels = channels, p.batch = batch, p.rows = rows, p.flags = flags, p.cu = cu_rows;
    p.g = g, p.g_stride = g_stride, p.x = x, p.x_stride = x_stride, p.dout = dout, p.dout_stride = dout_stride;
    p.dg = dg, p.dg_stride = dg_stride, p.dx = dx, p.dx_stride = dx_stride, p.saves = const_cast<float*>(saves);
    p.state_in = dstate, p.state_out = dstate_in, p.state_off = reinterpret_cast<const long long*>(state_off);
    const bool gb = flags & GLM53F_KDA_SCAN_G_BF16, xb = flags & GLM53F_KDA_SCAN_X_BF16;
    if (!matrices_ok(p, {{g, g_stride, gb}, {x, x_stride, xb}, {dout, dout_stride, xb}, {dg, dg_stride, gb}, {dx, dx_stride, xb}}, p.vec)) return kInvalid;
    if (!state_ok(saves) || state_off == nullptr || (reinterpret_cast<uintptr_t>(dstate) & 3) || (reinterpret_cast<uintptr_t>(dstate_in) & 3)) return kInvalid;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return kInvalid;
    return tiles_launch<true>(p, max_len, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
