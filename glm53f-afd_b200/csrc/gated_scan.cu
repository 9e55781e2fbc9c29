// Gated linear recurrence, channel by channel: h_t = a_t h_{t-1} + c_t x_t, with a_t = e^g_t or the sigmoid of g_t, c_t = 1 or 1 - a_t.
//
// Row by row (decode), as a scan over packed sequences (prefill), and backwards: with e_t = a_{t+1} D_{t+1} the gradient that reaches row t from
// the rows behind it, D_t = dy_t + e_t, so e runs through the same recurrence from the other end; dx_t = c_t D_t and
// dg_t = D_t a'_t (h_{t-1} - [c = 1 - a] x_t), a' the gate's slope.
//
// Bound by HBM: a few operations a value, each value read once and written once.  Rows compose: over rows i..j the recurrence is
// h_j = A h_{i-1} + B with A the product of the a.  A tile is kRows rows of 64 channels; its values stay in registers (eight rows of two
// channels a thread, all loads in flight at once) while the warps' (A, B) meet in shared memory and the tile's in global memory, so a sequence is divided
// over the GPU and still read once: a tile says its (A, B), then looks at those of the tiles before it up to the nearest
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

struct Record;
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
    // The workspace: [0] the counter, [1] whether somebody gave up; what tiles said, [slot][stripe][channel].
    unsigned* control;
    Record* records;
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
// Two channels of a row; bf16 pairs stay packed.
template <bool BF16>
struct Pair {
    float2 v;
    __device__ __forceinline__ float get(int i) const { return i ? v.y : v.x; }
};
template <>
struct Pair<true> {
    uint32_t v;
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i ? v & 0xffff0000u : v << 16); }
};
// `valid` of two channels of a row, each an access of its own; the others 0.
template <bool BF16>
__device__ __forceinline__ Pair<BF16> load_apart(const unsigned char* p, int valid) {
    Pair<BF16> r;
    if constexpr (BF16) {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
        r.v = (valid > 0 ? (uint32_t)__ldg(q) : 0u) | (valid > 1 ? (uint32_t)__ldg(q + 1) << 16 : 0u);
    } else {
        const float* q = reinterpret_cast<const float*>(p);
        r.v = make_float2(valid > 0 ? __ldg(q) : 0.0f, valid > 1 ? __ldg(q + 1) : 0.0f);
    }
    return r;
}
template <bool BF16>
__device__ __forceinline__ Pair<BF16> load_pair(const unsigned char* p, int valid, bool vec) {
    if (!vec) return load_apart<BF16>(p, valid);
    Pair<BF16> r;
    if constexpr (BF16) r.v = valid > 0 ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
    else r.v = valid > 0 ? __ldg(reinterpret_cast<const float2*>(p)) : make_float2(0.0f, 0.0f);
    return r;
}
template <bool BF16>
__device__ __forceinline__ void store_pair(unsigned char* to, int valid, bool vec, float v0, float v1) {
    if constexpr (BF16) {
        uint16_t* p = reinterpret_cast<uint16_t*>(to);
        if (vec) {
            if (valid > 0) *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v0, v1);
        } else {
            if (valid > 0) p[0] = f32_to_bf16_bits(v0);
            if (valid > 1) p[1] = f32_to_bf16_bits(v1);
        }
    } else {
        float* p = reinterpret_cast<float*>(to);
        if (vec) {
            if (valid > 0) *reinterpret_cast<float2*>(p) = make_float2(v0, v1);
        } else {
            if (valid > 0) p[0] = v0;
            if (valid > 1) p[1] = v1;
        }
    }
}
template <bool BF16>
constexpr int kBytes = BF16 ? 2 : 4;

// A thread's place in a matrix of rows: its first row's two channels, and the bytes between rows.
struct Walk {
    unsigned char* at;
    long long step;
    __device__ __forceinline__ Walk(const void* base, long long row, long long stride, int channel, int size)
        : at(static_cast<unsigned char*>(const_cast<void*>(base)) + (row * stride + channel) * size), step(stride * size) {}
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The rows of a tile that are on their way to a thread: places of shared memory that only it reads, so no barrier is needed between the copies and it.
template <bool BF16, int THREADS>
struct Inbox {
    Pair<BF16> v[kPer][THREADS];
    // Asks for m rows.
    __device__ __forceinline__ void ask(const Walk& w, int m, int valid, bool vec) {
        if (valid <= 0) return;
        const unsigned char* p = w.at;
#pragma unroll
        for (int r = 0; r < kPer; ++r, p += w.step) {
            if (r >= m) break;
            Pair<BF16>* to = &v[r][threadIdx.x];
            if (vec) copy_async<2 * kBytes<BF16>>(to, p);
            else if (!BF16 && valid > 1) copy_async<4>(to, p), copy_async<4>(reinterpret_cast<float*>(to) + 1, p + 4);
            else *to = load_apart<BF16>(p, valid);
        }
    }
    __device__ __forceinline__ Pair<BF16> get(int r) const { return v[r][threadIdx.x]; }
};

// e^x for x <= 0 or little above, to two units in the last place or so: the power of two of x log2(e) and what its rounding left.  Below 2^-126: 0.
__device__ __forceinline__ float exp_of(float x) {
    x = max_nan(x, -200.0f);  // (-inf: no infinities among the parts)
    const float t = x * kLog2e, rest = fmaf(x, kLog2e, -t), e = ex2_ftz(t);
    return fmaf(e, rest * 0.69314718f, e);
}
// a, and 1 - a without the cancellation where a is near one.  Of the sigmoid both from e^-|g|: no overflow, and the smaller one keeps its digits.
// Of e^g by the series of the exponential where a > 1/2.
template <bool SIGMOID, bool REST>
__device__ __forceinline__ void gate(float g, float& a, float& rest) {
    if constexpr (SIGMOID) {
        const float e = exp_of(-fabsf(g)), d = 1.0f + e;
        float r = rcp_approx(d);
        r = fmaf(r, fmaf(-d, r, 1.0f), r);  // (to half a step and a little)
        const float small = e * r;
        a = g < 0.0f ? small : r, rest = g < 0.0f ? r : small;
    } else {
        a = exp_of(g);
        if constexpr (REST) {
            float s = fmaf(g, 2.7557319e-6f, 2.4801587e-5f);  // 1 / 9!, 1 / 8!, ...
            s = fmaf(g, s, 1.9841270e-4f);
            s = fmaf(g, s, 1.3888889e-3f);
            s = fmaf(g, s, 8.3333333e-3f);
            s = fmaf(g, s, 4.1666667e-2f);
            s = fmaf(g, s, 1.6666667e-1f);
            s = fmaf(g, s, 0.5f);
            rest = fabsf(g) < 0.6931472f ? -fmaf(g * g, s, g) : 1.0f - a;
        } else {
            rest = 1.0f;
        }
    }
}

// ---- between tiles ------------------------------------------------------------------------------------------------------------
// What a tile says of a channel, in one access of 16 bytes: its (A, B), its end state, and which of the two are there.
struct __align__(16) Record {
    float a, b, whole;
    unsigned said;
};
__device__ __forceinline__ void say(Record* to, const Record& r) {
    asm volatile(
        "{\n\t.reg .b64 x, y;\n\t.reg .b128 z;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\tmov.b128 z, {x, y};\n\t"
        "st.relaxed.gpu.global.b128 [%0], z;\n\t}" ::"l"(to),
        "f"(r.a), "f"(r.b), "f"(r.whole), "r"(r.said)
        : "memory");
}
__device__ __forceinline__ Record heard(const Record* from) {
    Record r;
    asm volatile(
        "{\n\t.reg .b64 x, y;\n\t.reg .b128 z;\n\tld.relaxed.gpu.global.b128 z, [%4];\n\tmov.b128 {x, y}, z;\n\t"
        "mov.b64 {%0, %1}, x;\n\tmov.b64 {%2, %3}, y;\n\t}"
        : "=f"(r.a), "=f"(r.b), "=f"(r.whole), "=r"(r.said)
        : "l"(from)
        : "memory");
    return r;
}

// The state that reaches this tile, for the threads below kChannels (a channel each), called by the whole block.  `count` tiles of its sequence lie before it (STEP -1) or behind
// it (STEP 1), `more`: one waits for its end state.  Each warp asks one of the nearest tiles, all channels; the chain runs from the nearest whole one.
template <int STEP, int WARPS>
__device__ __forceinline__ float join(const ScanParams& p, Record (*near)[kChannels], long long slot, int stripe, int count, float A, float B, float start, bool more) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long pitch = (long long)p.stripes * kChannels;
    Record* mine = p.records + slot * pitch + stripe * kChannels;
    if (tid < kChannels && more) say(mine + tid, count == 0 ? Record{A, B, fmaf(A, start, B), kWhole} : Record{A, B, 0.0f, kPart});
    if (count == 0) return start;
    const int window = min(count, WARPS);
    const Record* theirs = mine + STEP * (1 + warp) * pitch;
    uint64_t t0 = 0;
    float h = 0.0f;
    for (int polls = 0;; ++polls) {
        if (warp < window) {
            const Record r0 = heard(theirs + lane), r1 = heard(theirs + 32 + lane);
            near[warp][lane] = r0, near[warp][32 + lane] = r1;
        }
        __syncthreads();
        bool found = true;
        if (tid < kChannels) {
            int d = 0;
            while (d < window && near[d][tid].said == kPart) ++d;
            found = d < window && near[d][tid].said == kWhole;
            if (found) {
                h = near[d][tid].whole;
                while (--d >= 0) h = fmaf(near[d][tid].a, h, near[d][tid].b);
            }
        }
        bool over = false;
        if (polls % 64 == 63) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            over = now - t0 > kWaitLimitNs || load_acquire(p.control + 1) != 0;
        }
        const int missing = __syncthreads_or(found ? 0 : 1);
        if (!missing) break;
        if (polls % 64 == 63 && __syncthreads_or(over)) {  // give up, and let the others know
            if (tid == 0) {
                atomicCAS(p.status, 0, STEP < 0 ? kStatusScanBefore : kStatusScanBehind);
                store_release(p.control + 1, 1u);
            }
            h = __int_as_float(0x7fc00000);
            break;
        }
    }
    if (tid < kChannels && more) say(mine + tid, Record{A, B, fmaf(A, h, B), kWhole});
    return h;
}

__global__ void scan_clear_kernel(const ScanParams p) {
    grid_ready();
    const long long n = p.tiles * kChannels;
    if (blockIdx.x == 0 && threadIdx.x < 2) p.control[threadIdx.x] = 0u;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) p.records[i].said = kNothing;
}

// Which tile a block is at.  LOOK: tiles come from the counter; otherwise the block walks its sequence's tiles, from the end that the pass starts at.
struct Place {
    int stripe, slot, b, first, n, tile, tiles;  // b < 0: no more
    __device__ __forceinline__ bool live() const { return b >= 0 && tile < tiles; }  // (a slot may lie between two sequences' tiles)
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

// A block's tiles, two known ahead: the copies of the next one's rows are asked for while this one is worked on.
template <int T, int WARPS, bool LOOK, bool REVERSE>
struct Tiles {
    Place (&ring)[3];
    unsigned ticket = 0;
    const bool guide = threadIdx.x / 32 == WARPS - 1;
    __device__ __forceinline__ Place next(const ScanParams& p, int i) {  // the guide's: tile i's place
        Place at;
        if constexpr (LOOK) {
            const unsigned now = __shfl_sync(0xffffffffu, ticket, 0);
            if ((threadIdx.x & 31) == 0) ticket = atomicAdd(p.control, 1u);
            place_ticket<T, REVERSE>(p, now, at);
        } else {
            place_walk<T, REVERSE>(p, i, at);
        }
        return at;
    }
    __device__ __forceinline__ void put(const ScanParams& p, int i) {
        if (!guide) return;
        const Place at = next(p, i);
        if ((threadIdx.x & 31) == 0) ring[i % 3] = at;
    }
    __device__ __forceinline__ Tiles(const ScanParams& p, Place (&r)[3]) : ring(r) {
        if (LOOK && guide && (threadIdx.x & 31) == 0) ticket = atomicAdd(p.control, 1u);
        put(p, 0);
        put(p, 1);
        __syncthreads();
    }
};

// This thread's rows of a tile, and how many there are.
template <int T>
__device__ __forceinline__ int rows_of(const Place& at, int& row0, long long& row) {
    row0 = at.tile * T + (threadIdx.x >> 5) * kPer;
    row = (long long)at.first + row0;
    return min(max(at.n - row0, 0), kPer);
}

template <bool GB, bool XB>
struct ForwardShared {
    Inbox<GB, kForwardWarps * 32> g;
    Inbox<XB, kForwardWarps * 32> x;
    Record near[kForwardWarps][kChannels];
    float4 agg[2][kForwardWarps][32];  // (A, B) of a warp's rows, two channels; two tiles' worth, so that one barrier a tile is enough
    float carry[kChannels];
    Place ring[3];
};

template <bool LOOK, bool GB, bool XB>
__global__ void __launch_bounds__(kForwardWarps * 32, 2) scan_forward_kernel(const ScanParams p) {
    constexpr int T = kForwardRows;
    extern __shared__ __align__(16) unsigned char smem[];
    auto& sh = *reinterpret_cast<ForwardShared<GB, XB>*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool vec = p.vec;
    float walk = 0.0f;  // a walking block's state between its tiles, a channel a thread of the first two warps
    grid_ready();
    Tiles<T, kForwardWarps, LOOK, false> tiles(p, sh.ring);
    auto ask = [&](const Place& at) {
        if (!at.live()) return;
        int row0;
        long long row;
        const int m = rows_of<T>(at, row0, row), c0 = at.stripe * kChannels + 2 * lane, valid = p.channels - c0;
        sh.g.ask(Walk(p.g, row, p.g_stride, c0, kBytes<GB>), m, valid, vec);
        sh.x.ask(Walk(p.x, row, p.x_stride, c0, kBytes<XB>), m, valid, vec);
    };
    ask(sh.ring[0]);
    for (int i = 0;; ++i) {
        const Place at = sh.ring[i % 3];
        if (at.b < 0) return;
        auto& agg = sh.agg[i & 1];
        int row0;
        long long row;
        const int m = rows_of<T>(at, row0, row), c0 = at.stripe * kChannels + 2 * lane, valid = p.channels - c0;
        float a[kPer][2], b[kPer][2];
        copies_done();
        if (at.live()) {
            with_flags(p.flags, [&](auto sigmoid, auto complement) {
#pragma unroll
                for (int r = 0; r < kPer; ++r) {
                    const Pair<GB> g = sh.g.get(r);
                    const Pair<XB> x = sh.x.get(r);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float rest;
                        gate<decltype(sigmoid)::value, decltype(complement)::value>(g.get(j), a[r][j], rest);
                        b[r][j] = decltype(complement)::value ? rest * x.get(j) : x.get(j);
                    }
                }
            });
            if (m < kPer)  // rows past the end leave the state as it is
#pragma unroll
                for (int r = 0; r < kPer; ++r)
                    if (r >= m) a[r][0] = a[r][1] = 1.0f, b[r][0] = b[r][1] = 0.0f;
            float A[2] = {1.0f, 1.0f}, B[2] = {0.0f, 0.0f};
#pragma unroll
            for (int r = 0; r < kPer; ++r)
#pragma unroll
                for (int j = 0; j < 2; ++j) A[j] *= a[r][j], B[j] = fmaf(a[r][j], B[j], b[r][j]);
            agg[warp][lane] = make_float4(A[0], B[0], A[1], B[1]);
        }
        __syncthreads();
        ask(sh.ring[(i + 1) % 3]);
        tiles.put(p, i + 2);
        if (!at.live()) continue;
        float TA = 1.0f, TB = 0.0f, start = walk;
        const int c = at.stripe * kChannels + tid;
        if (tid < kChannels) {  // a channel a thread
#pragma unroll
            for (int w = 0; w < kForwardWarps; ++w) {
                const float2 ab = reinterpret_cast<const float2*>(agg[w])[tid];
                TA *= ab.x, TB = fmaf(ab.x, TB, ab.y);
            }
            if (at.tile == 0 && c < p.channels) start = p.state_in[p.state_off[at.b] + c];
        }
        float h0 = start;
        if constexpr (LOOK) h0 = join<-1, kForwardWarps>(p, sh.near, at.slot, at.stripe, at.tile, TA, TB, start, at.tile + 1 < at.tiles);
        else walk = fmaf(TA, h0, TB);
        if (tid < kChannels) {
            sh.carry[tid] = h0;
            if (at.n == 0 && c < p.channels) p.state_out[p.state_off[at.b] + c] = h0;
        }
        __syncthreads();
        float h[2] = {sh.carry[2 * lane], sh.carry[2 * lane + 1]};
        for (int w = 0; w < warp; ++w) {
            const float4 ab = agg[w][lane];
            h[0] = fmaf(ab.x, h[0], ab.y), h[1] = fmaf(ab.z, h[1], ab.w);
        }
        if (p.saves != nullptr && (warp * kPer) % kSave == 0 && (m > 0 || row0 == 0))
            store_pair<false>(reinterpret_cast<unsigned char*>(p.saves + ((long long)slot_of(at.first, at.b, kSave) + row0 / kSave) * p.channels + c0), valid,
                              p.channels % 2 == 0, h[0], h[1]);
        Walk out(p.out, row, p.out_stride, c0, kBytes<XB>);
#pragma unroll
        for (int r = 0; r < kPer; ++r, out.at += out.step) {
            h[0] = fmaf(a[r][0], h[0], b[r][0]), h[1] = fmaf(a[r][1], h[1], b[r][1]);
            if (r < m && p.out != nullptr) store_pair<XB>(out.at, valid, vec, h[0], h[1]);
        }
        if (m > 0 && row0 + m == at.n) {
            float* s = p.state_out + p.state_off[at.b] + c0;
            if (valid > 0) s[0] = h[0];
            if (valid > 1) s[1] = h[1];
        }
    }
}

template <bool GB, bool XB>
struct BackwardShared {
    struct Rows {
        Inbox<GB, kBackwardWarps * 32> g;
        Inbox<XB, kBackwardWarps * 32> x, dy;
    } rows[2];  // (a tile's are read again at its end, when the next one's are on their way)
    Record near[kBackwardWarps][kChannels];
    float4 agg[2][kBackwardWarps][32];
    float2 back[2][kBackwardWarps][32];  // what a warp's rows add to e
    float carry[kChannels];
    Place ring[3];
};

// As the forward pass from the other end, e in h's place: D_t = dy_t + e_t, e_{t-1} = a_t D_t.  The h of the tile's rows are formed again from the saved state at its start.
template <bool LOOK, bool GB, bool XB>
__global__ void __launch_bounds__(kBackwardWarps * 32, XB ? 3 : 2) scan_backward_kernel(const ScanParams p) {
    constexpr int T = kBackwardRows;
    extern __shared__ __align__(16) unsigned char smem[];
    auto& sh = *reinterpret_cast<BackwardShared<GB, XB>*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool vec = p.vec;
    float walk = 0.0f;
    grid_ready();
    Tiles<T, kBackwardWarps, LOOK, true> tiles(p, sh.ring);
    auto ask = [&](const Place& at, auto& to) {
        if (!at.live()) return;
        int row0;
        long long row;
        const int m = rows_of<T>(at, row0, row), c0 = at.stripe * kChannels + 2 * lane, valid = p.channels - c0;
        to.g.ask(Walk(p.g, row, p.g_stride, c0, kBytes<GB>), m, valid, vec);
        to.x.ask(Walk(p.x, row, p.x_stride, c0, kBytes<XB>), m, valid, vec);
        to.dy.ask(Walk(p.dout, row, p.dout_stride, c0, kBytes<XB>), m, valid, vec);
    };
    ask(sh.ring[0], sh.rows[0]);
    for (int i = 0;; ++i) {
        const Place at = sh.ring[i % 3];
        if (at.b < 0) return;
        auto& agg = sh.agg[i & 1];
        auto& back = sh.back[i & 1];
        const auto& in = sh.rows[i & 1];
        int row0;
        long long row;
        const int m = rows_of<T>(at, row0, row), c0 = at.stripe * kChannels + 2 * lane, valid = p.channels - c0;
        const float* save = p.saves + ((long long)slot_of(at.first, at.b, kSave) + at.tile) * p.channels + c0;
        float before[2] = {at.live() && valid > 0 ? __ldg(save) : 0.0f, at.live() && valid > 1 ? __ldg(save + 1) : 0.0f};
        copies_done();
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
            constexpr bool S = decltype(sigmoid)::value, C = decltype(complement)::value;
            float a[kPer][2], b[kPer][2];
            if (at.live()) {
#pragma unroll
                for (int r = 0; r < kPer; ++r) {
                    const Pair<GB> g = in.g.get(r);
                    const Pair<XB> x = in.x.get(r);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float rest;
                        gate<S, C>(g.get(j), a[r][j], rest);
                        b[r][j] = C ? rest * x.get(j) : x.get(j);
                        if (r >= m) a[r][j] = 1.0f, b[r][j] = 0.0f;
                    }
                }
                float A[2] = {1.0f, 1.0f}, B[2] = {0.0f, 0.0f}, F[2] = {0.0f, 0.0f};
#pragma unroll
                for (int r = 0; r < kPer; ++r)
#pragma unroll
                    for (int j = 0; j < 2; ++j) A[j] *= a[r][j], B[j] = fmaf(a[r][j], B[j], b[r][j]);
#pragma unroll
                for (int r = kPer - 1; r >= 0; --r) {
                    const Pair<XB> dy = in.dy.get(r);
#pragma unroll
                    for (int j = 0; j < 2; ++j) F[j] = a[r][j] * ((r < m ? dy.get(j) : 0.0f) + F[j]);
                }
                agg[warp][lane] = make_float4(A[0], B[0], A[1], B[1]);
                back[warp][lane] = make_float2(F[0], F[1]);
            }
            __syncthreads();
            ask(sh.ring[(i + 1) % 3], sh.rows[(i + 1) & 1]);
            tiles.put(p, i + 2);
            if (!at.live()) return;
            // The states before this warp's rows, and before each of them.
            for (int w = 0; w < warp; ++w) {
                const float4 ab = agg[w][lane];
                before[0] = fmaf(ab.x, before[0], ab.y), before[1] = fmaf(ab.z, before[1], ab.w);
            }
#pragma unroll
            for (int r = 0; r < kPer; ++r)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float h = before[j];
                    before[j] = fmaf(a[r][j], h, b[r][j]);
                    b[r][j] = h;
                }
            float TA = 1.0f, TF = 0.0f, start = walk;
            const int c = at.stripe * kChannels + tid;
            if (tid < kChannels) {
#pragma unroll
                for (int w = kBackwardWarps - 1; w >= 0; --w) {
                    const float wa = reinterpret_cast<const float2*>(agg[w])[tid].x;
                    TA *= wa, TF = fmaf(wa, TF, reinterpret_cast<const float*>(back[w])[tid]);
                }
                if (at.tile + 1 == at.tiles) start = c < p.channels && p.state_in != nullptr ? p.state_in[p.state_off[at.b] + c] : 0.0f;
            }
            float e0 = start;
            if constexpr (LOOK) e0 = join<1, kBackwardWarps>(p, sh.near, at.slot, at.stripe, at.tiles - 1 - at.tile, TA, TF, start, at.tile > 0);
            else walk = fmaf(TA, e0, TF);
            if (tid < kChannels) {
                sh.carry[tid] = e0;
                if (at.n == 0 && c < p.channels && p.state_out != nullptr) p.state_out[p.state_off[at.b] + c] = e0;
            }
            __syncthreads();
            float e[2] = {sh.carry[2 * lane], sh.carry[2 * lane + 1]};
            for (int w = kBackwardWarps - 1; w > warp; --w) {
                const float4 ab = agg[w][lane];
                const float2 f = back[w][lane];
                e[0] = fmaf(ab.x, e[0], f.x), e[1] = fmaf(ab.z, e[1], f.y);
            }
            Walk dxs(p.dx, row + kPer - 1, p.dx_stride, c0, kBytes<XB>), dgs(p.dg, row + kPer - 1, p.dg_stride, c0, kBytes<GB>);
#pragma unroll
            for (int r = kPer - 1; r >= 0; --r, dxs.at -= dxs.step, dgs.at -= dgs.step) {
                if (r >= m) continue;
                const Pair<GB> g = in.g.get(r);
                const Pair<XB> x = in.x.get(r), dy = in.dy.get(r);
                float dg[2], dx[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float d = dy.get(j) + e[j];
                    float again = a[r][j], rest = 1.0f;
                    if constexpr (C || S) gate<S, C>(g.get(j), again, rest);  // (its other half again, from shared memory rather than kept)
                    const float slope = S ? again * rest : again;
                    dx[j] = C ? rest * d : d;
                    dg[j] = d * slope * (C ? b[r][j] - x.get(j) : b[r][j]);
                    e[j] = again * d;
                }
                store_pair<XB>(dxs.at, valid, vec, dx[0], dx[1]);
                store_pair<GB>(dgs.at, valid, vec, dg[0], dg[1]);
            }
            if (row0 == 0 && m > 0 && p.state_out != nullptr) {
                float* s = p.state_out + p.state_off[at.b] + c0;
                if (valid > 0) s[0] = e[0];
                if (valid > 1) s[1] = e[1];
            }
        });
    }
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
        Walk gs(p.g, row, p.g_stride, c0, kBytes<GB>), xs(p.x, row, p.x_stride, c0, kBytes<XB>), out(p.out, row, p.out_stride, c0, kBytes<XB>);
#pragma unroll
        for (int r = 0; r < kPer; ++r, gs.at += gs.step, xs.at += xs.step) {
            const int v = r < m ? valid : 0;
            g[r] = load_pair<GB>(gs.at, v, p.vec);
            x[r] = load_pair<XB>(xs.at, v, p.vec);
        }
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
#pragma unroll
            for (int r = 0; r < kPer; ++r, out.at += out.step) {
                if (r >= m) break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float a, rest;
                    gate<decltype(sigmoid)::value, decltype(complement)::value>(g[r].get(j), a, rest);
                    h[j] = fmaf(a, h[j], decltype(complement)::value ? rest * x[r].get(j) : x[r].get(j));
                }
                if (p.out != nullptr) store_pair<XB>(out.at, valid, p.vec, h[0], h[1]);
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
    long long slots, stripes, records, bytes;
    Layout(int64_t channels, int64_t batch, int64_t rows, int tile_rows) {
        slots = rows / tile_rows + batch;
        stripes = (channels + kChannels - 1) / kChannels;
        records = 256;
        bytes = records + slots * stripes * kChannels * (long long)sizeof(Record);
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
        p.records = reinterpret_cast<Record*>(w + at.records);
        p.slots = (int)at.slots;
        p.tiles = at.slots * at.stripes;
        const long long clear = (p.tiles * kChannels + 1023) / 1024, some = 4ll * sm_count();
        const int rc = launch_early(scan_clear_kernel, dim3((unsigned)(clear < some ? clear : some)), 256, 0, stream, p);
        if (rc != 0) return rc;
    }
    return with_types(p.flags, look, [&](auto l, auto gb, auto xb) {
        constexpr bool L = decltype(l)::value, G = decltype(gb)::value, X = decltype(xb)::value;
        auto launch = [&](auto kernel, size_t shared, int per_sm) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
            if (e != cudaSuccess) return (int)e;
            const long long most = (long long)per_sm * sm_count();
            if (L) blocks = p.tiles < most ? p.tiles : most;
            return launch_early(kernel, dim3((unsigned)blocks), threads, shared, stream, p);
        };
        if constexpr (BACKWARD) return launch(scan_backward_kernel<L, G, X>, sizeof(BackwardShared<G, X>), X ? 3 : 2);
        else return launch(scan_forward_kernel<L, G, X>, sizeof(ForwardShared<G, X>), 2);
    });
}

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
