// Gated linear recurrence, channel by channel: h_t = a_t h_{t-1} + c_t x_t, with a_t = e^g_t or the sigmoid of g_t, c_t = 1 or 1 - a_t.
//
// Row by row (decode), as a scan over packed sequences (prefill), and backwards: with e_t = a_{t+1} D_{t+1} the gradient that reaches row t from
// the rows behind it, D_t = dy_t + e_t, so e runs through the same recurrence from the other end; dx_t = c_t D_t and
// dg_t = D_t a'_t (h_{t-1} - [c = 1 - a] x_t), a' the gate's slope.
//
// Bound by HBM: a few operations a value, each value read once and written once.  Rows compose: over rows i..j the recurrence is
// h_j = A h_{i-1} + B with A the product of the a.  A tile is 64 rows of 64 channels.  A sequence is divided over the GPU and still read once: a tile says its
// (A, B) in global memory, looks at those of the tiles before it up to the nearest whose end state is known, and says its own.  Tiles are taken from
// a counter in their order, so whatever a tile waits for is with a block that runs already; the wait is bounded all the same (status 160).
//
// What passes between tiles takes 1 to 2 us, longer than a tile's share of the memory time (0.75 us), so several tiles of a block are under way at once, one block an SM:
//   a producer warp    finds the tiles and copies their rows into a ring of shared memory by tensor copies (64 x 64 boxes), two to three ahead;
//   two groups of eight warps, a tile each in turn: the (A, B) of the eight rows of every warp; then, when the state that reaches the tile before
//                      is there, the rows of that one, whose gates are formed again from shared memory: registers would hold only half as many;
//   pairs of chain warps, a channel a lane, a tile in turn: the tile's (A, B) from the warps', what passes between tiles, every warp's start.
// (With all of a tile done by one set of threads, two blocks an SM, 65,536 rows x 1,024 channels took 198 us, of 12,600 cycles a tile 4,300 in the wait for
// the state and 2,100 in asking for rows.)
//
// The states between tiles come from one chain of h <- A h + B whatever a tile found ready: the same bits every time, with any workspace and beside any other request.

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "kda_internal.h"
#include "tensor_map.cuh"

namespace kda {
namespace {

constexpr int kChannels = 64;  // of a tile: two a lane
constexpr int kRows = 64;      // of a tile
constexpr int kPer = 8;        // rows of a warp
constexpr int kWarps = kRows / kPer;  // of a group
constexpr int kGroups = 2;
constexpr int kAcross = 8;     // tiles that a look takes in at once
constexpr int kMostShared = 226 * 1024;
constexpr int kMost = 1 << 30;  // channels, rows: their tiles' ends are ints

// Every wait is bounded; the codes say which one gave up.
enum : int { kStatusScanChain = 160, kStatusScanEmpty = 161, kStatusScanFull = 162, kStatusScanSums = 163, kStatusScanStart = 164 };
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
    // Rows that lie on 16 bytes come by tensor copies: (channel, row) maps of the inputs, boxes of a tile.
    int boxes;
    CUtensorMap tm_g, tm_x, tm_dout;
};

// Tile slots: sequence b's tiles lie at cu[b] / 64 + b and behind.  Every sequence has a slot at least, slots ascend with b, and rows / 64 + batch are enough.
__device__ __forceinline__ int slot_of(int first, int b) { return first / kRows + b; }

// The sequence that slot lies in, by a converged warp: the last b with slot_of(cu[b], b) <= slot.
__device__ int sequence_of(const int32_t* cu, int batch, int slot) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = batch;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const bool below = at < n && slot_of(__ldg(cu + lo + at), lo + at) <= slot;
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
    __device__ __forceinline__ float2 get() const { return v; }
};
template <>
struct Pair<true> {
    uint32_t v;
    __device__ __forceinline__ float2 get() const { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
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

// A tile's rows of one matrix.  Where they come by boxes all of them do; else each thread asks for its own channels of its warp's rows, which only it reads.
template <bool BF16>
struct __align__(128) Inbox {
    static constexpr uint32_t kBoxBytes = kRows * kChannels * kBytes<BF16>;
    Pair<BF16> v[kWarps][kPer][32];
    __device__ __forceinline__ float2 get(int warp, int r) const { return v[warp][r][threadIdx.x & 31].get(); }
    __device__ __forceinline__ void box(const CUtensorMap& tm, int channel, int row, uint64_t* bar) {
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(v)),
                     "l"(reinterpret_cast<uint64_t>(&tm)), "r"(smem_u32(bar)), "r"(channel), "r"(row)
                     : "memory");
    }
    __device__ __forceinline__ void ask(int warp, const Walk& w, int m, int valid, bool vec) {
        if (valid <= 0) return;
        const unsigned char* p = w.at;
#pragma unroll 2
        for (int r = 0; r < m; ++r, p += w.step) {
            Pair<BF16>* to = &v[warp][r][threadIdx.x & 31];
            if (vec) copy_async<2 * kBytes<BF16>>(to, p);
            else if (!BF16 && valid > 1) copy_async<4>(to, p), copy_async<4>(reinterpret_cast<float*>(to) + 1, p + 4);
            else *to = load_apart<BF16>(p, valid);
        }
    }
};

__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 ex2_two(float2 t) { return make_float2(ex2_ftz(t.x), ex2_ftz(t.y)); }
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// a, and with REST 1 - a without the cancellation where a is near one.  Below 2^-126: 0.
//   e^g: the exponent's rounding costs |g| 2^-24 of a, beside the instruction's own error: 1.4 u measured where a is near one (u = 2^-24; -0.1 u on average, so that it does not grow with what
//     a channel remembers), 2.6 u for a > 1/2, 8.4 u at g = -10.  1 - a by the exponential's series where a > 1/2.
//   sigmoid: both from e^-|g|, whose exponent's rounding is made good, so that the smaller one keeps its digits: no overflow either.
template <bool SIGMOID, bool REST>
__device__ __forceinline__ void gate(float2 g, float2& a, float2& rest) {
    if constexpr (SIGMOID) {
        const float2 m = make_float2(min_nan(fabsf(g.x), 200.0f), min_nan(fabsf(g.y), 200.0f));
        const float2 t = mul2(m, two(-kLog2e)), left = fma2(m, two(-kLog2e), make_float2(-t.x, -t.y));
        float2 e = ex2_two(t);
        e = fma2(e, mul2(left, two(0.69314718f)), e);
        // 1 / (1 + e) by Newton's steps from the best straight line on [1, 2] (1/17 off, so 1/289, 1.2e-5, 1.4e-10): with the units for special functions
        // busy with the exponentials of both passes, theirs would be the bound.
        const float2 d = make_float2(1.0f + e.x, 1.0f + e.y), minus = make_float2(-d.x, -d.y);
        float2 r = fma2(d, two(-8.0f / 17.0f), two(24.0f / 17.0f));
#pragma unroll
        for (int i = 0; i < 3; ++i) r = fma2(r, fma2(minus, r, two(1.0f)), r);
        const float2 small = mul2(e, r);
        a = make_float2(g.x < 0.0f ? small.x : r.x, g.y < 0.0f ? small.y : r.y);
        rest = make_float2(g.x < 0.0f ? r.x : small.x, g.y < 0.0f ? r.y : small.y);
    } else {
        a = ex2_two(mul2(g, two(kLog2e)));
        if constexpr (REST) {
            float2 s = fma2(g, two(2.7557319e-6f), two(2.4801587e-5f));  // 1 / 9!, 1 / 8!, ...
            s = fma2(g, s, two(1.9841270e-4f));
            s = fma2(g, s, two(1.3888889e-3f));
            s = fma2(g, s, two(8.3333333e-3f));
            s = fma2(g, s, two(4.1666667e-2f));
            s = fma2(g, s, two(1.6666667e-1f));
            s = fma2(g, s, two(0.5f));
            s = fma2(mul2(g, g), s, g);
            rest = make_float2(fabsf(g.x) < 0.6931472f ? -s.x : 1.0f - a.x, fabsf(g.y) < 0.6931472f ? -s.y : 1.0f - a.y);
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

// The state that reaches the tile in `slot` from the `count` > 0 tiles of its sequence before it (STEP -1) or behind it (STEP 1), a channel a lane: the chain from the nearest
// whole tile on, over (A, B) of those in between.
template <int STEP>
__device__ float look(const ScanParams& p, const Record* mine, int count) {
    const long long pitch = STEP * (long long)p.stripes * kChannels;
    uint64_t t0 = 0;
    float h = 0.0f;
    bool found = false;
    for (int polls = 0; !found; ++polls) {
        // Outwards in steps of kAcross, twice at most: a lane's chain lies in registers.
        Record near[kAcross], far[kAcross];
        int whole = -1;
#pragma unroll
        for (int d = 0; d < kAcross; ++d) near[d] = d < count ? heard(mine + (d + 1) * pitch) : Record{0.0f, 0.0f, 0.0f, kNothing};
        bool parts = true;
#pragma unroll
        for (int d = 0; d < kAcross; ++d) {
            if (parts && near[d].said == kWhole) whole = d;
            parts = parts && near[d].said == kPart;
        }
        if (parts) {
#pragma unroll
            for (int d = 0; d < kAcross; ++d) far[d] = d + kAcross < count ? heard(mine + (d + kAcross + 1) * pitch) : Record{0.0f, 0.0f, 0.0f, kNothing};
#pragma unroll
            for (int d = 0; d < kAcross; ++d) {
                if (parts && far[d].said == kWhole) whole = d + kAcross;
                parts = parts && far[d].said == kPart;
            }
            if (whole >= 0) {
#pragma unroll
                for (int d = kAcross - 1; d >= 0; --d) {
                    if (d + kAcross == whole) h = far[d].whole;
                    else if (d + kAcross < whole) h = fmaf(far[d].a, h, far[d].b);
                }
            }
        }
        if (whole >= 0) {
#pragma unroll
            for (int d = kAcross - 1; d >= 0; --d) {
                if (d == whole) h = near[d].whole;
                else if (d < whole) h = fmaf(near[d].a, h, near[d].b);
            }
            found = true;
        }
        if (!found && polls % 64 == 63) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > kWaitLimitNs || load_acquire(p.control + 1) != 0) {  // give up, and let the others know
                atomicCAS(p.status, 0, kStatusScanChain);
                store_release(p.control + 1, 1u);
                return __int_as_float(0x7fc00000);
            }
        }
    }
    return h;
}
// The same, and what is said of this tile: its (A, B) at once, its end state when it is known, where `more`: another tile waits for it.
template <int STEP>
__device__ __forceinline__ float join(const ScanParams& p, long long slot, int stripe, int channel, int count, float A, float B, float start, bool more) {
    Record* mine = p.records + (slot * p.stripes + stripe) * kChannels + channel;
    if (count == 0) {
        if (more) say(mine, Record{A, B, fmaf(A, start, B), kWhole});
        return start;
    }
    if (more) say(mine, Record{A, B, 0.0f, kPart});
    const float h = look<STEP>(p, mine, count);
    if (more) say(mine, Record{A, B, fmaf(A, h, B), kWhole});
    return h;
}

__global__ void scan_clear_kernel(const __grid_constant__ ScanParams p) {
    grid_ready();
    const long long n = p.tiles * kChannels;
    if (blockIdx.x == 0 && threadIdx.x < 2) p.control[threadIdx.x] = 0u;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) p.records[i].said = kNothing;
}

// A tile's place.
struct Place {
    int stripe, slot, b, first, n, tile, tiles;  // b < 0: no more tiles
};
__device__ __forceinline__ void place_sequence(const ScanParams& p, Place& at) {
    at.first = min(max(__ldg(p.cu + at.b), 0), p.rows);
    at.n = max(min(__ldg(p.cu + at.b + 1), p.rows) - at.first, 0);
    at.tiles = max((at.n + kRows - 1) / kRows, 1);  // a sequence without rows has a tile all the same: its state passes through
}

// A block's tiles one after another, by a converged warp.  LOOK: from the counter, sequences' tiles forwards (backwards with REVERSE), the stripes of channels fastest;
// otherwise all of a sequence's 64 channels, then another one's.
template <bool LOOK, bool REVERSE>
struct Tiles {
    unsigned ticket = 0;
    long long item = blockIdx.x;
    int walked = 0;
    Place seen;
    __device__ __forceinline__ Tiles(const ScanParams& p) {
        if (LOOK && (threadIdx.x & 31) == 0) ticket = atomicAdd(p.control, 1u);
        seen.b = -1;
    }
    __device__ __forceinline__ Place next(const ScanParams& p) {
        Place at;
        if constexpr (LOOK) {
            for (;;) {
                const unsigned now = __shfl_sync(0xffffffffu, ticket, 0);
                if ((threadIdx.x & 31) == 0) ticket = atomicAdd(p.control, 1u);  // the next one, on its way
                at.b = -1;
                if (now >= p.tiles) return at;
                at.stripe = (int)(now % p.stripes);
                const int i = (int)(now / p.stripes);
                at.slot = REVERSE ? p.slots - 1 - i : i;
                at.b = sequence_of(p.cu, p.batch, at.slot);
                place_sequence(p, at);
                at.tile = at.slot - slot_of(at.first, at.b);
                if (at.tile >= 0 && at.tile < at.tiles) return at;  // (else a slot between two sequences, or before the first one's rows)
            }
        } else {
            if (seen.b >= 0 && walked == seen.tiles) item += gridDim.x, seen.b = -1;
            if (seen.b < 0) {
                at.b = -1;
                if (item >= (long long)p.stripes * p.batch) return at;
                seen.stripe = (int)(item % p.stripes), seen.b = (int)(item / p.stripes);
                place_sequence(p, seen);
                walked = 0;
            }
            at = seen;
            at.tile = REVERSE ? at.tiles - 1 - walked : walked;
            at.slot = slot_of(at.first, at.b) + at.tile;
            ++walked;
            return at;
        }
    }
};

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

template <bool GB, bool XB>
struct ForwardTile {
    Inbox<GB> g;
    Inbox<XB> x;
    float2 sums[kWarps][kChannels];  // (A, B) of a warp's rows; then in A's place the state before them
    static constexpr uint32_t kBoxBytes = Inbox<GB>::kBoxBytes + Inbox<XB>::kBoxBytes;
};
template <bool GB, bool XB>
struct BackwardTile {
    Inbox<GB> g;
    Inbox<XB> x, dy;
    float2 sums[kWarps][kChannels];  // as above
    float back[kWarps][kChannels];   // what a warp's rows add to e; then the e behind them
    static constexpr uint32_t kBoxBytes = Inbox<GB>::kBoxBytes + 2 * Inbox<XB>::kBoxBytes;
};
template <typename TILE>
struct Shared {
    static constexpr int kRing0 = kMostShared / (int)(sizeof(TILE) + sizeof(Place) + 32), kRing = kRing0 < 8 ? kRing0 : 8;
    static_assert(kRing >= 2 * kGroups, "a group holds two tiles");
    TILE tile[kRing];
    uint64_t full[kRing], summed[kRing], started[kRing], empty[kRing];
    Place place[kRing];
    uint32_t control[2];
};
// Chain warps: pairs, a tile each in turn.  A walking block has one, which carries the state.
template <bool LOOK>
constexpr int kPairs = LOOK ? 3 : 1;
template <bool LOOK>
constexpr int kThreads = 32 * (kGroups * kWarps + 2 * kPairs<LOOK> + 1);

// The ring's position of the i-th tile of a block, and the parity of its barriers' phases.
template <int RING>
struct Turn {
    int s;
    uint32_t parity;
    __device__ __forceinline__ explicit Turn(int i) : s(i % RING), parity(i / RING & 1) {}
    __device__ __forceinline__ void step(int n) {
        s += n;
        if (s >= RING) s -= RING, parity ^= 1;
    }
};

// The warps' common frame: barriers, roles, the end.  PASS: load(at, tile, bar) asks for a tile's boxes, ask(at, tile, warp) for a thread's rows without boxes,
// sum(at, tile, warp) forms the warp's sums, chain(at, tile, channel) what reaches the tile, finish(at, tile, warp) the rows.
template <typename TILE, bool LOOK, bool REVERSE, typename PASS>
__device__ __forceinline__ void run(const ScanParams& p, PASS& pass) {
    using S = Shared<TILE>;
    constexpr int R = S::kRing;
    extern __shared__ __align__(128) unsigned char smem[];
    S& sh = *reinterpret_cast<S*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < R; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.summed[s], kWarps);
            mbar_init(&sh.started[s], 2);
            mbar_init(&sh.empty[s], kWarps);
        }
        sh.control[0] = sh.control[1] = 0u;
        mbar_init_fence();
    }
    __syncthreads();
    const WaitCtx ctx{&sh.control[0], &sh.control[1], p.status};
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx, code)); };
    grid_ready();
    if (warp < kGroups * kWarps) {
        const int group = warp / kWarps, w = warp % kWarps;
        Turn<R> now(group), last(group);
        bool pending = false;
        auto finish = [&] {
            if (!wait(&sh.started[last.s], last.parity, kStatusScanStart)) return false;
            pass.finish(sh.place[last.s], sh.tile[last.s], w);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[last.s]);
            return true;
        };
        // Without boxes: the copies of this group's next tile, while it has work left.
        auto next = [&](const Turn<R>& t) {
            if (p.boxes) return true;
            if (!wait(&sh.full[t.s], t.parity, kStatusScanFull)) return false;
            if (sh.place[t.s].b >= 0) pass.ask(sh.place[t.s], sh.tile[t.s], w);
            return true;
        };
        bool ok = next(now);
        while (ok) {
            if (p.boxes) {
                ok = wait(&sh.full[now.s], now.parity, kStatusScanFull);
                if (!ok) break;
            } else {
                copies_done();
            }
            const bool more = sh.place[now.s].b >= 0;
            Turn<R> after = now;
            after.step(kGroups);
            if (more) {
                pass.sum(sh.place[now.s], sh.tile[now.s], w);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.summed[now.s]);
                // (a ring of three tiles a group has room for the next one before the last is done)
                if (R >= 3 * kGroups) ok = next(after);
            }
            if (ok && pending) ok = finish();
            if (!more) break;
            if (R < 3 * kGroups) ok = ok && next(after);
            last = now, pending = true, now = after;
        }
    } else if (warp < kGroups * kWarps + 2 * kPairs<LOOK>) {
        const int i = warp - kGroups * kWarps, channel = (i & 1) * 32 + lane;
        Turn<R> now(i / 2);
        for (;;) {
            if (!wait(&sh.full[now.s], now.parity, kStatusScanFull) || sh.place[now.s].b < 0) break;
            if (!wait(&sh.summed[now.s], now.parity, kStatusScanSums)) break;
            pass.chain(sh.place[now.s], sh.tile[now.s], channel);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.started[now.s]);
                sh.control[0] = sh.control[0] + 1u;
            }
            now.step(kPairs<LOOK>);
        }
    } else {
        Tiles<LOOK, REVERSE> tiles(p);
        Turn<R> now(0);
        constexpr int kEnds = kGroups > kPairs<LOOK> ? kGroups : kPairs<LOOK>;  // every group and every pair meets an end
        int ends = 0;
        Place at;
        at.b = 0;
        for (int i = 0; ends < kEnds; ++i) {
            if (i >= R && !wait(&sh.empty[now.s], now.parity ^ 1u, kStatusScanEmpty)) break;
            if (at.b >= 0) at = tiles.next(p);
            if (lane == 0) {
                sh.place[now.s] = at;
                if (at.b >= 0 && at.n > 0 && p.boxes) {
                    mbar_arrive_expect_tx(&sh.full[now.s], TILE::kBoxBytes);
                    pass.load(at, sh.tile[now.s], &sh.full[now.s]);
                } else {
                    mbar_arrive(&sh.full[now.s]);
                }
            }
            ends += at.b < 0;
            now.step(1);
        }
    }
    if (sh.control[1]) {  // after a wait that gave up, copies into this block's shared memory may still be in flight: a bounded time for them
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {
        }
    }
}

// A warp's rows of a tile: how many there are, and the first one's place.
__device__ __forceinline__ int rows_of(const Place& at, int warp, long long& row) {
    const int row0 = at.tile * kRows + warp * kPer;
    row = (long long)at.first + row0;
    return min(max(at.n - row0, 0), kPer);
}

template <bool LOOK, bool GB, bool XB>
struct Forward {
    using TILE = ForwardTile<GB, XB>;
    const ScanParams& p;
    float walk = 0.0f;  // a walking block's state between its tiles
    __device__ __forceinline__ explicit Forward(const ScanParams& q) : p(q) {}
    __device__ __forceinline__ void load(const Place& at, TILE& t, uint64_t* bar) const {
        const int c = at.stripe * kChannels, row = at.first + at.tile * kRows;
        t.g.box(p.tm_g, c, row, bar);
        t.x.box(p.tm_x, c, row, bar);
    }
    __device__ __forceinline__ void ask(const Place& at, TILE& t, int w) const {
        long long row;
        const int m = rows_of(at, w, row), c = at.stripe * kChannels + 2 * (threadIdx.x & 31);
        t.g.ask(w, Walk(p.g, row, p.g_stride, c, kBytes<GB>), m, p.channels - c, p.vec);
        t.x.ask(w, Walk(p.x, row, p.x_stride, c, kBytes<XB>), m, p.channels - c, p.vec);
    }
    __device__ __forceinline__ void sum(const Place& at, TILE& t, int w) const {
        long long row;
        const int m = rows_of(at, w, row), lane = threadIdx.x & 31;
        float2 A = two(1.0f), B = two(0.0f);
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
            constexpr bool S = decltype(sigmoid)::value, C = decltype(complement)::value;
#pragma unroll
            for (int r = 0; r < kPer; ++r) {
                float2 a, rest, b = t.x.get(w, r);
                gate<S, C>(t.g.get(w, r), a, rest);
                if constexpr (C) b = mul2(rest, b);
                if (r < m) A = mul2(A, a), B = fma2(a, B, b);  // rows past the end leave the state as it is
            }
        });
        reinterpret_cast<float4*>(t.sums[w])[lane] = make_float4(A.x, B.x, A.y, B.y);
    }
    __device__ __forceinline__ void chain(const Place& at, TILE& t, int channel) {
        const int c = at.stripe * kChannels + channel;
        const bool ok = c < p.channels;
        float TA = 1.0f, TB = 0.0f, h = at.tile == 0 ? (ok ? p.state_in[p.state_off[at.b] + c] : 0.0f) : walk;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ab = t.sums[w][channel];
            TA *= ab.x, TB = fmaf(ab.x, TB, ab.y);
        }
        if constexpr (LOOK) h = join<-1>(p, at.slot, at.stripe, channel, at.tile, TA, TB, h, at.tile + 1 < at.tiles);
        else walk = fmaf(TA, h, TB);
        if (p.saves != nullptr && ok) p.saves[(long long)at.slot * p.channels + c] = h;
        if (at.n == 0 && ok) p.state_out[p.state_off[at.b] + c] = h;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ab = t.sums[w][channel];
            t.sums[w][channel].x = h;
            h = fmaf(ab.x, h, ab.y);
        }
    }
    __device__ __forceinline__ void finish(const Place& at, const TILE& t, int w) const {
        long long row;
        const int m = rows_of(at, w, row), lane = threadIdx.x & 31, c = at.stripe * kChannels + 2 * lane, valid = p.channels - c;
        if (m == 0) return;
        const float4 s = reinterpret_cast<const float4*>(t.sums[w])[lane];
        float2 h = make_float2(s.x, s.z);
        Walk out(p.out, row, p.out_stride, c, kBytes<XB>);
        const bool vec = p.vec, write = p.out != nullptr;
        // (The gates of all rows before the first store: the compiler moves no load from shared memory over a store, and a row would wait for the one before it.)
        float2 a[kPer], b[kPer];
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
            constexpr bool S = decltype(sigmoid)::value, C = decltype(complement)::value;
#pragma unroll
            for (int r = 0; r < kPer; ++r) {
                float2 rest;
                b[r] = t.x.get(w, r);
                gate<S, C>(t.g.get(w, r), a[r], rest);
                if constexpr (C) b[r] = mul2(rest, b[r]);
            }
        });
        if (m == kPer && vec && valid > 0 && write) {
#pragma unroll
            for (int r = 0; r < kPer; ++r, out.at += out.step) {
                h = fma2(a[r], h, b[r]);
                store_pair<XB>(out.at, 2, true, h.x, h.y);
            }
        } else {
#pragma unroll
            for (int r = 0; r < kPer; ++r, out.at += out.step) {
                if (r >= m) break;
                h = fma2(a[r], h, b[r]);
                if (write) store_pair<XB>(out.at, valid, vec, h.x, h.y);
            }
        }
        if (at.tile * kRows + w * kPer + m == at.n) {
            float* to = p.state_out + p.state_off[at.b] + c;
            if (valid > 0) to[0] = h.x;
            if (valid > 1) to[1] = h.y;
        }
    }
};

// As the forward pass from the other end, e in h's place: D_t = dy_t + e_t, e_{t-1} = a_t D_t.  The h of the tile's rows are formed again from the saved state at its start.
template <bool LOOK, bool GB, bool XB>
struct Backward {
    using TILE = BackwardTile<GB, XB>;
    const ScanParams& p;
    float walk = 0.0f;
    __device__ __forceinline__ explicit Backward(const ScanParams& q) : p(q) {}
    __device__ __forceinline__ void load(const Place& at, TILE& t, uint64_t* bar) const {
        const int c = at.stripe * kChannels, row = at.first + at.tile * kRows;
        t.g.box(p.tm_g, c, row, bar);
        t.x.box(p.tm_x, c, row, bar);
        t.dy.box(p.tm_dout, c, row, bar);
    }
    __device__ __forceinline__ void ask(const Place& at, TILE& t, int w) const {
        long long row;
        const int m = rows_of(at, w, row), c = at.stripe * kChannels + 2 * (threadIdx.x & 31);
        t.g.ask(w, Walk(p.g, row, p.g_stride, c, kBytes<GB>), m, p.channels - c, p.vec);
        t.x.ask(w, Walk(p.x, row, p.x_stride, c, kBytes<XB>), m, p.channels - c, p.vec);
        t.dy.ask(w, Walk(p.dout, row, p.dout_stride, c, kBytes<XB>), m, p.channels - c, p.vec);
    }
    __device__ __forceinline__ void sum(const Place& at, TILE& t, int w) const {
        long long row;
        const int m = rows_of(at, w, row), lane = threadIdx.x & 31;
        float2 A = two(1.0f), B = two(0.0f), F = two(0.0f);
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
            constexpr bool S = decltype(sigmoid)::value, C = decltype(complement)::value;
#pragma unroll
            for (int r = 0; r < kPer; ++r) {
                float2 a, rest, b = t.x.get(w, r);
                gate<S, C>(t.g.get(w, r), a, rest);
                if constexpr (C) b = mul2(rest, b);
                if (r < m) {
                    A = mul2(A, a), B = fma2(a, B, b);
                    F = fma2(A, t.dy.get(w, r), F);  // sum of a_0 .. a_r dy_r: what reaches the rows before these
                }
            }
        });
        reinterpret_cast<float4*>(t.sums[w])[lane] = make_float4(A.x, B.x, A.y, B.y);
        reinterpret_cast<float2*>(t.back[w])[lane] = F;
    }
    __device__ __forceinline__ void chain(const Place& at, TILE& t, int channel) {
        const int c = at.stripe * kChannels + channel;
        const bool ok = c < p.channels;
        float h = ok ? __ldg(p.saves + (long long)at.slot * p.channels + c) : 0.0f;
        float TA = 1.0f, TF = 0.0f, e = at.tile + 1 == at.tiles ? (ok && p.state_in != nullptr ? p.state_in[p.state_off[at.b] + c] : 0.0f) : walk;
#pragma unroll
        for (int w = kWarps - 1; w >= 0; --w) {
            const float a = t.sums[w][channel].x;
            TA *= a, TF = fmaf(a, TF, t.back[w][channel]);
        }
        if constexpr (LOOK) e = join<1>(p, at.slot, at.stripe, channel, at.tiles - 1 - at.tile, TA, TF, e, at.tile > 0);
        else walk = fmaf(TA, e, TF);
        if (at.n == 0 && ok && p.state_out != nullptr) p.state_out[p.state_off[at.b] + c] = e;
        float A[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ab = t.sums[w][channel];
            t.sums[w][channel].x = h;
            h = fmaf(ab.x, h, ab.y);
            A[w] = ab.x;
        }
#pragma unroll
        for (int w = kWarps - 1; w >= 0; --w) {
            const float f = t.back[w][channel];
            t.back[w][channel] = e;
            e = fmaf(A[w], e, f);
        }
    }
    __device__ __forceinline__ void finish(const Place& at, const TILE& t, int w) const {
        long long row;
        const int m = rows_of(at, w, row), lane = threadIdx.x & 31, c = at.stripe * kChannels + 2 * lane, valid = p.channels - c;
        if (m == 0) return;
        const float4 s = reinterpret_cast<const float4*>(t.sums[w])[lane];
        float2 h = make_float2(s.x, s.z), e = reinterpret_cast<const float2*>(t.back[w])[lane];
        Walk dxs(p.dx, row + kPer - 1, p.dx_stride, c, kBytes<XB>), dgs(p.dg, row + kPer - 1, p.dg_stride, c, kBytes<GB>);
        const bool vec = p.vec;
        with_flags(p.flags, [&](auto sigmoid, auto complement) {
            constexpr bool S = decltype(sigmoid)::value, C = decltype(complement)::value;
            float2 a[kPer], from[kPer], rest[kPer];  // from: h before the row, less x where the gate decides over both
#pragma unroll
            for (int r = 0; r < kPer; ++r) {
                const float2 x = t.x.get(w, r);
                gate<S, C>(t.g.get(w, r), a[r], rest[r]);
                from[r] = C ? make_float2(h.x - x.x, h.y - x.y) : h;
                h = fma2(a[r], h, C ? mul2(rest[r], x) : x);
            }
#pragma unroll
            for (int r = kPer - 1; r >= 0; --r, dxs.at -= dxs.step, dgs.at -= dgs.step) {
                if (r >= m) continue;
                const float2 dy = t.dy.get(w, r), d = make_float2(dy.x + e.x, dy.y + e.y), slope = S ? mul2(a[r], rest[r]) : a[r];
                const float2 dx = C ? mul2(rest[r], d) : d, dg = mul2(mul2(d, slope), from[r]);
                e = mul2(a[r], d);
                store_pair<XB>(dxs.at, valid, vec, dx.x, dx.y);
                store_pair<GB>(dgs.at, valid, vec, dg.x, dg.y);
            }
        });
        if (at.tile == 0 && w == 0 && p.state_out != nullptr) {
            float* to = p.state_out + p.state_off[at.b] + c;
            if (valid > 0) to[0] = e.x;
            if (valid > 1) to[1] = e.y;
        }
    }
};

template <bool LOOK, bool GB, bool XB>
__global__ void __launch_bounds__(kThreads<LOOK>, 1) scan_forward_kernel(const __grid_constant__ ScanParams p) {
    Forward<LOOK, GB, XB> pass(p);
    run<ForwardTile<GB, XB>, LOOK, false>(p, pass);
}
template <bool LOOK, bool GB, bool XB>
__global__ void __launch_bounds__(kThreads<LOOK>, 1) scan_backward_kernel(const __grid_constant__ ScanParams p) {
    Backward<LOOK, GB, XB> pass(p);
    run<BackwardTile<GB, XB>, LOOK, true>(p, pass);
}

// Row by row, two channels a thread, eight rows' loads in flight.
constexpr int kStepThreads = 128;
template <bool GB, bool XB>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(const __grid_constant__ ScanParams p) {
    grid_ready();
    const int parts = (p.channels + 2 * kStepThreads - 1) / (2 * kStepThreads);
    const int b = blockIdx.x / parts, c0 = (int)(blockIdx.x % parts) * 2 * kStepThreads + 2 * (int)threadIdx.x, valid = min(p.channels - c0, 2);
    if (valid <= 0) return;
    const int first = __ldg(p.cu + b);
    int n = max(__ldg(p.cu + b + 1) - first, 0);
    if (p.keep != nullptr) n = min(n, max(__ldg(p.keep + b), 0));
    const long long off = p.state_off[b] + c0;
    float2 h = make_float2(p.state_in[off], valid > 1 ? p.state_in[off + 1] : 0.0f);
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
                float2 a, rest, b = x[r].get();
                gate<decltype(sigmoid)::value, decltype(complement)::value>(g[r].get(), a, rest);
                if constexpr (decltype(complement)::value) b = mul2(rest, b);
                h = fma2(a, h, b);
                if (p.out != nullptr) store_pair<XB>(out.at, valid, p.vec, h.x, h.y);
            }
        });
    }
    if (p.state_out != nullptr) {
        p.state_out[off] = h.x;
        if (valid > 1) p.state_out[off + 1] = h.y;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
constexpr int kAllFlags = GLM53F_KDA_SCAN_SIGMOID | GLM53F_KDA_SCAN_COMPLEMENT | GLM53F_KDA_SCAN_G_BF16 | GLM53F_KDA_SCAN_X_BF16;

struct Layout {  // of the workspace: bytes from its start
    long long slots, stripes, records, bytes;
    Layout(int64_t channels, int64_t batch, int64_t rows) {
        slots = rows / kRows + batch;
        stripes = (channels + kChannels - 1) / kChannels;
        records = 256;
        bytes = records + slots * stripes * kChannels * (long long)sizeof(Record);
    }
};

// Whether a call's sequences are divided, or one block walks each 64 channels of a sequence.  A walked tile has nothing to wait for: 0.6 us by itself and 0.87 with all SMs at it, against
// 1.3 us a tile of an SM's share and 5 us more where tiles look back; without tensor copies 1.3 to 3.1 us against 1.9 to 3.5.  A walk takes as long as its
// busiest block.  Measured, us walked and divided (f32 g, bf16 x): 4,096 channels 100 rows 4.0 and 6.4, 2,000 rows 22.6 and 23.6, 4,000 rows 39.9 and 38.1, 8,192 rows 76 and 69;
// 1,024 channels 1,000 rows 11.6 and 9.2, 16 x 1,000 rows 27 and 43; 64 channels 300 rows 5.4 and 5.8, 3,000 rows 29 and 7.6; there and back 2,048 channels, 16,289 rows in four sequences 163 and 200;
// 1,001 channels (no tensor copies) 1,000 rows 41 and 13.  Backwards alone: 4,096 channels 100 rows 4.4 and 7.0, 8,192 rows 138 and 109; 1,024 channels 1,000 rows 18 and 12, 16 x 1,000 rows 47 and 65, 65,536 rows
// 989 and 241; 64 channels 3,000 rows 43 and 8; four sequences as above 87 and 116; the rule's losses: 4,096 channels 2,000 rows 38 and 33, 64 channels 300 rows 6.8 and 6.3, both walked.
bool divide(const Layout& at, int batch, int max_len, bool boxes) {
    if (max_len <= kRows) return false;
    const long long items = at.stripes * batch, sms = sm_count(), longest = (max_len + kRows - 1) / kRows, tiles = at.slots * at.stripes;
    const long long share = (tiles + sms - 1) / sms;
    const long long walked = items <= sms || share + longest / 2 < longest ? longest : share + longest / 2;  // by the busiest block
    return walked > (boxes ? 2 * share + 7 : share + 2);
}

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

// A map of rows that lie on 16 bytes, for boxes of a tile.
bool row_boxes(CUtensorMap* tm, const Matrix& m, int channels, int rows) {
    const long long size = m.bf16 ? 2 : 4;
    EncodeTiled enc = encode_tiled();
    if (enc == nullptr || rows < 1 || (reinterpret_cast<uintptr_t>(m.p) & 15) || m.stride * size % 16) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)channels, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(m.stride * size)};
    const cuuint32_t box[2] = {kChannels, kRows}, estr[2] = {1u, 1u};
    return enc(tm, m.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(m.p), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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

// The launch over tiles: with sequences of more than one tile and a workspace that holds what tiles say, taken from the counter; else a block walks (sequence, stripe) after
// (sequence, stripe).
template <bool BACKWARD>
int tiles_launch(ScanParams& p, int max_len, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    const Layout at(p.channels, p.batch, p.rows);
    if (at.stripes * p.batch > 0x7fffffff || at.slots * at.stripes > 0x7fffffff) return kInvalid;
    p.stripes = (int)at.stripes;
    p.status = status_word();
    if (p.status == nullptr) return (int)cudaErrorUnknown;
    const bool gb = p.flags & GLM53F_KDA_SCAN_G_BF16, xb = p.flags & GLM53F_KDA_SCAN_X_BF16;
    p.boxes = row_boxes(&p.tm_g, {p.g, p.g_stride, gb}, p.channels, p.rows) && row_boxes(&p.tm_x, {p.x, p.x_stride, xb}, p.channels, p.rows) &&
              (!BACKWARD || row_boxes(&p.tm_dout, {p.dout, p.dout_stride, xb}, p.channels, p.rows));
    p.tiles = at.stripes * p.batch;
    const bool look = workspace != nullptr && workspace_bytes >= at.bytes && divide(at, p.batch, max_len, p.boxes);
    if (look) {
        auto* w = static_cast<unsigned char*>(workspace);
        p.control = reinterpret_cast<unsigned*>(w);
        p.records = reinterpret_cast<Record*>(w + at.records);
        p.slots = (int)at.slots;
        p.tiles = at.slots * at.stripes;
        const long long clear = (p.tiles * kChannels + 1023) / 1024, some = 4ll * sm_count();
        const int rc = launch_early(scan_clear_kernel, dim3((unsigned)(clear < some ? clear : some)), 256, 0, stream, p);
        if (rc != 0) return rc;
    }
    const long long blocks = p.tiles < sm_count() ? p.tiles : sm_count();
    return with_types(p.flags, look, [&](auto l, auto g_bf16, auto x_bf16) {
        constexpr bool L = decltype(l)::value, G = decltype(g_bf16)::value, X = decltype(x_bf16)::value;
        auto launch = [&](auto kernel, size_t shared) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
            if (e != cudaSuccess) return (int)e;
            return launch_early(kernel, dim3((unsigned)blocks), kThreads<L>, shared, stream, p);
        };
        if constexpr (BACKWARD) return launch(scan_backward_kernel<L, G, X>, sizeof(Shared<BackwardTile<G, X>>));
        else return launch(scan_forward_kernel<L, G, X>, sizeof(Shared<ForwardTile<G, X>>));
    });
}

bool common_ok(int32_t channels, int32_t batch, const int32_t* cu, int32_t flags) {
    return channels >= 1 && channels <= kMost && batch >= 0 && (flags & ~kAllFlags) == 0 && (batch == 0 || cu != nullptr);
}
bool state_ok(const void* state) { return state != nullptr && (reinterpret_cast<uintptr_t>(state) & 3) == 0; }

}  // namespace
}  // namespace kda

extern "C" int64_t glm53f_kda_scan_workspace_bytes(int32_t channels, int32_t batch, int32_t rows) {
    using namespace kda;
    if (channels < 1 || channels > kMost || batch < 1 || rows < 0 || rows > kMost) return 0;
    return Layout(channels, batch, rows).bytes;
}

extern "C" int64_t glm53f_kda_scan_saves_rows(int32_t batch, int32_t rows) { return batch < 1 || rows < 0 ? 0 : (int64_t)rows / kda::kRows + batch; }

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
    if (!common_ok(channels, batch, cu_rows, flags) || rows < 0 || rows > kMost || max_len < 0 || max_len > rows || workspace_bytes < 0) return kInvalid;
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
    if (!common_ok(channels, batch, cu_rows, flags) || rows < 0 || rows > kMost || max_len < 0 || max_len > rows || workspace_bytes < 0) return kInvalid;
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
