// recurrence.cu -- the gated linear recurrence: forward over a sequence, its
// backward pass, and the single-token step.  Per (batch row, time, channel):
//   s = sigmoid(r),  y = c softplus(lambda) s,  a = exp(-y),
//   beta = sqrt(1 - a^2),   h_t = keep_t a h_{t-1} + beta sigmoid(i) x
// (keep_t = 0 where a reset cuts the state, else 1).
//
// Backward, with G_t = dL/dh_t including what later tokens pass back:
//   G_t = dh_t + C_{t+1},  C_t = keep_t a_t G_t,
//   dx = G beta sigmoid(i),  di = dx x (1 - sigmoid(i)),
//   E  = y dL/dy = G (sigmoid(i) x a^2 (y / beta) - y a keep h_{t-1}),
//   dr = E (1 - s),  dlambda = sigmoid(lambda)/softplus(lambda) sum E.
// Writing the decay's gradient as E = y dL/dy keeps y / beta = O(sqrt(y))
// in place of 1 / beta, so gates that close completely (y = 0) give 0.
#include "common.cuh"
#include "internal.h"
#include "scan_math.cuh"
#include "tma.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>
#include <utility>
#include <vector>

namespace mb {

__device__ unsigned int g_recurrence_error = 0;

namespace {

// ---- gates ------------------------------------------------------------------
// Two elements at a time in packed FP32 (one issue slot per pair and
// operation); what is left per element are the special-function operations,
// five forward and seven backward (FP16 tensors eight).  Approximate exponentials, reciprocals and
// roots have relative errors of 2^-22 or less.  PRECISE (FP32 tensors) adds
// what their rounding needs: the exponent's product with log2(e) in two parts
// and a longer series.  For FP16 tensors the rounding to 2^-11 hides both: in
// the gates, which count once, while the decay counts for as long as the FP32
// state lives and is right to its last place for all (decay_of).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN operand stays one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float rsqrt_approx(float v) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// exp(-v), v above -120 and, PRECISE, below 1e30.
template <bool PRECISE>
__device__ __forceinline__ float2 exp_neg(float2 v) {
    const float2 t = __fmul2_rn(v, both(kLog2e));
    float2 e = make_float2(ex2_approx(-t.x), ex2_approx(-t.y));
    if (PRECISE) {  // 2^-(v log2 e) = 2^-t (1 + ln 2 d), d = t - v log2 e with log2 e in two parts
        float2 d = __ffma2_rn(v, both(-kLog2e), t);
        d = __ffma2_rn(v, both(-1.92596303e-8f), d);
        e = __ffma2_rn(e, __fmul2_rn(d, both(kLn2)), e);
    }
    return e;
}

// The decay gate's preactivation, held where exp(-v) is finite: sigmoid(-80) =
// 2e-35 and sigmoid(150) = 1 stand for what lies beyond.
template <bool PRECISE, bool BELOW = true>
__device__ __forceinline__ float2 clamp_gate(float2 v) {
    if (BELOW) v = make_float2(max_nan(v.x, -80.f), max_nan(v.y, -80.f));
    if (PRECISE) v = make_float2(min_nan(v.x, 150.f), min_nan(v.y, 150.f));
    return v;
}

// E = exp(v) of the input gate, sigmoid(v) = E / (1 + E), 1 - sigmoid(v) = 1 / (1 +
// E): right down to the smallest normal E, v held from above only (at `top`,
// where E and its products stay finite).
template <bool PRECISE>
__device__ __forceinline__ float2 exp_gate(float2 v, float top) {
    v = make_float2(max_nan(-v.x, -top), max_nan(-v.y, -top));
    if (PRECISE) v = make_float2(min_nan(v.x, 150.f), min_nan(v.y, 150.f));
    return exp_neg<PRECISE>(v);
}

// a = exp(-y) and m = 1 - a^2, m without cancellation for y near 0 and a
// rounded once there: an approximate exponential is off by up to 2^-23 and on
// average by a quarter of 2^-24, which adds up over the tokens that an FP32
// state lives.  So near 0 both come from d = 1 - a by its Taylor series, a = 1 -
// d and m = d (2 - d).
// PRECISE: below y = 1/2 the series to y^9 (relative error < (1/2)^9 / 10! =
// 6e-10); above, d = 1 - exp(-y): 2^-22 a / (1 - a) < 4e-7.
// Else: a series to y^5 and an exponential made 5 * 2^-24 too small, which is
// more than it is ever off: both bound a from below, so the larger one is
// right everywhere, without comparing and selecting.  Worst where they meet,
// near y = 0.25: 6e-7 of a, 3e-6 of m.  With the plain exponential instead, up to
// 1.4 * 2^-24 off near 1, 8 x 4096 x 4096 took 248 us, with the series 255;
// backward 8 x 2048 x 4096 271 and 292.
template <bool PRECISE>
__device__ __forceinline__ void decay_of(float2 y, float2 &a, float2 &m) {
    if (PRECISE) {
        const float2 e = exp_neg<PRECISE>(y);
        float2 q = __ffma2_rn(y, both(1.f / 362880), both(-1.f / 40320));
        q = __ffma2_rn(y, q, both(1.f / 5040));
        q = __ffma2_rn(y, q, both(-1.f / 720));
        q = __ffma2_rn(y, q, both(1.f / 120));
        q = __ffma2_rn(y, q, both(-1.f / 24));
        q = __ffma2_rn(y, q, both(1.f / 6));
        q = __ffma2_rn(y, q, both(-0.5f));
        q = __ffma2_rn(y, q, both(1.f));
        const float2 s = __fmul2_rn(y, q), l = __ffma2_rn(e, both(-1.f), both(1.f));
        const float2 d = make_float2(y.x < 0.5f ? s.x : l.x, y.y < 0.5f ? s.y : l.y);
        const float2 r = __ffma2_rn(d, both(-1.f), both(1.f));
        a = make_float2(y.x < 0.5f ? r.x : e.x, y.y < 0.5f ? r.y : e.y);
        m = __fmul2_rn(d, __ffma2_rn(d, both(-1.f), both(2.f)));
    } else {
        const float2 t = __ffma2_rn(y, both(-kLog2e), both(-5 * kLog2e / 16777216));
        const float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
        float2 q = __ffma2_rn(y, both(-1.f / 120), both(1.f / 24));
        q = __ffma2_rn(y, q, both(-1.f / 6));
        q = __ffma2_rn(y, q, both(0.5f));
        q = __ffma2_rn(y, q, both(-1.f));
        const float2 r = __ffma2_rn(y, q, both(1.f)), s = __fmul2_rn(y, q), l = __fadd2_rn(e, both(-1.f));
        a = make_float2(fmaxf(r.x, e.x), fmaxf(r.y, e.y));
        const float2 d = make_float2(fmaxf(s.x, l.x), fmaxf(s.y, l.y));  // a - 1
        m = __fmul2_rn(d, __ffma2_rn(d, both(-1.f), both(-2.f)));
    }
}

// 1 / sqrt(m + 1e-37): finite for m = 0, where m times it is 0 as it should be.
constexpr float kTiny = 1e-37f;

// 1 / (1 + e): sigmoid(v) for e = exp(-v).
__device__ __forceinline__ float2 sigmoid_of(float2 e) {
    const float2 q = __fadd2_rn(e, both(1.f));
    return make_float2(rcp_approx(q.x), rcp_approx(q.y));
}

// e = exp(-r), s = sigmoid(r) and the decay y = csp s, a = exp(-y), m = 1 - a^2.
// FINITE: so is e, and 1 - s = e s; else infinity just gives s = 0.
template <bool PRECISE, bool FINITE = PRECISE>
__device__ __forceinline__ void decay(float2 r, float2 csp, float2 &e, float2 &s, float2 &a, float2 &m) {
    e = exp_neg<PRECISE>(clamp_gate<PRECISE, FINITE>(r));
    s = sigmoid_of(e);
    decay_of<PRECISE>(__fmul2_rn(csp, s), a, m);
}

// Forward: a and b = sqrt(1 - a^2) sigmoid(i) x.  With E = exp(i), q = 1 + E and
// m = 1 - a^2, sqrt(m) / q = m / sqrt(m q^2): one root for both.  sigmoid(20) is 1
// to 2e-9, a fraction of a step of FP32, and q^2 finite.
template <bool PRECISE>
__device__ __forceinline__ void forward_gates(float2 r, float2 i, float2 x, float2 csp, float2 &a, float2 &b) {
    float2 e, s, m;
    decay<PRECISE>(r, csp, e, s, a, m);
    const float2 E = exp_gate<PRECISE>(i, 20.f), q = __fadd2_rn(E, both(1.f));
    const float2 t = __ffma2_rn(__fmul2_rn(m, q), q, both(kTiny));
    const float2 w = __fmul2_rn(m, make_float2(rsqrt_approx(t.x), rsqrt_approx(t.y)));
    // FP16: E x is finite.  FP32: w x is at most x.
    b = PRECISE ? __fmul2_rn(__fmul2_rn(w, x), E) : __fmul2_rn(w, __fmul2_rn(E, x));
}

// softplus(lambda), and c times it (finite: 0 times it has to be 0), once per
// channel and call.
__device__ __forceinline__ float channel_softplus(float l) { return fmaxf(l, 0.f) + log1pf(expf(-fabsf(l))); }
__device__ __forceinline__ float channel_decay(float c, float l) { return min_nan(c * channel_softplus(l), 1e30f); }

struct FwdParams {
    const void *x, *r, *i;
    const float *lambda, *h0;
    const int32_t *lengths;
    const uint8_t *resets;
    void *h;
    float *hN;
    int B, L, D;
    float c;
    unsigned row_first;  // per tensor map: see fetch_box
    int64_t sx[2], sr[2], si[2], sh[2];
};
struct BwdParams {
    FwdParams f;
    const void *dh;
    const float *dhN;
    void *dx, *dr, *di;
    float *dh0, *part;
    int64_t sdh[2], sdx[2], sdr[2], sdi[2];
};

__device__ __forceinline__ int row_length(const FwdParams &p, int b) {
    return p.lengths ? min(max(p.lengths[b], 0), p.L) : p.L;
}

constexpr int kThreads = 128;

// ---- tiles of a sequence ----------------------------------------------------
// A CTA of W warps owns one tile of the time axis, W * S tokens of 32 * VEC
// channels; warp w holds S consecutive tokens in registers.  The recurrence is
// affine in the state that enters a span, h_out = P h_in + H, so
//   1. each warp reduces its S tokens to (P, H), and the warps' maps are
//      composed through shared memory into the tile's,
//   2. the state entering the tile comes from the tiles before it, and
//   3. each warp walks its S tokens again, from registers, and writes h.
// Every tensor is read and written once, for any split of the time axis.
//
// Step 2 crosses CTAs.  Tiles are handed out by an atomic ticket, time-major
// (all rows' and channels' first tiles, then all second ones), so every tile
// before a running one is running or done and waiting for it ends.  Tiles form
// groups: a tile publishes its map to the later tiles of its group, and the
// group's last tile publishes the state leaving the group.  So the serial
// chain over a long sequence has one hop per group, each tile composes the
// same maps in the same order on every run (a scheme that takes whatever state
// is ready first would not), and results repeat bit for bit.
// A published value is one machine word that says itself whether it is there:
// the workspace starts as all ones bits (a NaN that no published value has).
constexpr int kMaxGroupShift = 4;
constexpr unsigned kErrRecurrenceTimeout = 64u;
constexpr uint32_t kEmpty = 0xffffffffu;

__device__ __forceinline__ float published(float v) {  // never the empty pattern
    return __float_as_uint(v) == kEmpty ? __uint_as_float(0x7fffffffu) : v;
}
__device__ __forceinline__ void put_map(float2 *slot, float P, float H) {
    const uint64_t w = (uint64_t)__float_as_uint(H) << 32 | __float_as_uint(published(P));
    asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(slot), "l"(w) : "memory");
}
__device__ __forceinline__ void put_state(float *slot, float h) {
    asm volatile("st.relaxed.gpu.global.b32 [%0], %1;" ::"l"(slot), "r"(__float_as_uint(published(h))) : "memory");
}
__device__ __forceinline__ uint64_t get_map(const float2 *slot) {
    uint64_t w;
    asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w) : "l"(slot) : "memory");
    return w;
}
__device__ __forceinline__ uint32_t get_state(const float *slot) {
    uint32_t w;
    asm volatile("ld.relaxed.gpu.global.b32 %0, [%1];" : "=r"(w) : "l"(slot) : "memory");
    return w;
}

// Bounded wait: 2 s, or at once after a wait of this call ran out (`gave_up`, a
// word of the call's workspace, is then no longer empty).
constexpr uint64_t kWaitNs = 2000000000ull;
struct Waiting {
    uint32_t *gave_up;
    uint64_t limit_ns, t0 = 0;
    int spins = 0;
    __device__ __forceinline__ Waiting(uint32_t *g, uint64_t limit) : gave_up(g), limit_ns(limit) {}
    __device__ __forceinline__ bool again() {
        if ((++spins & 63) == 0) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > limit_ns || *(volatile uint32_t *)gave_up != kEmpty) {
                *(volatile uint32_t *)gave_up = 0;
                atomicOr(&g_recurrence_error, kErrRecurrenceTimeout);
                return false;
            }
        }
        return true;
    }
};

// VEC consecutive elements.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
    return *reinterpret_cast<const Pack<T, VEC> *>(p);
}

// Affine maps h -> P h + H of a thread's channels.  A reset drops what enters
// even where that is infinite or NaN, so it is not P = 0 but a set sign bit of P
// (products of decays, which have none, keep it); CUTS: whether the call has
// resets at all.  with_flag turns a run-time flag into such a template argument.
template <typename F>
__device__ __forceinline__ void with_flag(bool flag, F &&f) {
    if (flag)
        f(std::true_type());
    else
        f(std::false_type());
}
__device__ __forceinline__ bool is_cut(float P) { return __float_as_int(P) < 0; }
template <int VEC>
struct Maps {
    Pack<float, VEC> P, H;
    __device__ __forceinline__ void identity() {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            P.v[e] = 1.f;
            H.v[e] = 0.f;
        }
    }
    // a reset: nothing of the state passes
    __device__ __forceinline__ void cut() {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            P.v[e] = -1.f;
            H.v[e] = 0.f;
        }
    }
    // then q, later in time
    template <bool CUTS = false>
    __device__ __forceinline__ void then(const Pack<float, VEC> &qP, const Pack<float, VEC> &qH) {
        if constexpr (VEC == 1) {
            H.v[0] = fmaf(qP.v[0], H.v[0], qH.v[0]);
            P.v[0] *= qP.v[0];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float2 p = make_float2(qP.v[e], qP.v[e + 1]);
                const float2 h = __ffma2_rn(p, make_float2(H.v[e], H.v[e + 1]), make_float2(qH.v[e], qH.v[e + 1]));
                const float2 n = __fmul2_rn(p, make_float2(P.v[e], P.v[e + 1]));
                H.v[e] = h.x;
                H.v[e + 1] = h.y;
                P.v[e] = n.x;
                P.v[e + 1] = n.y;
            }
        }
        if (CUTS)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (is_cut(qP.v[e])) {
                    P.v[e] = qP.v[e];
                    H.v[e] = qH.v[e];
                }
    }
    __device__ __forceinline__ void apply(const float (&s)[VEC], float (&h)[VEC], bool cuts) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            h[e] = fmaf(P.v[e], s[e], H.v[e]);
            if (cuts && is_cut(P.v[e])) h[e] = H.v[e];
        }
    }
};
// A CTA's maps in shared memory, by warp or by tile of the group.
template <int VEC, int N>
struct MapRows {
    Pack<float, VEC> P[N][32], H[N][32];
};

template <int VEC>
__device__ __forceinline__ void wait_maps(const float2 *slot, uint32_t *gave_up, Pack<float, VEC> &P,
                                          Pack<float, VEC> &H, uint64_t limit_ns = kWaitNs) {
    Waiting wt(gave_up, limit_ns);
    bool ready;
    do {
        uint64_t w[VEC];
        ready = true;
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[k] = get_map(slot + k);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            ready &= (uint32_t)w[k] != kEmpty;
            P.v[k] = __uint_as_float((uint32_t)w[k]);
            H.v[k] = __uint_as_float((uint32_t)(w[k] >> 32));
        }
    } while (!ready && wt.again());
}
template <int VEC>
__device__ __forceinline__ void wait_states(const float *slot, uint32_t *gave_up, float (&h)[VEC],
                                            uint64_t limit_ns = kWaitNs) {
    Waiting wt(gave_up, limit_ns);
    bool ready;
    do {
        uint32_t w[VEC];
        ready = true;
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[k] = get_state(slot + k);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            ready &= w[k] != kEmpty;
            h[k] = __uint_as_float(w[k]);
        }
    } while (!ready && wt.again());
}

// v / d by a product with floor(2^32 / d): at most one below the quotient.
struct Divisor {
    unsigned d, m;
    __device__ __forceinline__ unsigned divide(unsigned v, unsigned &rest) const {
        unsigned q = __umulhi(v, m);
        rest = v - q * d;
        if (rest >= d) {
            ++q;
            rest -= d;
        }
        return q;
    }
};

struct Chains {
    unsigned int *ticket;  // and behind it the word of Waiting
    float2 *maps;      // [chains, tiles, channels of a tile]
    float *states;     // [chains, groups, channels of a tile]
    const float *csp;  // [dim] c * softplus(lambda)
    Divisor blocks;    // channel blocks of a row
    Divisor chains;    // rows * blocks
    int tiles, groups, group, group_shift;  // tiles of a chain, in groups of `group` = 1 << group_shift
};

// Hands out tickets one ahead: next() gives the ticket drawn by the call
// before it (or at the start) and draws another, whose latency then hides
// behind a tile's work.  Each call syncs the CTA.
struct Tickets {
    unsigned int *counter, *shared;  // shared: two places, used in turn
    unsigned int ahead = 0, turn = 0;
    __device__ __forceinline__ Tickets(unsigned int *c, unsigned int *s) : counter(c), shared(s) {
        if (c && threadIdx.x == 0) ahead = atomicAdd(counter, 1u) + 1u;  // the counter starts as all ones bits
    }
    __device__ __forceinline__ unsigned int next() {
        turn ^= 1;
        if (threadIdx.x == 0) shared[turn] = ahead;
        __syncthreads();
        const unsigned int v = shared[turn];
        if (threadIdx.x == 0) ahead = atomicAdd(counter, 1u) + 1u;
        return v;
    }
};

// What a ticket stands for: time-major, all chains' k-th tiles together.
struct Tile {
    int chain, k, g, j, b, d, n, t0, cnt;  // tile k of its chain is tile j of group g
    bool live, in;
};
template <int VEC>
__device__ __forceinline__ Tile place_tile(const Chains &c, const FwdParams &p, unsigned v) {
    Tile t;
    unsigned chain, block;
    t.k = (int)c.chains.divide(v, chain);
    t.chain = (int)chain;
    t.g = t.k >> c.group_shift;
    t.j = t.k - (t.g << c.group_shift);
    t.b = (int)c.blocks.divide(chain, block);
    t.d = ((int)block * 32 + (threadIdx.x & 31)) * VEC;
    t.in = t.d < p.D;
    t.n = row_length(p, t.b);
    return t;
}

// The map from the state at the start of tile k's group to the state entering
// this warp's tokens.  Warps wait for the maps of the group's earlier tiles
// between them; `wm` holds the maps of this tile's warps.  Syncs the CTA.
template <int VEC, int W>
__device__ __forceinline__ Maps<VEC> prefix_maps(const Chains &c, const Tile &t, const MapRows<VEC, W> &wm,
                                                 MapRows<VEC, (1 << kMaxGroupShift) - 1> &gm, bool cuts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int j = t.j;
    for (int tile = warp; tile < j; tile += W) {
        Pack<float, VEC> P, H;
        wait_maps<VEC>(c.maps + ((int64_t)t.chain * c.tiles + t.k - j + tile) * (32 * VEC) + lane * VEC,
                       c.ticket + 1, P, H);
        gm.P[tile][lane] = P;
        gm.H[tile][lane] = H;
    }
    __syncthreads();
    Maps<VEC> m;
    m.identity();
    with_flag(cuts, [&](auto flag) {
        constexpr bool CUTS = decltype(flag)::value;
        for (int q = 0; q < j; ++q) m.template then<CUTS>(gm.P[q][lane], gm.H[q][lane]);
        for (int w = 0; w < warp; ++w) m.template then<CUTS>(wm.P[w][lane], wm.H[w][lane]);
    });
    return m;
}

// The state at the start of tile k's group, where a group went before it.
// Every warp waits for itself, so that the group's last warp can pass the
// state on without another barrier.
template <int VEC>
__device__ __forceinline__ void group_state(const Chains &c, const Tile &t, float (&s)[VEC]) {
    if (t.g > 0)
        wait_states<VEC>(c.states + ((int64_t)t.chain * c.groups + t.g - 1) * (32 * VEC) + (threadIdx.x & 31) * VEC,
                         c.ticket + 1, s);
}
template <int VEC>
__device__ __forceinline__ void leave_group(const Chains &c, const Tile &t, const float (&h)[VEC]) {
    float *slot = c.states + ((int64_t)t.chain * c.groups + t.g) * (32 * VEC) + (threadIdx.x & 31) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) put_state(slot + e, h[e]);
}

// The tile's own map (warp maps in order), published for the group's later tiles.
template <int VEC, int W>
__device__ __forceinline__ void publish_map(const Chains &c, const Tile &t, const MapRows<VEC, W> &wm, bool cuts) {
    const int lane = threadIdx.x & 31;
    Maps<VEC> m;
    m.identity();
    with_flag(cuts, [&](auto flag) {
#pragma unroll
        for (int w = 0; w < W; ++w) m.template then<decltype(flag)::value>(wm.P[w][lane], wm.H[w][lane]);
    });
    float2 *slot = c.maps + ((int64_t)t.chain * c.tiles + t.k) * (32 * VEC) + lane * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) put_map(slot + e, m.P.v[e], m.H.v[e]);
}

// WALK: the state entering this warp's tokens (h) and the state leaving the
// tile (s) from the state entering it (s), through the maps of the tile's warps.
template <int VEC, int W>
__device__ __forceinline__ void walk_state(const MapRows<VEC, W> &wm, float (&s)[VEC], float (&h)[VEC], bool cuts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    with_flag(cuts, [&](auto flag) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const Pack<float, VEC> P = wm.P[w][lane], H = wm.H[w][lane];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (w == warp) h[e] = s[e];
                s[e] = fmaf(P.v[e], s[e], H.v[e]);
                if (decltype(flag)::value && is_cut(P.v[e])) s[e] = H.v[e];
            }
        }
    });
}

// Which of this warp's tokens cut the state.
__device__ __forceinline__ uint32_t cut_mask(const FwdParams &p, int b, int t0, int cnt) {
    if (!p.resets) return 0;
    const int lane = threadIdx.x & 31;
    const bool z = lane < cnt && p.resets[(int64_t)b * p.L + t0 + lane] != 0;
    return __ballot_sync(0xffffffffu, z);
}

// ---- a tile's inputs in shared memory -----------------------------------------------
// N tensors of TT tokens x 32 * VEC channels, NB buffers in turn.  With TMA
// (16-byte aligned rows) one thread fetches a tile by one bulk tensor copy per
// tensor, completing on the buffer's mbarrier: no other thread spends an
// instruction on addresses.  Elsewhere each thread copies the elements that it
// will read itself.
template <typename T, int VEC, int TT, int N, int NB>
struct TileIn {
    alignas(128) Pack<T, VEC> v[NB][N][TT][32];
    alignas(16) uint64_t full[NB];
    LostCopies lost;
};
struct TileMaps {
    CUtensorMap m[5];
};
// Order of a tensor map's outer two dimensions: time then row, or row then
// time (the larger stride last).
__device__ __forceinline__ void fetch_box(void *dst, const CUtensorMap *map, uint64_t *bar, int d, int t, int b,
                                          bool row_first) {
    tma_load_3d(dst, map, bar, d, row_first ? b : t, row_first ? t : b);
}

// Waits for buffer `buf` in its `use`-th use.  A wait that runs out is reported;
// the CTA goes on, with wrong values.
__device__ __forceinline__ void await_box(uint64_t *full, int buf, uint32_t use, LostCopies *lost,
                                          uint64_t limit_ns = kWaitNs) {
    if (!await_copy(full, buf, use & 1, lost, limit_ns)) atomicOr(&g_recurrence_error, kErrRecurrenceTimeout);
}

// Without TMA: FP32 elements are copied to shared memory asynchronously.  FP16
// ones are too small for that; they wait in registers (held) and go to shared
// memory when their tile's turn comes (put_held).
template <typename T, int N, int S>
struct Held {
    T v[N][S];
};
template <typename T>
__device__ __forceinline__ void copy_one(Pack<T, 1> *dst, T &held, const T *src) {
    if constexpr (sizeof(T) == 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    else
        held = *src;
}
template <typename T, int N, int S, int TT>
__device__ __forceinline__ void put_held(Pack<T, 1> (&dst)[N][TT][32], const Held<T, N, S> &held, int row, int cnt) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (j < cnt) dst[k][row + j][threadIdx.x & 31].v[0] = held.v[k][j];
    }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's S x VEC elements in pairs: along the channels, or along time
// where it has one channel.  Element (token j, channel e) is number j * VEC + e.
template <typename T, int VEC, int S>
__device__ __forceinline__ float2 pair_of(const Pack<T, VEC> (&in)[S], int q) {
    const int k = 2 * q;
    return make_float2(cvt_f32(in[k / VEC].v[k % VEC]), cvt_f32(in[(k + 1) / VEC].v[(k + 1) % VEC]));
}
template <int VEC>
__device__ __forceinline__ float2 channel_pair(const float (&v)[VEC], int q) {
    return make_float2(v[(2 * q) % VEC], v[(2 * q + 1) % VEC]);
}
__device__ __forceinline__ float &half_of(float2 &v, int k) { return k & 1 ? v.y : v.x; }

// ---- forward --------------------------------------------------------------------
// Persistent CTAs take tiles by ticket; the next tile's inputs are fetched once
// every warp has this tile's in registers, while it waits for its state and
// writes h.  With enough chains to fill the GPU
// (walks()), a CTA walks one chain from its first tile to its last instead
// (WALK): no tickets, nothing published, the state stays in registers.
// Bound by bytes for many warps (64 x 512 x 4096 FP16: 219 us, 4.9 TB/s), by
// latency below: 8 x 4096 x 4096 (512 chains, 12.5 warps an SM) 254 to 257 us
// with the special-function unit 57% and issue 49% busy; 1 x 131072 x 2048 FP32
// 806 us (5.3 TB/s).
template <typename T, int VEC, int S, int W, bool WALK>
struct FwdSmem {
    TileIn<T, VEC, S * W, 3, 1> in;
    MapRows<VEC, W> wm[WALK ? 2 : 1];
    MapRows<VEC, WALK ? 1 : (1 << kMaxGroupShift) - 1> gm;
    unsigned int ticket[2];
};

template <typename T, int VEC, int S, int W, int CTAS, bool TMA, bool WALK>
__global__ void __launch_bounds__(32 * W, CTAS)
    recurrence_fwd_kernel(const FwdParams p, const Chains ch, const __grid_constant__ TileMaps maps) {
    constexpr bool PRECISE = sizeof(T) == 4;
    constexpr int TT = S * W, NP = S * VEC / 2;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    auto &sm = *reinterpret_cast<FwdSmem<T, VEC, S, W, WALK> *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned total = ch.chains.d * (unsigned)ch.tiles;
    const bool cuts = p.resets != nullptr;

    if (TMA) {
        if (tid == 0) {
            mbar_init(&sm.in.full[0], 1);
            sm.in.lost = LostCopies{};
            fence_mbar_init();
        }
        __syncthreads();
    }
    auto place = [&](unsigned v) {
        Tile t = place_tile<VEC>(ch, p, v);
        t.t0 = t.k * TT + warp * S;
        t.live = t.k == 0 || t.k * TT < t.n;  // else behind the row's end
        t.cnt = t.in ? min(max(t.n - t.t0, 0), S) : 0;
        return t;
    };
    Held<T, 3, TMA ? 1 : S> held;
    auto fetch = [&](const Tile &t) {
        if constexpr (TMA) {
            if (tid == 0 && !sm.in.lost.flag) {
                uint64_t *bar = &sm.in.full[0];
                mbar_arrive_expect_tx(bar, 3 * TT * 32 * VEC * sizeof(T));
                const int d0 = t.d, t0 = t.t0;  // of thread 0: the tile's first channel and token
                fetch_box(sm.in.v[0][0], &maps.m[0], bar, d0, t0, t.b, p.row_first & 1);
                fetch_box(sm.in.v[0][1], &maps.m[1], bar, d0, t0, t.b, p.row_first & 2);
                fetch_box(sm.in.v[0][2], &maps.m[2], bar, d0, t0, t.b, p.row_first & 4);
            }
        } else {
            const T *px = static_cast<const T *>(p.x) + t.b * p.sx[0] + t.t0 * p.sx[1] + t.d;
            const T *pr = static_cast<const T *>(p.r) + t.b * p.sr[0] + t.t0 * p.sr[1] + t.d;
            const T *pi = static_cast<const T *>(p.i) + t.b * p.si[0] + t.t0 * p.si[1] + t.d;
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (j < t.cnt) {
                    if constexpr (VEC == 1) {
                        copy_one<T>(&sm.in.v[0][0][warp * S + j][lane], held.v[0][j], pr + j * p.sr[1]);
                        copy_one<T>(&sm.in.v[0][1][warp * S + j][lane], held.v[1][j], pi + j * p.si[1]);
                        copy_one<T>(&sm.in.v[0][2][warp * S + j][lane], held.v[2][j], px + j * p.sx[1]);
                    }
                }
            copy_commit();
        }
    };

    Tickets tickets(WALK ? nullptr : ch.ticket, sm.ticket);
    unsigned v = WALK ? blockIdx.x : tickets.next();
    if (v >= total) return;
    Tile t = place(v);
    fetch(t);
    float csp[VEC], s[VEC];
    if (WALK) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            csp[e] = t.in ? channel_decay(p.c, p.lambda[t.d + e]) : 0.f;
            s[e] = t.in && p.h0 ? p.h0[(int64_t)t.b * p.D + t.d + e] : 0.f;
        }
    }
    for (uint32_t it = 0;; ++it) {
        Tile tn = t;
        bool next;
        if (WALK) {
            ++tn.k;
            tn.t0 += TT;
            tn.cnt = t.in ? min(max(t.n - tn.t0, 0), S) : 0;
            next = tn.k * TT < t.n;
        } else {
            v = tickets.next();  // its barrier also frees sm.wm and sm.gm
            next = v < total;
            if (next) tn = place(v);
        }
        if constexpr (TMA) {
            await_box(sm.in.full, 0, it, &sm.in.lost);
        } else {
            copy_wait<0>();
            put_held(sm.in.v[0], held, warp * S, t.cnt);
        }
        if (t.live) {
            if (!WALK)
#pragma unroll
                for (int e = 0; e < VEC; ++e) csp[e] = t.in ? ch.csp[t.d + e] : 0.f;
            float2 a[NP], b[NP];
            {
                Pack<T, VEC> r[S], gi[S], x[S];
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    r[j] = sm.in.v[0][0][warp * S + j][lane];
                    gi[j] = sm.in.v[0][1][warp * S + j][lane];
                    x[j] = sm.in.v[0][2][warp * S + j][lane];
                }
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    forward_gates<PRECISE>(pair_of<T, VEC, S>(r, q), pair_of<T, VEC, S>(gi, q),
                                           pair_of<T, VEC, S>(x, q), channel_pair<VEC>(csp, q), a[q], b[q]);
            }
            if (t.cnt < S) {  // what the buffer holds behind the end does not count
#pragma unroll
                for (int k = 0; k < S * VEC; ++k)
                    if (k / VEC >= t.cnt) {
                        half_of(a[k / 2], k) = 1.f;
                        half_of(b[k / 2], k) = 0.f;
                    }
            }
            const uint32_t cut = cut_mask(p, t.b, t.t0, min(max(t.n - t.t0, 0), S));
            Maps<VEC> own;
            own.identity();
            with_flag(cut != 0, [&](auto flag) {
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    Pack<float, VEC> P, H;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        P.v[e] = half_of(a[(j * VEC + e) / 2], j * VEC + e);
                        H.v[e] = half_of(b[(j * VEC + e) / 2], j * VEC + e);
                    }
                    if (decltype(flag)::value && (cut >> j & 1)) own.cut();
                    own.then(P, H);
                }
            });
            float h[VEC];
            auto &wm = sm.wm[WALK ? t.k & 1 : 0];
            wm.P[warp][lane] = own.P;
            wm.H[warp][lane] = own.H;
            __syncthreads();
            if (next) fetch(tn);  // every warp has read the buffer
            if constexpr (WALK) {
                walk_state<VEC, W>(wm, s, h, cuts);
                if (!next && warp == 0 && t.in && p.hN)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) p.hN[(int64_t)t.b * p.D + t.d + e] = s[e];
            } else {
                const bool more = (t.k + 1) * TT < t.n;  // a later tile waits for this one
                const bool last = t.j == ch.group - 1;
                if (warp == 0 && more && !last) publish_map<VEC, W>(ch, t, wm, cuts);
                Maps<VEC> m = prefix_maps<VEC, W>(ch, t, wm, sm.gm, cuts);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    s[e] = t.in && p.h0 && t.g == 0 ? p.h0[(int64_t)t.b * p.D + t.d + e] : 0.f;
                group_state<VEC>(ch, t, s);
                if (warp == W - 1 && (last || !more)) {
                    Maps<VEC> end = m;
                    with_flag(cuts, [&](auto flag) { end.template then<decltype(flag)::value>(own.P, own.H); });
                    end.apply(s, h, cuts);
                    if (more)
                        leave_group<VEC>(ch, t, h);
                    else if (t.in && p.hN)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) p.hN[(int64_t)t.b * p.D + t.d + e] = h[e];
                }
                m.apply(s, h, cuts);
            }
            T *ph = static_cast<T *>(p.h) + t.b * p.sh[0] + t.t0 * p.sh[1] + t.d;
            with_flag(cut != 0, [&](auto flag) {
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (j < t.cnt) {
                        Pack<T, VEC> o;
                        if (decltype(flag)::value && (cut >> j & 1))
#pragma unroll
                            for (int e = 0; e < VEC; ++e) h[e] = 0.f;
                        if constexpr (VEC == 1) {
                            h[0] = fmaf(half_of(a[j / 2], j), h[0], half_of(b[j / 2], j));
                            o.v[0] = cvt_out<T>(h[0]);
                        } else {
#pragma unroll
                            for (int e = 0; e < VEC; e += 2) {
                                const int q = (j * VEC + e) / 2;
                                const float2 n = __ffma2_rn(a[q], make_float2(h[e], h[e + 1]), b[q]);
                                o.v[e] = cvt_out<T>(h[e] = n.x);
                                o.v[e + 1] = cvt_out<T>(h[e + 1] = n.y);
                            }
                        }
                        *reinterpret_cast<Pack<T, VEC> *>(ph + j * p.sh[1]) = o;
                    }
            });
        } else if (next) {
            // Behind the row's end there is nothing to compute, but every warp has to have
            // seen this phase of the fetch barrier before the next one is armed: one that
            // finds it two phases on takes the parity for the present one and stands.
            __syncthreads();
            fetch(tn);
        }
        if (!next) break;
        t = tn;
    }
    if (TMA) drain_copies(sm.in.full, 1, &sm.in.lost, kWaitNs);
}

// ---- backward -------------------------------------------------------------------
// The same tiles and chains with time reversed; what runs along a chain is
// C_t = keep_t a_t G_t, the part of the gradient that reaches h_{t-1}.  Across
// the wait a thread keeps dh and sigmoid(r), or exp(-r); the decay is computed
// again (one exponential) rather than held.  8 x 2048 x 4096 FP16 takes 306 us
// (3.5 TB/s; issue 53% at 12.5 warps an SM, and time follows the count of
// instructions), with 1 - sigmoid(r) as a difference, without its reciprocal,
// 10 less; 8 x 1024 x 4096 FP32 194 (5.5).
template <typename T, int VEC, int S, int W, bool WALK>
struct BwdSmem {
    TileIn<T, VEC, S * W, 5, 2> in;
    MapRows<VEC, W> wm[WALK ? 2 : 1];
    MapRows<VEC, WALK ? 1 : (1 << kMaxGroupShift) - 1> gm;
    Pack<float, VEC> sums[W][32];
    unsigned int ticket[2];
};

template <typename T, int VEC, int S, int W, int CTAS, bool TMA, bool WALK>
__global__ void __launch_bounds__(32 * W, CTAS)
    recurrence_bwd_kernel(const BwdParams p, const Chains ch, const __grid_constant__ TileMaps maps) {
    constexpr bool PRECISE = sizeof(T) == 4;
    constexpr int TT = S * W, NP = S * VEC / 2;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    auto &sm = *reinterpret_cast<BwdSmem<T, VEC, S, W, WALK> *>(smem_raw);
    const FwdParams &f = p.f;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned total = ch.chains.d * (unsigned)ch.tiles;
    const bool cuts = f.resets != nullptr;
    const int trow = (W - 1 - warp) * S;  // this warp's first token in the tile: warp 0 holds the last ones

    if (TMA) {
        if (tid == 0) {
            mbar_init(&sm.in.full[0], 1);
            mbar_init(&sm.in.full[1], 1);
            sm.in.lost = LostCopies{};
            fence_mbar_init();
        }
        __syncthreads();
    }
    auto place = [&](unsigned v) {
        Tile t = place_tile<VEC>(ch, f, v);
        const int row_tiles = max((t.n + TT - 1) / TT, 1);
        t.live = t.k < row_tiles;
        t.t0 = (row_tiles - 1 - t.k) * TT + trow;
        t.cnt = t.in && t.live ? min(max(t.n - t.t0, 0), S) : 0;
        return t;
    };
    Held<T, 5, TMA ? 1 : S> held;
    auto fetch = [&](const Tile &t, int buf) {
        if constexpr (TMA) {
            if (tid == 0 && !sm.in.lost.flag) {
                uint64_t *bar = &sm.in.full[buf];
                mbar_arrive_expect_tx(bar, 5 * TT * 32 * VEC * sizeof(T));
                // A dead tile lies before time 0: its copies read zeros.
                const int d0 = t.d, t0 = t.t0 - trow;
                fetch_box(sm.in.v[buf][0], &maps.m[0], bar, d0, t0, t.b, f.row_first & 1);
                fetch_box(sm.in.v[buf][1], &maps.m[1], bar, d0, t0, t.b, f.row_first & 2);
                fetch_box(sm.in.v[buf][2], &maps.m[2], bar, d0, t0, t.b, f.row_first & 4);
                fetch_box(sm.in.v[buf][3], &maps.m[3], bar, d0, t0, t.b, f.row_first & 8);
                fetch_box(sm.in.v[buf][4], &maps.m[4], bar, d0, t0 - 1, t.b, f.row_first & 16);
            }
        } else {
            const T *pr = static_cast<const T *>(f.r) + t.b * f.sr[0] + t.t0 * f.sr[1] + t.d;
            const T *pg = static_cast<const T *>(p.dh) + t.b * p.sdh[0] + t.t0 * p.sdh[1] + t.d;
            const T *px = static_cast<const T *>(f.x) + t.b * f.sx[0] + t.t0 * f.sx[1] + t.d;
            const T *pi = static_cast<const T *>(f.i) + t.b * f.si[0] + t.t0 * f.si[1] + t.d;
            const T *ph = static_cast<const T *>(f.h) + t.b * f.sh[0] + (t.t0 - 1) * f.sh[1] + t.d;
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (j < t.cnt) {
                    const int row = trow + j;
                    if constexpr (VEC == 1) {
                        copy_one<T>(&sm.in.v[buf][0][row][lane], held.v[0][j], pr + j * f.sr[1]);
                        copy_one<T>(&sm.in.v[buf][1][row][lane], held.v[1][j], px + j * f.sx[1]);
                        copy_one<T>(&sm.in.v[buf][2][row][lane], held.v[2][j], pi + j * f.si[1]);
                        copy_one<T>(&sm.in.v[buf][3][row][lane], held.v[3][j], pg + j * p.sdh[1]);
                        if (t.t0 + j > 0) copy_one<T>(&sm.in.v[buf][4][row][lane], held.v[4][j], ph + j * f.sh[1]);
                    }
                }
        }
    };

    Tickets tickets(WALK ? nullptr : ch.ticket, sm.ticket);
    unsigned v = WALK ? blockIdx.x : tickets.next();
    if (v >= total) return;
    Tile t = place(v);
    fetch(t, 0);
    if (!TMA) copy_commit();
    float csp[VEC], s[VEC], sum[VEC] = {};
    if (WALK) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            csp[e] = t.in ? channel_decay(f.c, f.lambda[t.d + e]) : 0.f;
            s[e] = t.in && p.dhN ? p.dhN[(int64_t)t.b * f.D + t.d + e] : 0.f;
        }
    }
    for (uint32_t it = 0;; ++it) {
        const int buf = it & 1;
        Tile tn = t;
        bool next;
        if (WALK) {
            ++tn.k;
            tn.t0 -= TT;
            tn.cnt = t.in ? S : 0;  // only the last tokens' tile can be short
            next = tn.t0 - trow >= 0;
        } else {
            v = tickets.next();  // its barrier also frees sm.wm, sm.gm and sm.sums
            next = v < total;
            if (next) tn = place(v);
        }
        if constexpr (TMA) {
            await_box(sm.in.full, buf, it >> 1, &sm.in.lost);
        } else {
            copy_wait<0>();
            put_held(sm.in.v[buf], held, trow, t.cnt);
        }
        // WALK: one row of sums per chain, else one per tile
        float *part = p.part + (WALK ? (int64_t)t.b : (int64_t)t.b * ch.tiles + t.k) * f.D + t.d;
        if (t.live) {
            // sigmoid(r) and 1 - sigmoid(r), or (FP16 tensors: fewer registers, one more
            // reciprocal later) the exp(-r) that gives both.  The difference of 1 and an
            // approximate sigmoid would lose dr of open gates: 1% at r = 12.
            float2 sg[NP], om[PRECISE ? NP : 1];
            if (!WALK)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    csp[e] = t.in ? ch.csp[t.d + e] : 0.f;
                    sum[e] = 0.f;
                }
            const uint32_t cut = cut_mask(f, t.b, t.t0, min(max(t.n - t.t0, 0), S));
            Pack<T, VEC> dh[S];
            Maps<VEC> own;
            own.identity();
            constexpr int TP = VEC == 1 ? 2 : 1;  // tokens whose pairs are computed together
#pragma unroll
            for (int j0 = S - TP; j0 >= 0; j0 -= TP) {
                float2 a[TP * VEC / 2];
                Pack<T, VEC> r[TP];
#pragma unroll
                for (int u = 0; u < TP; ++u) {
                    r[u] = sm.in.v[buf][0][trow + j0 + u][lane];
                    dh[j0 + u] = sm.in.v[buf][3][trow + j0 + u][lane];
                }
#pragma unroll
                for (int z = 0; z < TP * VEC / 2; ++z) {
                    const int q = j0 * VEC / 2 + z;
                    float2 e, m;
                    decay<PRECISE, true>(pair_of<T, VEC, TP>(r, z), channel_pair<VEC>(csp, z), e, sg[q], a[z], m);
                    if (PRECISE)
                        om[q] = __fmul2_rn(e, sg[q]);
                    else
                        sg[q] = e;
                }
#pragma unroll
                for (int u = TP - 1; u >= 0; --u)
                    if (j0 + u < t.cnt) {  // what the buffer holds behind the end does not count
                        const Pack<T, VEC> &g = dh[j0 + u];
                        if (cut >> (j0 + u) & 1) {
                            own.cut();
                        } else if constexpr (VEC == 1) {
                            const float av = half_of(a[0], u);
                            own.H.v[0] = av * (own.H.v[0] + cvt_f32(g.v[0]));
                            own.P.v[0] *= av;
                        } else {
#pragma unroll
                            for (int e = 0; e < VEC; e += 2) {
                                const float2 av = a[e / 2];
                                const float2 h = __fmul2_rn(
                                    av, __fadd2_rn(make_float2(own.H.v[e], own.H.v[e + 1]),
                                                   make_float2(cvt_f32(g.v[e]), cvt_f32(g.v[e + 1]))));
                                const float2 P = __fmul2_rn(av, make_float2(own.P.v[e], own.P.v[e + 1]));
                                own.H.v[e] = h.x;
                                own.H.v[e + 1] = h.y;
                                own.P.v[e] = P.x;
                                own.P.v[e + 1] = P.y;
                            }
                        }
                    }
            }
            float C[VEC];
            auto &wm = sm.wm[WALK ? t.k & 1 : 0];
            wm.P[warp][lane] = own.P;
            wm.H[warp][lane] = own.H;
            __syncthreads();
            // Every warp is done with the tile before, so the other buffer is free.
            if (next) fetch(tn, buf ^ 1);
            if (!TMA) copy_commit();
            if constexpr (WALK) {
                walk_state<VEC, W>(wm, s, C, cuts);
                if (!next && warp == 0 && t.in && p.dh0)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) p.dh0[(int64_t)t.b * f.D + t.d + e] = s[e];
            } else {
                const bool more = t.t0 - trow > 0;  // an earlier tile waits for this one
                const bool last = t.j == ch.group - 1;
                if (warp == 0 && more && !last) publish_map<VEC, W>(ch, t, wm, cuts);
                Maps<VEC> m = prefix_maps<VEC, W>(ch, t, wm, sm.gm, cuts);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    s[e] = t.in && p.dhN && t.g == 0 ? p.dhN[(int64_t)t.b * f.D + t.d + e] : 0.f;
                group_state<VEC>(ch, t, s);
                if (warp == W - 1 && (last || !more)) {
                    Maps<VEC> end = m;
                    with_flag(cuts, [&](auto flag) { end.template then<decltype(flag)::value>(own.P, own.H); });
                    end.apply(s, C, cuts);
                    if (more)
                        leave_group<VEC>(ch, t, C);
                    else if (t.in && p.dh0)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) p.dh0[(int64_t)t.b * f.D + t.d + e] = C[e];
                }
                m.apply(s, C, cuts);
            }

            T *qx = static_cast<T *>(p.dx) + t.b * p.sdx[0] + t.t0 * p.sdx[1] + t.d;
            T *qr = static_cast<T *>(p.dr) + t.b * p.sdr[0] + t.t0 * p.sdr[1] + t.d;
            T *qi = static_cast<T *>(p.di) + t.b * p.sdi[0] + t.t0 * p.sdi[1] + t.d;
#pragma unroll
            for (int j0 = S - TP; j0 >= 0; j0 -= TP) {
                if (j0 >= t.cnt) continue;
                Pack<T, VEC> x[TP], gi[TP], hp[TP], ox[TP], orr[TP], oi[TP];
                float2 a[TP * VEC / 2], m[TP * VEC / 2], y[TP * VEC / 2], G[TP * VEC / 2];  // G = dh + C
                float2 os[TP * VEC / 2];                                                    // 1 - sigmoid(r)
#pragma unroll
                for (int z = 0; z < TP * VEC / 2; ++z) {
                    const int q = j0 * VEC / 2 + z;
                    const float2 s = PRECISE ? sg[q] : sigmoid_of(sg[q]);
                    os[z] = PRECISE ? om[PRECISE ? q : 0] : __fmul2_rn(sg[q], s);
                    y[z] = __fmul2_rn(channel_pair<VEC>(csp, z), s);
                    decay_of<PRECISE>(y[z], a[z], m[z]);
                }
                if constexpr (VEC == 1) {
#pragma unroll
                    for (int u = TP - 1; u >= 0; --u) {
                        const float g = cvt_f32(dh[j0 + u].v[0]) + C[0];
                        half_of(G[0], u) = g;
                        if (j0 + u < t.cnt) C[0] = cut >> (j0 + u) & 1 ? 0.f : half_of(a[0], u) * g;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        const Pack<T, VEC> &g = dh[j0];
                        G[e / 2] = __fadd2_rn(make_float2(cvt_f32(g.v[e]), cvt_f32(g.v[e + 1])),
                                              make_float2(C[e], C[e + 1]));
                        const float2 n = __fmul2_rn(a[e / 2], G[e / 2]);
                        C[e] = n.x;
                        C[e + 1] = n.y;
                    }
                    if (cut >> j0 & 1)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) C[e] = 0.f;
                }
#pragma unroll
                for (int u = 0; u < TP; ++u) {
                    x[u] = sm.in.v[buf][1][trow + j0 + u][lane];
                    gi[u] = sm.in.v[buf][2][trow + j0 + u][lane];
                    hp[u] = sm.in.v[buf][4][trow + j0 + u][lane];
                    if (t.t0 + j0 + u == 0 || (cut >> (j0 + u) & 1))  // the initial state, or none
#pragma unroll
                        for (int e = 0; e < VEC; ++e) hp[u].v[e] = cvt_out<T>(0.f);
                }
#pragma unroll
                for (int z = 0; z < TP * VEC / 2; ++z) {
                    const float2 xv = pair_of<T, VEC, TP>(x, z), av = a[z];
                    float2 prev = pair_of<T, VEC, TP>(hp, z);
                    if (t.t0 + j0 == 0 && f.h0 && !(cut >> j0 & 1)) {  // h_{-1}, in FP32
                        prev.x = f.h0[(int64_t)t.b * f.D + t.d + (2 * z) % VEC];
                        if (VEC > 1) prev.y = f.h0[(int64_t)t.b * f.D + t.d + (2 * z + 1) % VEC];
                    }
                    const float2 ei = exp_gate<PRECISE>(pair_of<T, VEC, TP>(gi, z), 80.f);
                    const float2 qi1 = __fadd2_rn(ei, both(1.f));
                    const float2 om1 = make_float2(rcp_approx(qi1.x), rcp_approx(qi1.y));  // 1 - sigmoid(i)
                    const float2 si = __fmul2_rn(ei, om1);
                    const float2 m2 = m[z], m1 = __fadd2_rn(m2, both(kTiny));
                    const float2 w = make_float2(rsqrt_approx(m1.x), rsqrt_approx(m1.y));
                    const float2 gs2 = __fmul2_rn(G[z], si);               // G sigmoid(i)
                    const float2 gx = __fmul2_rn(gs2, __fmul2_rn(m2, w));  // * sqrt(m)
                    const float2 gi2 = __fmul2_rn(__fmul2_rn(gx, xv), om1);
                    // E = a (G si x a (y / sqrt(m)) - y G h_{t-1}); y / sqrt(m) first, it tends to 0
                    const float2 u1 = __fmul2_rn(__fmul2_rn(gs2, xv), __fmul2_rn(av, __fmul2_rn(y[z], w)));
                    const float2 u2 = __ffma2_rn(__fmul2_rn(__fmul2_rn(y[z], both(-1.f)), G[z]), prev, u1);
                    const float2 E = __fmul2_rn(av, u2);
                    const float2 gr = __fmul2_rn(E, os[z]);
#pragma unroll
                    for (int hlf = 0; hlf < 2; ++hlf) {
                        const int k = 2 * z + hlf, u = k / VEC, e = k % VEC;
                        ox[u].v[e] = cvt_out<T>(hlf ? gx.y : gx.x);
                        oi[u].v[e] = cvt_out<T>(hlf ? gi2.y : gi2.x);
                        orr[u].v[e] = cvt_out<T>(hlf ? gr.y : gr.x);
                        if (VEC > 1 || j0 + u < t.cnt) sum[e] += hlf ? E.y : E.x;
                    }
                }
#pragma unroll
                for (int u = 0; u < TP; ++u)
                    if (VEC > 1 || j0 + u < t.cnt) {
                        const int j = j0 + u;
                        *reinterpret_cast<Pack<T, VEC> *>(qx + j * p.sdx[1]) = ox[u];
                        *reinterpret_cast<Pack<T, VEC> *>(qi + j * p.sdi[1]) = oi[u];
                        *reinterpret_cast<Pack<T, VEC> *>(qr + j * p.sdr[1]) = orr[u];
                    }
            }
            // the sum of E per channel, warps in order
            if (!WALK || !next) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) sm.sums[warp][lane].v[e] = sum[e];
                __syncthreads();
                if (warp == 0 && t.in)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        float z = 0.f;
#pragma unroll
                        for (int w = 0; w < W; ++w) z += sm.sums[w][lane].v[e];
                        part[e] = z;
                    }
            }
        } else {  // behind the row's end
            if (warp == 0 && t.in)
#pragma unroll
                for (int e = 0; e < VEC; ++e) part[e] = 0.f;
            if (next) fetch(tn, buf ^ 1);
            if (!TMA) copy_commit();
        }
        if (!next) break;
        t = tn;
    }
    if (TMA) drain_copies(sm.in.full, 2, &sm.in.lost, kWaitNs);
}

// dlambda[d] = sigmoid(lambda)/softplus(lambda) * sum of the tiles' sums of E,
// in a fixed order: warp w adds rows w, w + 16, ..., then the warps in order.
// The quotient tends to 1 for very negative lambda.
constexpr int kSumWarps = 16;
__global__ void __launch_bounds__(32 * kSumWarps)
    recurrence_dlambda_kernel(const float *__restrict__ part, const float *__restrict__ lambda,
                              float *__restrict__ dlambda, int64_t rows, int D) {
    __shared__ float sm[kSumWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (d < D)
        for (int64_t k = warp; k < rows; k += kSumWarps) s += part[k * D + d];
    sm[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && d < D) {
#pragma unroll
        for (int w = 1; w < kSumWarps; ++w) s += sm[w][lane];
        const float l = lambda[d];
        dlambda[d] = s * (l < -20.f ? 1.f : 1.f / (1.f + expf(-l)) / channel_softplus(l));
    }
}

// ---- single token -----------------------------------------------------------------
// A thread serves VEC channels of `rows` batch rows, so that its softplus of
// lambda serves them all, and loads two rows before it stores either (a store
// may be to the loaded state, so the compiler keeps their order).  Bound by
// bytes for large batches, by latency for small ones: 4096 x 5120 FP16 takes 58
// us (5.8 TB/s), with one row loaded at a time 68, with four 59; 256 x 5120 12.3,
// 13.3 and 12.3; 4096 x 5120 FP32 82 us each way.
constexpr int kStepAhead = 2;
template <typename T>
struct StepParams {
    const T *x, *r, *i;
    T *h;
    const float *lambda, *s_in;
    float *s_out;
    int64_t xrs, rrs, irs, hrs;
    int B, D, rows;
    float c;
};
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) recurrence_step_kernel(const StepParams<T> p) {
    constexpr bool PRECISE = sizeof(T) == 4;
    const int d = (blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (d >= p.D) return;
    float csp[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) csp[e] = channel_decay(p.c, p.lambda[d + e]);
    const int64_t b0 = (int64_t)blockIdx.y * p.rows, b1 = min(b0 + p.rows, (int64_t)p.B);
    for (int64_t b = b0; b < b1; b += kStepAhead) {
        Pack<T, VEC> x[kStepAhead], r[kStepAhead], gi[kStepAhead];
        Pack<float, VEC> s[kStepAhead];
#pragma unroll
        for (int k = 0; k < kStepAhead; ++k)
            if (b + k < b1) {
                x[k] = load_pack<T, VEC>(p.x + (b + k) * p.xrs + d);
                r[k] = load_pack<T, VEC>(p.r + (b + k) * p.rrs + d);
                gi[k] = load_pack<T, VEC>(p.i + (b + k) * p.irs + d);
                s[k] = load_pack<float, VEC>(p.s_in + (b + k) * p.D + d);
            }
#pragma unroll
        for (int k = 0; k < kStepAhead; ++k) {
            if (b + k >= b1) break;
            Pack<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const int f = VEC == 1 ? 0 : e + 1;
                float2 a, bt;
                forward_gates<PRECISE>(make_float2(cvt_f32(r[k].v[e]), cvt_f32(r[k].v[f])),
                                       make_float2(cvt_f32(gi[k].v[e]), cvt_f32(gi[k].v[f])),
                                       make_float2(cvt_f32(x[k].v[e]), cvt_f32(x[k].v[f])),
                                       make_float2(csp[e], csp[f]), a, bt);
                s[k].v[e] = fmaf(a.x, s[k].v[e], bt.x);
                if (VEC > 1) s[k].v[f] = fmaf(a.y, s[k].v[f], bt.y);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) o.v[e] = cvt_out<T>(s[k].v[e]);
            *reinterpret_cast<Pack<float, VEC> *>(p.s_out + (b + k) * p.D + d) = s[k];
            *reinterpret_cast<Pack<T, VEC> *>(p.h + (b + k) * p.hrs + d) = o;
        }
    }
}

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Every row starts at a multiple of VEC elements' bytes.
template <typename T, int VEC>
bool vector_rows(const void *p, const int64_t *s) {
    return aligned_to(p, sizeof(T) * VEC) && s[0] % VEC == 0 && s[1] % VEC == 0;
}

// Rows of an output must not overlap one another.
bool output_rows_disjoint(const int64_t *s, int B, int L, int D) {
    if (L > 1 && s[1] < D) return false;
    if (B > 1 && s[0] < D) return false;
    if (B > 1 && L > 1 && s[0] < (L - 1) * s[1] + D && s[1] < (B - 1) * s[0] + D) return false;
    return true;
}

int check_args(const MambaRecurrenceArgs *a, bool backward) {
    MB_CHECK_ARG(a, "gated_recurrence: null args");
    MB_CHECK_ARG(a->batch >= 0 && a->seqlen >= 0 && a->dim >= 0, "gated_recurrence: negative size");
    MB_CHECK_ARG(a->dtype == MAMBA_F32 || a->dtype == MAMBA_F16, "gated_recurrence: bad dtype");
    MB_CHECK_ARG(a->c > 0.f && a->c <= 3.0e38f, "gated_recurrence: c must be positive and finite");
    if (a->batch == 0 || a->dim == 0) return 0;
    MB_CHECK_ARG(a->lambda && (a->seqlen == 0 || (a->x && a->r && a->i && a->h)), "gated_recurrence: null pointer");
    const size_t es = dtype_size(a->dtype);
    MB_CHECK_ARG(aligned_to(a->x, es) && aligned_to(a->r, es) && aligned_to(a->i, es) && aligned_to(a->h, es) &&
                     aligned_to(a->lambda, 4) && aligned_to(a->initial_state, 4) && aligned_to(a->final_state, 4) &&
                     aligned_to(a->lengths, 4),
                 "gated_recurrence: pointers must be aligned to their element type");
    MB_CHECK_ARG(backward || a->seqlen == 0 || (a->h != a->x && a->h != a->r && a->h != a->i),
                 "gated_recurrence: h may not be one of the inputs");
    MB_CHECK_ARG(backward || !a->final_state || a->final_state != a->initial_state,
                 "gated_recurrence: final_state may not be initial_state");
    MB_CHECK_ARG(backward || output_rows_disjoint(a->h_stride, a->batch, a->seqlen, a->dim),
                 "gated_recurrence: rows of h overlap (strides)");
    return 0;
}

FwdParams fwd_params(const MambaRecurrenceArgs *a) {
    FwdParams p{};
    p.x = a->x;
    p.r = a->r;
    p.i = a->i;
    p.lambda = a->lambda;
    p.h0 = a->initial_state;
    p.lengths = a->lengths;
    p.resets = a->resets;
    p.h = a->h;
    p.hN = a->final_state;
    p.B = a->batch;
    p.L = a->seqlen;
    p.D = a->dim;
    p.c = a->c;
    for (int k = 0; k < 2; ++k) {
        p.sx[k] = a->x_stride[k];
        p.sr[k] = a->r_stride[k];
        p.si[k] = a->i_stride[k];
        p.sh[k] = a->h_stride[k];
    }
    return p;
}

// Tile shapes: channels a thread holds, tokens a warp holds, warps, CTAs per SM.
// The ...One shapes, without tensor maps, serve any alignment and strides.
template <int VEC_, int S_, int W_, int CTAS_, bool TMA_ = true>
struct Shape {
    static constexpr int VEC = VEC_, S = S_, W = W_, CTAS = CTAS_, tile = S_ * W_;
    static constexpr bool TMA = TMA_;
};
// FP16 walking, 8 x 4096 x 4096: 257 us; 8 warps a CTA 314; one channel a thread
// 286 to 293.  Backward 8 x 2048 x 4096: 308, 8 warps 306 to 308.
template <typename T> struct Shapes;
template <> struct Shapes<__half> {
    using Fwd = Shape<2, 16, 4, 4>;
    using FwdOne = Shape<1, 16, 4, 4, false>;
    using FwdWalk = Shape<2, 16, 4, 4>;
    using Bwd = Shape<2, 8, 4, 4>;
    using BwdOne = Shape<1, 8, 4, 3, false>;
    using BwdWalk = Shape<2, 8, 4, 4>;
};
template <> struct Shapes<float> {
    using Fwd = Shape<1, 16, 8, 3>;
    using FwdOne = Shape<1, 8, 4, 6, false>;
    using FwdWalk = Shape<2, 8, 4, 5>;
    using Bwd = Shape<1, 8, 4, 4>;
    using BwdOne = Shape<1, 8, 4, 4, false>;
    using BwdWalk = Shape<1, 8, 4, 4>;
};

// Token positions are 32-bit numbers, up to two tiles behind the sequence's end.
constexpr int kMaxSeqlen = 0x7fffffff - 256;

// The chains of a call and where its workspace holds what.
struct Plan {
    Chains ch;
    size_t bytes, csp_bytes, part_bytes, ones_bytes;
};
template <typename Sh>
bool plan_chains(const MambaRecurrenceArgs *a, bool backward, Plan &pl) {
    const int cw = 32 * Sh::VEC;
    Chains &c = pl.ch;
    c = Chains{};
    const int64_t blocks = ceil_div64(a->dim, cw), tiles = std::max<int64_t>(1, ceil_div64(a->seqlen, Sh::tile));
    if (blocks * a->batch > 0x7fffffffLL || blocks * a->batch * tiles > 0x7fffffffLL) return false;
    if (a->seqlen > kMaxSeqlen) return false;
    auto divisor = [](int64_t d) {
        return Divisor{(unsigned)d, d == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / (unsigned long long)d)};
    };
    c.blocks = divisor(blocks);
    c.chains = divisor(blocks * a->batch);
    c.tiles = (int)tiles;
    // A chain's latency is its groups' hand-overs plus a group's length of maps to
    // compose.  Groups of 4 everywhere: 1 x 524288 x 64 FP16 931 us instead of 303;
    // of 16 everywhere: 1 x 131072 x 2048 FP32 820 instead of 807, 1 x 16384 x 4096
    // FP16 175 instead of 173.
    c.group_shift = std::min(kMaxGroupShift, tiles <= 128 ? 2 : tiles <= 1024 ? 3 : 4);
    c.group = 1 << c.group_shift;
    c.groups = ceil_div((int)tiles, c.group);
    // csp, the backward's partial sums, then what starts as all ones bits:
    // the ticket, the maps and the states (a multiple of 16 bytes: cw is 32 at least)
    auto up = [](size_t v) { return (v + 15) / 16 * 16; };
    pl.csp_bytes = up((size_t)a->dim * sizeof(float));
    pl.part_bytes = backward ? up((size_t)a->batch * tiles * a->dim * sizeof(float)) : 0;
    pl.ones_bytes = 256;
    if (tiles > 1) pl.ones_bytes += (size_t)c.chains.d * cw * (tiles * sizeof(float2) + c.groups * sizeof(float));
    pl.bytes = pl.csp_bytes + pl.part_bytes + pl.ones_bytes;
    return true;
}
template <typename T>
size_t workspace_bytes(const MambaRecurrenceArgs *a, bool backward) {
    using S = Shapes<T>;
    Plan p, q;
    if (!(backward ? plan_chains<typename S::Bwd>(a, true, p) : plan_chains<typename S::Fwd>(a, false, p))) return 0;
    if (!(backward ? plan_chains<typename S::BwdOne>(a, true, q) : plan_chains<typename S::FwdOne>(a, false, q)))
        return 0;
    return std::max(p.bytes, q.bytes);
}

}  // namespace

// What either channel width needs, so that the size does not depend on pointers.
size_t recurrence_workspace_bytes(const MambaRecurrenceArgs *a, bool backward) {
    if (!a || a->batch <= 0 || a->seqlen < 0 || a->dim <= 0) return 0;
    return a->dtype == MAMBA_F16 ? workspace_bytes<__half>(a, backward) : workspace_bytes<float>(a, backward);
}

namespace {

// Opts a kernel into its shared memory, once per device.
template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes) {
    static std::mutex mu;
    static std::vector<std::pair<const void *, int>> done;
    int dev = 0;
    MB_CUDA_TRY(cudaGetDevice(&dev));
    const std::pair<const void *, int> key(reinterpret_cast<const void *>(kernel), dev);
    std::lock_guard<std::mutex> lk(mu);
    if (std::find(done.begin(), done.end(), key) != done.end()) return 0;
    MB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.push_back(key);
    return 0;
}

// Prepares the workspace: c * softplus(lambda) per channel, and all ones bits
// from the ticket on.
__global__ void __launch_bounds__(256)
    recurrence_init_kernel(const float *__restrict__ lambda, float c, int D, float *__restrict__ csp,
                           uint4 *__restrict__ ones, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = (int64_t)gridDim.x * 256;
    for (int64_t d = i; d < D; d += stride) csp[d] = channel_decay(c, lambda[d]);
    for (int64_t k = i; k < n; k += stride) ones[k] = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
}

// Launches one variant.  Tickets: the workspace's preparation, then as many
// persistent CTAs as fit; walking: one CTA per chain, no preparation.
template <typename Sh, bool WALK, typename Kernel, typename Params>
int launch_tiles(Kernel kernel, const Params &p, const FwdParams &f, Plan &pl, const TileMaps &maps, size_t smem,
                 void *ws, cudaStream_t st, const char *what) {
    Chains &c = pl.ch;
    if (allow_smem(kernel, smem)) return -1;
    const int64_t sms = device_sm_count();
    int64_t grid = c.chains.d;
    if (!WALK) {
        uint8_t *base = static_cast<uint8_t *>(ws);
        float *csp = reinterpret_cast<float *>(base);
        base += pl.csp_bytes + pl.part_bytes;
        c.csp = csp;
        c.ticket = reinterpret_cast<unsigned int *>(base);
        c.maps = reinterpret_cast<float2 *>(base + 256);
        c.states = reinterpret_cast<float *>(c.maps + (int64_t)c.chains.d * c.tiles * 32 * Sh::VEC);
        const int64_t ones = (int64_t)pl.ones_bytes / 16;
        const int64_t init = std::min<int64_t>(8 * sms, std::max<int64_t>(ceil_div64(ones, 1024), ceil_div64(f.D, 256)));
        recurrence_init_kernel<<<(unsigned)init, 256, 0, st>>>(f.lambda, f.c, f.D, csp, reinterpret_cast<uint4 *>(base),
                                                               ones);
        if (launch_status(what)) return -1;
        grid = std::min(grid * c.tiles, Sh::CTAS * sms);
    }
    kernel<<<(unsigned)grid, 32 * Sh::W, smem, st>>>(p, c, maps);
    return launch_status(what);
}

// Whether CTAs should walk whole chains: where the chains fill the resident
// CTAs of `Sh` in nearly whole rounds, walking spares the hand-over of states
// between CTAs; with fewer chains it would leave SMs empty.  FP16, by ticket and
// walking: 8 x 4096 x 4096 265 and 257 us, 64 x 512 x 4096 277 and 220, 4 x 4096
// x 2048 87 and 148, 1 x 16384 x 4096 173 and 520; backward 8 x 2048 x 4096 340
// and 308, 4 x 2048 x 2048 107 and 171.  0.6 lies where the two meet: at 0.54
// (16 x 2048 x 2560) forward 171 and 184, backward (16 x 1024 x 2560) 220 and 222.
template <typename Sh>
bool walks(const Plan &pl) {
    const int64_t slots = (int64_t)Sh::CTAS * device_sm_count(), chains = pl.ch.chains.d;
    return chains * 10 >= ceil_div64(chains, slots) * slots * 6 || pl.ch.tiles == 1;
}

// Tensor map of [batch, seqlen, dim] with boxes of `tokens` x `chans`; false
// where the hardware cannot describe it (the caller then takes the kernels
// without tensor maps).  The outer dimension with the larger stride comes last.
// Aligned tensors with tensor copies and with each thread's own: 8 x 4096 x 4096
// FP16 257 and 560 us, backward 8 x 2048 x 4096 308 and 430, 8 x 2048 x 4096
// FP32 189 and 310, backward 8 x 1024 x 4096 196 and 286.
template <typename T>
bool encode_tile(CUtensorMap *m, const void *ptr, const int64_t *s, int B, int L, int D, int chans, int tokens,
                 unsigned bit, unsigned &row_first) {
    constexpr int64_t es = sizeof(T);
    if (!ptr || !aligned_to(ptr, 16)) return false;
    // a dimension of one element has no stride of its own
    const int64_t row = ((int64_t)D * es + 15) / 16 * 16;
    int64_t st = L > 1 ? s[1] * es : row, sb = B > 1 ? s[0] * es : st * std::max(L, 1);
    const bool swap = B > 1 && L > 1 && sb < st;
    if (B > 1 && L == 1) st = row;
    const int64_t s1 = swap ? sb : st, s2 = swap ? st : std::max(sb, s1);
    if (s1 < D * es || s1 % 16 || s2 % 16 || s1 >= (1ll << 40) || s2 >= (1ll << 40)) return false;
    if (B > 1 && !swap && sb != s2) return false;
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)(swap ? B : L), (cuuint64_t)(swap ? L : B)};
    const cuuint64_t strides[2] = {(cuuint64_t)s1, (cuuint64_t)s2};
    const cuuint32_t box[3] = {(cuuint32_t)chans, (cuuint32_t)(swap ? 1 : tokens), (cuuint32_t)(swap ? tokens : 1)};
    const cuuint32_t one[3] = {1, 1, 1};
    if (swap) row_first |= bit;
    return enc(m, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3,
               const_cast<void *>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename Sh, bool WALK>
int launch_forward(const FwdParams &p, Plan &pl, const TileMaps &maps, void *ws, cudaStream_t st) {
    return launch_tiles<Sh, WALK>(recurrence_fwd_kernel<T, Sh::VEC, Sh::S, Sh::W, Sh::CTAS, Sh::TMA, WALK>, p, p, pl, maps,
                                  sizeof(FwdSmem<T, Sh::VEC, Sh::S, Sh::W, WALK>), ws, st, "gated_recurrence kernel");
}
// The forward's tensors (x, r, i first: the order of the kernel's buffers).
template <typename T, typename Sh>
bool forward_maps(FwdParams &p, TileMaps &maps) {
    p.row_first = 0;
    if (p.D % Sh::VEC || p.L == 0) return false;
    auto enc = [&](int k, const void *ptr, const int64_t *s) {
        return encode_tile<T>(&maps.m[k], ptr, s, p.B, p.L, p.D, 32 * Sh::VEC, Sh::tile, 1u << k, p.row_first);
    };
    return enc(0, p.r, p.sr) && enc(1, p.i, p.si) && enc(2, p.x, p.sx) && vector_rows<T, Sh::VEC>(p.h, p.sh);
}
template <typename T>
int choose_forward(const MambaRecurrenceArgs *a, void *ws, cudaStream_t st) {
    using S = Shapes<T>;
    FwdParams p = fwd_params(a);
    TileMaps maps;
    Plan pl;
    const char *many = "gated_recurrence: too many tiles or tokens";
    MB_CHECK_ARG(plan_chains<typename S::FwdWalk>(a, false, pl), many);
    if (walks<typename S::FwdWalk>(pl) && forward_maps<T, typename S::FwdWalk>(p, maps))
        return launch_forward<T, typename S::FwdWalk, true>(p, pl, maps, ws, st);
    if (forward_maps<T, typename S::Fwd>(p, maps)) {
        MB_CHECK_ARG(plan_chains<typename S::Fwd>(a, false, pl), many);
        return launch_forward<T, typename S::Fwd, false>(p, pl, maps, ws, st);
    }
    MB_CHECK_ARG(plan_chains<typename S::FwdOne>(a, false, pl), many);
    return walks<typename S::FwdOne>(pl) ? launch_forward<T, typename S::FwdOne, true>(p, pl, maps, ws, st)
                                         : launch_forward<T, typename S::FwdOne, false>(p, pl, maps, ws, st);
}

template <typename T, typename Sh, bool WALK>
int launch_backward(BwdParams &p, Plan &pl, const TileMaps &maps, void *ws, cudaStream_t st) {
    p.part = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + pl.csp_bytes);
    return launch_tiles<Sh, WALK>(recurrence_bwd_kernel<T, Sh::VEC, Sh::S, Sh::W, Sh::CTAS, Sh::TMA, WALK>, p, p.f, pl, maps,
                                  sizeof(BwdSmem<T, Sh::VEC, Sh::S, Sh::W, WALK>), ws, st,
                                  "gated_recurrence_backward kernel");
}
// The backward's tensors (r, x, i, dh, h: the order of the kernel's buffers).
template <typename T, typename Sh>
bool backward_maps(BwdParams &p, TileMaps &maps) {
    FwdParams &f = p.f;
    f.row_first = 0;
    if (f.D % Sh::VEC || f.L == 0) return false;
    auto enc = [&](int k, const void *ptr, const int64_t *s) {
        return encode_tile<T>(&maps.m[k], ptr, s, f.B, f.L, f.D, 32 * Sh::VEC, Sh::tile, 1u << k, f.row_first);
    };
    return enc(0, f.r, f.sr) && enc(1, f.x, f.sx) && enc(2, f.i, f.si) && enc(3, p.dh, p.sdh) && enc(4, f.h, f.sh) &&
           vector_rows<T, Sh::VEC>(p.dx, p.sdx) && vector_rows<T, Sh::VEC>(p.dr, p.sdr) &&
           vector_rows<T, Sh::VEC>(p.di, p.sdi);
}
template <typename T>
int choose_backward(const MambaRecurrenceArgs *a, BwdParams &p, const MambaRecurrenceGrads *g, void *ws,
                    cudaStream_t st) {
    using S = Shapes<T>;
    TileMaps maps;
    Plan pl;
    const char *many = "gated_recurrence_backward: too many tiles or tokens";
    int64_t rows = a->batch;
    MB_CHECK_ARG(plan_chains<typename S::BwdWalk>(a, true, pl), many);
    if (walks<typename S::BwdWalk>(pl) && backward_maps<T, typename S::BwdWalk>(p, maps)) {
        if (launch_backward<T, typename S::BwdWalk, true>(p, pl, maps, ws, st)) return -1;
    } else if (backward_maps<T, typename S::Bwd>(p, maps)) {
        MB_CHECK_ARG(plan_chains<typename S::Bwd>(a, true, pl), many);
        if (launch_backward<T, typename S::Bwd, false>(p, pl, maps, ws, st)) return -1;
        rows *= pl.ch.tiles;
    } else {
        MB_CHECK_ARG(plan_chains<typename S::BwdOne>(a, true, pl), many);
        const bool walk = walks<typename S::BwdOne>(pl);
        if (walk ? launch_backward<T, typename S::BwdOne, true>(p, pl, maps, ws, st)
                 : launch_backward<T, typename S::BwdOne, false>(p, pl, maps, ws, st))
            return -1;
        if (!walk) rows *= pl.ch.tiles;
    }
    recurrence_dlambda_kernel<<<(unsigned)ceil_div(a->dim, 32), 32 * kSumWarps, 0, st>>>(p.part, a->lambda,
                                                                                         g->dlambda, rows, a->dim);
    return launch_status("gated_recurrence_backward sum kernel");
}

}  // namespace

int recurrence_forward(const MambaRecurrenceArgs *a, void *ws, size_t ws_bytes, cudaStream_t st) {
    if (check_args(a, false)) return -1;
    if (a->batch == 0 || a->dim == 0) return 0;
    const size_t need = recurrence_workspace_bytes(a, false);
    MB_CHECK_ARG(need, "gated_recurrence: too many tiles or tokens");
    MB_CHECK_ARG(ws && ws_bytes >= need && aligned_to(ws, 16),
                 "gated_recurrence: workspace too small or not 16-byte aligned");
    return a->dtype == MAMBA_F16 ? choose_forward<__half>(a, ws, st) : choose_forward<float>(a, ws, st);
}

int recurrence_backward(const MambaRecurrenceArgs *a, const MambaRecurrenceGrads *g, void *ws, size_t ws_bytes,
                        cudaStream_t st) {
    if (check_args(a, true)) return -1;
    MB_CHECK_ARG(g, "gated_recurrence_backward: null gradients");
    if (a->dim == 0) return 0;
    MB_CHECK_ARG(g->dlambda && aligned_to(g->dlambda, 4), "gated_recurrence_backward: dlambda");
    if (a->batch == 0) {
        MB_CUDA_TRY(cudaMemsetAsync(g->dlambda, 0, (size_t)a->dim * 4, st));
        return 0;
    }
    MB_CHECK_ARG(a->seqlen == 0 || (g->dh && g->dx && g->dr && g->di), "gated_recurrence_backward: null pointer");
    const size_t es = dtype_size(a->dtype);
    MB_CHECK_ARG(aligned_to(g->dh, es) && aligned_to(g->dx, es) && aligned_to(g->dr, es) && aligned_to(g->di, es) &&
                     aligned_to(g->dfinal_state, 4) && aligned_to(g->dinitial_state, 4),
                 "gated_recurrence_backward: pointers must be aligned to their element type");
    if (a->seqlen > 0) {
        const void *in[5] = {a->x, a->r, a->i, a->h, g->dh};
        for (const void *p : in)
            MB_CHECK_ARG(p != g->dx && p != g->dr && p != g->di,
                         "gated_recurrence_backward: a gradient may not be one of the inputs");
        MB_CHECK_ARG(g->dx != g->dr && g->dx != g->di && g->dr != g->di,
                     "gated_recurrence_backward: the gradients need memory of their own");
    }
    MB_CHECK_ARG(!g->dinitial_state || (g->dinitial_state != g->dfinal_state && g->dinitial_state != a->initial_state),
                 "gated_recurrence_backward: dinitial_state may not be dfinal_state or initial_state");
    MB_CHECK_ARG(output_rows_disjoint(g->dx_stride, a->batch, a->seqlen, a->dim) &&
                     output_rows_disjoint(g->dr_stride, a->batch, a->seqlen, a->dim) &&
                     output_rows_disjoint(g->di_stride, a->batch, a->seqlen, a->dim),
                 "gated_recurrence_backward: rows of a gradient overlap (strides)");
    const size_t need = recurrence_workspace_bytes(a, true);
    MB_CHECK_ARG(need, "gated_recurrence_backward: too many tiles or tokens");
    MB_CHECK_ARG(ws && ws_bytes >= need && aligned_to(ws, 16),
                 "gated_recurrence_backward: workspace too small or not 16-byte aligned");
    BwdParams p{};
    p.f = fwd_params(a);
    p.dh = g->dh;
    p.dhN = g->dfinal_state;
    p.dx = g->dx;
    p.dr = g->dr;
    p.di = g->di;
    p.dh0 = g->dinitial_state;
    for (int k = 0; k < 2; ++k) {
        p.sdh[k] = g->dh_stride[k];
        p.sdx[k] = g->dx_stride[k];
        p.sdr[k] = g->dr_stride[k];
        p.sdi[k] = g->di_stride[k];
    }
    return a->dtype == MAMBA_F16 ? choose_backward<__half>(a, p, g, ws, st) : choose_backward<float>(a, p, g, ws, st);
}

namespace {

// Waits that nothing ends, through the kernels' own helpers: for a published
// state and for a box.  The words outlive the call and stay as they are.
__device__ uint32_t g_wait_selftest[2] = {kEmpty, kEmpty};
__global__ void recurrence_wait_selftest_kernel(uint64_t limit_ns) {
    __shared__ uint64_t full[1];
    __shared__ LostCopies lost;
    if (threadIdx.x != 0) return;
    float h[1];
    wait_states<1>(reinterpret_cast<const float *>(&g_wait_selftest[1]), &g_wait_selftest[0], h, limit_ns);
    const bool reported = *(volatile uint32_t *)&g_wait_selftest[0] != kEmpty;
    *(volatile uint32_t *)&g_wait_selftest[0] = kEmpty;
    lost = LostCopies{};
    mbar_init(&full[0], 1);
    fence_mbar_init();
    if (reported) await_box(full, 0, 0, &lost, limit_ns);
    drain_copies(full, 1, &lost, limit_ns);
}

}  // namespace

int recurrence_wait_selftest(uint64_t limit_ns, cudaStream_t st) {
    recurrence_wait_selftest_kernel<<<1, 32, 0, st>>>(limit_ns);
    return launch_status("gated_recurrence wait self-test kernel");
}

unsigned recurrence_error_flags(bool clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_recurrence_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (clear && v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_recurrence_error, &z, sizeof(z));
    }
    return v;
}

int recurrence_step(const void *x, int64_t xrs, const void *r, int64_t rrs, const void *i, int64_t irs,
                    const float *lambda, const float *state_in, float *state_out, void *h, int64_t hrs, int batch,
                    int dim, float c, int dtype, cudaStream_t st) {
    MB_CHECK_ARG(batch >= 0 && dim >= 0, "gated_recurrence_step: negative size");
    MB_CHECK_ARG(dtype == MAMBA_F32 || dtype == MAMBA_F16, "gated_recurrence_step: bad dtype");
    MB_CHECK_ARG(c > 0.f && c <= 3.0e38f, "gated_recurrence_step: c must be positive and finite");
    if (batch == 0 || dim == 0) return 0;
    MB_CHECK_ARG(x && r && i && lambda && state_in && state_out && h, "gated_recurrence_step: null pointer");
    const size_t es = dtype_size(dtype);
    MB_CHECK_ARG(aligned_to(x, es) && aligned_to(r, es) && aligned_to(i, es) && aligned_to(h, es) &&
                     aligned_to(lambda, 4) && aligned_to(state_in, 4) && aligned_to(state_out, 4),
                 "gated_recurrence_step: pointers must be aligned to their element type");
    MB_CHECK_ARG(batch == 1 || hrs >= dim, "gated_recurrence_step: rows of h overlap (stride)");
    MB_CHECK_ARG(h != x && h != r && h != i, "gated_recurrence_step: h may not be one of the inputs");
    auto run = [&](auto zero) {
        using T = decltype(zero);
        StepParams<T> p{static_cast<const T *>(x), static_cast<const T *>(r), static_cast<const T *>(i),
                        static_cast<T *>(h), lambda, state_in, state_out, xrs, rrs, irs, hrs, batch, dim, 1, c};
        const bool vec = dim % 4 == 0 && xrs % 4 == 0 && rrs % 4 == 0 && irs % 4 == 0 && hrs % 4 == 0 &&
                         aligned_to(x, 4 * es) && aligned_to(r, 4 * es) && aligned_to(i, 4 * es) &&
                         aligned_to(h, 4 * es) && aligned_to(state_in, 16) && aligned_to(state_out, 16);
        const int blocks = ceil_div(dim, kThreads * (vec ? 4 : 1));
        // several rows per thread once one row each would fill the GPU four times over:
        // 4096 x 5120 FP16 58 us, with one row each 80; 1024 x 5120 22 and 27; FP32 82 and 95
        p.rows = (int64_t)blocks * batch >= 16LL * device_sm_count() ? 4 : 1;
        p.rows = std::max(p.rows, ceil_div(batch, 65535));  // the grid's limit
        const dim3 grid((unsigned)blocks, (unsigned)ceil_div(batch, p.rows));
        if (vec)
            recurrence_step_kernel<T, 4><<<grid, kThreads, 0, st>>>(p);
        else
            recurrence_step_kernel<T, 1><<<grid, kThreads, 0, st>>>(p);
    };
    if (dtype == MAMBA_F16)
        run(__half());
    else
        run(0.f);
    return launch_status("gated_recurrence_step kernel");
}

}  // namespace mb
