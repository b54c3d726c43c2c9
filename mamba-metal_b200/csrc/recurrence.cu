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

namespace mb {

__device__ unsigned int g_recurrence_error = 0;

namespace {

// Gates of one element.  FP16 tensors: single-instruction exponentials and
// reciprocals (relative error ~2^-22, far below FP16's 2^-11 rounding).
// FP32 tensors: the CUDA math library's FP32 functions.
template <bool PRECISE>
__device__ __forceinline__ float exp_neg(float v) {  // exp(-v)
    return PRECISE ? expf(-v) : ex2_approx(-v * kLog2e);
}

// sigmoid(v) and 1 - sigmoid(v), each without cancellation.
template <bool PRECISE>
__device__ __forceinline__ void sigmoid2(float v, float &s, float &om) {
    const float e = exp_neg<PRECISE>(fabsf(v));
    const float t = PRECISE ? __fdiv_rn(1.f, 1.f + e) : rcp_approx(1.f + e);
    const float u = e * t;
    s = v >= 0.f ? t : u;
    om = v >= 0.f ? u : t;
}

// 1 - a^2 = -expm1(-2y) for a = exp(-y).  FP16 tensors: below y = 0.03 the
// series 2y - 2y^2 + 4/3 y^3 (relative error < y^3/3 = 9e-6), above it
// fma(-a, a, 1), whose absolute error of ~4e-7 is then below 7e-6 of it.
template <bool PRECISE>
__device__ __forceinline__ float one_minus_a2(float y, float a) {
    if (PRECISE) return -expm1f(-2.f * y);
    const float series = 2.f * y * fmaf(y, fmaf(y, 2.f / 3.f, -1.f), 1.f);
    return y < 0.03f ? series : fmaf(-a, a, 1.f);
}

template <bool PRECISE>
__device__ __forceinline__ float sqrt_gate(float m) {
    if (PRECISE) return sqrtf(m);
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(m));
    return r;
}

// softplus(lambda): per channel, so the accurate form for both types.
__device__ __forceinline__ float softplus_channel(float l) { return fmaxf(l, 0.f) + log1pf(expf(-fabsf(l))); }

// beta = sqrt(m) and q = y / beta; q -> sqrt(y / 2) -> 0 as the gate closes.
template <bool PRECISE>
__device__ __forceinline__ void root_gate(float m, float y, float &beta, float &q) {
    if (PRECISE) {
        beta = sqrtf(m);
        q = beta <= 1e-18f ? 0.f : __fdiv_rn(y, beta);
    } else {
        const float r = rsqrtf(m);
        beta = m <= 1e-36f ? 0.f : m * r;  // a NaN stays one
        q = m <= 1e-36f ? 0.f : y * r;
    }
}

struct Decay {
    float s, om, y, a;
};
template <bool PRECISE>
__device__ __forceinline__ Decay decay(float r, float csp) {
    Decay d;
    sigmoid2<PRECISE>(r, d.s, d.om);
    d.y = csp * d.s;
    d.a = exp_neg<PRECISE>(d.y);
    return d;
}

struct FwdParams {
    const void *x, *r, *i;
    const float *lambda, *h0;
    const int32_t *lengths;
    const uint8_t *resets;
    void *h;
    float *hN;
    int B, L, D;
    float c;
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
// groups of kGroup: a tile publishes its map to the later tiles of its group,
// and the group's last tile publishes the state leaving the group.  So the
// serial chain over a long sequence has one hop per group, each tile composes
// the same maps in the same order on every run (a scheme that takes whatever
// state is ready first would not), and results repeat bit for bit.
// A published value is one machine word that says itself whether it is there:
// the workspace starts as all ones bits (a NaN that no published value has).
constexpr int kGroup = 8;
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

// Bounded wait (2 s, or at once after another CTA's wait ran out).
struct Waiting {
    uint64_t t0 = 0;
    int spins = 0;
    __device__ __forceinline__ bool again() {
        if ((++spins & 63) == 0) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > 2000000000ull || *(volatile unsigned int *)&g_recurrence_error) {
                atomicOr(&g_recurrence_error, kErrRecurrenceTimeout);
                return false;
            }
        }
        return true;
    }
};

template <int VEC>
__device__ __forceinline__ void wait_maps(const float2 *slot, float2 (&m)[VEC]) {
    Waiting wt;
    bool ready;
    do {
        uint64_t w[VEC];
        ready = true;
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[k] = get_map(slot + k);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            ready &= (uint32_t)w[k] != kEmpty;
            m[k] = make_float2(__uint_as_float((uint32_t)w[k]), __uint_as_float((uint32_t)(w[k] >> 32)));
        }
    } while (!ready && wt.again());
}
template <int VEC>
__device__ __forceinline__ void wait_states(const float *slot, float (&h)[VEC]) {
    Waiting wt;
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

struct Chains {
    unsigned int *ticket;
    float2 *maps;    // [chains, tiles, channels of a tile]
    float *states;   // [chains, groups, channels of a tile]
    int blocks;      // channel blocks of a row
    int chains;      // rows * blocks
    int tiles;
};

// Hands out tickets one ahead: next() gives the ticket drawn by the call
// before it (or at the start) and draws another, whose latency then hides
// behind a tile's work.  Each call syncs the CTA.
struct Tickets {
    unsigned int *counter, *shared;  // shared: two places, used in turn
    unsigned int ahead = 0, turn = 0;
    __device__ __forceinline__ Tickets(unsigned int *c, unsigned int *s) : counter(c), shared(s) {
        if (threadIdx.x == 0) ahead = atomicAdd(counter, 1u) + 1u;  // the counter starts as all ones bits
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

// The map from the state at the start of tile k's group to the state entering
// this warp's tokens (m), for the last warp also to the state leaving the
// tile (end).  Warps wait for the maps of the group's earlier tiles between
// them; `wm` holds the maps of this tile's warps.  Syncs the CTA.
template <int VEC, int W>
__device__ __forceinline__ void prefix_maps(const Chains &c, int chain, int k, const float2 (*wm)[VEC * 32],
                                            float2 (*gm)[VEC * 32], float2 (&m)[VEC], float2 (&end)[VEC]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cw = VEC * 32;
    const int g = k / kGroup, j = k % kGroup;
#pragma unroll
    for (int q = 0; q < (kGroup - 1 + W - 1) / W; ++q) {
        const int tile = warp + q * W;
        if (tile < j) {
            float2 t[VEC];
            wait_maps<VEC>(c.maps + ((int64_t)chain * c.tiles + g * kGroup + tile) * cw + lane * VEC, t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) gm[tile][e * 32 + lane] = t[e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) m[e] = make_float2(1.f, 0.f);
    auto then = [&](float2 &f, const float2 &q) {
        f.y = fmaf(q.x, f.y, q.y);
        f.x *= q.x;
    };
    for (int t = 0; t < j; ++t)
#pragma unroll
        for (int e = 0; e < VEC; ++e) then(m[e], gm[t][e * 32 + lane]);
    for (int w = 0; w < warp; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) then(m[e], wm[w][e * 32 + lane]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        end[e] = m[e];
        then(end[e], wm[warp][e * 32 + lane]);
    }
}

// The state at the start of tile k's group: `first`, or what the group before
// left.  Every warp waits for itself, so that the group's last warp can pass
// the state on without another barrier.
template <int VEC>
__device__ __forceinline__ void group_state(const Chains &c, int chain, int k, float (&s)[VEC]) {
    const int lane = threadIdx.x & 31, g = k / kGroup, groups = (c.tiles + kGroup - 1) / kGroup;
    if (g > 0) wait_states<VEC>(c.states + ((int64_t)chain * groups + g - 1) * (VEC * 32) + lane * VEC, s);
}
template <int VEC>
__device__ __forceinline__ void leave_group(const Chains &c, int chain, int k, const float (&h)[VEC]) {
    const int lane = threadIdx.x & 31, groups = (c.tiles + kGroup - 1) / kGroup;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        put_state(c.states + ((int64_t)chain * groups + k / kGroup) * (VEC * 32) + lane * VEC + e, h[e]);
}

// The tile's own map (warp maps in order), published for the group's later tiles.
template <int VEC, int W>
__device__ __forceinline__ void publish_map(const Chains &c, int chain, int k, const float2 (*wm)[VEC * 32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        float2 m = make_float2(1.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 q = wm[w][e * 32 + lane];
            m.y = fmaf(q.x, m.y, q.y);
            m.x *= q.x;
        }
        put_map(c.maps + ((int64_t)chain * c.tiles + k) * (VEC * 32) + lane * VEC + e, m.x, m.y);
    }
}

// VEC consecutive elements, as loaded and as FP32.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
    return *reinterpret_cast<const Pack<T, VEC> *>(p);
}

// Which of this warp's tokens cut the state.
__device__ __forceinline__ uint32_t cut_mask(const FwdParams &p, int b, int t0, int cnt) {
    if (!p.resets) return 0;
    const int lane = threadIdx.x & 31;
    const bool z = lane < cnt && p.resets[(int64_t)b * p.L + t0 + lane] != 0;
    return __ballot_sync(0xffffffffu, z);
}

// Copies VEC elements to this thread's own place in shared memory,
// asynchronously where they make at least the 4 bytes cp.async takes.
template <typename T, int VEC>
__device__ __forceinline__ void copy_pack(Pack<T, VEC> *dst, const T *src) {
    if constexpr (sizeof(T) * VEC >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src),
                     "n"((int)(sizeof(T) * VEC))
                     : "memory");
    else
        *dst = load_pack<T, VEC>(src);
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool PRECISE>
__device__ __forceinline__ float channel_softplus(float l) {
    return PRECISE ? softplus_channel(l) : softplus_fast(l);
}

// Which tile a ticket stands for: time-major, all chains' k-th tiles together.
struct Tile {
    int chain, k, b, d, n, t0, cnt;
    bool live, in;
};

// ---- forward --------------------------------------------------------------------
// Persistent CTAs: the copies of the next tile's x, r and i into shared memory
// run while the current tile is computed and waits for its state.  A thread
// reads back only what it copied itself, so no barrier guards the buffers.
template <typename T, int VEC, int S, int W>
struct FwdSmem {
    Pack<T, VEC> in[2][3][S][32 * W];
    float2 wm[W][32 * VEC], gm[kGroup][32 * VEC];
    unsigned int ticket[2];
};

template <typename T, int VEC, int S, int W, int CTAS>
__global__ void __launch_bounds__(32 * W, CTAS) recurrence_fwd_kernel(const FwdParams p, const Chains ch) {
    constexpr bool PRECISE = sizeof(T) == 4;
    constexpr int cw = 32 * VEC, TT = S * W;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    auto &sm = *reinterpret_cast<FwdSmem<T, VEC, S, W> *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned total = (unsigned)ch.chains * (unsigned)ch.tiles;

    auto place = [&](unsigned v) {
        Tile t;
        t.k = (int)(v / (unsigned)ch.chains);
        t.chain = (int)(v - (unsigned)t.k * (unsigned)ch.chains);
        t.b = t.chain / ch.blocks;
        t.d = (t.chain - t.b * ch.blocks) * cw + lane * VEC;
        t.n = row_length(p, t.b);
        t.t0 = t.k * TT + warp * S;
        t.live = t.k == 0 || t.k * TT < t.n;  // else behind the row's end
        t.in = t.d < p.D;
        t.cnt = t.in ? min(max(t.n - t.t0, 0), S) : 0;
        return t;
    };
    auto fetch = [&](const Tile &t, int buf) {
        const T *px = static_cast<const T *>(p.x) + t.b * p.sx[0] + t.t0 * p.sx[1] + t.d;
        const T *pr = static_cast<const T *>(p.r) + t.b * p.sr[0] + t.t0 * p.sr[1] + t.d;
        const T *pi = static_cast<const T *>(p.i) + t.b * p.si[0] + t.t0 * p.si[1] + t.d;
#pragma unroll
        for (int j = 0; j < S; ++j)
            if (j < t.cnt) {
                copy_pack<T, VEC>(&sm.in[buf][0][j][tid], pr + j * p.sr[1]);
                copy_pack<T, VEC>(&sm.in[buf][1][j][tid], pi + j * p.si[1]);
                copy_pack<T, VEC>(&sm.in[buf][2][j][tid], px + j * p.sx[1]);
            }
    };

    Tickets tickets(ch.ticket, sm.ticket);
    unsigned v = tickets.next();
    if (v >= total) return;
    Tile t = place(v);
    fetch(t, 0);
    copy_commit();
    for (int buf = 0;; buf ^= 1) {
        const unsigned vn = tickets.next();  // its barrier also frees sm.wm and sm.gm
        Tile tn{};
        if (vn < total) {
            tn = place(vn);
            fetch(tn, buf ^ 1);
        }
        copy_commit();
        copy_wait<1>();
        if (t.live) {
            float a[S][VEC], bt[S][VEC], csp[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) csp[e] = t.in ? p.c * channel_softplus<PRECISE>(p.lambda[t.d + e]) : 0.f;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const Pack<T, VEC> r = sm.in[buf][0][j][tid], gi = sm.in[buf][1][j][tid], x = sm.in[buf][2][j][tid];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const Decay g = decay<PRECISE>(cvt_f32(r.v[e]), csp[e]);
                    float si, om;
                    sigmoid2<PRECISE>(cvt_f32(gi.v[e]), si, om);
                    const float bv = sqrt_gate<PRECISE>(one_minus_a2<PRECISE>(g.y, g.a)) * si * cvt_f32(x.v[e]);
                    a[j][e] = j < t.cnt ? g.a : 1.f;  // what the buffer holds behind the end does not count
                    bt[j][e] = j < t.cnt ? bv : 0.f;
                }
            }
            const uint32_t cut = cut_mask(p, t.b, t.t0, min(max(t.n - t.t0, 0), S));
            if (cut)
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (cut >> j & 1)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) a[j][e] = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float P = 1.f, H = 0.f;
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    H = fmaf(a[j][e], H, bt[j][e]);
                    P *= a[j][e];
                }
                sm.wm[warp][e * 32 + lane] = make_float2(P, H);
            }
            __syncthreads();
            const bool more = (t.k + 1) * TT < t.n;  // a later tile waits for this one
            const bool last = t.k % kGroup == kGroup - 1;
            if (warp == 0 && more && !last) publish_map<VEC, W>(ch, t.chain, t.k, sm.wm);
            float2 m[VEC], end[VEC];
            prefix_maps<VEC, W>(ch, t.chain, t.k, sm.wm, sm.gm, m, end);
            float s[VEC], h[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                s[e] = t.in && p.h0 && t.k < kGroup ? p.h0[(int64_t)t.b * p.D + t.d + e] : 0.f;
            group_state<VEC>(ch, t.chain, t.k, s);
            if (warp == W - 1 && (last || !more)) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[e] = fmaf(end[e].x, s[e], end[e].y);
                if (more)
                    leave_group<VEC>(ch, t.chain, t.k, h);
                else if (t.in && p.hN)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) p.hN[(int64_t)t.b * p.D + t.d + e] = h[e];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[e] = fmaf(m[e].x, s[e], m[e].y);
            T *ph = static_cast<T *>(p.h) + t.b * p.sh[0] + t.t0 * p.sh[1] + t.d;
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (j < t.cnt) {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        h[e] = fmaf(a[j][e], h[e], bt[j][e]);
                        o.v[e] = cvt_out<T>(h[e]);
                    }
                    *reinterpret_cast<Pack<T, VEC> *>(ph + j * p.sh[1]) = o;
                }
        }
        if (vn >= total) break;
        t = tn;
    }
}

// ---- backward -------------------------------------------------------------------
// The same tiles and chains with time reversed; what runs along a chain is
// C_t = keep_t a_t G_t, the part of the gradient that reaches h_{t-1}.
template <typename T, int VEC, int S, int W>
struct BwdSmem {
    Pack<T, VEC> in[2][5][S][32 * W];
    float2 wm[W][32 * VEC], gm[kGroup][32 * VEC];
    float sums[W][32 * VEC];
    unsigned int ticket[2];
};

template <typename T, int VEC, int S, int W, int CTAS>
__global__ void __launch_bounds__(32 * W, CTAS) recurrence_bwd_kernel(const BwdParams p, const Chains ch) {
    constexpr bool PRECISE = sizeof(T) == 4;
    constexpr int cw = 32 * VEC, TT = S * W;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    auto &sm = *reinterpret_cast<BwdSmem<T, VEC, S, W> *>(smem_raw);
    const FwdParams &f = p.f;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned total = (unsigned)ch.chains * (unsigned)ch.tiles;

    auto place = [&](unsigned v) {
        Tile t;
        t.k = (int)(v / (unsigned)ch.chains);
        t.chain = (int)(v - (unsigned)t.k * (unsigned)ch.chains);
        t.b = t.chain / ch.blocks;
        t.d = (t.chain - t.b * ch.blocks) * cw + lane * VEC;
        t.n = row_length(f, t.b);
        const int row_tiles = max((t.n + TT - 1) / TT, 1);
        t.live = t.k < row_tiles;
        t.t0 = (row_tiles - 1 - t.k) * TT + (W - 1 - warp) * S;  // warp 0 holds the tile's last tokens
        t.in = t.d < f.D;
        t.cnt = t.in && t.live ? min(max(t.n - t.t0, 0), S) : 0;
        return t;
    };
    auto fetch = [&](const Tile &t, int buf) {
        const T *pr = static_cast<const T *>(f.r) + t.b * f.sr[0] + t.t0 * f.sr[1] + t.d;
        const T *pg = static_cast<const T *>(p.dh) + t.b * p.sdh[0] + t.t0 * p.sdh[1] + t.d;
        const T *px = static_cast<const T *>(f.x) + t.b * f.sx[0] + t.t0 * f.sx[1] + t.d;
        const T *pi = static_cast<const T *>(f.i) + t.b * f.si[0] + t.t0 * f.si[1] + t.d;
        const T *ph = static_cast<const T *>(f.h) + t.b * f.sh[0] + (t.t0 - 1) * f.sh[1] + t.d;
#pragma unroll
        for (int j = 0; j < S; ++j)
            if (j < t.cnt) {
                copy_pack<T, VEC>(&sm.in[buf][0][j][tid], pr + j * f.sr[1]);
                copy_pack<T, VEC>(&sm.in[buf][1][j][tid], pg + j * p.sdh[1]);
                copy_pack<T, VEC>(&sm.in[buf][2][j][tid], px + j * f.sx[1]);
                copy_pack<T, VEC>(&sm.in[buf][3][j][tid], pi + j * f.si[1]);
                if (t.t0 + j > 0) copy_pack<T, VEC>(&sm.in[buf][4][j][tid], ph + j * f.sh[1]);
            }
    };

    Tickets tickets(ch.ticket, sm.ticket);
    unsigned v = tickets.next();
    if (v >= total) return;
    Tile t = place(v);
    fetch(t, 0);
    copy_commit();
    for (int buf = 0;; buf ^= 1) {
        const unsigned vn = tickets.next();  // its barrier also frees sm.wm and sm.gm
        Tile tn{};
        if (vn < total) {
            tn = place(vn);
            fetch(tn, buf ^ 1);
        }
        copy_commit();
        copy_wait<1>();
        float *part = p.part + ((int64_t)t.b * ch.tiles + t.k) * f.D + t.d;
        if (t.live) {
            float a[S][VEC], y[S][VEC], om[S][VEC], csp[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) csp[e] = t.in ? f.c * channel_softplus<PRECISE>(f.lambda[t.d + e]) : 0.f;
            const uint32_t cut = cut_mask(f, t.b, t.t0, min(max(t.n - t.t0, 0), S));
            float2 own[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) own[e] = make_float2(1.f, 0.f);
#pragma unroll
            for (int j = S - 1; j >= 0; --j) {
                const Pack<T, VEC> r = sm.in[buf][0][j][tid], dh = sm.in[buf][1][j][tid];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const Decay g = decay<PRECISE>(cvt_f32(r.v[e]), csp[e]);
                    a[j][e] = g.a;
                    y[j][e] = g.y;
                    om[j][e] = g.om;
                    if (j < t.cnt) {  // what the buffer holds behind the end does not count
                        const float ak = cut >> j & 1 ? 0.f : g.a;
                        own[e].y = ak * (cvt_f32(dh.v[e]) + own[e].y);
                        own[e].x *= ak;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) sm.wm[warp][e * 32 + lane] = own[e];
            __syncthreads();
            const bool more = t.t0 - (W - 1 - warp) * S > 0;  // an earlier tile waits for this one
            const bool last = t.k % kGroup == kGroup - 1;
            if (warp == 0 && more && !last) publish_map<VEC, W>(ch, t.chain, t.k, sm.wm);
            float2 m[VEC], end[VEC];
            prefix_maps<VEC, W>(ch, t.chain, t.k, sm.wm, sm.gm, m, end);
            float s[VEC], C[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                s[e] = t.in && p.dhN && t.k < kGroup ? p.dhN[(int64_t)t.b * f.D + t.d + e] : 0.f;
            group_state<VEC>(ch, t.chain, t.k, s);
            if (warp == W - 1 && (last || !more)) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) C[e] = fmaf(end[e].x, s[e], end[e].y);
                if (more)
                    leave_group<VEC>(ch, t.chain, t.k, C);
                else if (t.in && p.dh0)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) p.dh0[(int64_t)t.b * f.D + t.d + e] = C[e];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) C[e] = fmaf(m[e].x, s[e], m[e].y);
            T *qx = static_cast<T *>(p.dx) + t.b * p.sdx[0] + t.t0 * p.sdx[1] + t.d;
            T *qr = static_cast<T *>(p.dr) + t.b * p.sdr[0] + t.t0 * p.sdr[1] + t.d;
            T *qi = static_cast<T *>(p.di) + t.b * p.sdi[0] + t.t0 * p.sdi[1] + t.d;
            float sum[VEC] = {};
#pragma unroll
            for (int j = S - 1; j >= 0; --j)
                if (j < t.cnt) {
                    const Pack<T, VEC> dh = sm.in[buf][1][j][tid], x = sm.in[buf][2][j][tid],
                                       gi = sm.in[buf][3][j][tid], hp = sm.in[buf][4][j][tid];
                    Pack<T, VEC> ox, orr, oi;
                    const bool keep = !(cut >> j & 1);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float av = a[j][e], yv = y[j][e], xv = cvt_f32(x.v[e]);
                        const float G = cvt_f32(dh.v[e]) + C[e];
                        C[e] = (keep ? av : 0.f) * G;
                        float si, omi, beta, q;
                        sigmoid2<PRECISE>(cvt_f32(gi.v[e]), si, omi);
                        root_gate<PRECISE>(one_minus_a2<PRECISE>(yv, av), yv, beta, q);
                        float prev = cvt_f32(hp.v[e]);
                        if (t.t0 + j == 0) prev = f.h0 ? f.h0[(int64_t)t.b * f.D + t.d + e] : 0.f;
                        if (!keep) prev = 0.f;
                        const float gx = G * beta * si;
                        const float E = G * (si * xv * av * av * q - yv * av * prev);
                        sum[e] += E;
                        ox.v[e] = cvt_out<T>(gx);
                        oi.v[e] = cvt_out<T>(gx * xv * omi);
                        orr.v[e] = cvt_out<T>(E * om[j][e]);
                    }
                    *reinterpret_cast<Pack<T, VEC> *>(qx + j * p.sdx[1]) = ox;
                    *reinterpret_cast<Pack<T, VEC> *>(qi + j * p.sdi[1]) = oi;
                    *reinterpret_cast<Pack<T, VEC> *>(qr + j * p.sdr[1]) = orr;
                }
            // the tile's sum of E per channel, warps in order
#pragma unroll
            for (int e = 0; e < VEC; ++e) sm.sums[warp][e * 32 + lane] = sum[e];
            __syncthreads();
            if (warp == 0 && t.in)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w) v += sm.sums[w][e * 32 + lane];
                    part[e] = v;
                }
        } else if (warp == 0 && t.in) {  // behind the row's end
#pragma unroll
            for (int e = 0; e < VEC; ++e) part[e] = 0.f;
        }
        if (vn >= total) break;
        t = tn;
    }
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
        float sg, om;
        const float l = lambda[d];
        sigmoid2<true>(l, sg, om);
        dlambda[d] = s * (l < -20.f ? 1.f : sg / softplus_channel(l));
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    recurrence_step_kernel(const T *__restrict__ x, int64_t xrs, const T *__restrict__ r, int64_t rrs,
                           const T *__restrict__ gi, int64_t irs, const float *__restrict__ lambda,
                           const float *s_in, float *s_out, T *__restrict__ h, int64_t hrs, int D, float c) {
    constexpr bool PRECISE = sizeof(T) == 4;
    const int d = blockIdx.x * kThreads + threadIdx.x;
    const int64_t b = blockIdx.y;
    if (d >= D) return;
    const Decay g = decay<PRECISE>(ld_f32(r + b * rrs + d), c * softplus_channel(lambda[d]));
    float si, om;
    sigmoid2<PRECISE>(ld_f32(gi + b * irs + d), si, om);
    const float bt = sqrt_gate<PRECISE>(one_minus_a2<PRECISE>(g.y, g.a)) * si * ld_f32(x + b * xrs + d);
    const float v = fmaf(g.a, s_in[b * D + d], bt);
    s_out[b * D + d] = v;
    h[b * hrs + d] = cvt_out<T>(v);
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
    MB_CHECK_ARG(a->batch <= 65535, "gated_recurrence: batch above 65535");
    if (a->batch == 0 || a->dim == 0) return 0;
    MB_CHECK_ARG(a->lambda && (a->seqlen == 0 || (a->x && a->r && a->i && a->h)), "gated_recurrence: null pointer");
    const size_t es = dtype_size(a->dtype);
    MB_CHECK_ARG(aligned_to(a->x, es) && aligned_to(a->r, es) && aligned_to(a->i, es) && aligned_to(a->h, es) &&
                     aligned_to(a->lambda, 4) && aligned_to(a->initial_state, 4) && aligned_to(a->final_state, 4) &&
                     aligned_to(a->lengths, 4),
                 "gated_recurrence: pointers must be aligned to their element type");
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

// Tile shapes: channels a thread holds (1 serves any alignment and channel
// count), tokens a warp holds, warps and CTAs per SM.
constexpr int kFwdS = 8, kFwdW = 4, kFwdCtas = 4;
constexpr int kBwdS = 8, kBwdW = 4, kBwdCtas = 4;
constexpr int fwd_vec(int dtype) { return dtype == MAMBA_F16 ? 4 : 2; }
constexpr int bwd_vec(int dtype) { return dtype == MAMBA_F16 ? 2 : 1; }

// The chains of a call and where its workspace holds what.
struct Plan {
    Chains ch;
    size_t bytes, part_bytes;
};
bool plan_chains(const MambaRecurrenceArgs *a, bool backward, int vec, Plan &pl) {
    const int tile = backward ? kBwdS * kBwdW : kFwdS * kFwdW, cw = 32 * vec;
    Chains &c = pl.ch;
    c = Chains{};
    const int64_t blocks = ceil_div64(a->dim, cw), tiles = std::max<int64_t>(1, ceil_div64(a->seqlen, tile));
    if (blocks * a->batch * tiles > 0x7fffffffLL) return false;
    c.blocks = (int)blocks;
    c.chains = (int)blocks * a->batch;
    c.tiles = (int)tiles;
    pl.bytes = 256 + (size_t)c.chains * cw * (tiles * sizeof(float2) + ceil_div64(tiles, kGroup) * sizeof(float));
    if (tiles == 1) pl.bytes = 256;
    pl.part_bytes = backward ? ((size_t)a->batch * tiles * a->dim * sizeof(float) + 15) / 16 * 16 : 0;
    return true;
}

}  // namespace

// The largest of the variants that the alignment could choose, so that the
// size does not depend on pointers.
size_t recurrence_workspace_bytes(const MambaRecurrenceArgs *a, bool backward) {
    if (!a || a->batch <= 0 || a->seqlen < 0 || a->dim <= 0) return 0;
    size_t need = 0;
    for (int vec : {1, backward ? bwd_vec(a->dtype) : fwd_vec(a->dtype)}) {
        Plan pl;
        if (!plan_chains(a, backward, vec, pl)) return 0;
        need = std::max(need, pl.bytes + pl.part_bytes);
    }
    return need;
}

namespace {

// Launches one variant: the workspace's part from the ticket on set to all
// ones bits, then persistent CTAs.
template <int VEC, typename Kernel, typename Params>
int launch_tiles(Kernel kernel, const Params &p, Plan &pl, int threads, int ctas, size_t smem, void *ws,
                 cudaStream_t st, const char *what) {
    Chains &c = pl.ch;
    uint8_t *base = static_cast<uint8_t *>(ws) + pl.part_bytes;
    c.ticket = reinterpret_cast<unsigned int *>(base);
    c.maps = reinterpret_cast<float2 *>(base + 256);
    c.states = reinterpret_cast<float *>(c.maps + (int64_t)c.chains * c.tiles * 32 * VEC);
    MB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    MB_CUDA_TRY(cudaMemsetAsync(base, 0xff, pl.bytes, st));
    const int64_t total = (int64_t)c.chains * c.tiles, most = (int64_t)ctas * device_sm_count();
    kernel<<<(unsigned)std::min(total, most), threads, smem, st>>>(p, c);
    return launch_status(what);
}

template <typename T, int VEC>
int launch_forward(const MambaRecurrenceArgs *a, void *ws, cudaStream_t st) {
    Plan pl;
    MB_CHECK_ARG(plan_chains(a, false, VEC, pl), "gated_recurrence: too many tiles");
    return launch_tiles<VEC>(recurrence_fwd_kernel<T, VEC, kFwdS, kFwdW, kFwdCtas>, fwd_params(a), pl, 32 * kFwdW,
                             kFwdCtas, sizeof(FwdSmem<T, VEC, kFwdS, kFwdW>), ws, st, "gated_recurrence kernel");
}
template <typename T>
int choose_forward(const MambaRecurrenceArgs *a, void *ws, cudaStream_t st) {
    constexpr int V = fwd_vec(sizeof(T) == 2 ? MAMBA_F16 : MAMBA_F32);
    const bool vec = a->dim % V == 0 && vector_rows<T, V>(a->x, a->x_stride) && vector_rows<T, V>(a->r, a->r_stride) &&
                     vector_rows<T, V>(a->i, a->i_stride) && vector_rows<T, V>(a->h, a->h_stride);
    return vec ? launch_forward<T, V>(a, ws, st) : launch_forward<T, 1>(a, ws, st);
}

template <typename T, int VEC>
int launch_backward(const MambaRecurrenceArgs *a, BwdParams &p, void *ws, cudaStream_t st, int &tiles) {
    Plan pl;
    MB_CHECK_ARG(plan_chains(a, true, VEC, pl), "gated_recurrence_backward: too many tiles");
    tiles = pl.ch.tiles;
    return launch_tiles<VEC>(recurrence_bwd_kernel<T, VEC, kBwdS, kBwdW, kBwdCtas>, p, pl, 32 * kBwdW, kBwdCtas,
                             sizeof(BwdSmem<T, VEC, kBwdS, kBwdW>), ws, st, "gated_recurrence_backward kernel");
}
template <typename T>
int choose_backward(const MambaRecurrenceArgs *a, BwdParams &p, const MambaRecurrenceGrads *g, void *ws,
                    cudaStream_t st) {
    constexpr int V = bwd_vec(sizeof(T) == 2 ? MAMBA_F16 : MAMBA_F32);
    const bool vec = a->dim % V == 0 && vector_rows<T, V>(a->x, a->x_stride) && vector_rows<T, V>(a->r, a->r_stride) &&
                     vector_rows<T, V>(a->i, a->i_stride) && vector_rows<T, V>(a->h, a->h_stride) &&
                     vector_rows<T, V>(g->dh, g->dh_stride) && vector_rows<T, V>(g->dx, g->dx_stride) &&
                     vector_rows<T, V>(g->dr, g->dr_stride) && vector_rows<T, V>(g->di, g->di_stride);
    int tiles = 0;
    if (vec ? launch_backward<T, V>(a, p, ws, st, tiles) : launch_backward<T, 1>(a, p, ws, st, tiles)) return -1;
    recurrence_dlambda_kernel<<<(unsigned)ceil_div(a->dim, 32), 32 * kSumWarps, 0, st>>>(
        p.part, a->lambda, g->dlambda, (int64_t)a->batch * tiles, a->dim);
    return launch_status("gated_recurrence_backward sum kernel");
}

}  // namespace

int recurrence_forward(const MambaRecurrenceArgs *a, void *ws, size_t ws_bytes, cudaStream_t st) {
    if (check_args(a, false)) return -1;
    if (a->batch == 0 || a->dim == 0) return 0;
    const size_t need = recurrence_workspace_bytes(a, false);
    MB_CHECK_ARG(need, "gated_recurrence: too many tiles");
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
    MB_CHECK_ARG(output_rows_disjoint(g->dx_stride, a->batch, a->seqlen, a->dim) &&
                     output_rows_disjoint(g->dr_stride, a->batch, a->seqlen, a->dim) &&
                     output_rows_disjoint(g->di_stride, a->batch, a->seqlen, a->dim),
                 "gated_recurrence_backward: rows of a gradient overlap (strides)");
    const size_t need = recurrence_workspace_bytes(a, true);
    MB_CHECK_ARG(need, "gated_recurrence_backward: too many tiles");
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
    p.part = static_cast<float *>(ws);
    for (int k = 0; k < 2; ++k) {
        p.sdh[k] = g->dh_stride[k];
        p.sdx[k] = g->dx_stride[k];
        p.sdr[k] = g->dr_stride[k];
        p.sdi[k] = g->di_stride[k];
    }
    return a->dtype == MAMBA_F16 ? choose_backward<__half>(a, p, g, ws, st) : choose_backward<float>(a, p, g, ws, st);
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
    MB_CHECK_ARG(batch <= 65535, "gated_recurrence_step: batch above 65535");
    if (batch == 0 || dim == 0) return 0;
    MB_CHECK_ARG(x && r && i && lambda && state_in && state_out && h, "gated_recurrence_step: null pointer");
    const size_t es = dtype_size(dtype);
    MB_CHECK_ARG(aligned_to(x, es) && aligned_to(r, es) && aligned_to(i, es) && aligned_to(h, es) &&
                     aligned_to(lambda, 4) && aligned_to(state_in, 4) && aligned_to(state_out, 4),
                 "gated_recurrence_step: pointers must be aligned to their element type");
    MB_CHECK_ARG(batch == 1 || hrs >= dim, "gated_recurrence_step: rows of h overlap (stride)");
    const dim3 grid((unsigned)ceil_div(dim, kThreads), (unsigned)batch);
    if (dtype == MAMBA_F16)
        recurrence_step_kernel<__half><<<grid, kThreads, 0, st>>>(
            static_cast<const __half *>(x), xrs, static_cast<const __half *>(r), rrs, static_cast<const __half *>(i),
            irs, lambda, state_in, state_out, static_cast<__half *>(h), hrs, dim, c);
    else
        recurrence_step_kernel<float><<<grid, kThreads, 0, st>>>(
            static_cast<const float *>(x), xrs, static_cast<const float *>(r), rrs, static_cast<const float *>(i), irs,
            lambda, state_in, state_out, static_cast<float *>(h), hrs, dim, c);
    return launch_status("gated_recurrence_step kernel");
}

}  // namespace mb
