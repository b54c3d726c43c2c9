// scan_bwd.cu -- gradients of the fused selective scan (selective_scan of
// scan.cu; Sources/CPURef/selective_scan_cpu.cpp:17-41).  Per (b, t, d), with
// dt = softplus(delta + dt_bias), a = e^(dt A), phi = (a - 1) / A (dt for A ->
// 0), w = B x, h_t = a h_{t-1} + phi w and q = dy SiLU(z):
//   g_t = C_t q_t + a_{t+1} g_{t+1}                      (over reversed time)
//   dz = dy SiLU'(z) (sum_n C h + D x)
//   dx = D q + sum_n g phi B,      dD = sum q x
//   dB = sum_d g phi x,            dC = sum_d q h_t
//   ddelta = sigmoid(delta + dt_bias) sum_n g a (A h_{t-1} + w)
//   dA = sum g (dt a h_{t-1} + w psi),   psi = (dt a - phi) / A
// a - 1 is evaluated without cancellation (e): phi = e / A.  With FP16 tensors a
// state and token has only e where |dt A| < 1/16 (h_t = h + e (h + w / A), a g =
// g + e g) and only a elsewhere (h_t = a (h + w / A) - w / A): from the other of
// the two, what a weak decay takes or a strong one leaves would be lost.  Of A
// the kernels keep A2 = A log2(e) and K2 = 1 / A2, with B log2(e) in place of B,
// so that w / A = w2 K2.  dA is summed as A dA = sum r dt ln 2 h_{t-1} + w2 g (dt
// a - phi) / log2(e) with r = g a A2.  A state with |A| < 1e-20 counts as 1e-20,
// where all of these are the limits.
//
// Three passes over time chunks:
//   1. forward: the state before every 8th token (a checkpoint), from zero at
//      the start of each chunk; with several chunks also each chunk's map
//      (its end state H, the reverse carry G and the sum of dt),
//   2. (several chunks) the state entering each chunk and the carry entering
//      it from behind,
//   3. backward, 8 tokens at a time: the states from the checkpoint on, kept in
//      tensor memory, then the reverse steps over them.
// A CTA holds 128 channels: a thread has 4 channels x 4 states, two channels to
// each packed operation, so a row's x, dt and q are one 16-byte access for 4
// channels, and the sums over channels (dB, dC) and states (dx, ddelta, y) are
// half done before the first shuffle.  dB and dC leave as one partial row per
// block of 128 channels, dA, dD and ddt_bias as one per chunk and batch; a last
// kernel adds them in order.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "scan_math.cuh"
#include "umma.cuh"

namespace mb {
namespace {

constexpr int kT = 8;        // tokens between checkpoints
constexpr int kCh = 128;     // channels (and threads) per CTA
constexpr int kN = 16;       // states, padded: fewer cost the same (8 x 2048 x 4096 with 4 states 3.17 ms, 16 3.17)
constexpr int kHalf = kT / 2;  // tokens that a thread stages, of two channels

struct ScanGradParams {
    const void *x, *delta, *dy, *z, *B, *C;
    const float *A, *D, *dt_bias, *h0, *dfinal;
    void *dx, *ddelta, *dz;
    float *dh0;
    // States are kept as [dim / 4 rounded up][16 states][4 channels].
    float *ck;    // [batch][subs][states] before every 8th token
    float *ck_dt; // [batch][subs][dim4] sum of dt before it, since the chunk's start
    float *H, *G; // [batch][chunks][states]
    float *S;     // [batch][chunks][dim]
    float *part_bc;  // [blocks][batch * L][32]
    float *part_a;   // [batch * chunks][sums_of(dim)]: dA [states], dD [dim], ddt_bias [dim]
    int batch, L, dim, N, chunk, chunks, subs, blocks;
    int64_t per;     // floats of one set of states
    int dim4;        // dim to the next multiple of 4
    bool pairs;      // two adjacent channels can be loaded and stored as one
    int64_t sx[3], sdelta[3], sdy[3], sz[3], sB[3], sC[3], sdx[3], sddelta[3], sdz[3];
};

__host__ __device__ __forceinline__ int64_t states_of(int dim) { return ((int64_t)dim + 3) / 4 * (4 * kN); }
// Floats of a partial row of dA, dD and ddt_bias, a multiple of 4.
__host__ __device__ __forceinline__ int64_t sums_of(int dim) { return states_of(dim) + (2 * (int64_t)dim + 3) / 4 * 4; }
__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 make2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 lo2(const float4 &v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(const float4 &v) { return make_float2(v.z, v.w); }

// max and min that keep a NaN
__device__ __forceinline__ float clamp_nan(float v, float lo, float hi) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(lo));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(hi));
    return r;
}

// e = 2^v - 1, and a = 2^v, for two states.
// FP16 tensors: where |dt A| is below 1/16 (near) e by the series to the fourth
// power (relative error 2e-7), elsewhere one approximate exponential a (2e-7;
// that of a - 1 is up to 2e-6).  Either is returned in e.
// FP32 tensors: v = j + f with j whole and |f| <= 1/2, 2^f - 1 = f q(f) with q
// interpolating (2^f - 1) / f at the six Chebyshev nodes of [-1/2, 1/2]
// (relative error 7e-8), a = 2^j (1 + f q), e = 2^j f q + (2^j - 1).
constexpr float kNear = 0.0625f * 1.4426950408889634f;
__device__ __forceinline__ bool is_near(float v) { return fabsf(v) < kNear; }
template <bool PRECISE>
__device__ __forceinline__ void exp2m1_2(float2 v, float2 &e, float2 &a) {
    if (PRECISE) {
        v.x = clamp_nan(v.x, -125.f, 127.f);
        v.y = clamp_nan(v.y, -125.f, 127.f);
        const float2 t = fadd2(v, make2(12582912.f));  // j in the low bits
        const float2 f = ffma2(fadd2(t, make2(-12582912.f)), make2(-1.f), v);
        float2 s = ffma2(f, make2(1.545316336e-04f), make2(1.339086331e-03f));
        s = ffma2(s, f, make2(9.618083015e-03f));
        s = ffma2(s, f, make2(5.550356954e-02f));
        s = ffma2(s, f, make2(2.402265072e-01f));
        s = ffma2(s, f, make2(6.931471825e-01f));
        s = fmul2(s, f);
        const float2 m = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                                     __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000));
        e = ffma2(m, s, fadd2(m, make2(-1.f)));
        a = ffma2(m, s, m);
        return;
    }
    constexpr float c1 = 0.69314718055994531f, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
    const float2 far = make_float2(ex2_approx(v.x), ex2_approx(v.y));
    float2 s = ffma2(v, make2(c4), make2(c3));
    s = ffma2(s, v, make2(c2));
    s = ffma2(s, v, make2(c1));
    s = fmul2(s, v);
    e = make_float2(is_near(v.x) ? s.x : far.x, is_near(v.y) ? s.y : far.y);
}
// (a - 1) K2 = phi / log2(e).
template <bool PRECISE>
__device__ __forceinline__ float2 phi_2(float2 v, float2 e, float2 K2) {
    if (PRECISE) return fmul2(e, K2);
    return ffma2(e, K2, make_float2(is_near(v.x) ? 0.f : -K2.x, is_near(v.y) ? 0.f : -K2.y));
}

// a x (FP16 tensors, near: x + e x).
template <bool PRECISE>
__device__ __forceinline__ float2 decay_2(float2 v, float2 e, float2 a, float2 x) {
    if (PRECISE) return fmul2(a, x);
    return ffma2(e, x, make_float2(is_near(v.x) ? x.x : 0.f, is_near(v.y) ? x.y : 0.f));
}
// h_t = a h + phi w (FP16 tensors: a (h + w / A) - w / A, near h + e (h + w / A)).
template <bool PRECISE>
__device__ __forceinline__ float2 step_2(float2 v, float2 e, float2 a, float2 w, float2 K2, float2 h) {
    if (PRECISE) return ffma2(fmul2(e, K2), w, fmul2(a, h));
    const float2 wk = fmul2(w, K2);
    return ffma2(e, fadd2(h, wk), make_float2(is_near(v.x) ? h.x : -wk.x, is_near(v.y) ? h.y : -wk.y));
}

// g (dt a - phi) / log2(e) from e, phi / log2(e) = (a - 1) / A2 and dt ln 2, and
// from g a and g phi.  The difference loses 2 d / x^2 of its value for an absolute
// error d of e, where x = dt A: so below |x| = 0.4 (d = 6e-8: 8e-7; FP32 tensors,
// whose e has a relative error, 0.25) phi (x / (1 - e^-x) - 1) by x/2 + x^2/12 -
// x^4/720 (the next term is 7e-7 of the sum at 0.4).  FP16 tensors: the roundings
// of g a and g phi are 3e-7 of the difference at 0.4 each.
template <bool PRECISE>
__device__ __forceinline__ float2 bend_2(float2 v, float2 e, float2 phi, float2 dt_ln2, float2 g, float2 ga,
                                         float2 gphi) {
    constexpr float c1 = 0.69314718055994531f, c2 = c1 * c1 / 12, c4 = -c1 * c1 * c1 * c1 / 720;
    constexpr float near = (PRECISE ? 0.25f : 0.4f) * kLog2e;
    const float2 far = PRECISE ? fmul2(g, ffma2(phi, make2(-1.f), ffma2(dt_ln2, e, dt_ln2)))
                               : ffma2(dt_ln2, ga, make_float2(-gphi.x, -gphi.y));
    float2 s = ffma2(fmul2(v, v), make2(c4), make2(c2));
    s = ffma2(s, v, make2(c1 / 2));
    s = fmul2(fmul2(s, v), gphi);
    return make_float2(fabsf(v.x) < near ? s.x : far.x, fabsf(v.y) < near ? s.y : far.y);
}

template <bool PRECISE>
__device__ __forceinline__ float softplus_of(float v) {
    return PRECISE ? fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))) : softplus_fast(v);
}
template <bool PRECISE>
__device__ __forceinline__ float sigmoid_of(float v) {
    const float e = PRECISE ? expf(-fabsf(v)) : ex2_approx(-fabsf(v) * kLog2e);
    const float t = PRECISE ? __fdiv_rn(1.f, 1.f + e) : rcp_approx(1.f + e);
    return v >= 0.f ? t : e * t;
}

// Two channels of one row.
template <typename T> struct Pair;
template <> struct Pair<float> {
    float2 v;
    __device__ __forceinline__ float2 f32() const { return v; }
    static __device__ __forceinline__ Pair of(float2 v) { return {v}; }
    static __device__ __forceinline__ Pair zero() { return {make_float2(0.f, 0.f)}; }
};
template <> struct Pair<__half> {
    __half2 v;
    __device__ __forceinline__ float2 f32() const { return __half22float2(v); }
    static __device__ __forceinline__ Pair of(float2 v) { return {__float22half2_rn(v)}; }
    static __device__ __forceinline__ Pair zero() { return {__float2half2_rn(0.f)}; }
};
template <typename T>
__device__ __forceinline__ Pair<T> load_pair(const T *p, int64_t sc, bool pairs, bool second) {
    if (pairs) return *reinterpret_cast<const Pair<T> *>(p);
    Pair<T> r = Pair<T>::zero();
    r.v.x = p[0];
    if (second) r.v.y = p[sc];
    return r;
}
template <typename T>
__device__ __forceinline__ void store_pair(T *p, int64_t sc, bool pairs, bool second, float2 v) {
    const Pair<T> r = Pair<T>::of(v);
    if (pairs) {
        *reinterpret_cast<Pair<T> *>(p) = r;
    } else {
        p[0] = r.v.x;
        if (second) p[sc] = r.v.y;
    }
}

// One thread's inputs of 8 tokens: channels 2 (tid % 64) and the next of the
// block, tokens 4 (tid / 64) .. + 3, and two of the 8 x 32 values of B and C.
// What lies behind the last token or channel is zero.
template <typename Tx, typename Td, typename Tb>
struct RawRows {
    Pair<Tx> x[kHalf], dy[kHalf], z[kHalf];
    Pair<Td> delta[kHalf];
    Tb bc[2];
    __device__ __forceinline__ void load(const ScanGradParams &p, int b, int t0, int end, int c, bool grads) {
        const bool second = c + 1 < p.dim;
#pragma unroll
        for (int k = 0; k < kHalf; ++k) {
            const int64_t t = t0 + k + (threadIdx.x >> 6) * kHalf;
            x[k] = dy[k] = z[k] = Pair<Tx>::zero();
            delta[k] = Pair<Td>::zero();
            if (t < end && c < p.dim) {
                x[k] = load_pair(static_cast<const Tx *>(p.x) + b * p.sx[0] + t * p.sx[1] + c * p.sx[2], p.sx[2],
                                 p.pairs, second);
                delta[k] = load_pair(static_cast<const Td *>(p.delta) + b * p.sdelta[0] + t * p.sdelta[1] +
                                         c * p.sdelta[2],
                                     p.sdelta[2], p.pairs, second);
                if (grads) {
                    dy[k] = load_pair(static_cast<const Tx *>(p.dy) + b * p.sdy[0] + t * p.sdy[1] + c * p.sdy[2],
                                      p.sdy[2], p.pairs, second);
                    if (p.z)
                        z[k] = load_pair(static_cast<const Tx *>(p.z) + b * p.sz[0] + t * p.sz[1] + c * p.sz[2],
                                         p.sz[2], p.pairs, second);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = threadIdx.x + k * kCh, n = at & 15;
            const int64_t t = t0 + (at >> 5);
            bc[k] = cvt_out<Tb>(0.f);
            if (t < end && n < p.N)
                bc[k] = at & 16 ? static_cast<const Tb *>(p.C)[b * p.sC[0] + t * p.sC[1] + n * p.sC[2]]
                                : static_cast<const Tb *>(p.B)[b * p.sB[0] + t * p.sB[1] + n * p.sB[2]];
        }
    }
    // B log2(e) and C, each value twice in a row: {B, B, C, C} per token and state,
    // state n at n % 4 * 4 + n / 4, so that the four lanes of a quad, 4 states
    // apart, read 64 bytes in a row (without that, two of them share banks).
    __device__ __forceinline__ void stage_bc(float4 (&bc4)[kT][kN]) const {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = threadIdx.x + k * kCh;
            const float v = cvt_f32<Tb>(bc[k]) * (at & 16 ? 1.f : kLog2e);
            reinterpret_cast<float2 *>(&bc4[at >> 5][(at & 3) * 4 + ((at >> 2) & 3)])[(at >> 4) & 1] = make2(v);
        }
    }
};

// A2 and K2 of a thread's 4 states x 4 channels.
__device__ __forceinline__ void load_A(const ScanGradParams &p, int c4, int n4, float2 (&A2)[4][2], float2 (&K2)[4][2]) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = c4 + 2 * h + e;
                v[e] = c < p.dim && n4 + s < p.N ? p.A[(int64_t)c * p.N + n4 + s] : 0.f;
                if (fabsf(v[e]) < 1e-20f) v[e] = 1e-20f;
                v[e] *= kLog2e;
            }
            A2[s][h] = make_float2(v[0], v[1]);
            K2[s][h] = make_float2(__frcp_rn(v[0]), __frcp_rn(v[1]));
        }
}

// A thread's states from the caller's [dim][N] rows (zero without any).
__device__ __forceinline__ void load_given(const ScanGradParams &p, const float *rows, int b, int c4, int n4,
                                           float2 (&v)[4][2]) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float q[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = c4 + 2 * h + e;
                q[e] = rows && c < p.dim && n4 + s < p.N ? rows[((int64_t)b * p.dim + c) * p.N + n4 + s] : 0.f;
            }
            v[s][h] = make_float2(q[0], q[1]);
        }
}
// A thread's states from and to the workspace.
__device__ __forceinline__ void load_states(const float *set, int dim, int c4, int n4, float2 (&v)[4][2]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c4 < dim) q = *reinterpret_cast<const float4 *>(set + (int64_t)c4 * kN + (n4 + s) * 4);
        v[s][0] = lo2(q);
        v[s][1] = hi2(q);
    }
}
__device__ __forceinline__ void store_states(float *set, int dim, int c4, int n4, const float2 (&v)[4][2]) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
        if (c4 < dim)
            *reinterpret_cast<float4 *>(set + (int64_t)c4 * kN + (n4 + s) * 4) =
                make_float4(v[s][0].x, v[s][0].y, v[s][1].x, v[s][1].y);
}

struct Place {
    int block, chunk, b;
};
__device__ __forceinline__ Place place(const ScanGradParams &p) {
    Place r;
    r.block = blockIdx.x % p.blocks;
    const int rest = blockIdx.x / p.blocks;
    r.chunk = rest % p.chunks;
    r.b = rest / p.chunks;
    return r;
}

// Pass 1: 0.82 ms of the call below; with its inputs fetched a round ahead (three
// CTAs an SM) 0.05 more.
template <typename Tx, typename Td, typename Tb, bool MULTI>
__global__ void __launch_bounds__(kCh, 4) scan_bwd_states_kernel(const ScanGradParams p) {
    constexpr bool PRECISE = sizeof(Tx) == 4;
    __shared__ __align__(16) float xs[2][kT][kCh], dts[2][kT][kCh], qs[MULTI ? 2 : 1][kT][MULTI ? kCh : 4];
    __shared__ float4 bc4[2][kT][kN];
    __shared__ __align__(16) float half_dt[2][2][kCh];  // sums of dt over the tokens of either half
    const Place at = place(p);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int l2 = (tid & 63) * 2, k0 = (tid >> 6) * kHalf, c2 = at.block * kCh + l2;  // what this thread stages
    const int l4 = warp * 32 + (lane >> 2) * 4, c4 = at.block * kCh + l4, n4 = (lane & 3) * 4;
    const int t_first = at.chunk * p.chunk, t_end = min(p.L, t_first + p.chunk);
    float2 bias = make2(0.f);
    if (p.dt_bias && c2 < p.dim) bias = make_float2(p.dt_bias[c2], c2 + 1 < p.dim ? p.dt_bias[c2 + 1] : 0.f);
    float2 A2[4][2], K2[4][2], h[4][2], P[4][2], G[4][2];
    load_A(p, c4, n4, A2, K2);
    load_given(p, at.chunk == 0 ? p.h0 : nullptr, at.b, c4, n4, h);
    float2 since[2] = {make2(0.f), make2(0.f)};  // sum of dt
    if (MULTI) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                P[s][i] = make2(1.f);
                G[s][i] = make2(0.f);
            }
    }
    float2 sum_dt = make2(0.f);  // of this thread's tokens
    RawRows<Tx, Td, Tb> raw;
    int buf = 0;
    for (int t0 = t_first; t0 < t_end; t0 += kT, buf ^= 1) {
        const int64_t sub = (int64_t)at.b * p.subs + t0 / kT;
        raw.load(p, at.b, t0, t_end, c2, MULTI);
        store_states(p.ck + sub * p.per, p.dim, c4, n4, h);
        if (MULTI) *reinterpret_cast<float2 *>(&half_dt[buf][tid >> 6][l2]) = sum_dt;
#pragma unroll
        for (int k = 0; k < kHalf; ++k) {
            const bool live = t0 + k0 + k < t_end;
            const float2 d = raw.delta[k].f32();
            float2 dt = make2(0.f);
            if (live && c2 < p.dim) dt.x = softplus_of<PRECISE>(d.x + bias.x);
            if (live && c2 + 1 < p.dim) dt.y = softplus_of<PRECISE>(d.y + bias.y);
            *reinterpret_cast<float2 *>(&xs[buf][k0 + k][l2]) = raw.x[k].f32();
            *reinterpret_cast<float2 *>(&dts[buf][k0 + k][l2]) = dt;
            if (MULTI) {
                sum_dt = fadd2(sum_dt, dt);
                float2 q = raw.dy[k].f32();
                if (p.z) {
                    const float2 z = raw.z[k].f32();
                    float2 gate, slope;
                    silu_grad<PRECISE>(z.x, gate.x, slope.x);
                    silu_grad<PRECISE>(z.y, gate.y, slope.y);
                    q = fmul2(q, gate);
                }
                *reinterpret_cast<float2 *>(&qs[buf][k0 + k][l2]) = q;
            }
        }
        raw.stage_bc(bc4[buf]);
        __syncthreads();  // the other buffer's readers are behind this barrier's predecessor
        if (MULTI && at.block * kCh + tid < p.dim4)
            p.ck_dt[sub * p.dim4 + at.block * kCh + tid] = half_dt[buf][0][tid] + half_dt[buf][1][tid];
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const float4 x4 = *reinterpret_cast<const float4 *>(&xs[buf][k][l4]);
            const float4 d4 = *reinterpret_cast<const float4 *>(&dts[buf][k][l4]);
            const float2 x2[2] = {lo2(x4), hi2(x4)}, d2[2] = {lo2(d4), hi2(d4)};
            float2 q2[2];
            if (MULTI) {
                const float4 q4 = *reinterpret_cast<const float4 *>(&qs[buf][k][l4]);
                q2[0] = lo2(q4);
                q2[1] = hi2(q4);
                since[0] = fadd2(since[0], d2[0]);
                since[1] = fadd2(since[1], d2[1]);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float4 bc = bc4[buf][k][s * 4 + (lane & 3)];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float2 e, a;
                    const float2 v = fmul2(d2[i], A2[s][i]);
                    exp2m1_2<PRECISE>(v, e, a);
                    h[s][i] = step_2<PRECISE>(v, e, a, fmul2(x2[i], lo2(bc)), K2[s][i], h[s][i]);
                    if (MULTI) {
                        // the decay since the chunk's start
                        if (PRECISE) {
                            P[s][i] = fmul2(a, P[s][i]);
                        } else {  // as a product the 16 P would spill (890 us in place of 821)
                            const float2 u = fmul2(since[i], A2[s][i]);
                            P[s][i] = make_float2(ex2_approx(u.x), ex2_approx(u.y));
                        }
                        G[s][i] = ffma2(P[s][i], fmul2(hi2(bc), q2[i]), G[s][i]);
                    }
                }
            }
        }
    }
    if (MULTI) {
        const int64_t chunk = (int64_t)at.b * p.chunks + at.chunk;
        store_states(p.H + chunk * p.per, p.dim, c4, n4, h);
        store_states(p.G + chunk * p.per, p.dim, c4, n4, G);
        *reinterpret_cast<float2 *>(&half_dt[buf][tid >> 6][l2]) = sum_dt;
        __syncthreads();
        if (at.block * kCh + tid < p.dim)
            p.S[chunk * p.dim + at.block * kCh + tid] = half_dt[buf][0][tid] + half_dt[buf][1][tid];
    }
}

// Pass 2: a thread per (batch, channel, state) walks the chunks, forward for
// the state that enters each (into H; chunk 0's is in its checkpoints already,
// so H there becomes 0), backward for the carry that enters it from behind
// (into G).
__global__ void __launch_bounds__(256) scan_bwd_carry_kernel(const ScanGradParams p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.batch * p.per) return;
    const int64_t b = i / p.per, at = i - b * p.per;
    const int d = (int)(at / (4 * kN)) * 4 + (int)(at & 3), n = (int)(at % (4 * kN)) / 4;
    if (d >= p.dim) return;
    float A2 = n < p.N ? p.A[(int64_t)d * p.N + n] : 0.f;
    if (fabsf(A2) < 1e-20f) A2 = 1e-20f;
    A2 *= kLog2e;
    float *H = p.H + b * p.chunks * p.per + at, *G = p.G + b * p.chunks * p.per + at;
    const float *S = p.S + b * p.chunks * p.dim + d;
    // 16 chunks' loads at a time: they do not wait for the stores between them
    constexpr int kAhead = 16;
    float h = 0.f;
    for (int k0 = 0; k0 < p.chunks; k0 += kAhead) {
        float end[kAhead], sum[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (k0 + u < p.chunks) {
                end[u] = H[(k0 + u) * p.per];
                sum[u] = S[(int64_t)(k0 + u) * p.dim];
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (k0 + u < p.chunks) {
                H[(k0 + u) * p.per] = h;
                h = k0 + u == 0 ? end[u] : fmaf(exp2f(A2 * sum[u]), h, end[u]);
            }
    }
    float g = p.dfinal && n < p.N ? p.dfinal[(b * p.dim + d) * p.N + n] : 0.f;
    for (int k0 = p.chunks - 1; k0 >= 0; k0 -= kAhead) {
        float own[kAhead], sum[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (k0 - u >= 0) {
                own[u] = G[(k0 - u) * p.per];
                sum[u] = S[(int64_t)(k0 - u) * p.dim];
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (k0 - u >= 0) {
                G[(k0 - u) * p.per] = g;
                g = fmaf(exp2f(A2 * sum[u]), g, own[u]);
            }
    }
}

// Sum over the 4 lanes of a quad: lane j is left with v[j]'s.
__device__ __forceinline__ float quad_sum(const float2 (&v)[2], int j) {
    const bool hi = j & 2, odd = j & 1;
    float a = hi ? v[1].x : v[0].x, b = hi ? v[1].y : v[0].y;
    a += __shfl_xor_sync(0xffffffffu, hi ? v[0].x : v[1].x, 2);
    b += __shfl_xor_sync(0xffffffffu, hi ? v[0].y : v[1].y, 2);
    return (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
}
// Sum over the 8 lanes with the same lane & 3: lane l is left with v[l >> 2]'s.
__device__ __forceinline__ float oct_sum(const float (&v)[8], int lane) {
    float a[4], b[2];
    const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        a[k] = (b4 ? v[4 + k] : v[k]) + __shfl_xor_sync(0xffffffffu, b4 ? v[k] : v[4 + k], 16);
#pragma unroll
    for (int k = 0; k < 2; ++k)
        b[k] = (b3 ? a[2 + k] : a[k]) + __shfl_xor_sync(0xffffffffu, b3 ? a[k] : a[2 + k], 8);
    return (b2 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, b2 ? b[0] : b[1], 4);
}

// A thread's 16 values to and from its lane of tensor memory, 16 columns from
// `at` on.  (These touch no other memory, so there is no memory clobber; the
// load waits for itself.)
__device__ __forceinline__ void tmem_put(uint32_t at, const float2 (&v)[4][2]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
        " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "f"(v[0][0].x), "f"(v[0][0].y), "f"(v[0][1].x), "f"(v[0][1].y), "f"(v[1][0].x), "f"(v[1][0].y),
        "f"(v[1][1].x), "f"(v[1][1].y), "f"(v[2][0].x), "f"(v[2][0].y), "f"(v[2][1].x), "f"(v[2][1].y),
        "f"(v[3][0].x), "f"(v[3][0].y), "f"(v[3][1].x), "f"(v[3][1].y));
}
__device__ __forceinline__ void tmem_get(uint32_t at, float2 (&v)[4][2]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0][0].x), "=f"(v[0][0].y), "=f"(v[0][1].x), "=f"(v[0][1].y), "=f"(v[1][0].x), "=f"(v[1][0].y),
          "=f"(v[1][1].x), "=f"(v[1][1].y), "=f"(v[2][0].x), "=f"(v[2][0].y), "=f"(v[2][1].x), "=f"(v[2][1].y),
          "=f"(v[3][0].x), "=f"(v[3][0].y), "=f"(v[3][1].x), "=f"(v[3][1].y)
        : "r"(at));
}

// 16 values each from 32 columns in a row.
__device__ __forceinline__ void tmem_get(uint32_t at, float2 (&v)[4][2], float2 (&w)[4][2]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
        " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0][0].x), "=f"(v[0][0].y), "=f"(v[0][1].x), "=f"(v[0][1].y), "=f"(v[1][0].x), "=f"(v[1][0].y),
          "=f"(v[1][1].x), "=f"(v[1][1].y), "=f"(v[2][0].x), "=f"(v[2][0].y), "=f"(v[2][1].x), "=f"(v[2][1].y),
          "=f"(v[3][0].x), "=f"(v[3][0].y), "=f"(v[3][1].x), "=f"(v[3][1].y), "=f"(w[0][0].x), "=f"(w[0][0].y),
          "=f"(w[0][1].x), "=f"(w[0][1].y), "=f"(w[1][0].x), "=f"(w[1][0].y), "=f"(w[1][1].x), "=f"(w[1][1].y),
          "=f"(w[2][0].x), "=f"(w[2][0].y), "=f"(w[2][1].x), "=f"(w[2][1].y), "=f"(w[3][0].x), "=f"(w[3][0].y),
          "=f"(w[3][1].x), "=f"(w[3][1].y)
        : "r"(at));
}

// Pass 3.  The states before each of 8 tokens are 128 columns of tensor memory
// (a thread's own lane), and with FP16 tensors the e or a of each token 128 more,
// so that the reverse steps do not evaluate it again; there the state behind a
// token is loaded too (the next one's), which costs less than to compute it.
//
// 42 instructions a state and token, about 18 of them packed (which take two issue
// slots), at 0.51 instructions a cycle and scheduler with two warps each: FMA pipe
// 46%, special functions 14%, DRAM 6%, none of them full; warps wait for the
// fixed latency of what they issued last as often as they issue.  8 x 2048 x 4096
// FP16: 2.29 ms with two CTAs an SM and 255 registers.  Measured when e
// stood for a as well (2.24): the states in shared memory 2.8 ms; three CTAs, 168
// registers and 128 columns 3.07; two CTAs without e 2.77; scalar operations
// 2.39; the next token's values loaded during the sums over lanes 2.28.
template <typename Tx, typename Td, typename Tb, bool MULTI>
__global__ void __launch_bounds__(kCh, 2) scan_bwd_kernel(const ScanGradParams p) {
    constexpr bool PRECISE = sizeof(Tx) == 4, KEEP_E = !PRECISE;
    constexpr uint32_t SLOT = KEEP_E ? 2 * kN : kN, COLUMNS = kT * SLOT;  // tensor-memory columns of a token, of all
    __shared__ __align__(16) float xs[kT][kCh];   // x, later dx
    __shared__ __align__(16) float dts[kT][kCh];  // dt, later the gradient of dt
    __shared__ __align__(16) float qs[kT][kCh];   // q, later sum_n C h + D x
    __shared__ __align__(16) float fz[kT][kCh];   // dy SiLU'(z)
    __shared__ __align__(16) float fd[kT][kCh];   // sigmoid(delta + dt_bias)
    __shared__ float4 bc4[kT][kN];
    __shared__ float red[kT][kCh / 32][2 * kN];   // dB, dC of each warp
    __shared__ float4 entry[MULTI ? 4 : 1][MULTI ? kCh : 1];  // the states entering the chunk
    __shared__ uint32_t tmem_base;
    const Place at = place(p);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, j = lane & 3;
    const int l2 = (tid & 63) * 2, k0 = (tid >> 6) * kHalf, c2 = at.block * kCh + l2;
    const int l4 = warp * 32 + (lane >> 2) * 4, c4 = at.block * kCh + l4, n4 = j * 4;
    const int t_first = at.chunk * p.chunk, t_end = min(p.L, t_first + p.chunk);
    const int64_t chunk = (int64_t)at.b * p.chunks + at.chunk;
    if (warp == 0) {
        tmem_alloc(&tmem_base, COLUMNS);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base + ((uint32_t)(warp * 32) << 16);
    float2 bias = make2(0.f);
    if (p.dt_bias && c2 < p.dim) bias = make_float2(p.dt_bias[c2], c2 + 1 < p.dim ? p.dt_bias[c2 + 1] : 0.f);
    float2 A2[4][2], K2[4][2], g[4][2], dA[4][2];
    load_A(p, c4, n4, A2, K2);
    if (MULTI)
        load_states(p.G + chunk * p.per, p.dim, c4, n4, g);
    else
        load_given(p, p.dfinal, at.b, c4, n4, g);
    float2 Dk[2];  // the skip's weights, in one lane of each quad
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = c4 + 2 * i;
        Dk[i] = make_float2(j == 0 && p.D && c < p.dim ? p.D[c] : 0.f, j == 0 && p.D && c + 1 < p.dim ? p.D[c + 1] : 0.f);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) dA[s][0] = dA[s][1] = make2(0.f);
    float2 dD = make2(0.f), dbias = make2(0.f);  // of this thread's tokens and channels
    RawRows<Tx, Td, Tb> raw;
    const int t_last = t_first + (t_end - 1 - t_first) / kT * kT;
    raw.load(p, at.b, t_last, t_end, c2, true);
    float2 h[4][2];
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto load_check = [&](int t) {
        const int64_t sub = (int64_t)at.b * p.subs + t / kT;
        load_states(p.ck + sub * p.per, p.dim, c4, n4, h);
        if (MULTI && at.chunk > 0 && c4 < p.dim) {
            sum = *reinterpret_cast<const float4 *>(p.ck_dt + sub * p.dim4 + c4);
        }
    };
    load_check(t_last);
    if (MULTI) {
        float2 in[4][2];
        load_states(p.H + chunk * p.per, p.dim, c4, n4, in);
#pragma unroll
        for (int s = 0; s < 4; ++s) entry[s][tid] = make_float4(in[s][0].x, in[s][0].y, in[s][1].x, in[s][1].y);
    }
    for (int t0 = t_last; t0 >= t_first; t0 -= kT) {
#pragma unroll
        for (int k = 0; k < kHalf; ++k) {
            const bool live = t0 + k0 + k < t_end;
            const float2 x = raw.x[k].f32(), dy = raw.dy[k].f32(), d = raw.delta[k].f32();
            const float2 pre = fadd2(d, bias);
            float2 dt = make2(0.f), q = dy, f = make2(0.f);
            if (live && c2 < p.dim) dt.x = softplus_of<PRECISE>(pre.x);
            if (live && c2 + 1 < p.dim) dt.y = softplus_of<PRECISE>(pre.y);
            if (p.z) {
                const float2 z = raw.z[k].f32();
                float2 gate, slope;
                silu_grad<PRECISE>(z.x, gate.x, slope.x);
                silu_grad<PRECISE>(z.y, gate.y, slope.y);
                q = fmul2(dy, gate);
                f = fmul2(dy, slope);
            }
            *reinterpret_cast<float2 *>(&xs[k0 + k][l2]) = x;
            *reinterpret_cast<float2 *>(&dts[k0 + k][l2]) = dt;
            *reinterpret_cast<float2 *>(&qs[k0 + k][l2]) = q;
            *reinterpret_cast<float2 *>(&fz[k0 + k][l2]) = f;
            *reinterpret_cast<float2 *>(&fd[k0 + k][l2]) =
                make_float2(sigmoid_of<PRECISE>(pre.x), sigmoid_of<PRECISE>(pre.y));
            dD = ffma2(q, x, dD);
        }
        raw.stage_bc(bc4);
        __syncthreads();
        if (MULTI && at.chunk > 0) {
            // the checkpoint holds the states from zero at the chunk's start
            const float2 sum2[2] = {lo2(sum), hi2(sum)};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float4 in = entry[s][tid];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 v = fmul2(A2[s][i], sum2[i]);
                    const float2 f = PRECISE ? make_float2(exp2f(v.x), exp2f(v.y))
                                             : make_float2(ex2_approx(v.x), ex2_approx(v.y));
                    h[s][i] = ffma2(f, i ? hi2(in) : lo2(in), h[s][i]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            tmem_put(tmem + k * SLOT, h);
            if (!KEEP_E && k + 1 == kT) break;  // FP16 tensors: h becomes the state behind the last token
            float2 ee[4][2];
            const float4 x4 = *reinterpret_cast<const float4 *>(&xs[k][l4]);
            const float4 d4 = *reinterpret_cast<const float4 *>(&dts[k][l4]);
            const float2 x2[2] = {lo2(x4), hi2(x4)}, d2[2] = {lo2(d4), hi2(d4)};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float2 B2 = *reinterpret_cast<const float2 *>(&bc4[k][s * 4 + j]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float2 e, a;
                    const float2 v = fmul2(d2[i], A2[s][i]);
                    exp2m1_2<PRECISE>(v, e, a);
                    if (KEEP_E) ee[s][i] = e;
                    h[s][i] = step_2<PRECISE>(v, e, a, fmul2(x2[i], B2), K2[s][i], h[s][i]);
                }
            }
            if (KEEP_E) tmem_put(tmem + k * SLOT + kN, ee);
        }
        tmem_wait_st();
#pragma unroll 1
        for (int k = kT - 1; k >= 0; --k) {
            const float4 x4 = *reinterpret_cast<const float4 *>(&xs[k][l4]);
            const float4 d4 = *reinterpret_cast<const float4 *>(&dts[k][l4]);
            const float4 q4 = *reinterpret_cast<const float4 *>(&qs[k][l4]);
            const float2 x2[2] = {lo2(x4), hi2(x4)}, d2[2] = {lo2(d4), hi2(d4)}, q2[2] = {lo2(q4), hi2(q4)};
            if (KEEP_E && k + 1 < kT) tmem_get(tmem + (k + 1) * SLOT, h);  // the state behind the token
            float2 y[2], dx[2], dd[2], dt_ln2[2];
            float v8[8];  // dB of the 4 states, dC of them: sums over the 4 channels
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                y[i] = fmul2(Dk[i], x2[i]);
                dx[i] = fmul2(Dk[i], q2[i]);
                dd[i] = make2(0.f);
                dt_ln2[i] = fmul2(d2[i], make2(kLn2));
            }
            auto use_state = [&](int s, int i, float2 C2, float2 ht, float2 &dC) {
                y[i] = ffma2(C2, ht, y[i]);
                dC = i ? ffma2(q2[i], ht, dC) : fmul2(q2[i], ht);
                g[s][i] = ffma2(C2, q2[i], g[s][i]);
            };
            if (KEEP_E) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const float2 C2 = reinterpret_cast<const float2 *>(&bc4[k][s * 4 + j])[1];
                    float2 dC;
#pragma unroll
                    for (int i = 0; i < 2; ++i) use_state(s, i, C2, h[s][i], dC);
                    v8[4 + s] = dC.x + dC.y;
                }
            }
            float2 hp[4][2], ee[4][2];
            if (KEEP_E)
                tmem_get(tmem + k * SLOT, hp, ee);
            else
                tmem_get(tmem + k * SLOT, hp);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float4 bc = bc4[k][s * 4 + j];
                const float2 B2 = lo2(bc);
                float2 dB, dC;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 v = fmul2(d2[i], A2[s][i]);
                    float2 e, a;
                    if (KEEP_E)
                        e = ee[s][i];
                    else
                        exp2m1_2<PRECISE>(v, e, a);
                    const float2 w = fmul2(x2[i], B2);
                    if (!KEEP_E) use_state(s, i, hi2(bc), step_2<PRECISE>(v, e, a, w, K2[s][i], hp[s][i]), dC);
                    const float2 gt = g[s][i];
                    const float2 hw = ffma2(w, K2[s][i], hp[s][i]);  // h_{t-1} + B x / A
                    const float2 ga = decay_2<PRECISE>(v, e, a, gt);
                    const float2 phi = phi_2<PRECISE>(v, e, K2[s][i]), gphi = fmul2(gt, phi);
                    g[s][i] = ga;
                    dB = i ? ffma2(gphi, x2[i], dB) : fmul2(gphi, x2[i]);
                    dx[i] = ffma2(gphi, B2, dx[i]);
                    const float2 r = fmul2(ga, A2[s][i]);
                    dd[i] = ffma2(r, hw, dd[i]);
                    const float2 bend = bend_2<PRECISE>(v, e, phi, dt_ln2[i], gt, ga, gphi);
                    dA[s][i] = ffma2(fmul2(r, dt_ln2[i]), hp[s][i], dA[s][i]);
                    dA[s][i] = ffma2(w, bend, dA[s][i]);
                }
                v8[s] = dB.x + dB.y;
                if (!KEEP_E) v8[4 + s] = dC.x + dC.y;
            }
            const float ys = quad_sum(y, j), dxs = quad_sum(dx, j), dds = quad_sum(dd, j);
            const float r = oct_sum(v8, lane);
            const int m = lane >> 2;  // dB of state n4 + m, or dC of n4 + m - 4
            __syncwarp();             // the quad has read this token's rows
            qs[k][l4 + j] = ys;
            xs[k][l4 + j] = dxs;
            dts[k][l4 + j] = dds * kLn2;
            red[k][warp][(m & 4) * 4 + n4 + (m & 3)] = m & 4 ? r : r * kLog2e;
        }
        if (t0 > t_first) {
            raw.load(p, at.b, t0 - kT, t_end, c2, true);
            load_check(t0 - kT);
        }
        __syncthreads();
        if (c2 < p.dim) {
            const bool second = c2 + 1 < p.dim;
#pragma unroll
            for (int k = 0; k < kHalf; ++k) {
                const int64_t t = t0 + k0 + k;
                if (t < t_end) {
                    auto pair = [&](const float (&v)[kT][kCh]) { return *reinterpret_cast<const float2 *>(&v[k0 + k][l2]); };
                    const float2 u = fmul2(pair(dts), pair(fd));
                    store_pair(static_cast<Tx *>(p.dx) + at.b * p.sdx[0] + t * p.sdx[1] + c2 * p.sdx[2], p.sdx[2],
                               p.pairs, second, pair(xs));
                    store_pair(static_cast<Td *>(p.ddelta) + at.b * p.sddelta[0] + t * p.sddelta[1] + c2 * p.sddelta[2],
                               p.sddelta[2], p.pairs, second, u);
                    if (p.z)
                        store_pair(static_cast<Tx *>(p.dz) + at.b * p.sdz[0] + t * p.sdz[1] + c2 * p.sdz[2], p.sdz[2],
                                   p.pairs, second, fmul2(pair(qs), pair(fz)));
                    dbias = fadd2(dbias, u);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = tid + k * kCh, t = i >> 5;
            if (t0 + t < t_end) {
                float s = 0.f;
#pragma unroll
                for (int v = 0; v < kCh / 32; ++v) s += red[t][v][i & 31];
                p.part_bc[(((int64_t)at.block * p.batch + at.b) * p.L + t0 + t) * (2 * kN) + (i & 31)] = s;
            }
        }
        __syncthreads();
    }
    float *part = p.part_a + chunk * sums_of(p.dim);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) dA[s][i] = fmul2(fmul2(dA[s][i], K2[s][i]), make2(kLog2e));
    store_states(part, p.dim, c4, n4, dA);
    // the two halves' sums of dD and ddt_bias
    *reinterpret_cast<float2 *>(&xs[tid >> 6][l2]) = dD;
    *reinterpret_cast<float2 *>(&dts[tid >> 6][l2]) = dbias;
    __syncthreads();
    if (at.block * kCh + tid < p.dim) {
        part += states_of(p.dim) + at.block * kCh + tid;
        part[0] = xs[0][tid] + xs[1][tid];
        part[p.dim] = dts[0][tid] + dts[1][tid];
    }
    if (at.chunk == 0 && p.dh0) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c4 + i < p.dim && n4 + s < p.N)
                    p.dh0[((int64_t)at.b * p.dim + c4 + i) * p.N + n4 + s] = i & 1 ? g[s][i / 2].y : g[s][i / 2].x;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem_base, COLUMNS);
}

struct ScanSumParams {
    const float *part_bc, *part_a;
    void *dB, *dC;
    float *dA, *dD, *ddt_bias;
    int64_t sdB[3], sdC[3], rows;  // rows = batch * L
    int blocks, parts, dim, N, L;
    unsigned bc_ctas;
};
// The partial rows' sums in order: the first bc_ctas CTAs add dB and dC over
// the channel blocks, the others dA, dD and ddt_bias over chunks and batch (warp
// v takes parts v, v + 8, ..., then the warps' sums are added).
template <typename Tb>
__global__ void __launch_bounds__(256) scan_bwd_sum_kernel(const ScanSumParams p) {
    __shared__ float sm[8][32];
    if (blockIdx.x < p.bc_ctas) {
        const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
        const int64_t row = i >> 5;
        const int m = (int)(i & 31), n = m & 15;
        if (row >= p.rows || n >= p.N) return;
        float s = 0.f;
#pragma unroll 4
        for (int k = 0; k < p.blocks; ++k) s += p.part_bc[(k * p.rows + row) * 32 + m];
        const int64_t b = row / p.L, t = row - b * p.L;
        if (m & 16) {
            if (p.dC) static_cast<Tb *>(p.dC)[b * p.sdC[0] + t * p.sdC[1] + n * p.sdC[2]] = cvt_out<Tb>(s);
        } else {
            if (p.dB) static_cast<Tb *>(p.dB)[b * p.sdB[0] + t * p.sdB[1] + n * p.sdB[2]] = cvt_out<Tb>(s);
        }
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t states = states_of(p.dim), cols = states + 2 * (int64_t)p.dim, row = sums_of(p.dim);
    const int64_t col = (int64_t)(blockIdx.x - p.bc_ctas) * 32 + lane;
    float s = 0.f;
    if (col < cols) {
#pragma unroll 8
        for (int k = warp; k < p.parts; k += 8) s += p.part_a[k * row + col];
    }
    sm[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || col >= cols) return;
#pragma unroll
    for (int v = 1; v < 8; ++v) s += sm[v][lane];
    if (col < states) {
        const int64_t d = col / (4 * kN) * 4 + (col & 3);
        const int n = (int)(col % (4 * kN)) / 4;
        if (d < p.dim && n < p.N && p.dA) p.dA[d * p.N + n] = s;
    } else if (col < states + p.dim) {
        if (p.dD) p.dD[col - states] = s;
    } else if (p.ddt_bias) {
        p.ddt_bias[col - states - p.dim] = s;
    }
}

// Tokens per chunk.  Passes 1 and 3 run 4 and 2 CTAs an SM, each as long as its
// chunk and some tokens' worth of work around it, and pass 1 costs about 0.4 of
// pass 3; several chunks add a tenth, and each a little to pass 2.  Taken: the
// number of chunks for which the rounds of CTAs are shortest (of 8 x 2048 x 4096
// and 3 x 333 x 203, 9 and 42 chunks: 3.13 ms and 55 us; 5 and 11 took 3.33 and
// 90).  At most 16384 tokens, about 21 ms with two CTAs an SM (FP16; chunks of 8192
// tokens take 10.4): a CTA keeps a half (FP32 a quarter) of its SM's tensor
// memory as long.
int chunk_length(int64_t batch, int64_t L, int64_t dim) {
    const int64_t ctas = batch * ceil_div64(dim, kCh), slots = 148 * 2, least_n = ceil_div64(L, 16384);
    int64_t best = 0;
    double least = 0;
    for (int64_t n = least_n; n <= least_n + 127 && n <= ceil_div64(L, kT); ++n) {
        const int64_t chunk = ceil_div64(ceil_div64(L, n), kT) * kT, all = ctas * ceil_div64(L, chunk);
        double cost = (ceil_div64(all, slots) + 0.8 * ceil_div64(all, 2 * slots)) * (double)(chunk + 8);
        if (chunk < L) cost = cost * 1.1 + 0.3 * n;
        if (best == 0 || cost < least) {
            best = chunk;
            least = cost;
        }
    }
    return (int)best;
}

size_t up(size_t v) { return (v + 255) / 256 * 256; }
struct Layout {
    size_t ck, ck_dt, H, G, S, bc, a, bytes;
    int chunk, chunks, subs, blocks;
};
Layout layout(const MambaScanArgs *a) {
    Layout l{};
    const size_t b = (size_t)a->batch, dim = (size_t)a->dim, L = (size_t)a->seqlen;
    l.chunk = chunk_length(a->batch, a->seqlen, a->dim);
    l.chunks = (int)ceil_div64(a->seqlen, l.chunk);
    l.subs = (int)ceil_div64(a->seqlen, kT);
    l.blocks = ceil_div(a->dim, kCh);
    size_t at = 0;
    auto take = [&](size_t floats) {
        const size_t v = at;
        at += up(floats * 4);
        return v;
    };
    const bool multi = l.chunks > 1;
    const size_t per = (size_t)states_of(a->dim);
    l.ck = take(b * l.subs * per);
    l.ck_dt = take(multi ? b * l.subs * ((dim + 3) / 4 * 4) : 0);
    l.H = take(multi ? b * l.chunks * per : 0);
    l.G = take(multi ? b * l.chunks * per : 0);
    l.S = take(multi ? b * l.chunks * dim : 0);
    l.bc = take(l.blocks * b * L * 2 * kN);
    l.a = take(b * l.chunks * (size_t)sums_of(a->dim));
    l.bytes = at;
    return l;
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename Tx, typename Td, typename Tb, bool MULTI>
int launch_passes(const ScanGradParams &p, cudaStream_t st) {
    const unsigned grid = (unsigned)(p.blocks * p.chunks * p.batch);
    scan_bwd_states_kernel<Tx, Td, Tb, MULTI><<<grid, kCh, 0, st>>>(p);
    if (launch_status("selective_scan_backward states kernel")) return -1;
    if (MULTI) {
        const int64_t n = (int64_t)p.batch * p.per;
        scan_bwd_carry_kernel<<<(unsigned)ceil_div64(n, 256), 256, 0, st>>>(p);
        if (launch_status("selective_scan_backward carry kernel")) return -1;
    }
    scan_bwd_kernel<Tx, Td, Tb, MULTI><<<grid, kCh, 0, st>>>(p);
    return launch_status("selective_scan_backward kernel");
}
template <typename Tx, typename Td, typename Tb>
int launch_all(const ScanGradParams &p, ScanSumParams &s, cudaStream_t st) {
    if (p.chunks > 1 ? launch_passes<Tx, Td, Tb, true>(p, st) : launch_passes<Tx, Td, Tb, false>(p, st)) return -1;
    s.bc_ctas = (unsigned)ceil_div64(s.rows * 32, 256);
    const int64_t grid = (int64_t)s.bc_ctas + ceil_div64(p.per + 2 * (int64_t)p.dim, 32);
    scan_bwd_sum_kernel<Tb><<<(unsigned)grid, 256, 0, st>>>(s);
    return launch_status("selective_scan_backward sum kernel");
}

int check(const MambaScanArgs *a) {
    const char *what = "selective_scan_backward";
    MB_CHECK_ARG(a, std::string(what) + ": null args");
    MB_CHECK_ARG(a->batch >= 0 && a->seqlen >= 0 && a->dim >= 0, std::string(what) + ": negative size");
    MB_CHECK_ARG(a->dstate >= 1 && a->dstate <= 16, std::string(what) + ": dstate must be in 1..16");
    const bool f32 = a->x_dtype == MAMBA_F32 && a->delta_dtype == MAMBA_F32 && a->bc_dtype == MAMBA_F32;
    const bool f16 = a->x_dtype == MAMBA_F16 && (a->delta_dtype == MAMBA_F16 || a->delta_dtype == MAMBA_F32) &&
                     (a->bc_dtype == MAMBA_F16 || (a->bc_dtype == MAMBA_F32 && a->delta_dtype == MAMBA_F32));
    MB_CHECK_ARG(f32 || f16, std::string(what) + ": unsupported combination of dtypes");
    const int64_t elems = (int64_t)a->batch * std::max(a->seqlen, 1);
    MB_CHECK_ARG(elems <= ((int64_t)1 << 31) / std::max(ceil_div(a->dim, kCh), 1) && a->seqlen <= 0x7fffffff - 256,
                 std::string(what) + ": too many elements");
    return 0;
}

}  // namespace

size_t selective_scan_backward_workspace_bytes(const MambaScanArgs *a) {
    if (!a || a->batch <= 0 || a->seqlen <= 0 || a->dim <= 0 || a->dstate < 1 || a->dstate > 16) return 0;
    return layout(a).bytes;
}

int selective_scan_backward(const MambaScanArgs *a, const MambaScanGrads *g, void *ws, size_t ws_bytes,
                            cudaStream_t st) {
    if (check(a)) return -1;
    MB_CHECK_ARG(g, "selective_scan_backward: null gradients");
    const size_t ex = dtype_size(a->x_dtype), ed = dtype_size(a->delta_dtype), eb = dtype_size(a->bc_dtype);
    MB_CHECK_ARG(aligned(g->dA, 4) && aligned(g->dD, 4) && aligned(g->ddt_bias, 4) && aligned(g->dinitial_state, 4) &&
                     aligned(g->dfinal_state, 4),
                 "selective_scan_backward: pointers must be aligned to their element type");
    if (a->batch == 0 || a->seqlen == 0 || a->dim == 0) {
        // no token: the sums are zero, and the initial state's gradient is the final state's
        const size_t dim = (size_t)a->dim, states = (size_t)a->batch * dim * a->dstate;
        if (dim && g->dA) MB_CUDA_TRY(cudaMemsetAsync(g->dA, 0, dim * a->dstate * 4, st));
        if (dim && g->dD) MB_CUDA_TRY(cudaMemsetAsync(g->dD, 0, dim * 4, st));
        if (dim && g->ddt_bias) MB_CUDA_TRY(cudaMemsetAsync(g->ddt_bias, 0, dim * 4, st));
        if (states && g->dinitial_state && g->dinitial_state != g->dfinal_state) {
            if (g->dfinal_state)
                MB_CUDA_TRY(cudaMemcpyAsync(g->dinitial_state, g->dfinal_state, states * 4, cudaMemcpyDeviceToDevice, st));
            else
                MB_CUDA_TRY(cudaMemsetAsync(g->dinitial_state, 0, states * 4, st));
        }
        if (a->dim == 0 && a->batch && a->seqlen) {
            MB_CHECK_ARG(!g->dB && !g->dC, "selective_scan_backward: no channels to sum dB and dC over");
        }
        return 0;
    }
    MB_CHECK_ARG(a->x && a->delta && a->A && a->B && a->C && g->dy && g->dx && g->ddelta,
                 "selective_scan_backward: null pointer");
    MB_CHECK_ARG(!a->z || g->dz, "selective_scan_backward: a gate needs dz");
    MB_CHECK_ARG(aligned(a->x, ex) && aligned(a->z, ex) && aligned(g->dy, ex) && aligned(g->dx, ex) &&
                     aligned(g->dz, ex) && aligned(a->delta, ed) && aligned(g->ddelta, ed) && aligned(a->B, eb) &&
                     aligned(a->C, eb) && aligned(g->dB, eb) && aligned(g->dC, eb) && aligned(a->A, 4) &&
                     aligned(a->D, 4) && aligned(a->dt_bias, 4) && aligned(a->initial_state, 4),
                 "selective_scan_backward: pointers must be aligned to their element type");
    const void *in[] = {a->x, a->delta, a->z, a->B, a->C, g->dy, a->A, a->D, a->dt_bias, a->initial_state,
                        g->dfinal_state};
    const void *out[] = {g->dx, g->ddelta, a->z ? g->dz : nullptr, g->dB, g->dC, g->dA, g->dD, g->ddt_bias,
                         g->dinitial_state};
    for (size_t i = 0; i < sizeof(out) / sizeof(out[0]); ++i) {
        if (!out[i]) continue;
        for (const void *p : in)
            MB_CHECK_ARG(out[i] != p, "selective_scan_backward: a gradient may not be one of the inputs");
        for (size_t k = 0; k < i; ++k)
            MB_CHECK_ARG(out[i] != out[k], "selective_scan_backward: the gradients need memory of their own");
    }
    MB_CHECK_ARG(ws && ws_bytes >= selective_scan_backward_workspace_bytes(a) && aligned(ws, 16),
                 "selective_scan_backward: workspace too small or not 16-byte aligned");
    // an output's elements lie apart
    auto apart = [&](const void *p, const int64_t *st3, int inner) {
        return !p || ((a->batch == 1 || st3[0] != 0) && (a->seqlen == 1 || st3[1] != 0) && (inner == 1 || st3[2] != 0));
    };
    MB_CHECK_ARG(apart(g->dx, g->dx_stride, a->dim) && apart(g->ddelta, g->ddelta_stride, a->dim) &&
                     (!a->z || apart(g->dz, g->dz_stride, a->dim)) && apart(g->dB, g->dB_stride, a->dstate) &&
                     apart(g->dC, g->dC_stride, a->dstate),
                 "selective_scan_backward: a gradient's elements overlap (strides)");
    const Layout l = layout(a);
    uint8_t *base = static_cast<uint8_t *>(ws);
    auto at = [&](size_t o) { return reinterpret_cast<float *>(base + o); };
    ScanGradParams p{};
    p.x = a->x;
    p.delta = a->delta;
    p.dy = g->dy;
    p.z = a->z;
    p.B = a->B;
    p.C = a->C;
    p.A = a->A;
    p.D = a->D;
    p.dt_bias = a->dt_bias;
    p.h0 = a->initial_state;
    p.dfinal = g->dfinal_state;
    p.dx = g->dx;
    p.ddelta = g->ddelta;
    p.dz = g->dz;
    p.dh0 = g->dinitial_state;
    p.ck = at(l.ck);
    p.ck_dt = at(l.ck_dt);
    p.H = at(l.H);
    p.G = at(l.G);
    p.S = at(l.S);
    p.part_bc = at(l.bc);
    p.part_a = at(l.a);
    p.batch = a->batch;
    p.L = a->seqlen;
    p.dim = a->dim;
    p.N = a->dstate;
    p.chunk = l.chunk;
    p.chunks = l.chunks;
    p.subs = l.subs;
    p.blocks = l.blocks;
    p.per = states_of(p.dim);
    p.dim4 = (p.dim + 3) / 4 * 4;
    ScanSumParams s{};
    for (int k = 0; k < 3; ++k) {
        p.sx[k] = a->x_stride[k];
        p.sdelta[k] = a->delta_stride[k];
        p.sdy[k] = g->dy_stride[k];
        p.sz[k] = a->z_stride[k];
        p.sB[k] = a->B_stride[k];
        p.sC[k] = a->C_stride[k];
        p.sdx[k] = g->dx_stride[k];
        p.sddelta[k] = g->ddelta_stride[k];
        p.sdz[k] = g->dz_stride[k];
        s.sdB[k] = g->dB_stride[k];
        s.sdC[k] = g->dC_stride[k];
    }
    // two channels at a time: adjacent, and every row start aligned for both
    auto even = [&](const void *v, const int64_t *st3, size_t es) {
        return !v || (st3[2] == 1 && st3[1] % 2 == 0 && st3[0] % 2 == 0 && aligned(v, 2 * es));
    };
    p.pairs = p.dim % 2 == 0 && even(p.x, p.sx, ex) && even(p.delta, p.sdelta, ed) && even(p.dy, p.sdy, ex) &&
              even(p.z, p.sz, ex) && even(p.dx, p.sdx, ex) && even(p.ddelta, p.sddelta, ed) &&
              (!p.z || even(p.dz, p.sdz, ex));
    s.part_bc = p.part_bc;
    s.part_a = p.part_a;
    s.dB = g->dB;
    s.dC = g->dC;
    s.dA = g->dA;
    s.dD = g->dD;
    s.ddt_bias = g->ddt_bias;
    s.rows = (int64_t)p.batch * p.L;
    s.blocks = p.blocks;
    s.parts = p.batch * p.chunks;
    s.dim = p.dim;
    s.N = p.N;
    s.L = p.L;
    if (a->x_dtype == MAMBA_F32) return launch_all<float, float, float>(p, s, st);
    if (a->delta_dtype == MAMBA_F16) return launch_all<__half, __half, __half>(p, s, st);
    return a->bc_dtype == MAMBA_F16 ? launch_all<__half, float, __half>(p, s, st)
                                    : launch_all<__half, float, float>(p, s, st);
}

}  // namespace mb
