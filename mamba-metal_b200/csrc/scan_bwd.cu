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
// a - 1 is evaluated without cancellation (e), psi too, and everything is kept
// as e: h_t = h + e (h + w / A), a g = g + e g, phi = e / A.  A state with
// |A| < 1e-20 counts as 1e-20, where these are the limits.
//
// Three passes over time chunks:
//   1. forward: the state before every 8th token (a checkpoint), from zero at
//      the start of each chunk; with several chunks also each chunk's map
//      (its end state H, the reverse carry G and the sum of dt),
//   2. (several chunks) the state entering each chunk and the carry entering
//      it from behind,
//   3. backward, 8 tokens at a time: the states from the checkpoint on into
//      shared memory, then the reverse steps over them.
// A CTA holds 128 channels: a thread has 4 channels x 4 states, so a row's x,
// dt and q are one 16-byte access for 4 channels, and the sums over channels
// (dB, dC) and states (dx, ddelta, y) are half done before the first shuffle.
// dB and dC leave as one partial row per block of 128 channels, dA, dD and
// ddt_bias as one per chunk and batch; a last kernel adds them in order.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "scan_math.cuh"

namespace mb {
namespace {

constexpr int kT = 8;        // tokens between checkpoints
constexpr int kCh = 128;     // channels (and threads) per CTA
constexpr int kN = 16;       // states, padded

struct ScanGradParams {
    const void *x, *delta, *dy, *z, *B, *C;
    const float *A, *D, *dt_bias, *h0, *dfinal;
    void *dx, *ddelta, *dz;
    float *dh0;
    float *ck;    // [batch][subs][dim][16] states before every 8th token
    float *ck_dt; // [batch][subs][dim] sum of dt before it, since the chunk's start
    float *H, *G; // [batch][chunks][dim][16]
    float *S;     // [batch][chunks][dim]
    float *part_bc;  // [blocks][batch * L][32]
    float *part_a;   // [batch * chunks][sums_of(dim)]: dA [dim][16], dD [dim], ddt_bias [dim]
    int batch, L, dim, N, chunk, chunks, subs, blocks;
    int64_t sx[3], sdelta[3], sdy[3], sz[3], sB[3], sC[3], sdx[3], sddelta[3], sdz[3];
};

// Floats of a partial row of dA, dD and ddt_bias, a multiple of 4.
__host__ __device__ __forceinline__ int64_t sums_of(int dim) { return ((int64_t)dim * (kN + 2) + 3) / 4 * 4; }
__device__ __forceinline__ float2 make2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float4 zero4() { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float at4(const float4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// e^(dt A) - 1 for two states.  FP16 tensors (v = dt A log2(e)): one
// approximate exponential less 1, or below 1/32 the series to v^4 (relative
// error below 2e-6 at the border, 6e-8 relative to e^v - 1 = O(1) elsewhere).
constexpr float kNear2 = 0.03125f * 1.4426950408889634f;
template <bool PRECISE>
__device__ __forceinline__ float2 expm1_2(float dt, float dt2, float2 A) {
    if (PRECISE) return make_float2(expm1f(dt * A.x), expm1f(dt * A.y));
    constexpr float c1 = 0.69314718055994531f, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
    const float2 v = __fmul2_rn(make2(dt2), A);
    float2 far = make_float2(ex2_approx(v.x), ex2_approx(v.y));
    far = __fadd2_rn(far, make2(-1.f));
    float2 s = __ffma2_rn(v, make2(c4), make2(c3));
    s = __ffma2_rn(s, v, make2(c2));
    s = __ffma2_rn(s, v, make2(c1));
    s = __fmul2_rn(s, v);
    return make_float2(fabsf(v.x) < kNear2 ? s.x : far.x, fabsf(v.y) < kNear2 ? s.y : far.y);
}

// psi = (dt a - phi) / A.  Where |dt A| is small, dt^2 (1/2 + v/3 + v^2/8 + ...).
template <bool PRECISE>
__device__ __forceinline__ float psi_1(float dt, float e, float phi, float A, float kI) {
    const float v = dt * A;
    const float far = (fmaf(dt, e, dt) - phi) * kI;
    float s;
    if (PRECISE) {
        s = fmaf(v, 1.f / 840, 1.f / 144);
        s = fmaf(s, v, 1.f / 30);
        s = fmaf(s, v, 1.f / 8);
    } else {
        s = fmaf(v, 1.f / 30, 1.f / 8);
    }
    s = fmaf(s, v, 1.f / 3);
    s = fmaf(s, v, 0.5f);
    s *= dt * dt;
    return fabsf(v) < (PRECISE ? 0.25f : 0.0625f) ? s : far;
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

// One thread's inputs of 8 tokens: channel `tid` of the block's rows, and two
// of the 8 x 32 values of B and C.
template <typename Tx, typename Td, typename Tb>
struct RawRows {
    Tx x[kT], dy[kT], z[kT];
    Td delta[kT];
    Tb bc[2];
    // Tokens behind `end` and channels behind the last are left unread: stage() skips them too.
    __device__ __forceinline__ void load(const ScanGradParams &p, int b, int t0, int end, int c, bool grads) {
        if (c < p.dim) {
            const Tx *px = static_cast<const Tx *>(p.x) + b * p.sx[0] + c * p.sx[2];
            const Td *pd = static_cast<const Td *>(p.delta) + b * p.sdelta[0] + c * p.sdelta[2];
            const Tx *pg = static_cast<const Tx *>(p.dy) + b * p.sdy[0] + c * p.sdy[2];
            const Tx *pz = static_cast<const Tx *>(p.z) + b * p.sz[0] + c * p.sz[2];
#pragma unroll
            for (int k = 0; k < kT; ++k) {
                const int64_t t = t0 + k;
                if (t < end) {
                    x[k] = px[t * p.sx[1]];
                    delta[k] = pd[t * p.sdelta[1]];
                    if (grads) {
                        dy[k] = pg[t * p.sdy[1]];
                        if (p.z) z[k] = pz[t * p.sz[1]];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = threadIdx.x + k * kCh, n = at & 15;
            const int64_t t = t0 + (at >> 5);
            if (t < end && n < p.N)
                bc[k] = at & 16 ? static_cast<const Tb *>(p.C)[b * p.sC[0] + t * p.sC[1] + n * p.sC[2]]
                                : static_cast<const Tb *>(p.B)[b * p.sB[0] + t * p.sB[1] + n * p.sB[2]];
        }
    }
};

// A, 1/A of a thread's 4 channels x 4 states.
__device__ __forceinline__ void load_A(const ScanGradParams &p, int c4, int n4, float2 (&A)[4][2], float2 (&kI)[4][2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int n = n4 + 2 * k + e;
                v[e] = c4 + i < p.dim && n < p.N ? p.A[(int64_t)(c4 + i) * p.N + n] : 0.f;
                if (fabsf(v[e]) < 1e-20f) v[e] = 1e-20f;
            }
            A[i][k] = make_float2(v[0], v[1]);
            kI[i][k] = make_float2(__frcp_rn(v[0]), __frcp_rn(v[1]));
        }
}

// Four states of each of a thread's channels, from [dim][16] rows or [dim][N] ones.
__device__ __forceinline__ void load_states(const float *rows, int dim, int N, int c4, int n4, float2 (&v)[4][2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 q = zero4();
        if (rows && c4 + i < dim) {
            const float *r = rows + (int64_t)(c4 + i) * N;
            if (N == kN) {
                q = *reinterpret_cast<const float4 *>(r + n4);
            } else {
                q.x = n4 + 0 < N ? r[n4 + 0] : 0.f;
                q.y = n4 + 1 < N ? r[n4 + 1] : 0.f;
                q.z = n4 + 2 < N ? r[n4 + 2] : 0.f;
                q.w = n4 + 3 < N ? r[n4 + 3] : 0.f;
            }
        }
        v[i][0] = make_float2(q.x, q.y);
        v[i][1] = make_float2(q.z, q.w);
    }
}
__device__ __forceinline__ void store_states(float *rows, int dim, int c4, int n4, const float2 (&v)[4][2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c4 + i < dim)
            *reinterpret_cast<float4 *>(rows + (int64_t)(c4 + i) * kN + n4) =
                make_float4(v[i][0].x, v[i][0].y, v[i][1].x, v[i][1].y);
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

// Pass 1.
template <typename Tx, typename Td, typename Tb, bool MULTI>
__global__ void __launch_bounds__(kCh) scan_bwd_states_kernel(const ScanGradParams p) {
    constexpr bool PRECISE = sizeof(Tx) == 4;
    __shared__ __align__(16) float xs[2][kT][kCh], dts[2][kT][kCh], qs[MULTI ? 2 : 1][kT][MULTI ? kCh : 4];
    __shared__ __align__(16) float bcs[2][kT][2 * kN];
    const Place at = place(p);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c = at.block * kCh + tid;  // the channel this thread stages
    const int l4 = warp * 32 + (lane >> 2) * 4, c4 = at.block * kCh + l4, n4 = (lane & 3) * 4;
    const int t_first = at.chunk * p.chunk, t_end = min(p.L, t_first + p.chunk);
    const float bias = p.dt_bias && c < p.dim ? p.dt_bias[c] : 0.f;
    float2 A[4][2], kI[4][2], h[4][2], P[4][2], G[4][2];
    load_A(p, c4, n4, A, kI);
    load_states(at.chunk == 0 && p.h0 ? p.h0 + (int64_t)at.b * p.dim * p.N : nullptr, p.dim, p.N, c4, n4, h);
    if (MULTI) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                P[i][k] = make2(1.f);
                G[i][k] = make2(0.f);
            }
    }
    float sum_dt = 0.f;
    RawRows<Tx, Td, Tb> raw;
    raw.load(p, at.b, t_first, t_end, c, MULTI);
    int buf = 0;
    for (int t0 = t_first; t0 < t_end; t0 += kT, buf ^= 1) {
        const int64_t sub = (int64_t)at.b * p.subs + t0 / kT;
        if (MULTI && c < p.dim) p.ck_dt[sub * p.dim + c] = sum_dt;
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const bool live = t0 + k < t_end && c < p.dim;
            const float dt = live ? softplus_of<PRECISE>(cvt_f32<Td>(raw.delta[k]) + bias) : 0.f;
            xs[buf][k][tid] = live ? cvt_f32<Tx>(raw.x[k]) : 0.f;
            dts[buf][k][tid] = dt;
            sum_dt += dt;
            if (MULTI) {
                float q = live ? cvt_f32<Tx>(raw.dy[k]) : 0.f;
                if (live && p.z) {
                    float gate, slope;
                    silu_grad<PRECISE>(cvt_f32<Tx>(raw.z[k]), gate, slope);
                    q *= gate;
                }
                qs[buf][k][tid] = q;
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = tid + k * kCh;
            (&bcs[buf][0][0])[i] = t0 + (i >> 5) < t_end && (i & 15) < p.N ? cvt_f32<Tb>(raw.bc[k]) : 0.f;
        }
        __syncthreads();  // the other buffer's readers are behind this barrier's predecessor
        if (t0 + kT < t_end) raw.load(p, at.b, t0 + kT, t_end, c, MULTI);
        store_states(p.ck + sub * p.dim * kN, p.dim, c4, n4, h);
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const float4 x4 = *reinterpret_cast<const float4 *>(&xs[buf][k][l4]);
            const float4 d4 = *reinterpret_cast<const float4 *>(&dts[buf][k][l4]);
            const float4 B4 = *reinterpret_cast<const float4 *>(&bcs[buf][k][n4]);
            float4 q4 = zero4(), C4 = zero4();
            if (MULTI) {
                q4 = *reinterpret_cast<const float4 *>(&qs[buf][k][l4]);
                C4 = *reinterpret_cast<const float4 *>(&bcs[buf][k][kN + n4]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float dt = at4(d4, i), dt2 = dt * kLog2e;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const float2 Bp = s ? make_float2(B4.z, B4.w) : make_float2(B4.x, B4.y);
                    const float2 e = expm1_2<PRECISE>(dt, dt2, A[i][s]);
                    const float2 w = __fmul2_rn(make2(at4(x4, i)), Bp);
                    h[i][s] = __ffma2_rn(e, __ffma2_rn(w, kI[i][s], h[i][s]), h[i][s]);
                    if (MULTI) {
                        const float2 Cp = s ? make_float2(C4.z, C4.w) : make_float2(C4.x, C4.y);
                        P[i][s] = __ffma2_rn(P[i][s], e, P[i][s]);
                        G[i][s] = __ffma2_rn(P[i][s], __fmul2_rn(Cp, make2(at4(q4, i))), G[i][s]);
                    }
                }
            }
        }
    }
    if (MULTI) {
        const int64_t chunk = (int64_t)at.b * p.chunks + at.chunk;
        store_states(p.H + chunk * p.dim * kN, p.dim, c4, n4, h);
        store_states(p.G + chunk * p.dim * kN, p.dim, c4, n4, G);
        if (c < p.dim) p.S[chunk * p.dim + c] = sum_dt;
    }
}

// Pass 2: a thread per (batch, channel, state) walks the chunks, forward for
// the state that enters each (into H; chunk 0's is in its checkpoints already,
// so H there becomes 0), backward for the carry that enters it from behind
// (into G).
__global__ void __launch_bounds__(256) scan_bwd_carry_kernel(const ScanGradParams p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)p.dim * kN;
    if (i >= p.batch * per) return;
    const int64_t b = i / per, at = i - b * per;
    const int d = (int)(at / kN), n = (int)(at % kN);
    float A = n < p.N ? p.A[(int64_t)d * p.N + n] : 0.f;
    if (fabsf(A) < 1e-20f) A = 1e-20f;
    float *H = p.H + b * p.chunks * per + at, *G = p.G + b * p.chunks * per + at;
    const float *S = p.S + b * p.chunks * p.dim + d;
    float h = 0.f;
#pragma unroll 4
    for (int k = 0; k < p.chunks; ++k) {
        const float end = H[k * per], P = expf(A * S[(int64_t)k * p.dim]);
        H[k * per] = h;
        h = k == 0 ? end : fmaf(P, h, end);
    }
    float g = p.dfinal && n < p.N ? p.dfinal[(b * p.dim + d) * p.N + n] : 0.f;
#pragma unroll 4
    for (int k = p.chunks - 1; k >= 0; --k) {
        const float own = G[k * per], P = expf(A * S[(int64_t)k * p.dim]);
        G[k * per] = g;
        g = fmaf(P, g, own);
    }
}

// Sum over the 4 lanes of a quad: lane j is left with v[j]'s.
__device__ __forceinline__ float quad_sum(const float (&v)[4], int j) {
    const bool hi = j & 2, odd = j & 1;
    float a = hi ? v[2] : v[0], b = hi ? v[3] : v[1];
    a += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 2);
    b += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 2);
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

struct BwdSmem {
    float4 states[kT][4][kCh];  // h before each token: [token][channel of the thread][thread]
    float x[kT][kCh];           // x, later dx
    float dt[kT][kCh];          // dt, later the gradient of dt
    float q[kT][kCh];           // q, later sum_n C h + D x
    float fz[kT][kCh];          // dy SiLU'(z)
    float fd[kT][kCh];          // sigmoid(delta + dt_bias)
    float bc[kT][2 * kN];
    float red[kT][kCh / 32][2 * kN];  // dB, dC of each warp
};

// Pass 3.
template <typename Tx, typename Td, typename Tb, bool MULTI>
__global__ void __launch_bounds__(kCh, 2) scan_bwd_kernel(const ScanGradParams p) {
    constexpr bool PRECISE = sizeof(Tx) == 4;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    BwdSmem &sm = *reinterpret_cast<BwdSmem *>(smem_raw);
    const Place at = place(p);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, j = lane & 3;
    const int c = at.block * kCh + tid;
    const int l4 = warp * 32 + (lane >> 2) * 4, c4 = at.block * kCh + l4, n4 = j * 4;
    const int t_first = at.chunk * p.chunk, t_end = min(p.L, t_first + p.chunk);
    const int64_t chunk = (int64_t)at.b * p.chunks + at.chunk;
    const float bias = p.dt_bias && c < p.dim ? p.dt_bias[c] : 0.f;
    float2 A[4][2], kI[4][2], g[4][2], dA[4][2];
    load_A(p, c4, n4, A, kI);
    if (MULTI)
        load_states(p.G + chunk * p.dim * kN, p.dim, kN, c4, n4, g);
    else
        load_states(p.dfinal ? p.dfinal + (int64_t)at.b * p.dim * p.N : nullptr, p.dim, p.N, c4, n4, g);
    float Dk[4];  // the skip's weights, in one lane of each quad
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        Dk[i] = j == 0 && p.D && c4 + i < p.dim ? p.D[c4 + i] : 0.f;
        dA[i][0] = dA[i][1] = make2(0.f);
    }
    float dD = 0.f, dbias = 0.f;
    RawRows<Tx, Td, Tb> raw;
    const int t_last = t_first + (t_end - 1 - t_first) / kT * kT;
    raw.load(p, at.b, t_last, t_end, c, true);
    for (int t0 = t_last; t0 >= t_first; t0 -= kT) {
        const int64_t sub = (int64_t)at.b * p.subs + t0 / kT;
        float2 h[4][2];
        load_states(p.ck + sub * p.dim * kN, p.dim, kN, c4, n4, h);
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const bool live = t0 + k < t_end && c < p.dim;
            const float xv = live ? cvt_f32<Tx>(raw.x[k]) : 0.f, dy = live ? cvt_f32<Tx>(raw.dy[k]) : 0.f;
            const float pre = live ? cvt_f32<Td>(raw.delta[k]) + bias : 0.f;
            float q = dy, fz = 0.f;
            if (p.z) {
                float gate, slope;
                silu_grad<PRECISE>(live ? cvt_f32<Tx>(raw.z[k]) : 0.f, gate, slope);
                q = dy * gate;
                fz = dy * slope;
            }
            sm.x[k][tid] = xv;
            sm.dt[k][tid] = live ? softplus_of<PRECISE>(pre) : 0.f;
            sm.q[k][tid] = q;
            sm.fz[k][tid] = fz;
            sm.fd[k][tid] = sigmoid_of<PRECISE>(pre);
            dD = fmaf(q, xv, dD);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = tid + k * kCh;
            (&sm.bc[0][0])[i] = t0 + (i >> 5) < t_end && (i & 15) < p.N ? cvt_f32<Tb>(raw.bc[k]) : 0.f;
        }
        __syncthreads();
        if (t0 > t_first) raw.load(p, at.b, t0 - kT, t_end, c, true);
        if (MULTI && at.chunk > 0) {
            // the checkpoint holds the states from zero at the chunk's start
            float2 in[4][2];
            load_states(p.H + chunk * p.dim * kN, p.dim, kN, c4, n4, in);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float s = c4 + i < p.dim ? p.ck_dt[sub * p.dim + c4 + i] : 0.f;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    h[i][k].x = fmaf(expf(A[i][k].x * s), in[i][k].x, h[i][k].x);
                    h[i][k].y = fmaf(expf(A[i][k].y * s), in[i][k].y, h[i][k].y);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const float4 x4 = *reinterpret_cast<const float4 *>(&sm.x[k][l4]);
            const float4 d4 = *reinterpret_cast<const float4 *>(&sm.dt[k][l4]);
            const float4 B4 = *reinterpret_cast<const float4 *>(&sm.bc[k][n4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sm.states[k][i][tid] = make_float4(h[i][0].x, h[i][0].y, h[i][1].x, h[i][1].y);
                if (k + 1 < kT) {
                    const float dt = at4(d4, i), dt2 = dt * kLog2e;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const float2 Bp = s ? make_float2(B4.z, B4.w) : make_float2(B4.x, B4.y);
                        const float2 e = expm1_2<PRECISE>(dt, dt2, A[i][s]);
                        const float2 w = __fmul2_rn(make2(at4(x4, i)), Bp);
                        h[i][s] = __ffma2_rn(e, __ffma2_rn(w, kI[i][s], h[i][s]), h[i][s]);
                    }
                }
            }
        }
#pragma unroll 1
        for (int k = kT - 1; k >= 0; --k) {
            const float4 x4 = *reinterpret_cast<const float4 *>(&sm.x[k][l4]);
            const float4 d4 = *reinterpret_cast<const float4 *>(&sm.dt[k][l4]);
            const float4 q4 = *reinterpret_cast<const float4 *>(&sm.q[k][l4]);
            const float4 B4 = *reinterpret_cast<const float4 *>(&sm.bc[k][n4]);
            const float4 C4 = *reinterpret_cast<const float4 *>(&sm.bc[k][kN + n4]);
            float2 bc[4] = {make2(0.f), make2(0.f), make2(0.f), make2(0.f)};  // dB, dC over the 4 channels
            float y[4], dx[4], dd[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 hv = sm.states[k][i][tid];
                const float dt = at4(d4, i), dt2 = dt * kLog2e, q = at4(q4, i), xv = at4(x4, i);
                float2 y2 = make2(0.f), dx2 = make2(0.f), dd2 = make2(0.f);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const float2 Bp = s ? make_float2(B4.z, B4.w) : make_float2(B4.x, B4.y);
                    const float2 Cp = s ? make_float2(C4.z, C4.w) : make_float2(C4.x, C4.y);
                    const float2 hp = s ? make_float2(hv.z, hv.w) : make_float2(hv.x, hv.y);
                    const float2 e = expm1_2<PRECISE>(dt, dt2, A[i][s]);
                    const float2 w = __fmul2_rn(make2(xv), Bp);
                    const float2 hw = __ffma2_rn(w, kI[i][s], hp);     // h_{t-1} + w / A
                    const float2 ht = __ffma2_rn(e, hw, hp);
                    y2 = __ffma2_rn(Cp, ht, y2);
                    bc[2 + s] = __ffma2_rn(make2(q), ht, bc[2 + s]);
                    const float2 gt = __ffma2_rn(Cp, make2(q), g[i][s]);
                    const float2 phi = __fmul2_rn(e, kI[i][s]);
                    const float2 gphi = __fmul2_rn(gt, phi);
                    bc[s] = __ffma2_rn(gphi, make2(xv), bc[s]);
                    dx2 = __ffma2_rn(gphi, Bp, dx2);
                    const float2 ga = __ffma2_rn(gt, e, gt);
                    g[i][s] = ga;
                    dd2 = __ffma2_rn(__fmul2_rn(ga, hw), A[i][s], dd2);
                    const float2 psi = make_float2(psi_1<PRECISE>(dt, e.x, phi.x, A[i][s].x, kI[i][s].x),
                                                   psi_1<PRECISE>(dt, e.y, phi.y, A[i][s].y, kI[i][s].y));
                    dA[i][s] = __ffma2_rn(__fmul2_rn(ga, make2(dt)), hp, dA[i][s]);
                    dA[i][s] = __ffma2_rn(__fmul2_rn(gt, w), psi, dA[i][s]);
                }
                y[i] = fmaf(Dk[i], xv, y2.x + y2.y);
                dx[i] = fmaf(Dk[i], q, dx2.x + dx2.y);
                dd[i] = dd2.x + dd2.y;
            }
            const float ys = quad_sum(y, j), dxs = quad_sum(dx, j), dds = quad_sum(dd, j);
            const float v[8] = {bc[0].x, bc[0].y, bc[1].x, bc[1].y, bc[2].x, bc[2].y, bc[3].x, bc[3].y};
            const float r = oct_sum(v, lane);
            const int m = lane >> 2;  // dB of state n4 + m, or dC of n4 + m - 4
            __syncwarp();             // the quad has read this token's rows
            sm.q[k][l4 + j] = ys;
            sm.x[k][l4 + j] = dxs;
            sm.dt[k][l4 + j] = dds;
            sm.red[k][warp][(m & 4) * 4 + n4 + (m & 3)] = r;
        }
        __syncthreads();
        if (c < p.dim) {
            Tx *dx = static_cast<Tx *>(p.dx) + at.b * p.sdx[0] + c * p.sdx[2];
            Td *dd = static_cast<Td *>(p.ddelta) + at.b * p.sddelta[0] + c * p.sddelta[2];
            Tx *dz = static_cast<Tx *>(p.dz) + at.b * p.sdz[0] + c * p.sdz[2];
#pragma unroll
            for (int k = 0; k < kT; ++k) {
                const int64_t t = t0 + k;
                if (t < t_end) {
                    const float u = sm.dt[k][tid] * sm.fd[k][tid];
                    dx[t * p.sdx[1]] = cvt_out<Tx>(sm.x[k][tid]);
                    dd[t * p.sddelta[1]] = cvt_out<Td>(u);
                    if (p.z) dz[t * p.sdz[1]] = cvt_out<Tx>(sm.q[k][tid] * sm.fz[k][tid]);
                    dbias += u;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = tid + k * kCh, t = i >> 5;
            if (t0 + t < t_end) {
                float s = 0.f;
#pragma unroll
                for (int v = 0; v < kCh / 32; ++v) s += sm.red[t][v][i & 31];
                p.part_bc[(((int64_t)at.block * p.batch + at.b) * p.L + t0 + t) * (2 * kN) + (i & 31)] = s;
            }
        }
        __syncthreads();
    }
    float *part = p.part_a + chunk * sums_of(p.dim);
    store_states(part, p.dim, c4, n4, dA);
    if (c < p.dim) {
        part[(int64_t)p.dim * 16 + c] = dD;
        part[(int64_t)p.dim * 17 + c] = dbias;
    }
    if (at.chunk == 0 && p.dh0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c4 + i < p.dim) {
                float *to = p.dh0 + ((int64_t)at.b * p.dim + c4 + i) * p.N;
                const float v[4] = {g[i][0].x, g[i][0].y, g[i][1].x, g[i][1].y};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n4 + k < p.N) to[n4 + k] = v[k];
            }
    }
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
    const int64_t cols = (int64_t)p.dim * (kN + 2), row = sums_of(p.dim), col = (int64_t)(blockIdx.x - p.bc_ctas) * 32 + lane;
    float s = 0.f;
    if (col < cols)
        for (int k = warp; k < p.parts; k += 8) s += p.part_a[k * row + col];
    sm[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || col >= cols) return;
#pragma unroll
    for (int v = 1; v < 8; ++v) s += sm[v][lane];
    if (col < (int64_t)p.dim * 16) {
        const int64_t d = col / kN;
        const int n = (int)(col % kN);
        if (n < p.N && p.dA) p.dA[d * p.N + n] = s;
    } else if (col < (int64_t)p.dim * 17) {
        if (p.dD) p.dD[col - (int64_t)p.dim * 16] = s;
    } else if (p.ddt_bias) {
        p.ddt_bias[col - (int64_t)p.dim * 17] = s;
    }
}

// Tokens per chunk: as few chunks as fill the GPU several times over with CTAs
// (two fit an SM), but at least 32 tokens each.
int chunk_length(int64_t batch, int64_t L, int64_t dim) {
    const int64_t blocks = batch * ceil_div64(dim, kCh), want = ceil_div64(8 * 148, std::max<int64_t>(blocks, 1));
    int64_t chunk = ceil_div64(ceil_div64(L, std::max<int64_t>(want, 1)), kT) * kT;
    chunk = std::max<int64_t>(chunk, 32);
    return (int)std::min<int64_t>(chunk, ceil_div64(L, kT) * kT);
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
    l.ck = take(b * l.subs * dim * kN);
    l.ck_dt = take(multi ? b * l.subs * dim : 0);
    l.H = take(multi ? b * l.chunks * dim * kN : 0);
    l.G = take(multi ? b * l.chunks * dim * kN : 0);
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
        const int64_t n = (int64_t)p.batch * p.dim * kN;
        scan_bwd_carry_kernel<<<(unsigned)ceil_div64(n, 256), 256, 0, st>>>(p);
        if (launch_status("selective_scan_backward carry kernel")) return -1;
    }
    auto kernel = scan_bwd_kernel<Tx, Td, Tb, MULTI>;
    MB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(BwdSmem)));
    kernel<<<grid, kCh, sizeof(BwdSmem), st>>>(p);
    return launch_status("selective_scan_backward kernel");
}
template <typename Tx, typename Td, typename Tb>
int launch_all(const ScanGradParams &p, ScanSumParams &s, cudaStream_t st) {
    if (p.chunks > 1 ? launch_passes<Tx, Td, Tb, true>(p, st) : launch_passes<Tx, Td, Tb, false>(p, st)) return -1;
    s.bc_ctas = (unsigned)ceil_div64(s.rows * 32, 256);
    const int64_t grid = (int64_t)s.bc_ctas + ceil_div64((int64_t)p.dim * (kN + 2), 32);
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
                     aligned(a->D, 4) && aligned(a->dt_bias, 4),
                 "selective_scan_backward: pointers must be aligned to their element type");
    MB_CHECK_ARG((!a->initial_state || aligned(a->initial_state, 16)) && aligned(g->dfinal_state, 16),
                 "selective_scan_backward: states must be 16-byte aligned");
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
