// conv_bwd.cu -- gradients of the depthwise causal conv of conv.cu
// (Sources/Kernels/causal_conv1d.metal:21-45 with the SiLU of
// MambaRuntime.cpp:96).  With pre_t = sum_k w_k x_{t-K+1+k} + bias and
// p_t = dy_t SiLU'(pre_t) (dy_t without the activation):
//   dx_t = sum_k w_k p_{t+K-1-k},  dw_k = sum_t p_t x_{t-K+1+k},  dbias = sum_t p_t
//
// One pass over x and dy that writes dx.  8 x 4096 x 4096 FP16, K 4, SiLU: 160-168
// us for 805 MB with 4 channels a thread and 128 registers (four CTAs an SM); with
// 154 registers 182, 102 registers 244, 2 channels a thread 227, 8 rows in flight
// instead of 4 203.  Neither bytes (DRAM 60%) nor issue slots (51%) are used up:
// 16 warps an SM with 4 rows of x and dy each in flight wait for memory.  A thread owns VEC
// channels and a run of timesteps; the last K inputs and the last K p_t stay in
// registers, so a run reads K - 1 rows before it (of x) and behind it (of
// both) again.  The sums of dw and dbias leave as one partial row per run and
// are added in a fixed order.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "scan_math.cuh"

namespace mb {
namespace {

struct ConvGradParams {
    const void *dy, *x;
    const float *w, *bias;
    void *dx;
    float *part;  // [runs * batch][K + 1][dim]: K taps, then the bias
    int64_t sdy[3], sx[3], sdx[3];
    int batch, L, D, run, runs, blocks;
    bool silu;
};

constexpr int kCbThreads = 128;
constexpr int kCbRows = 4;  // rows of x and dy in flight

// Channels a thread where rows allow it.  FP32: with 4 a thread needs 188
// registers (8 x 4096 x 1000 115 us, with 2 93).  FP16 with 5 to 8 taps, 188 to 228
// registers: 8 x 4096 x 4096 219, 242, 264, 301 us, with 2 channels 221, 282, 292,
// 302; 8 x 4096 x 1000 63, 71, 78, 90 and 58, 82, 85, 90; 1 x 4096 x 2048 20.7,
// 25.4, 27.4, 35.7 and 18.7, 25.8, 27.5, 31.6.
template <typename T> constexpr int kWideChannels = sizeof(T) == 2 ? 4 : 2;

// A row's VEC channels as loaded, and as pairs.
template <typename T, int VEC> struct RowVec;
template <typename T> struct RowVec<T, 1> {
    using Raw = T;
    static __device__ __forceinline__ void unpack(const T &r, float2 *f) { f[0] = make_float2(cvt_f32<T>(r), 0.f); }
    static __device__ __forceinline__ T pack(const float2 *f) { return cvt_out<T>(f[0].x); }
    static __device__ __forceinline__ T zero() { return cvt_out<T>(0.f); }
};
template <> struct RowVec<__half, 4> {
    using Raw = uint2;
    static __device__ __forceinline__ void unpack(const uint2 &r, float2 *f) {
        f[0] = __half22float2(*reinterpret_cast<const __half2 *>(&r.x));
        f[1] = __half22float2(*reinterpret_cast<const __half2 *>(&r.y));
    }
    static __device__ __forceinline__ uint2 pack(const float2 *f) {
        const __half2 a = __float22half2_rn(f[0]), b = __float22half2_rn(f[1]);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    static __device__ __forceinline__ uint2 zero() { return make_uint2(0u, 0u); }
};
template <> struct RowVec<__half, 2> {
    using Raw = __half2;
    static __device__ __forceinline__ void unpack(const __half2 &r, float2 *f) { f[0] = __half22float2(r); }
    static __device__ __forceinline__ __half2 pack(const float2 *f) { return __float22half2_rn(f[0]); }
    static __device__ __forceinline__ __half2 zero() { return __float2half2_rn(0.f); }
};
template <> struct RowVec<float, 2> {
    using Raw = float2;
    static __device__ __forceinline__ void unpack(const float2 &r, float2 *f) { f[0] = r; }
    static __device__ __forceinline__ float2 pack(const float2 *f) { return f[0]; }
    static __device__ __forceinline__ float2 zero() { return make_float2(0.f, 0.f); }
};
// SiLU'(v) = t (1 + v e t) with e = e^-v and t = 1 / (1 + e), for two values of
// FP16 tensors (approximate exponential and reciprocal, 2^-22 each).  e ends at
// 2^126, where t is the smallest normal number; a NaN stays one.
__device__ __forceinline__ float min_nan(float v, float hi) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 silu_slope_2(float2 v) {
    const float2 one = make_float2(1.f, 1.f), n = __fmul2_rn(v, make_float2(-kLog2e, -kLog2e));
    const float2 e = make_float2(ex2_approx(min_nan(n.x, 126.f)), ex2_approx(min_nan(n.y, 126.f)));
    float2 t = __fadd2_rn(e, one);
    t = make_float2(rcp_approx(t.x), rcp_approx(t.y));
    return __fmul2_rn(t, __ffma2_rn(v, __fmul2_rn(e, t), one));
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kCbThreads, sizeof(T) == 2 && K <= 4 ? 4 : 1) conv1d_bwd_kernel(const ConvGradParams p) {
    using Rv = RowVec<T, VEC>;
    using Raw = typename Rv::Raw;
    constexpr bool PRECISE = sizeof(T) == 4;
    const int block = blockIdx.x % p.blocks, rest = blockIdx.x / p.blocks;
    const int run = rest % p.runs, b = rest / p.runs;
    const int d0 = (block * kCbThreads + threadIdx.x) * VEC;
    if (d0 >= p.D) return;
    const int t0 = run * p.run, t1 = min(p.L, t0 + p.run);
    const T *x = static_cast<const T *>(p.x) + b * p.sx[0] + d0 * p.sx[2];
    const T *dy = static_cast<const T *>(p.dy) + b * p.sdy[0] + d0 * p.sdy[2];
    T *dx = static_cast<T *>(p.dx) + b * p.sdx[0] + d0 * p.sdx[2];
    auto row = [&](const T *v, const int64_t *s, int t) {
        return t < p.L ? *reinterpret_cast<const Raw *>(v + (int64_t)t * s[1]) : Rv::zero();
    };
    // channels in pairs: one packed operation for two (VEC 1: the second half idles)
    constexpr int P = (VEC + 1) / 2;
    float2 w[K][P], bias[P];
    auto pair = [&](auto &&get) { return make_float2(get(0), VEC > 1 ? get(1) : 0.f); };
#pragma unroll
    for (int c = 0; c < P; ++c) {
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][c] = pair([&](int e) { return p.w[(int64_t)(d0 + 2 * c + e) * K + k]; });
        bias[c] = p.bias ? pair([&](int e) { return p.bias[d0 + 2 * c + e]; }) : make_float2(0.f, 0.f);
    }
    float2 win[K][P] = {};  // x_{s-K+1} .. x_s
    float2 pw[K][P] = {};   // p_{s-K+1} .. p_s
    float2 dw[K][P] = {}, db[P] = {};
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int t = t0 - K + 1 + k;
        if (t >= 0) Rv::unpack(row(x, p.sx, t), win[k]);
    }
    Raw xr[kCbRows], yr[kCbRows];
#pragma unroll
    for (int r = 0; r < kCbRows; ++r) {
        xr[r] = row(x, p.sx, t0 + r);
        yr[r] = row(dy, p.sdy, t0 + r);
    }
    // the next rows to fetch and to write
    const T *xn = x + (int64_t)(t0 + kCbRows) * p.sx[1], *yn = dy + (int64_t)(t0 + kCbRows) * p.sdy[1];
    T *out_at = dx + (int64_t)(t0 - K + 1) * p.sdx[1];
    const int s1 = t1 + K - 1;  // rows behind the run complete its last gradients
    // one row: SUM, it belongs to the run (its p_t counts in dw); PUT, a gradient is complete with it
    auto one_row = [&](const Raw &xv, const Raw &yv, bool sum, bool put) {
        Rv::unpack(xv, win[K - 1]);
        Rv::unpack(yv, pw[K - 1]);
        if (p.silu) {
#pragma unroll
            for (int c = 0; c < P; ++c) {
                float2 pre = bias[c], slope;
#pragma unroll
                for (int k = 0; k < K; ++k) pre = __ffma2_rn(win[k][c], w[k][c], pre);
                if (PRECISE) {
                    float g;
                    silu_grad<true>(pre.x, g, slope.x);
                    if (VEC > 1) silu_grad<true>(pre.y, g, slope.y);
                    else slope.y = 0.f;
                } else {
                    slope = silu_slope_2(pre);
                }
                pw[K - 1][c] = __fmul2_rn(pw[K - 1][c], slope);
            }
        }
        if (sum) {
#pragma unroll
            for (int c = 0; c < P; ++c) {
#pragma unroll
                for (int k = 0; k < K; ++k) dw[k][c] = __ffma2_rn(pw[K - 1][c], win[k][c], dw[k][c]);
                db[c] = __fadd2_rn(db[c], pw[K - 1][c]);
            }
        }
        if (put) {
            float2 out[P];
#pragma unroll
            for (int c = 0; c < P; ++c) {
                out[c] = __fmul2_rn(w[0][c], pw[K - 1][c]);
#pragma unroll
                for (int k = 1; k < K; ++k) out[c] = __ffma2_rn(w[k][c], pw[K - 1 - k][c], out[c]);
            }
            *reinterpret_cast<Raw *>(out_at) = Rv::pack(out);
        }
        out_at += p.sdx[1];
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int c = 0; c < P; ++c) {
                win[k][c] = win[k + 1][c];
                pw[k][c] = pw[k + 1][c];
            }
    };
    for (int sb = t0; sb < s1; sb += kCbRows) {
        Raw xc[kCbRows], yc[kCbRows];
#pragma unroll
        for (int r = 0; r < kCbRows; ++r) {
            xc[r] = xr[r];
            yc[r] = yr[r];
        }
        if (sb + 2 * kCbRows <= p.L) {
#pragma unroll
            for (int r = 0; r < kCbRows; ++r) {
                xr[r] = *reinterpret_cast<const Raw *>(xn);
                yr[r] = *reinterpret_cast<const Raw *>(yn);
                xn += p.sx[1];
                yn += p.sdy[1];
            }
        } else if (sb + kCbRows < s1) {
#pragma unroll
            for (int r = 0; r < kCbRows; ++r) {
                xr[r] = row(x, p.sx, sb + kCbRows + r);
                yr[r] = row(dy, p.sdy, sb + kCbRows + r);
            }
        }
        if (sb >= t0 + K - 1 && sb + kCbRows <= t1) {  // inside the run: no conditions
#pragma unroll
            for (int r = 0; r < kCbRows; ++r) one_row(xc[r], yc[r], true, true);
        } else {
#pragma unroll
            for (int r = 0; r < kCbRows; ++r) {
                const int s = sb + r;
                one_row(xc[r], yc[r], s < t1, s - K + 1 >= t0 && s - K + 1 < t1);
            }
        }
    }
    float *part = p.part + (int64_t)rest * (K + 1) * p.D + d0;
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int c = 0; c < P; ++c) {
            const float2 v = k < K ? dw[k < K ? k : 0][c] : db[c];
            part[(int64_t)k * p.D + 2 * c] = v.x;
            if (VEC > 1) part[(int64_t)k * p.D + 2 * c + 1] = v.y;
        }
}

// dw and dbias from the partial rows, in a fixed order: warp v of a CTA adds
// rows v, v + warps, ... of 32 channels and one tap, then the warps' sums are added
// in order.
template <int THREADS>
__global__ void __launch_bounds__(THREADS)
    conv1d_bwd_sum_kernel(const float *__restrict__ part, float *__restrict__ dw, float *__restrict__ dbias, int parts,
                          int K, int D) {
    __shared__ float sm[THREADS / 32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane, k = blockIdx.y;
    if (k == K ? !dbias : !dw) return;
    float s = 0.f;
    if (d < D)
        for (int i = warp; i < parts; i += THREADS / 32) s += part[((int64_t)i * (K + 1) + k) * D + d];
    sm[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && d < D) {
#pragma unroll
        for (int v = 1; v < THREADS / 32; ++v) s += sm[v][lane];
        if (k == K)
            dbias[d] = s;
        else
            dw[(int64_t)d * K + k] = s;
    }
}

// Timesteps per thread: 128, fewer where that leaves less than 256 threads an SM (8
// x 4096 x 1000 FP16 and 1 x 4096 x 2048, with the sums of the partial rows: 56
// and 21 us; for 512 threads 55 and 24, 1024 66 and 24).
int run_length(int64_t batch, int64_t L, int64_t D) {
    int run = 128;
    while (run > 16 && batch * ceil_div64(L, run) * ceil_div64(D, 4) < 148 * 256) run /= 2;
    return run;
}

template <typename T, int K>
int launch_conv_bwd(ConvGradParams &p, int vec, cudaStream_t st) {
    p.blocks = ceil_div(p.D, kCbThreads * vec);
    const int64_t grid = (int64_t)p.blocks * p.runs * p.batch;
    MB_CHECK_ARG(grid <= 0x7fffffff, "causal_conv1d_backward: too many elements");
    if (vec == kWideChannels<T>)
        conv1d_bwd_kernel<T, K, kWideChannels<T>><<<(unsigned)grid, kCbThreads, 0, st>>>(p);
    else if (vec == 2)
        conv1d_bwd_kernel<T, K, 2><<<(unsigned)grid, kCbThreads, 0, st>>>(p);
    else
        conv1d_bwd_kernel<T, K, 1><<<(unsigned)grid, kCbThreads, 0, st>>>(p);
    return launch_status("causal_conv1d_backward kernel");
}
template <typename T>
int launch_conv_bwd(ConvGradParams &p, int K, int vec, cudaStream_t st) {
    switch (K) {
        case 1: return launch_conv_bwd<T, 1>(p, vec, st);
        case 2: return launch_conv_bwd<T, 2>(p, vec, st);
        case 3: return launch_conv_bwd<T, 3>(p, vec, st);
        case 4: return launch_conv_bwd<T, 4>(p, vec, st);
        case 5: return launch_conv_bwd<T, 5>(p, vec, st);
        case 6: return launch_conv_bwd<T, 6>(p, vec, st);
        case 7: return launch_conv_bwd<T, 7>(p, vec, st);
        default: return launch_conv_bwd<T, 8>(p, vec, st);
    }
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Rows of n channels at a time: channels adjacent, every row start aligned.
bool vector_rows(const void *v, const int64_t *s, int64_t es, int n) {
    return s[2] == 1 && aligned(v, (size_t)(n * es)) && s[1] % n == 0 && s[0] % n == 0;
}

int check(const MambaConvGradArgs *a) {
    MB_CHECK_ARG(a, "causal_conv1d_backward: null args");
    MB_CHECK_ARG(a->batch >= 0 && a->seqlen >= 0 && a->dim >= 0, "causal_conv1d_backward: negative size");
    MB_CHECK_ARG(a->K >= 1 && a->K <= 8, "causal_conv1d_backward: K must be in 1..8");
    MB_CHECK_ARG(a->dtype == MAMBA_F32 || a->dtype == MAMBA_F16, "causal_conv1d_backward: bad dtype");
    MB_CHECK_ARG(a->seqlen <= 0x7fffffff - 256, "causal_conv1d_backward: sequence too long");
    return 0;
}

}  // namespace

size_t causal_conv1d_backward_workspace_bytes(const MambaConvGradArgs *a) {
    if (!a || a->batch <= 0 || a->seqlen <= 0 || a->dim <= 0 || a->K < 1 || a->K > 8) return 0;
    return (size_t)a->batch * ceil_div64(a->seqlen, run_length(a->batch, a->seqlen, a->dim)) * (a->K + 1) * a->dim * 4;
}

int causal_conv1d_backward(const MambaConvGradArgs *a, void *ws, size_t ws_bytes, cudaStream_t st) {
    if (check(a)) return -1;
    if (a->dim == 0) return 0;
    MB_CHECK_ARG(aligned(a->dw, 4) && aligned(a->dbias, 4),
                 "causal_conv1d_backward: pointers must be aligned to their element type");
    MB_CHECK_ARG(!a->dw || a->dw != a->dbias, "causal_conv1d_backward: dw and dbias need memory of their own");
    if (a->batch == 0 || a->seqlen == 0) {
        if (a->dw) MB_CUDA_TRY(cudaMemsetAsync(a->dw, 0, (size_t)a->dim * a->K * 4, st));
        if (a->dbias) MB_CUDA_TRY(cudaMemsetAsync(a->dbias, 0, (size_t)a->dim * 4, st));
        return 0;
    }
    const size_t es = dtype_size(a->dtype);
    MB_CHECK_ARG(a->dy && a->x && a->w && a->dx, "causal_conv1d_backward: null pointer");
    MB_CHECK_ARG(aligned(a->dy, es) && aligned(a->x, es) && aligned(a->dx, es) && aligned(a->w, 4) && aligned(a->bias, 4),
                 "causal_conv1d_backward: pointers must be aligned to their element type");
    MB_CHECK_ARG(a->dx != a->x && a->dx != a->dy, "causal_conv1d_backward: dx needs memory of its own");
    MB_CHECK_ARG((a->batch == 1 || a->dx_stride[0] != 0) && (a->seqlen == 1 || a->dx_stride[1] != 0) &&
                     (a->dim == 1 || a->dx_stride[2] != 0),
                 "causal_conv1d_backward: the elements of dx overlap (strides)");
    MB_CHECK_ARG(ws && ws_bytes >= causal_conv1d_backward_workspace_bytes(a) && aligned(ws, 16),
                 "causal_conv1d_backward: workspace too small or not 16-byte aligned");
    ConvGradParams p{};
    p.dy = a->dy;
    p.x = a->x;
    p.w = a->w;
    p.bias = a->bias;
    p.dx = a->dx;
    p.part = static_cast<float *>(ws);
    for (int k = 0; k < 3; ++k) {
        p.sdy[k] = a->dy_stride[k];
        p.sx[k] = a->x_stride[k];
        p.sdx[k] = a->dx_stride[k];
    }
    p.batch = a->batch;
    p.L = a->seqlen;
    p.D = a->dim;
    p.run = run_length(a->batch, a->seqlen, a->dim);
    p.runs = ceil_div(p.L, p.run);
    p.silu = a->silu != 0;
    MB_CHECK_ARG((int64_t)p.runs * p.batch <= 0x7fffffff, "causal_conv1d_backward: too many elements");
    int vec = a->dtype == MAMBA_F16 ? kWideChannels<__half> : kWideChannels<float>;
    while (vec > 1 && !(p.D % vec == 0 && vector_rows(a->x, p.sx, (int64_t)es, vec) &&
                        vector_rows(a->dy, p.sdy, (int64_t)es, vec) && vector_rows(a->dx, p.sdx, (int64_t)es, vec)))
        vec /= 2;
    if (a->dtype == MAMBA_F16 ? launch_conv_bwd<__half>(p, a->K, vec, st) : launch_conv_bwd<float>(p, a->K, vec, st))
        return -1;
    if (!a->dw && !a->dbias) return 0;
    // 32 warps to a CTA where that is one round of CTAs (777 channels, 282 rows 3.7 us, 5.2 with 8), else 8 (4096
    // channels, 256 rows 8.5, with 32 15.8)
    const dim3 grid((unsigned)ceil_div(p.D, 32), (unsigned)(a->K + 1));
    if (grid.x * grid.y <= 2u * (unsigned)device_sm_count())
        conv1d_bwd_sum_kernel<1024><<<grid, 1024, 0, st>>>(p.part, a->dw, a->dbias, p.runs * p.batch, a->K, p.D);
    else
        conv1d_bwd_sum_kernel<256><<<grid, 256, 0, st>>>(p.part, a->dw, a->dbias, p.runs * p.batch, a->K, p.D);
    return launch_status("causal_conv1d_backward sum kernel");
}

}  // namespace mb
