// block_norm.cu -- the join between two blocks of a residual stack, in one
// pass: the norm behind a block with its gate, the scaled residual add, and
// the norm before the next block.  Per row of `cols` channels:
//   n  = y * rstd_post,            rstd_post = rsqrt(mean(y^2) + eps)
//   r' = rho * r + w_post * n * SiLU(z)
//   out = w_pre * r' * rstd_pre,   rstd_pre = rsqrt(mean(r'^2) + eps)
//
// Backward, with R = dL/dr' in all (directly and through the second norm):
//   R  = dr' + rstd_pre (g - m mean(g m)),  g = dout * w_pre, m = r' rstd_pre
//   dr = rho R,   dw_pre = sum dout m,
//   dw_post = sum R n SiLU(z),   dz = R w_post n SiLU'(z),
//   dy = rstd_post (v - n mean(v n)),  v = R w_post SiLU(z)
// where means are over the row and sums over the rows.
#include "common.cuh"
#include "internal.h"
#include "scan_math.cuh"

#include <algorithm>

namespace mb {

namespace {

struct NormParams {
    const void *y, *z;
    const float *res, *w_post, *w_pre;
    float *res_out;
    void *out;
    float *rstd_post, *rstd_pre;
    int64_t rows, sy, sz;
    int cols;
    float rho, eps;
};
struct NormGradParams {
    NormParams f;
    const float *dres_out;
    const void *dout;
    float *dres;
    void *dy, *dz;
    float *part_post, *part_pre;  // [parts, cols] column sums, or NULL
    int64_t sdy, sdz;
};

// SiLU(z) and its derivative.  FP16 tensors: one approximate exponential and
// reciprocal (relative error ~2^-22, far below FP16's 2^-11).
template <bool PRECISE>
__device__ __forceinline__ void silu_grad(float z, float &g, float &dg) {
    const float e = PRECISE ? expf(-fabsf(z)) : ex2_approx(-fabsf(z) * kLog2e);
    const float t = PRECISE ? __fdiv_rn(1.f, 1.f + e) : rcp_approx(1.f + e), u = e * t;
    const float s = z >= 0.f ? t : u, om = z >= 0.f ? u : t;
    g = z * s;
    dg = s * fmaf(z, om, 1.f);
}

constexpr int kMaxCols = 16384;
constexpr int kMaxParts = 444;  // CTAs (and column-sum partials) of the backward pass

// N consecutive elements as FP32; N = 8 by 16-byte accesses.
template <int N>
__device__ __forceinline__ void load_n(const float *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 q = *reinterpret_cast<const float4 *>(p + k);
            v[k] = q.x;
            v[k + 1] = q.y;
            v[k + 2] = q.z;
            v[k + 3] = q.w;
        }
    }
}
template <int N>
__device__ __forceinline__ void load_n(const __half *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = __half2float(*p);
    } else {
        const uint4 raw = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
            v[2 * k] = f.x;
            v[2 * k + 1] = f.y;
        }
    }
}
template <int N>
__device__ __forceinline__ void store_n(float *p, const float (&v)[N]) {
    if constexpr (N == 1) {
        *p = v[0];
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4)
            *reinterpret_cast<float4 *>(p + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    }
}
template <int N>
__device__ __forceinline__ void store_n(__half *p, const float (&v)[N]) {
    if constexpr (N == 1) {
        *p = __float2half_rn(v[0]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <int N>
__device__ __forceinline__ void load_weight(const float *w, int c, float (&v)[N]) {
    if (w) {
        load_n(w + c, v);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 1.f;
    }
}

// Sum over the CTA, the same bits in every thread.  `sm` holds two sets of
// 32 partials used in turn, so one barrier per sum suffices: a set is
// overwritten only after the barrier of the sum in between.
__device__ __forceinline__ float block_sum(float v, float *sm, int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) return v;
    float *s = sm + 32 * turn;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? s[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One CTA per row, the row in registers: thread t holds NV groups of VEC
// channels, group j at channel (j * threads + t) * VEC.
template <typename T, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) block_norm_kernel(const NormParams p) {
    constexpr bool PRECISE = sizeof(T) == 4;
    __shared__ float sm[64];
    int turn = 0;
    const float inv_cols = 1.f / (float)p.cols;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *y = static_cast<const T *>(p.y) + row * p.sy;
        const T *z = p.z ? static_cast<const T *>(p.z) + row * p.sz : nullptr;
        float v[NV][VEC], gz[NV][VEC], r[NV][VEC];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                load_n(y + c, v[j]);
                if (z) load_n(z + c, gz[j]);
                load_n(p.res + row * p.cols + c, r[j]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) ss = fmaf(v[j][k], v[j][k], ss);
            }
        }
        const float rs = rsqrtf(block_sum(ss, sm, turn) * inv_cols + p.eps);
        float ss2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                float w[VEC];
                load_weight(p.w_post, c, w);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float n = v[j][k] * rs * w[k];
                    if (z) {
                        float g, dg;
                        silu_grad<PRECISE>(gz[j][k], g, dg);
                        n *= g;
                    }
                    r[j][k] = fmaf(p.rho, r[j][k], n);
                    ss2 = fmaf(r[j][k], r[j][k], ss2);
                }
                store_n(p.res_out + row * p.cols + c, r[j]);
            }
        }
        if (threadIdx.x == 0 && p.rstd_post) p.rstd_post[row] = rs;
        if (!p.out) continue;
        const float rp = rsqrtf(block_sum(ss2, sm, turn) * inv_cols + p.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                float w[VEC];
                load_weight(p.w_pre, c, w);
#pragma unroll
                for (int k = 0; k < VEC; ++k) w[k] *= r[j][k] * rp;
                store_n(static_cast<T *>(p.out) + row * p.cols + c, w);
            }
        }
        if (threadIdx.x == 0 && p.rstd_pre) p.rstd_pre[row] = rp;
    }
}

// Backward: CTA k walks rows k, k + CTAs, ... and keeps the column sums of
// its rows in registers; they leave as one partial row per CTA.
template <typename T, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) block_norm_bwd_kernel(const NormGradParams p) {
    constexpr bool PRECISE = sizeof(T) == 4;
    __shared__ float sm[64];
    int turn = 0;
    const int cols = p.f.cols;
    const float inv_cols = 1.f / (float)cols;
    float acc_post[NV][VEC] = {}, acc_pre[NV][VEC] = {};
    for (int64_t row = blockIdx.x; row < p.f.rows; row += gridDim.x) {
        const T *y = static_cast<const T *>(p.f.y) + row * p.f.sy;
        const T *z = p.f.z ? static_cast<const T *>(p.f.z) + row * p.f.sz : nullptr;
        const T *go = p.dout ? static_cast<const T *>(p.dout) + row * cols : nullptr;
        const float rs = p.f.rstd_post[row], rp = go ? p.f.rstd_pre[row] : 0.f;
        float R[NV][VEC], n[NV][VEC], gz[NV][VEC], d[NV][VEC], m[NV][VEC];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                load_n(y + c, n[j]);
                if (z) load_n(z + c, gz[j]);
                if (p.dres_out) load_n(p.dres_out + row * cols + c, R[j]);
                if (go) {
                    load_n(go + c, d[j]);
                    load_n(p.f.res_out + row * cols + c, m[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                float w[VEC];
                load_weight(p.f.w_pre, c, w);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    n[j][k] *= rs;
                    if (!p.dres_out) R[j][k] = 0.f;
                    if (go) {
                        m[j][k] *= rp;
                        acc_pre[j][k] = fmaf(d[j][k], m[j][k], acc_pre[j][k]);
                        d[j][k] *= w[k];
                        dot = fmaf(d[j][k], m[j][k], dot);
                    }
                }
            }
        }
        const float mean = go ? block_sum(dot, sm, turn) * inv_cols : 0.f;
        float dot2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                float w[VEC], o[VEC];
                load_weight(p.f.w_post, c, w);
                if (go) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        R[j][k] = fmaf(rp, fmaf(-m[j][k], mean, d[j][k]), R[j][k]);
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) o[k] = p.f.rho * R[j][k];
                store_n(p.dres + row * cols + c, o);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float g = 1.f, dg = 0.f;
                    if (z) silu_grad<PRECISE>(gz[j][k], g, dg);
                    const float Rn = R[j][k] * n[j][k];
                    acc_post[j][k] = fmaf(Rn, g, acc_post[j][k]);
                    o[k] = Rn * w[k] * dg;
                    R[j][k] *= w[k] * g;
                    dot2 = fmaf(R[j][k], n[j][k], dot2);
                }
                if (z) store_n(static_cast<T *>(p.dz) + row * p.sdz + c, o);
            }
        }
        const float mean2 = block_sum(dot2, sm, turn) * inv_cols;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                float o[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) o[k] = rs * fmaf(-n[j][k], mean2, R[j][k]);
                store_n(static_cast<T *>(p.dy) + row * p.sdy + c, o);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + threadIdx.x) * VEC;
        if (c < cols) {
            if (p.part_post) store_n(p.part_post + (int64_t)blockIdx.x * cols + c, acc_post[j]);
            if (p.part_pre) store_n(p.part_pre + (int64_t)blockIdx.x * cols + c, acc_pre[j]);
        }
    }
}

// Column sums of the partial rows, in a fixed order: warp w of a CTA adds
// rows w, w + 8, ... of 32 columns, then the warps' sums are added in order.
// blockIdx.y: 0 = dw_post, 1 = dw_pre.
constexpr int kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads)
    block_norm_sum_kernel(const float *__restrict__ part_post, const float *__restrict__ part_pre,
                          float *__restrict__ dw_post, float *__restrict__ dw_pre, int parts, int cols) {
    __shared__ float sm[kSumThreads / 32][32];
    const float *part = blockIdx.y ? part_pre : part_post;
    float *dw = blockIdx.y ? dw_pre : dw_post;
    if (!dw) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < cols)
        for (int k = warp; k < parts; k += kSumThreads / 32) s += part[(int64_t)k * cols + c];
    sm[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < kSumThreads / 32; ++k) s += sm[k][lane];
        dw[c] = s;
    }
}

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_args(const MambaBlockNormArgs *a, const char *what) {
    MB_CHECK_ARG(a, std::string(what) + ": null args");
    MB_CHECK_ARG(a->rows >= 0 && a->cols >= 0, std::string(what) + ": negative size");
    MB_CHECK_ARG(a->dtype == MAMBA_F32 || a->dtype == MAMBA_F16, std::string(what) + ": bad dtype");
    MB_CHECK_ARG(a->cols <= kMaxCols, std::string(what) + ": more than 16384 channels");
    MB_CHECK_ARG(a->eps > 0.f && a->eps <= 3.0e38f, std::string(what) + ": eps must be positive and finite");
    MB_CHECK_ARG(a->residual_scale - a->residual_scale == 0.f, std::string(what) + ": residual_scale must be finite");
    if (a->rows == 0 || a->cols == 0) return 0;
    MB_CHECK_ARG(a->y && a->residual_out, std::string(what) + ": null pointer");
    const size_t es = dtype_size(a->dtype);
    MB_CHECK_ARG(aligned_to(a->y, es) && aligned_to(a->z, es) && aligned_to(a->out, es) && aligned_to(a->residual, 4) &&
                     aligned_to(a->residual_out, 4) && aligned_to(a->w_post, 4) && aligned_to(a->w_pre, 4) &&
                     aligned_to(a->rstd_post, 4) && aligned_to(a->rstd_pre, 4),
                 std::string(what) + ": pointers must be aligned to their element type");
    return 0;
}

NormParams norm_params(const MambaBlockNormArgs *a) {
    NormParams p{};
    p.y = a->y;
    p.z = a->z;
    p.res = a->residual;
    p.w_post = a->w_post;
    p.w_pre = a->w_pre;
    p.res_out = a->residual_out;
    p.out = a->out;
    p.rstd_post = a->rstd_post;
    p.rstd_pre = a->rstd_pre;
    p.rows = a->rows;
    p.cols = a->cols;
    p.sy = a->y_stride;
    p.sz = a->z_stride;
    p.rho = a->residual_scale;
    p.eps = a->eps;
    return p;
}

// 16-byte accesses: 8 channels at a time, every row start aligned.
bool vector_rows(const MambaBlockNormArgs *a) {
    const int64_t es = (int64_t)dtype_size(a->dtype);
    return a->cols % 8 == 0 && aligned_to(a->y, 16) && aligned_to(a->z, 16) && aligned_to(a->out, 16) &&
           aligned_to(a->residual, 16) && aligned_to(a->residual_out, 16) && aligned_to(a->w_post, 16) &&
           aligned_to(a->w_pre, 16) && (a->y_stride * es) % 16 == 0 && (!a->z || (a->z_stride * es) % 16 == 0);
}

int threads_for(int cols, int per_thread) { return std::max(32, (ceil_div(cols, per_thread) + 31) / 32 * 32); }

template <typename T>
int launch_fwd(const NormParams &p, bool vec, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(p.rows, 0x7fffffff);
    if (vec && p.cols <= 4096)
        block_norm_kernel<T, 8, 1, 512><<<grid, threads_for(p.cols, 8), 0, st>>>(p);
    else if (vec)
        block_norm_kernel<T, 8, 2, 1024><<<grid, threads_for(p.cols, 16), 0, st>>>(p);
    else if (p.cols <= 4096)
        block_norm_kernel<T, 1, 4, 1024><<<grid, threads_for(p.cols, 4), 0, st>>>(p);
    else
        block_norm_kernel<T, 1, 16, 1024><<<grid, threads_for(p.cols, 16), 0, st>>>(p);
    return launch_status("block_norm kernel");
}

template <typename T>
int launch_bwd(const NormGradParams &p, bool vec, unsigned grid, cudaStream_t st) {
    const int cols = p.f.cols;
    if (vec && cols <= 4096)
        block_norm_bwd_kernel<T, 8, 1, 512><<<grid, threads_for(cols, 8), 0, st>>>(p);
    else if (vec)
        block_norm_bwd_kernel<T, 8, 2, 1024><<<grid, threads_for(cols, 16), 0, st>>>(p);
    else if (cols <= 4096)
        block_norm_bwd_kernel<T, 1, 4, 1024><<<grid, threads_for(cols, 4), 0, st>>>(p);
    else
        block_norm_bwd_kernel<T, 1, 16, 1024><<<grid, threads_for(cols, 16), 0, st>>>(p);
    return launch_status("block_norm_backward kernel");
}

}  // namespace

size_t block_norm_workspace_bytes(const MambaBlockNormArgs *a) {
    if (!a || a->rows <= 0 || a->cols <= 0 || a->cols > kMaxCols) return 0;
    // two sets of partial rows, each starting on a 16-byte boundary
    return 2 * (((size_t)std::min<int64_t>(a->rows, kMaxParts) * a->cols + 3) / 4 * 4) * sizeof(float);
}

int block_norm(const MambaBlockNormArgs *a, cudaStream_t st) {
    if (check_args(a, "block_norm")) return -1;
    if (a->rows == 0 || a->cols == 0) return 0;
    MB_CHECK_ARG(a->residual, "block_norm: null pointer");
    const NormParams p = norm_params(a);
    const bool vec = vector_rows(a);
    return a->dtype == MAMBA_F16 ? launch_fwd<__half>(p, vec, st) : launch_fwd<float>(p, vec, st);
}

int block_norm_backward(const MambaBlockNormArgs *a, const MambaBlockNormGrads *g, void *ws, size_t ws_bytes,
                        cudaStream_t st) {
    if (check_args(a, "block_norm_backward")) return -1;
    MB_CHECK_ARG(g, "block_norm_backward: null gradients");
    if (a->cols == 0) return 0;
    MB_CHECK_ARG(aligned_to(g->dw_post, 4) && aligned_to(g->dw_pre, 4),
                 "block_norm_backward: pointers must be aligned to their element type");
    if (a->rows == 0) {
        if (g->dw_post) MB_CUDA_TRY(cudaMemsetAsync(g->dw_post, 0, (size_t)a->cols * 4, st));
        if (g->dw_pre) MB_CUDA_TRY(cudaMemsetAsync(g->dw_pre, 0, (size_t)a->cols * 4, st));
        return 0;
    }
    MB_CHECK_ARG(a->rstd_post && g->dresidual && g->dy && (g->dout || g->dresidual_out),
                 "block_norm_backward: null pointer");
    MB_CHECK_ARG(!g->dout || a->rstd_pre, "block_norm_backward: dout needs rstd_pre");
    MB_CHECK_ARG(!a->z || g->dz, "block_norm_backward: a gate needs dz");
    const size_t es = dtype_size(a->dtype);
    MB_CHECK_ARG(aligned_to(g->dout, es) && aligned_to(g->dy, es) && aligned_to(g->dz, es) &&
                     aligned_to(g->dresidual_out, 4) && aligned_to(g->dresidual, 4),
                 "block_norm_backward: pointers must be aligned to their element type");
    MB_CHECK_ARG(a->rows == 1 || (g->dy_stride >= a->cols && (!a->z || g->dz_stride >= a->cols)),
                 "block_norm_backward: rows of a gradient overlap (strides)");
    MB_CHECK_ARG(ws && ws_bytes >= block_norm_workspace_bytes(a) && aligned_to(ws, 16),
                 "block_norm_backward: workspace too small or not 16-byte aligned");
    const unsigned grid = (unsigned)std::min<int64_t>(a->rows, kMaxParts);
    NormGradParams p{};
    p.f = norm_params(a);
    p.dres_out = g->dresidual_out;
    p.dout = g->dout;
    p.dres = g->dresidual;
    p.dy = g->dy;
    p.dz = g->dz;
    p.sdy = g->dy_stride;
    p.sdz = g->dz_stride;
    float *part = static_cast<float *>(ws);
    if (g->dw_post) p.part_post = part;
    if (g->dw_pre) p.part_pre = part + ((int64_t)grid * a->cols + 3) / 4 * 4;
    const bool vec = vector_rows(a) && aligned_to(g->dout, 16) && aligned_to(g->dresidual_out, 16) &&
                     aligned_to(g->dresidual, 16) && aligned_to(g->dy, 16) && aligned_to(g->dz, 16) &&
                     (g->dy_stride * (int64_t)es) % 16 == 0 && (!a->z || (g->dz_stride * (int64_t)es) % 16 == 0);
    if (a->dtype == MAMBA_F16 ? launch_bwd<__half>(p, vec, grid, st) : launch_bwd<float>(p, vec, grid, st)) return -1;
    if (!g->dw_post && !g->dw_pre) return 0;
    block_norm_sum_kernel<<<dim3((unsigned)ceil_div(a->cols, 32), 2), kSumThreads, 0, st>>>(
        p.part_post, p.part_pre, g->dw_post, g->dw_pre, (int)grid, a->cols);
    return launch_status("block_norm_backward sum kernel");
}

}  // namespace mb
