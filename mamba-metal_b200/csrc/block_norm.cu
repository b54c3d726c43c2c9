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
#include "rows.cuh"
#include "scan_math.cuh"

#include <algorithm>

namespace mb {

__device__ unsigned int g_block_norm_error = 0;

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

// With many rows (RING): persistent CTAs whose rows arrive through shared
// memory.  One thread fetches each row by untiled bulk copies (one per tensor)
// into a ring of `stages` rows, that far ahead, so that loads stay in flight
// through a row's two sums and the threads spend no registers on them.  A
// row's place is free again behind the first sum, when every thread has the
// row in registers.  Bound by bytes.  32768 x 2048 FP16, with the ring and
// without: forward 162 and 182 us (5.8 and 5.2 TB/s), backward 289 and 324;
// 16384 x 4096 164 and 205; unaligned 32768 x 2047 332 and 535.
// Resident threads per SM.  32768 x 2048 FP16: forward 160 us, with 768 threads
// 180, with 1280 207 (57 registers a thread, they no longer fit); backward 276,
// with 512 336.
constexpr int kRingThreads = 1024, kRingBwdThreads = 768;


// One CTA per row, the row in registers: thread t holds NV groups of VEC
// channels, group j at channel (j * threads + t) * VEC.
template <typename T, int VEC, int NV, int MAXT, bool RING, int CTAS = 1>
__global__ void __launch_bounds__(MAXT, CTAS) block_norm_kernel(const NormParams p, const RingRow<3> ring) {
    constexpr bool PRECISE = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kMaxStages];
    __shared__ LostCopies lost;
    __shared__ float sm[64];
    int turn = 0;
    const float inv_cols = 1.f / (float)p.cols;
    RingPlace at;
    if (RING) start_ring<3>(ring, smem, full, &lost, p.rows);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const uint8_t *place = smem + at.s * ring.stage;
        auto at_place = [&](int k) { return place + ring.offset[k] + (VEC == 1 ? ring.shift(k, row) : 0u); };
        const T *y = RING ? reinterpret_cast<const T *>(at_place(0)) : static_cast<const T *>(p.y) + row * p.sy;
        const T *z = RING ? reinterpret_cast<const T *>(at_place(1)) : static_cast<const T *>(p.z) + row * p.sz;
        const float *res = RING ? reinterpret_cast<const float *>(at_place(2)) : p.res + row * p.cols;
        if (RING) await_row(full, at, &lost, &g_block_norm_error);
        float v[NV][VEC], gz[NV][VEC], r[NV][VEC];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                load_n(y + c, v[j]);
                if (p.z) load_n(z + c, gz[j]);
                load_n(res + c, r[j]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) ss = fmaf(v[j][k], v[j][k], ss);
            }
        }
        const float rs = rsqrtf(block_sum(ss, sm, turn) * inv_cols + p.eps);
        if (RING) {
            const int64_t ahead = row + (int64_t)ring.stages * gridDim.x;
            if (threadIdx.x == 0 && ahead < p.rows && !lost.flag) fetch_row<3>(ring, smem, full, ahead, at.s);
            at.step(ring.stages);
        }
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
                    if (p.z) {
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
    if (RING) drain_copies(full, ring.stages, &lost, kWaitNs);
}

// Backward: CTA k walks rows k, k + CTAs, ... and keeps the column sums of
// its rows in registers; they leave as one partial row per CTA.
template <typename T, int VEC, int NV, int MAXT, bool RING, int CTAS = 1>
__global__ void __launch_bounds__(MAXT, CTAS) block_norm_bwd_kernel(const NormGradParams p, const RingRow<5> ring) {
    constexpr bool PRECISE = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kMaxStages];
    __shared__ LostCopies lost;
    __shared__ float sm[64];
    int turn = 0;
    const int cols = p.f.cols;
    const float inv_cols = 1.f / (float)cols;
    float acc_post[NV][VEC] = {}, acc_pre[NV][VEC] = {};
    const bool first = p.dout != nullptr;  // the second norm's output has a gradient
    RingPlace at;
    if (RING) start_ring<5>(ring, smem, full, &lost, p.f.rows);
    float rs_next = p.f.rstd_post[blockIdx.x], rp_next = first ? p.f.rstd_pre[blockIdx.x] : 0.f;  // grid <= rows
    for (int64_t row = blockIdx.x; row < p.f.rows; row += gridDim.x) {
        const uint8_t *place = smem + at.s * ring.stage;
        auto at_place = [&](int k) { return place + ring.offset[k] + (VEC == 1 ? ring.shift(k, row) : 0u); };
        const T *y = RING ? reinterpret_cast<const T *>(at_place(0)) : static_cast<const T *>(p.f.y) + row * p.f.sy;
        const T *z = RING ? reinterpret_cast<const T *>(at_place(1)) : static_cast<const T *>(p.f.z) + row * p.f.sz;
        const T *go = RING ? reinterpret_cast<const T *>(at_place(2)) : static_cast<const T *>(p.dout) + row * cols;
        const float *dro = RING ? reinterpret_cast<const float *>(at_place(3)) : p.dres_out + row * cols;
        const float *r1 = RING ? reinterpret_cast<const float *>(at_place(4)) : p.f.res_out + row * cols;
        // this row's factors were loaded a row ago, the next row's are on their way
        const float rs = rs_next, rp = rp_next;
        const int64_t after = row + gridDim.x;
        if (after < p.f.rows) {
            rs_next = p.f.rstd_post[after];
            if (first) rp_next = p.f.rstd_pre[after];
        }
        if (RING) await_row(full, at, &lost, &g_block_norm_error);
        float R[NV][VEC], n[NV][VEC], gz[NV][VEC], d[NV][VEC], m[NV][VEC];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                load_n(y + c, n[j]);
                if (p.f.z) load_n(z + c, gz[j]);
                if (p.dres_out) load_n(dro + c, R[j]);
                if (first) {
                    load_n(go + c, d[j]);
                    load_n(r1 + c, m[j]);
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
                    if (first) {
                        m[j][k] *= rp;
                        acc_pre[j][k] = fmaf(d[j][k], m[j][k], acc_pre[j][k]);
                        d[j][k] *= w[k];
                        dot = fmaf(d[j][k], m[j][k], dot);
                    }
                }
            }
        }
        // (without dout the sum is 0, and its barrier still frees the ring's place)
        const float mean = RING || first ? block_sum(dot, sm, turn) * inv_cols : 0.f;
        if (RING) {
            const int64_t ahead = row + (int64_t)ring.stages * gridDim.x;
            if (threadIdx.x == 0 && ahead < p.f.rows && !lost.flag) fetch_row<5>(ring, smem, full, ahead, at.s);
            at.step(ring.stages);
        }
        float dot2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                float w[VEC], o[VEC];
                load_weight(p.f.w_post, c, w);
                if (first) {
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
                    if (p.f.z) silu_grad<PRECISE>(gz[j][k], g, dg);
                    const float Rn = R[j][k] * n[j][k];
                    acc_post[j][k] = fmaf(Rn, g, acc_post[j][k]);
                    o[k] = Rn * w[k] * dg;
                    R[j][k] *= w[k] * g;
                    dot2 = fmaf(R[j][k], n[j][k], dot2);
                }
                if (p.f.z) store_n(static_cast<T *>(p.dz) + row * p.sdz + c, o);
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
    if (RING) drain_copies(full, ring.stages, &lost, kWaitNs);
}

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

// Rows of partial column sums of the backward pass at most.
int64_t max_parts(int64_t rows, int cols) {
    const int ctas = std::min(16, ring_ctas(threads_for(cols, cols <= 4096 ? 8 : 16), kRingBwdThreads));
    return std::min<int64_t>(rows, std::max(kDirectParts, 148 * ctas));
}

template <typename T, int VEC, int NV, int MAXT>
int ring_fwd(const NormParams &p, const RingRow<3> &r, int ctas, int threads, cudaStream_t st) {
    auto kernel = block_norm_kernel<T, VEC, NV, MAXT, true>;
    if (allow_smem(kernel)) return -1;
    kernel<<<(unsigned)(ctas * device_sm_count()), threads, (size_t)r.stage * r.stages, st>>>(p, r);
    return launch_status("block_norm kernel");
}
template <typename T>
int launch_fwd(const NormParams &p, bool vec, cudaStream_t st) {
    RingRow<3> r{};
    if (p.cols <= 8192) {
        const uint32_t half = (uint32_t)(p.cols * sizeof(T));
        r.src[0] = p.y;
        r.src[1] = p.z;
        r.src[2] = p.res;
        r.stride[0] = p.sy * (int64_t)sizeof(T);
        r.stride[1] = p.sz * (int64_t)sizeof(T);
        r.stride[2] = p.cols * 4LL;
        r.bytes[0] = half;
        r.bytes[1] = p.z ? half : 0;
        r.bytes[2] = (uint32_t)p.cols * 4;
        const bool one = p.cols <= 4096;
        const int threads = threads_for(p.cols, one ? 8 : 16);
        int ctas = ring_ctas(threads, kRingThreads);
        if (plan_ring<3>(r, p.rows, ctas)) {
            if (vec)
                return one ? ring_fwd<T, 8, 1, 512>(p, r, ctas, threads, st)
                           : ring_fwd<T, 8, 2, 512>(p, r, ctas, threads, st);
            return one ? ring_fwd<T, 1, 8, 512>(p, r, ctas, threads, st)
                       : ring_fwd<T, 1, 16, 512>(p, r, ctas, threads, st);
        }
    }
    const unsigned grid = (unsigned)std::min<int64_t>(p.rows, 0x7fffffff);
    if (vec && p.cols <= 4096)
        block_norm_kernel<T, 8, 1, 512, false><<<grid, threads_for(p.cols, 8), 0, st>>>(p, r);
    else if (vec)
        block_norm_kernel<T, 8, 2, 1024, false><<<grid, threads_for(p.cols, 16), 0, st>>>(p, r);
    else if (p.cols <= 4096)
        block_norm_kernel<T, 1, 4, 1024, false><<<grid, threads_for(p.cols, 4), 0, st>>>(p, r);
    else
        block_norm_kernel<T, 1, 16, 1024, false><<<grid, threads_for(p.cols, 16), 0, st>>>(p, r);
    return launch_status("block_norm kernel");
}

template <typename T, int VEC, int NV, int MAXT, int CTAS>
int ring_bwd(const NormGradParams &p, const RingRow<5> &r, unsigned grid, int threads, cudaStream_t st) {
    auto kernel = block_norm_bwd_kernel<T, VEC, NV, MAXT, true, CTAS>;
    if (allow_smem(kernel)) return -1;
    kernel<<<grid, threads, (size_t)r.stage * r.stages, st>>>(p, r);
    return launch_status("block_norm_backward kernel");
}
// grid: CTAs to launch at most; set to those launched (rows of partial sums).
template <typename T>
int launch_bwd(const NormGradParams &p, bool vec, unsigned &grid, cudaStream_t st) {
    const int cols = p.f.cols;
    RingRow<5> r{};
    if (cols <= 8192) {
        const uint32_t half = (uint32_t)(cols * sizeof(T)), whole = (uint32_t)cols * 4;
        const void *src[5] = {p.f.y, p.f.z, p.dout, p.dres_out, p.f.res_out};
        const int64_t stride[5] = {p.f.sy * (int64_t)sizeof(T), p.f.sz * (int64_t)sizeof(T), half, whole, whole};
        for (int k = 0; k < 5; ++k) {
            r.src[k] = src[k];
            r.stride[k] = stride[k];
            r.bytes[k] = k < 3 ? half : whole;
            if (!src[k] || (k == 4 && !p.dout)) r.bytes[k] = 0;
        }
        const bool one = cols <= 4096;
        const int threads = threads_for(cols, one ? 8 : 16);
        int ctas = std::min(16, ring_ctas(threads, kRingBwdThreads));
        if (plan_ring<5>(r, p.f.rows, ctas)) {
            grid = std::min(grid, (unsigned)(ctas * device_sm_count()));
            if (!one)
                return vec ? ring_bwd<T, 8, 2, 512, 1>(p, r, grid, threads, st)
                           : ring_bwd<T, 1, 16, 512, 1>(p, r, grid, threads, st);
            if (!vec) return ring_bwd<T, 1, 8, 512, 1>(p, r, grid, threads, st);
            // three CTAs fit by 80 registers a thread; with fewer, more registers are faster
            return threads <= 256 && ctas >= 3 ? ring_bwd<T, 8, 1, 256, 3>(p, r, grid, threads, st)
                                               : ring_bwd<T, 8, 1, 512, 1>(p, r, grid, threads, st);
        }
    }
    grid = std::min(grid, (unsigned)kDirectParts);
    if (vec && cols <= 4096)
        block_norm_bwd_kernel<T, 8, 1, 512, false><<<grid, threads_for(cols, 8), 0, st>>>(p, r);
    else if (vec)
        block_norm_bwd_kernel<T, 8, 2, 1024, false><<<grid, threads_for(cols, 16), 0, st>>>(p, r);
    else if (cols <= 4096)
        block_norm_bwd_kernel<T, 1, 4, 1024, false><<<grid, threads_for(cols, 4), 0, st>>>(p, r);
    else
        block_norm_bwd_kernel<T, 1, 16, 1024, false><<<grid, threads_for(cols, 16), 0, st>>>(p, r);
    return launch_status("block_norm_backward kernel");
}

}  // namespace

size_t block_norm_workspace_bytes(const MambaBlockNormArgs *a) {
    if (!a || a->rows <= 0 || a->cols <= 0 || a->cols > kMaxCols) return 0;
    // two sets of partial rows, each starting on a 16-byte boundary
    return 2 * (((size_t)max_parts(a->rows, a->cols) * a->cols + 3) / 4 * 4) * sizeof(float);
}

int block_norm(const MambaBlockNormArgs *a, cudaStream_t st) {
    if (check_args(a, "block_norm")) return -1;
    if (a->rows == 0 || a->cols == 0) return 0;
    MB_CHECK_ARG(a->residual, "block_norm: null pointer");
    MB_CHECK_ARG(!a->out || (a->out != a->y && a->out != a->z && a->out != a->residual && a->out != a->residual_out),
                 "block_norm: out needs memory of its own");
    MB_CHECK_ARG(a->residual_out != a->y && a->residual_out != a->z, "block_norm: residual_out may not be y or z");
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
    const void *in[4] = {a->y, a->z, g->dout, a->residual_out};
    for (const void *p : in)
        MB_CHECK_ARG(p != g->dy && p != g->dresidual && (!p || p != g->dz),
                     "block_norm_backward: a gradient may not be one of the inputs");
    MB_CHECK_ARG(g->dy != g->dz && static_cast<void *>(g->dresidual) != g->dy &&
                     static_cast<void *>(g->dresidual) != g->dz && g->dresidual_out != g->dy &&
                     (!g->dz || g->dresidual_out != g->dz),
                 "block_norm_backward: the gradients need memory of their own");
    MB_CHECK_ARG(a->rows == 1 || (g->dy_stride >= a->cols && (!a->z || g->dz_stride >= a->cols)),
                 "block_norm_backward: rows of a gradient overlap (strides)");
    MB_CHECK_ARG(ws && ws_bytes >= block_norm_workspace_bytes(a) && aligned_to(ws, 16),
                 "block_norm_backward: workspace too small or not 16-byte aligned");
    unsigned grid = (unsigned)max_parts(a->rows, a->cols);  // launch_bwd may take fewer
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
    if (g->dw_pre) p.part_pre = part + ((int64_t)grid * a->cols + 3) / 4 * 4;  // grid is still the most
    const bool vec = vector_rows(a) && aligned_to(g->dout, 16) && aligned_to(g->dresidual_out, 16) &&
                     aligned_to(g->dresidual, 16) && aligned_to(g->dy, 16) && aligned_to(g->dz, 16) &&
                     (g->dy_stride * (int64_t)es) % 16 == 0 && (!a->z || (g->dz_stride * (int64_t)es) % 16 == 0);
    if (a->dtype == MAMBA_F16 ? launch_bwd<__half>(p, vec, grid, st) : launch_bwd<float>(p, vec, grid, st)) return -1;
    if (!g->dw_post && !g->dw_pre) return 0;
    column_sum_kernel<><<<dim3((unsigned)ceil_div(a->cols, 32), 2), kSumThreads, 0, st>>>(
        p.part_post, p.part_pre, g->dw_post, g->dw_pre, (int)grid, a->cols);
    return launch_status("block_norm_backward sum kernel");
}

namespace {

// A wait for a row that nothing fetches, through the kernels' own helper.
__global__ void block_norm_wait_selftest_kernel(uint64_t limit_ns) {
    __shared__ uint64_t full[2];
    __shared__ LostCopies lost;
    if (threadIdx.x != 0) return;
    lost = LostCopies{};
    for (int s = 0; s < 2; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    RingPlace at;
    await_row(full, at, &lost, &g_block_norm_error, limit_ns);
    at.step(2);
    await_row(full, at, &lost, &g_block_norm_error, limit_ns);  // at once
    drain_copies(full, 2, &lost, limit_ns);
}

}  // namespace

int block_norm_wait_selftest(uint64_t limit_ns, cudaStream_t st) {
    block_norm_wait_selftest_kernel<<<1, 32, 0, st>>>(limit_ns);
    return launch_status("block_norm wait self-test kernel");
}

unsigned block_norm_error_flags(bool clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_block_norm_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (clear && v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_block_norm_error, &z, sizeof(z));
    }
    return v;
}

}  // namespace mb
