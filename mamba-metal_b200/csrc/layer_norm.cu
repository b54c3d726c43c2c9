// layer_norm.cu -- layer norm over rows of channels and its gradients:
//   y = (x - mean) * rstd * w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
// Backward, with n = (x - mean) rstd and u = dout * w:
//   dx = rstd (u - mean(u) - n mean(u n)),   dw = sum dout n,   db = sum dout
// where means are over the row and sums over the rows.
//
// The deviation is a second sum over the row held in registers, not
// mean(x^2) - mean^2, which cancels where the mean is large.  Bound by bytes:
// each pass reads its rows once.  With many rows the next one is loaded ahead:
// into registers (forward), or through the ring of rows.cuh (backward, whose
// registers hold the column sums, and rows that are not 16-byte aligned).
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace mb {

__device__ unsigned int g_layer_norm_error = 0;

namespace {

struct LayerNormParams {
    const void *x;
    const float *w, *b;
    void *out;
    float *mean, *rstd;
    int64_t rows, sx, so;
    int cols;
    float eps;
};
struct LayerNormGradParams {
    const void *dout, *x;
    const float *w, *mean, *rstd;
    void *dx;
    float *part_w, *part_b;  // [parts, cols] column sums, or NULL
    int64_t rows, sg, sx, sdx;
    int cols;
};

// One CTA per row at a time, the row in registers: thread t holds NV groups of
// VEC channels, group j at channel (j * threads + t) * VEC.
template <typename TX, typename TO, int VEC, int NV, int MAXT, bool RING>
__global__ void __launch_bounds__(MAXT) layer_norm_kernel(const LayerNormParams p, const RingRow<1> ring) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kMaxStages];
    __shared__ LostCopies lost;
    __shared__ float sm[64];
    int turn = 0;
    const float inv_cols = 1.f / (float)p.cols;
    RingPlace at;
    if (RING) start_ring<1>(ring, smem, full, &lost, p.rows);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const TX *x = RING ? reinterpret_cast<const TX *>(smem + at.s * ring.stage + (VEC <= 2 ? ring.shift(0, row) : 0u))
                           : static_cast<const TX *>(p.x) + row * p.sx;
        if (RING) await_row(full, at, &lost, &g_layer_norm_error);
        float v[NV][VEC];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                load_n(x + c, v[j]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) s += v[j][k];
            }
        }
        const float mean = block_sum(s, sm, turn) * inv_cols;
        if (RING) {
            const int64_t ahead = row + (int64_t)ring.stages * gridDim.x;
            if (threadIdx.x == 0 && ahead < p.rows && !lost.flag) fetch_row<1>(ring, smem, full, ahead, at.s);
            at.step(ring.stages);
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v[j][k] -= mean;
                    ss = fmaf(v[j][k], v[j][k], ss);
                }
            }
        }
        const float rs = rsqrtf(block_sum(ss, sm, turn) * inv_cols + p.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                float w[VEC], b[VEC];
                load_weight(p.w, c, w);
                if (p.b) load_n(p.b + c, b);
#pragma unroll
                for (int k = 0; k < VEC; ++k) w[k] = fmaf(v[j][k] * rs, w[k], p.b ? b[k] : 0.f);
                store_n(static_cast<TO *>(p.out) + row * p.so + c, w);
            }
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rs;
        }
    }
    if (RING) drain_copies(full, ring.stages, &lost, kWaitNs);
}

// VEC elements as loaded.
template <typename T, int VEC> struct RawGroup;
template <> struct RawGroup<float, 2> { using Type = uint2; };
template <> struct RawGroup<__half, 2> { using Type = uint32_t; };
template <> struct RawGroup<float, 4> { using Type = uint4; };
template <> struct RawGroup<__half, 4> { using Type = uint2; };
template <> struct RawGroup<__half, 8> { using Type = uint4; };

// The same for rows of 16-byte accesses, or of pairs, with the CTA's next row on its way in
// registers while this one's sums are made.  32 channels a thread: one or two
// warps for a row of 2048, whose barriers cost little.
template <typename TX, typename TO, int VEC, int NV>
__global__ void __launch_bounds__(512) layer_norm_ahead_kernel(const LayerNormParams p) {
    using Raw = typename RawGroup<TX, VEC>::Type;
    __shared__ float sm[64];
    int turn = 0;
    const float inv_cols = 1.f / (float)p.cols;
    Raw raw[NV];
    auto fetch = [&](int64_t row) {
        const TX *x = static_cast<const TX *>(p.x) + row * p.sx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) raw[j] = *reinterpret_cast<const Raw *>(x + c);
        }
    };
    fetch(blockIdx.x);  // grid <= rows
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        float v[NV][VEC];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                load_n(reinterpret_cast<const TX *>(&raw[j]), v[j]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) s += v[j][k];
            }
        }
        if (row + gridDim.x < p.rows) fetch(row + gridDim.x);
        const float mean = block_sum(s, sm, turn) * inv_cols;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v[j][k] -= mean;
                    ss = fmaf(v[j][k], v[j][k], ss);
                }
            }
        }
        const float rs = rsqrtf(block_sum(ss, sm, turn) * inv_cols + p.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < p.cols) {
                float w[VEC], b[VEC];
                load_weight(p.w, c, w);
                if (p.b) load_n(p.b + c, b);
#pragma unroll
                for (int k = 0; k < VEC; ++k) w[k] = fmaf(v[j][k] * rs, w[k], p.b ? b[k] : 0.f);
                store_n(static_cast<TO *>(p.out) + row * p.so + c, w);
            }
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rs;
        }
    }
}

// Backward: CTA k walks rows k, k + CTAs, ... and keeps the column sums of its
// rows in registers; they leave as one partial row per CTA.
template <typename TX, typename TO, int VEC, int NV, int MAXT, bool RING>
__global__ void __launch_bounds__(MAXT) layer_norm_bwd_kernel(const LayerNormGradParams p, const RingRow<2> ring) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kMaxStages];
    __shared__ LostCopies lost;
    __shared__ float2 sm[64];
    int turn = 0;
    const int cols = p.cols;
    const float inv_cols = 1.f / (float)cols;
    float acc_w[NV][VEC] = {}, acc_b[NV][VEC] = {};
    RingPlace at;
    if (RING) start_ring<2>(ring, smem, full, &lost, p.rows);
    float mean_next = p.mean[blockIdx.x], rs_next = p.rstd[blockIdx.x];  // grid <= rows
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const uint8_t *place = smem + at.s * ring.stage;
        auto at_place = [&](int k) { return place + ring.offset[k] + (VEC <= 2 ? ring.shift(k, row) : 0u); };
        const TX *x = RING ? reinterpret_cast<const TX *>(at_place(0)) : static_cast<const TX *>(p.x) + row * p.sx;
        const TO *g = RING ? reinterpret_cast<const TO *>(at_place(1)) : static_cast<const TO *>(p.dout) + row * p.sg;
        // this row's statistics were loaded a row ago, the next row's are on their way
        const float mean = mean_next, rs = rs_next;
        const int64_t after = row + gridDim.x;
        if (after < p.rows) {
            mean_next = p.mean[after];
            rs_next = p.rstd[after];
        }
        if (RING) await_row(full, at, &lost, &g_layer_norm_error);
        float n[NV][VEC], u[NV][VEC];
        float2 dot = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                load_n(x + c, n[j]);
                load_n(g + c, u[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
                float w[VEC];
                load_weight(p.w, c, w);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    n[j][k] = (n[j][k] - mean) * rs;
                    acc_w[j][k] = fmaf(u[j][k], n[j][k], acc_w[j][k]);
                    acc_b[j][k] += u[j][k];
                    u[j][k] *= w[k];
                    dot.x += u[j][k];
                    dot.y = fmaf(u[j][k], n[j][k], dot.y);
                }
            }
        }
        dot = block_sum2(dot, sm, turn);
        if (RING) {
            const int64_t ahead = row + (int64_t)ring.stages * gridDim.x;
            if (threadIdx.x == 0 && ahead < p.rows && !lost.flag) fetch_row<2>(ring, smem, full, ahead, at.s);
            at.step(ring.stages);
        }
        const float mean_u = dot.x * inv_cols, mean_un = dot.y * inv_cols;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            if (c < cols) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) u[j][k] = rs * (fmaf(-n[j][k], mean_un, u[j][k]) - mean_u);
                store_n(static_cast<TX *>(p.dx) + row * p.sdx + c, u[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + threadIdx.x) * VEC;
        if (c < cols) {
            if (p.part_w) store_n(p.part_w + (int64_t)blockIdx.x * cols + c, acc_w[j]);
            if (p.part_b) store_n(p.part_b + (int64_t)blockIdx.x * cols + c, acc_b[j]);
        }
    }
    if (RING) drain_copies(full, ring.stages, &lost, kWaitNs);
}

// Channels of a group with 16-byte accesses: 8 of FP16 rows, 4 where a row is
// FP32 (32 bytes a thread would leave half of each access's sectors, or banks,
// to the next).
template <typename TX, typename TO> constexpr int kGroup = sizeof(TX) + sizeof(TO) == 4 ? 8 : 4;

// Resident threads per SM of the ring kernels.  32768 x 2048 backward, FP32 to
// FP16 and FP16 to FP16, 16 channels a thread: 1536 threads 118 and 84 us, 1024
// 124 and 106; 8 channels a thread, 2048 threads 118 and 99, 1024 129; 32
// channels a thread, 768 threads 178 and 142.
constexpr int kLnThreads = 1024, kLnBwdThreads = 1536;
constexpr int kLnBwdChannels = 16;  // channels a thread of the backward ring
// Channels and resident threads per SM of the kernel that loads a row ahead.
// Forward, FP32 to FP16 and FP16 to FP16: 72 and 61 us (bytes alone 62 and 41); 768
// threads 88 and 73; 64 channels a thread 137 and 63; through the ring, 8 channels a
// thread, 95 and 92.
constexpr int kLnAheadChannels = 32, kLnAheadThreads = 1024;
constexpr int kLnSumThreads = 1024;

int ln_ctas(int threads, bool backward) {
    return backward ? std::min(16, ring_ctas(threads, kLnBwdThreads)) : ring_ctas(threads, kLnThreads);
}
// Rows of partial column sums of the backward pass at most.
int64_t ln_parts(int64_t rows, int cols) {
    const int ctas = ln_ctas(threads_for(cols, kLnBwdChannels), true);
    return std::min<int64_t>(rows, std::max(kDirectParts, 148 * ctas));
}

template <typename TX, typename TO, int NV>
int ring_ln(const LayerNormParams &p, const RingRow<1> &r, int ctas, int threads, cudaStream_t st) {
    auto kernel = layer_norm_kernel<TX, TO, 1, NV, 512, true>;
    if (allow_smem(kernel)) return -1;
    kernel<<<(unsigned)(ctas * device_sm_count()), threads, (size_t)r.stage * r.stages, st>>>(p, r);
    return launch_status("layer_norm kernel");
}
// How a call's rows can be accessed: 16 bytes at a time, in pairs of channels
// (every row of an even width), or one by one.
enum Access { kSingle, kPairs, kWide };

template <typename TX, typename TO, int V>
int launch_ln_groups(const LayerNormParams &p, cudaStream_t st) {
    if (p.rows >= 2 * device_sm_count()) {  // with fewer rows nothing is ahead
        const int threads = threads_for(p.cols, kLnAheadChannels);
        const int ctas = std::min(32, kLnAheadThreads / threads);
        const unsigned grid = (unsigned)std::min<int64_t>(p.rows, (int64_t)device_sm_count() * ctas);
        layer_norm_ahead_kernel<TX, TO, V, kLnAheadChannels / V><<<grid, threads, 0, st>>>(p);
    } else if (p.cols <= 4096) {
        layer_norm_kernel<TX, TO, V, 8 / V, 512, false>
            <<<(unsigned)p.rows, threads_for(p.cols, 8), 0, st>>>(p, RingRow<1>{});
    } else {
        layer_norm_kernel<TX, TO, V, 16 / V, 1024, false>
            <<<(unsigned)p.rows, threads_for(p.cols, 16), 0, st>>>(p, RingRow<1>{});
    }
    return launch_status("layer_norm kernel");
}
template <typename TX, typename TO>
int launch_ln(const LayerNormParams &p, Access access, cudaStream_t st) {
    if (access == kWide) return launch_ln_groups<TX, TO, kGroup<TX, TO>>(p, st);
    if (access == kPairs) return launch_ln_groups<TX, TO, 2>(p, st);
    RingRow<1> r{};
    if (p.cols <= 8192) {
        r.src[0] = p.x;
        r.stride[0] = p.sx * (int64_t)sizeof(TX);
        r.bytes[0] = (uint32_t)(p.cols * sizeof(TX));
        const bool one = p.cols <= 4096;
        const int threads = threads_for(p.cols, one ? 8 : 16);
        int ctas = ln_ctas(threads, false);
        if (plan_ring<1>(r, p.rows, ctas))
            return one ? ring_ln<TX, TO, 8>(p, r, ctas, threads, st) : ring_ln<TX, TO, 16>(p, r, ctas, threads, st);
    }
    const unsigned grid = (unsigned)std::min<int64_t>(p.rows, 0x7fffffff);
    if (p.cols <= 4096)
        layer_norm_kernel<TX, TO, 1, 4, 1024, false><<<grid, threads_for(p.cols, 4), 0, st>>>(p, r);
    else
        layer_norm_kernel<TX, TO, 1, 16, 1024, false><<<grid, threads_for(p.cols, 16), 0, st>>>(p, r);
    return launch_status("layer_norm kernel");
}

template <typename TX, typename TO, int VEC, int NV>
int ring_ln_bwd(const LayerNormGradParams &p, const RingRow<2> &r, unsigned grid, int threads, cudaStream_t st) {
    auto kernel = layer_norm_bwd_kernel<TX, TO, VEC, NV, 512, true>;
    if (allow_smem(kernel)) return -1;
    kernel<<<grid, threads, (size_t)r.stage * r.stages, st>>>(p, r);
    return launch_status("layer_norm_backward kernel");
}
// grid: CTAs to launch at most; set to those launched (rows of partial sums).
template <typename TX, typename TO>
int launch_ln_bwd(const LayerNormGradParams &p, Access access, unsigned &grid, cudaStream_t st) {
    constexpr int V = kGroup<TX, TO>;
    const int cols = p.cols;
    RingRow<2> r{};
    if (cols <= 8192) {
        r.src[0] = p.x;
        r.src[1] = p.dout;
        r.stride[0] = p.sx * (int64_t)sizeof(TX);
        r.stride[1] = p.sg * (int64_t)sizeof(TO);
        r.bytes[0] = (uint32_t)(cols * sizeof(TX));
        r.bytes[1] = (uint32_t)(cols * sizeof(TO));
        const int threads = threads_for(cols, kLnBwdChannels);
        int ctas = ln_ctas(threads, true);
        if (plan_ring<2>(r, p.rows, ctas)) {
            grid = std::min(grid, (unsigned)(ctas * device_sm_count()));
            if (access == kWide) return ring_ln_bwd<TX, TO, V, kLnBwdChannels / V>(p, r, grid, threads, st);
            if (access == kPairs) return ring_ln_bwd<TX, TO, 2, kLnBwdChannels / 2>(p, r, grid, threads, st);
            return ring_ln_bwd<TX, TO, 1, kLnBwdChannels>(p, r, grid, threads, st);
        }
    }
    grid = std::min(grid, (unsigned)kDirectParts);
    const int eight = threads_for(cols, 8), sixteen = threads_for(cols, 16);
    if (access == kWide && cols <= 4096)
        layer_norm_bwd_kernel<TX, TO, V, 8 / V, 512, false><<<grid, eight, 0, st>>>(p, r);
    else if (access == kWide)
        layer_norm_bwd_kernel<TX, TO, V, 16 / V, 1024, false><<<grid, sixteen, 0, st>>>(p, r);
    else if (access == kPairs && cols <= 4096)
        layer_norm_bwd_kernel<TX, TO, 2, 4, 512, false><<<grid, eight, 0, st>>>(p, r);
    else if (access == kPairs)
        layer_norm_bwd_kernel<TX, TO, 2, 8, 1024, false><<<grid, sixteen, 0, st>>>(p, r);
    else if (cols <= 4096)
        layer_norm_bwd_kernel<TX, TO, 1, 4, 1024, false><<<grid, threads_for(cols, 4), 0, st>>>(p, r);
    else
        layer_norm_bwd_kernel<TX, TO, 1, 16, 1024, false><<<grid, sixteen, 0, st>>>(p, r);
    return launch_status("layer_norm_backward kernel");
}

bool float_dtype(int dt) { return dt == MAMBA_F32 || dt == MAMBA_F16; }
// Every row starts on a boundary of `bytes`.
bool aligned_rows(const void *p, int64_t stride, int dtype, int64_t bytes) {
    return aligned_to(p, (size_t)bytes) && (stride * (int64_t)dtype_size(dtype)) % bytes == 0;
}
bool pair_rows(const void *p, int64_t stride, int dtype) {
    return aligned_rows(p, stride, dtype, 2 * (int64_t)dtype_size(dtype));
}

int check_ln(const MambaLayerNormArgs *a, const std::string &what) {
    MB_CHECK_ARG(a, what + ": null args");
    MB_CHECK_ARG(a->rows >= 0 && a->cols >= 0, what + ": negative size");
    MB_CHECK_ARG(float_dtype(a->x_dtype) && float_dtype(a->out_dtype), what + ": bad dtype");
    MB_CHECK_ARG(a->cols <= kMaxCols, what + ": more than 16384 channels");
    if (a->rows == 0 || a->cols == 0) return 0;
    MB_CHECK_ARG(a->x, what + ": null pointer");
    MB_CHECK_ARG(aligned_to(a->x, dtype_size(a->x_dtype)) && aligned_to(a->w, 4) && aligned_to(a->b, 4) &&
                     aligned_to(a->mean, 4) && aligned_to(a->rstd, 4),
                 what + ": pointers must be aligned to their element type");
    return 0;
}

}  // namespace

int layer_norm(const MambaLayerNormArgs *a, cudaStream_t st) {
    if (check_ln(a, "layer_norm")) return -1;
    MB_CHECK_ARG(a->eps > 0.f && a->eps <= 3.0e38f, "layer_norm: eps must be positive and finite");
    if (a->rows == 0 || a->cols == 0) return 0;
    MB_CHECK_ARG(a->out, "layer_norm: null pointer");
    MB_CHECK_ARG(aligned_to(a->out, dtype_size(a->out_dtype)),
                 "layer_norm: pointers must be aligned to their element type");
    MB_CHECK_ARG(a->out != a->x, "layer_norm: out needs memory of its own");
    MB_CHECK_ARG(a->rows == 1 || a->out_stride >= a->cols, "layer_norm: rows of out overlap (strides)");
    LayerNormParams p{};
    p.x = a->x;
    p.w = a->w;
    p.b = a->b;
    p.out = a->out;
    p.mean = a->mean;
    p.rstd = a->rstd;
    p.rows = a->rows;
    p.cols = a->cols;
    p.eps = a->eps;
    p.sx = a->x_stride;
    p.so = a->out_stride;
    Access access = kSingle;
    if (a->cols % 8 == 0 && aligned_rows(a->x, a->x_stride, a->x_dtype, 16) &&
        aligned_rows(a->out, a->out_stride, a->out_dtype, 16) && aligned_to(a->w, 16) && aligned_to(a->b, 16))
        access = kWide;
    else if (a->cols % 2 == 0 && pair_rows(a->x, a->x_stride, a->x_dtype) &&
             pair_rows(a->out, a->out_stride, a->out_dtype) && aligned_to(a->w, 8) && aligned_to(a->b, 8))
        access = kPairs;
    if (a->x_dtype == MAMBA_F16)
        return a->out_dtype == MAMBA_F16 ? launch_ln<__half, __half>(p, access, st) : launch_ln<__half, float>(p, access, st);
    return a->out_dtype == MAMBA_F16 ? launch_ln<float, __half>(p, access, st) : launch_ln<float, float>(p, access, st);
}

size_t layer_norm_workspace_bytes(const MambaLayerNormArgs *a) {
    if (!a || a->rows <= 0 || a->cols <= 0 || a->cols > kMaxCols) return 0;
    // two sets of partial rows, each starting on a 16-byte boundary
    return 2 * (((size_t)ln_parts(a->rows, a->cols) * a->cols + 3) / 4 * 4) * sizeof(float);
}

int layer_norm_backward(const MambaLayerNormArgs *a, const MambaLayerNormGrads *g, void *ws, size_t ws_bytes,
                        cudaStream_t st) {
    if (check_ln(a, "layer_norm_backward")) return -1;
    MB_CHECK_ARG(g, "layer_norm_backward: null gradients");
    if (a->cols == 0) return 0;
    MB_CHECK_ARG(aligned_to(g->dw, 4) && aligned_to(g->db, 4),
                 "layer_norm_backward: pointers must be aligned to their element type");
    if (a->rows == 0) {
        if (g->dw) MB_CUDA_TRY(cudaMemsetAsync(g->dw, 0, (size_t)a->cols * 4, st));
        if (g->db) MB_CUDA_TRY(cudaMemsetAsync(g->db, 0, (size_t)a->cols * 4, st));
        return 0;
    }
    MB_CHECK_ARG(a->mean && a->rstd && g->dout && g->dx, "layer_norm_backward: null pointer");
    MB_CHECK_ARG(aligned_to(g->dout, dtype_size(a->out_dtype)) && aligned_to(g->dx, dtype_size(a->x_dtype)),
                 "layer_norm_backward: pointers must be aligned to their element type");
    MB_CHECK_ARG(g->dx != a->x && g->dx != g->dout, "layer_norm_backward: dx needs memory of its own");
    MB_CHECK_ARG(!g->dw || g->dw != g->db, "layer_norm_backward: dw and db need memory of their own");
    MB_CHECK_ARG(a->rows == 1 || g->dx_stride >= a->cols, "layer_norm_backward: rows of dx overlap (strides)");
    MB_CHECK_ARG(ws && ws_bytes >= layer_norm_workspace_bytes(a) && aligned_to(ws, 16),
                 "layer_norm_backward: workspace too small or not 16-byte aligned");
    unsigned grid = (unsigned)ln_parts(a->rows, a->cols);  // launch_ln_bwd may take fewer
    LayerNormGradParams p{};
    p.dout = g->dout;
    p.x = a->x;
    p.w = a->w;
    p.mean = a->mean;
    p.rstd = a->rstd;
    p.dx = g->dx;
    p.rows = a->rows;
    p.cols = a->cols;
    p.sg = g->dout_stride;
    p.sx = a->x_stride;
    p.sdx = g->dx_stride;
    float *part = static_cast<float *>(ws);
    if (g->dw) p.part_w = part;
    if (g->db) p.part_b = part + ((int64_t)grid * a->cols + 3) / 4 * 4;  // grid is still the most
    Access access = kSingle;
    if (a->cols % 8 == 0 && aligned_rows(a->x, a->x_stride, a->x_dtype, 16) &&
        aligned_rows(g->dout, g->dout_stride, a->out_dtype, 16) && aligned_rows(g->dx, g->dx_stride, a->x_dtype, 16) &&
        aligned_to(a->w, 16))
        access = kWide;
    else if (a->cols % 2 == 0 && pair_rows(a->x, a->x_stride, a->x_dtype) &&
             pair_rows(g->dout, g->dout_stride, a->out_dtype) && pair_rows(g->dx, g->dx_stride, a->x_dtype) &&
             aligned_to(a->w, 8))
        access = kPairs;
    int rc;
    if (a->x_dtype == MAMBA_F16)
        rc = a->out_dtype == MAMBA_F16 ? launch_ln_bwd<__half, __half>(p, access, grid, st)
                                       : launch_ln_bwd<__half, float>(p, access, grid, st);
    else
        rc = a->out_dtype == MAMBA_F16 ? launch_ln_bwd<float, __half>(p, access, grid, st)
                                       : launch_ln_bwd<float, float>(p, access, grid, st);
    if (rc) return -1;
    if (!g->dw && !g->db) return 0;
    column_sum_kernel<kLnSumThreads><<<dim3((unsigned)ceil_div(a->cols, 32), 2), kLnSumThreads, 0, st>>>(
        p.part_w, p.part_b, g->dw, g->db, (int)grid, a->cols);
    return launch_status("layer_norm_backward sum kernel");
}

namespace {

// A wait for a row that nothing fetches, through the kernels' own helpers.
__global__ void layer_norm_wait_selftest_kernel(uint64_t limit_ns) {
    __shared__ uint64_t full;
    __shared__ LostCopies lost;
    if (threadIdx.x != 0) return;
    lost = LostCopies{};
    mbar_init(&full, 1);
    fence_mbar_init();
    await_row(&full, RingPlace{}, &lost, &g_layer_norm_error, limit_ns);
    drain_copies(&full, 1, &lost, limit_ns);
}

}  // namespace

int layer_norm_wait_selftest(uint64_t limit_ns, cudaStream_t st) {
    layer_norm_wait_selftest_kernel<<<1, 32, 0, st>>>(limit_ns);
    return launch_status("layer_norm wait self-test kernel");
}

unsigned layer_norm_error_flags(bool clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_layer_norm_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (clear && v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_layer_norm_error, &z, sizeof(z));
    }
    return v;
}

}  // namespace mb
