// dropout.cu -- dropout from a counter-based generator, with an optional
// residual add:
//   out[i] = [residual[i] +] (word(i) >= p 2^32 ? x[i] / (1 - p) : 0)
// where i = row * cols + col and word(i) is number i % 4 of the Philox4x32-10
// block (J. K. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011) with counter (i / 4, offset) and key seed.  The mask is a function
// of (seed, offset, i), so the backward pass is the same map on the gradient
// and nothing is stored.
//
// Bound by bytes.  A block of four numbers costs 20 wide products and 20
// three-input exclusive ors, 10 integer operations per element against 22 that
// fit in the time of an FP16 element's 4 bytes.
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace mb {
namespace {

struct DropoutParams {
    const void *x;
    const float *res;
    void *out;
    const uint64_t *state;  // {seed, offset} or NULL
    uint64_t seed, offset;
    int64_t rows, cols, sx, sr, so;
    uint32_t threshold;
    float scale;
};

__device__ __forceinline__ uint4 philox(uint64_t counter, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)offset,
             c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

constexpr int kDropThreads = 256;
constexpr int kDropVec = 8, kDropUnroll = 2;  // elements of a group, groups a thread has in flight

// Groups of 8 elements within a row (a contiguous tensor counts as one row): 32768
// x 2048 FP16 with the FP32 residual 112 us, with groups of 4 (16 bytes of out) 116.
template <typename TX, typename TO, bool NONE>
__global__ void __launch_bounds__(kDropThreads) dropout_vec_kernel(const DropoutParams p) {
    constexpr int VEC = kDropVec;
    const uint64_t seed = p.state ? p.state[0] : p.seed, offset = p.offset + (p.state ? p.state[1] : 0);
    const int64_t per_row = p.cols / VEC, groups = p.rows * per_row;
    int64_t g = (int64_t)blockIdx.x * (kDropThreads * kDropUnroll) + threadIdx.x;
    float v[kDropUnroll][VEC], r[kDropUnroll][VEC];
    int64_t row[kDropUnroll], col[kDropUnroll];
#pragma unroll
    for (int u = 0; u < kDropUnroll; ++u) {
        const int64_t at = g + u * kDropThreads;
        if (at < groups) {
            row[u] = p.rows == 1 ? 0 : at / per_row;
            col[u] = (at - row[u] * per_row) * VEC;
            load_n(static_cast<const TX *>(p.x) + row[u] * p.sx + col[u], v[u]);
            if (p.res) load_n(p.res + row[u] * p.sr + col[u], r[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < kDropUnroll; ++u) {
        const int64_t at = g + u * kDropThreads;
        if (at < groups) {
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                const uint4 w = philox((uint64_t)at * (VEC / 4) + h, offset, seed);
                const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float &e = v[u][4 * h + k];
                    const bool keep = !NONE && word[k] >= p.threshold;
                    const float add = p.res ? r[u][4 * h + k] : 0.f;
                    e = keep ? (p.res ? fmaf(e, p.scale, add) : e * p.scale) : add;
                }
            }
            store_n(static_cast<TO *>(p.out) + row[u] * p.so + col[u], v[u]);
        }
    }
    // the end of a single row, behind its last whole group
    const int64_t i = per_row * VEC + threadIdx.x;
    if (p.rows == 1 && blockIdx.x == 0 && i < p.cols) {
        const uint4 w = philox((uint64_t)i / 4, offset, seed);
        const uint32_t word = i & 2 ? (i & 1 ? w.w : w.z) : (i & 1 ? w.y : w.x);
        const float e = ld_f32(static_cast<const TX *>(p.x) + i), add = p.res ? p.res[i] : 0.f;
        const bool keep = !NONE && word >= p.threshold;
        static_cast<TO *>(p.out)[i] = cvt_out<TO>(keep ? (p.res ? fmaf(e, p.scale, add) : e * p.scale) : add);
    }
}

// Any sizes, strides and alignment: one block of four numbers per thread.
template <typename TX, typename TO, bool NONE>
__global__ void __launch_bounds__(kDropThreads) dropout_any_kernel(const DropoutParams p) {
    const uint64_t seed = p.state ? p.state[0] : p.seed, offset = p.offset + (p.state ? p.state[1] : 0);
    const int64_t n = p.rows * p.cols, g = (int64_t)blockIdx.x * kDropThreads + threadIdx.x;
    if (4 * g >= n) return;
    const uint4 w = philox((uint64_t)g, offset, seed);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    int64_t row = p.rows == 1 ? 0 : 4 * g / p.cols, col = 4 * g - row * p.cols;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (4 * g + k < n) {
            const float e = ld_f32(static_cast<const TX *>(p.x) + row * p.sx + col);
            const bool keep = !NONE && word[k] >= p.threshold;
            const float add = p.res ? p.res[row * p.sr + col] : 0.f;
            static_cast<TO *>(p.out)[row * p.so + col] =
                cvt_out<TO>(keep ? (p.res ? fmaf(e, p.scale, add) : e * p.scale) : add);
        }
        if (++col == p.cols) {
            col = 0;
            ++row;
        }
    }
}

template <typename TX, typename TO, bool NONE>
int launch_dropout(const DropoutParams &p, bool vec, cudaStream_t st) {
    const int64_t n = p.rows * p.cols;
    const int64_t ctas = ceil_div64(n, vec ? kDropVec * kDropUnroll * kDropThreads : 4 * kDropThreads);
    MB_CHECK_ARG(ctas <= 0x7fffffff, "dropout: too many elements");
    if (vec)
        dropout_vec_kernel<TX, TO, NONE><<<(unsigned)ctas, kDropThreads, 0, st>>>(p);
    else
        dropout_any_kernel<TX, TO, NONE><<<(unsigned)ctas, kDropThreads, 0, st>>>(p);
    return launch_status("dropout kernel");
}
template <typename TX, typename TO>
int launch_dropout(const DropoutParams &p, bool vec, bool none, cudaStream_t st) {
    return none ? launch_dropout<TX, TO, true>(p, vec, st) : launch_dropout<TX, TO, false>(p, vec, st);
}

}  // namespace

int dropout(const MambaDropoutArgs *a, cudaStream_t st) {
    MB_CHECK_ARG(a, "dropout: null args");
    MB_CHECK_ARG(a->rows >= 0 && a->cols >= 0, "dropout: negative size");
    MB_CHECK_ARG((a->x_dtype == MAMBA_F32 || a->x_dtype == MAMBA_F16) &&
                     (a->out_dtype == MAMBA_F32 || a->out_dtype == MAMBA_F16),
                 "dropout: bad dtype");
    MB_CHECK_ARG(a->p >= 0.f && a->p <= 1.f, "dropout: p must lie between 0 and 1");
    if (a->rows == 0 || a->cols == 0) return 0;
    MB_CHECK_ARG(a->rows <= (int64_t)1 << 40 && a->cols <= (int64_t)1 << 40 && a->rows <= ((int64_t)1 << 40) / a->cols,
                 "dropout: too many elements");
    MB_CHECK_ARG(a->x && a->out, "dropout: null pointer");
    const size_t ex = dtype_size(a->x_dtype), eo = dtype_size(a->out_dtype);
    MB_CHECK_ARG(aligned_to(a->x, ex) && aligned_to(a->out, eo) && aligned_to(a->residual, 4) && aligned_to(a->state, 8),
                 "dropout: pointers must be aligned to their element type");
    MB_CHECK_ARG(a->rows == 1 || a->out_stride >= a->cols, "dropout: rows of out overlap (strides)");
    MB_CHECK_ARG(a->out != a->x || (ex == eo && (a->rows == 1 || a->x_stride == a->out_stride)),
                 "dropout: out may be x only in x's type and strides");
    MB_CHECK_ARG(static_cast<const void *>(a->residual) != a->out ||
                     (eo == 4 && (a->rows == 1 || a->residual_stride == a->out_stride)),
                 "dropout: out may be residual only as FP32 of its strides");
    DropoutParams p{};
    p.x = a->x;
    p.res = a->residual;
    p.out = a->out;
    p.state = a->state;
    p.seed = a->seed;
    p.offset = a->offset;
    p.rows = a->rows;
    p.cols = a->cols;
    p.sx = a->x_stride;
    p.sr = a->residual_stride;
    p.so = a->out_stride;
    // p 2^32 to the nearest whole number (p = 1: every element is dropped)
    const double share = (double)a->p, border = nearbyint(share * 4294967296.0);
    const bool none = border >= 4294967296.0;
    p.threshold = none ? 0u : (uint32_t)border;
    p.scale = none ? 0.f : (float)(1.0 / (1.0 - share));
    if (p.rows > 1 && p.sx == p.cols && p.so == p.cols && (!p.res || p.sr == p.cols)) {
        p.cols *= p.rows;
        p.rows = 1;
    }
    // single rows may end anywhere
    const bool vec = (p.cols % 8 == 0 || p.rows == 1) && aligned_to(p.x, 16) && aligned_to(p.out, 16) && aligned_to(p.res, 16) &&
                     (p.rows == 1 || ((p.sx * (int64_t)ex) % 16 == 0 && (p.so * (int64_t)eo) % 16 == 0 &&
                                      (!p.res || p.sr % 4 == 0)));
    if (a->x_dtype == MAMBA_F16)
        return a->out_dtype == MAMBA_F16 ? launch_dropout<__half, __half>(p, vec, none, st)
                                         : launch_dropout<__half, float>(p, vec, none, st);
    return a->out_dtype == MAMBA_F16 ? launch_dropout<float, __half>(p, vec, none, st)
                                     : launch_dropout<float, float>(p, vec, none, st);
}

}  // namespace mb
