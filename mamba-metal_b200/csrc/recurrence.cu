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

namespace mb {

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
    float *dlambda, *dh0, *part;
    int64_t sdh[2], sdx[2], sdr[2], sdi[2];
};

__device__ __forceinline__ int row_length(const FwdParams &p, int b) {
    return p.lengths ? min(max(p.lengths[b], 0), p.L) : p.L;
}

constexpr int kThreads = 128;

// One thread per (row, channel), walking time.
template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_fwd_kernel(const FwdParams p) {
    constexpr bool PRECISE = sizeof(T) == 4;
    const int d = blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
    if (d >= p.D) return;
    const int n = row_length(p, b);
    const float csp = p.c * softplus_channel(p.lambda[d]);
    const T *x = static_cast<const T *>(p.x) + b * p.sx[0] + d;
    const T *r = static_cast<const T *>(p.r) + b * p.sr[0] + d;
    const T *gi = static_cast<const T *>(p.i) + b * p.si[0] + d;
    T *ho = static_cast<T *>(p.h) + b * p.sh[0] + d;
    float h = p.h0 ? p.h0[(int64_t)b * p.D + d] : 0.f;
    for (int t = 0; t < n; ++t) {
        const Decay g = decay<PRECISE>(ld_f32(r + t * p.sr[1]), csp);
        float si, om;
        sigmoid2<PRECISE>(ld_f32(gi + t * p.si[1]), si, om);
        const float bt = sqrt_gate<PRECISE>(one_minus_a2<PRECISE>(g.y, g.a)) * si * ld_f32(x + t * p.sx[1]);
        if (p.resets && p.resets[(int64_t)b * p.L + t]) h = 0.f;
        h = fmaf(g.a, h, bt);
        ho[t * p.sh[1]] = cvt_out<T>(h);
    }
    if (p.hN) p.hN[(int64_t)b * p.D + d] = h;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_bwd_kernel(const BwdParams p) {
    constexpr bool PRECISE = sizeof(T) == 4;
    const FwdParams &f = p.f;
    const int d = blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
    if (d >= f.D) return;
    const int n = row_length(f, b);
    const float csp = f.c * softplus_channel(f.lambda[d]);
    const T *x = static_cast<const T *>(f.x) + b * f.sx[0] + d;
    const T *r = static_cast<const T *>(f.r) + b * f.sr[0] + d;
    const T *gi = static_cast<const T *>(f.i) + b * f.si[0] + d;
    const T *h = static_cast<const T *>(f.h) + b * f.sh[0] + d;
    const T *dh = static_cast<const T *>(p.dh) + b * p.sdh[0] + d;
    T *dx = static_cast<T *>(p.dx) + b * p.sdx[0] + d;
    T *dr = static_cast<T *>(p.dr) + b * p.sdr[0] + d;
    T *di = static_cast<T *>(p.di) + b * p.sdi[0] + d;
    float C = p.dhN ? p.dhN[(int64_t)b * f.D + d] : 0.f, sum = 0.f;
    for (int t = n - 1; t >= 0; --t) {
        const Decay g = decay<PRECISE>(ld_f32(r + t * f.sr[1]), csp);
        float si, om;
        sigmoid2<PRECISE>(ld_f32(gi + t * f.si[1]), si, om);
        const float m = one_minus_a2<PRECISE>(g.y, g.a), beta = sqrt_gate<PRECISE>(m);
        const float q = beta > 1e-18f ? g.y / beta : 0.f;
        const bool keep = !(f.resets && f.resets[(int64_t)b * f.L + t]);
        float prev = t ? ld_f32(h + (t - 1) * f.sh[1]) : (f.h0 ? f.h0[(int64_t)b * f.D + d] : 0.f);
        if (!keep) prev = 0.f;
        const float G = ld_f32(dh + t * p.sdh[1]) + C, xv = ld_f32(x + t * f.sx[1]);
        const float gx = G * beta * si;
        const float E = G * (si * xv * g.a * g.a * q - g.y * g.a * prev);
        dx[t * p.sdx[1]] = cvt_out<T>(gx);
        di[t * p.sdi[1]] = cvt_out<T>(gx * xv * om);
        dr[t * p.sdr[1]] = cvt_out<T>(E * g.om);
        sum += E;
        C = keep ? g.a * G : 0.f;
    }
    if (p.dh0) p.dh0[(int64_t)b * f.D + d] = C;
    p.part[(int64_t)b * f.D + d] = sum;
}

// dlambda[d] = sigmoid(lambda)/softplus(lambda) * sum of the partial sums of
// E, added in row order.  The quotient tends to 1 for very negative lambda.
__global__ void __launch_bounds__(kThreads)
    recurrence_dlambda_kernel(const float *__restrict__ part, const float *__restrict__ lambda,
                              float *__restrict__ dlambda, int64_t rows, int D) {
    const int d = blockIdx.x * kThreads + threadIdx.x;
    if (d >= D) return;
    float s = 0.f;
    for (int64_t k = 0; k < rows; ++k) s += part[k * D + d];
    float sg, om;
    const float l = lambda[d];
    sigmoid2<true>(l, sg, om);
    dlambda[d] = s * (l < -20.f ? 1.f : sg / softplus_channel(l));
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

}  // namespace

size_t recurrence_workspace_bytes(const MambaRecurrenceArgs *a, bool backward) {
    if (!a || a->batch <= 0 || a->seqlen < 0 || a->dim <= 0 || !backward) return 0;
    return (size_t)a->batch * a->dim * sizeof(float);
}

int recurrence_forward(const MambaRecurrenceArgs *a, void *ws, size_t ws_bytes, cudaStream_t st) {
    if (check_args(a, false)) return -1;
    if (a->batch == 0 || a->dim == 0) return 0;
    const FwdParams p = fwd_params(a);
    const dim3 grid((unsigned)ceil_div(a->dim, kThreads), (unsigned)a->batch);
    if (a->dtype == MAMBA_F16)
        recurrence_fwd_kernel<__half><<<grid, kThreads, 0, st>>>(p);
    else
        recurrence_fwd_kernel<float><<<grid, kThreads, 0, st>>>(p);
    return launch_status("gated_recurrence kernel");
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
    MB_CHECK_ARG(ws && ws_bytes >= recurrence_workspace_bytes(a, true) && aligned_to(ws, 16),
                 "gated_recurrence_backward: workspace too small or not 16-byte aligned");
    BwdParams p{};
    p.f = fwd_params(a);
    p.dh = g->dh;
    p.dhN = g->dfinal_state;
    p.dx = g->dx;
    p.dr = g->dr;
    p.di = g->di;
    p.dlambda = g->dlambda;
    p.dh0 = g->dinitial_state;
    p.part = static_cast<float *>(ws);
    for (int k = 0; k < 2; ++k) {
        p.sdh[k] = g->dh_stride[k];
        p.sdx[k] = g->dx_stride[k];
        p.sdr[k] = g->dr_stride[k];
        p.sdi[k] = g->di_stride[k];
    }
    const dim3 grid((unsigned)ceil_div(a->dim, kThreads), (unsigned)a->batch);
    if (a->dtype == MAMBA_F16)
        recurrence_bwd_kernel<__half><<<grid, kThreads, 0, st>>>(p);
    else
        recurrence_bwd_kernel<float><<<grid, kThreads, 0, st>>>(p);
    if (launch_status("gated_recurrence_backward kernel")) return -1;
    recurrence_dlambda_kernel<<<(unsigned)ceil_div(a->dim, kThreads), kThreads, 0, st>>>(p.part, a->lambda,
                                                                                          g->dlambda, a->batch, a->dim);
    return launch_status("gated_recurrence_backward sum kernel");
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
