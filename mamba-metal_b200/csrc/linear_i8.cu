// linear_i8.cu -- linear layer in 8-bit integers, for serving: activations
// quantised per token, weights per output channel, both symmetric.
//   quantise:  scale[t] = max|x[t]| / 127,  q = round(x / scale) (half to even)
//   product:   y[t, n] = x_scale[t] w_scale[n] sum_k xq[t, k] wq[n, k] + bias[n]
// The sums are exact 32-bit integers (k <= 131071: 128 * 128 * 131071 < 2^31),
// so the result does not depend on how K is split.
#include "common.cuh"
#include "internal.h"

#include <algorithm>

namespace mb {

namespace {

// ---- row quantiser ----------------------------------------------------------
constexpr int kQThreads = 256;
constexpr int kQRegs = 4;  // groups of VEC channels cached per thread

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

// round(x / s) with ties to even, of the exact quotient: the product with the
// reciprocal may land on the wrong side of a half, so the remainder
// d = x - k s, which fma gives exactly here (|d| <= s/2 (1 + 2^-16) is a
// multiple of half of s's last place), decides.  For scales below 2^-100, whose
// reciprocal or half may not be a normal number, the quotient is divided out;
// it is then compared the same way.
__device__ __forceinline__ int quantise(float x, float s, float inv, bool tiny) {
    if (tiny) {
        const double q = (double)x / (double)s;  // exact to 2^-53: decides every tie of 24-bit operands
        return max(-127, min(127, __double2int_rn(q)));
    }
    const float k = rintf(x * inv);
    const float d = fmaf(-k, s, x), half = 0.5f * s;
    int q = (int)k;
    if (fabsf(d) >= half) {
        const bool tie = fabsf(d) == half;
        if (!tie || (q & 1)) q += d > 0.f ? 1 : -1;
    }
    return max(-127, min(127, q));
}

template <typename T, int VEC, int TPR>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ q, int64_t ldq,
                         float *__restrict__ scale, int64_t rows, int cols) {
    __shared__ uint32_t sm[kQThreads / 32];
    const int tid = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kQThreads / TPR) + threadIdx.x / TPR;
    if (TPR == 32 && row >= rows) return;  // TPR 256: one row per CTA, always inside
    const T *xr = x + row * ldx;
    int8_t *qr = q + row * ldq;
    float v[kQRegs][VEC];
    uint32_t m = 0;  // largest |x| as bits: ordered like the values, infinity and NaN above all numbers
#pragma unroll
    for (int j = 0; j < kQRegs; ++j) {
        const int64_t c = (int64_t)(j * TPR + tid) * VEC;
        if (c < cols) {
            load_n(xr + c, v[j]);
#pragma unroll
            for (int k = 0; k < VEC; ++k) m = max(m, __float_as_uint(v[j][k]) & 0x7fffffffu);
        }
    }
    for (int64_t c = (int64_t)(kQRegs * TPR + tid) * VEC; c < cols; c += TPR * VEC) {
        float u[VEC];
        load_n(xr + c, u);
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = max(m, __float_as_uint(u[k]) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kQThreads / 32; ++k) m = max(m, sm[k]);
    }
    const bool bad = m >= 0x7f800000u;  // an infinity or NaN in the row: scale NaN, q 0
    const float s = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(m), 127.f);
    const bool zero = bad || s == 0.f, tiny = s < 7.9e-31f;
    const float inv = zero ? 0.f : __fdiv_rn(1.f, s);
    if (tid == 0) scale[row] = s;
    auto emit = [&](int64_t c, const float (&u)[VEC]) {
        int r[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) r[k] = zero ? 0 : quantise(u[k], s, inv, tiny);
        if constexpr (VEC == 1) {
            qr[c] = (int8_t)r[0];
        } else {
            uint32_t w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                w[h] = (r[4 * h] & 0xff) | (r[4 * h + 1] & 0xff) << 8 | (r[4 * h + 2] & 0xff) << 16 |
                       (uint32_t)r[4 * h + 3] << 24;
            *reinterpret_cast<uint2 *>(qr + c) = make_uint2(w[0], w[1]);
        }
    };
#pragma unroll
    for (int j = 0; j < kQRegs; ++j) {
        const int64_t c = (int64_t)(j * TPR + tid) * VEC;
        if (c < cols) emit(c, v[j]);
    }
    for (int64_t c = (int64_t)(kQRegs * TPR + tid) * VEC; c < cols; c += TPR * VEC) {
        float u[VEC];
        load_n(xr + c, u);
        emit(c, u);
    }
}

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T, int VEC>
int launch_quantize(const T *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int cols,
                    cudaStream_t st) {
    if (cols <= 32 * VEC * kQRegs && rows > 4LL * device_sm_count()) {
        const int64_t grid = ceil_div64(rows, kQThreads / 32);
        MB_CHECK_ARG(grid <= 0x7fffffffLL, "quantize_rows: too many rows");
        quantize_rows_kernel<T, VEC, 32><<<(unsigned)grid, kQThreads, 0, st>>>(x, ldx, q, ldq, scale, rows, cols);
    } else {
        MB_CHECK_ARG(rows <= 0x7fffffffLL, "quantize_rows: too many rows");
        quantize_rows_kernel<T, VEC, kQThreads><<<(unsigned)rows, kQThreads, 0, st>>>(x, ldx, q, ldq, scale, rows,
                                                                                      cols);
    }
    return launch_status("quantize_rows kernel");
}

// ---- product ------------------------------------------------------------------
struct I8Params {
    const int8_t *x, *w;
    const float *xs, *ws, *bias;
    void *y;
    int64_t ldx, ldw, ldy, rows;
    int n, k, mode;
};

__device__ __forceinline__ void emit_i8(const I8Params &p, int64_t t, int n, int acc) {
    float v = (float)acc * p.xs[t] * p.ws[n];
    if (p.bias) v += p.bias[n];
    if (p.mode == 0)
        static_cast<__half *>(p.y)[t * p.ldy + n] = __float2half_rn(v);
    else if (p.mode == 1)
        static_cast<float *>(p.y)[t * p.ldy + n] += v;
    else
        static_cast<float *>(p.y)[t * p.ldy + n] = v;
}

// Any strides and alignment: 64 x 64 outputs per CTA, 64 bytes of K staged at
// a time by single bytes, 4 x 4 outputs per thread by dp4a.
constexpr int kDT = 64, kDPitch = 68;
__global__ void __launch_bounds__(256) linear_i8_dp4a_kernel(const I8Params p) {
    __shared__ __align__(16) int8_t sx[kDT][kDPitch], sw[kDT][kDPitch];
    const int64_t t0 = (int64_t)blockIdx.y * kDT;
    const int n0 = blockIdx.x * kDT, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 64) {
        for (int e = threadIdx.x; e < kDT * 64; e += 256) {
            const int r = e >> 6, c = e & 63;
            const bool in = k0 + c < p.k;
            sx[r][c] = in && t0 + r < p.rows ? p.x[(t0 + r) * p.ldx + k0 + c] : (int8_t)0;
            sw[r][c] = in && n0 + r < p.n ? p.w[(int64_t)(n0 + r) * p.ldw + k0 + c] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
            int a[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[j] = *reinterpret_cast<const int *>(&sx[ty + 16 * j][c]);
                b[j] = *reinterpret_cast<const int *>(&sw[tx + 16 * j][c]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t t = t0 + ty + 16 * i;
            const int n = n0 + tx + 16 * j;
            if (t < p.rows && n < p.n) emit_i8(p, t, n, acc[i][j]);
        }
}

}  // namespace

int quantize_rows(const void *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int cols, int dtype,
                  cudaStream_t st) {
    MB_CHECK_ARG(rows >= 0 && cols >= 0, "quantize_rows: negative size");
    MB_CHECK_ARG(dtype == MAMBA_F32 || dtype == MAMBA_F16, "quantize_rows: bad dtype");
    if (rows == 0) return 0;
    MB_CHECK_ARG(scale && aligned_to(scale, 4) && (cols == 0 || (x && q)), "quantize_rows: null pointer");
    MB_CHECK_ARG(aligned_to(x, dtype_size(dtype)), "quantize_rows: pointers must be aligned to their element type");
    MB_CHECK_ARG(rows == 1 || ldq >= cols, "quantize_rows: rows of q overlap (stride)");
    const bool vec = cols % 8 == 0 && aligned_to(x, 16) && (ldx * (int64_t)dtype_size(dtype)) % 16 == 0 &&
                     aligned_to(q, 8) && ldq % 8 == 0;
    if (dtype == MAMBA_F16) {
        auto *p = static_cast<const __half *>(x);
        return vec ? launch_quantize<__half, 8>(p, ldx, q, ldq, scale, rows, cols, st)
                   : launch_quantize<__half, 1>(p, ldx, q, ldq, scale, rows, cols, st);
    }
    auto *p = static_cast<const float *>(x);
    return vec ? launch_quantize<float, 8>(p, ldx, q, ldq, scale, rows, cols, st)
               : launch_quantize<float, 1>(p, ldx, q, ldq, scale, rows, cols, st);
}

int linear_i8(const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w, int64_t ldw, const float *w_scale,
              const float *bias, void *y, int64_t ldy, int64_t rows, int n, int k, int mode, cudaStream_t st) {
    MB_CHECK_ARG(rows >= 0 && n >= 0 && k >= 0, "linear_i8: negative size");
    MB_CHECK_ARG(mode >= 0 && mode <= 2, "linear_i8: bad epilogue mode");
    MB_CHECK_ARG(k <= 131071, "linear_i8: k above 131071 could overflow the 32-bit sums");
    if (rows == 0 || n == 0) return 0;
    MB_CHECK_ARG(x_scale && w_scale && y && (k == 0 || (x && w)), "linear_i8: null pointer");
    MB_CHECK_ARG(aligned_to(x_scale, 4) && aligned_to(w_scale, 4) && aligned_to(bias, 4) &&
                     aligned_to(y, mode == 0 ? 2 : 4),
                 "linear_i8: pointers must be aligned to their element type");
    MB_CHECK_ARG((rows == 1 || (ldx >= k && ldy >= n)) && (n == 1 || ldw >= k), "linear_i8: a row stride is below its row");
    MB_CHECK_ARG(rows <= 65535LL * kDT, "linear_i8: too many rows");
    I8Params p{};
    p.x = x;
    p.w = w;
    p.xs = x_scale;
    p.ws = w_scale;
    p.bias = bias;
    p.y = y;
    p.ldx = ldx;
    p.ldw = ldw;
    p.ldy = ldy;
    p.rows = rows;
    p.n = n;
    p.k = k;
    p.mode = mode;
    linear_i8_dp4a_kernel<<<dim3((unsigned)ceil_div(n, kDT), (unsigned)ceil_div64(rows, kDT)), 256, 0, st>>>(p);
    return launch_status("linear_i8 kernel");
}

}  // namespace mb
