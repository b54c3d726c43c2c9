// linear_i8.cu -- linear layer in 8-bit integers, for serving: activations
// quantised per token, weights per output channel, both symmetric.
//   quantise:  scale[t] = max|x[t]| / 127,  q = round(x / scale) (half to even)
//   product:   y[t, n] = x_scale[t] w_scale[n] sum_k xq[t, k] wq[n, k] + bias[n]
// The sums are exact 32-bit integers (k <= 131071: 128 * 128 * 131071 < 2^31),
// so the result does not depend on how K is split.
#include "common.cuh"
#include "internal.h"
#include "tma.cuh"
#include "umma.cuh"

#include <algorithm>
#include <mutex>
#include <vector>

namespace mb {

__device__ unsigned int g_linear_i8_error = 0;

namespace {

// ---- row quantiser ----------------------------------------------------------
// One read and one write of the row, which is held in registers as it was
// loaded.  Bound by bytes as long as an element costs few instructions: the
// largest magnitude is taken over packed FP16 bits, and the rounding stays in
// the FMA pipe (a conversion instruction has a quarter of its rate): 16384 x
// 2048 FP16 takes 29 us (3.5 TB/s), 66 with conversions; 16384 x 8192 FP32 109
// (6.2 TB/s).
constexpr int kQThreads = 256;
// Groups of VEC channels a thread holds.  FP16 rows: 4 (65536 x 512 takes 33
// us, with 8 it takes 43; 16384 x 2048 takes 29 with either); FP32 rows: 8
// (16384 x 8192 takes 109 us, with 4 it takes 119).
template <int VEC>
constexpr int kQRegs = VEC == 8 ? 4 : 8;

// VEC elements as loaded: 16 bytes, or one element.
template <typename T, int VEC>
struct Raw {
    uint32_t w[VEC == 1 ? 1 : 4];
};
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T *p) {
    Raw<T, VEC> r;
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 2)
            r.w[0] = __half_as_ushort(*p);
        else
            r.w[0] = __float_as_uint(*p);
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        r.w[0] = v.x;
        r.w[1] = v.y;
        r.w[2] = v.z;
        r.w[3] = v.w;
    }
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ float element(const Raw<T, VEC> &r, int k) {
    if constexpr (sizeof(T) == 2)
        return __half2float(__ushort_as_half((unsigned short)(r.w[k / 2] >> (16 * (k & 1)))));
    else
        return __uint_as_float(r.w[k]);
}
// Largest magnitudes as bits, which are ordered like the values with infinity
// and NaN above all numbers; FP16: of the two halves of a word each for itself.
template <typename T, int VEC>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const Raw<T, VEC> &r) {
#pragma unroll
    for (uint32_t w : r.w) m = sizeof(T) == 2 ? __vmaxu2(m, w & 0x7fff7fffu) : max(m, w & 0x7fffffffu);
    return m;
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

// Four elements, for a scale of 2^-100 or more: adding 1.5 * 2^23 rounds the
// product with the reciprocal to an integer, which is then the sum's low byte
// (|x| <= 127 s (1 + 2^-24), so it is 127 at most).  `off` is set where the
// remainder says that quantise() has to look at a half.
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], float s, float inv, float half, bool &off) {
    const float magic = 12582912.f;
    uint32_t t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float v = fmaf(x[k], inv, magic);
        off |= fabsf(fmaf(-(v - magic), s, x[k])) >= half;
        t[k] = __float_as_uint(v);
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

template <typename T, int VEC, int TPR>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ q, int64_t ldq,
                         float *__restrict__ scale, int64_t rows, int cols) {
    constexpr int REGS = kQRegs<VEC>;
    __shared__ uint32_t sm[kQThreads / 32];
    const int tid = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kQThreads / TPR) + threadIdx.x / TPR;
    if (TPR == 32 && row >= rows) return;
    const bool in = row < rows;  // rows of a CTA share its barrier
    const T *xr = x + row * ldx;
    int8_t *qr = q + row * ldq;
    Raw<T, VEC> v[REGS];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < REGS; ++j) {
        const int64_t c = (int64_t)(j * TPR + tid) * VEC;
        if (in && c < cols)
            v[j] = load_raw<T, VEC>(xr + c);
        else
            v[j] = Raw<T, VEC>{};
    }
#pragma unroll
    for (int j = 0; j < REGS; ++j) m = max_bits(m, v[j]);
    for (int64_t c = (int64_t)(REGS * TPR + tid) * VEC; in && c < cols; c += TPR * VEC)
        m = max_bits(m, load_raw<T, VEC>(xr + c));
    if (sizeof(T) == 2) m = max(m >> 16, m & 0xffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TPR / 32; ++k) m = max(m, sm[threadIdx.x / TPR * (TPR / 32) + k]);
        if (!in) return;
    }
    const float top = sizeof(T) == 2 ? __half2float(__ushort_as_half((unsigned short)m)) : __uint_as_float(m);
    const bool bad = !(top < INFINITY);  // an infinity or NaN in the row: scale NaN, q 0
    const float s = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(top, 127.f);
    const bool zero = bad || s == 0.f, tiny = s < 7.9e-31f;
    const float inv = zero ? 0.f : __fdiv_rn(1.f, s), half = 0.5f * s;
    if (tid == 0) scale[row] = s;
    auto emit = [&](int64_t c, const Raw<T, VEC> &u) {
        if constexpr (VEC == 1) {
            qr[c] = (int8_t)(zero ? 0 : quantise(element(u, 0), s, inv, tiny));
        } else {
            uint32_t w[VEC / 4];
            bool off = zero || tiny;
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                const float e[4] = {element(u, 4 * h), element(u, 4 * h + 1), element(u, 4 * h + 2),
                                    element(u, 4 * h + 3)};
                w[h] = quantise4(e, s, inv, half, off);
            }
            if (off) {
#pragma unroll
                for (int h = 0; h < VEC / 4; ++h) {
                    w[h] = 0;
                    for (int k = 0; k < 4 && !zero; ++k)
                        w[h] |= (uint32_t)(quantise(element(u, 4 * h + k), s, inv, tiny) & 0xff) << (8 * k);
                }
            }
            if constexpr (VEC == 8)
                *reinterpret_cast<uint2 *>(qr + c) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint32_t *>(qr + c) = w[0];
        }
    };
#pragma unroll
    for (int j = 0; j < REGS; ++j) {
        const int64_t c = (int64_t)(j * TPR + tid) * VEC;
        if (c < cols) emit(c, v[j]);
    }
    for (int64_t c = (int64_t)(REGS * TPR + tid) * VEC; c < cols; c += TPR * VEC)
        emit(c, load_raw<T, VEC>(xr + c));
}

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T, int VEC, int TPR>
int launch_quantize(const T *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int cols,
                    cudaStream_t st) {
    const int64_t grid = ceil_div64(rows, kQThreads / TPR);
    // The fewest threads a row that hold it, while every SM still gets a CTA:
    // 16384 x 2560 FP16 takes 39 us, with a whole CTA a row 62; 1024 x 2048
    // takes 10, with four CTAs per SM asked for 12.
    if constexpr (TPR < kQThreads)
        if (cols > TPR * VEC * kQRegs<VEC> || grid <= device_sm_count())
            return launch_quantize<T, VEC, 2 * TPR>(x, ldx, q, ldq, scale, rows, cols, st);
    MB_CHECK_ARG(grid <= 0x7fffffffLL, "quantize_rows: too many rows");
    quantize_rows_kernel<T, VEC, TPR><<<(unsigned)grid, kQThreads, 0, st>>>(x, ldx, q, ldq, scale, rows, cols);
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

// ---- tensor cores -----------------------------------------------------------------
// A persistent kernel of CTA pairs (clusters of two, cta_group::2), the shape
// of the FP16 projection GEMM: a pair owns 256 tokens x BN channels; per 128
// bytes of K each CTA loads its 128 rows of x and BN / 2 rows of w by TMA
// (128-byte swizzle) into a ring of stages, one thread of the even CTA issues
// tcgen05.mma.kind::i8 over both CTAs' operands, and the 32-bit sums land in
// both CTAs' TMEM, two accumulators in turn.  Eight epilogue warps scale the
// sums (warp w: TMEM lanes of quarter w % 4, every other chunk of 32 columns)
// and send them out through swizzled shared-memory boxes by bulk tensor stores
// (adds for mode 1), or element by element where y's rows are not 16-byte
// aligned.
//
// Bound by the tensor cores for large calls: 16384 x 8192 x 2048 takes 180 to
// 191 us alone (2.9 to 3.05 POP/s, tensor pipe 69% active), 156 with the
// epilogue skipped.  Decode-sized calls are bound by latency: 256 x 10240 x 2560
// takes 20 us with a cold L2.
// Every mbarrier wait is bounded (2 s); on timeout the role stops, bit 7 of the
// device status is set, and both CTAs still reach the final cluster barrier.
constexpr int kBK = 128, kUK = 32;          // bytes of K per stage and per MMA
constexpr int kStages = 5, kEpiWarps = 8, kThreads = 64 + 32 * kEpiWarps;
constexpr int kStageX = 128 * kBK, kStageW = 128 * kBK, kStageBytes = kStageX + kStageW;
constexpr int kAccCols = 256;
constexpr int kBox = 32 * 128;              // 32 rows x 128 bytes
constexpr int kSmemBytes = kStages * kStageBytes + kEpiWarps * 2 * kBox + 1024 /* alignment */ + 256 /* barriers */;
static_assert(kSmemBytes <= 232448, "shared memory");
constexpr unsigned kErrLinearI8Timeout = 128u;

struct PairParams {
    I8Params g;
    int BN, m_tiles, n_tiles, kblocks;
    uint32_t idesc, tx_bytes;
    bool boxes;  // y's rows allow bulk tensor stores
};

__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, uint64_t limit_ns = 2000000000ull) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait_bounded(bar, parity, limit_ns) ? 1 : 0;
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// 32 rows x 32 columns (a lane holds a row) without a bulk store: turned round
// in a shared-memory box, so that a warp writes a row's 32 columns at once.
__device__ __forceinline__ void store_block(const I8Params &g, uint8_t *box, int64_t row0, int c0,
                                            const float (&f)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 8; ++j)  // 16-byte chunk j of a row at j ^ (row % 8): no bank conflicts either way
        *reinterpret_cast<float4 *>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
            make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
    __syncwarp();
    const int rows = (int)min((int64_t)32, g.rows - row0);
    if (c0 + lane < g.n) {
        const int64_t o0 = row0 * g.ldy + c0 + lane;
#pragma unroll 8
        for (int r = 0; r < rows; ++r) {
            const float v =
                *reinterpret_cast<const float *>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            if (g.mode == 0)
                static_cast<__half *>(g.y)[o0 + r * g.ldy] = __float2half_rn(v);
            else if (g.mode == 1)
                static_cast<float *>(g.y)[o0 + r * g.ldy] += v;
            else
                static_cast<float *>(g.y)[o0 + r * g.ldy] = v;
        }
    }
    __syncwarp();
}

__global__ void __launch_bounds__(kThreads, 1)
    linear_i8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                          const __grid_constant__ CUtensorMap map_y, const PairParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *epi = smem + kStages * kStageBytes;
    uint64_t *full = reinterpret_cast<uint64_t *>(epi + kEpiWarps * 2 * kBox);
    uint64_t *empty = full + kStages, *tfull = empty + kStages, *tempty = tfull + 2, *drain = tempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = p.m_tiles * p.n_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 2 * kEpiWarps);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_w);
        prefetch_tensormap(&map_y);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 2 * kAccCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full0 = mapa_shared(smem_u32(&full[0]), 0);
            uint32_t it = 0;
            for (int tile = pair; tile < tiles && ok; tile += npairs) {
                const int mt = tile / p.n_tiles, nt = tile % p.n_tiles;
                const int xrow = mt * 256 + (int)rank * 128, wrow = nt * p.BN + (int)rank * (p.BN >> 1);
                for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
                    const uint32_t s = it % kStages, ph = (it / kStages) & 1;
                    if (!mbar_wait_bounded(&empty[s], ph ^ 1)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], p.tx_bytes);
                    uint8_t *a = smem + s * kStageBytes;
                    tma_load_2d_pair(a, &map_x, full0 + s * 8, kb * kBK, xrow);
                    tma_load_2d_pair(a + kStageX, &map_w, full0 + s * 8, kb * kBK, wrow);
                }
            }
            if (rank == 0) {  // every copy of both CTAs has landed before the even CTA leaves
                const uint32_t first = it > (uint32_t)kStages ? it - kStages : 0;
                for (uint32_t j = first; j < it; ++j)
                    if (!mbar_wait_bounded_cluster(&full[j % kStages], (j / kStages) & 1)) ok = false;
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t it = 0, tcount = 0;
            for (int tile = pair; tile < tiles && ok; tile += npairs, ++tcount) {
                const uint32_t b = tcount & 1, tph = (tcount >> 1) & 1;
                if (!mbar_wait_bounded_cluster(&tempty[b], tph ^ 1)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem + b * kAccCols;
                for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
                    const uint32_t s = it % kStages, ph = (it / kStages) & 1;
                    if (!mbar_wait_bounded_cluster(&full[s], ph)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + s * kStageBytes), b_addr = a_addr + kStageX;
#pragma unroll
                    for (int k = 0; k < kBK / kUK; ++k)
                        umma_i8_pair(d_tmem, smem_desc_sw128(a_addr + k * kUK), smem_desc_sw128(b_addr + k * kUK),
                                     p.idesc, (kb | k) != 0);
                    umma_commit_pair(&empty[s], 0x3);
                }
                if (!ok) break;
                umma_commit_pair(&tfull[b], 0x3);
            }
            umma_commit_pair(drain, 0x1);  // every issued MMA completes before TMEM may be freed
            if (!mbar_wait_bounded(drain, 0)) ok = false;
        }
    } else {
        const int quarter = warp & 3, egroup = (warp - 2) >> 2;
        uint8_t *boxes = epi + (warp - 2) * 2 * kBox;
        const uint32_t tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
        const I8Params &g = p.g;
        const int cstep = g.mode == 0 ? 64 : 32;  // columns of one 128-byte box row
        uint32_t tcount = 0, nbox = 0;
        for (int tile = pair; tile < tiles; tile += npairs, ++tcount) {
            const uint32_t b = tcount & 1, tph = (tcount >> 1) & 1;
            const int mt = tile / p.n_tiles, nt = tile % p.n_tiles;
            const int64_t row0 = (int64_t)mt * 256 + rank * 128 + quarter * 32, row = row0 + lane;
            const float xs = row < g.rows ? g.xs[row] : 0.f;
            // The scales and biases of this warp's columns, one column per lane and
            // 32 columns, fetched before the sums are there and handed round by
            // shuffle: chunk q of cstep columns starts at column (2 q + egroup) cstep.
            float wsc[4], wbi[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int j = 32 * q, c = nt * p.BN + (2 * (j / cstep) + egroup) * cstep + j % cstep + lane;
                wsc[q] = c < g.n ? __ldg(g.ws + c) : 0.f;
                wbi[q] = g.bias && c < g.n ? __ldg(g.bias + c) : 0.f;
            }
            if (!warp_wait(&tfull[b], tph)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16) + b * kAccCols;
#pragma unroll
            for (int q = 0; q < 4; ++q) {  // chunks of 64 columns: only q = 0, 1
                const int c = (2 * q + egroup) * cstep;
                if (c >= p.BN) break;
                const int col = nt * p.BN + c;
                if (col >= g.n || row0 >= g.rows) break;  // the same for the whole warp
                uint8_t *box = boxes + (nbox & 1) * kBox;
                // an FP16 box takes 64 columns: of a BN that is an odd multiple of 32 the last 32
                // go out without one, since the box's other half would be the next tile's
                const bool boxed = p.boxes && (g.mode != 0 || c + 32 < p.BN);
                // the bulk store that last read this box has finished reading it
                if (lane == 0) bulk_wait_group_read<1>();
                __syncwarp();
#pragma unroll
                for (int hlf = 0; hlf < 2; ++hlf) {
                    if (hlf && g.mode != 0) break;
                    const int c0 = col + 32 * hlf;
                    if (c + 32 * hlf >= p.BN) break;  // BN is a multiple of 32
                    uint32_t v[32];
                    tmem_ld_32x32b_x32(tl + c + 32 * hlf, v);
                    tmem_wait_ld();
                    float f[32];
                    const float wl = g.mode == 0 ? wsc[(2 * q + hlf) & 3] : wsc[q];
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        f[j] = (float)(int)v[j] * xs * __shfl_sync(0xffffffffu, wl, j);
                    if (g.bias) {
                        const float bl = g.mode == 0 ? wbi[(2 * q + hlf) & 3] : wbi[q];
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] += __shfl_sync(0xffffffffu, bl, j);
                    }
                    if (!boxed) {
                        store_block(g, box, row0, c0, f);
                        continue;
                    }
                    // row `lane` of a 32-row box with the TMA 128-byte swizzle: chunk j at j ^ (row % 8)
                    if (g.mode == 0) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const __half2 h = __floats2half2_rn(f[8 * j + 2 * q], f[8 * j + 2 * q + 1]);
                                w[q] = *reinterpret_cast<const uint32_t *>(&h);
                            }
                            *reinterpret_cast<uint4 *>(box + lane * 128 + (((4 * hlf + j) ^ (lane & 7)) << 4)) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4 *>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                                make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                    }
                }
                if (!boxed) continue;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (g.mode == 1)
                        tma_reduce_add_2d(&map_y, box, col, (int)row0);
                    else
                        tma_store_2d(&map_y, box, col, (int)row0);
                    bulk_commit_group();
                }
                ++nbox;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0)
                    mbar_arrive(&tempty[b]);
                else
                    mbar_arrive_cluster(tempty0 + b * 8);
            }
        }
        if (lane == 0) bulk_wait_group_all();
        __syncwarp();
    }
    if (!ok) atomicOr(&g_linear_i8_error, kErrLinearI8Timeout);
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 2 * kAccCols);
    }
}

// 2-D map over row-major rows with 128-byte-swizzled boxes of 128 bytes x
// box_rows; loads outside the matrix read zeros, stores outside are dropped.
bool encode_rows(CUtensorMap *m, CUtensorMapDataType t, int esize, const void *ptr, int64_t rows, int64_t cols,
                 int64_t ld, int box_rows) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * esize)};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / esize), (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return enc(m, t, 2, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t pair_launch(int pairs, cudaLaunchAttribute *attr, cudaStream_t st) {
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = 2;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * pairs, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

// CTA pairs that fit on the current device at once (asked once per device),
// -1 on an error, 0 on a device without these tensor cores.
int device_pairs() {
    static std::mutex mu;
    static std::vector<int> cache;
    int dev = 0;
    MB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if ((int)cache.size() <= dev) cache.resize(dev + 1, -1);
    if (cache[dev] < 0) {
        int major = 0, n = 0;
        MB_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
        if (major == 10) {
            MB_CUDA_TRY(cudaFuncSetAttribute(linear_i8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kSmemBytes));
            cudaLaunchAttribute attr{};
            cudaLaunchConfig_t cfg = pair_launch(148, &attr, nullptr);
            MB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, linear_i8_pair_kernel, &cfg));
        }
        cache[dev] = n;
    }
    return cache[dev];
}

// Columns per tile: the multiple of 32 with the least rounds of tiles over the
// pairs, each round costing what a CTA loads per byte of K (128 rows of x and
// BN / 2 of w).  Against 256 everywhere: 777 x 203 x 1000 14.3 us instead of
// 18.5, 256 x 2560 x 5120 22.6 instead of 24.6; 256 x 10240 x 2560 and large
// calls take the same time with either.
int choose_bn(int64_t m_tiles, int n, int pairs) {
    int best = 256;
    int64_t cost = INT64_MAX;
    for (int bn = 256; bn >= 32; bn -= 32) {
        const int64_t rounds = ceil_div64(m_tiles * ceil_div(n, bn), pairs), c = rounds * (128 + bn / 2);
        if (c < cost) {
            cost = c;
            best = bn;
        }
    }
    return best;
}

int launch_pairs(const I8Params &g, int pairs, cudaStream_t st) {
    PairParams p{};
    p.g = g;
    p.m_tiles = (int)ceil_div64(g.rows, 256);
    p.BN = choose_bn(p.m_tiles, g.n, pairs);
    const int64_t tiles = (int64_t)p.m_tiles * ceil_div(g.n, p.BN);
    MB_CHECK_ARG(tiles <= 0x7fffffff, "linear_i8: too many tiles");
    p.n_tiles = ceil_div(g.n, p.BN);
    p.kblocks = ceil_div(g.k, kBK);
    p.idesc = idesc_s8_s32acc(256, p.BN);
    p.tx_bytes = (uint32_t)(2 * (kStageX + (p.BN / 2) * kBK));
    const int es = g.mode == 0 ? 2 : 4;
    p.boxes = aligned_to(g.y, 16) && (g.ldy * es) % 16 == 0;
    CUtensorMap mx, mw, my;
    bool enc = encode_rows(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.x, g.rows, g.k, g.ldx, 128) &&
               encode_rows(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.w, g.n, g.k, g.ldw, p.BN / 2);
    if (enc && p.boxes)
        enc = encode_rows(&my, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, es, g.y,
                          g.rows, g.n, g.ldy, 32);
    else
        my = mx;
    MB_CHECK_ARG(enc, "linear_i8: tensor map encoding failed");
    cudaLaunchAttribute attr{};
    const cudaLaunchConfig_t cfg = pair_launch((int)std::min<int64_t>(tiles, pairs), &attr, st);
    MB_CUDA_TRY(cudaLaunchKernelEx(&cfg, linear_i8_pair_kernel, mx, mw, my, p));
    return launch_status("linear_i8 (tcgen05, CTA pairs) kernel");
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
    MB_CHECK_ARG(!q || (static_cast<const void *>(q) != x && static_cast<void *>(q) != scale),
                 "quantize_rows: q needs memory of its own");
    const int wide = 16 / (int)dtype_size(dtype);  // elements of 16 bytes
    const bool vec = cols % wide == 0 && aligned_to(x, 16) && (rows == 1 || (ldx % wide == 0 && ldq % wide == 0)) &&
                     aligned_to(q, wide);
    if (dtype == MAMBA_F16) {
        auto *p = static_cast<const __half *>(x);
        return vec ? launch_quantize<__half, 8, 32>(p, ldx, q, ldq, scale, rows, cols, st)
                   : launch_quantize<__half, 1, 32>(p, ldx, q, ldq, scale, rows, cols, st);
    }
    auto *p = static_cast<const float *>(x);
    return vec ? launch_quantize<float, 4, 32>(p, ldx, q, ldq, scale, rows, cols, st)
               : launch_quantize<float, 1, 32>(p, ldx, q, ldq, scale, rows, cols, st);
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
    const void *in[5] = {x, w, x_scale, w_scale, bias};
    for (const void *v : in) MB_CHECK_ARG(v != y, "linear_i8: y may not be one of the inputs");
    I8Params p{};
    p.x = x;
    p.w = w;
    p.xs = x_scale;
    p.ws = w_scale;
    p.bias = bias;
    p.y = y;
    // a single row has no stride of its own
    const int64_t k16 = ((int64_t)k + 15) / 16 * 16, n16 = ((int64_t)n + 15) / 16 * 16;
    p.ldx = ldx = rows == 1 ? k16 : ldx;
    p.ldw = ldw = n == 1 ? k16 : ldw;
    p.ldy = rows == 1 ? n16 : ldy;
    p.rows = rows;
    p.n = n;
    p.k = k;
    p.mode = mode;
    if (k > 0 && aligned_to(x, 16) && aligned_to(w, 16) && ldx % 16 == 0 && ldw % 16 == 0 &&
        rows <= 0x7fffffff - 256) {
        const int pairs = device_pairs();
        if (pairs < 0) return -1;
        if (pairs > 0) return launch_pairs(p, pairs, st);
    }
    MB_CHECK_ARG(rows <= 65535LL * kDT, "linear_i8: too many rows");
    linear_i8_dp4a_kernel<<<dim3((unsigned)ceil_div(n, kDT), (unsigned)ceil_div64(rows, kDT)), 256, 0, st>>>(p);
    return launch_status("linear_i8 kernel");
}

namespace {

// A wait for sums that nothing computes, through the epilogue's own helper.
__global__ void linear_i8_wait_selftest_kernel(uint64_t limit_ns) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        fence_mbar_init();
    }
    __syncwarp();
    if (!warp_wait(&bar, 0, limit_ns)) atomicOr(&g_linear_i8_error, kErrLinearI8Timeout);
}

}  // namespace

int linear_i8_wait_selftest(uint64_t limit_ns, cudaStream_t st) {
    linear_i8_wait_selftest_kernel<<<1, 32, 0, st>>>(limit_ns);
    return launch_status("linear_i8 wait self-test kernel");
}

unsigned linear_i8_error_flags(bool clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_linear_i8_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (clear && v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_linear_i8_error, &z, sizeof(z));
    }
    return v;
}

}  // namespace mb
