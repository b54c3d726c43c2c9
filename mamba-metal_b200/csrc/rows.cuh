// rows.cuh -- helpers of the kernels that walk rows of channels (block norm,
// layer norm): vector accesses, sums over a CTA, rows fetched ahead through a
// ring in shared memory, and column sums of partial rows.
#pragma once

#include <algorithm>
#include <mutex>
#include <utility>
#include <vector>

#include "common.cuh"
#include "tma.cuh"

namespace mb {
namespace {

constexpr int kMaxCols = 16384;
constexpr int kDirectParts = 296;  // CTAs of the backward pass without a ring: few, so that their partial sums are

// N consecutive elements as FP32; N = 8 by 16-byte accesses, N = 4 and 2 by one of their size.
template <int N>
__device__ __forceinline__ void load_n(const float *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = *p;
    } else if constexpr (N == 2) {
        const float2 q = *reinterpret_cast<const float2 *>(p);
        v[0] = q.x;
        v[1] = q.y;
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
    } else if constexpr (N == 2) {
        const float2 q = __half22float2(*reinterpret_cast<const __half2 *>(p));
        v[0] = q.x;
        v[1] = q.y;
    } else if constexpr (N == 4) {
        const uint2 raw = *reinterpret_cast<const uint2 *>(p);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
        v[0] = a.x;
        v[1] = a.y;
        v[2] = b.x;
        v[3] = b.y;
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
    } else if constexpr (N == 2) {
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
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
    } else if constexpr (N == 2) {
        *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(v[0], v[1]);
    } else if constexpr (N == 4) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
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

// Sum over the CTA, the same bits in every thread, and a barrier: what a thread
// read from shared memory before it is read when any thread returns (shuffles
// alone do not order memory).  `sm` holds two sets of 32 partials used in turn,
// so one barrier per sum suffices: a set is overwritten only after the barrier
// of the sum in between.
__device__ __forceinline__ float block_sum(float v, float *sm, int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) {
        __syncwarp();
        return v;
    }
    float *s = sm + 32 * turn;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? s[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The same for two sums at once; `sm` holds two sets of 32 pairs.
__device__ __forceinline__ float2 block_sum2(float2 v, float2 *sm, int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (blockDim.x == 32) {
        __syncwarp();
        return v;
    }
    float2 *s = sm + 32 * turn;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? s[threadIdx.x & 31] : make_float2(0.f, 0.f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

// The ring: persistent CTAs whose rows arrive through shared memory.  One
// thread fetches each row by untiled bulk copies (one per tensor) into a ring
// of `stages` rows, that far ahead.  A wait that runs out sets the kernel's
// error word.
constexpr unsigned kErrRowTimeout = 256u;
constexpr int kMaxStages = 4;
constexpr int kRingBytes = 224 * 1024;                    // shared memory of an SM, with room for the static parts

template <int N>
struct RingRow {
    const void *src[N];  // first row of each tensor
    int64_t stride[N];   // bytes between rows
    uint32_t bytes[N];   // bytes of a row, 0: tensor absent
    uint32_t offset[N];  // within a stage
    uint32_t stage;      // bytes of a stage
    int stages;
    // Bulk copies start and end on 16-byte boundaries: a row that does not is
    // copied with the bytes around it (of its neighbours, or in the 16 bytes of
    // memory that its first or last byte lies in) and starts this far behind
    // its place.
    __device__ __forceinline__ uint32_t shift(int k, int64_t row) const {
        return (uint32_t)(reinterpret_cast<uintptr_t>(src[k]) + row * stride[k]) & 15u;
    }
};

template <int N>
__device__ __forceinline__ void fetch_row(const RingRow<N> &r, uint8_t *ring, uint64_t *full, int64_t row, int s) {
    uint32_t bytes[N], total = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        bytes[k] = r.bytes[k] ? (r.shift(k, row) + r.bytes[k] + 15) / 16 * 16 : 0;
        total += bytes[k];
    }
    mbar_arrive_expect_tx(&full[s], total);
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (bytes[k])
            bulk_load(ring + s * r.stage + r.offset[k],
                      static_cast<const uint8_t *>(r.src[k]) + row * r.stride[k] - r.shift(k, row), bytes[k], &full[s]);
}
// Place s of the ring in use, and the parity of that use.
struct RingPlace {
    int s = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void step(int stages) {
        if (++s == stages) {
            s = 0;
            parity ^= 1;
        }
    }
};
// Waits for the row at a place.  A wait that runs out is reported; the CTA goes
// on, with wrong values.
constexpr uint64_t kWaitNs = 2000000000ull;
__device__ __forceinline__ void await_row(uint64_t *full, const RingPlace &at, LostCopies *lost, unsigned *error,
                                          uint64_t limit_ns = kWaitNs) {
    if (!await_copy(full, at.s, at.parity, lost, limit_ns)) atomicOr(error, kErrRowTimeout);
}
// Sets the ring up and fetches the first rows; rows first, first + step, ...
template <int N>
__device__ __forceinline__ void start_ring(const RingRow<N> &r, uint8_t *ring, uint64_t *full, LostCopies *lost,
                                           int64_t rows) {
    if (threadIdx.x == 0) {
        *lost = LostCopies{};
        for (int s = 0; s < r.stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
        int64_t row = blockIdx.x;
        for (int s = 0; s < r.stages && row < rows; ++s, row += gridDim.x) fetch_row<N>(r, ring, full, row, s);
    }
    __syncthreads();
}

// Column sums of the partial rows, in a fixed order: warp w of a CTA of v adds
// rows w, w + v, ... of 32 columns, then the warps' sums are added in order.
// blockIdx.y: which of the two sums (NULL: not wanted).
constexpr int kSumThreads = 256;
template <int THREADS = kSumThreads>
__global__ void __launch_bounds__(THREADS)
    column_sum_kernel(const float *__restrict__ part0, const float *__restrict__ part1, float *__restrict__ sum0,
                      float *__restrict__ sum1, int parts, int cols) {
    __shared__ float sm[THREADS / 32][32];
    const float *part = blockIdx.y ? part1 : part0;
    float *dw = blockIdx.y ? sum1 : sum0;
    if (!dw) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < cols)
        for (int k = warp; k < parts; k += THREADS / 32) s += part[(int64_t)k * cols + c];
    sm[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < THREADS / 32; ++k) s += sm[k][lane];
        dw[c] = s;
    }
}

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int threads_for(int cols, int per_thread) { return std::max(32, (ceil_div(cols, per_thread) + 31) / 32 * 32); }

// Opts a kernel into the shared memory of its ring, once per device.
template <typename Kernel>
int allow_smem(Kernel kernel) {
    static std::mutex mu;
    static std::vector<std::pair<const void *, int>> done;
    int dev = 0;
    MB_CUDA_TRY(cudaGetDevice(&dev));
    const std::pair<const void *, int> key(reinterpret_cast<const void *>(kernel), dev);
    std::lock_guard<std::mutex> lk(mu);
    if (std::find(done.begin(), done.end(), key) != done.end()) return 0;
    MB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
    done.push_back(key);
    return 0;
}

// CTAs per SM that a ring kernel wants.
int ring_ctas(int threads, int resident) { return std::max(1, std::min(32, resident / threads)); }
// Lays a ring out and lowers the CTAs per SM until each has room for two rows
// (one, if at most two CTAs share the SM).  False where a row is larger than that, or
// where CTAs would get too few rows for a ring to pay: with one or two nothing
// is ahead.  Asking for 2, 3 or 6 rows a CTA measures the same.
template <int N>
bool plan_ring(RingRow<N> &r, int64_t rows, int &ctas_per_sm) {
    uint32_t at = 0;
    for (int k = 0; k < N; ++k) {
        r.offset[k] = at;
        if (r.bytes[k]) at += (r.bytes[k] + 30 + 127) / 128 * 128;  // and what surrounds an unaligned row
    }
    r.stage = at;
    for (;; --ctas_per_sm) {
        r.stages = (int)std::min<uint32_t>(kMaxStages, (uint32_t)(kRingBytes / ctas_per_sm - 2048) / std::max(at, 1u));
        if (r.stages >= 2 || (r.stages == 1 && ctas_per_sm == 2) || ctas_per_sm == 1) break;
    }
    return r.stages >= 1 && rows >= 3LL * ctas_per_sm * device_sm_count();
}

}  // namespace
}  // namespace mb
