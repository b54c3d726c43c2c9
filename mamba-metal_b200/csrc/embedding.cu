// embedding.cu -- embedding lookup with scaling, and the table's gradient:
//   out[t] = scale * table[id_t]                      (0 for ids outside the table)
//   dtable[v] = scale * sum_{t : id_t = v} dout[t]    (in order of t)
//
// Lookup: a gather, bound by bytes (the rows that occur, once, and out).
//
// Gradient: no atomics, so that the sums have one order.  The ids are sorted
// with their positions, the sorted list is cut into parts of equal length, and
// one CTA sums the rows of a part, id by id.  An id that lies within one part is
// finished there; the sums of one that spans several leave as partial rows,
// which a second kernel adds in order.  Frequent ids so cost no more than others.
// Rows of the table that no token names are zeroed beside the sums, each row
// of the table being written once.  Bound by bytes: dout once, the table once.
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace mb {

__device__ unsigned int g_embedding_error = 0;

namespace {

// ---- lookup -------------------------------------------------------------------
// 32768 x 2048 FP16 into FP32 and into FP16: 128 threads and 4 tokens in flight
// 53 and 32 us, 256 threads 58 and 44, 512 72 and 65, 8 tokens 68 and 44.
constexpr int kLookupThreads = 128;
constexpr int kLookupTokens = 4;  // tokens a thread has in flight

__device__ __forceinline__ int64_t token_id(const void *ids, bool wide, int64_t t) {
    return wide ? static_cast<const int64_t *>(ids)[t] : (int64_t) static_cast<const int32_t *>(ids)[t];
}

struct LookupParams {
    const void *ids;
    const void *table;
    void *out;
    int64_t tokens, vocab, table_stride, out_stride;
    int dim;
    bool wide;
    float scale;
};

// Threads (x) cover a row in groups of VEC elements, (y) different tokens.
template <typename TT, typename TO, int VEC, int TOKENS>
__global__ void __launch_bounds__(kLookupThreads) embedding_kernel(const LookupParams p) {
    const int64_t t0 = (int64_t)blockIdx.x * (blockDim.y * TOKENS) + threadIdx.y;
    int64_t id[TOKENS];
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
        const int64_t t = t0 + k * blockDim.y;
        id[k] = t < p.tokens ? token_id(p.ids, p.wide, t) : -1;
        if (id[k] >= p.vocab) id[k] = -1;
    }
    for (int c = threadIdx.x * VEC; c < p.dim; c += blockDim.x * VEC) {
        float v[TOKENS][VEC];
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            if (id[k] >= 0) {
                load_n(static_cast<const TT *>(p.table) + id[k] * p.table_stride + c, v[k]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < TOKENS; ++k) {
            const int64_t t = t0 + k * blockDim.y;
            if (t >= p.tokens) break;
            if (id[k] >= 0) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] *= p.scale;
            }
            store_n(static_cast<TO *>(p.out) + t * p.out_stride + c, v[k]);
        }
    }
}

int pow2_at_least(int v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

template <typename TT, typename TO, int VEC>
int launch_lookup(const LookupParams &p, cudaStream_t st) {
    const int tx = std::min(kLookupThreads, pow2_at_least(p.dim / VEC)), ty = kLookupThreads / tx;
    // few tokens: more CTAs instead (256 x 2560 2.5 us, 3.6 with 4 tokens each)
    const bool few = p.tokens < (int64_t)ty * kLookupTokens * 2 * device_sm_count();
    const int64_t grid = ceil_div64(p.tokens, (int64_t)ty * (few ? 1 : kLookupTokens));
    MB_CHECK_ARG(grid <= 0x7fffffff, "embedding: too many tokens");
    if (few)
        embedding_kernel<TT, TO, VEC, 1><<<(unsigned)grid, dim3(tx, ty), 0, st>>>(p);
    else
        embedding_kernel<TT, TO, VEC, kLookupTokens><<<(unsigned)grid, dim3(tx, ty), 0, st>>>(p);
    return launch_status("embedding kernel");
}

// 16 bytes of out a thread: FP32 rows written 32 bytes a thread leave half of
// each access's sectors empty (32768 x 2048 into FP32, 256 threads: 71 us in
// place of 58).  Rows of an even width that are not 16-byte aligned: pairs.
template <typename TT, typename TO>
int launch_lookup(const LookupParams &p, bool vec, bool pairs, cudaStream_t st) {
    if (vec) return launch_lookup<TT, TO, 16 / (int)sizeof(TO)>(p, st);
    return pairs ? launch_lookup<TT, TO, 2>(p, st) : launch_lookup<TT, TO, 1>(p, st);
}

// ---- sort -----------------------------------------------------------------------
// Stable, 8 bits at a time, least significant first.  Up to kTinyTokens tokens
// one CTA runs all passes in shared memory, up to 8 times as many a cluster of 8
// CTAs (32768 tokens, 16 bits: 18 us in one launch, by the kernels below 18 in
// four); above that each pass counts the
// digits of every tile and then moves the tile's items, whose places a CTA
// finds from the counts itself while there are few tiles (kFewTiles), and from
// their running sums, made by a kernel in between, when there are many.  That
// kernel is one CTA, whose time grows with the tokens: two passes over 2^17, 2^18
// and 2^20 tokens 28, 54 and 210 us, beside 126, 243 and 927 for the sums of rows
// of 256.
constexpr int kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 256, kSortItems = 4, kSortTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kFewTiles = 64;
constexpr int kTinyThreads = 1024, kTinyItems = 4, kTinyTokens = kTinyThreads * kTinyItems, kTinyWarps = kTinyThreads / 32;

// Key of a token: its id, or `vocab` (behind all ids) for one outside the table.
__device__ __forceinline__ uint32_t token_key(const void *ids, bool wide, int64_t t, uint32_t vocab) {
    const int64_t id = token_id(ids, wide, t);
    return id >= 0 && id < (int64_t)vocab ? (uint32_t)id : vocab;
}

struct SortPass {
    const void *ids;  // first pass: the keys come from here; NULL: from keys_in, pos_in
    const uint32_t *keys_in, *pos_in;
    uint32_t *keys_out, *pos_out;
    uint32_t *hist;  // [tiles][kDigits] counts, or with many tiles [kDigits][tiles] first places
    uint32_t n, vocab;
    int shift, bits, tiles;
    bool wide, few;
};
__device__ __forceinline__ uint32_t pass_key(const SortPass &p, uint32_t i) {
    return p.ids ? token_key(p.ids, p.wide, i, p.vocab) : p.keys_in[i];
}

// Place of each of a warp's items among the warp's items of the same digit
// (items in the order k * 32 + lane; digit kDigits: no item); `count` [kDigits]
// ends as the warp's numbers.  The lanes of one digit find each other by a match.
template <int ITEMS, typename Count, typename Digit>
__device__ __forceinline__ void rank_in_warp(Count *count, uint32_t (&rank)[ITEMS], Digit digit) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const uint32_t d = digit(k), same = __match_any_sync(0xffffffffu, d);
        const uint32_t before = d < kDigits ? count[d] : 0;
        rank[k] = before + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (d < kDigits && lane == __ffs(same) - 1) count[d] = (Count)(before + __popc(same));
        __syncwarp();
    }
}
// Exclusive sum over kDigits threads' values (the CTA's first kDigits threads; all call).
__device__ __forceinline__ uint32_t exclusive_digits(uint32_t v, uint32_t *warp_sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t in = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += u;
    }
    if (warp < kDigits / 32 && lane == 31) warp_sum[warp] = in;
    __syncthreads();
    uint32_t base = 0;
    for (int w = 0; w < warp && w < kDigits / 32; ++w) base += warp_sum[w];
    __syncthreads();
    return base + in - v;
}

// All passes over at most CTAS * kTinyTokens tokens, by one cluster.  CTA r holds
// places r * kTinyTokens .. of the list in shared memory; in each pass the CTAs
// tell each other their numbers of each digit and write their items to the
// places' owners.
template <int CTAS>
struct TinySmem {
    uint64_t item[kTinyTokens];  // position, key above it
    uint32_t total[CTAS][kDigits];
    uint16_t count[kTinyWarps][kDigits];
    uint32_t warp_sum[kDigits / 32];
};
__device__ __forceinline__ void store_cluster(uint32_t addr, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
template <int CTAS>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kTinyThreads) sort_small_kernel(const SortPass p) {
    static_assert(CTAS * kTinyTokens <= 65536, "places fit 16 bits");
    extern __shared__ __align__(16) uint8_t smem_raw[];
    TinySmem<CTAS> &sm = *reinterpret_cast<TinySmem<CTAS> *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t self = CTAS > 1 ? cluster_ctarank() : 0, base = self * kTinyTokens;
    uint32_t key[kTinyItems], pos[kTinyItems], rank[kTinyItems];
#pragma unroll
    for (int k = 0; k < kTinyItems; ++k) {
        const uint32_t i = base + warp * (32 * kTinyItems) + k * 32 + lane;
        key[k] = i < p.n ? token_key(p.ids, p.wide, i, p.vocab) : 0;
        pos[k] = i;
    }
    if (CTAS > 1) cluster_sync();  // every CTA has started: its shared memory may be written
    for (int shift = 0; shift < p.bits; shift += kDigitBits) {
        if (shift > 0) {
#pragma unroll
            for (int k = 0; k < kTinyItems; ++k) {
                const int i = warp * (32 * kTinyItems) + k * 32 + lane;
                key[k] = (uint32_t)(sm.item[i] >> 32);
                pos[k] = (uint32_t)sm.item[i];
            }
        }
        for (int d = tid; d < kTinyWarps * kDigits / 2; d += kTinyThreads) reinterpret_cast<uint32_t *>(sm.count)[d] = 0;
        __syncthreads();
        auto digit = [&](int k) {
            const uint32_t i = base + warp * (32 * kTinyItems) + k * 32 + lane;
            return i < p.n ? key[k] >> shift & (kDigits - 1) : (uint32_t)kDigits;
        };
        rank_in_warp<kTinyItems>(sm.count[warp], rank, digit);
        __syncthreads();
        uint32_t all = 0, before = 0;
        if (tid < kDigits) {
#pragma unroll
            for (int w = 0; w < kTinyWarps; ++w) all += sm.count[w][tid];
            if (CTAS > 1) {
                const uint32_t at = smem_u32(&sm.total[self][tid]);
#pragma unroll
                for (int r = 0; r < CTAS; ++r) store_cluster(mapa_shared(at, r), all);
            }
        }
        if (CTAS > 1) {
            cluster_sync();  // also: every CTA has its items in registers
            all = 0;
            if (tid < kDigits) {
#pragma unroll
                for (int r = 0; r < CTAS; ++r) {
                    const uint32_t v = sm.total[r][tid];
                    if (r < (int)self) before += v;
                    all += v;
                }
            }
        }
        uint32_t run = exclusive_digits(all, sm.warp_sum) + before;
        if (tid < kDigits) {
            uint16_t c[kTinyWarps];  // loads that wait for no store
#pragma unroll
            for (int w = 0; w < kTinyWarps; ++w) c[w] = sm.count[w][tid];
#pragma unroll
            for (int w = 0; w < kTinyWarps; ++w) {
                sm.count[w][tid] = (uint16_t)run;
                run += c[w];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kTinyItems; ++k) {
            const uint32_t d = digit(k);
            if (d < kDigits) {
                const uint32_t to = sm.count[warp][d] + rank[k];
                const uint64_t item = (uint64_t)key[k] << 32 | pos[k];
                if (CTAS > 1)
                    store_cluster(mapa_shared(smem_u32(&sm.item[to % kTinyTokens]), to / kTinyTokens), item);
                else
                    sm.item[to] = item;
            }
        }
        if (CTAS > 1)
            cluster_sync();
        else
            __syncthreads();
    }
    for (uint32_t i = tid; i < kTinyTokens && base + i < p.n; i += kTinyThreads) {
        p.keys_out[base + i] = (uint32_t)(sm.item[i] >> 32);
        p.pos_out[base + i] = (uint32_t)sm.item[i];
    }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortPass p) {
    __shared__ uint32_t count[kDigits];
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (uint32_t)kSortTile;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = base + k * kSortThreads + threadIdx.x;
        if (i < p.n) atomicAdd(&count[pass_key(p, i) >> p.shift & (kDigits - 1)], 1u);  // whole numbers: any order
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads)
        p.hist[p.few ? (size_t)blockIdx.x * kDigits + d : (size_t)d * p.tiles + blockIdx.x] = count[d];
}

// Exclusive sums of `n` counts in place, one CTA.
__global__ void __launch_bounds__(1024) sort_sum_kernel(uint32_t *v, uint32_t n) {
    __shared__ uint32_t warp_sum[32];
    __shared__ uint32_t carry;
    if (threadIdx.x == 0) carry = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t base = 0; base < n; base += 4096) {
        uint32_t e[4], s = 0;
        const uint32_t at = base + threadIdx.x * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            e[k] = at + k < n ? v[at + k] : 0;
            s += e[k];
        }
        uint32_t in = s;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += u;
        }
        __syncthreads();  // the last round's readers of warp_sum and carry are done
        if (lane == 31) warp_sum[warp] = in;
        __syncthreads();
        if (warp == 0) {
            uint32_t w = warp_sum[lane];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += u;
            }
            warp_sum[lane] = w;
        }
        __syncthreads();
        uint32_t run = carry + (warp ? warp_sum[warp - 1] : 0) + in - s;
        const uint32_t total = warp_sum[31];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (at + k < n) v[at + k] = run;
            run += e[k];
        }
        __syncthreads();
        if (threadIdx.x == 0) carry += total;
    }
}

// Moves a tile's items to their places.  Warp w of the tile holds items
// w * 32 * kSortItems + k * 32 + lane, so equal digits keep their order.
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(const SortPass p) {
    static_assert(kSortThreads == kDigits, "a thread per digit");
    __shared__ uint32_t count[kSortWarps][kDigits];
    __shared__ uint32_t warp_sum[kDigits / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digit_of = threadIdx.x;
    // first place of this tile's items of digit `digit_of`
    uint32_t first = 0;
    if (p.few) {
        uint32_t before = 0, all = 0;
#pragma unroll 8
        for (int t = 0; t < p.tiles; ++t) {
            const uint32_t c = p.hist[(size_t)t * kDigits + digit_of];
            if (t < (int)blockIdx.x) before += c;
            all += c;
        }
        first = exclusive_digits(all, warp_sum) + before;
    } else {
        first = p.hist[(size_t)digit_of * p.tiles + blockIdx.x];
    }
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) count[w][digit_of] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (uint32_t)kSortTile + warp * (32 * kSortItems);
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = base + k * 32 + lane;
        key[k] = i < p.n ? pass_key(p, i) : 0;
    }
    rank_in_warp<kSortItems>(count[warp], rank, [&](int k) {
        return base + k * 32 + lane < p.n ? key[k] >> p.shift & (kDigits - 1) : (uint32_t)kDigits;
    });
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w][digit_of];
        count[w][digit_of] = first;
        first += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = base + k * 32 + lane;
        if (i < p.n) {
            const uint32_t to = count[warp][key[k] >> p.shift & (kDigits - 1)] + rank[k];
            p.keys_out[to] = key[k];
            p.pos_out[to] = p.ids ? i : p.pos_in[i];
        }
    }
}

constexpr int kSmallCtas = 8;
template <int CTAS>
int launch_small(const SortPass &p, cudaStream_t st) {
    if (allow_smem(sort_small_kernel<CTAS>)) return -1;
    sort_small_kernel<CTAS><<<CTAS, kTinyThreads, sizeof(TinySmem<CTAS>), st>>>(p);
    return launch_status("embedding_backward sort kernel");
}

// ---- sums -----------------------------------------------------------------------
// The sorted list is cut into equal parts, one per CTA and about as many as fit
// the GPU at once, so that an id that occurs often spans few of them.  Rows of
// dout arrive through a ring in shared memory, fetched ahead by bulk copies.
constexpr unsigned kErrEmbeddingTimeout = 512u;
constexpr int kSumThreadsE = 256;
constexpr int kSumStages = 8;
constexpr int kZeroRows = 16;  // table rows that a CTA looks after

struct SumParams {
    const uint32_t *keys, *pos;
    const void *dout;
    float *dtable;
    float *part;  // [parts][2][dim]: slot 0 an id begun in an earlier part, 1 one that goes on in the next
    int64_t dout_stride, table_stride;
    uint32_t n, vocab, len;  // len: sorted tokens per part
    int dim, parts, cols, stages;  // cols: columns of a CTA
    uint32_t stage;                // bytes of a row's place in the ring
    float scale;
    bool accumulate;
};

template <int VEC>
__device__ __forceinline__ void put_row(const SumParams &p, uint32_t key, int c, const float (&s)[VEC]) {
    float *to = p.dtable + (int64_t)key * p.table_stride + c;
    float v[VEC];
    if (p.accumulate) load_n(to, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = p.accumulate ? fmaf(s[e], p.scale, v[e]) : s[e] * p.scale;
    store_n(to, v);
}

// Rows of the table that no token names become zero.
__device__ void zero_rows(const SumParams &p, int64_t tile) {
    __shared__ uint8_t present[kZeroRows];
    const uint32_t v0 = (uint32_t)(tile * kZeroRows), v1 = (uint32_t)min((int64_t)p.vocab, (tile + 1) * kZeroRows);
    if (v0 + threadIdx.x < v1) {
        const uint32_t v = v0 + threadIdx.x;
        uint32_t lo = 0, hi = p.n;  // the first sorted token with an id of v or more
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (p.keys[mid] < v)
                lo = mid + 1;
            else
                hi = mid;
        }
        present[threadIdx.x] = lo < p.n && p.keys[lo] == v;
    }
    __syncthreads();
    const bool vec = p.dim % 4 == 0 && p.table_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.dtable) % 16 == 0;
    for (uint32_t v = v0; v < v1; ++v) {
        if (present[v - v0]) continue;
        float *row = p.dtable + (int64_t)v * p.table_stride;
        if (vec)
            for (int c = threadIdx.x * 4; c < p.dim; c += kSumThreadsE * 4)
                *reinterpret_cast<float4 *>(row + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        else
            for (int c = threadIdx.x; c < p.dim; c += kSumThreadsE) row[c] = 0.f;
    }
}

// Waits for the row at a place of the ring.  A wait that runs out is reported; the
// CTA goes on, with wrong values.
__device__ __forceinline__ void await_sum_row(uint64_t *full, const RingPlace &at, LostCopies *lost,
                                              uint64_t limit_ns = kWaitNs) {
    if (!await_copy(full, at.s, at.parity, lost, limit_ns)) atomicOr(&g_embedding_error, kErrEmbeddingTimeout);
}

// blockIdx.x: part, and behind the parts tiles of the table to zero; blockIdx.y:
// block of columns (the zeroing has one).  A thread has NV groups of VEC columns,
// group g at column (g * threads + t) * VEC.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kSumThreadsE) embedding_sum_kernel(const SumParams p) {
    if (blockIdx.x >= (unsigned)p.parts) {
        if (blockIdx.y == 0) zero_rows(p, blockIdx.x - p.parts);
        return;
    }
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t full[kSumStages];
    __shared__ LostCopies lost;
    const uint32_t first = blockIdx.x * p.len, end = min(p.n, first + p.len);
    const int c0 = blockIdx.y * p.cols, cols = min(p.cols, p.dim - c0);
    // a row's columns start at `from`; what precedes them in their 16 bytes is copied too
    auto from = [&](uint32_t pos) {
        return reinterpret_cast<const uint8_t *>(static_cast<const T *>(p.dout) + (int64_t)pos * p.dout_stride + c0);
    };
    auto fetch = [&](uint32_t pos, int s) {
        const uint8_t *src = from(pos);
        const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(src) & 15u;
        const uint32_t bytes = (shift + cols * (uint32_t)sizeof(T) + 15) / 16 * 16;
        mbar_arrive_expect_tx(&full[s], bytes);
        bulk_load(ring + s * p.stage, src - shift, bytes, &full[s]);
    };
    // tokens outside the table are last: nothing behind the first of them counts
    uint32_t live = end;
    if (first < end && p.keys[end - 1] >= p.vocab) {
        uint32_t lo = first, hi = end - 1;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (p.keys[mid] < p.vocab)
                lo = mid + 1;
            else
                hi = mid;
        }
        live = lo;
    }
    if (threadIdx.x == 0) {
        lost = LostCopies{};
        for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
        for (int s = 0; s < p.stages && first + s < live; ++s) fetch(p.pos[first + s], s);
    }
    __syncthreads();
    if (first >= live) return;
    // the next row to fetch, looked up a row ahead
    uint32_t fetch_pos = first + p.stages < live ? p.pos[first + p.stages] : 0;
    float sum[NV][VEC] = {};
    uint32_t id = p.keys[first];
    bool begun = first > 0 && p.keys[first - 1] == id;  // the current id begun in an earlier part
    RingPlace at;
    uint32_t next = first + 1 < p.n ? p.keys[first + 1] : p.vocab;
    for (uint32_t i = first; i < live; ++i) {
        const uint32_t after = i + 2 < p.n ? p.keys[i + 2] : p.vocab;  // on its way while the row is added
        const uint32_t shift = VEC <= 2 ? (uint32_t)reinterpret_cast<uintptr_t>(from(p.pos[i])) & 15u : 0u;
        await_sum_row(full, at, &lost);
        const T *row = reinterpret_cast<const T *>(ring + at.s * p.stage + shift);
#pragma unroll
        for (int g = 0; g < NV; ++g) {
            const int c = (g * kSumThreadsE + threadIdx.x) * VEC;
            if (c < cols) {
                float v[VEC];
                load_n(row + c, v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[g][e] += v[e];
            }
        }
        __syncthreads();  // the row's place is free
        if (threadIdx.x == 0 && i + p.stages < live) {
            if (!lost.flag) fetch(fetch_pos, at.s);
            if (i + p.stages + 1 < live) fetch_pos = p.pos[i + p.stages + 1];
        }
        at.step(p.stages);
        const bool ends = next != id;
        if (ends || i + 1 == live) {
#pragma unroll
            for (int g = 0; g < NV; ++g) {
                const int c = (g * kSumThreadsE + threadIdx.x) * VEC;
                if (c < cols) {
                    if (!begun && ends)
                        put_row(p, id, c0 + c, sum[g]);
                    else
                        store_n(p.part + ((int64_t)blockIdx.x * 2 + (begun ? 0 : 1)) * p.dim + c0 + c, sum[g]);
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[g][e] = 0.f;
            }
            begun = false;
        }
        id = next;
        next = after;
    }
    drain_copies(full, p.stages, &lost, kWaitNs);
}

// blockIdx.x: the part in which an id begins that goes on in the next ones.
template <int VEC>
__global__ void __launch_bounds__(kSumThreadsE) embedding_join_kernel(const SumParams p) {
    const uint32_t first = blockIdx.x * p.len;
    if (p.n - first <= p.len) return;  // the last part
    const uint32_t end = first + p.len, id = p.keys[end];  // end: the next part's first
    if (id >= p.vocab || p.keys[end - 1] != id) return;
    if (first > 0 && p.keys[first - 1] == id) return;  // begun earlier
    // the last part that starts with the id: each warp looks at 32 at once
    int last = blockIdx.x + 1;
    for (;;) {
        const int part = last + 1 + (threadIdx.x & 31);
        const uint32_t other = __ballot_sync(0xffffffffu, part >= p.parts || p.keys[(uint32_t)part * p.len] != id);
        if (other) {
            last += __ffs(other) - 1;
            break;
        }
        last += 32;
    }
    const int c = (blockIdx.y * kSumThreadsE + threadIdx.x) * VEC;
    if (c >= p.dim) return;
    float sum[VEC];
    load_n(p.part + ((int64_t)blockIdx.x * 2 + 1) * p.dim + c, sum);
#pragma unroll 8
    for (int k = blockIdx.x + 1; k <= last; ++k) {
        float v[VEC];
        load_n(p.part + (int64_t)k * 2 * p.dim + c, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += v[e];
    }
    put_row(p, id, c, sum);
}

// Sorted tokens per part, and the parts.  Four CTAs an SM by shared memory.
uint32_t part_length(int64_t n) { return (uint32_t)std::max<int64_t>(4, ceil_div64(n, 148 * 4)); }

template <typename T, int VEC, int NV>
int launch_sums(SumParams &p, cudaStream_t st) {
    p.cols = kSumThreadsE * VEC * NV;
    const int cols = std::min(p.cols, p.dim);
    p.stage = (uint32_t)((cols * sizeof(T) + 30) / 128 * 128 + 128);
    p.stages = (int)std::max<uint32_t>(2, std::min<uint32_t>(kSumStages, kRingBytes / 4 / p.stage));
    auto kernel = embedding_sum_kernel<T, VEC, NV>;
    if (allow_smem(kernel)) return -1;
    const int64_t zero = p.accumulate ? 0 : ceil_div64(p.vocab, kZeroRows);
    MB_CHECK_ARG(p.parts + zero <= 0x7fffffff, "embedding_backward: too many rows");
    kernel<<<dim3((unsigned)(p.parts + zero), (unsigned)ceil_div(p.dim, p.cols)), kSumThreadsE,
             (size_t)p.stage * p.stages, st>>>(p);
    if (launch_status("embedding_backward sum kernel")) return -1;
    if (p.parts == 1) return 0;
    constexpr int JV = VEC <= 2 ? VEC : 4;
    embedding_join_kernel<JV><<<dim3((unsigned)p.parts, (unsigned)ceil_div(p.dim, kSumThreadsE * JV)), kSumThreadsE, 0,
                                st>>>(p);
    return launch_status("embedding_backward join kernel");
}

struct Layout {
    size_t keys[2], pos[2], hist, part, bytes;
    int tiles, parts;
};
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
Layout layout(int64_t n, int dim) {
    Layout l{};
    l.tiles = (int)ceil_div64(n, kSortTile);
    l.parts = (int)ceil_div64(n, part_length(n));
    size_t at = 0;
    for (int k = 0; k < 2; ++k) {
        l.keys[k] = at;
        at += up256((size_t)n * 4);
        l.pos[k] = at;
        at += up256((size_t)n * 4);
    }
    l.hist = at;
    at += up256((size_t)l.tiles * kDigits * 4);
    l.part = at;
    at += up256((size_t)l.parts * 2 * dim * 4);
    l.bytes = at;
    return l;
}

// A wait for a row that nothing fetches, through the kernel's own helpers.
__global__ void embedding_wait_selftest_kernel(uint64_t limit_ns) {
    __shared__ uint64_t full;
    __shared__ LostCopies lost;
    if (threadIdx.x != 0) return;
    lost = LostCopies{};
    mbar_init(&full, 1);
    fence_mbar_init();
    await_sum_row(&full, RingPlace{}, &lost, limit_ns);
    drain_copies(&full, 1, &lost, limit_ns);
}

constexpr int64_t kMaxTokens = (int64_t)1 << 30;

int check_embedding(const MambaEmbeddingArgs *a, const std::string &what) {
    MB_CHECK_ARG(a, what + ": null args");
    MB_CHECK_ARG(a->tokens >= 0 && a->vocab >= 0 && a->dim >= 0, what + ": negative size");
    MB_CHECK_ARG(a->tokens <= kMaxTokens, what + ": more than 2^30 tokens");
    MB_CHECK_ARG(a->vocab < (int64_t)1 << 31, what + ": more than 2^31 - 1 rows");
    MB_CHECK_ARG(a->id_bytes == 4 || a->id_bytes == 8, what + ": ids must have 4 or 8 bytes");
    MB_CHECK_ARG(a->scale - a->scale == 0.f, what + ": scale must be finite");
    MB_CHECK_ARG((a->table_dtype == MAMBA_F32 || a->table_dtype == MAMBA_F16) &&
                     (a->out_dtype == MAMBA_F32 || a->out_dtype == MAMBA_F16),
                 what + ": bad dtype");
    MB_CHECK_ARG(aligned_to(a->ids, (size_t)a->id_bytes), what + ": pointers must be aligned to their element type");
    return 0;
}

}  // namespace

int embedding_wait_selftest(uint64_t limit_ns, cudaStream_t st) {
    embedding_wait_selftest_kernel<<<1, 32, 0, st>>>(limit_ns);
    return launch_status("embedding wait self-test kernel");
}

unsigned embedding_error_flags(bool clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_embedding_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (clear && v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_embedding_error, &z, sizeof(z));
    }
    return v;
}

int embedding(const MambaEmbeddingArgs *a, cudaStream_t st) {
    if (check_embedding(a, "embedding")) return -1;
    if (a->tokens == 0 || a->dim == 0) return 0;
    MB_CHECK_ARG(a->ids && a->out && (a->table || a->vocab == 0), "embedding: null pointer");
    const int64_t et = (int64_t)dtype_size(a->table_dtype), eo = (int64_t)dtype_size(a->out_dtype);
    MB_CHECK_ARG(aligned_to(a->table, (size_t)et) && aligned_to(a->out, (size_t)eo),
                 "embedding: pointers must be aligned to their element type");
    MB_CHECK_ARG(a->out != a->table && a->out != a->ids, "embedding: out needs memory of its own");
    MB_CHECK_ARG(a->tokens == 1 || a->out_stride >= a->dim, "embedding: rows of out overlap (strides)");
    LookupParams p{};
    p.ids = a->ids;
    p.table = a->table;
    p.out = a->out;
    p.tokens = a->tokens;
    p.vocab = a->vocab;
    p.table_stride = a->table_stride;
    p.out_stride = a->out_stride;
    p.dim = a->dim;
    p.wide = a->id_bytes == 8;
    p.scale = a->scale;
    const bool vec = a->dim % 8 == 0 && aligned_to(a->table, 16) && aligned_to(a->out, 16) &&
                     (a->table_stride * et) % 16 == 0 && (a->out_stride * eo) % 16 == 0;
    const bool pairs = a->dim % 2 == 0 && aligned_to(a->table, (size_t)(2 * et)) && aligned_to(a->out, (size_t)(2 * eo)) &&
                       a->table_stride % 2 == 0 && a->out_stride % 2 == 0;
    if (a->table_dtype == MAMBA_F16)
        return a->out_dtype == MAMBA_F16 ? launch_lookup<__half, __half>(p, vec, pairs, st)
                                         : launch_lookup<__half, float>(p, vec, pairs, st);
    return a->out_dtype == MAMBA_F16 ? launch_lookup<float, __half>(p, vec, pairs, st)
                                     : launch_lookup<float, float>(p, vec, pairs, st);
}

size_t embedding_workspace_bytes(const MambaEmbeddingArgs *a) {
    if (!a || a->tokens <= 0 || a->dim <= 0 || a->tokens > kMaxTokens) return 0;
    return layout(a->tokens, a->dim).bytes;
}

int embedding_backward(const MambaEmbeddingArgs *a, const void *dout, int64_t dout_stride, float *dtable,
                       int64_t dtable_stride, int accumulate, void *ws, size_t ws_bytes, cudaStream_t st) {
    if (check_embedding(a, "embedding_backward")) return -1;
    if (a->vocab == 0 || a->dim == 0) return 0;
    MB_CHECK_ARG(dtable, "embedding_backward: null pointer");
    MB_CHECK_ARG(aligned_to(dtable, 4) && aligned_to(dout, dtype_size(a->out_dtype)),
                 "embedding_backward: pointers must be aligned to their element type");
    MB_CHECK_ARG(a->vocab == 1 || dtable_stride >= a->dim, "embedding_backward: rows of dtable overlap (strides)");
    if (a->tokens > 0) {
        MB_CHECK_ARG(a->ids && dout, "embedding_backward: null pointer");
        MB_CHECK_ARG(dtable != dout && dtable != a->ids, "embedding_backward: dtable needs memory of its own");
        MB_CHECK_ARG(ws && ws_bytes >= embedding_workspace_bytes(a) && aligned_to(ws, 16),
                     "embedding_backward: workspace too small or not 16-byte aligned");
    }
    if (a->tokens == 0) {
        if (accumulate) return 0;
        const size_t row = (size_t)a->dim * 4, pitch = a->vocab == 1 ? row : (size_t)dtable_stride * 4;
        if (pitch == row)
            MB_CUDA_TRY(cudaMemsetAsync(dtable, 0, row * (size_t)a->vocab, st));
        else
            MB_CUDA_TRY(cudaMemset2DAsync(dtable, pitch, 0, row, (size_t)a->vocab, st));
        return 0;
    }
    const Layout l = layout(a->tokens, a->dim);
    uint8_t *base = static_cast<uint8_t *>(ws);
    SortPass s{};
    s.n = (uint32_t)a->tokens;
    s.vocab = (uint32_t)a->vocab;
    s.tiles = l.tiles;
    s.few = l.tiles <= kFewTiles;
    s.wide = a->id_bytes == 8;
    s.hist = reinterpret_cast<uint32_t *>(base + l.hist);
    s.bits = 1;
    while (s.bits < 32 && (a->vocab >> s.bits) != 0) ++s.bits;  // keys are 0 .. vocab
    auto words = [&](size_t o) { return reinterpret_cast<uint32_t *>(base + o); };
    if (a->tokens <= kSmallCtas * kTinyTokens) {
        s.ids = a->ids;
        s.keys_out = words(l.keys[0]);
        s.pos_out = words(l.pos[0]);
        if (a->tokens <= kTinyTokens ? launch_small<1>(s, st) : launch_small<kSmallCtas>(s, st)) return -1;
    } else {
        int to = 0;
        for (s.shift = 0; s.shift < s.bits; s.shift += kDigitBits, to ^= 1) {
            s.ids = s.shift == 0 ? a->ids : nullptr;
            s.keys_in = words(l.keys[to ^ 1]);
            s.pos_in = words(l.pos[to ^ 1]);
            s.keys_out = words(l.keys[to]);
            s.pos_out = words(l.pos[to]);
            sort_count_kernel<<<(unsigned)l.tiles, kSortThreads, 0, st>>>(s);
            if (!s.few) sort_sum_kernel<<<1, 1024, 0, st>>>(s.hist, (uint32_t)l.tiles * kDigits);
            sort_move_kernel<<<(unsigned)l.tiles, kSortThreads, 0, st>>>(s);
            if (launch_status("embedding_backward sort kernels")) return -1;
        }
    }
    SumParams p{};
    p.keys = s.keys_out;
    p.pos = s.pos_out;
    p.dout = dout;
    p.dtable = dtable;
    p.part = reinterpret_cast<float *>(base + l.part);
    p.dout_stride = dout_stride;
    p.table_stride = dtable_stride;
    p.n = s.n;
    p.vocab = s.vocab;
    p.dim = a->dim;
    p.parts = l.parts;
    p.len = part_length(a->tokens);
    p.scale = a->scale;
    p.accumulate = accumulate != 0;
    const bool vec = a->dim % 8 == 0 && aligned_to(dout, 16) && aligned_to(dtable, 16) && dtable_stride % 4 == 0 &&
                     (dout_stride * (int64_t)dtype_size(a->out_dtype)) % 16 == 0;
    const bool pairs = a->dim % 2 == 0 && aligned_to(dout, 2 * dtype_size(a->out_dtype)) && aligned_to(dtable, 8) &&
                       dtable_stride % 2 == 0 && dout_stride % 2 == 0;
    // up to 2048 columns a CTA
    if (a->out_dtype == MAMBA_F16) {
        if (vec) return launch_sums<__half, 8, 1>(p, st);
        return pairs ? launch_sums<__half, 2, 4>(p, st) : launch_sums<__half, 1, 8>(p, st);
    }
    if (vec) return launch_sums<float, 4, 2>(p, st);
    return pairs ? launch_sums<float, 2, 4>(p, st) : launch_sums<float, 1, 8>(p, st);
}

}  // namespace mb
