// embedding.cu -- embedding lookup with scaling, and the table's gradient:
//   out[t] = scale * table[id_t]                      (0 for ids outside the table)
//   dtable[v] = scale * sum_{t : id_t = v} dout[t]    (in order of t)
//
// Lookup: a gather, bound by bytes (the rows that occur, once, and out).
//
// Gradient: no atomics, so that the sums have one order.  The ids are sorted
// with their positions (stable, least significant digit first), the sorted
// list is cut into chunks of equal length, and one CTA sums the rows of a
// chunk, id by id.  An id that lies within one chunk is finished there; the
// sums of one that spans several leave as partial rows, which a second kernel
// adds in order.  Frequent ids so cost no more than others.
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace mb {
namespace {

// ---- lookup -------------------------------------------------------------------
constexpr int kLookupThreads = 256;
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
template <typename TT, typename TO, int VEC>
__global__ void __launch_bounds__(kLookupThreads) embedding_kernel(const LookupParams p) {
    const int64_t t0 = (int64_t)blockIdx.x * (blockDim.y * kLookupTokens) + threadIdx.y;
    int64_t id[kLookupTokens];
#pragma unroll
    for (int k = 0; k < kLookupTokens; ++k) {
        const int64_t t = t0 + k * blockDim.y;
        id[k] = t < p.tokens ? token_id(p.ids, p.wide, t) : -1;
        if (id[k] >= p.vocab) id[k] = -1;
    }
    for (int c = threadIdx.x * VEC; c < p.dim; c += blockDim.x * VEC) {
        float v[kLookupTokens][VEC];
#pragma unroll
        for (int k = 0; k < kLookupTokens; ++k) {
            if (id[k] >= 0) {
                load_n(static_cast<const TT *>(p.table) + id[k] * p.table_stride + c, v[k]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < kLookupTokens; ++k) {
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

template <typename TT, typename TO>
int launch_lookup(const LookupParams &p, bool vec, cudaStream_t st) {
    const int tx = std::min(kLookupThreads, pow2_at_least(vec ? p.dim / 8 : p.dim)), ty = kLookupThreads / tx;
    const int64_t grid = ceil_div64(p.tokens, (int64_t)ty * kLookupTokens);
    MB_CHECK_ARG(grid <= 0x7fffffff, "embedding: too many tokens");
    if (vec)
        embedding_kernel<TT, TO, 8><<<(unsigned)grid, dim3(tx, ty), 0, st>>>(p);
    else
        embedding_kernel<TT, TO, 1><<<(unsigned)grid, dim3(tx, ty), 0, st>>>(p);
    return launch_status("embedding kernel");
}

// ---- sort -----------------------------------------------------------------------
constexpr int kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 512, kSortItems = 8, kSortTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32;

// Key of a token: its id, or `vocab` (behind all ids) for one outside the table.
__device__ __forceinline__ uint32_t token_key(const void *ids, bool wide, int64_t t, uint32_t vocab) {
    const int64_t id = token_id(ids, wide, t);
    return id >= 0 && id < (int64_t)vocab ? (uint32_t)id : vocab;
}

struct SortPass {
    const void *ids;  // first pass: the keys come from here; NULL: from keys_in, pos_in
    const uint32_t *keys_in, *pos_in;
    uint32_t *keys_out, *pos_out;
    uint32_t *hist;  // [kDigits][tiles]: counts, then first places
    uint32_t n, vocab;
    int shift, tiles;
    bool wide;
};
__device__ __forceinline__ uint32_t pass_key(const SortPass &p, uint32_t i) {
    return p.ids ? token_key(p.ids, p.wide, i, p.vocab) : p.keys_in[i];
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
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) p.hist[(size_t)d * p.tiles + blockIdx.x] = count[d];
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
// w * 32 * kSortItems + k * 32 + lane and counts its digits round by round (the
// lanes of one digit find each other by a match), so equal digits keep their order.
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(const SortPass p) {
    __shared__ uint32_t count[kSortWarps][kDigits];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int d = threadIdx.x; d < kSortWarps * kDigits; d += kSortThreads) count[d / kDigits][d % kDigits] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (uint32_t)kSortTile + warp * (32 * kSortItems);
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = base + k * 32 + lane;
        key[k] = i < p.n ? pass_key(p, i) : 0;
    }
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = base + k * 32 + lane;
        const uint32_t d = i < p.n ? key[k] >> p.shift & (kDigits - 1) : kDigits;  // kDigits: no item
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        const uint32_t before = d < kDigits ? count[warp][d] : 0;
        rank[k] = before + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (d < kDigits && lane == __ffs(same) - 1) count[warp][d] = before + __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
        uint32_t run = p.hist[(size_t)d * p.tiles + blockIdx.x];
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = count[w][d];
            count[w][d] = run;
            run += c;
        }
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

// ---- sums -----------------------------------------------------------------------
constexpr int kChunk = 16;       // sorted tokens per CTA
constexpr int kSumRows = 8;      // rows a thread has in flight
constexpr int kSumCtaThreads = 256;

struct SumParams {
    const uint32_t *keys, *pos;
    const void *dout;
    float *dtable;
    float *part;  // [chunks][2][dim]: slot 0 an id begun in an earlier chunk, 1 one that goes on in the next
    int64_t dout_stride, table_stride;
    uint32_t n, vocab;
    int dim, chunks;
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

// blockIdx.x: chunk; blockIdx.y: block of columns.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumCtaThreads) embedding_sum_kernel(const SumParams p) {
    __shared__ uint32_t key[kChunk + 2], pos[kChunk];  // key[1 + k]: token k of the chunk, around it its neighbours
    const uint32_t first = blockIdx.x * (uint32_t)kChunk;
    if (threadIdx.x < kChunk + 2) {
        const uint32_t i = first + threadIdx.x - 1;  // wraps at -1: beyond n
        key[threadIdx.x] = i < p.n ? p.keys[i] : p.vocab;
    }
    if (threadIdx.x < kChunk) pos[threadIdx.x] = first + threadIdx.x < p.n ? p.pos[first + threadIdx.x] : 0;
    __syncthreads();
    const int c = (blockIdx.y * kSumCtaThreads + threadIdx.x) * VEC;
    if (c >= p.dim) return;
    float sum[VEC] = {};
    bool begun = key[0] == key[1] && first > 0;  // the current id begun in an earlier chunk
#pragma unroll 1
    for (int k0 = 0; k0 < kChunk; k0 += kSumRows) {
        float v[kSumRows][VEC];
#pragma unroll
        for (int k = 0; k < kSumRows; ++k)
            if (key[1 + k0 + k] < p.vocab)
                load_n(static_cast<const T *>(p.dout) + (int64_t)pos[k0 + k] * p.dout_stride + c, v[k]);
#pragma unroll
        for (int k = 0; k < kSumRows; ++k) {
            const uint32_t id = key[1 + k0 + k];
            if (id >= p.vocab) return;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] += v[k][e];
            const bool last = k0 + k == kChunk - 1, ends = key[2 + k0 + k] != id;
            if (ends || last) {
                if (!begun && ends)
                    put_row(p, id, c, sum);
                else
                    store_n(p.part + ((int64_t)blockIdx.x * 2 + (begun ? 0 : 1)) * p.dim + c, sum);
                begun = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
            }
        }
    }
}

// blockIdx.x: the chunk in which an id begins that goes on in the next ones.
template <int VEC>
__global__ void __launch_bounds__(kSumCtaThreads) embedding_join_kernel(const SumParams p) {
    const uint32_t first = blockIdx.x * (uint32_t)kChunk, end = first + kChunk;  // end: the next chunk's first
    if (end >= p.n) return;
    const uint32_t id = p.keys[end];
    if (id >= p.vocab || p.keys[end - 1] != id) return;
    if (first > 0 && p.keys[first - 1] == id) return;  // begun earlier
    // one behind the id's last token
    uint32_t lo = end, hi = p.n;
    while (lo + 1 < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (p.keys[mid] == id)
            lo = mid;
        else
            hi = mid;
    }
    const int last = (int)(lo / kChunk);
    const int c = (blockIdx.y * kSumCtaThreads + threadIdx.x) * VEC;
    if (c >= p.dim) return;
    float sum[VEC];
    load_n(p.part + ((int64_t)blockIdx.x * 2 + 1) * p.dim + c, sum);
#pragma unroll 4
    for (int k = blockIdx.x + 1; k <= last; ++k) {
        float v[VEC];
        load_n(p.part + (int64_t)k * 2 * p.dim + c, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += v[e];
    }
    put_row(p, id, c, sum);
}

template <typename T>
int launch_sums(const SumParams &p, bool vec, cudaStream_t st) {
    const dim3 grid((unsigned)p.chunks, (unsigned)ceil_div(vec ? p.dim / 8 : p.dim, kSumCtaThreads));
    if (vec) {
        embedding_sum_kernel<T, 8><<<grid, kSumCtaThreads, 0, st>>>(p);
        embedding_join_kernel<8><<<grid, kSumCtaThreads, 0, st>>>(p);
    } else {
        embedding_sum_kernel<T, 1><<<grid, kSumCtaThreads, 0, st>>>(p);
        embedding_join_kernel<1><<<grid, kSumCtaThreads, 0, st>>>(p);
    }
    return launch_status("embedding_backward sum kernels");
}

struct Layout {
    size_t keys[2], pos[2], hist, part, bytes;
    int tiles, chunks;
};
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
Layout layout(int64_t n, int dim) {
    Layout l{};
    l.tiles = (int)ceil_div64(n, kSortTile);
    l.chunks = (int)ceil_div64(n, kChunk);
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
    at += up256((size_t)l.chunks * 2 * dim * 4);
    l.bytes = at;
    return l;
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
    if (a->table_dtype == MAMBA_F16)
        return a->out_dtype == MAMBA_F16 ? launch_lookup<__half, __half>(p, vec, st)
                                         : launch_lookup<__half, float>(p, vec, st);
    return a->out_dtype == MAMBA_F16 ? launch_lookup<float, __half>(p, vec, st) : launch_lookup<float, float>(p, vec, st);
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
    const size_t row = (size_t)a->dim * 4, pitch = a->vocab == 1 ? row : (size_t)dtable_stride * 4;
    if (!accumulate) {
        if (pitch == row)
            MB_CUDA_TRY(cudaMemsetAsync(dtable, 0, row * (size_t)a->vocab, st));
        else
            MB_CUDA_TRY(cudaMemset2DAsync(dtable, pitch, 0, row, (size_t)a->vocab, st));
    }
    if (a->tokens == 0) return 0;
    const Layout l = layout(a->tokens, a->dim);
    uint8_t *base = static_cast<uint8_t *>(ws);
    SortPass s{};
    s.n = (uint32_t)a->tokens;
    s.vocab = (uint32_t)a->vocab;
    s.tiles = l.tiles;
    s.wide = a->id_bytes == 8;
    s.hist = reinterpret_cast<uint32_t *>(base + l.hist);
    int bits = 1;
    while (bits < 32 && (a->vocab >> bits) != 0) ++bits;  // keys are 0 .. vocab
    int to = 0;
    for (s.shift = 0; s.shift < bits; s.shift += kDigitBits, to ^= 1) {
        s.ids = s.shift == 0 ? a->ids : nullptr;
        s.keys_in = reinterpret_cast<uint32_t *>(base + l.keys[to ^ 1]);
        s.pos_in = reinterpret_cast<uint32_t *>(base + l.pos[to ^ 1]);
        s.keys_out = reinterpret_cast<uint32_t *>(base + l.keys[to]);
        s.pos_out = reinterpret_cast<uint32_t *>(base + l.pos[to]);
        sort_count_kernel<<<(unsigned)l.tiles, kSortThreads, 0, st>>>(s);
        sort_sum_kernel<<<1, 1024, 0, st>>>(s.hist, (uint32_t)l.tiles * kDigits);
        sort_move_kernel<<<(unsigned)l.tiles, kSortThreads, 0, st>>>(s);
        if (launch_status("embedding_backward sort kernels")) return -1;
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
    p.chunks = l.chunks;
    p.scale = a->scale;
    p.accumulate = accumulate != 0;
    const bool vec = a->dim % 8 == 0 && aligned_to(dout, 16) && aligned_to(dtable, 16) && dtable_stride % 4 == 0 &&
                     (dout_stride * (int64_t)dtype_size(a->out_dtype)) % 16 == 0;
    return a->out_dtype == MAMBA_F16 ? launch_sums<__half>(p, vec, st) : launch_sums<float>(p, vec, st);
}

}  // namespace mb
