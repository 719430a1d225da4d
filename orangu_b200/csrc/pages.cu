// Operators over the pages of a cache that the caller holds: the entry points ob_pages_* (checks, handle, workspace), and the kernels that
// move pages and positions or bound the keys of a page.  Attention is in pages_attention.cu, the choice of pages in pages_select.cu.
//
// What moves data is bound by its bytes: whole 16-byte words, several in flight per thread, one launch for all layers, keys and
// values.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "mixers_common.cuh"
#include "pages.h"
#include "runtime.h"

using namespace obrt;

struct ob_pages {
    ob_ctx *ctx;
    ob_pages_desc d;
    uint64_t layer_bytes;  // from a layer's pages to the next one's
    uint8_t *workspace;    // PG_COUNTERS words that are zero between launches, as many PagePiece, then partial results
    std::vector<PageMaps> maps;  // of every layer
};

namespace {

struct MoveArgs {
    uint8_t *k, *v;
    uint64_t layer_bytes;
    uint32_t n_pages, n_kv, row_bytes;  // of one position's key or value
    int32_t *tables;
    uint32_t n_seq, stride;
    __device__ __forceinline__ uint8_t *pool(uint32_t layer, uint32_t value) const { return (value ? v : k) + layer * layer_bytes; }
    __device__ __forceinline__ uint64_t page_bytes() const { return (uint64_t)n_kv * KV_PAGE * row_bytes; }
};

constexpr uint32_t MOVE_THREADS = 256, MOVE_WORDS = 4;  // 16-byte words of a thread in flight

// One page of one layer's keys or values; the whole CTA.
__device__ __forceinline__ void copy_page(const uint8_t *src, uint8_t *dst, uint32_t words) {
    const uint4 *s = reinterpret_cast<const uint4 *>(src);
    uint4 *d = reinterpret_cast<uint4 *>(dst);
    uint32_t i = threadIdx.x;
    for (; i + (MOVE_WORDS - 1) * MOVE_THREADS < words; i += MOVE_WORDS * MOVE_THREADS) {
        uint4 x[MOVE_WORDS];
#pragma unroll
        for (uint32_t u = 0; u < MOVE_WORDS; ++u) x[u] = __ldcs(s + i + u * MOVE_THREADS);
#pragma unroll
        for (uint32_t u = 0; u < MOVE_WORDS; ++u) __stcs(d + i + u * MOVE_THREADS, x[u]);
    }
    for (; i < words; i += MOVE_THREADS) __stcs(d + i, __ldcs(s + i));
}

// grid (pairs, layers x 2)
__global__ void __launch_bounds__(MOVE_THREADS) pages_copy_kernel(const __grid_constant__ MoveArgs a, const int32_t *__restrict__ src, const int32_t *__restrict__ dst) {
    ob::pdl_wait();
    const int32_t s = src[blockIdx.x], d = dst[blockIdx.x];
    if ((uint32_t)s >= a.n_pages || (uint32_t)d >= a.n_pages || s == d) return;
    uint8_t *pool = a.pool(blockIdx.y >> 1, blockIdx.y & 1);
    copy_page(pool + (uint64_t)s * a.page_bytes(), pool + (uint64_t)d * a.page_bytes(), (uint32_t)(a.page_bytes() / 16));
}

// grid (children, layers x 2 + 1): the last row of CTAs writes the tables
__global__ void __launch_bounds__(MOVE_THREADS) pages_fork_kernel(const __grid_constant__ MoveArgs a, uint32_t n_layer, const int32_t *__restrict__ parent,
                                                                  const int32_t *__restrict__ child, const uint32_t *__restrict__ n_pos, const int32_t *__restrict__ fresh) {
    ob::pdl_wait();
    const int32_t p = parent[blockIdx.x], c = child[blockIdx.x], f = fresh[blockIdx.x];
    if ((uint32_t)p >= a.n_seq || (uint32_t)c >= a.n_seq || p == c) return;
    const uint32_t n = min(n_pos[blockIdx.x], a.stride * KV_PAGE), whole = n / KV_PAGE;
    const int32_t *from = a.tables + (uint64_t)p * a.stride;
    if (blockIdx.y == 2 * n_layer) {
        int32_t *to = a.tables + (uint64_t)c * a.stride;
        for (uint32_t i = threadIdx.x; i < whole; i += MOVE_THREADS) to[i] = from[i];
        if (threadIdx.x == 0 && n % KV_PAGE) to[whole] = f;
        return;
    }
    if (n % KV_PAGE == 0) return;
    const int32_t s = from[whole];
    if ((uint32_t)s >= a.n_pages || (uint32_t)f >= a.n_pages || s == f) return;
    uint8_t *pool = a.pool(blockIdx.y >> 1, blockIdx.y & 1);
    copy_page(pool + (uint64_t)s * a.page_bytes(), pool + (uint64_t)f * a.page_bytes(), (uint32_t)(a.page_bytes() / 16));
}

// grid (sequences, layers x 2, groups of heads): every word is read before the first is written.  A thread holds KEEP_WORDS of the
// words (head, j, 16 bytes); `heads` of them a CTA so that they fit.
constexpr uint32_t KEEP_WORDS = 4;
__global__ void __launch_bounds__(MOVE_THREADS) pages_keep_kernel(const __grid_constant__ MoveArgs a, uint32_t most, const uint32_t *__restrict__ n_ctx, const int32_t *__restrict__ kept,
                                                                  uint32_t kept_stride, const uint32_t *__restrict__ n_kept) {
    __shared__ uint64_t s_from[64], s_to[64];  // bytes of head 0's row in a layer's pool; ~0: none
    ob::pdl_wait();
    const uint32_t n = min(n_kept[blockIdx.x], most), ctx = n_ctx[blockIdx.x];
    if (n == 0) return;
    const int32_t *table = a.tables + (uint64_t)blockIdx.x * a.stride;
    if (threadIdx.x < 2 * n) {
        const uint32_t j = threadIdx.x >> 1;
        const int32_t i = threadIdx.x & 1 ? kept[(uint64_t)blockIdx.x * kept_stride + j] : (int32_t)j;
        uint64_t at = ~0ull;
        const uint64_t x = (uint64_t)ctx + (uint32_t)i;
        if ((uint32_t)i < 64 && x < (uint64_t)a.stride * KV_PAGE) {
            const int32_t id = table[x / KV_PAGE];
            if ((uint32_t)id < a.n_pages) at = (uint64_t)id * a.page_bytes() + x % KV_PAGE * a.row_bytes;
        }
        (threadIdx.x & 1 ? s_from : s_to)[j] = at;
    }
    __syncthreads();
    uint8_t *pool = a.pool(blockIdx.y >> 1, blockIdx.y & 1);
    const uint32_t row = a.row_bytes / 16, head_words = n * row, fit = max(1u, KEEP_WORDS * MOVE_THREADS / head_words);
    for (uint32_t h0 = blockIdx.z * fit; h0 < a.n_kv; h0 += gridDim.z * fit) {
        const uint32_t words = min(fit, a.n_kv - h0) * head_words;
        uint4 x[KEEP_WORDS];
        uint8_t *to[KEEP_WORDS];
#pragma unroll
        for (uint32_t u = 0; u < KEEP_WORDS; ++u) {
            const uint32_t i = u * MOVE_THREADS + threadIdx.x, h = h0 + i / head_words, j = i % head_words / row, c = i % row;
            to[u] = nullptr;
            if (i < words && s_from[j] != ~0ull && s_to[j] != ~0ull && s_from[j] != s_to[j]) {
                const uint64_t off = (uint64_t)h * KV_PAGE * a.row_bytes + c * 16;
                x[u] = *reinterpret_cast<const uint4 *>(pool + s_from[j] + off);
                to[u] = pool + s_to[j] + off;
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < KEEP_WORDS; ++u)
            if (to[u]) *reinterpret_cast<uint4 *>(to[u]) = x[u];
    }
}

// Bounds of a page's keys.  A warp per (page, head): 16 bytes a lane, HD / 8 lanes a row, the lanes' maxima and minima of f16 or bf16 pairs;
// then the unit d = max(|hi|, |lo|) / 127 and the codes ceil(hi / d), floor(lo / d), so that a code times d is no tighter than the keys
// (by more than the division's rounding).  Reading the keys bounds it.
template <typename T> struct Pair;
template <> struct Pair<__half> {
    using V = __half2;
    static __device__ __forceinline__ float2 f(V v) { return __half22float2(v); }
};
template <> struct Pair<bf16> {
    using V = __nv_bfloat162;
    static __device__ __forceinline__ float2 f(V v) { return __bfloat1622float2(v); }
};
constexpr float BOUND_MOST = 1e18f;  // what larger keys count as: the scores stay finite
__device__ __forceinline__ float bounded(float v) { return v != v ? 0.0f : fminf(fmaxf(v, -BOUND_MOST), BOUND_MOST); }

template <typename T, int HD>
__global__ void __launch_bounds__(256) pages_bounds_kernel(const __grid_constant__ PageView pg, const uint32_t *__restrict__ first_pos, const uint32_t *__restrict__ n_pos, int8_t *codes, float *scales) {
    using V = typename Pair<T>::V;
    constexpr uint32_t LANES = HD / 8, STEP = 32 / LANES, ROWS = KV_PAGE / STEP;  // lanes a row, rows a load, loads
    ob::pdl_wait();
    const uint32_t lane = threadIdx.x & 31, unit = blockIdx.x * 8 + (threadIdx.x >> 5), seq = blockIdx.y, room = pg.stride * KV_PAGE;
    const uint32_t from = first_pos[seq], to = min(n_pos[seq], room);
    const uint32_t page = from / KV_PAGE + unit / pg.n_kv, head = unit % pg.n_kv;
    if (from >= to || page >= (to + KV_PAGE - 1) / KV_PAGE) return;
    const int32_t id = pg.tables[(uint64_t)seq * pg.stride + page];
    if ((uint32_t)id >= pg.n_pages) return;
    const uint32_t filled = min(to - page * KV_PAGE, (uint32_t)KV_PAGE);
    const uint64_t at = (uint64_t)id * pg.n_kv + head;
    const uint4 *k = reinterpret_cast<const uint4 *>(static_cast<const T *>(pg.k) + at * KV_PAGE * HD);
    uint4 x[ROWS];
#pragma unroll
    for (uint32_t i = 0; i < ROWS; ++i) {
        const uint32_t row = i * STEP + lane / LANES;
        x[i] = ob::ldg128_stream(k + (row < filled ? i * 32 + lane : lane % LANES));  // rows that are not filled: the first one again
    }
    V hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) hi[e] = lo[e] = reinterpret_cast<const V *>(&x[0])[e];
#pragma unroll
    for (uint32_t i = 1; i < ROWS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const V v = reinterpret_cast<const V *>(&x[i])[e];
            hi[e] = __hmax2(hi[e], v), lo[e] = __hmin2(lo[e], v);
        }
#pragma unroll
    for (uint32_t o = LANES; o < 32; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            hi[e] = __hmax2(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
            lo[e] = __hmin2(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
        }
    float h[8], l[8], top = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 a = Pair<T>::f(hi[e]), b = Pair<T>::f(lo[e]);
        h[2 * e] = bounded(a.x), h[2 * e + 1] = bounded(a.y), l[2 * e] = bounded(b.x), l[2 * e + 1] = bounded(b.y);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(fabsf(h[e]), fabsf(l[e])));
    top = ob::warp_max(top);
    const float d = __fdiv_rn(top, 127.0f), by = d > 0.0f ? d : 1.0f;
    if (lane < 2 * LANES) {  // the first LANES lanes write the largest, the next ones the smallest
        const bool low = lane >= LANES;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float c = low ? floorf(__fdiv_rn(l[e], by)) : ceilf(__fdiv_rn(h[e], by));
            w[e / 4] |= ((uint32_t)(int)fminf(fmaxf(c, -127.0f), 127.0f) & 255u) << (e % 4 * 8);
        }
        *reinterpret_cast<uint2 *>(codes + at * 2 * HD + lane * 8) = make_uint2(w[0], w[1]);
    }
    if (lane == 0) scales[at] = d;
}

// ---------------------------------------------------------------------------------------------------- checks
int bad(const ob_pages *p, const char *who, const char *what) { return fail(p ? p->ctx : nullptr, OB_ERR_INVALID, std::string(who) + ": " + what); }
bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Device memory of the context's GPU.
bool on_device(const ob_ctx *ctx, const void *p) {
    cudaPointerAttributes at{};
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return (at.type == cudaMemoryTypeDevice && at.device == ctx->device) || at.type == cudaMemoryTypeManaged;
}
struct Named {
    const void *p;
    const char *name;
    size_t align;
};
template <size_t N>
int check_pointers(ob_pages *p, const char *who, const Named (&list)[N]) {
    for (const Named &n : list) {
        if (!n.p) return fail(p->ctx, OB_ERR_INVALID, std::string(who) + ": " + n.name + " is null");
        if (!aligned(n.p, n.align)) return fail(p->ctx, OB_ERR_INVALID, std::string(who) + ": " + n.name + " is not aligned to " + std::to_string(n.align) + " bytes");
        if (!on_device(p->ctx, n.p)) return fail(p->ctx, OB_ERR_INVALID, std::string(who) + ": " + n.name + " is not memory of the context's device");
    }
    return OB_OK;
}
// Queries or outputs: rows of n_head vectors.
int check_rows(ob_pages *p, const char *who, const char *name, uint64_t stride, uint32_t n_head) {
    if (stride < (uint64_t)n_head * p->d.head_dim || stride % 8)
        return fail(p->ctx, OB_ERR_INVALID, std::string(who) + ": " + name + " has to be a multiple of 8 and at least n_head * head_dim");
    return OB_OK;
}
int check_heads(ob_pages *p, const char *who, uint32_t n_head) {
    if (n_head == 0 || n_head % p->d.n_head_kv) return fail(p->ctx, OB_ERR_INVALID, std::string(who) + ": n_head has to be a multiple of n_head_kv");
    if (n_head / p->d.n_head_kv > PG_MAX_GROUP) return fail(p->ctx, OB_ERR_UNSUPPORTED, std::string(who) + ": more than 16 query heads per key/value head");
    return OB_OK;
}

PageView view(const ob_pages *p, uint32_t layer) {
    const ob_pages_desc &d = p->d;
    PageView v{};
    v.k = static_cast<const uint8_t *>(d.k) + layer * p->layer_bytes;
    v.v = static_cast<const uint8_t *>(d.v) + layer * p->layer_bytes;
    v.is_bf16 = d.type == OB_TYPE_BF16;
    v.n_pages = d.n_pages, v.n_kv = d.n_head_kv, v.dim = d.head_dim;
    v.tables = d.tables, v.n_seq = d.n_seq, v.stride = d.table_stride;
    return v;
}
MoveArgs moves(const ob_pages *p) {
    const ob_pages_desc &d = p->d;
    return MoveArgs{static_cast<uint8_t *>(d.k), static_cast<uint8_t *>(d.v), p->layer_bytes, d.n_pages, d.n_head_kv, d.head_dim * 2, d.tables, d.n_seq, d.table_stride};
}
void use_workspace(const ob_pages *p, PagedAttnArgs &a) {
    a.counters = reinterpret_cast<uint32_t *>(p->workspace);
    a.pieces = reinterpret_cast<PagePiece *>(p->workspace + PG_COUNTERS * 4);
    a.partial = reinterpret_cast<float *>(p->workspace + PG_COUNTERS * (4 + sizeof(PagePiece)));
}
cudaStream_t stream_of(const ob_pages *p, void *stream) { return stream ? static_cast<cudaStream_t>(stream) : p->ctx->stream; }
int launched(ob_pages *p, const char *who, cudaError_t e, uint32_t kernels = 1) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(p->ctx, OB_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
    }
    p->ctx->launches += kernels;
    return OB_OK;
}

}  // namespace

extern "C" {

int ob_pages_create(ob_ctx *ctx, const ob_pages_desc *desc, ob_pages **out) {
    if (out) *out = nullptr;
    if (!ctx || !desc || !out) return fail(ctx, OB_ERR_INVALID, "pages_create: null argument");
    const ob_pages_desc &d = *desc;
    std::lock_guard<std::mutex> g(ctx->mu);
    Bind b(ctx);
    if (d.type != OB_TYPE_F16 && d.type != OB_TYPE_BF16) return fail(ctx, OB_ERR_UNSUPPORTED, "pages_create: pages are f16 (OB_TYPE_F16) or bfloat16 (OB_TYPE_BF16)");
    if (d.head_dim != 64 && d.head_dim != 128) return fail(ctx, OB_ERR_UNSUPPORTED, "pages_create: head_dim has to be 64 or 128");
    if (!d.n_layer || !d.n_pages || !d.n_head_kv || !d.n_seq || !d.table_stride) return fail(ctx, OB_ERR_INVALID, "pages_create: a size is zero");
    if (d.n_layer > 16383 || d.n_head_kv > 4096 || d.n_pages > 0x7fffffffu || d.table_stride > (1u << 27) || d.n_seq > (1u << 24))
        return fail(ctx, OB_ERR_UNSUPPORTED, "pages_create: a size is too large");
    const uint64_t elems = (uint64_t)d.n_pages * d.n_head_kv * KV_PAGE * d.head_dim;
    if (d.n_layer > 1 && (d.layer_stride < elems || d.layer_stride % 8)) return fail(ctx, OB_ERR_INVALID, "pages_create: layer_stride has to be a multiple of 8 and at least a layer's pages");
    if (!d.k || !d.v || !d.tables) return fail(ctx, OB_ERR_INVALID, "pages_create: null argument");
    if (!aligned(d.k, 16) || !aligned(d.v, 16) || !aligned(d.tables, 4)) return fail(ctx, OB_ERR_INVALID, "pages_create: pages have to be aligned to 16 bytes, tables to 4");
    if (!on_device(ctx, d.k) || !on_device(ctx, d.v) || !on_device(ctx, d.tables)) return fail(ctx, OB_ERR_INVALID, "pages_create: pages and tables have to be memory of the context's device");
    ob_pages *p = new (std::nothrow) ob_pages{ctx, d, d.n_layer > 1 ? d.layer_stride * 2 : 0, nullptr, {}};
    if (!p) return fail(ctx, OB_ERR_OOM, "pages_create: out of memory");
    p->maps.resize(d.n_layer);
    for (uint32_t l = 0; l < d.n_layer; ++l)
        if (!make_page_maps(view(p, l), &p->maps[l])) {
            delete p;
            return fail(ctx, OB_ERR_UNSUPPORTED, "pages_create: no tensor map of the pages can be made (n_pages * n_head_kv * 16 rows have to be below 2^31)");
        }
    void *ws = nullptr;
    cudaError_t e = cudaMalloc(&ws, PG_WORKSPACE);
    if (e == cudaSuccess) {
        e = cudaMemsetAsync(ws, 0, PG_COUNTERS * 4, ctx->stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);  // calls come on any stream
        if (e != cudaSuccess) cudaFree(ws);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        delete p;
        return fail(ctx, e == cudaErrorMemoryAllocation ? OB_ERR_OOM : OB_ERR_CUDA, std::string("pages_create: ") + cudaGetErrorString(e));
    }
    p->workspace = static_cast<uint8_t *>(ws);
    *out = p;
    return OB_OK;
}

void ob_pages_destroy(ob_pages *p) {
    if (!p) return;
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    cudaFree(p->workspace);
    delete p;
}

int ob_pages_attention_tree(ob_pages *p, uint32_t layer, uint32_t n_seq, const void *q, uint64_t q_stride, uint32_t n_tokens, const int32_t *first_token, const uint32_t *n_ctx,
                            const uint64_t *visible, uint32_t n_head, uint32_t max_drafts, uint32_t max_ctx, float scale, void *out, uint64_t out_stride, void *stream) {
    const char *who = "pages_attention_tree";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (layer >= p->d.n_layer) return bad(p, who, "no such layer");
    if (n_seq > p->d.n_seq) return bad(p, who, "more sequences than tables");
    if (int rc = check_heads(p, who, n_head)) return rc;
    if (max_drafts > PG_MAX_DRAFTS) return fail(p->ctx, OB_ERR_UNSUPPORTED, "pages_attention_tree: more than 64 drafted tokens of a sequence");
    if (n_tokens > 0x7fffffffu) return bad(p, who, "too many tokens");
    if (!std::isfinite(scale) || scale <= 0.0f) return bad(p, who, "scale has to be finite and above zero");
    if (int rc = check_rows(p, who, "q_stride", q_stride, n_head)) return rc;
    if (int rc = check_rows(p, who, "out_stride", out_stride, n_head)) return rc;
    if (n_seq == 0 || n_tokens == 0 || max_drafts == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{q, "q", 16}, {first_token, "first_token", 4}, {n_ctx, "n_ctx", 4}, {visible, "visible", 8}, {out, "out", 16}})) return rc;
    PagedAttnArgs a{};
    a.pg = view(p, layer);
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.group = n_head / p->d.n_head_kv, a.n_units = n_seq, a.scale = scale;
    a.first = first_token, a.n_ctx = n_ctx, a.visible = visible, a.n_tokens = n_tokens, a.max_drafts = max_drafts, a.max_ctx = max_ctx;
    use_workspace(p, a);
    if (max_drafts * a.group > PG_FEW_ROWS) {
        // (the walk over all tiles counts them in 31 bits)
        if ((uint64_t)n_seq * p->d.n_head_kv * (((uint64_t)p->d.table_stride + 7) / 8) * ((max_drafts * a.group + 127) / 128) >= (1ull << 31))
            return fail(p->ctx, OB_ERR_CAPACITY, "pages_attention_tree: the tables of all sequences together have room for too many positions");
        return launched(p, who, launch_pages_tree_tc5(a, p->maps[layer], p->ctx->sm_count, stream_of(p, stream)), 2);
    }
    return launched(p, who, launch_pages_attention(a, true, p->ctx->sm_count, stream_of(p, stream)));
}

int ob_pages_attention(ob_pages *p, uint32_t layer, uint32_t n_rows, const void *q, uint64_t q_stride, const int32_t *row_seq, const uint32_t *n_pos, uint32_t n_head,
                       const int32_t *selected, uint32_t n_select, float scale, void *out, uint64_t out_stride, void *stream) {
    const char *who = "pages_attention";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (layer >= p->d.n_layer) return bad(p, who, "no such layer");
    if (!row_seq && n_rows > p->d.n_seq) return bad(p, who, "more rows than tables");
    if (int rc = check_heads(p, who, n_head)) return rc;
    if (n_rows > (1u << 24)) return bad(p, who, "too many rows");
    if (n_select == 0 || n_select > p->d.table_stride) return bad(p, who, "n_select has to be at least 1 and at most table_stride");
    if (!std::isfinite(scale) || scale <= 0.0f) return bad(p, who, "scale has to be finite and above zero");
    if (int rc = check_rows(p, who, "q_stride", q_stride, n_head)) return rc;
    if (int rc = check_rows(p, who, "out_stride", out_stride, n_head)) return rc;
    if (n_rows == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{q, "q", 16}, {n_pos, "n_pos", 4}, {selected, "selected", 4}, {out, "out", 16}})) return rc;
    if (row_seq)
        if (int rc = check_pointers(p, who, {{row_seq, "row_seq", 4}})) return rc;
    PagedAttnArgs a{};
    a.pg = view(p, layer);
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.group = n_head / p->d.n_head_kv, a.n_units = n_rows, a.scale = scale;
    a.list = selected, a.n_list = n_select, a.n_pos = n_pos, a.row_seq = row_seq;
    use_workspace(p, a);
    return launched(p, who, launch_pages_attention(a, false, p->ctx->sm_count, stream_of(p, stream)));
}

int ob_pages_select(ob_pages *p, const int8_t *codes, const float *scales, uint32_t n_rows, const void *q, uint64_t q_stride, const int32_t *row_seq, const uint32_t *n_pos, uint32_t n_head,
                    uint32_t max_pos, uint32_t n_select, uint32_t keep_first, uint32_t keep_last, int32_t *selected, void *stream) {
    const char *who = "pages_select";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (!row_seq && n_rows > p->d.n_seq) return bad(p, who, "more rows than tables");
    if (int rc = check_heads(p, who, n_head)) return rc;
    if (n_rows > (1u << 24)) return bad(p, who, "too many rows");
    if (n_select == 0 || n_select > p->d.table_stride) return bad(p, who, "n_select has to be at least 1 and at most table_stride");
    if ((uint64_t)keep_first + keep_last > n_select) return bad(p, who, "keep_first + keep_last is more than n_select");
    if (std::min<uint64_t>(((uint64_t)max_pos + KV_PAGE - 1) / KV_PAGE, p->d.table_stride) > PG_SELECT_PAGES)
        return fail(p->ctx, OB_ERR_CAPACITY, "pages_select: a row has more than " + std::to_string(PG_SELECT_PAGES) + " pages");
    if (int rc = check_rows(p, who, "q_stride", q_stride, n_head)) return rc;
    if (n_rows == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{codes, "codes", 16}, {scales, "scales", 4}, {q, "q", 16}, {n_pos, "n_pos", 4}, {selected, "selected", 4}})) return rc;
    if (row_seq)
        if (int rc = check_pointers(p, who, {{row_seq, "row_seq", 4}})) return rc;
    PagedSelectArgs a{};
    a.pg = view(p, 0);
    a.codes = codes, a.scales = scales, a.q = q, a.q_stride = q_stride, a.group = n_head / p->d.n_head_kv, a.n_rows = n_rows, a.n_pos = n_pos, a.row_seq = row_seq;
    a.max_pos = max_pos, a.n_select = n_select, a.keep_first = keep_first, a.keep_last = keep_last, a.selected = selected;
    a.keys = reinterpret_cast<uint32_t *>(p->workspace + PG_COUNTERS * (4 + sizeof(PagePiece)));
    uint32_t kernels = 0;
    const cudaError_t e = launch_pages_select(a, p->ctx->sm_count, stream_of(p, stream), &kernels);
    return launched(p, who, e, kernels);
}

int ob_pages_bounds(ob_pages *p, uint32_t layer, uint32_t n_seq, const uint32_t *first_pos, const uint32_t *n_pos, uint32_t max_new, int8_t *codes, float *scales, void *stream) {
    const char *who = "pages_bounds";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (layer >= p->d.n_layer) return bad(p, who, "no such layer");
    if (n_seq > p->d.n_seq) return bad(p, who, "more sequences than tables");
    if (n_seq > 65535) return fail(p->ctx, OB_ERR_UNSUPPORTED, "pages_bounds: more than 65535 sequences");
    if (n_seq == 0 || max_new == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{first_pos, "first_pos", 4}, {n_pos, "n_pos", 4}, {codes, "codes", 16}, {scales, "scales", 4}})) return rc;
    const PageView v = view(p, layer);
    const uint64_t pages = std::min<uint64_t>((uint64_t)(max_new - 1) / KV_PAGE + 2, p->d.table_stride);  // positions that do not begin a page touch one more
    const uint64_t ctas = (pages * v.n_kv + 7) / 8;
    if (ctas > 0x7fffffffull) return fail(p->ctx, OB_ERR_UNSUPPORTED, "pages_bounds: too many pages");
    const dim3 grid((uint32_t)ctas, n_seq);
    auto kernel = v.is_bf16 ? (v.dim == 64 ? pages_bounds_kernel<bf16, 64> : pages_bounds_kernel<bf16, 128>) : (v.dim == 64 ? pages_bounds_kernel<__half, 64> : pages_bounds_kernel<__half, 128>);
    return launched(p, who, ob::launch_pdl(kernel, grid, dim3(256), 0, stream_of(p, stream), v, first_pos, n_pos, codes, scales));
}

int ob_pages_copy(ob_pages *p, uint32_t n, const int32_t *src, const int32_t *dst, void *stream) {
    const char *who = "pages_copy";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (n > 0x7fffffffu) return bad(p, who, "too many pages");
    if (n == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{src, "src", 4}, {dst, "dst", 4}})) return rc;
    return launched(p, who, ob::launch_pdl(pages_copy_kernel, dim3(n, 2 * p->d.n_layer), dim3(MOVE_THREADS), 0, stream_of(p, stream), moves(p), src, dst));
}

int ob_pages_fork(ob_pages *p, uint32_t n, const int32_t *parent, const int32_t *child, const uint32_t *n_pos, const int32_t *fresh, void *stream) {
    const char *who = "pages_fork";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (n > 0x7fffffffu) return bad(p, who, "too many sequences");
    if (n == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{parent, "parent", 4}, {child, "child", 4}, {n_pos, "n_pos", 4}, {fresh, "fresh", 4}})) return rc;
    return launched(p, who, ob::launch_pdl(pages_fork_kernel, dim3(n, 2 * p->d.n_layer + 1), dim3(MOVE_THREADS), 0, stream_of(p, stream), moves(p), p->d.n_layer, parent, child, n_pos, fresh));
}

int ob_pages_keep(ob_pages *p, uint32_t n_seq, const uint32_t *n_ctx, const int32_t *kept, uint32_t kept_stride, const uint32_t *n_kept, void *stream) {
    const char *who = "pages_keep";
    if (!p) return bad(p, who, "null argument");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (n_seq > p->d.n_seq) return bad(p, who, "more sequences than tables");
    if (kept_stride == 0 || kept_stride > PG_MAX_DRAFTS) return bad(p, who, "kept_stride has to be 1 to 64");
    if (n_seq == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{n_ctx, "n_ctx", 4}, {kept, "kept", 4}, {n_kept, "n_kept", 4}})) return rc;
    // Heads are shared out over CTAs while there are few of them.
    const uint32_t z = std::min(p->d.n_head_kv, std::max(1u, (uint32_t)(4ull * p->ctx->sm_count / ((uint64_t)n_seq * 2 * p->d.n_layer))));
    return launched(p, who, ob::launch_pdl(pages_keep_kernel, dim3(n_seq, 2 * p->d.n_layer, z), dim3(MOVE_THREADS), 0, stream_of(p, stream), moves(p), kept_stride, n_ctx, kept, kept_stride, n_kept));
}

}  // extern "C"
