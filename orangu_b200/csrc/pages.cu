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
    ob_ctx *ctx;           // null once the context is gone
    ob_pages_desc d;
    uint64_t layer_bytes;  // from a layer's pages to the next one's
    PageWorkspace ws;      // PG_COUNTERS words that are zero between launches, as many PagePiece, then partial results
    uint32_t untold;       // who was not told of a wait that was given up: SYNCHRONIZE, PAGES_SYNCHRONIZE
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

// grid (pairs, layers x 2): a page of one pool lies together.  1.07 GB of pages copied: 319 us, 6.7 TB/s, the bytes.
__global__ void __launch_bounds__(MOVE_THREADS) pages_copy_kernel(const __grid_constant__ MoveArgs a, const int32_t *__restrict__ src, const int32_t *__restrict__ dst) {
    ob::pdl_release();
    ob::pdl_wait();
    const int32_t s = src[blockIdx.x], d = dst[blockIdx.x];
    if ((uint32_t)s >= a.n_pages || (uint32_t)d >= a.n_pages || s == d) return;
    uint8_t *pool = a.pool(blockIdx.y >> 1, blockIdx.y & 1);
    copy_page(pool + (uint64_t)s * a.page_bytes(), pool + (uint64_t)d * a.page_bytes(), (uint32_t)(a.page_bytes() / 16));
}

// grid (children, layers x 2 + 1): the last row of CTAs writes the tables.  Eight children at 1000 positions: 3.0 us in a graph, a launch and two reads that
// depend on each other.
__global__ void __launch_bounds__(MOVE_THREADS) pages_fork_kernel(const __grid_constant__ MoveArgs a, uint32_t n_layer, const int32_t *__restrict__ parent,
                                                                  const int32_t *__restrict__ child, const uint32_t *__restrict__ n_pos, const int32_t *__restrict__ fresh) {
    ob::pdl_release();
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

// x / d for x below 65536 by the high half of a product.
struct Divide {
    uint32_t d, m;
    __host__ __device__ explicit Divide(uint32_t by) : d(by), m(by > 1 ? 0xffffffffu / by + 1 : 0u) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return d > 1 ? __umulhi(x, m) : x; }
};

// grid (sequences, shares of the (layer, keys or values, head) pools): every word of a pool's head is read before the first is written.  A CTA
// takes as many of them at a time as its threads hold words (KEEP_WORDS of 16 bytes each), so that a few positions a head fill it, too.  64 sequences, 8
// positions each, 81 MB read and written: 13.9 us in a graph, 5.8 TB/s in pieces of 256 bytes.
constexpr uint32_t KEEP_WORDS = 4;
__global__ void __launch_bounds__(MOVE_THREADS, 6) pages_keep_kernel(const __grid_constant__ MoveArgs a, uint32_t pools, const Divide kv, uint32_t most, const uint32_t *__restrict__ n_ctx,
                                                                     const int32_t *__restrict__ kept, uint32_t kept_stride, const uint32_t *__restrict__ n_kept) {
    __shared__ uint64_t s_from[64], s_to[64];  // bytes of head 0's row in a layer's pool; equal: nothing to do
    ob::pdl_release();
    ob::pdl_wait();
    {
        const uint32_t j = threadIdx.x >> 1, ctx = n_ctx[blockIdx.x];
        const int32_t i = j < most && (threadIdx.x & 1) ? kept[(uint64_t)blockIdx.x * kept_stride + j] : (int32_t)j;
        const uint64_t x = (uint64_t)ctx + (uint32_t)i;
        uint64_t at = ~0ull;
        if (j < most && (uint32_t)i < 64 && x < (uint64_t)a.stride * KV_PAGE) {
            const int32_t id = a.tables[(uint64_t)blockIdx.x * a.stride + x / KV_PAGE];
            if ((uint32_t)id < a.n_pages) at = (uint64_t)id * a.page_bytes() + x % KV_PAGE * a.row_bytes;
        }
        const uint64_t other = __shfl_xor_sync(0xffffffffu, at, 1);
        if (at == ~0ull || other == ~0ull) at = 0;  // either is not there: both are the same place
        if (j < 64) (threadIdx.x & 1 ? s_from : s_to)[j] = at;
    }
    const uint32_t n = min(n_kept[blockIdx.x], most), shift = a.row_bytes == 128 ? 3 : 4, unit = n << shift;  // words of a pool's head
    __syncthreads();
    if (n == 0) return;
    const Divide by_n(n);
    const uint32_t fit = KEEP_WORDS * MOVE_THREADS / unit, total = pools * a.n_kv;
#pragma unroll 1
    for (uint32_t p0 = blockIdx.y * fit; p0 < total; p0 += gridDim.y * fit) {
        const uint32_t words = min(fit, total - p0) * unit;
        uint4 x[KEEP_WORDS];
        uint8_t *to[KEEP_WORDS];
#pragma unroll
        for (uint32_t u = 0; u < KEEP_WORDS; ++u) {
            const uint32_t i = u * MOVE_THREADS + threadIdx.x, row = i >> shift, p = by_n(row), j = row - p * n;
            to[u] = nullptr;
            if (i < words && s_from[j] != s_to[j]) {
                const uint32_t pool = kv(p0 + p), head = p0 + p - pool * a.n_kv;
                uint8_t *base = a.pool(pool >> 1, pool & 1) + (uint64_t)head * KV_PAGE * a.row_bytes + ((i & ((1u << shift) - 1)) << 4);
                x[u] = *reinterpret_cast<const uint4 *>(base + s_from[j]);
                to[u] = base + s_to[j];
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
// (by more than the division's rounding).  Reading the keys bounds it: 65,536 positions of 8 heads of 128, 31 us with nothing in the caches (6.0 TB/s), 26 in a
// loop; with plain loads and a division per code it were instructions, 640 a page and head (4.3 TB/s).
// Two values in a word: plain words and instructions (through the types of the headers the compiler takes the halves apart: 1000
// instructions a page instead of the few hundred there are).
template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ float2 f(uint32_t v) {
        float2 r;
        asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(v));
        return r;
    }
};
template <> struct Pair<bf16> {
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ float2 f(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
};
constexpr uint32_t SIGNS = 0x80008000u;
constexpr uint32_t BOUND_DEPTH = 3;   // pages of a warp's ring: 96 KB a CTA with 128 entries a key
constexpr float BOUND_MOST = 1e18f;  // what larger keys count as: the scores stay finite
__device__ __forceinline__ float bounded(float v) { return v != v ? 0.0f : fminf(fmaxf(v, -BOUND_MOST), BOUND_MOST); }

// grid (CTAs of a sequence, sequences): warp w of a sequence has head w % n_kv of every `step`th page from w / n_kv on; the next page's number
// and keys are on their way while a page is done.
template <typename T, int HD>
__global__ void __launch_bounds__(256) pages_bounds_kernel(const __grid_constant__ PageView pg, uint32_t step, const uint32_t *__restrict__ first_pos, const uint32_t *__restrict__ n_pos, int8_t *codes,
                                                           float *scales) {
    using P = Pair<T>;
    constexpr uint32_t LANES = HD / 8, STEP = 32 / LANES, ROWS = KV_PAGE / STEP;  // lanes a row, rows a load, loads
    ob::pdl_release();
    ob::pdl_wait();
    const uint32_t lane = threadIdx.x & 31, w = blockIdx.x * 8 + (threadIdx.x >> 5), seq = blockIdx.y, first = w / pg.n_kv, head = w - first * pg.n_kv;
    const uint32_t from = first_pos[seq], to = min(n_pos[seq], pg.stride * KV_PAGE), end = (to + KV_PAGE - 1) / KV_PAGE;
    if (from >= to || first >= step) return;
    const int32_t *table = pg.tables + (uint64_t)seq * pg.stride;
    auto page_of = [&](uint32_t p) {
        const int32_t id = p < end ? table[p] : -1;
        return (uint32_t)id < pg.n_pages ? id : -1;
    };
    extern __shared__ __align__(16) uint4 ring[];  // [warp][BOUND_DEPTH][page's keys of a head]
    constexpr uint32_t WORDS = KV_PAGE * HD / 8;
    uint4 *own = ring + (threadIdx.x >> 5) * BOUND_DEPTH * WORDS;
    auto request = [&](uint32_t p, int32_t id, uint32_t slot) {
        if (id >= 0) {
            const uint4 *k = reinterpret_cast<const uint4 *>(static_cast<const T *>(pg.k) + ((uint64_t)id * pg.n_kv + head) * KV_PAGE * HD) + lane;
            const uint32_t filled = min(to - p * KV_PAGE, (uint32_t)KV_PAGE), dst = smem_addr(own + slot * WORDS + lane);
#pragma unroll
            for (uint32_t i = 0; i < ROWS; ++i) cp16(dst + i * 512, i * STEP + lane / LANES < filled ? k + i * 32 : k - lane / LANES * LANES, true);  // rows that are not filled: the first one again
        }
        cp_commit();
    };
    // From the exchange on the first LANES lanes have the largest keys, the next ones the smallest with their sign turned: floor(x) = -ceil(-x).
    const bool low = lane / LANES & 1;
    auto bound = [&](int32_t id, uint32_t slot) {
        const uint4 *x = own + slot * WORDS + lane, x0 = x[0];
        uint32_t hi[4] = {x0.x, x0.y, x0.z, x0.w}, lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) lo[e] = hi[e] ^ SIGNS;
#pragma unroll
        for (uint32_t i = 1; i < ROWS; ++i) {
            const uint4 xi = x[i * 32];
            const uint32_t v[4] = {xi.x, xi.y, xi.z, xi.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) hi[e] = P::max(hi[e], v[e]), lo[e] = P::max(lo[e], v[e] ^ SIGNS);
        }
        if constexpr (STEP == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = P::max(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], 16));
                lo[e] = P::max(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], 16));
            }
        }
        float b[8], top = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, low ? hi[e] : lo[e], LANES);
            const float2 f = P::f(P::max(low ? lo[e] : hi[e], got));
            b[2 * e] = f.x, b[2 * e + 1] = f.y;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(b[e]));
        if (__any_sync(0xffffffffu, !(top <= BOUND_MOST))) {
            top = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                b[e] = bounded(b[e]);
                top = fmaxf(top, b[e]);
            }
        }
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // (not negative: ordered as its bits are)
        const float d = __fdiv_rn(top, 127.0f), by = d > 0.0f ? d : 1.0f;
        // The quotient's next whole number by way of a product with about 1 / d, which is off by less than 2^-14 (127 times 2^-22 and 2^-24):
        // where that may be on the other side of one, the division is done, but not for those near 127, whose code is 127 either way.
        constexpr float MAGIC = 12582912.0f;  // 1.5 2^23: adding it rounds to whole numbers, which are then the low bits
        const float inverse = __frcp_rn(by);
        float r[8];
        bool near = !(by > 1e-37f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float q = b[e] * inverse;
            near |= q < 126.9f && fabsf(q - ((q + MAGIC) - MAGIC)) < 2.5e-4f;
            r[e] = fminf((q + 0.5f) + MAGIC, MAGIC + 127.0f);
        }
        if (near) {
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
                float y = b[0];
#pragma unroll
                for (int k = 1; k < 8; ++k) y = e == k ? b[k] : y;
                y = fminf(ceilf(__fdiv_rn(y, by)), 127.0f) + MAGIC;
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = e == k ? y : r[k];
            }
        }
        const uint64_t at = (uint64_t)id * pg.n_kv + head;
        if (lane < 2 * LANES) {
            uint32_t c[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t a = __byte_perm(__float_as_uint(r[4 * e]), __float_as_uint(r[4 * e + 1]), 0x0040), z = __byte_perm(__float_as_uint(r[4 * e + 2]), __float_as_uint(r[4 * e + 3]), 0x0040);
                c[e] = __byte_perm(a, z, 0x5410);
                if (low) c[e] = __vneg4(c[e]);
            }
            *reinterpret_cast<uint2 *>(codes + at * 2 * HD + lane * 8) = make_uint2(c[0], c[1]);
        }
        if (lane == 0) scales[at] = d;
    };
    uint32_t page = from / KV_PAGE + first, slot = 0;
    int32_t id[BOUND_DEPTH];  // pages of this turn and the next ones
#pragma unroll
    for (uint32_t i = 0; i < BOUND_DEPTH; ++i) id[i] = page_of(page + i * step);
#pragma unroll
    for (uint32_t i = 0; i + 1 < BOUND_DEPTH; ++i) request(page + i * step, id[i], i);
#pragma unroll 1
    for (; page < end; page += step) {
        const int32_t after = page_of(page + BOUND_DEPTH * step);
        cp_wait<BOUND_DEPTH - 2>();
        __syncwarp();
        request(page + (BOUND_DEPTH - 1) * step, id[BOUND_DEPTH - 1], slot == 0 ? BOUND_DEPTH - 1 : slot - 1);
        if (id[0] >= 0) bound(id[0], slot);
#pragma unroll
        for (uint32_t i = 0; i + 1 < BOUND_DEPTH; ++i) id[i] = id[i + 1];
        id[BOUND_DEPTH - 1] = after;
        slot = slot + 1 == BOUND_DEPTH ? 0 : slot + 1;
    }
    cp_wait<0>();
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
    a.counters = reinterpret_cast<uint32_t *>(p->ws.mem);
    a.pieces = reinterpret_cast<PagePiece *>(p->ws.mem + PG_COUNTERS * 4);
    a.partial = reinterpret_cast<float *>(p->ws.mem + PG_COUNTERS * (4 + sizeof(PagePiece)));
    a.status = p->ws.status;
}
// Whether a wait was given up since `who` was last told.
constexpr uint32_t SYNCHRONIZE = 1, PAGES_SYNCHRONIZE = 2;
bool take_status(ob_pages *p, uint32_t who) {
    volatile uint32_t *word = p->ws.status;
    if (*word) *word = 0, p->untold = SYNCHRONIZE | PAGES_SYNCHRONIZE;
    const bool mine = p->untold & who;
    p->untold &= ~who;
    return mine;
}
// The state that a new handle's workspace has, before any stream's next work.
cudaError_t clear(const ob_ctx *ctx, const PageWorkspace &ws) {
    *ws.status = 0;
    const cudaError_t e = cudaMemsetAsync(ws.mem, 0, PG_COUNTERS * 4, ctx->stream);
    return e == cudaSuccess ? cudaStreamSynchronize(ctx->stream) : e;
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

bool obrt::pages_gave_up(ob_ctx *ctx) {
    std::lock_guard<std::mutex> l(ctx->pages_mu);
    bool any = false;
    for (ob_pages *p : ctx->pages) any |= take_status(p, SYNCHRONIZE);
    return any;
}
void obrt::close_pages(ob_ctx *ctx) {
    for (ob_pages *p : ctx->pages) p->ctx = nullptr;  // the handles are their owners' to destroy
    ctx->pages.clear();
    for (const PageWorkspace &w : ctx->page_workspaces) cudaFree(w.mem), cudaFreeHost(w.status);  // (the first waits for the device)
    ctx->page_workspaces.clear(), ctx->free_page_workspaces.clear();
}

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
    if (d.n_layer > 16383 || d.n_head_kv > 4096 || d.n_pages > 0x7fffffffu || d.table_stride > (1u << 26) || d.n_seq > (1u << 24))
        return fail(ctx, OB_ERR_UNSUPPORTED, "pages_create: a size is too large");
    const uint64_t elems = (uint64_t)d.n_pages * d.n_head_kv * KV_PAGE * d.head_dim;
    if (d.n_layer > 1 && (d.layer_stride < elems || d.layer_stride % 8)) return fail(ctx, OB_ERR_INVALID, "pages_create: layer_stride has to be a multiple of 8 and at least a layer's pages");
    if (!d.k || !d.v || !d.tables) return fail(ctx, OB_ERR_INVALID, "pages_create: null argument");
    if (!aligned(d.k, 16) || !aligned(d.v, 16) || !aligned(d.tables, 4)) return fail(ctx, OB_ERR_INVALID, "pages_create: pages have to be aligned to 16 bytes, tables to 4");
    if (!on_device(ctx, d.k) || !on_device(ctx, d.v) || !on_device(ctx, d.tables)) return fail(ctx, OB_ERR_INVALID, "pages_create: pages and tables have to be memory of the context's device");
    ob_pages *p = new (std::nothrow) ob_pages{ctx, d, d.n_layer > 1 ? d.layer_stride * 2 : 0, {}, 0, {}};
    if (!p) return fail(ctx, OB_ERR_OOM, "pages_create: out of memory");
    try {  // (all that could throw, before there is anything on the device)
        std::lock_guard<std::mutex> l(ctx->pages_mu);
        p->maps.resize(d.n_layer);
        ctx->pages.reserve(ctx->pages.size() + 1);
        ctx->page_workspaces.reserve(ctx->page_workspaces.size() + 1);
        ctx->free_page_workspaces.reserve(ctx->page_workspaces.size() + 1);
    } catch (const std::bad_alloc &) {
        delete p;
        return fail(ctx, OB_ERR_OOM, "pages_create: out of memory");
    }
    for (uint32_t l = 0; l < d.n_layer; ++l)
        if (!make_page_maps(view(p, l), &p->maps[l])) {
            delete p;
            return fail(ctx, OB_ERR_UNSUPPORTED, "pages_create: no tensor map of the pages can be made (n_pages * n_head_kv * 16 rows have to be below 2^31)");
        }
    PageWorkspace ws{};
    cudaError_t e = cudaSuccess;
    if (!ctx->free_page_workspaces.empty()) {  // one that a destroyed handle has left
        ws = ctx->free_page_workspaces.back();
        ctx->free_page_workspaces.pop_back();
    } else {
        e = cudaMalloc(&ws.mem, PG_WORKSPACE);
        if (e == cudaSuccess) e = cudaHostAlloc(&ws.status, sizeof(uint32_t), cudaHostAllocMapped | cudaHostAllocPortable);  // (one address on both sides)
        if (e == cudaSuccess) e = clear(ctx, ws);
        if (e == cudaSuccess) ctx->page_workspaces.push_back(ws);
    }
    if (e != cudaSuccess) {
        cudaFree(ws.mem), cudaFreeHost(ws.status);
        cudaGetLastError();
        delete p;
        return fail(ctx, e == cudaErrorMemoryAllocation ? OB_ERR_OOM : OB_ERR_CUDA, std::string("pages_create: ") + cudaGetErrorString(e));
    }
    p->ws = ws;
    {
        std::lock_guard<std::mutex> l(ctx->pages_mu);
        ctx->pages.push_back(p);
    }
    *out = p;
    return OB_OK;
}

void ob_pages_destroy(ob_pages *p) {
    if (!p) return;
    if (ob_ctx *ctx = p->ctx) {
        std::lock_guard<std::mutex> g(ctx->mu);
        Bind b(ctx);
        {
            std::lock_guard<std::mutex> l(ctx->pages_mu);
            ctx->pages.erase(std::find(ctx->pages.begin(), ctx->pages.end(), p));
        }
        // For the next handle, unless the device cannot be waited for (while a stream of it is captured): kernels may be using it still then, and it
        // only goes with the context.
        if (cudaDeviceSynchronize() == cudaSuccess && clear(ctx, p->ws) == cudaSuccess)
            ctx->free_page_workspaces.push_back(p->ws);  // (there is room: ob_pages_create)
        else
            cudaGetLastError();
    }
    delete p;
}

int ob_pages_synchronize(ob_pages *p, void *stream) {
    const char *who = "pages_synchronize";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    ob_ctx *ctx = p->ctx;
    Bind b(ctx);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(stream_of(p, stream), &capture);
    if (e == cudaSuccess && capture == cudaStreamCaptureStatusNone) e = cudaStreamSynchronize(stream_of(p, stream));  // (others may launch meanwhile)
    std::lock_guard<std::mutex> g(ctx->mu);
    if (e != cudaSuccess) return launched(p, who, e);
    if (capture != cudaStreamCaptureStatusNone) return bad(p, who, "the stream is being captured");
    std::lock_guard<std::mutex> l(ctx->pages_mu);
    if (take_status(p, PAGES_SYNCHRONIZE)) return fail(ctx, OB_ERR_CUDA, "pages_synchronize: attention of drafted tokens gave up a bounded wait (pipeline barrier); its output is not valid");
    return OB_OK;
}

int ob_pages_wait_selftest(ob_pages *p, void *stream) {
    const char *who = "pages_wait_selftest";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    return launched(p, who, launch_pages_wait_selftest(p->ws.status, stream_of(p, stream)));
}

int ob_pages_attention_tree(ob_pages *p, uint32_t layer, uint32_t n_seq, const void *q, uint64_t q_stride, uint32_t n_tokens, const int32_t *first_token, const uint32_t *n_ctx,
                            const uint64_t *visible, uint32_t n_head, uint32_t max_drafts, uint32_t max_ctx, float scale, void *out, uint64_t out_stride, void *stream) {
    const char *who = "pages_attention_tree";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
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
        // (the walk over all pieces counts their tiles, and PG_START more for each, in 31 bits)
        if ((uint64_t)n_seq * p->d.n_head_kv * (((uint64_t)p->d.table_stride + PG_PAGES - 1) / PG_PAGES + PG_START) * ((max_drafts * a.group + 127) / 128) >= (1ull << 31))
            return fail(p->ctx, OB_ERR_CAPACITY, "pages_attention_tree: the tables of all sequences together have room for too many positions");
        return launched(p, who, launch_pages_tree_tc5(a, p->maps[layer], p->ctx->sm_count, stream_of(p, stream)), 2);
    }
    return launched(p, who, launch_pages_attention(a, true, p->ctx->sm_count, stream_of(p, stream)));
}

int ob_pages_attention(ob_pages *p, uint32_t layer, uint32_t n_rows, const void *q, uint64_t q_stride, const int32_t *row_seq, const uint32_t *n_pos, uint32_t n_head,
                       const int32_t *selected, uint32_t n_select, float scale, void *out, uint64_t out_stride, void *stream) {
    const char *who = "pages_attention";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (layer >= p->d.n_layer) return bad(p, who, "no such layer");
    if (!row_seq && n_rows > p->d.n_seq) return bad(p, who, "more rows than tables");
    if (int rc = check_heads(p, who, n_head)) return rc;
    if (n_rows > (1u << 24)) return bad(p, who, "too many rows");
    if (n_select == 0 || n_select > PG_SELECT_PAGES) return bad(p, who, "n_select has to be 1 to 131072");
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
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (!row_seq && n_rows > p->d.n_seq) return bad(p, who, "more rows than tables");
    if (int rc = check_heads(p, who, n_head)) return rc;
    if (n_rows > (1u << 24)) return bad(p, who, "too many rows");
    if (n_select == 0 || n_select > PG_SELECT_PAGES) return bad(p, who, "n_select has to be 1 to 131072");
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
    a.keys = reinterpret_cast<uint32_t *>(p->ws.mem + PG_COUNTERS * (4 + sizeof(PagePiece)));
    uint32_t kernels = 0;
    const cudaError_t e = launch_pages_select(a, p->ctx->sm_count, stream_of(p, stream), &kernels);
    return launched(p, who, e, kernels);
}

int ob_pages_bounds(ob_pages *p, uint32_t layer, uint32_t n_seq, const uint32_t *first_pos, const uint32_t *n_pos, uint32_t max_new, int8_t *codes, float *scales, void *stream) {
    const char *who = "pages_bounds";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (layer >= p->d.n_layer) return bad(p, who, "no such layer");
    if (n_seq > p->d.n_seq) return bad(p, who, "more sequences than tables");
    if (n_seq > 65535) return fail(p->ctx, OB_ERR_UNSUPPORTED, "pages_bounds: more than 65535 sequences");
    if (n_seq == 0 || max_new == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{first_pos, "first_pos", 4}, {n_pos, "n_pos", 4}, {codes, "codes", 16}, {scales, "scales", 4}})) return rc;
    const PageView v = view(p, layer);
    const uint64_t pages = std::min<uint64_t>((uint64_t)(max_new - 1) / KV_PAGE + 2, p->d.table_stride);  // positions that do not begin a page touch one more
    // Warps for all places (two CTAs an SM with 128 entries, four with 64), each for several pages where there are that many.
    const uint32_t bytes = 8 * BOUND_DEPTH * KV_PAGE * v.dim * 2;
    const uint64_t warps = std::min<uint64_t>(pages, std::max<uint64_t>(1, 2048ull / v.dim * p->ctx->sm_count / ((uint64_t)n_seq * v.n_kv))) * v.n_kv;
    const dim3 grid((uint32_t)((warps + 7) / 8), n_seq);
    auto kernel = v.is_bf16 ? (v.dim == 64 ? pages_bounds_kernel<bf16, 64> : pages_bounds_kernel<bf16, 128>) : (v.dim == 64 ? pages_bounds_kernel<__half, 64> : pages_bounds_kernel<__half, 128>);
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([] {
            for (auto k : {pages_bounds_kernel<bf16, 64>, pages_bounds_kernel<bf16, 128>, pages_bounds_kernel<__half, 64>, pages_bounds_kernel<__half, 128>})
                if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * BOUND_DEPTH * KV_PAGE * 128 * 2)) return e;
            return cudaSuccess;
        }))
        return launched(p, who, e);
    return launched(p, who, ob::launch_pdl(kernel, grid, dim3(256), bytes, stream_of(p, stream), v, (uint32_t)(warps / v.n_kv), first_pos, n_pos, codes, scales));
}

int ob_pages_copy(ob_pages *p, uint32_t n, const int32_t *src, const int32_t *dst, void *stream) {
    const char *who = "pages_copy";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (n > 0x7fffffffu) return bad(p, who, "too many pages");
    if (n == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{src, "src", 4}, {dst, "dst", 4}})) return rc;
    return launched(p, who, ob::launch_pdl(pages_copy_kernel, dim3(n, 2 * p->d.n_layer), dim3(MOVE_THREADS), 0, stream_of(p, stream), moves(p), src, dst));
}

int ob_pages_fork(ob_pages *p, uint32_t n, const int32_t *parent, const int32_t *child, const uint32_t *n_pos, const int32_t *fresh, void *stream) {
    const char *who = "pages_fork";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (n > 0x7fffffffu) return bad(p, who, "too many sequences");
    if (n == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{parent, "parent", 4}, {child, "child", 4}, {n_pos, "n_pos", 4}, {fresh, "fresh", 4}})) return rc;
    return launched(p, who, ob::launch_pdl(pages_fork_kernel, dim3(n, 2 * p->d.n_layer + 1), dim3(MOVE_THREADS), 0, stream_of(p, stream), moves(p), p->d.n_layer, parent, child, n_pos, fresh));
}

int ob_pages_keep(ob_pages *p, uint32_t n_seq, const uint32_t *n_ctx, const int32_t *kept, uint32_t kept_stride, const uint32_t *n_kept, void *stream) {
    const char *who = "pages_keep";
    if (!p || !p->ctx) return bad(p, who, "no handle, or its context is gone");
    std::lock_guard<std::mutex> g(p->ctx->mu);
    Bind b(p->ctx);
    if (n_seq > p->d.n_seq) return bad(p, who, "more sequences than tables");
    if (kept_stride == 0 || kept_stride > PG_MAX_DRAFTS) return bad(p, who, "kept_stride has to be 1 to 64");
    if (n_seq == 0) return OB_OK;
    if (int rc = check_pointers(p, who, {{n_ctx, "n_ctx", 4}, {kept, "kept", 4}, {n_kept, "n_kept", 4}})) return rc;
    // About two turns a CTA where all of its places are taken (six an SM), one where they are not.
    const uint64_t total = 2ull * p->d.n_layer * p->d.n_head_kv;
    if (total > 65535) return fail(p->ctx, OB_ERR_UNSUPPORTED, "pages_keep: n_layer * n_head_kv above 32767");
    const uint64_t few = std::max<uint64_t>(1, 12ull * p->ctx->sm_count / n_seq), turns = (total * kept_stride * (p->d.head_dim / 8) + KEEP_WORDS * MOVE_THREADS - 1) / (KEEP_WORDS * MOVE_THREADS);
    return launched(p, who, ob::launch_pdl(pages_keep_kernel, dim3(n_seq, (uint32_t)std::max<uint64_t>(1, std::min(few, turns))), dim3(MOVE_THREADS), 0, stream_of(p, stream), moves(p), 2 * p->d.n_layer,
                                           Divide(p->d.n_head_kv), kept_stride, n_ctx, kept, kept_stride, n_kept));
}

}  // extern "C"
