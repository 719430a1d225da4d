// What the mma.sync forms of attention over pages share (pages_attention.cu, pages_q4.cu): how the pages of all (unit, key/value head) pieces are shared
// out over the CTAs, and how the parts of a piece are added up.
#pragma once

#include <type_traits>

#include "mixers_common.cuh"
#include "pages.h"

namespace ob {

namespace {

template <typename T> struct Half2;
template <> struct Half2<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
    static constexpr uint32_t ONES = 0x3c003c00u, EXPONENT = 0x7c007c00u;
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Half2<bf16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
    static constexpr uint32_t ONES = 0x3f803f80u, EXPONENT = 0x7f807f80u;
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma_bf16(c, a, b0, b1); }
};

// The first product of a sum.
template <typename T> __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32, PA_CTAS = 3;  // CTAs an SM: one's start and end under another's pages
constexpr int PA_ROWS = 16;

// Shared memory: each warp's ring of DEPTH pages' keys and values (SLOT bytes), then the results.
template <int HD>
struct PaResult {
    static constexpr int PITCH = HD + 4;             // floats of an output row on its way between warps
    static constexpr int PART = PA_ROWS * (HD + 2);  // floats of a partial result
    static constexpr int BYTES = PA_WARPS * PA_ROWS * (PITCH + 2) * 4;
};

// Pages of a CTA.  Adding up the parts of a piece of n pages takes as long as some of them, so that there are not many more parts than the
// square root of n; and a piece that begins in the middle of a CTA's share costs that CTA a second start and end, so that shares are up to
// 1 / PA_MORE larger where no piece has to.  One sequence, 16 rows of 128, in a graph: 14.2 -> 9.9 us of 512 positions, 17.8 -> 13.3 of 2048,
// 26.2 -> 20.6 of 8192; 8 sequences of 2048 21.7 -> 18.2 us.  (Half of it for lists, whose rows are few: 128 pages 8.5 us, 9.2 without the half.)
constexpr uint32_t PA_LEAST = 2 * PA_WARPS, PA_MORE = 4;

// A sequence, `block` of its tokens (tree) or row (list) as the walk sees it.
struct PaUnit {
    uint32_t row0, rows, drafts, ctx, limit, n_pages;  // rows: tokens of the unit, the first of them `row0`; drafts: those at ctx, ctx + 1, ...
};
__device__ __forceinline__ PaUnit pa_tree_unit(const PagedAttnArgs &a, uint32_t unit) {
    PaUnit u{};
    const uint32_t s = a.blocks > 1 ? unit / a.blocks : unit, skip = (unit - s * a.blocks) * a.block;
    const int32_t f0 = a.first[s], f1 = a.first[s + 1];
    const uint32_t ctx = a.n_ctx[s];
    if (f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens) return u;
    const uint32_t room = a.pg.stride * KV_PAGE, n = min((uint32_t)(f1 - f0), a.max_drafts);
    if (skip >= n) return u;
    u.row0 = (uint32_t)f0 + skip;
    u.rows = min(n - skip, a.block);
    // without bits all that is before a block is context
    u.ctx = min(ctx, room);
    u.drafts = n;
    if (!a.visible) u.ctx = min(u.ctx + skip, room), u.drafts = u.rows;
    u.limit = min(u.ctx + u.drafts, room);
    u.n_pages = (u.limit + KV_PAGE - 1) / KV_PAGE;
    return u;
}
// Pieces in the order (unit, head); every warp holds the same walk.  Where the grid has a CTA for every `per` pages of every piece, a piece begins a new
// CTA (`apart`): none has the end of one and the start of the next.  UNIT: where a cut piece
// costs nothing, the least share is so many pages, and no more.
template <bool TREE, uint32_t UNIT = 0>
struct PaWalk {
    uint64_t at, end, per;  // pages of this CTA, pages a CTA; with `apart`, every piece counts as a multiple of `per`
    uint32_t unit, head, page;
    bool apart;
    PaUnit u;

    __device__ __forceinline__ void start(const PagedAttnArgs &a) {
        const uint32_t lane = threadIdx.x & 31;
        const uint64_t pieces = (uint64_t)a.n_units * a.pg.n_kv;
        apart = false;
        if constexpr (!TREE) {
            share(pieces * a.n_list, pieces);
            uint32_t parts = 1;
            if (pieces <= gridDim.x)  // (then everything fits 32 bits)
                for (uint32_t more = 0; more < 2 && !apart; ++more) {
                    const uint32_t each = (uint32_t)per + more * ((uint32_t)per / PA_MORE + 1);
                    parts = (a.n_list + each - 1) / each;
                    apart = (uint32_t)pieces * parts <= gridDim.x;
                    if (apart) per = each;
                }
            const uint64_t total = apart ? pieces * parts * per : pieces * a.n_list;
            at = min(total, blockIdx.x * per), end = min(total, at + per);
            const uint64_t item = apart ? blockIdx.x / parts : at / a.n_list;
            page = apart ? blockIdx.x % parts * (uint32_t)per : (uint32_t)(at % a.n_list);
            unit = (uint32_t)(item / a.pg.n_kv), head = (uint32_t)(item % a.pg.n_kv);
            u.n_pages = a.n_list;
        } else {
            auto load = [&](uint32_t s0) { return s0 + lane < a.n_units ? pa_tree_unit(a, s0 + lane) : PaUnit{}; };
            const PaUnit front = load(0);  // (up to 32 sequences are read once)
            uint64_t total = 0;
            for (uint32_t s0 = 0; s0 < a.n_units; s0 += 32) total += (uint32_t)warp_sum_i((int)(s0 ? load(s0) : front).n_pages);
            total *= a.pg.n_kv;
            share(total, pieces);
            uint32_t each = 1;
            if (pieces <= gridDim.x && per < a.apart)
                for (uint32_t more = 0; more < 2 && !apart; ++more) {
                    each = (uint32_t)per + more * ((uint32_t)per / PA_MORE + 1);  // (about a piece's pages at most: 32 bits)
                    uint64_t parts = 0;
                    for (uint32_t s0 = 0; s0 < a.n_units; s0 += 32) parts += (uint32_t)warp_sum_i((int)(((s0 ? load(s0) : front).n_pages + each - 1) / each));
                    parts *= a.pg.n_kv;
                    apart = parts <= gridDim.x;
                    if (apart) per = each, total = parts * per;
                }
            at = min(total, blockIdx.x * per), end = min(total, at + per);
            uint64_t before = 0;
            unit = head = page = 0, u = PaUnit{};
            for (uint32_t s0 = 0; at < end; s0 += 32) {
                if (s0 >= a.n_units) {  // (not while nobody writes the lengths meanwhile)
                    at = end;
                    break;
                }
                const PaUnit x = s0 ? load(s0) : front;
                const uint32_t span = apart ? (x.n_pages + each - 1) / each * each : x.n_pages;
                uint32_t sum = span;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= (uint32_t)o) sum += up;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, at < (before + sum) * a.pg.n_kv);
                if (hit) {
                    const int src = __ffs(hit) - 1;
                    auto of = [&](uint32_t v) { return __shfl_sync(0xffffffffu, v, src); };
                    unit = s0 + src;
                    u = PaUnit{of(x.row0), of(x.rows), of(x.drafts), of(x.ctx), of(x.limit), of(x.n_pages)};
                    const uint64_t off = at - (before + of(sum - span)) * a.pg.n_kv;  // pages of all heads: up to 2^38
                    const uint32_t length = of(span);
                    head = off >> 32 ? (uint32_t)(off / length) : (uint32_t)off / length, page = (uint32_t)(off - (uint64_t)head * length);
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
    }
    __device__ __forceinline__ void share(uint64_t total, uint64_t pieces) {
        const float piece = (float)total / (float)pieces;  // pages of a piece, about
        const uint64_t even = total >> 32 ? (total + gridDim.x - 1) / gridDim.x : total ? ((uint32_t)total - 1) / gridDim.x + 1 : 0;
        if constexpr (UNIT != 0) per = max(even, (uint64_t)UNIT);
        else per = max(even, (uint64_t)max(PA_LEAST, (uint32_t)sqrtf(TREE ? piece : 0.5f * piece)));
    }
    __device__ __forceinline__ bool more() const { return at < end; }
    __device__ __forceinline__ uint32_t last() const { return (uint32_t)min((uint64_t)u.n_pages, page + (end - at)); }  // the present piece is pages [page, last())
    __device__ __forceinline__ void next(const PagedAttnArgs &a) {
        at = apart ? end : at + (last() - page);
        page = 0;
        if (at >= end || ++head < a.pg.n_kv) return;
        head = 0;
        if constexpr (!TREE) {
            ++unit;
        } else {
            do {
                if (++unit >= a.n_units) {
                    at = end;
                    return;
                }
                u = pa_tree_unit(a, unit);
            } while (u.n_pages == 0);
        }
    }
};

// The end of a piece: the warps' parts of its rows in shared memory (so: [warp][row][PITCH] outputs, sml: [warp][row][2] maximum and sum; all of them
// written, no barrier since) become outputs, or a part that others go on with.  The maxima and sums are those of weights made 2^raise times as large.
// The whole CTA.  DEEP: entries of parts under way.
template <typename T, int HD, bool TREE, uint32_t DEEP = 16>
__device__ __forceinline__ void pa_finish(const PagedAttnArgs &a, const PaWalk<TREE> &wk, const float *so, const float *sml, uint32_t row0, uint32_t n_rows, uint32_t head, uint32_t to, float raise,
                                          uint32_t &s_last) {
    using H = Half2<T>;
    using S = PaResult<HD>;
    __syncthreads();
    constexpr int VEC = HD / 4;  // of a row, four entries each
    const bool whole = wk.page == 0 && to == wk.u.n_pages;
    const uint64_t origin = wk.at - wk.page;  // of the whole piece, in pages of all
    auto slot = [&](uint32_t c) { return a.partial + (2ull * c + (origin > c * wk.per ? 1 : 0)) * S::PART; };  // a CTA has a part of two pieces at most
    float *part = slot(blockIdx.x);
    auto store = [&](uint32_t r, uint32_t c, float4 x, float l, float top) {
        const float f = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // nothing seen: 0; a sum that is no number stays none
        const uint32_t t = TREE ? r / a.group : 0u;
        *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + (uint64_t)(row0 + t) * a.out_stride + (uint64_t)(head * a.group + r - t * a.group) * HD + 4 * c) =
            make_uint2(H::pack(x.x * f, x.y * f), H::pack(x.z * f, x.w * f));
        if (TREE && a.stats && c == 0) a.stats[(uint64_t)(row0 + t) * a.group * a.pg.n_kv + head * a.group + r - t * a.group] = make_float2(top - raise, f);
    };
    for (uint32_t i = threadIdx.x; i < n_rows * VEC; i += PA_THREADS) {
        const uint32_t r = i / VEC, c = i % VEC;
        float top = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < PA_WARPS; ++k) top = fmaxf(top, sml[2 * (k * PA_ROWS + r)]);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < PA_WARPS; ++k) {
            const float mk = sml[2 * (k * PA_ROWS + r)], lk = sml[2 * (k * PA_ROWS + r) + 1], f = mk == -INFINITY ? 0.0f : pow2(mk - top);
            if (mk == -INFINITY && lk == 0.0f) continue;
            const float4 y = *reinterpret_cast<const float4 *>(so + (k * PA_ROWS + r) * S::PITCH + 4 * c);
            l = fmaf(lk, f, l);
            x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
        }
        if (whole) {
            store(r, c, x, l, top);
        } else {
            __stcg(reinterpret_cast<float4 *>(part + r * HD + 4 * c), x);
            if (c == 0) __stcg(reinterpret_cast<float2 *>(part + PA_ROWS * HD + 2 * r), make_float2(top, l));
        }
    }
    if (whole) {
        __syncthreads();  // (the rings are written again)
        return;
    }
    // ---- the last part to arrive adds them all up
    const uint32_t c0 = (uint32_t)(origin / wk.per), c1 = (uint32_t)((origin + wk.u.n_pages - 1) / wk.per);  // CTAs that have one
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicInc(a.counters + c0, c1 - c0) == c1 - c0;  // (one piece at most begins in a CTA and goes on in others)
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    // 16 entries of parts under way at once: a sequence of 32,000 positions, whose eight pieces have 55 parts each, takes 51 us for 16 rows of
    // 128 and 49 us for 4; with one row after the other 16 rows took 67 us
    auto add_up = [&](auto rows) {
        constexpr uint32_t MINE = decltype(rows)::value, APART = PA_THREADS / VEC, AHEAD = DEEP / MINE;  // rows of a thread, from one to the next, parts
        const uint32_t r0 = threadIdx.x / VEC, c = threadIdx.x % VEC;
        float top[MINE], l[MINE];
        float4 x[MINE];
#pragma unroll
        for (uint32_t j = 0; j < MINE; ++j) top[j] = -INFINITY, l[j] = 0.0f, x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (uint32_t k = c0; k <= c1; k += AHEAD) {
            float2 ml[AHEAD][MINE];
            float4 y[AHEAD][MINE];
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (uint32_t j = 0; j < MINE; ++j) {
                    const uint32_t r = r0 + j * APART;
                    const float *from_k = slot(k + i);
                    ml[i][j] = make_float2(-INFINITY, 0.0f), y[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (k + i <= c1 && r < n_rows) {
                        ml[i][j] = __ldcg(reinterpret_cast<const float2 *>(from_k + PA_ROWS * HD + 2 * r));
                        y[i][j] = __ldcg(reinterpret_cast<const float4 *>(from_k + r * HD + 4 * c));
                    }
                }
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (uint32_t j = 0; j < MINE; ++j) {
                    const float2 ml1 = ml[i][j];
                    const float4 y1 = y[i][j];
                    const float higher = fmaxf(top[j], ml1.x), f0 = top[j] == -INFINITY ? 0.0f : pow2(top[j] - higher), f1 = ml1.x == -INFINITY ? 0.0f : pow2(ml1.x - higher);
                    top[j] = higher;
                    l[j] = fmaf(ml1.y, f1, l[j] * f0);
                    x[j].x = fmaf(y1.x, f1, x[j].x * f0), x[j].y = fmaf(y1.y, f1, x[j].y * f0), x[j].z = fmaf(y1.z, f1, x[j].z * f0), x[j].w = fmaf(y1.w, f1, x[j].w * f0);
                }
        }
#pragma unroll
        for (uint32_t j = 0; j < MINE; ++j)
            if (r0 + j * APART < n_rows) store(r0 + j * APART, c, x[j], l[j], top[j]);
    };
    if (n_rows * VEC <= PA_THREADS)
        add_up(std::integral_constant<uint32_t, 1>{});
    else
        add_up(std::integral_constant<uint32_t, PA_ROWS * VEC / PA_THREADS>{});
}

}  // namespace

}  // namespace ob
