// Attention over the pages of a cache for few rows a key/value head: the tokens of a tree of drafts with the query heads that share
// the head (ob_pages_attention_tree), or the heads of one token over a list of pages (ob_pages_attention).
//
//   out_r = sum_x w_rx v_x,  w_rx = 2^(s_rx - m_r) / sum_x 2^(s_rx - m_r),  s_rx = scale log2(e) q_r . k_x  over the positions x that row r sees
//
// in one pass with the running maximum m_r and sum.  A CTA has the (up to 16) rows of one key/value head and a stretch of the sequence's
// pages, which its four warps take in turn, each through a ring of its own: no barrier until the end.  Both products are mma.sync m16n8k16
// (f16 or bf16, fp32 accumulators): the bytes of the cache are the bound, and 16 rows fill its tile where a tcgen05 tile needs 128.
// Weights enter as value and remainder of the cache's type, since 8 or 11 bits of weight alone would be the largest error of the result: f16 ones
// are off by 2^-22 then, bf16 ones by 2^-16.  The sum of the weights is one more product, with ones, of the same rounded weights (that of
// pages_tc5.cu is of the weights before their rounding: the difference is 2^-32 of the largest a position at most, PG_RAISE).
//
// The pages of all (sequence, key/value head) pieces, laid end to end, are shared out evenly over the CTAs, whatever the lengths; a CTA walks
// through the pieces that lie in its part, or has a part of one piece only where there are CTAs enough for that.  A piece that is cut leaves (m, sum, output) in fp32 and the last of its CTAs to arrive -- a
// counter tells, which goes back to zero by itself -- adds the parts up in order, so the result does not depend on who was last.
//
// 32 sequences of 8192, 16 rows a head of 128: 195 us, 5.5 TB/s.  64 rows over 64 listed pages of random places, 8 heads of 128: 49 us, 5.4 TB/s.
#include <algorithm>
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

constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32, PA_CTAS = 3;  // CTAs an SM: one's start and end under another's pages
constexpr int PA_ROWS = 16;

template <int HD>
struct PaShape {
    static constexpr int PAGE_BYTES = KV_PAGE * HD * 2, SLOT = 2 * PAGE_BYTES;  // keys, then values
    static constexpr int DEPTH = 256 / HD;
    static constexpr int RINGS = PA_WARPS * DEPTH * SLOT;                       // 64 KB
    static constexpr int PITCH = HD + 4;                                        // floats of an output row on its way between warps
    static constexpr int PART = PA_ROWS * (HD + 2);                             // floats of a partial result
    static_assert(PA_WARPS * PA_ROWS * (PITCH + 2) * 4 <= RINGS, "the warps' results meet in the rings");
};

// Pages of a CTA.  Adding up the parts of a piece of n pages takes as long as some of them, so that there are not many more parts than the
// square root of n; and a piece that begins in the middle of a CTA's share costs that CTA a second start and end, so that shares are up to
// 1 / PA_MORE larger where no piece has to.  One sequence, 16 rows of 128, in a graph: 14.2 -> 9.9 us of 512 positions, 17.8 -> 13.3 of 2048,
// 26.2 -> 20.6 of 8192; 8 sequences of 2048 21.7 -> 18.2 us.  (Half of it for lists, whose rows are few: 128 pages 8.5 us, 9.2 without the half.)
constexpr uint32_t PA_LEAST = 2 * PA_WARPS, PA_MORE = 4;

// A sequence (tree) or row (list) as the walk sees it.
struct PaUnit {
    uint32_t row0, drafts, ctx, limit, n_pages;
};
__device__ __forceinline__ PaUnit pa_tree_unit(const PagedAttnArgs &a, uint32_t s) {
    PaUnit u{};
    const int32_t f0 = a.first[s], f1 = a.first[s + 1];
    if (f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens) return u;
    const uint32_t room = a.pg.stride * KV_PAGE;
    u.row0 = (uint32_t)f0;
    u.drafts = min((uint32_t)(f1 - f0), a.max_drafts);
    u.ctx = min(a.n_ctx[s], room);
    u.limit = min(u.ctx + u.drafts, room);
    u.n_pages = (u.limit + KV_PAGE - 1) / KV_PAGE;
    return u;
}
// Pieces in the order (unit, head); every warp holds the same walk.  Where the grid has a CTA for every `per` pages of every piece, a piece begins a new
// CTA (`apart`): none has the end of one and the start of the next.
template <bool TREE>
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
            if (pieces <= gridDim.x)
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
                    u = PaUnit{of(x.row0), of(x.drafts), of(x.ctx), of(x.limit), of(x.n_pages)};
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
        per = max(even, (uint64_t)max(PA_LEAST, (uint32_t)sqrtf(TREE ? piece : 0.5f * piece)));
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

template <typename T, int HD, bool TREE>
__global__ void __launch_bounds__(PA_THREADS, PA_CTAS) pages_attention_kernel(const __grid_constant__ PagedAttnArgs a) {
    using H = Half2<T>;
    using S = PaShape<HD>;
    constexpr int DEPTH = S::DEPTH, KS = HD / 16, CHUNKS = HD / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_last;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_release();
    pdl_wait();

    const uint32_t room = a.pg.stride * KV_PAGE;  // positions a table can name
    const float scale2 = a.scale * 1.4426950408889634f;
    const uint32_t k_row = (lane >> 4) * 8 + (lane & 7), k_half = lane >> 3 & 1, v_row = (lane >> 3 & 1) * 8 + (lane & 7), v_half = lane >> 4;
    PaWalk<TREE> wk;
    wk.start(a);
    for (; wk.more(); wk.next(a)) {
        // ---- which rows, which pages
        const uint32_t head = wk.head, unit = wk.unit;
        uint32_t seq = unit, row0 = unit, n_rows = a.group, ctx = 0, limit, drafts = 0;
        const int32_t *list = nullptr;
        if constexpr (TREE) {
            row0 = wk.u.row0, drafts = wk.u.drafts, n_rows = drafts * a.group, ctx = wk.u.ctx, limit = wk.u.limit;
        } else {
            const int32_t s = a.row_seq ? a.row_seq[unit] : (int32_t)unit;
            limit = (uint32_t)s < a.pg.n_seq ? min(a.n_pos[unit], room) : 0u;
            seq = (uint32_t)s < a.pg.n_seq ? (uint32_t)s : 0u;
            list = a.list + ((uint64_t)unit * a.pg.n_kv + head) * a.n_list;
        }
        const uint32_t from = wk.page + warp, to = wk.last();
        const uint32_t n_steps = to > from ? (to - from + PA_WARPS - 1) / PA_WARPS : 0u;  // pages of this warp
        const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;

        // ---- page numbers: lane i has those of step 32 j + i, and of the 32 after them
        auto look = [&](uint32_t step, int32_t &logical) {  // page of a step, or -1
            logical = -1;
            if (step >= n_steps) return -1;
            const uint32_t i = from + step * PA_WARPS;
            const int32_t p = TREE ? (int32_t)i : list[i];
            if ((uint32_t)p >= a.pg.stride || (uint32_t)p * KV_PAGE >= limit) return -1;
            const int32_t id = table[p];
            logical = p;
            return (uint32_t)id < a.pg.n_pages ? id : -1;
        };
        int32_t log_now, log_next, id_now = look(lane, log_now), id_next = look(32 + lane, log_next);
        uint32_t block = 0;  // steps 32 block ..: log_now, id_now
        auto numbers = [&](uint32_t step, int32_t &id, int32_t &logical) {  // steps [32 block, 32 block + 64)
            const bool next = step / 32 != block;
            id = __shfl_sync(0xffffffffu, next ? id_next : id_now, step & 31);
            logical = __shfl_sync(0xffffffffu, next ? log_next : log_now, step & 31);
        };

        const uint32_t base = smem_addr(smem) + warp * DEPTH * S::SLOT;
        const uint64_t page_elems = (uint64_t)a.pg.n_kv * KV_PAGE * HD, head_elems = (uint64_t)head * KV_PAGE * HD;
        auto request = [&](uint32_t step) {  // copies of a step's keys and values
            if (step < n_steps) {
                int32_t id, logical;
                numbers(step, id, logical);
                if (id >= 0) {
                    const uint64_t off = ((uint64_t)id * page_elems + head_elems) * 2;
                    const uint8_t *k = static_cast<const uint8_t *>(a.pg.k) + off, *v = static_cast<const uint8_t *>(a.pg.v) + off;
                    const uint32_t dst = base + step % DEPTH * S::SLOT, there = limit - (uint32_t)logical * KV_PAGE;  // rows of the page that hold positions
#pragma unroll
                    for (int i = 0; i < 2 * HD / 32; ++i) {
                        const uint32_t c = i * 32 + lane, row = c / CHUNKS, at = row * HD * 2 + (((c % CHUNKS) ^ (row & 7)) << 4);
                        cp16(dst + at, k + c * 16, row < there);
                        cp16(dst + S::PAGE_BYTES + at, v + c * 16, row < there);
                    }
                }
            }
            cp_commit();
        };
#pragma unroll 1
        for (int i = 0; i < DEPTH - 1; ++i) request(i);

        // ---- queries: rows (token, head of the group) as A fragments
        uint32_t q[KS][4];
        uint64_t seen[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = lane / 4 + 8 * h, t = TREE ? r / a.group : 0u;
            const bool live = r < n_rows;
            const uint64_t token = row0 + t;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(a.q) + (live ? token * a.q_stride + (uint64_t)(head * a.group + r - t * a.group) * HD : 0u));
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                q[s][h] = live ? src[s * 8 + (lane & 3)] : 0u;
                q[s][2 + h] = live ? src[s * 8 + 4 + (lane & 3)] : 0u;
            }
            seen[h] = 0;
            if constexpr (TREE)
                if (live) seen[h] = a.visible[token] & (drafts < 64 ? (1ull << drafts) - 1 : ~0ull);
        }

        float o[HD / 8][4], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

#pragma unroll 1
        for (uint32_t step = 0; step < n_steps; ++step) {
            cp_wait<DEPTH - 2>();
            __syncwarp();
            if (step / 32 != block) {
                block = step / 32;
                id_now = id_next, log_now = log_next;
                id_next = look(32 * (block + 1) + lane, log_next);
            }
            request(step + DEPTH - 1);
            int32_t id, logical;
            numbers(step, id, logical);
            if (id < 0) continue;
            const uint32_t ks = base + step % DEPTH * S::SLOT, vs = ks + S::PAGE_BYTES, pos0 = (uint32_t)logical * KV_PAGE;

            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t f[4];
                ldsm4(f, ks + k_row * HD * 2 + (((2 * k + k_half) ^ (k_row & 7)) << 4));
                H::mma(s[0], q[k], f[0], f[1]);
                H::mma(s[1], q[k], f[2], f[3]);
            }
            const bool drafted = TREE && pos0 + KV_PAGE > ctx, ragged = pos0 + KV_PAGE > limit;
            uint32_t hidden = 0;  // a bit per element of s that its row does not see
            if (drafted || ragged) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = pos0 + n * 8 + (lane & 3) * 2 + (e & 1);
                        bool see = x < limit;
                        if (TREE && x >= ctx) see = see && (seen[e >> 1] >> ((x - ctx) & 63) & 1);  // x - ctx < drafts where x < limit
                        if (!see) s[n][e] = -INFINITY, hidden |= 1u << (n * 4 + e);
                    }
            }
            float now[2];
            bool grown = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                now[h] = x * scale2;
                grown |= now[h] > m[h] + PG_SLACK;  // (the first time, too)
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float top = fmaxf(m[h], now[h]), keep = m[h] == -INFINITY ? 0.0f : pow2(m[h] - top);
                    m[h] = top;
                    sum[2 * h] *= keep, sum[2 * h + 1] *= keep;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) o[n][2 * h] *= keep, o[n][2 * h + 1] *= keep;
                }
            }
            uint32_t w[4], rest[4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float off = m[h] == -INFINITY ? 0.0f : PG_RAISE<T> - m[h];
                    const float e0 = pow2(fmaf(s[n][2 * h], scale2, off)), e1 = pow2(fmaf(s[n][2 * h + 1], scale2, off));
                    const uint32_t u = H::pack(e0, e1);
                    w[2 * n + h] = u;
                    const float2 r = H::unpack(u);
                    rest[2 * n + h] = H::pack(e0 - r.x, e1 - r.y);
                }
            H::mma(sum, w, H::ONES, H::ONES);
            H::mma(sum, rest, H::ONES, H::ONES);
            bool odd = false;  // a drafted token's value is not finite: 0 times it would reach rows that do not see the token
            if (drafted) {
#pragma unroll 1
                for (int i = lane; i < 2 * HD; i += 32) {
                    uint32_t u[4];
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(vs + i * 16));
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd |= (u[e] & H::EXPONENT & 0xffffu) == (H::EXPONENT & 0xffffu) || (u[e] & H::EXPONENT & 0xffff0000u) == (H::EXPONENT & 0xffff0000u);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
#pragma unroll
                for (int n = 0; n < HD / 8; n += 2) {
                    uint32_t f[4];
                    ldsm4t(f, vs + v_row * HD * 2 + (((n + v_half) ^ (v_row & 7)) << 4));
                    H::mma(o[n], w, f[0], f[1]);
                    H::mma(o[n + 1], w, f[2], f[3]);
                    H::mma(o[n], rest, f[0], f[1]);
                    H::mma(o[n + 1], rest, f[2], f[3]);
                }
            } else {  // term by term, those that a row sees
#pragma unroll 1
                for (uint32_t j = 0; j < KV_PAGE; ++j) {
                    const uint32_t src = (lane & ~3u) | (j & 7) >> 1;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 p = H::unpack(__shfl_sync(0xffffffffu, j < 8 ? w[h] : w[2 + h], src));
                        const float2 r = H::unpack(__shfl_sync(0xffffffffu, j < 8 ? rest[h] : rest[2 + h], src));
                        const float x = j & 1 ? p.y + r.y : p.x + r.x;
                        const bool see = !(__shfl_sync(0xffffffffu, hidden, src) >> ((j >> 3) * 4 + 2 * h + (j & 1)) & 1);
#pragma unroll
                        for (int n = 0; n < HD / 8; ++n) {
                            uint32_t u;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(vs + j * HD * 2 + ((n ^ (j & 7)) << 4) + (lane & 3) * 4));
                            const float2 v = H::unpack(u);
                            if (see) o[n][2 * h] = fmaf(x, v.x, o[n][2 * h]), o[n][2 * h + 1] = fmaf(x, v.y, o[n][2 * h + 1]);
                        }
                    }
                }
            }
        }
        cp_wait<0>();
        __syncthreads();

        // ---- the warps' parts of a row meet in shared memory
        float *so = reinterpret_cast<float *>(smem), *sml = so + PA_WARPS * PA_ROWS * S::PITCH;  // [warp][row]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = warp * PA_ROWS + 8 * h + lane / 4;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2 *>(so + r * S::PITCH + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
            if ((lane & 3) == 0) sml[2 * r] = m[h], sml[2 * r + 1] = sum[2 * h];
        }
        __syncthreads();
        constexpr int VEC = HD / 4;  // of a row, four entries each
        const bool whole = wk.page == 0 && to == wk.u.n_pages;
        const uint64_t origin = wk.at - wk.page;  // of the whole piece, in pages of all
        auto slot = [&](uint32_t c) { return a.partial + (2ull * c + (origin > c * wk.per ? 1 : 0)) * S::PART; };  // a CTA has a part of two pieces at most
        float *part = slot(blockIdx.x);
        auto store = [&](uint32_t r, uint32_t c, float4 x, float l) {
            const float f = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // nothing seen: 0; a sum that is no number stays none
            const uint32_t t = TREE ? r / a.group : 0u;
            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + (uint64_t)(row0 + t) * a.out_stride + (uint64_t)(head * a.group + r - t * a.group) * HD + 4 * c) =
                make_uint2(H::pack(x.x * f, x.y * f), H::pack(x.z * f, x.w * f));
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
                store(r, c, x, l);
            } else {
                __stcg(reinterpret_cast<float4 *>(part + r * HD + 4 * c), x);
                if (c == 0) __stcg(reinterpret_cast<float2 *>(part + PA_ROWS * HD + 2 * r), make_float2(top, l));
            }
        }
        if (whole) {
            __syncthreads();  // (the rings are written again)
            continue;
        }
        // ---- the last part to arrive adds them all up
        const uint32_t c0 = (uint32_t)(origin / wk.per), c1 = (uint32_t)((origin + wk.u.n_pages - 1) / wk.per);  // CTAs that have one
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) s_last = atomicInc(a.counters + c0, c1 - c0) == c1 - c0;  // (one piece at most begins in a CTA and goes on in others)
        __syncthreads();
        if (!s_last) continue;
        __threadfence();
        // 16 entries of parts are under way at once: a sequence of 32,000 positions, whose eight pieces have 55 parts each, takes 51 us for 16 rows of
        // 128 and 49 us for 4; with one row after the other 16 rows took 67 us
        auto add_up = [&](auto rows) {
            constexpr uint32_t MINE = decltype(rows)::value, APART = PA_THREADS / VEC, AHEAD = 16 / MINE;  // rows of a thread, from one to the next, parts
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
                if (r0 + j * APART < n_rows) store(r0 + j * APART, c, x[j], l[j]);
        };
        if (n_rows * VEC <= PA_THREADS)
            add_up(std::integral_constant<uint32_t, 1>{});
        else
            add_up(std::integral_constant<uint32_t, PA_ROWS * VEC / PA_THREADS>{});
    }
}

template <typename T, int HD, bool TREE>
cudaError_t launch(PagedAttnArgs a, int sm_count, cudaStream_t st) {
    using S = PaShape<HD>;
    auto kernel = pages_attention_kernel<T, HD, TREE>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::RINGS); })) return e;
    const uint64_t pages = TREE ? (std::min(a.max_ctx, a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE : a.n_list;  // (tree: about, of a sequence)
    const uint64_t most = std::min<uint64_t>({(uint64_t)sm_count * PA_CTAS, PG_COUNTERS, PG_PARTIAL / (2 * S::PART * 4)});
    const uint64_t grid = std::min(most, std::max<uint64_t>(1, a.n_units * ((pages + PA_LEAST - 1) / PA_LEAST) * a.pg.n_kv));
    return launch_pdl(kernel, dim3((uint32_t)grid), dim3(PA_THREADS), S::RINGS, st, a);
}

template <typename T>
cudaError_t launch_dim(const PagedAttnArgs &a, bool tree, int sm_count, cudaStream_t st) {
    if (a.pg.dim == 64) return tree ? launch<T, 64, true>(a, sm_count, st) : launch<T, 64, false>(a, sm_count, st);
    return tree ? launch<T, 128, true>(a, sm_count, st) : launch<T, 128, false>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_pages_attention(const PagedAttnArgs &a, bool tree, int sm_count, cudaStream_t st) {
    return a.pg.is_bf16 ? launch_dim<bf16>(a, tree, sm_count, st) : launch_dim<__half>(a, tree, sm_count, st);
}

}  // namespace ob
