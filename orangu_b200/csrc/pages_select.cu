// Which pages a row reads (ob_pages_select): a score for every page of the row's sequence, per key/value head, from bounds of the page's
// keys in 8 bits, and the best n_select of them.
//
//   q_h,e ~ dq_h c_h,e  with dq_h = max_e |q_h,e| / 127, c = rint(q / dq);  hi_e, lo_e: codes of the page's largest and smallest key, unit d
//   score = max over the heads h of  (dq_h d) * sum_e max(c_h,e hi_e, c_h,e lo_e)  =  (dq_h d) * (sum_e max(c, 0) hi_e + sum_e min(c, 0) lo_e)
//
// The sum is a whole number below 2^24 and the two products are single roundings, so a score has one value whatever the order of
// the terms, and so has the choice.  The sums are an s8 product of length 2 dim: mma.sync m16n8k32 with 16 pages as rows, whose codes go
// from memory straight into the fragments (a lane's 16 bytes serve two steps; the order of the terms inside a step is free), and the
// heads as columns: a page's best head is two exchanges away.  Nor do the queries need shared memory: four lanes hold a head's codes just
// where the fragments want them.  What bounds the scores is the reading of the codes, 2 dim + 4 bytes a page; with eight pages as columns and
// the heads as rows, four times as many instructions did (51 us for 64 rows of 6 to 24 k positions, 8 heads of 128; now 27 us for the 120 MB, and
// 8 for the choice).  With rows half as long the two take 29 us instead of 36: starts, chains of loads and the rounds of the choice are the larger part.  Rings of
// cp.async in shared memory, codes brought to the L2 cache ahead, the first codes before the queries and fewer warps with more registers all took 35 to 38.
//
// Scores are kept as 32-bit words in their order.  Many of them are made by a kernel of their own, a warp per 128 pages (fewer where there are few), neighbouring warps
// the heads of the same pages, whose codes lie together; few of them in the CTA that picks.  A CTA per (row, head) then picks: counts in
// 2048 equal parts of the range, as often as the part with the border still holds more than are wanted (two times as a rule),
// and the list is written in ascending order.
#include <algorithm>

#include "mixers_common.cuh"
#include "pages.h"
#include "pages_pick.cuh"

namespace ob {

namespace {

constexpr uint32_t SEL_HELD = 32768;       // words that the picking CTA holds in shared memory; with more they are read again from the workspace
constexpr uint32_t SEL_FUSED = 512;        // pages of a row up to which the picking CTA makes the scores, too
constexpr float SEL_MOST = 1e18f;          // what larger queries count as: products of two units and a sum stay finite

__device__ __forceinline__ float2 as_float2(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
__device__ __forceinline__ float2 as_float2(uint32_t u, bf16) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Larger scores have larger words; what is no number has the smallest.
__device__ __forceinline__ uint32_t ordered(float s) {
    if (s != s) return 0u;
    const uint32_t u = __float_as_uint(s + 0.0f);  // (-0 is 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A row's sequence and pages.
struct SelRow {
    const int32_t *table;
    uint32_t n_pages;
};
__device__ __forceinline__ SelRow sel_row(const PagedSelectArgs &a, uint32_t row) {
    const int32_t s = a.row_seq ? a.row_seq[row] : (int32_t)row;
    const bool known = (uint32_t)s < a.pg.n_seq;
    const uint32_t n_pos = known ? min(min(a.n_pos[row], a.max_pos), a.pg.stride * KV_PAGE) : 0u;
    return SelRow{a.pg.tables + (uint64_t)(known ? s : 0) * a.pg.stride, (n_pos + KV_PAGE - 1) / KV_PAGE};
}

// One warp's queries of a (row, key/value head) as B fragments.  MANY: more than eight heads, in two sets of columns.  Load i of a lane is
// bytes 64 i + 16 (lane % 4) .. + 15 of a page's codes (largest keys, then smallest); its words 0, 1 and 2, 3 are the two halves of a step's
// 32.  So lane l has entries 64 i + 16 (l % 4) .. + 15 of heads l / 4 and l / 4 + 8.
template <typename T, int HD, bool MANY>
struct SelQuery {
    static constexpr int LOADS = 2 * HD / 64, SETS = MANY ? 2 : 1, HEADS = 8 * SETS, PER = HD / 32;  // PER: entries of a lane while codes are made
    uint32_t pos[SETS][LOADS / 2][4], neg[SETS][LOADS / 2][4];  // codes above and below zero: they meet the largest and the smallest keys
    float unit[SETS][2];                                        // of this lane's two columns; -1: no such head

    // own: HEADS x HD entries of shared memory that are this warp's: the queries, whose places their codes take.  A head after the other in a
    // loop that is not unrolled: the instructions are fetched from memory by every SM (32 entries a lane side by side took 8 us), and all
    // loads at once.
    __device__ __forceinline__ void load(const PagedSelectArgs &a, uint32_t row, uint32_t head, T *own) {
        const uint32_t lane = threadIdx.x & 31, words = a.group * HD / 8;  // of 16 bytes
        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (uint64_t)row * a.q_stride + (uint64_t)head * a.group * HD);
        uint4 v[HEADS * HD / 256];
#pragma unroll
        for (uint32_t i = 0; i < HEADS * HD / 256; ++i) v[i] = i * 32 + lane < words ? __ldg(src + i * 32 + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < HEADS * HD / 256; ++i) reinterpret_cast<uint4 *>(own)[i * 32 + lane] = v[i];
        __syncwarp();
        float mine = -1.0f;  // lane h: head h's unit
#pragma unroll 1
        for (uint32_t h = 0; h < a.group; ++h) {  // (the places of the others are zero, as are their codes)
            constexpr float MAGIC = 12582912.0f;  // 1.5 2^23: adding it rounds to whole numbers, which are then the low bits
            const uint32_t *at = reinterpret_cast<const uint32_t *>(own + h * HD) + lane * (PER / 2);
            float x[PER], top = 0.0f;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const float2 f = as_float2(at[e / 2], T());
                x[e] = e % 2 ? f.y : f.x;
                top = fmaxf(top, fabsf(x[e]));
            }
            bool odd = !(top <= SEL_MOST);
#pragma unroll
            for (int e = 0; e < PER; ++e) odd |= x[e] != x[e];
            if (odd) {
                top = 0.0f;
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -SEL_MOST), SEL_MOST);
                    top = fmaxf(top, fabsf(x[e]));
                }
            }
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // (not negative: ordered as its bits are)
            const float d = __fdiv_rn(top, 127.0f), by = d > 0.0f ? d : 1.0f;
            if (lane == h) mine = d;
            // rint(x / d) by way of a product with about 1 / d, which is off by less than 2^-14 (127 times 2^-22 and 2^-24): only where that
            // may cross a half, or d is too small for an inverse, is the division done.
            const float inverse = __frcp_rn(by);
            float far = 0.0f, t[PER];  // far: how far from a whole number
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                t[e] = x[e] * inverse;
                far = fmaxf(far, fabsf(t[e] - ((t[e] + MAGIC) - MAGIC)));
            }
            if (!(far < 0.4999f) || !(by > 1e-37f)) {
#pragma unroll 1
                for (int e = 0; e < PER; ++e) {
                    float y = x[0];
#pragma unroll
                    for (int k = 1; k < PER; ++k) y = e == k ? x[k] : y;
                    y = __fdiv_rn(y, by);
#pragma unroll
                    for (int k = 0; k < PER; ++k) t[k] = e == k ? y : t[k];
                }
            }
            uint32_t c = 0;  // (a quotient is 127 and a little at most, which rounds to 127)
#pragma unroll
            for (int e = 0; e < PER; ++e) c |= (__float_as_uint(t[e] + MAGIC) & 255u) << (8 * e);
            int8_t *code = reinterpret_cast<int8_t *>(own + h * HD);  // (all lanes have read: the maximum is theirs)
            if constexpr (PER == 4) reinterpret_cast<uint32_t *>(code)[lane] = c;
            else reinterpret_cast<uint16_t *>(code)[lane] = (uint16_t)c;
        }
        __syncwarp();
#pragma unroll
        for (int m = 0; m < SETS; ++m) {
#pragma unroll
            for (int e = 0; e < 2; ++e) unit[m][e] = __shfl_sync(0xffffffffu, mine, (lane & 3) * 2 + e + 8 * m);
#pragma unroll
            for (int i = 0; i < LOADS / 2; ++i) {
                const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const int8_t *>(own + (lane / 4 + 8 * m) * HD) + i * 64 + (lane & 3) * 16);
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) pos[m][i][w] = __vmaxs4(u[w], 0u), neg[m][i][w] = __vmins4(u[w], 0u);
            }
        }
    }
    // Words of pages first + step k + i, i < 16, below `end` of the row, handed to put(page, word) by the lanes that have them.
    template <typename P>
    __device__ __forceinline__ void score(const PagedSelectArgs &a, const SelRow &r, uint32_t head, uint32_t first, uint32_t end, uint32_t step, P put) const {
        const uint32_t lane = threadIdx.x & 31;
        auto page_of = [&](uint32_t p) {
            const int32_t id = p < end ? r.table[p] : -1;
            return (uint32_t)id < a.pg.n_pages ? id : -1;
        };
        int32_t id[2] = {page_of(first + lane / 4), page_of(first + lane / 4 + 8)};  // this lane's two rows of a product
#pragma unroll 1
        for (uint32_t p0 = first; p0 < end; p0 += step) {
            uint4 x[2][LOADS];
            float d[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint64_t at = (uint64_t)(uint32_t)max(id[u], 0) * a.pg.n_kv + head;
                const int8_t *src = a.codes + at * (2 * HD) + (lane & 3) * 16;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) x[u][i] = ldg128_stream(src + i * 64);  // (of page 0 where there is none)
                d[u] = id[u] < 0 ? __int_as_float(0x7fc00000) : __ldg(a.scales + at);    // a page that is not there: no number
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) id[u] = page_of(p0 + step + lane / 4 + 8 * u);
            float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int m = 0; m < SETS; ++m) {
                int c[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const uint32_t(&w)[4] = i < LOADS / 2 ? pos[m][i % (LOADS / 2)] : neg[m][i % (LOADS / 2)];
                    const uint32_t a0[4] = {x[0][i].x, x[1][i].x, x[0][i].y, x[1][i].y}, a1[4] = {x[0][i].z, x[1][i].z, x[0][i].w, x[1][i].w};
                    mma_s8(c, a0, w[0], w[1]);
                    mma_s8(c, a1, w[2], w[3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (unit[m][e & 1] >= 0.0f) best[e >> 1] = fmaxf(best[e >> 1], __fmul_rn(__fmul_rn(unit[m][e & 1], d[e >> 1]), (float)c[e]));
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float y = best[u];
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
                const uint32_t p = p0 + lane / 4 + 8 * u;
                if ((lane & 3) == 0 && p < end) put(p, p < a.keep_first || p + a.keep_last >= r.n_pages ? SEL_FORCED : d[u] != d[u] ? 0u : ordered(y));
            }
        }
    }
};

// A warp per (row, `unit` pages, key/value head), heads side by side.
template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(256, MANY ? 2 : 4) pages_score_kernel(const __grid_constant__ PagedSelectArgs a, uint32_t row0, uint32_t unit, uint32_t units, uint32_t pitch) {
    __shared__ __align__(16) T s_query[8][MANY ? 16 : 8][HD];
    pdl_release();
    pdl_wait();
    const uint32_t w = blockIdx.x * 8 + (threadIdx.x >> 5), head = w % a.pg.n_kv, part = w / a.pg.n_kv % units;
    const uint32_t row = row0 + w / a.pg.n_kv / units;
    if (row >= a.n_rows) return;
    const SelRow r = sel_row(a, row);
    const uint32_t first = part * unit;
    if (r.n_pages <= a.n_select || first >= r.n_pages) return;  // (all of the row's pages are taken without a score)
    SelQuery<T, HD, MANY> q;
    q.load(a, row, head, &s_query[threadIdx.x >> 5][0][0]);
    uint32_t *keys = a.keys + ((uint64_t)(row - row0) * a.pg.n_kv + head) * pitch;
    q.score(a, r, head, first, min(first + unit, r.n_pages), 16, [&](uint32_t p, uint32_t key) { keys[p] = key; });
}

// A CTA per (row, key/value head).
template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(256) pages_score_pick_kernel(const __grid_constant__ PagedSelectArgs a) {
    extern __shared__ __align__(16) uint32_t held[];
    __shared__ __align__(16) T s_query[8][MANY ? 16 : 8][HD];
    pdl_release();
    pdl_wait();
    const uint32_t head = blockIdx.x % a.pg.n_kv, row = blockIdx.x / a.pg.n_kv, warp = threadIdx.x >> 5;
    const SelRow r = sel_row(a, row);
    int32_t *out = a.selected + (uint64_t)blockIdx.x * a.n_select;
    if (r.n_pages <= a.n_select) {  // all of them
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < a.n_select; i += 256) out[i] = i < r.n_pages ? (int32_t)i : -1;
        return;
    }
    uint32_t lo = 0xffffffffu, hi = 0;
    SelQuery<T, HD, MANY> q;
    q.load(a, row, head, &s_query[warp][0][0]);
    q.score(a, r, head, warp * 16, r.n_pages, 8 * 16, [&](uint32_t p, uint32_t key) {
        held[p] = key;
        if (key != SEL_FORCED) lo = min(lo, key), hi = max(hi, key);
    });
    pick<256>(a.n_select - a.keep_first - a.keep_last, held, r.n_pages, lo, hi, out);
}
template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) pages_pick_kernel(const __grid_constant__ PagedSelectArgs a, uint32_t row0, uint32_t pitch) {
    extern __shared__ __align__(16) uint32_t held[];
    pdl_release();
    pdl_wait();
    const uint32_t head = blockIdx.x % a.pg.n_kv, row = row0 + blockIdx.x / a.pg.n_kv;
    const uint32_t n = sel_row(a, row).n_pages;
    int32_t *out = a.selected + ((uint64_t)row * a.pg.n_kv + head) * a.n_select;
    if (n <= a.n_select) {
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < a.n_select; i += THREADS) out[i] = i < n ? (int32_t)i : -1;
        return;
    }
    const uint32_t *from = a.keys + (uint64_t)blockIdx.x * pitch;
    const bool fits = n <= SEL_HELD;
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        const uint32_t key = __ldcg(from + i);
        if (fits) held[i] = key;
        if (key != SEL_FORCED) lo = min(lo, key), hi = max(hi, key);
    }
    pick<THREADS>(a.n_select - a.keep_first - a.keep_last, fits ? held : from, n, lo, hi, out);
}

template <typename T, int HD, bool MANY>
cudaError_t launch(PagedSelectArgs a, int sm_count, cudaStream_t st, uint32_t *launches) {
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(pages_pick_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_HELD * 4); })) return e;
    const uint32_t pages = std::max(1u, (std::min(a.max_pos, a.pg.stride * KV_PAGE) + KV_PAGE - 1) / KV_PAGE);
    const uint64_t pairs = (uint64_t)a.n_rows * a.pg.n_kv;
    *launches = 1;
    // One kernel while a CTA per SM scores its own pages at once.
    if (pages <= SEL_FUSED && pairs <= (uint64_t)sm_count) return launch_pdl(pages_score_pick_kernel<T, HD, MANY>, dim3((uint32_t)pairs), dim3(256), pages * 4, st, a);
    const uint32_t unit = pairs * pages >= 128ull * 32 * sm_count ? 128 : pairs * pages >= 64ull * 32 * sm_count ? 64 : 32;  // (up to 32 warps an SM)
    const uint32_t pitch = (pages + 7) / 8 * 8, units = (pages + unit - 1) / unit;
    const uint64_t fit = std::min<uint64_t>(PG_KEYS_BYTES / ((uint64_t)pitch * 4 * a.pg.n_kv), 0x7fffffffu / ((uint64_t)units * a.pg.n_kv));  // rows of a batch
    if (fit == 0) return cudaErrorInvalidConfiguration;
    *launches = 0;
    for (uint64_t row = 0; row < a.n_rows; row += fit) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(fit, a.n_rows - row);
        PagedSelectArgs b = a;
        b.n_rows = (uint32_t)row + rows;
        // (no early start for the scores: their CTAs would crowd on the SMs that are done first; 121 us instead of 93 with the attention that follows, 64 rows)
        pages_score_kernel<T, HD, MANY><<<(uint32_t)(((uint64_t)rows * units * a.pg.n_kv + 7) / 8), 256, 0, st>>>(b, (uint32_t)row, unit, units, pitch);
        if (cudaError_t e = cudaGetLastError()) return e;
        const dim3 grid(rows * a.pg.n_kv);
        const size_t held = (size_t)std::min(pages, SEL_HELD) * 4;
        if (cudaError_t e = pages <= 4096 ? launch_pdl(pages_pick_kernel<256>, grid, dim3(256), held, st, b, (uint32_t)row, pitch)
                                          : launch_pdl(pages_pick_kernel<1024>, grid, dim3(1024), held, st, b, (uint32_t)row, pitch)) return e;
        *launches += 2;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_pages_select(const PagedSelectArgs &a, int sm_count, cudaStream_t st, uint32_t *launches) {
    auto pick = [&](auto few, auto many) { return a.group > 8 ? many(a, sm_count, st, launches) : few(a, sm_count, st, launches); };
    if (a.pg.is_bf16) return a.pg.dim == 64 ? pick(launch<bf16, 64, false>, launch<bf16, 64, true>) : pick(launch<bf16, 128, false>, launch<bf16, 128, true>);
    return a.pg.dim == 64 ? pick(launch<__half, 64, false>, launch<__half, 64, true>) : pick(launch<__half, 128, false>, launch<__half, 128, true>);
}

}  // namespace ob
