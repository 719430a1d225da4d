// Which pages a row reads (ob_pages_select): a score for every page of the row's sequence, per key/value head, from bounds of the page's
// keys in 8 bits, and the best n_select of them.
//
//   q_h,e ~ dq_h c_h,e  with dq_h = max_e |q_h,e| / 127, c = rint(q / dq);  hi_e, lo_e: codes of the page's largest and smallest key, unit d
//   score = max over the heads h of  (dq_h d) * sum_e max(c_h,e hi_e, c_h,e lo_e)  =  (dq_h d) * (sum_e max(c, 0) hi_e + sum_e min(c, 0) lo_e)
//
// The sum is a whole number below 2^24 and the two products are single roundings, so a score has one value whatever the order of
// the terms, and so has the choice.  A row's sum over (hi, lo) is one row of an s8 product of length 2 dim: mma.sync m16n8k32 with the
// heads as the 16 rows and 8 pages as columns, whose codes go from memory straight into the fragments (a lane's 16 bytes serve
// two steps; the order of the terms inside a step is free).  What bounds it is the reading of the codes, 2 dim + 4 bytes a page.
//
// One cluster per (row, head): its CTAs share the pages, keep the scores as ordered 32-bit words in shared memory, and find the
// n_select'th by four rounds of 8 bits, adding the CTAs' histograms up through distributed shared memory.  Pages above it are taken, and
// of those that equal it the first ones; the list is written in ascending order without another pass over memory.
#include <cooperative_groups.h>

#include <algorithm>

#include "mixers_common.cuh"
#include "pages.h"

namespace ob {

namespace {

namespace cg = cooperative_groups;

constexpr int SEL_WARPS = 8, SEL_THREADS = SEL_WARPS * 32;
constexpr uint32_t SEL_CLUSTER = 8;        // most CTAs of a cluster
constexpr uint32_t SEL_KEYS = 16384;       // most pages of a CTA
constexpr float SEL_MOST = 1e18f;          // what larger queries count as: products of two units and a sum stay finite

__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(bf16 v) { return __bfloat162float(v); }

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

// MANY: more than eight heads a key/value head; the lower half of the product's rows is empty otherwise.
template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(SEL_THREADS, MANY ? 2 : 4) pages_select_kernel(const __grid_constant__ PagedSelectArgs a, uint32_t n_cta, uint32_t cap) {
    constexpr int LOADS = 2 * HD / 64;  // 16-byte loads of a lane per page: a quarter of the page's codes
    extern __shared__ __align__(16) uint32_t keys[];  // [cap]
    __shared__ __align__(16) int8_t s_code[PG_MAX_GROUP][HD];
    __shared__ float s_unit[PG_MAX_GROUP];
    __shared__ uint32_t s_hist[4][256], s_warp[2][SEL_WARPS], s_pick[3], s_count[2];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = n_cta > 1 ? cg::this_cluster().block_rank() : 0u;
    pdl_release();
    pdl_wait();
    const uint32_t pair = blockIdx.x / n_cta, head = pair % a.pg.n_kv, row = pair / a.pg.n_kv;
    const int32_t s = a.row_seq ? a.row_seq[row] : (int32_t)row;
    const bool known = (uint32_t)s < a.pg.n_seq;
    const uint32_t n_pos = known ? min(min(a.n_pos[row], a.max_pos), a.pg.stride * KV_PAGE) : 0u, n_pages = (n_pos + KV_PAGE - 1) / KV_PAGE;
    const int32_t *table = a.pg.tables + (uint64_t)(known ? s : 0) * a.pg.stride;
    int32_t *out = a.selected + (uint64_t)pair * a.n_select;
    if (n_pages <= a.n_select) {  // all of them (every CTA of the cluster leaves here)
        if (rank == 0)
            for (uint32_t i = threadIdx.x; i < a.n_select; i += SEL_THREADS) out[i] = i < n_pages ? (int32_t)i : -1;
        return;
    }
    const uint32_t share = (n_pages + n_cta - 1) / n_cta, p0 = min(rank * share, n_pages), n = min(share, n_pages - p0);  // this CTA's pages

    // ---- the queries' codes
    constexpr uint32_t HEADS = MANY ? 16 : 8, WORDS = MANY ? 4 : 2;  // words of an A fragment that are not always zero
#pragma unroll 1
    for (uint32_t h = warp; h < HEADS; h += SEL_WARPS) {
        float x[HD / 32], top = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            x[i] = h < a.group ? as_float(static_cast<const T *>(a.q)[(uint64_t)row * a.q_stride + (uint64_t)(head * a.group + h) * HD + i * 32 + lane]) : 0.0f;
            if (x[i] != x[i]) x[i] = 0.0f;
            x[i] = fminf(fmaxf(x[i], -SEL_MOST), SEL_MOST);
            top = fmaxf(top, fabsf(x[i]));
        }
        top = warp_max(top);
        const float d = __fdiv_rn(top, 127.0f), by = d > 0.0f ? d : 1.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) s_code[h][i * 32 + lane] = (int8_t)fminf(fmaxf(rintf(__fdiv_rn(x[i], by)), -127.0f), 127.0f);
        if (lane == 0) s_unit[h] = h < a.group ? d : -1.0f;
    }
    for (uint32_t i = threadIdx.x; i < 4 * 256; i += SEL_THREADS) (&s_hist[0][0])[i] = 0u;
    __syncthreads();
    // Load i of a lane is bytes 64 i + 16 (lane % 4) .. + 15 of a page's codes; its words 0, 1 and 2, 3 are the two halves of a step's 32.
    uint32_t f[LOADS][2][WORDS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < (int)WORDS; ++e) {
                const uint32_t at = i * 64 + (lane & 3) * 16 + j * 8 + e / (WORDS / 2) * 4, h = lane / 4 + (MANY ? e & 1 : 0) * 8;
                const uint32_t c = *reinterpret_cast<const uint32_t *>(&s_code[h][at % HD]);
                f[i][j][e] = at < HD ? __vmaxs4(c, 0u) : __vmins4(c, 0u);  // largest keys meet the positive codes, smallest the others
            }
    const float unit0 = s_unit[lane / 4], unit1 = MANY ? s_unit[lane / 4 + 8] : -1.0f;
    auto product = [&](int(&c)[4], const uint32_t(&w)[WORDS], uint32_t b0, uint32_t b1) {
        if constexpr (MANY) {
            mma_s8(c, w, b0, b1);
        } else {
            const uint32_t x[4] = {w[0], 0u, w[1], 0u};
            mma_s8(c, x, b0, b1);
        }
    };

    // ---- scores: a warp takes eight pages at a time, two such groups in flight
    const uint64_t rec = 2 * HD;
    const uint32_t col = (lane & 3) * 2;  // this lane's two columns of a product
    auto page_of = [&](uint32_t i) {
        if (i >= n) return -1;
        const int32_t id = table[p0 + i];
        return (uint32_t)id < a.pg.n_pages ? id : -1;
    };
    constexpr int AHEAD = 2;
    int32_t id[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) id[u] = page_of((warp + u * SEL_WARPS) * 8 + lane / 4);
    for (uint32_t g = warp; g * 8 < n; g += AHEAD * SEL_WARPS) {
        uint4 x[AHEAD][LOADS];
        float d[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint64_t at = (uint64_t)(uint32_t)max(id[u], 0) * a.pg.n_kv + head;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) x[u][i] = id[u] < 0 ? make_uint4(0, 0, 0, 0) : ldg128_stream(a.codes + at * rec + i * 64 + (lane & 3) * 16);
            d[u] = id[u] < 0 ? __int_as_float(0x7fc00000) : __ldg(a.scales + at);  // a page that is not there: no number
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) id[u] = page_of((g + (AHEAD + u) * SEL_WARPS) * 8 + lane / 4);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            int c[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                product(c, f[i][0], x[u][i].x, x[u][i].y);
                product(c, f[i][1], x[u][i].z, x[u][i].w);
            }
            float best[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float dp = __shfl_sync(0xffffffffu, d[u], (col + e) * 4);
                const float s0 = unit0 < 0.0f ? -INFINITY : __fmul_rn(__fmul_rn(unit0, dp), (float)c[e]);
                float y = s0;
                if (MANY && unit1 >= 0.0f) y = fmaxf(y, __fmul_rn(__fmul_rn(unit1, dp), (float)c[2 + e]));  // (fmaxf gives -inf only where no head is: heads of a page that is not there are all no numbers)
                if (dp != dp) y = dp;
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
                best[e] = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
            }
            const uint32_t i = (g + u * SEL_WARPS) * 8 + col;
            if (lane < 4) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (i + e < n) {
                        const uint32_t p = p0 + i + e;
                        keys[i + e] = p < a.keep_first || p + a.keep_last >= n_pages ? 0xffffffffu : ordered(best[e]);
                    }
            }
        }
    }
    __syncthreads();

    // ---- the n_select'th largest word
    uint32_t prefix = 0, want = a.n_select;  // of the words that begin with the prefix, the want'th largest is looked for
    int shift = 24;
#pragma unroll 1
    for (int round = 0;; ++round, shift -= 8) {
        uint32_t *hist = s_hist[round];
        for (uint32_t i = threadIdx.x; i < (n + 31) / 32 * 32; i += SEL_THREADS) {
            const uint32_t k = i < n ? keys[i] : 0u;
            const bool in = i < n && (round == 0 || (k >> (shift + 8)) == prefix);
            const uint32_t digit = in ? (k >> shift) & 255u : 256u;
            const uint32_t same = __match_any_sync(0xffffffffu, digit);  // scores are close together: one addition for equal digits
            if (in && lane == (uint32_t)__ffs(same) - 1) atomicAdd(hist + digit, __popc(same));
        }
        if (n_cta > 1) cg::this_cluster().sync();
        else __syncthreads();
        uint32_t total = 0;  // thread t: digit 255 - t
        const uint32_t digit = 255 - threadIdx.x;
        if (n_cta > 1) {
            for (uint32_t c = 0; c < n_cta; ++c) total += cg::this_cluster().map_shared_rank(hist, c)[digit];
        } else {
            total = hist[digit];
        }
        uint32_t upto = total;  // words with this digit or a larger one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += up;
        }
        if (lane == 31) s_warp[round & 1][warp] = upto;
        __syncthreads();
        for (uint32_t w = 0; w < warp; ++w) upto += s_warp[round & 1][w];
        if (upto >= want && upto - total < want) s_pick[0] = digit, s_pick[1] = want - (upto - total), s_pick[2] = total;
        __syncthreads();
        prefix = prefix << 8 | s_pick[0];
        want = s_pick[1];
        if (round == 3 || want == s_pick[2]) break;  // (all words that begin so are taken: no need to look further)
        __syncthreads();
    }
    // ---- words that begin with more than the prefix: all; with the prefix: the first `want` of all CTAs
    const uint32_t span = (n + SEL_WARPS - 1) / SEL_WARPS, w0 = min(warp * span, n), w1 = min(w0 + span, n);  // this warp's pages
    uint32_t above = 0, equal = 0;
    for (uint32_t i = w0 + lane; i < w1; i += 32) above += keys[i] >> shift > prefix, equal += keys[i] >> shift == prefix;
    above = warp_sum_i(above), equal = warp_sum_i(equal);
    if (lane == 0) s_warp[0][warp] = above, s_warp[1][warp] = equal;
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t x = 0, y = 0;
        for (int w = 0; w < SEL_WARPS; ++w) x += s_warp[0][w], y += s_warp[1][w];
        s_count[0] = x, s_count[1] = y;
    }
    if (n_cta > 1) cg::this_cluster().sync();
    else __syncthreads();
    above = equal = 0;  // before this warp
    for (uint32_t c = 0; c < rank; ++c) {
        const uint32_t *r = cg::this_cluster().map_shared_rank(s_count, c);
        above += r[0], equal += r[1];
    }
    for (uint32_t w = 0; w < warp; ++w) above += s_warp[0][w], equal += s_warp[1][w];
    for (uint32_t i = w0; i < w1; i += 32) {
        const uint32_t k = i + lane < w1 ? keys[i + lane] >> shift : 0u;
        const bool live = i + lane < w1;
        const uint32_t gt = __ballot_sync(0xffffffffu, live && k > prefix), eq = __ballot_sync(0xffffffffu, live && k == prefix), below = (1u << lane) - 1;
        const uint32_t ga = above + __popc(gt & below), ea = equal + __popc(eq & below);
        if ((gt >> lane & 1) || ((eq >> lane & 1) && ea < want)) out[ga + min(ea, want)] = (int32_t)(p0 + i + lane);
        above += __popc(gt), equal += __popc(eq);
    }
    if (n_cta > 1) cg::this_cluster().sync();  // nobody leaves while its counts may still be read
}

template <typename T, int HD, bool MANY>
cudaError_t launch(const PagedSelectArgs &a, int sm_count, cudaStream_t st) {
    auto kernel = pages_select_kernel<T, HD, MANY>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_KEYS * 4); })) return e;
    const uint32_t pages = std::max(1u, (std::min(a.max_pos, a.pg.stride * KV_PAGE) + KV_PAGE - 1) / KV_PAGE);
    const uint64_t pairs = (uint64_t)a.n_rows * a.pg.n_kv;
    // More CTAs a row while the SMs are not all taken four times and a CTA keeps 64 pages (a group of eight for each warp), or while a CTA's
    // words would not fit.
    uint32_t c = 1;
    while (c < SEL_CLUSTER && ((pairs * c * 2 <= 4ull * sm_count && pages / (2 * c) >= 64) || (pages + c - 1) / c > SEL_KEYS)) c *= 2;
    const uint32_t cap = (pages + c - 1) / c;
    if (pairs * c > 0x7fffffffull || cap > SEL_KEYS) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = c, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((uint32_t)(pairs * c));
    cfg.blockDim = dim3(SEL_THREADS);
    cfg.dynamicSmemBytes = (size_t)cap * 4;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a, c, cap);
}

}  // namespace

uint32_t pages_select_most() { return SEL_CLUSTER * SEL_KEYS; }

cudaError_t launch_pages_select(const PagedSelectArgs &a, int sm_count, cudaStream_t st) {
    auto pick = [&](auto few, auto many) { return a.group > 8 ? many(a, sm_count, st) : few(a, sm_count, st); };
    if (a.pg.is_bf16) return a.pg.dim == 64 ? pick(launch<bf16, 64, false>, launch<bf16, 64, true>) : pick(launch<bf16, 128, false>, launch<bf16, 128, true>);
    return a.pg.dim == 64 ? pick(launch<__half, 64, false>, launch<__half, 64, true>) : pick(launch<__half, 128, false>, launch<__half, 128, true>);
}

}  // namespace ob
