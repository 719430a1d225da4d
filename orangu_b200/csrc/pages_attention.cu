// Attention over the pages of a cache for few rows a key/value head: the tokens of a tree of drafts with the query heads that share
// the head (ob_pages_attention_tree), or the heads of one token over a list of pages (ob_pages_attention).
//
//   out_r = sum_x w_rx v_x,  w_rx = 2^(s_rx - m_r) / sum_x 2^(s_rx - m_r),  s_rx = scale log2(e) q_r . k_x  over the positions x that row r sees
//
// in one pass with the running maximum m_r and sum.  A CTA has the (up to 16) rows of one key/value head and a stretch of the sequence's
// pages, which its four warps take in turn, each through a ring of its own: no barrier until the end.  Both products are mma.sync m16n8k16
// (f16 or bf16, fp32 accumulators): the bytes of the cache are the bound, and 16 rows fill its tile where a tcgen05 tile needs 128.
// Weights of bf16 caches enter as value and remainder, since 8 bits of weight would be the largest error of the result; f16 has 11.
// The sum of the weights is one more product, with ones, of the same rounded weights.
//
// Few rows of long sequences are cut into stretches over CTAs; each leaves (m, sum, output) in fp32 and the last one to arrive -- a
// counter tells, which goes back to zero by itself -- adds them up in the order of the stretches, so the result does not depend on
// who was last.
#include <algorithm>

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

constexpr float PA_SLACK = 8.0f;  // growth of the maximum (powers of two) that is put up with before the output is rescaled
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

template <typename T, int HD, bool TREE>
__global__ void __launch_bounds__(PA_THREADS, PA_CTAS) pages_attention_kernel(const __grid_constant__ PagedAttnArgs a) {
    using H = Half2<T>;
    using S = PaShape<HD>;
    constexpr int DEPTH = S::DEPTH, KS = HD / 16, CHUNKS = HD / 8;
    constexpr bool REMAINDER = H::ONES == 0x3f803f80u;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_last;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_release();
    pdl_wait();

    // ---- which rows, which pages
    uint32_t b = blockIdx.x;
    const uint32_t head = b % a.pg.n_kv;
    b /= a.pg.n_kv;
    const uint32_t chunk = b % a.max_chunks, unit = b / a.max_chunks, item = unit * a.pg.n_kv + head;
    const uint32_t room = a.pg.stride * KV_PAGE;  // positions a table can name
    uint32_t seq = unit, row0 = unit, n_rows, ctx = 0, limit, n_pages, drafts = 0;
    const int32_t *list = nullptr;
    if constexpr (TREE) {
        const int32_t f0 = a.first[unit], f1 = a.first[unit + 1];
        if (f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens) return;
        row0 = (uint32_t)f0;
        drafts = min((uint32_t)(f1 - f0), a.max_drafts);
        n_rows = drafts * a.group;
        ctx = min(a.n_ctx[unit], room);
        limit = min(ctx + drafts, room);
        n_pages = (limit + KV_PAGE - 1) / KV_PAGE;
    } else {
        const int32_t s = a.row_seq ? a.row_seq[unit] : (int32_t)unit;
        n_rows = a.group;
        limit = (uint32_t)s < a.pg.n_seq ? min(a.n_pos[unit], room) : 0u;
        seq = (uint32_t)s < a.pg.n_seq ? (uint32_t)s : 0u;
        list = a.list + (uint64_t)item * a.n_list;
        n_pages = a.n_list;
    }
    // (a sequence longer than the caller's bound has longer stretches, not more of them)
    const uint32_t even = (n_pages + a.max_chunks - 1) / a.max_chunks, per = max(a.chunk, (even + PA_WARPS - 1) / PA_WARPS * PA_WARPS);
    const uint32_t n_chunks = max(1u, (n_pages + per - 1) / per);
    if (chunk >= n_chunks) return;
    const uint32_t from = chunk * per + warp, to = min(chunk * per + per, n_pages);
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
    const float scale2 = a.scale * 1.4426950408889634f;
    const uint32_t k_row = (lane >> 4) * 8 + (lane & 7), k_half = lane >> 3 & 1, v_row = (lane >> 3 & 1) * 8 + (lane & 7), v_half = lane >> 4;

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
            grown |= now[h] > m[h] + PA_SLACK;  // (the first time, too)
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
                const float off = m[h] == -INFINITY ? 0.0f : -m[h];
                const float e0 = pow2(fmaf(s[n][2 * h], scale2, off)), e1 = pow2(fmaf(s[n][2 * h + 1], scale2, off));
                const uint32_t u = H::pack(e0, e1);
                w[2 * n + h] = u;
                if constexpr (REMAINDER) {
                    const float2 r = H::unpack(u);
                    rest[2 * n + h] = H::pack(e0 - r.x, e1 - r.y);
                }
            }
        H::mma(sum, w, H::ONES, H::ONES);
        if constexpr (REMAINDER) H::mma(sum, rest, H::ONES, H::ONES);
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
                if constexpr (REMAINDER) {
                    H::mma(o[n], rest, f[0], f[1]);
                    H::mma(o[n + 1], rest, f[2], f[3]);
                }
            }
        } else {  // term by term, those that a row sees
#pragma unroll 1
            for (uint32_t j = 0; j < KV_PAGE; ++j) {
                const uint32_t src = (lane & ~3u) | (j & 7) >> 1;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 p = H::unpack(__shfl_sync(0xffffffffu, j < 8 ? w[h] : w[2 + h], src));
                    float x = j & 1 ? p.y : p.x;
                    if constexpr (REMAINDER) {
                        const float2 r = H::unpack(__shfl_sync(0xffffffffu, j < 8 ? rest[h] : rest[2 + h], src));
                        x += j & 1 ? r.y : r.x;
                    }
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
    const bool whole = n_chunks == 1;
    float *part = a.partial + (uint64_t)(item * a.max_chunks + chunk) * S::PART;
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
    if (whole) return;

    // ---- the last stretch to arrive adds them all up
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicInc(a.counters + item, n_chunks - 1) == n_chunks - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    const float *parts = a.partial + (uint64_t)item * a.max_chunks * S::PART;
    for (uint32_t i = threadIdx.x; i < n_rows * VEC; i += PA_THREADS) {
        const uint32_t r = i / VEC, c = i % VEC;
        float top = -INFINITY, l = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (uint32_t k = 0; k < n_chunks; ++k) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(parts + k * S::PART + PA_ROWS * HD + 2 * r));
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(parts + k * S::PART + r * HD + 4 * c));
            if (ml.x == -INFINITY && ml.y == 0.0f) continue;
            const float higher = fmaxf(top, ml.x), f0 = top == -INFINITY ? 0.0f : pow2(top - higher), f1 = ml.x == -INFINITY ? 0.0f : pow2(ml.x - higher);
            top = higher;
            l = fmaf(ml.y, f1, l * f0);
            x.x = fmaf(y.x, f1, x.x * f0), x.y = fmaf(y.y, f1, x.y * f0), x.z = fmaf(y.z, f1, x.z * f0), x.w = fmaf(y.w, f1, x.w * f0);
        }
        store(r, c, x, l);
    }
}

template <typename T, int HD, bool TREE>
cudaError_t launch(PagedAttnArgs a, int sm_count, cudaStream_t st) {
    using S = PaShape<HD>;
    auto kernel = pages_attention_kernel<T, HD, TREE>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::RINGS); })) return e;
    const uint64_t items = (uint64_t)a.n_units * a.pg.n_kv;
    const uint32_t most = TREE ? (std::min(a.max_ctx, a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE : a.n_list;
    // Stretches: a CTA for every place where there are fewer items, several rounds of them where there are more, so that the last round's
    // idle SMs and sequences of different lengths cost little; a stretch has two pages a warp at least.
    const uint64_t slots = (uint64_t)sm_count * PA_CTAS, least = 2 * PA_WARPS;
    uint64_t chunks = items >= 4 * slots ? 1 : items >= slots ? (4 * slots + items - 1) / items : slots / items;
    const uint64_t fit = items <= PG_COUNTERS ? PG_PARTIAL / (items * S::PART * 4) : 1;
    chunks = std::max<uint64_t>(1, std::min({chunks, fit, (most + least - 1) / least}));
    a.chunk = (uint32_t)(((most + chunks - 1) / chunks + PA_WARPS - 1) / PA_WARPS * PA_WARPS);
    a.max_chunks = (uint32_t)std::max<uint64_t>(1, (most + a.chunk - 1) / std::max(1u, a.chunk));
    const uint64_t grid = items * a.max_chunks;
    if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
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
