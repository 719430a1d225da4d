// Attention over the pages of a cache for few rows a key/value head: the tokens of a tree of drafts with the query heads that share
// the head (ob_pages_attention_tree), or the heads of one token over a list of pages (ob_pages_attention).
//
//   out_r = sum_x w_rx v_x,  w_rx = 2^(s_rx - m_r) / sum_x 2^(s_rx - m_r),  s_rx = scale log2(e) q_r . k_x  over the positions x that row r sees
//
// in one pass with the running maximum m_r and sum.  A CTA has the rows of one key/value head (up to 16 MT WR) and a stretch of the
// sequence's pages.  Its warps are WR x WK: WR groups of 16 MT rows share the pages of a ring, WK rings take pages in turn, so that no
// barrier is wider than the warps that share a ring; with 16 or 32 rows every warp has a ring of its own and there is none.  Both products are
// mma.sync m16n8k16 (f16 or bf16, fp32 accumulators): the bytes of the cache are the bound up to about 128 rows a head, and 16 rows
// fill its tile where a tcgen05 tile needs 128.  Weights of bf16 caches enter as value and remainder, since 8 bits of weight would
// be the largest error of the result; f16 has 11.  The sum of the weights is one more product, with ones, of the same rounded weights.
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

__device__ __forceinline__ void group_sync(uint32_t id, uint32_t threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

constexpr float PA_SLACK = 8.0f;  // growth of the maximum (powers of two) that is put up with before the output is rescaled
constexpr int PA_WARPS = 8, PA_THREADS = PA_WARPS * 32;

template <int HD, int MT, int WR>
struct PaShape {
    static constexpr int WK = PA_WARPS / WR, MR = 16 * MT * WR;           // rings, rows
    static constexpr int PAGE_BYTES = KV_PAGE * HD * 2, SLOT = 2 * PAGE_BYTES;  // keys, then values
    static constexpr int DEPTH = 24 / WK;
    static constexpr int RING = WK * DEPTH * SLOT;
    static constexpr int PITCH = HD + 4;                                   // floats of an output row on its way between warps
    static constexpr int MERGE = WK * MR * (PITCH + 2) * 4;
    static constexpr int BYTES = RING > MERGE ? RING : MERGE;
};

template <typename T, int HD, int MT, int WR, bool TREE>
__global__ void __launch_bounds__(PA_THREADS, 1) pages_attention_kernel(const __grid_constant__ PagedAttnArgs a) {
    using H = Half2<T>;
    using S = PaShape<HD, MT, WR>;
    constexpr int WK = S::WK, MR = S::MR, DEPTH = S::DEPTH, KS = HD / 16, CHUNKS = HD / 8;
    constexpr bool REMAINDER = sizeof(T) == 2 && H::ONES == 0x3f803f80u;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_last;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ring = warp / WR, wr = warp % WR;
    pdl_release();
    pdl_wait();

    // ---- which rows, which pages
    uint32_t b = blockIdx.x;
    const uint32_t tile = b % a.row_tiles;
    b /= a.row_tiles;
    const uint32_t head = b % a.pg.n_kv;
    b /= a.pg.n_kv;
    const uint32_t chunk = b % a.max_chunks, unit = b / a.max_chunks, item = (unit * a.pg.n_kv + head) * a.row_tiles + tile;
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
        if (tile * MR >= n_rows) return;
    } else {
        const int32_t s = a.row_seq ? a.row_seq[unit] : (int32_t)unit;
        n_rows = a.group;
        limit = (uint32_t)s < a.pg.n_seq ? min(a.n_pos[unit], room) : 0u;
        seq = (uint32_t)s < a.pg.n_seq ? (uint32_t)s : 0u;
        list = a.list + ((uint64_t)unit * a.pg.n_kv + head) * a.n_list;
        n_pages = a.n_list;
    }
    // (a sequence longer than the caller's bound has longer stretches, not more of them)
    const uint32_t even = (n_pages + a.max_chunks - 1) / a.max_chunks, per = max(a.chunk, (even + WK - 1) / WK * WK);
    const uint32_t n_chunks = max(1u, (n_pages + per - 1) / per);
    if (chunk >= n_chunks) return;
    const uint32_t from = chunk * per, to = min(from + per, n_pages);
    const uint32_t n_steps = to > from + ring ? (to - from - ring + WK - 1) / WK : 0u;
    const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;

    // ---- queries: rows (token, head of the group) of this warp as A fragments
    const uint32_t r_lane = tile * MR + wr * 16 * MT + lane / 4;
    uint32_t q[MT][KS][4];
    uint64_t seen[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = r_lane + 16 * t + 8 * h;
            const bool live = r < n_rows;
            const uint64_t token = row0 + (TREE ? r / a.group : 0u);
            const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(a.q) + (live ? token * a.q_stride + (uint64_t)(head * a.group + r % a.group) * HD : 0u));
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                q[t][s][h] = live ? src[s * 8 + (lane & 3)] : 0u;
                q[t][s][2 + h] = live ? src[s * 8 + 4 + (lane & 3)] : 0u;
            }
            seen[t][h] = 0;
            if constexpr (TREE)
                if (live) seen[t][h] = a.visible[token] & (drafts < 64 ? (1ull << drafts) - 1 : ~0ull);
        }

    // ---- page numbers: lane i has those of step 32 j + i, and of the 32 after them
    auto look = [&](uint32_t step, int32_t &logical) {  // page of a step, or -1
        logical = -1;
        if (step >= n_steps) return -1;
        const uint32_t i = from + ring + step * WK;
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

    const uint32_t base = smem_addr(smem) + ring * DEPTH * S::SLOT;
    const uint64_t page_elems = (uint64_t)a.pg.n_kv * KV_PAGE * HD, head_elems = (uint64_t)head * KV_PAGE * HD;
    auto request = [&](uint32_t step) {  // copies of a step's keys and values, by the warps that share the ring
        if (step < n_steps) {
            int32_t id, logical;
            numbers(step, id, logical);
            if (id >= 0) {
                const uint64_t off = ((uint64_t)id * page_elems + head_elems) * 2;
                const uint8_t *k = static_cast<const uint8_t *>(a.pg.k) + off, *v = static_cast<const uint8_t *>(a.pg.v) + off;
                const uint32_t dst = base + step % DEPTH * S::SLOT, there = limit - (uint32_t)logical * KV_PAGE;  // rows of the page that hold positions
#pragma unroll
                for (int i = 0; i < 2 * HD / (32 * WR); ++i) {
                    const uint32_t c = i * 32 * WR + wr * 32 + lane, row = c / CHUNKS, at = row * HD * 2 + (((c % CHUNKS) ^ (row & 7)) << 4);
                    cp16(dst + at, k + c * 16, row < there);
                    cp16(dst + S::PAGE_BYTES + at, v + c * 16, row < there);
                }
            }
        }
        cp_commit();
    };

    float o[MT][HD / 8][4], sum[MT][4], m[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t][0] = m[t][1] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[t][e] = 0.0f;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][n][e] = 0.0f;
    }
    const float scale2 = a.scale * 1.4426950408889634f;
    const uint32_t k_row = (lane >> 4) * 8 + (lane & 7), k_half = lane >> 3 & 1, v_row = (lane >> 3 & 1) * 8 + (lane & 7), v_half = lane >> 4;

#pragma unroll 1
    for (int i = 0; i < DEPTH - 1; ++i) request(i);
#pragma unroll 1
    for (uint32_t step = 0; step < n_steps; ++step) {
        cp_wait<DEPTH - 2>();
        if constexpr (WR > 1) group_sync(1 + ring, WR * 32);
        else __syncwarp();
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

        float s[MT][2][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][n][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t f[4];
            ldsm4(f, ks + k_row * HD * 2 + (((2 * k + k_half) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                H::mma(s[t][0], q[t][k], f[0], f[1]);
                H::mma(s[t][1], q[t][k], f[2], f[3]);
            }
        }
        const bool drafted = TREE && pos0 + KV_PAGE > ctx, ragged = pos0 + KV_PAGE > limit;
        uint32_t hidden[MT];  // a bit per element of s that its row does not see
#pragma unroll
        for (int t = 0; t < MT; ++t) hidden[t] = 0;
        if (drafted || ragged) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = pos0 + n * 8 + (lane & 3) * 2 + (e & 1);
                        bool see = x < limit;
                        if (TREE && x >= ctx) see = see && (seen[t][e >> 1] >> ((x - ctx) & 63) & 1);  // x - ctx < drafts where x < limit
                        if (!see) s[t][n][e] = -INFINITY, hidden[t] |= 1u << (n * 4 + e);
                    }
        }
        float now[MT][2];
        bool grown = false;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = fmaxf(fmaxf(s[t][0][2 * h], s[t][0][2 * h + 1]), fmaxf(s[t][1][2 * h], s[t][1][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                now[t][h] = x * scale2;
                grown |= now[t][h] > m[t][h] + PA_SLACK;  // (the first time, too)
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float top = fmaxf(m[t][h], now[t][h]), keep = m[t][h] == -INFINITY ? 0.0f : pow2(m[t][h] - top);
                    m[t][h] = top;
                    sum[t][2 * h] *= keep, sum[t][2 * h + 1] *= keep;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) o[t][n][2 * h] *= keep, o[t][n][2 * h + 1] *= keep;
                }
        }
        uint32_t w[MT][4], rest[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float off = m[t][h] == -INFINITY ? 0.0f : -m[t][h];
                    const float e0 = pow2(fmaf(s[t][n][2 * h], scale2, off)), e1 = pow2(fmaf(s[t][n][2 * h + 1], scale2, off));
                    const uint32_t u = H::pack(e0, e1);
                    w[t][2 * n + h] = u;
                    if constexpr (REMAINDER) {
                        const float2 r = H::unpack(u);
                        rest[t][2 * n + h] = H::pack(e0 - r.x, e1 - r.y);
                    }
                }
            H::mma(sum[t], w[t], H::ONES, H::ONES);
            if constexpr (REMAINDER) H::mma(sum[t], rest[t], H::ONES, H::ONES);
        }
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
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    H::mma(o[t][n], w[t], f[0], f[1]);
                    H::mma(o[t][n + 1], w[t], f[2], f[3]);
                    if constexpr (REMAINDER) {
                        H::mma(o[t][n], rest[t], f[0], f[1]);
                        H::mma(o[t][n + 1], rest[t], f[2], f[3]);
                    }
                }
            }
        } else {  // term by term, those that a row sees
#pragma unroll 1
            for (uint32_t j = 0; j < KV_PAGE; ++j) {
                const uint32_t src = (lane & ~3u) | (j & 7) >> 1;
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t word = j < 8 ? w[t][h] : w[t][2 + h], low = j < 8 ? rest[t][h] : rest[t][2 + h];
                        const float2 p = H::unpack(__shfl_sync(0xffffffffu, word, src));
                        float x = j & 1 ? p.y : p.x;
                        if constexpr (REMAINDER) {
                            const float2 r = H::unpack(__shfl_sync(0xffffffffu, low, src));
                            x += j & 1 ? r.y : r.x;
                        }
                        const bool see = !(__shfl_sync(0xffffffffu, hidden[t], src) >> ((j >> 3) * 4 + 2 * h + (j & 1)) & 1);
#pragma unroll
                        for (int n = 0; n < HD / 8; ++n) {
                            uint32_t u;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(vs + j * HD * 2 + ((n ^ (j & 7)) << 4) + (lane & 3) * 4));
                            const float2 v = H::unpack(u);
                            if (see) o[t][n][2 * h] = fmaf(x, v.x, o[t][n][2 * h]), o[t][n][2 * h + 1] = fmaf(x, v.y, o[t][n][2 * h + 1]);
                        }
                    }
            }
        }
    }
    cp_wait<0>();
    __syncthreads();

    // ---- the rings' parts of a row meet in shared memory
    float *so = reinterpret_cast<float *>(smem), *sml = so + WK * MR * S::PITCH;  // [ring][row]
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = ring * MR + wr * 16 * MT + 16 * t + 8 * h + lane / 4;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
                *reinterpret_cast<float2 *>(so + r * S::PITCH + n * 8 + (lane & 3) * 2) = make_float2(o[t][n][2 * h], o[t][n][2 * h + 1]);
            if ((lane & 3) == 0) sml[2 * r] = m[t][h], sml[2 * r + 1] = sum[t][2 * h];
        }
    __syncthreads();
    const uint32_t here = min((uint32_t)MR, n_rows - tile * MR);
    constexpr int VEC = HD / 4;  // of a row, four entries each
    const bool whole = n_chunks == 1;
    float *part = a.partial + (uint64_t)(item * a.max_chunks + chunk) * MR * (HD + 2);
    auto store = [&](uint32_t r, uint32_t c, float4 x, float l) {
        const float f = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // nothing seen: 0; a sum that is no number stays none
        const uint32_t g = tile * MR + r;
        const uint64_t token = row0 + (TREE ? g / a.group : 0u);
        uint2 u = make_uint2(H::pack(x.x * f, x.y * f), H::pack(x.z * f, x.w * f));
        *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + token * a.out_stride + (uint64_t)(head * a.group + g % a.group) * HD + 4 * c) = u;
    };
    for (uint32_t i = threadIdx.x; i < here * VEC; i += PA_THREADS) {
        const uint32_t r = i / VEC, c = i % VEC;
        float top = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < WK; ++k) top = fmaxf(top, sml[2 * (k * MR + r)]);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            const float mk = sml[2 * (k * MR + r)], f = mk == -INFINITY ? 0.0f : pow2(mk - top);
            if (mk == -INFINITY && sml[2 * (k * MR + r) + 1] == 0.0f) continue;
            const float4 y = *reinterpret_cast<const float4 *>(so + (k * MR + r) * S::PITCH + 4 * c);
            l = fmaf(sml[2 * (k * MR + r) + 1], f, l);
            x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
        }
        if (whole) {
            store(r, c, x, l);
        } else {
            __stcg(reinterpret_cast<float4 *>(part + (uint64_t)r * HD + 4 * c), x);
            if (c == 0) __stcg(reinterpret_cast<float2 *>(part + (uint64_t)MR * HD + 2 * r), make_float2(top, l));
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
    const float *parts = a.partial + (uint64_t)item * a.max_chunks * MR * (HD + 2);
    constexpr uint64_t STEP = (uint64_t)MR * (HD + 2);
    for (uint32_t i = threadIdx.x; i < here * VEC; i += PA_THREADS) {
        const uint32_t r = i / VEC, c = i % VEC;
        float top = -INFINITY, l = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t k = 0; k < n_chunks; ++k) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(parts + k * STEP + (uint64_t)MR * HD + 2 * r));
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(parts + k * STEP + (uint64_t)r * HD + 4 * c));
            if (ml.x == -INFINITY && ml.y == 0.0f) continue;
            const float new_top = fmaxf(top, ml.x), f0 = top == -INFINITY ? 0.0f : pow2(top - new_top), f1 = ml.x == -INFINITY ? 0.0f : pow2(ml.x - new_top);
            top = new_top;
            l = fmaf(ml.y, f1, l * f0);
            x.x = fmaf(y.x, f1, x.x * f0), x.y = fmaf(y.y, f1, x.y * f0), x.z = fmaf(y.z, f1, x.z * f0), x.w = fmaf(y.w, f1, x.w * f0);
        }
        store(r, c, x, l);
    }
}

template <typename T, int HD, int MT, int WR, bool TREE>
cudaError_t launch(PagedAttnArgs a, int sm_count, cudaStream_t st) {
    using S = PaShape<HD, MT, WR>;
    auto kernel = pages_attention_kernel<T, HD, MT, WR, TREE>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES); })) return e;
    const uint64_t rows = TREE ? (uint64_t)a.max_drafts * a.group : a.group;
    a.row_tiles = (uint32_t)((rows + S::MR - 1) / S::MR);
    const uint64_t items = (uint64_t)a.n_units * a.pg.n_kv * a.row_tiles;
    const uint32_t most = TREE ? (std::min(a.max_ctx, a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE : a.n_list;
    // Stretches: a CTA for every SM where there are fewer items, several rounds of them where there are more, so that the last round's
    // idle SMs and sequences of different lengths cost little; a stretch has two pages a ring at least.
    const uint64_t slots = sm_count;
    uint64_t chunks = items >= 4 * slots ? 1 : items >= slots ? (4 * slots + items - 1) / items : slots / items;
    const uint64_t fit = items <= PG_COUNTERS ? PG_PARTIAL / (items * S::MR * (HD + 2) * 4) : 1;
    chunks = std::max<uint64_t>(1, std::min({chunks, fit, (uint64_t)(most + 2 * S::WK - 1) / (2 * S::WK)}));
    a.chunk = (uint32_t)(((most + chunks - 1) / chunks + S::WK - 1) / S::WK * S::WK);
    a.max_chunks = (uint32_t)std::max<uint64_t>(1, (most + a.chunk - 1) / std::max(1u, a.chunk));
    const uint64_t grid = items * a.max_chunks;
    if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    return launch_pdl(kernel, dim3((uint32_t)grid), dim3(PA_THREADS), S::BYTES, st, a);
}

template <typename T, int HD>
cudaError_t launch_rows(const PagedAttnArgs &a, bool tree, int sm_count, cudaStream_t st) {
    if (!tree) return launch<T, HD, 1, 1, false>(a, sm_count, st);
    const uint32_t rows = a.max_drafts * a.group;
    if (rows <= 16) return launch<T, HD, 1, 1, true>(a, sm_count, st);
    if (rows <= 32) return launch<T, HD, 2, 1, true>(a, sm_count, st);
    if (rows <= 64) return launch<T, HD, 2, 2, true>(a, sm_count, st);
    return launch<T, HD, 2, 4, true>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_pages_attention(PagedAttnArgs a, bool tree, int sm_count, cudaStream_t st) {
    if (a.pg.is_bf16) return a.pg.dim == 64 ? launch_rows<bf16, 64>(a, tree, sm_count, st) : launch_rows<bf16, 128>(a, tree, sm_count, st);
    return a.pg.dim == 64 ? launch_rows<__half, 64>(a, tree, sm_count, st) : launch_rows<__half, 128>(a, tree, sm_count, st);
}

}  // namespace ob
