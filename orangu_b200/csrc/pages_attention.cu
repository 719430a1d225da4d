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

#include "pages_walk.cuh"

namespace ob {

namespace {

template <int HD>
struct PaShape {
    static constexpr int PAGE_BYTES = KV_PAGE * HD * 2, SLOT = 2 * PAGE_BYTES;  // keys, then values
    static constexpr int DEPTH = 256 / HD;
    static constexpr int RINGS = PA_WARPS * DEPTH * SLOT;                       // 64 KB
    static constexpr int PITCH = PaResult<HD>::PITCH, PART = PaResult<HD>::PART;
    static_assert(PaResult<HD>::BYTES <= RINGS, "the warps' results meet in the rings");
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
            row0 = wk.u.row0, drafts = wk.u.drafts, n_rows = wk.u.rows * a.group, ctx = wk.u.ctx, limit = wk.u.limit;
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
                if (live) seen[h] = (a.visible ? a.visible[token] : (2ull << t) - 1) & (drafts < 64 ? (1ull << drafts) - 1 : ~0ull);
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
        pa_finish<T, HD, TREE>(a, wk, so, sml, row0, n_rows, head, to, PG_RAISE<T>, s_last);
    }
}

template <typename T, int HD, bool TREE>
cudaError_t launch(PagedAttnArgs a, int sm_count, cudaStream_t st) {
    using S = PaShape<HD>;
    auto kernel = pages_attention_kernel<T, HD, TREE>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::RINGS); })) return e;
    const uint64_t pages = TREE ? (std::min(a.max_ctx, a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE : a.n_list;  // (tree: about, of a sequence)
    const uint64_t most = std::min<uint64_t>({(uint64_t)sm_count * PA_CTAS, PG_COUNTERS, PG_PARTS / (2 * S::PART * 4)});
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
