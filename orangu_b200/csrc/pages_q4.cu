// Attention over pages in 4 bits (layout: pages_q4.cuh) for few rows (token, query head) a key/value head: the mathematics of pages_attention.cu, whose
// walk and sums of parts it shares, with the entries made f16 numbers on their way into the products.  They are that exactly, so nothing is lost here that the codes have.
//
// Both products are mma.sync m16n8k16 with the page's side as its 16 rows: scores^T = keys x queries^T (16 positions x 8 rows), then
// output^T += values^T x weights^T (16 dimensions x 8 rows), whose weights come out of the scores' registers by one exchange of 8 x 8 halves.  Up to 8
// rows are half the products that 16 rows on the other side would be.  The order of a product's terms is free: a lane takes 16 neighbouring bytes of a key and
// of two values.  Queries are f16; bfloat16 ones become that after a power of two per row has been taken out (their 8 bits fit, and what
// falls below 2^-24 of 2^14 is less than 2^-38 of the row's largest).  Weights enter as value and remainder, raised by 2^7, as over f16 pages: the value alone is off by up to
// 2^-11, which is more than a bfloat16 output's own rounding where values cancel.
//
// 9 bits for two entries: a page of a head is 18 HD bytes, keys and values, and with 128 entries about 373 instructions of the loop (4-bit words to entries 176, products 24, copies, scores
// and weights the rest), 401 with starts and ends.  In the time of the bytes an SM can issue 396 (at 1.9 GHz): the two floors are the same, and there is little room for a gap.  64
// sequences of 4 to 16 k, 8 heads of 128, 4 rows: 183 us, 3.8 TB/s (115 with the copies alone), 64 of 64 entries 121 us.  59 % of the issue slots are used and no pipe more than 42 %;
// what the warps, 16 an SM, wait for most are the latencies of their own instructions.  More CTAs an SM, deeper rings, products apart or two sums of scores at once changed nothing.
#include <algorithm>

#include "pages_q4.cuh"
#include "pages_walk.cuh"

namespace ob {

namespace {

template <int HD>
struct P4Shape {
    static constexpr uint32_t BLOCK = Q4Block<HD>::BYTES, SLOT = 2 * BLOCK;
    static constexpr int DEPTH = HD == 128 ? 4 : 5;
    static constexpr int RINGS = PA_WARPS * DEPTH * SLOT;
    static_assert(PaResult<HD>::BYTES <= RINGS && SLOT % 16 == 0, "the warps' results meet in the rings");
};

__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // of 8 x 8 halves, two of a row a lane
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// NT: columns of eight rows.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(PA_THREADS, NT == 1 ? 4 : 3) pages_q4_attention_kernel(const __grid_constant__ PagedAttnArgs a) {
    using F = Half2<__half>;
    using S = P4Shape<HD>;
    using B = Q4Block<HD>;
    constexpr int DEPTH = S::DEPTH, KW = HD / 32, MT = HD / 16;  // words of a lane: of a key, of two values; tiles of dimensions
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_last;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_release();
    pdl_wait();

    const float scale2 = a.scale * 1.4426950408889634f;
    // this lane's places in a block
    const uint32_t k_at = g * B::ROW + t * (HD / 8), k_unit = B::CODES + 2 * (g * B::GROUPS + t * (HD / 4) / Q4_GROUP);
    const uint32_t v_at = t * HD + 8 * B::eight(t, g * (HD / 64)), v_unit = B::CODES + 2 * (g * (HD / 8) / Q4_GROUP * KV_PAGE + 2 * t);
    PaWalk<true> wk;
    wk.start(a);
    for (; wk.more(); wk.next(a)) {
        const uint32_t head = wk.head, seq = a.blocks > 1 ? wk.unit / a.blocks : wk.unit;
        const uint32_t row0 = wk.u.row0, n_rows = wk.u.rows * a.group, ctx = wk.u.ctx, limit = wk.u.limit, drafts = wk.u.drafts;
        const uint32_t from = wk.page + warp, to = wk.last();
        const uint32_t n_steps = to > from ? (to - from + PA_WARPS - 1) / PA_WARPS : 0u;  // pages of this warp
        const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;

        // ---- page numbers: lane i has those of step 32 j + i, and of the 32 after them
        auto look = [&](uint32_t step) {  // page of a step, or -1
            if (step >= n_steps) return -1;
            const int32_t id = table[from + step * PA_WARPS];
            return (uint32_t)id < a.pg.n_pages ? id : -1;
        };
        int32_t id_now = look(lane), id_next = look(32 + lane);
        uint32_t block = 0;  // steps 32 block ..: id_now
        auto number = [&](uint32_t step) { return __shfl_sync(0xffffffffu, step / 32 != block ? id_next : id_now, step & 31); };  // steps [32 block, 32 block + 64)

        const uint32_t base = smem_addr(smem) + warp * DEPTH * S::SLOT;
        // copies of a step's keys and values, 16 bytes a lane and turn; in the turn that has the end of the keys and the start of the values the lanes go apart
        constexpr uint32_t WORDS = S::BLOCK / 16, KEY_TURNS = WORDS / 32, ODD = WORDS % 32;
        static_assert(ODD <= 16, "the second turn of the values begins behind the lanes that had the keys' end");
        const uint8_t *k_base = static_cast<const uint8_t *>(a.pg.k) + (uint64_t)head * S::BLOCK + lane * 16, *v_base = static_cast<const uint8_t *>(a.pg.v) + (uint64_t)head * S::BLOCK + lane * 16;
        const uint64_t page_bytes = (uint64_t)a.pg.n_kv * S::BLOCK;
        auto request = [&](uint32_t step, uint32_t place) {
            if (step < n_steps) {
                const int32_t id = number(step);
                if (id >= 0) {
                    const uint64_t off = (uint32_t)id * page_bytes;
                    const uint8_t *k = k_base + off, *v = v_base + off;
                    const uint32_t dst = base + place + lane * 16;
#pragma unroll
                    for (uint32_t i = 0; i < KEY_TURNS; ++i) {
                        cp16(dst + i * 512, k + i * 512, true);
                        cp16(dst + S::BLOCK + i * 512, v + i * 512, true);
                    }
                    if (lane < ODD) cp16(dst + KEY_TURNS * 512, k + KEY_TURNS * 512, true);
                    else if (lane < 2 * ODD) cp16(dst + S::BLOCK + KEY_TURNS * 512 - ODD * 16, v + KEY_TURNS * 512 - ODD * 16, true);
                }
            }
            cp_commit();
        };
#pragma unroll 1
        for (int i = 0; i < DEPTH - 1; ++i) request(i, i * S::SLOT);

        // ---- queries as B fragments: lane (g, t) has entries t HD / 4 .. of row g of each set of eight
        uint32_t q[NT][HD / 8];
        float fac[NT][2];  // of this lane's columns 2 t, 2 t + 1
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t r = n * 8 + g, tok = r / a.group;
            const bool live = r < n_rows;
            const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (live ? (uint64_t)(row0 + tok) * a.q_stride + (uint64_t)(head * a.group + r - tok * a.group) * HD + t * (HD / 4) : 0u));
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                const uint4 x = live ? src[i] : make_uint4(0, 0, 0, 0);
                q[n][4 * i] = x.x, q[n][4 * i + 1] = x.y, q[n][4 * i + 2] = x.z, q[n][4 * i + 3] = x.w;
            }
            float mine = 1.0f;
            if constexpr (!std::is_same<T, __half>::value) {
                uint32_t top = 0;  // the largest magnitude's bits
#pragma unroll
                for (int i = 0; i < HD / 8; ++i) top = max(top, max(q[n][i] & 0x7fffu, q[n][i] >> 16 & 0x7fffu));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^14 is the largest's power of two afterwards; none is taken out of rows with infinities or no numbers, nor of zeros
                const int e = top == 0 || top >= 0x7f80u ? 0 : max(-112, min(112, 14 - ((int)(top >> 7) - 127)));
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                mine = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int i = 0; i < HD / 8; ++i) {
                    const float2 x = Half2<T>::unpack(q[n][i]);
                    q[n][i] = F::pack(x.x * up, x.y * up);
                }
            }
            fac[n][0] = __shfl_sync(0xffffffffu, mine, 8 * t) * scale2, fac[n][1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4) * scale2;
        }

        float o[MT][NT][4], sum[NT][2], m[NT][2], off[NT][2];  // off: what is added to a score's exponent
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            sum[n][0] = sum[n][1] = off[n][0] = off[n][1] = 0.0f, m[n][0] = m[n][1] = -INFINITY;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.0f;
        }

        uint32_t place = 0, ahead = (DEPTH - 1) * S::SLOT;  // of this step, of the one that is asked for
        int32_t id = number(0);
#pragma unroll 1
        for (uint32_t step = 0; step < n_steps; ++step) {
            cp_wait<DEPTH - 2>();
            __syncwarp();
            if (step / 32 != block) {
                block = step / 32;
                id_now = id_next;
                id_next = look(32 * (block + 1) + lane);
            }
            request(step + DEPTH - 1, ahead);
            const int32_t now = id;
            const uint32_t ks = base + place;
            id = number(step + 1);
            ahead = place;
            place = place == (DEPTH - 1) * S::SLOT ? 0 : place + S::SLOT;
            if (now < 0) continue;
            const uint32_t vs = ks + S::BLOCK, pos0 = (from + step * PA_WARPS) * KV_PAGE;

            // ---- scores of positions g and g + 8 (rows) for rows 2 t, 2 t + 1 of each set
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
            {
                uint32_t w0[KW], w1[KW];
                lds_words(w0, ks + k_at);
                lds_words(w1, ks + k_at + 8 * B::ROW);
                const uint32_t d0 = lds16(ks + k_unit) * 0x10001u, d1 = lds16(ks + k_unit + 16 * B::GROUPS) * 0x10001u, n0 = q4_offset(d0), n1 = q4_offset(d1);
#pragma unroll
                for (int i = 0; i < KW; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t f[4] = {q4_field(w0[i], 2 * h, d0, n0), q4_field(w1[i], 2 * h, d1, n1), q4_field(w0[i], 2 * h + 1, d0, n0), q4_field(w1[i], 2 * h + 1, d1, n1)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) F::mma(s[n], f, q[n][4 * i + 2 * h], q[n][4 * i + 2 * h + 1]);
                    }
            }
            const bool drafted = pos0 + KV_PAGE > ctx, ragged = pos0 + KV_PAGE > limit;
            if (drafted) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t r = n * 8 + 2 * t + c, tok = r / a.group;
                        uint64_t seen = 0;
                        if (r < n_rows) seen = (a.visible ? a.visible[row0 + tok] : (2ull << tok) - 1) & (drafts < 64 ? (1ull << drafts) - 1 : ~0ull);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x = pos0 + g + 8 * h;
                            if (x >= limit || (x >= ctx && !(seen >> ((x - ctx) & 63) & 1))) s[n][2 * h + c] = -INFINITY;
                        }
                    }
            }
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) grown |= fmaxf(s[n][c], s[n][2 + c]) * fac[n][c] > m[n][c] + PG_SLACK;  // (the first time, too)
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float x = fmaxf(s[n][c], s[n][2 + c]) * fac[n][c];
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float top = fmaxf(m[n][c], x), keep = m[n][c] == -INFINITY ? 0.0f : pow2(m[n][c] - top);
                        m[n][c] = top, off[n][c] = top == -INFINITY ? 0.0f : PG_RAISE<__half> - top;
                        sum[n][c] *= keep;
#pragma unroll
                        for (int i = 0; i < MT; ++i) o[i][n][c] *= keep, o[i][n][2 + c] *= keep;
                    }
            }
            uint32_t w[NT][2], rest[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float e0 = pow2(fmaf(s[n][2 * h], fac[n][0], off[n][0])), e1 = pow2(fmaf(s[n][2 * h + 1], fac[n][1], off[n][1]));
                    sum[n][0] += e0, sum[n][1] += e1;
                    const uint32_t u = F::pack(e0, e1);
                    const float2 r = F::unpack(u);
                    w[n][h] = transposed(u), rest[n][h] = transposed(F::pack(e0 - r.x, e1 - r.y));
                }
            }
            // ---- outputs of the lane's dimensions: positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9
            uint32_t u0 = lds32(vs + v_unit), u1 = lds32(vs + v_unit + 16);
            if (ragged) {  // what nobody has written counts as zero, whatever is there
                const uint32_t x = pos0 + 2 * t;
                u0 &= (x < limit ? 0xffffu : 0u) | (x + 1 < limit ? 0xffff0000u : 0u);
                u1 &= (x + 8 < limit ? 0xffffu : 0u) | (x + 9 < limit ? 0xffff0000u : 0u);
            }
            const uint32_t n0 = q4_offset(u0), n1 = q4_offset(u1);
            uint32_t v0[KW], v1[KW];
            lds_words(v0, vs + v_at);
            lds_words(v1, vs + v_at + 4 * HD);
#pragma unroll
            for (int i = 0; i < KW; i += 2)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t f[4] = {q4_field(v0[i], j, u0, n0), q4_field(v0[i + 1], j, u0, n0), q4_field(v1[i], j, u1, n1), q4_field(v1[i + 1], j, u1, n1)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        F::mma(o[2 * i + j][n], f, w[n][0], w[n][1]);
                        F::mma(o[2 * i + j][n], f, rest[n][0], rest[n][1]);
                    }
                }
        }
        cp_wait<0>();
        __syncthreads();

        // ---- the warps' parts of a row meet in shared memory: lane (g, t) has dimensions g HD / 8 .. of rows 2 t, 2 t + 1
        constexpr int PITCH = PaResult<HD>::PITCH;
        float *so = reinterpret_cast<float *>(smem), *sml = so + PA_WARPS * PA_ROWS * PITCH;  // [warp][row]
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t r = warp * PA_ROWS + n * 8 + 2 * t + c;
#pragma unroll
                for (int i = 0; i < MT; i += 2) *reinterpret_cast<float4 *>(so + r * PITCH + g * (HD / 8) + 2 * i) = make_float4(o[i][n][c], o[i][n][2 + c], o[i + 1][n][c], o[i + 1][n][2 + c]);
                float l = sum[n][c];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) sml[2 * r] = m[n][c], sml[2 * r + 1] = l;
            }
        pa_finish<T, HD, true, NT == 1 ? 8 : 16>(a, wk, so, sml, row0, n_rows, head, to, PG_RAISE<__half>, s_last);
    }
}

template <typename T, int HD, int NT>
cudaError_t launch(const PagedAttnArgs &a, int sm_count, cudaStream_t st) {
    using S = P4Shape<HD>;
    auto kernel = pages_q4_attention_kernel<T, HD, NT>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::RINGS); })) return e;
    const uint64_t pages = (std::min<uint64_t>(a.max_ctx, (uint64_t)a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE;  // about, of a sequence
    const uint64_t most = std::min<uint64_t>({(uint64_t)sm_count * (NT == 1 ? 4 : 3), PG_COUNTERS, PG_PARTS / (2 * PaResult<HD>::PART * 4)});
    const uint64_t grid = std::min(most, std::max<uint64_t>(1, a.n_units * ((pages + PA_LEAST - 1) / PA_LEAST) * a.pg.n_kv));
    return launch_pdl(kernel, dim3((uint32_t)grid), dim3(PA_THREADS), S::RINGS, st, a);
}
template <typename T>
cudaError_t launch_dim(const PagedAttnArgs &a, int sm_count, cudaStream_t st) {
    const bool few = std::min(a.max_drafts, a.block) * a.group <= 8;
    if (a.pg.dim == 64) return few ? launch<T, 64, 1>(a, sm_count, st) : launch<T, 64, 2>(a, sm_count, st);
    return few ? launch<T, 128, 1>(a, sm_count, st) : launch<T, 128, 2>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_pages_q4_attention(const PagedAttnArgs &a, bool q_bf16, int sm_count, cudaStream_t st) {
    return q_bf16 ? launch_dim<bf16>(a, sm_count, st) : launch_dim<__half>(a, sm_count, st);
}

}  // namespace ob
