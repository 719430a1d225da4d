// The weights that every position gets, added up over the rows and query heads that see it (ob_pages_attention_tokens with masses).
//
//   mass[s][h][x] += sum over the tokens and heads r of h's group that see x of 2^(s_rx - m_r) / l_r
//
// A weight is known only when its row's sum is, so the scores are made a second time: from the keys alone, half of the cache's bytes, with the rows'
// maxima and inverse sums that the attention before has left.  Scores kept in memory instead would take a limit on the context, and from a few
// rows on more bytes than the keys: 8 a row and position against 72 (4 bits, 128 entries) or 256.
//
// A warp has pages of its own, two at a time, from memory into the fragments of mma.sync m16n8k16 (16 positions as rows, the order of a product's terms is free: a lane
// takes a quarter of a key), and adds up in registers over all rows, in order; the CTA's warps share the rows' queries in shared memory, up to 256 at
// a time, and go through the pages of a (sequence, head) with them.  A position has one writer: no atomics.
#include <algorithm>

#include "pages_q4.cuh"
#include "pages_walk.cuh"

namespace ob {

namespace {

constexpr uint32_t MS_WARPS = 8, MS_COLS = 256;  // columns (rows of queries) in shared memory at a time
constexpr uint32_t MS_PAGES = 2;                 // pages of a warp at a time

// Q4: pages in 4 bits, and queries as f16 numbers with a power of two per row.
template <typename T, int HD, bool Q4>
__global__ void __launch_bounds__(MS_WARPS * 32, 2) pages_mass_kernel(const __grid_constant__ PagedAttnArgs a, float *mass, uint64_t mass_stride, uint32_t held) {
    using TQ = typename std::conditional<Q4, __half, T>::type;
    using F = Half2<TQ>;
    using B = Q4Block<HD>;
    constexpr int KW = HD / 32;  // 16-byte words of a lane's quarter of a row
    extern __shared__ __align__(16) uint4 s_q[];                            // [held / 8][KW][lane]
    float4 *s_row = reinterpret_cast<float4 *>(s_q + held / 8 * KW * 32);  // [held]: factor of the scores, maximum, inverse of the sum, token
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_release();
    pdl_wait();
    const uint32_t seq = blockIdx.z, head = blockIdx.y;
    const int32_t f0 = a.first[seq], f1 = a.first[seq + 1];
    if (f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens) return;
    const uint32_t room = a.pg.stride * KV_PAGE, n = min((uint32_t)(f1 - f0), a.max_drafts), ctx = min(a.n_ctx[seq], room), limit = (uint32_t)min((uint64_t)ctx + n, (uint64_t)room);
    const uint32_t n_pages = (limit + KV_PAGE - 1) / KV_PAGE, n_cols = n * a.group;
    const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;
    const float scale2 = a.scale * 1.4426950408889634f;

    auto keys = [&](uint32_t (&f)[HD / 16][4], uint32_t page) {  // positions g and g + 8 of a page as A fragments
        if constexpr (Q4) {
            const uint8_t *k = static_cast<const uint8_t *>(a.pg.k) + ((uint64_t)page * a.pg.n_kv + head) * B::BYTES;
            uint32_t w0[KW], w1[KW];
            const uint8_t *at = k + g * B::ROW + t * (HD / 8);
            if constexpr (HD == 128) {
                const uint4 x = *reinterpret_cast<const uint4 *>(at), y = *reinterpret_cast<const uint4 *>(at + 8 * B::ROW);
                w0[0] = x.x, w0[1] = x.y, w0[KW - 2] = x.z, w0[KW - 1] = x.w, w1[0] = y.x, w1[1] = y.y, w1[KW - 2] = y.z, w1[KW - 1] = y.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(at), y = *reinterpret_cast<const uint2 *>(at + 8 * B::ROW);
                w0[0] = x.x, w0[1] = x.y, w1[0] = y.x, w1[1] = y.y;
            }
            const uint16_t *unit = reinterpret_cast<const uint16_t *>(k + B::CODES) + g * B::GROUPS + t * (HD / 4) / Q4_GROUP;
            const uint32_t d0 = unit[0] * 0x10001u, d1 = unit[8 * B::GROUPS] * 0x10001u, n0 = q4_offset(d0), n1 = q4_offset(d1);
#pragma unroll
            for (int w = 0; w < KW; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f[2 * w + h][0] = q4_field(w0[w], 2 * h, d0, n0), f[2 * w + h][1] = q4_field(w1[w], 2 * h, d1, n1);
                    f[2 * w + h][2] = q4_field(w0[w], 2 * h + 1, d0, n0), f[2 * w + h][3] = q4_field(w1[w], 2 * h + 1, d1, n1);
                }
        } else {
            const uint4 *k = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.pg.k) + (((uint64_t)page * a.pg.n_kv + head) * KV_PAGE + g) * HD + t * (HD / 4));
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const uint4 x = __ldg(k + w), y = __ldg(k + w + HD);  // (eight rows on: 8 HD entries of two bytes)
                f[2 * w][0] = x.x, f[2 * w][1] = y.x, f[2 * w][2] = x.y, f[2 * w][3] = y.y;
                f[2 * w + 1][0] = x.z, f[2 * w + 1][1] = y.z, f[2 * w + 1][2] = x.w, f[2 * w + 1][3] = y.w;
            }
        }
    };
    const uint32_t step = gridDim.x * MS_WARPS * MS_PAGES, mine = warp * MS_PAGES;
    auto page_of = [&](uint32_t p) {
        const int32_t id = p < n_pages ? table[p] : -1;
        return (uint32_t)id < a.pg.n_pages ? id : -1;
    };
    uint32_t page0 = blockIdx.x * MS_WARPS * MS_PAGES;
    int32_t id[MS_PAGES], next[MS_PAGES];
#pragma unroll
    for (uint32_t i = 0; i < MS_PAGES; ++i) id[i] = page_of(page0 + mine + i);
    bool staged = false;
#pragma unroll 1
    for (; page0 < n_pages; page0 += step) {
#pragma unroll
        for (uint32_t i = 0; i < MS_PAGES; ++i) next[i] = page_of(page0 + step + mine + i);
        float acc[MS_PAGES][2];
#pragma unroll
        for (uint32_t i = 0; i < MS_PAGES; ++i) acc[i][0] = acc[i][1] = 0.0f;
        uint32_t f[MS_PAGES][HD / 16][4];  // the pages' keys (of pages that are not there: of page 0, for nothing)
#pragma unroll
        for (uint32_t i = 0; i < MS_PAGES; ++i) keys(f[i], max(id[i], 0));
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < n_cols; c0 += held) {
            const uint32_t cols = min(n_cols - c0, held), sets = (cols + 7) / 8;
            if (!staged || n_cols > held) {
            __syncthreads();
            // ---- queries: a warp a set of eight rows at a time, as B fragments
            for (uint32_t k = warp; k < sets; k += MS_WARPS) {
                const uint32_t r = c0 + k * 8 + g, tok = r / a.group;
                const bool live = r < n_cols;
                const uint64_t token = (uint64_t)(uint32_t)f0 + tok;
                const uint32_t h = head * a.group + r - tok * a.group;
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (live ? token * a.q_stride + (uint64_t)h * HD + t * (HD / 4) : 0u));
                uint32_t q[HD / 8];
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    const uint4 x = live ? src[i] : make_uint4(0, 0, 0, 0);
                    q[4 * i] = x.x, q[4 * i + 1] = x.y, q[4 * i + 2] = x.z, q[4 * i + 3] = x.w;
                }
                float factor = 1.0f;
                if constexpr (Q4 && !std::is_same<T, __half>::value) {
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) top = max(top, max(q[i] & 0x7fffu, q[i] >> 16 & 0x7fffu));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = top == 0 || top >= 0x7f80u ? 0 : max(-112, min(112, 14 - ((int)(top >> 7) - 127)));
                    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                    factor = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) {
                        const float2 x = Half2<T>::unpack(q[i]);
                        q[i] = F::pack(x.x * up, x.y * up);
                    }
                }
#pragma unroll
                for (int i = 0; i < KW; ++i) s_q[(k * KW + i) * 32 + lane] = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
                if (t == 0) {
                    const float2 st = live ? a.stats[token * a.group * a.pg.n_kv + h] : make_float2(0.0f, 0.0f);
                    // a row that sees nothing has a maximum of minus infinity and an inverse of zero
                    s_row[k * 8 + g] = make_float4(factor * scale2, st.x == -INFINITY ? 0.0f : st.x, st.y, __uint_as_float(live ? tok : 0xffffffffu));
                }
            }
            __syncthreads();
            staged = true;
            }
            const uint32_t pos0 = (page0 + mine) * KV_PAGE;
            const bool drafted = pos0 + MS_PAGES * KV_PAGE > ctx;
            float part[MS_PAGES][2];  // sums of some rows, then of those: errors grow with the square root of what one sum would have
#pragma unroll
            for (uint32_t i = 0; i < MS_PAGES; ++i) part[i][0] = part[i][1] = 0.0f;
#pragma unroll 1
            for (uint32_t k = 0; k < sets; ++k) {
                float s[MS_PAGES][4];
#pragma unroll
                for (uint32_t i = 0; i < MS_PAGES; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    const uint4 q = s_q[(k * KW + w) * 32 + lane];
#pragma unroll
                    for (uint32_t i = 0; i < MS_PAGES; ++i) {
                        F::mma(s[i], f[i][2 * w], q.x, q.y);
                        F::mma(s[i], f[i][2 * w + 1], q.z, q.w);
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float4 row = s_row[k * 8 + 2 * t + c];
                    const uint32_t tok = __float_as_uint(row.w);
                    const bool live = row.z != 0.0f;  // (a row that is none, or sees nothing)
                    uint64_t bits = 0;
                    if (drafted && live && a.visible) bits = a.visible[(uint32_t)f0 + tok];
#pragma unroll
                    for (uint32_t i = 0; i < MS_PAGES; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float w = pow2(fmaf(s[i][2 * h + c], row.x, -row.y)) * row.z;
                            bool see = live;
                            if (drafted) {
                                const uint32_t x = pos0 + i * KV_PAGE + g + 8 * h;
                                see = see && (x < ctx || (x < limit && (a.visible ? (bits >> ((x - ctx) & 63) & 1) != 0 : x - ctx <= tok)));
                            }
                            part[i][h] += see ? w : 0.0f;
                        }
                }
                if ((k & 7) == 7 || k + 1 == sets)
#pragma unroll
                    for (uint32_t i = 0; i < MS_PAGES; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) acc[i][h] += part[i][h], part[i][h] = 0.0f;
            }
        }
        float *at = mass + ((uint64_t)seq * a.pg.n_kv + head) * mass_stride;
#pragma unroll
        for (uint32_t i = 0; i < MS_PAGES; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v = acc[i][h];
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                const uint32_t x = (page0 + mine + i) * KV_PAGE + g + 8 * h;
                if (t == 0 && id[i] >= 0 && x < limit) at[x] = x < ctx ? at[x] + v : v;
            }
            id[i] = next[i];
        }
    }
}

template <typename T, int HD, bool Q4>
cudaError_t launch(const PagedAttnArgs &a, uint32_t n_seq, float *mass, uint64_t stride, int sm_count, cudaStream_t st) {
    auto kernel = pages_mass_kernel<T, HD, Q4>;
    constexpr size_t COLUMN = HD * 2 + sizeof(float4);
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MS_COLS * COLUMN); })) return e;
    const uint64_t pages = (std::min<uint64_t>(a.max_ctx, (uint64_t)a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE;  // about
    const uint64_t chunks = (pages + MS_WARPS * MS_PAGES - 1) / (MS_WARPS * MS_PAGES);
    // Four rounds of CTAs' places (two an SM) for lengths that differ; a CTA begins with three loads that depend on each other, and the queries.
    const uint64_t most = std::max<uint64_t>(1, 8ull * sm_count / ((uint64_t)n_seq * a.pg.n_kv));
    const uint32_t held = (uint32_t)std::min<uint64_t>(MS_COLS, ((uint64_t)a.max_drafts * a.group + 7) / 8 * 8);
    return launch_pdl(kernel, dim3((uint32_t)std::max<uint64_t>(1, std::min(chunks, most)), a.pg.n_kv, n_seq), dim3(MS_WARPS * 32), held * COLUMN, st, a, mass, stride, held);
}
template <typename T>
cudaError_t launch_dim(const PagedAttnArgs &a, bool q4, uint32_t n_seq, float *mass, uint64_t stride, int sm_count, cudaStream_t st) {
    if (a.pg.dim == 64) return q4 ? launch<T, 64, true>(a, n_seq, mass, stride, sm_count, st) : launch<T, 64, false>(a, n_seq, mass, stride, sm_count, st);
    return q4 ? launch<T, 128, true>(a, n_seq, mass, stride, sm_count, st) : launch<T, 128, false>(a, n_seq, mass, stride, sm_count, st);
}

}  // namespace

cudaError_t launch_pages_mass(const PagedAttnArgs &a, bool q_bf16, bool q4, uint32_t n_seq, float *mass, uint64_t mass_stride, int sm_count, cudaStream_t st) {
    return q_bf16 ? launch_dim<bf16>(a, q4, n_seq, mass, mass_stride, sm_count, st) : launch_dim<__half>(a, q4, n_seq, mass, mass_stride, sm_count, st);
}

}  // namespace ob
