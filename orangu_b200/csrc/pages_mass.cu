// The weights that every position gets, added up over the rows and query heads that see it (ob_pages_attention_tokens with masses).
//
//   mass[s][h][x] += sum over the tokens and heads r of h's group that see x of 2^(s_rx - m_r) / l_r
//
// A weight is known only when its row's sum is, so the scores are made a second time: from the keys alone, half of the cache's bytes, with the rows'
// maxima and inverse sums that the attention before has left.  Scores kept in memory instead would take a limit on the context, and from a few
// rows on more bytes than the keys: 8 a row and position against 72 (4 bits, 128 entries) or 256.
//
// The pages of all (sequence, key/value head) pieces are shared out evenly (pages_walk.cuh); a warp has two pages at a time, through a ring of its own, as the rows of
// mma.sync m16n8k16, and adds up in registers over the rows of queries, eight columns at a time, in order.  The CTA's warps share the queries in
// shared memory, up to 128 at a time; with more the pages are gone through again.  A position has one writer: no atomics.
//
// One row a sequence: the bytes of the keys (32 sequences of 1 to 4 k in bfloat16 pages, 8 heads of 128: about 24 us of the 97 that attention and this take).  Many rows: the
// tensor cores are busy 46 % of the time at 128 rows; pages_mass_tc5.cu is for those.
#include <algorithm>

#include "pages_q4.cuh"
#include "pages_walk.cuh"

namespace ob {

namespace {

constexpr uint32_t MS_COLS = 128;  // columns (rows of queries) in shared memory at a time
constexpr uint32_t MS_PAGES = 2;   // pages of a step

template <int HD, bool Q4>
struct MsShape {
    static constexpr uint32_t BLOCK = Q4 ? Q4Block<HD>::BYTES : KV_PAGE * HD * 2, STEP = MS_PAGES * BLOCK, DEPTH = Q4 ? 4 : 2 * 128 / HD, RINGS = PA_WARPS * DEPTH * STEP;
    static constexpr uint32_t COLUMN = HD * 2 + sizeof(float4);  // a query, and its factor, maximum, inverse of the sum and token
};

// Q4: pages in 4 bits, and queries as f16 numbers with a power of two per row.
template <typename T, int HD, bool Q4>
__global__ void __launch_bounds__(PA_THREADS, 3) pages_mass_kernel(const __grid_constant__ PagedAttnArgs a, float *mass, uint64_t mass_stride, uint32_t held) {
    using TQ = typename std::conditional<Q4, __half, T>::type;
    using F = Half2<TQ>;
    using B = Q4Block<HD>;
    using S = MsShape<HD, Q4>;
    constexpr uint32_t KW = HD / 32, DEPTH = S::DEPTH;  // KW: 16-byte words of a lane's quarter of a row
    extern __shared__ __align__(128) uint8_t smem[];
    uint4 *s_q = reinterpret_cast<uint4 *>(smem + S::RINGS);               // [held / 8][KW][lane]
    float4 *s_row = reinterpret_cast<float4 *>(s_q + held / 8 * KW * 32);  // [held]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_release();
    pdl_wait();
    const float scale2 = a.scale * 1.4426950408889634f;
    const uint32_t base = smem_addr(smem) + warp * DEPTH * S::STEP;
    PaWalk<true> wk;
    wk.start(a);
    for (; wk.more(); wk.next(a)) {
        const uint32_t head = wk.head, seq = wk.unit, row0 = wk.u.row0, n_cols = wk.u.rows * a.group, ctx = wk.u.ctx, limit = wk.u.limit;
        const uint32_t from = wk.page + warp * MS_PAGES, to = wk.last(), n_steps = to > from ? (to - from + PA_WARPS * MS_PAGES - 1) / (PA_WARPS * MS_PAGES) : 0u;
        const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;
        float *at = mass + ((uint64_t)seq * a.pg.n_kv + head) * mass_stride;
        const uint8_t *pool = static_cast<const uint8_t *>(a.pg.k) + (uint64_t)head * S::BLOCK;
        const uint64_t page_bytes = (uint64_t)a.pg.n_kv * S::BLOCK;
        auto page_of = [&](uint32_t i) { return from + i / MS_PAGES * (PA_WARPS * MS_PAGES) + i % MS_PAGES; };  // the warp's i-th page
        auto look = [&](uint32_t i) {
            const int32_t id = page_of(i) < to ? table[page_of(i)] : -1;
            return (uint32_t)id < a.pg.n_pages ? id : -1;
        };
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < n_cols; c0 += held) {
            const uint32_t cols = min(n_cols - c0, held), sets = (cols + 7) / 8;
            // ---- page numbers: lane i has those of the warp's page 32 j + i, and of the 32 after them
            int32_t id_now = look(lane), id_next = look(32 + lane);
            uint32_t block = 0;
            auto number = [&](uint32_t i) { return __shfl_sync(0xffffffffu, i / 32 != block ? id_next : id_now, i & 31); };
            auto request = [&](uint32_t step) {
                if (step < n_steps)
#pragma unroll
                    for (uint32_t k = 0; k < MS_PAGES; ++k) {
                        const int32_t id = number(step * MS_PAGES + k);
                        if (id < 0) continue;
                        const uint8_t *src = pool + (uint32_t)id * page_bytes;
                        const uint32_t dst = base + step % DEPTH * S::STEP + k * S::BLOCK;
#pragma unroll
                        for (uint32_t c = lane; c < S::BLOCK / 16; c += 32) {
                            const uint32_t row = c / (HD / 8);  // (16-bit pages: 16-byte words of a row exchanged, for ldmatrix)
                            cp16(dst + (Q4 ? c * 16 : row * HD * 2 + (((c % (HD / 8)) ^ (row & 7)) << 4)), src + c * 16, true);
                        }
                    }
                cp_commit();
            };
#pragma unroll 1
            for (uint32_t i = 0; i + 1 < DEPTH; ++i) request(i);
            __syncthreads();  // (of the columns before)
            // ---- rows: a row that sees nothing has a maximum of minus infinity and an inverse of zero; it counts as a row of zeros, as one that is none does
            for (uint32_t c = threadIdx.x; c < sets * 8; c += PA_THREADS) {
                const uint32_t r = c0 + c, tok = r / a.group;
                const float2 st = r < n_cols ? a.stats[((uint64_t)row0 + tok) * a.group * a.pg.n_kv + head * a.group + r - tok * a.group] : make_float2(0.0f, 0.0f);
                s_row[c] = make_float4(scale2, st.y != 0.0f ? -st.x : 0.0f, st.y, __uint_as_float(tok));
            }
            __syncthreads();
            // ---- queries: a warp a set of eight at a time, as B fragments; the order of a product's terms is that of the keys
#pragma unroll 2
            for (uint32_t k = warp; k < sets; k += PA_WARPS) {
                const uint32_t r = c0 + k * 8 + g, tok = r / a.group, h = head * a.group + r - tok * a.group;
                const bool counts = r < n_cols && s_row[k * 8 + g].z != 0.0f;
                const T *row = static_cast<const T *>(a.q) + (r < n_cols ? ((uint64_t)row0 + tok) * a.q_stride + (uint64_t)h * HD : 0u);
                uint32_t q[HD / 8];
                if constexpr (Q4) {
#pragma unroll
                    for (uint32_t i = 0; i < KW; ++i) {
                        const uint4 x = counts ? reinterpret_cast<const uint4 *>(row + t * (HD / 4))[i] : make_uint4(0, 0, 0, 0);
                        q[4 * i] = x.x, q[4 * i + 1] = x.y, q[4 * i + 2] = x.z, q[4 * i + 3] = x.w;
                    }
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < HD / 8; ++i) q[i] = counts ? reinterpret_cast<const uint32_t *>(row)[i * 4 + t] : 0u;
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
                for (uint32_t i = 0; i < KW; ++i) s_q[(k * KW + i) * 32 + lane] = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
                if (Q4 && !std::is_same<T, __half>::value && t == 0) s_row[k * 8 + g].x = factor * scale2;
            }
            __syncthreads();
#pragma unroll 1
            for (uint32_t step = 0; step < n_steps; ++step) {
                cp_wait<DEPTH - 2>();
                __syncwarp();
                if (step * MS_PAGES / 32 != block) {
                    block = step * MS_PAGES / 32;
                    id_now = id_next;
                    id_next = look(32 * (block + 1) + lane);
                }
                request(step + DEPTH - 1);
                const uint32_t page = page_of(step * MS_PAGES), pos0 = page * KV_PAGE, ks = base + step % DEPTH * S::STEP;
                bool there[MS_PAGES];
                float old[MS_PAGES][2];  // what is added to: lane (g, 0) has positions g and g + 8 of the pages
#pragma unroll
                for (uint32_t i = 0; i < MS_PAGES; ++i) {
                    there[i] = number(step * MS_PAGES + i) >= 0;
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        const uint32_t x = pos0 + i * KV_PAGE + g + 8 * h;
                        old[i][h] = t == 0 && there[i] && (c0 > 0 ? x < limit : x < ctx) ? at[x] : 0.0f;
                    }
                }
                uint32_t f[MS_PAGES][HD / 16][4];
#pragma unroll
                for (uint32_t i = 0; i < MS_PAGES; ++i) {
                    const uint32_t k = ks + i * S::BLOCK;
                    if constexpr (Q4) {
                        uint32_t w0[KW], w1[KW];
                        lds_words(w0, k + g * B::ROW + t * (HD / 8));
                        lds_words(w1, k + (g + 8) * B::ROW + t * (HD / 8));
                        const uint32_t unit = k + B::CODES + 2 * (g * B::GROUPS + t * (HD / 4) / Q4_GROUP);
                        const uint32_t d0 = lds16(unit) * 0x10001u, d1 = lds16(unit + 16 * B::GROUPS) * 0x10001u, n0 = q4_offset(d0), n1 = q4_offset(d1);
#pragma unroll
                        for (uint32_t w = 0; w < KW; ++w)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                f[i][2 * w + h][0] = q4_field(w0[w], 2 * h, d0, n0), f[i][2 * w + h][1] = q4_field(w1[w], 2 * h, d1, n1);
                                f[i][2 * w + h][2] = q4_field(w0[w], 2 * h + 1, d0, n0), f[i][2 * w + h][3] = q4_field(w1[w], 2 * h + 1, d1, n1);
                            }
                    } else {
                        const uint32_t row = lane & 15;
#pragma unroll
                        for (uint32_t w = 0; w < HD / 16; ++w) ldsm4(f[i][w], k + row * HD * 2 + (((2 * w + (lane >> 4)) ^ (row & 7)) << 4));
                    }
                }
                const bool drafted = pos0 + MS_PAGES * KV_PAGE > ctx;
                float acc[MS_PAGES][2], part[MS_PAGES][2];  // sums of 64 rows, then of those: errors grow with the square root of what one sum would have
#pragma unroll
                for (uint32_t i = 0; i < MS_PAGES; ++i) acc[i][0] = acc[i][1] = part[i][0] = part[i][1] = 0.0f;
                // N sets of eight columns from set k on: products of several sums under way at once
                auto add = [&](auto sets_at_once, auto masked, uint32_t k) {
                    constexpr uint32_t N = decltype(sets_at_once)::value;
                    float s[N][MS_PAGES][4];
#pragma unroll
                    for (uint32_t w = 0; w < KW; ++w)
#pragma unroll
                        for (uint32_t m = 0; m < N; ++m) {
                            const uint4 q = s_q[((k + m) * KW + w) * 32 + lane];
#pragma unroll
                            for (uint32_t i = 0; i < MS_PAGES; ++i) {
                                if (w == 0) mma_first<TQ>(s[m][i], f[i][0], q.x, q.y);
                                else F::mma(s[m][i], f[i][2 * w], q.x, q.y);
                                F::mma(s[m][i], f[i][2 * w + 1], q.z, q.w);
                            }
                        }
#pragma unroll
                    for (uint32_t m = 0; m < N; ++m)
#pragma unroll
                        for (uint32_t c = 0; c < 2; ++c) {
                            const float4 row = s_row[(k + m) * 8 + 2 * t + c];
                            uint64_t bits = 0;
                            const uint32_t tok = __float_as_uint(row.w);
                            if (decltype(masked)::value && a.visible && row.z != 0.0f) bits = a.visible[row0 + tok];
#pragma unroll
                            for (uint32_t i = 0; i < MS_PAGES; ++i)
#pragma unroll
                                for (uint32_t h = 0; h < 2; ++h) {
                                    const float e = pow2(fmaf(s[m][i][2 * h + c], row.x, row.y));
                                    if constexpr (decltype(masked)::value) {
                                        const uint32_t x = pos0 + i * KV_PAGE + g + 8 * h;
                                        if (row.z != 0.0f && (x < ctx || (x < limit && (a.visible ? (bits >> ((x - ctx) & 63) & 1) != 0 : x - ctx <= tok)))) part[i][h] = fmaf(e, row.z, part[i][h]);
                                    } else {
                                        if (row.z != 0.0f) part[i][h] = fmaf(e, row.z, part[i][h]);  // (a column of zeros: an infinite entry of a key would make it none)
                                    }
                                }
                        }
                };
                auto all = [&](auto masked) {
                    uint32_t k = 0;
                    using one = std::integral_constant<uint32_t, 1>;
                    using two = std::integral_constant<uint32_t, 2>;
#pragma unroll 1
                    for (; k + 1 < sets; k += 2) {
                        add(two(), masked, k);
                        if ((k & 7) == 6)
#pragma unroll
                            for (uint32_t i = 0; i < MS_PAGES; ++i)
#pragma unroll
                                for (uint32_t h = 0; h < 2; ++h) acc[i][h] += part[i][h], part[i][h] = 0.0f;
                    }
                    if (k < sets) add(one(), masked, k);
                };
                if (drafted) all(std::true_type());
                else all(std::false_type());
#pragma unroll
                for (uint32_t i = 0; i < MS_PAGES; ++i)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) acc[i][h] += part[i][h];
#pragma unroll
                for (uint32_t i = 0; i < MS_PAGES; ++i)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        float v = acc[i][h];
                        v += __shfl_xor_sync(0xffffffffu, v, 1);
                        v += __shfl_xor_sync(0xffffffffu, v, 2);
                        const uint32_t x = pos0 + i * KV_PAGE + g + 8 * h;
                        if (t == 0 && there[i] && x < limit) at[x] = old[i][h] + v;
                    }
            }
            cp_wait<0>();
        }
        __syncthreads();  // (the queries are written again)
    }
}

template <typename T, int HD, bool Q4>
cudaError_t launch(PagedAttnArgs a, uint32_t n_seq, float *mass, uint64_t stride, int sm_count, cudaStream_t st) {
    using S = MsShape<HD, Q4>;
    auto kernel = pages_mass_kernel<T, HD, Q4>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::RINGS + MS_COLS * S::COLUMN); })) return e;
    const uint64_t pages = (std::min<uint64_t>(a.max_ctx, (uint64_t)a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE;  // about, of a sequence
    const uint32_t held = (uint32_t)std::min<uint64_t>(MS_COLS, ((uint64_t)a.max_drafts * a.group + 7) / 8 * 8), bytes = S::RINGS + held * S::COLUMN;
    const uint64_t most = (uint64_t)sm_count * std::min<uint32_t>(3, 227 * 1024 / (bytes + 1024));
    a.block = a.max_drafts, a.blocks = 1, a.n_units = n_seq;  // whole sequences
    a.apart = 0;
    const uint64_t grid = std::min(most, std::max<uint64_t>(1, n_seq * ((pages + PA_LEAST - 1) / PA_LEAST) * a.pg.n_kv));
    return launch_pdl(kernel, dim3((uint32_t)grid), dim3(PA_THREADS), bytes, st, a, mass, stride, held);
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
