// The weights that every position gets, added up over many rows (pages_mass.cu has the mathematics and the form for few): scores on the fifth-generation
// tensor cores with the positions as the 128 rows of a product, so that a thread has a position and adds up over its columns (rows of queries) by itself.
//
//   warps 0-7  bring tiles of keys and queries into shared memory (two of 64 KB wait while one is worked on), turn scores into weights and add them up: a
//              thread has a position and half of the 128 columns
//   warp 8     issues the products: scores (tensor memory, two places) = keys x queries
//
// One operand stays and the other streams: with up to 128 columns the queries of a (sequence, head) stay and its keys go by; with more the keys of 128
// positions stay and the queries go by.  The pages of all pieces are shared out evenly (pages_walk.cuh), a tile is eight of them.  A position has one
// writer, columns are added up in order: no atomics.  Its floor is the special function unit's, 16 powers of two a clock: 500 tokens of 4 heads a head at 12,000, 8 heads of 128, 46 us.
// It takes 200 us (the mma.sync form 627; 236 with a least share of the square root of a piece's pages, as attention has it, for which there were too few CTAs): a warp's step of 128 positions and 64 columns is some 1100 instructions, of which weights are a third, and issues half of the
// time; tiles of queries come anew for every 128 positions (bfloat16 ones over 4-bit pages are made f16 each time: 366 us).  All waits are bounded; after one that was given up
// every warp still goes through its loop, so that none is missed at a barrier.
#include <algorithm>

#include "pages_q4.cuh"
#include "pages_walk.cuh"
#include "tc5_common.cuh"

namespace ob {

namespace {

constexpr uint32_t MT_ROWS = 128, MT_PAGES = MT_ROWS / KV_PAGE, MT_BLOCK = MT_ROWS * 128;  // a tile's positions, and columns; blocks of 64 entries
constexpr int MT_SOFT = 256, MT_MMA_WARP = 8, MT_THREADS = 9 * 32, MT_CTAS = 2;
constexpr uint32_t MT_TMEM = 256;
// mbarriers and small arrays, byte offsets behind the operand tiles
constexpr uint32_t MB_FULL = 0, MB_DONE = 16, MB_EMPTY = 32, MB_SLOT = 48, MB_ABORT = 52, MB_ROWS = 64, MB_XCHG = MB_ROWS + 4 * MT_ROWS * 16, MB_BYTES = MB_XCHG + 2 * MT_ROWS * 4;
template <int HD> struct MtPlan {
    static constexpr uint32_t TILE = HD / 64 * MT_BLOCK, BAR = 3 * TILE, BYTES = BAR + MB_BYTES;  // what stays, and two that stream
    static_assert(MT_CTAS * (BYTES + 1024) <= 228 * 1024, "shared memory");
};

// c / group for c below 2^24 and groups up to 16; magic = 2^32 / group, rounded up (0: one).
__device__ __forceinline__ uint32_t token_of(uint32_t c, uint32_t magic) { return magic ? __umulhi(c, magic) : c; }
__device__ __forceinline__ void mt_sync() { asm volatile("bar.sync 1, %0;" ::"n"(MT_SOFT) : "memory"); }

// One tile on its way into shared memory: `issue` asks for it, `finish` writes what came by way of registers.  256 threads, 16 bytes of the tile each and turn.
template <int HD> struct MtTurns {
    static constexpr uint32_t WORDS = HD / 8, TURNS = MT_ROWS * WORDS / MT_SOFT;  // 16-byte words of a row
    static __device__ __forceinline__ uint32_t row(uint32_t i) { return (i * MT_SOFT + threadIdx.x) / WORDS; }
    static __device__ __forceinline__ uint32_t word() { return threadIdx.x % WORDS; }
    static __device__ __forceinline__ uint32_t place(uint32_t i) {  // in the swizzled tile
        const uint32_t r = row(i), c = word();
        return c / 8 * MT_BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    }
};
// Keys of pages page0 ..; pages from `end` on, or that are not there, are zero.
template <typename T, int HD, bool Q4> struct MtKeys : MtTurns<HD> {
    using M = MtTurns<HD>;
    using B = Q4Block<HD>;
    uint32_t code[Q4 ? M::TURNS : 1], unit[Q4 ? M::TURNS : 1];
    __device__ __forceinline__ void issue(const PagedAttnArgs &a, const int32_t *table, uint32_t head, uint32_t page0, uint32_t end, uint32_t tile) {
#pragma unroll
        for (uint32_t i = 0; i < M::TURNS; ++i) {
            const uint32_t r = M::row(i), page = page0 + r / KV_PAGE;
            const int32_t id = page < end ? table[page] : -1;
            const bool there = (uint32_t)id < a.pg.n_pages;
            const uint64_t at = (uint64_t)(there ? (uint32_t)id : 0u) * a.pg.n_kv + head;
            if constexpr (Q4) {
                const uint8_t *block = static_cast<const uint8_t *>(a.pg.k) + at * B::BYTES;
                code[i] = __ldg(reinterpret_cast<const uint32_t *>(block + B::key(r % KV_PAGE, M::word())));
                unit[i] = there ? __ldg(reinterpret_cast<const uint16_t *>(block + B::unit(false, r % KV_PAGE, M::word() / 4))) : 0u;
            } else {
                cp16(tile + M::place(i), static_cast<const T *>(a.pg.k) + (at * KV_PAGE + r % KV_PAGE) * HD + M::word() * 8, there);
            }
        }
    }
    __device__ __forceinline__ void finish(uint8_t *tile) {
        if constexpr (Q4) {
#pragma unroll
            for (uint32_t i = 0; i < M::TURNS; ++i) {
                const uint32_t d = unit[i] * 0x10001u, n = q4_offset(d);
                *reinterpret_cast<uint4 *>(tile + M::place(i)) = make_uint4(q4_field(code[i], 0, d, n), q4_field(code[i], 1, d, n), q4_field(code[i], 2, d, n), q4_field(code[i], 3, d, n));
            }
        }
    }
};
// Columns c0 .. of the piece's n_cols as rows of a tile, and what is known of each, two neighbours together where both are read at once: minus its maximum, the
// inverse of its sum, its token (-1: none, or it sees nothing: no weights, whatever its scores), and its factor where they are not all the same.
struct MtRows {
    float pair[MT_ROWS / 2][4];  // maximum, maximum, inverse, inverse
    int32_t token[MT_ROWS];
    float factor[MT_ROWS];
};
__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
template <typename T, int HD, bool Q4> struct MtQueries : MtTurns<HD> {
    using M = MtTurns<HD>;
    static constexpr bool FACTORS = Q4 && !std::is_same<T, __half>::value;  // bfloat16 queries become f16 ones (pages_q4.cu)
    uint4 word[FACTORS ? M::TURNS : 1];
    float2 stat;
    __device__ __forceinline__ void issue(const PagedAttnArgs &a, uint32_t row0, uint32_t head, uint32_t n_cols, uint32_t c0, uint32_t magic, uint32_t tile) {
        const T *base = static_cast<const T *>(a.q) + (uint64_t)row0 * a.q_stride + (uint64_t)head * a.group * HD + M::word() * 8;
#pragma unroll
        for (uint32_t i = 0; i < M::TURNS; ++i) {
            const uint32_t c = c0 + M::row(i), tok = token_of(c, magic);
            const bool live = c < n_cols;
            const T *src = live ? base + tok * a.q_stride + (c - tok * a.group) * HD : base;
            if constexpr (FACTORS) word[i] = live ? *reinterpret_cast<const uint4 *>(src) : make_uint4(0, 0, 0, 0);
            else cp16(tile + M::place(i), src, live);
        }
        const uint32_t c = c0 + threadIdx.x, tok = token_of(c, magic);
        stat = make_float2(0.0f, 0.0f);
        if (threadIdx.x < MT_ROWS && c < n_cols) stat = a.stats[((uint64_t)row0 + tok) * a.group * a.pg.n_kv + head * a.group + c - tok * a.group];
    }
    __device__ __forceinline__ void finish(uint32_t c0, uint32_t magic, float scale2, uint8_t *tile, MtRows &rows) {
        if constexpr (FACTORS) {
#pragma unroll
            for (uint32_t i = 0; i < M::TURNS; ++i) {
                uint32_t u[4] = {word[i].x, word[i].y, word[i].z, word[i].w}, top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7fffu, u[e] >> 16 & 0x7fffu));
#pragma unroll
                for (uint32_t o = 1; o < M::WORDS; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                const int e = top == 0 || top >= 0x7f80u ? 0 : max(-112, min(112, 14 - ((int)(top >> 7) - 127)));
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float2 f = Half2<T>::unpack(u[x]);
                    u[x] = Half2<__half>::pack(f.x * up, f.y * up);
                }
                *reinterpret_cast<uint4 *>(tile + M::place(i)) = make_uint4(u[0], u[1], u[2], u[3]);
                if (M::word() == 0) rows.factor[M::row(i)] = __uint_as_float((uint32_t)(127 - e) << 23) * scale2;
            }
        }
        if (threadIdx.x < MT_ROWS) {
            float *pair = rows.pair[threadIdx.x / 2] + threadIdx.x % 2;
            pair[0] = stat.y != 0.0f ? -stat.x : 0.0f, pair[2] = stat.y;
            rows.token[threadIdx.x] = stat.y != 0.0f ? (int32_t)token_of(c0 + threadIdx.x, magic) : -1;
        }
    }
};

template <typename T, int HD, bool Q4>
__global__ void __launch_bounds__(MT_THREADS, MT_CTAS) pages_mass_tc5_kernel(const __grid_constant__ PagedAttnArgs a, float *mass, uint64_t mass_stride) {
    using P = MtPlan<HD>;
    using TP = typename std::conditional<Q4, __half, T>::type;  // of the operands
    constexpr uint32_t TILE = P::TILE;
    constexpr bool FACTORS = MtQueries<T, HD, Q4>::FACTORS;
    static_assert(sizeof(MtRows) == 16 * MT_ROWS, "as many bytes as are set apart");
    extern __shared__ __align__(1024) uint8_t smem[];  // (no other shared memory: the operand tiles' swizzle counts on the alignment)
    const uint32_t sbase = smem_u32(smem), bar = sbase + P::BAR, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile uint32_t *abort = reinterpret_cast<volatile uint32_t *>(smem + P::BAR + MB_ABORT);
    if (threadIdx.x == 0) {
        for (uint32_t b = 0; b < 2; ++b) {
            mbar_init(bar + MB_FULL + 8 * b, 8);
            mbar_init(bar + MB_DONE + 8 * b, 1);
            mbar_init(bar + MB_EMPTY + 8 * b, 8);
        }
        *abort = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MT_MMA_WARP) tmem_alloc(bar + MB_SLOT, MT_TMEM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_release();  // (only now: a CTA of the next kernel must not take the tensor memory first, it would keep it until this grid is done)
    pdl_wait();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + P::BAR + MB_SLOT);
    PaWalk<true, MT_PAGES> wk;
    wk.start(a);
    uint32_t n = 0;  // products so far: number n has place n % 2 of what streams, and of the scores
    if (warp == MT_MMA_WARP) {
        constexpr uint32_t F16 = std::is_same<TP, __half>::value ? (1u << 7) | (1u << 10) : 0u;  // the operands' format bits: zero for f16
        const uint32_t idesc = umma_idesc_bf16(MT_ROWS) & ~F16;
        const uint64_t stays = umma_desc_sw128(sbase), streams[2] = {umma_desc_sw128(sbase + TILE), umma_desc_sw128(sbase + 2 * TILE)};
        for (; wk.more(); wk.next(a)) {
            const uint32_t cols = wk.u.rows * a.group, tiles = (wk.last() - wk.page + MT_PAGES - 1) / MT_PAGES, sets = (cols + MT_ROWS - 1) / MT_ROWS;
            const bool keys_stream = sets == 1;
#pragma unroll 1
            for (uint32_t i = 0; i < tiles * sets; ++i, ++n) {
                const uint32_t b = n & 1;
                mbar_wait_warp(bar + MB_FULL + 8 * b, n >> 1 & 1u, abort);
                mbar_wait_warp(bar + MB_EMPTY + 8 * b, (n >> 1 & 1u) ^ 1u, abort);
                tc_fence_after();
                const uint64_t s = streams[b], keys = keys_stream ? s : stays, queries = keys_stream ? stays : s;
#pragma unroll
                for (uint32_t k = 0; k < HD / 16; ++k)
                    umma_bf16_warp(tmem + b * MT_ROWS, keys + (k / 4) * (MT_BLOCK >> 4) + 2 * (k % 4), queries + (k / 4) * (MT_BLOCK >> 4) + 2 * (k % 4), idesc, k ? 1u : 0u);
                umma_commit_warp(bar + MB_DONE + 8 * b);
            }
        }
    } else {
        const uint32_t r = warp % 4 * 32 + lane, half = warp / 4;  // this thread's position of a tile, and columns
        const uint32_t from = tmem + ((warp % 4 * 32) << 16) + half * 64;
        const float scale2 = a.scale * 1.4426950408889634f;
        const uint32_t magic = a.group > 1 ? 0xffffffffu / a.group + 1 : 0u;
        MtRows *rows = reinterpret_cast<MtRows *>(smem + P::BAR + MB_ROWS);  // of product n at n % 4 (with keys that stream: of the piece at 0)
        volatile float *xchg = reinterpret_cast<volatile float *>(smem + P::BAR + MB_XCHG);
        float *pending = nullptr;  // where the sum of the tile before goes: the other half's part is known only after the next barrier
        float pending_old = 0.0f, pending_sum = 0.0f;
        uint32_t turn = 0;
        auto settle = [&]() {  // behind a barrier
            if (pending) *pending = pending_old + (pending_sum + xchg[(turn ^ 1) * MT_ROWS + r]);
            pending = nullptr;
        };
        auto fence = []() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); };
        auto arrive = [&](uint32_t b) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar + MB_FULL + 8 * b);
        };
        for (; wk.more(); wk.next(a)) {
            const uint32_t head = wk.head, seq = wk.unit, row0 = wk.u.row0, n_cols = wk.u.rows * a.group, ctx = wk.u.ctx, limit = wk.u.limit, last = wk.last();
            const uint32_t tiles = (last - wk.page + MT_PAGES - 1) / MT_PAGES, sets = (n_cols + MT_ROWS - 1) / MT_ROWS;
            const bool keys_stream = sets == 1;
            const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;
            float *out = mass + ((uint64_t)seq * a.pg.n_kv + head) * mass_stride;
            MtKeys<T, HD, Q4> keys;
            MtQueries<T, HD, Q4> queries;
            const uint32_t groups = keys_stream ? 1u : tiles, length = keys_stream ? tiles : sets;  // times that something stays, and what goes by meanwhile
#pragma unroll 1
            for (uint32_t group = 0; group < groups; ++group) {
                // What streams: number i into the place of product n0 + i.
                const uint32_t n0 = n;
                auto place = [&](uint32_t i) { return TILE + (n0 + i & 1) * TILE; };
                auto issue = [&](uint32_t i) {
                    if (keys_stream) keys.issue(a, table, head, wk.page + i * MT_PAGES, last, sbase + place(i));
                    else queries.issue(a, row0, head, n_cols, i * MT_ROWS, magic, sbase + place(i));
                };
                auto finish = [&](uint32_t i) {
                    if (keys_stream) keys.finish(smem + place(i));
                    else queries.finish(i * MT_ROWS, magic, scale2, smem + place(i), rows[n0 + i & 3]);
                };
                mt_sync();  // (all have read the rows of the piece before, and its products are done)
                settle();
                if (keys_stream) {
                    queries.issue(a, row0, head, n_cols, 0, magic, sbase);
                    queries.finish(0, magic, scale2, smem, rows[0]);
                } else {
                    keys.issue(a, table, head, wk.page + group * MT_PAGES, last, sbase);
                    keys.finish(smem);
                }
#pragma unroll 1
                for (uint32_t i = 0; i < min(length, 2u); ++i) {
                    issue(i);
                    finish(i);
                    cp_commit();
                    cp_wait<0>();
                    fence();
                    arrive(n0 + i & 1);
                }
                float sum = 0.0f;
#pragma unroll 1
                for (uint32_t i = 0; i < length; ++i, ++n) {
                    const uint32_t b = n & 1, x = (wk.page + (keys_stream ? i : group) * MT_PAGES) * KV_PAGE + r;
                    const bool first = keys_stream || i == 0, ends = keys_stream || i + 1 == length;
                    mbar_wait_warp(bar + MB_DONE + 8 * b, n >> 1 & 1u, abort);
                    mt_sync();  // (the columns' rows that others have written, and their parts of the sums)
                    tc_fence_after();
                    settle();
                    if (i + 2 < length) issue(i + 2);
                    cp_commit();
                    if (first) sum = 0.0f;
                    const MtRows &col = rows[keys_stream ? 0u : n & 3];
                    float part = 0.0f;
                    // Without bits a position is seen by the tokens from `least` on.
                    const int32_t least = x < ctx ? 0 : x < limit ? (int32_t)(x - ctx) : 0x7fffffff;
                    const bool inside = x - r + MT_ROWS <= ctx, bits = a.visible && !inside;  // (alike for all threads)
                    const bool plain = inside && __all_sync(0xffffffffu, min(col.token[half * 64 + lane], col.token[half * 64 + 32 + lane]) >= 0);  // every column sees every position
#pragma unroll 1
                    for (uint32_t c = 0; c < 64; c += 16) {
                        const uint32_t c0 = half * 64 + c;
                        uint32_t u[16];
                        tmem_ld16(from + b * MT_ROWS + c, u);
                        tmem_ld_wait();
                        float p[2] = {0.0f, 0.0f};
                        if (!bits) {
#pragma unroll
                            for (uint32_t e = 0; e < 16; e += 2) {
                                const float4 w = *reinterpret_cast<const float4 *>(col.pair[(c0 + e) / 2]);
                                float2 k = make_float2(scale2, scale2);
                                if constexpr (FACTORS) k = *reinterpret_cast<const float2 *>(col.factor + c0 + e);
                                float f0, f1;
                                fma2(f0, f1, __uint_as_float(u[e]), __uint_as_float(u[e + 1]), k.x, k.y, w.x, w.y);
                                f0 = pow2(f0), f1 = pow2(f1);
                                if (plain) {
                                    fma2(p[0], p[1], f0, f1, w.z, w.w, p[0], p[1]);
                                } else {
                                    const int2 tok = *reinterpret_cast<const int2 *>(col.token + c0 + e);
                                    if (tok.x >= least) p[0] = fmaf(f0, w.z, p[0]);
                                    if (tok.y >= least) p[1] = fmaf(f1, w.w, p[1]);
                                }
                            }
                        } else {
#pragma unroll 1
                            for (uint32_t e = 0; e < 16; ++e) {
                                const float *w = col.pair[(c0 + e) / 2] + e % 2;
                                const int32_t tok = col.token[c0 + e];
                                bool see = x < ctx && tok >= 0;
                                if (x >= ctx && x < limit && tok >= 0) see = a.visible[row0 + tok] >> ((x - ctx) & 63) & 1;
                                float s = __uint_as_float(u[0]);
#pragma unroll
                                for (uint32_t k = 1; k < 16; ++k) s = e == k ? __uint_as_float(u[k]) : s;
                                if (see) p[0] = fmaf(pow2(fmaf(s, FACTORS ? col.factor[c0 + e] : scale2, w[0])), w[2], p[0]);
                            }
                        }
                        part += p[0] + p[1];
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar + MB_EMPTY + 8 * b);
                    sum += part;
                    if (ends) {
                        if (half) {
                            xchg[turn * MT_ROWS + r] = sum;
                        } else {
                            const uint32_t page = x / KV_PAGE;
                            if (page < last && x < limit && (uint32_t)table[page] < a.pg.n_pages) {
                                pending = out + x, pending_sum = sum;
                                pending_old = x < ctx ? out[x] : 0.0f;
                            }
                        }
                        turn ^= 1;
                    }
                    if (i + 2 < length) {
                        finish(i + 2);
                        cp_wait<0>();
                        fence();
                        arrive(b);
                    }
                }
            }
        }
        mt_sync();
        settle();
    }
    __syncwarp();
    if (*abort && lane == 0) {
        *reinterpret_cast<volatile uint32_t *>(a.status) = 1u;
        __threadfence_system();
    }
    if (*abort)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // (products that are still under way end before the memory goes away)
    cp_wait<0>();
    tc_fence_before();
    __syncthreads();
    if (warp == MT_MMA_WARP) tmem_dealloc(tmem, MT_TMEM);
}

template <typename T, int HD, bool Q4>
cudaError_t launch(PagedAttnArgs a, uint32_t n_seq, float *mass, uint64_t stride, int sm_count, cudaStream_t st) {
    using P = MtPlan<HD>;
    auto kernel = pages_mass_tc5_kernel<T, HD, Q4>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::BYTES); })) return e;
    const uint64_t pages = (std::min<uint64_t>(a.max_ctx, (uint64_t)a.pg.stride * KV_PAGE) + a.max_drafts + KV_PAGE - 1) / KV_PAGE;  // about, of a sequence
    a.block = a.max_drafts, a.blocks = 1, a.n_units = n_seq;  // whole sequences
    a.apart = 0;
    const uint64_t grid = std::min<uint64_t>((uint64_t)sm_count * MT_CTAS, std::max<uint64_t>(1, n_seq * ((pages + MT_PAGES - 1) / MT_PAGES) * a.pg.n_kv));
    return launch_pdl(kernel, dim3((uint32_t)grid), dim3(MT_THREADS), P::BYTES, st, a, mass, stride);
}
template <typename T>
cudaError_t launch_dim(const PagedAttnArgs &a, bool q4, uint32_t n_seq, float *mass, uint64_t stride, int sm_count, cudaStream_t st) {
    if (a.pg.dim == 64) return q4 ? launch<T, 64, true>(a, n_seq, mass, stride, sm_count, st) : launch<T, 64, false>(a, n_seq, mass, stride, sm_count, st);
    return q4 ? launch<T, 128, true>(a, n_seq, mass, stride, sm_count, st) : launch<T, 128, false>(a, n_seq, mass, stride, sm_count, st);
}

}  // namespace

cudaError_t launch_pages_mass_tc5(const PagedAttnArgs &a, bool q_bf16, bool q4, uint32_t n_seq, float *mass, uint64_t mass_stride, int sm_count, cudaStream_t st) {
    return q_bf16 ? launch_dim<bf16>(a, q4, n_seq, mass, mass_stride, sm_count, st) : launch_dim<__half>(a, q4, n_seq, mass, mass_stride, sm_count, st);
}

}  // namespace ob
