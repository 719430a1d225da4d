// Attention of drafted tokens on the fifth-generation tensor cores: the form of ob_pages_attention_tree for more rows (drafted token, query
// head) a key/value head than the mma.sync kernel of pages_attention.cu keeps up with.  The mathematics is the same.
//
// The tiles of 64 positions of all (rows, sequence, key/value head) pieces are laid end to end and shared out evenly: every SM has one CTA with
// the same number of tiles, whatever the lengths of the contexts, and walks through the pieces that lie in its part.  A piece that
// is cut leaves (maximum, sum, output) in fp32, and a second kernel, launched along, adds them up over all SMs (the last of a piece's
// CTAs to arrive doing it alone took as long as all the rest: 181 us for 8 x 64 tokens of 4 heads a key/value head at 8192).
//
//   warps 0-7  softmax: four warps per stream, a thread per row.  Scores come from tensor memory, weights go back into the same
//              columns, as value and remainder of the cache's type: one of 8 or 11 bits alone would be the largest error of the result.
//   warps 8, 9 issue the products of a stream each: scores = queries (shared memory) x keys, output += weights (tensor memory) x values
//   warps 10, 11 issue the TMA loads of keys and of values, pages of 16 rows x 64 columns each, straight from the cache into the swizzled operand
//              tiles, each into a ring of its own
//
// There are two streams of scores.  Up to 128 rows (WIDE false) they are the even and the odd tiles of the same rows, with an output each;
// above that they are two tiles of 128 rows that share keys and values.  A stream has two places for scores: while one's weights
// are made, the other's are multiplied and its next scores come.  Tiles of 128 positions with one place a stream, 16 softmax warps and one that
// issued all products took 25.6 us for one sequence of 512 positions and 48 rows a key/value head, 52 us for eight of 4096 and 64, and this form 17.4
// and 43 to 46 (then without remainders of f16 weights, now 18.4 and 47); with keys and values through one ring, in order, 32 sequences of 8192 with 128
// rows took 230 us over bfloat16 pages, with a ring each 216 (keys are wanted two steps before their values: of one order only the values were ahead).
//
// What bounds it (head dimension 128): up to 128 rows the bytes, 217 to 240 us for 32 sequences of 8192 with 128 rows (floor 167, 4.6 to 5 TB/s).  Above,
// the chain of a step (scores, weights and their remainders, two products): the tensor cores work 54 % of the time and the special function unit 36 %; 727 us
// for 32 sequences of 8192 with 512 rows in a call of its own, 855 in a loop, where the clocks fall under the power limit (floor 335).  A part of the powers of
// two on the fused multiply-adds, 1/8 to 1/2 of them, took from 2 % less to 6 % more.
//
// Over 4-bit pages (Q4) warps make the f16 operand tiles out of codes, where TMA brings them otherwise.  Four warps
// do it, two for keys and two for values.  8 x 16 tokens of 4 heads at 8192: 67 us (f16 pages 61); with three quarters of any one part left out, making of tiles, softmax, products or
// copies, 56 to 66: no one of them bounds it, and 17 are the same at 512 positions.  1000 tokens of 8 heads at 8000: 405 us, 685 TFLOP/s of scores and values
// (1030 with the products of the remainders).
//
// Context positions are seen by every row: only tiles that reach past the context, or have a page that is not there, are masked, a 64-bit word
// per thread.  There, values of positions that nobody has, or that are no numbers, are set to zero in shared memory (0 times them
// would reach rows that do not see them); what rows do see of the latter is added at the end.  All waits are bounded.
#include <algorithm>
#include <cstring>

#include "mixers_common.cuh"
#include "pages.h"
#include "pages_q4.cuh"
#include "tc5_common.cuh"

namespace ob {

namespace {

constexpr uint32_t PG_ROWS = 128, PG_KEYS = PG_PAGES * KV_PAGE, PG_BLOCK = PG_KEYS * 128, PG_QBLOCK = PG_ROWS * 128;  // a tile's positions; blocks of 64 columns
constexpr int PG_SOFT = 256, PG_MMA_WARP = 8, PG_TMA_WARP = 10, PG_THREADS = 12 * 32;
constexpr int P4_TURNS = 2, P4_CODE_WARPS = 2 * P4_TURNS, P4_AHEAD = 2, P4_THREADS = 16 * 32;  // over 4-bit pages: warps for keys and for values; their tiles under way; whole warpgroups
constexpr uint32_t PG_TMEM_S = 0, PG_TMEM_O = 256, PG_TMEM_COLS = 512;
constexpr uint32_t PG_LEAST = 4;        // units of a CTA

// mbarriers and small arrays, byte offsets
constexpr uint32_t PG_STAGES = 12;      // at most
constexpr uint32_t PB_K_FULL = 0, PB_K_EMPTY = PB_K_FULL + 8 * PG_STAGES, PB_V_FULL = PB_K_EMPTY + 8 * PG_STAGES, PB_V_EMPTY = PB_V_FULL + 8 * PG_STAGES, PB_S_FULL = PB_V_EMPTY + 8 * PG_STAGES /* [stream][place] */,
                   PB_P_FULL = PB_S_FULL + 32, PB_PV_DONE = PB_P_FULL + 32, PB_O_FULL = PB_PV_DONE + 16, PB_Q_FULL = PB_O_FULL + 16, PB_SLOT = PB_Q_FULL + 8, PB_ABORT = PB_SLOT + 4, PB_ODD = PB_ABORT + 4,
                   PB_TOP = PB_ODD + 8, PB_BYTES = PB_TOP + 4 * PG_ROWS * 4;
template <int HD, bool WIDE, bool Q4 = false>
struct PgPlan {
    static constexpr uint32_t NB = HD / 64, OPERAND = NB * PG_BLOCK, ROWS = NB * PG_QBLOCK, Q = (WIDE ? 2 : 1) * ROWS;  // (16 KB at least: outputs leave by way of it)
    // Places of the two rings.  Values are wanted two steps after their keys: they get more.  Where the streams take every other tile, the numbers are
    // even, so that a place is always the same stream's within a piece: waits go by the parity of a phase, and a stream that runs ahead must not ask
    // for a place's next tile before the one before, the other stream's, has arrived.
    // Where both streams take all tiles, two share a place: half the waits (32 sequences of 8192 with 512 rows, bf16: 720 us, and 773 with a place a tile).
    static constexpr uint32_t P4_CODES = Q4 ? P4_CODE_WARPS * P4_AHEAD * PG_PAGES * Q4Block<HD>::BYTES : 0;  // codes on their way
    static constexpr uint32_t G = WIDE && !Q4 ? 2 : 1, PLACE = G * OPERAND, FIT = (227 * 1024 - PB_BYTES - Q - P4_CODES) / PLACE, EVEN = WIDE ? 1 : 2;
    // Over 4-bit pages a place is always made by the same warp (waits go by parity here, too: a warp that went on to places that others had made
    // before could take an earlier phase for the one it waits for): multiples of P4_TURNS.
    static constexpr uint32_t KST = Q4 ? (FIT >= 20 ? 8 : FIT >= 8 ? 4 : 2) : std::min(FIT / 3 / EVEN * EVEN + WIDE, PG_STAGES);
    static constexpr uint32_t VST = Q4 ? (FIT >= 20 ? 12 : 4) : std::min((FIT - KST) / EVEN * EVEN, PG_STAGES);
    static constexpr uint32_t K = Q, V = K + KST * PLACE, CODES = V + VST * PLACE, BAR = CODES + P4_CODES, BYTES = BAR + PB_BYTES;
    static constexpr uint32_t MR = WIDE ? 2 * PG_ROWS : PG_ROWS;
    static constexpr uint64_t PART = (uint64_t)MR * (HD + 2);  // floats of a partial result
    static_assert(KST >= 2 && VST >= 3 && KST + VST <= FIT && PG_STAGES % 2 == 0 && (WIDE || (KST % 2 == 0 && VST % 2 == 0)) && BYTES <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b, float c) {
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float &d0, float &d1, float a0, float a1) {
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(PG_SOFT) : "memory"); }

template <typename T> __device__ __forceinline__ uint32_t pack16(float a, float b);
template <> __device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack16<bf16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack16(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
__device__ __forceinline__ float2 unpack16(uint32_t u, bf16) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ float from16(__half v) { return __half2float(v); }
__device__ __forceinline__ float from16(bf16 v) { return __bfloat162float(v); }
template <typename T> constexpr uint32_t EXPONENT16 = 0x7c00u;
template <> constexpr uint32_t EXPONENT16<bf16> = 0x7f80u;

// The end of a warp that gave up a wait, or found that another had: the word that the host reads (ob_pages_synchronize), and time for copies that
// are still in flight to land before the shared memory goes away.
__device__ __forceinline__ void gave_up(uint32_t *status) {
    if ((threadIdx.x & 31) == 0) {
        *reinterpret_cast<volatile uint32_t *>(status) = 1u;
        __threadfence_system();
    }
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
}

// A sequence as the walk sees it.
struct PgSeq {
    uint32_t row0, drafts, ctx, limit, n_pages, n_tiles, n_rt;  // n_rt: tiles of rows
};
template <uint32_t MR>
__device__ __forceinline__ PgSeq pg_seq(const PagedAttnArgs &a, uint32_t unit) {
    PgSeq q{};
    const uint32_t s = a.blocks > 1 ? unit / a.blocks : unit, skip = (unit - s * a.blocks) * a.block;  // (more than one block: all that is before it is context)
    const int32_t f0 = a.first[s], f1 = a.first[s + 1];
    const uint32_t ctx = a.n_ctx[s], room = a.pg.stride * KV_PAGE;  // (all loads before the first decision)
    if (f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens) return q;
    const uint32_t n = min((uint32_t)(f1 - f0), a.max_drafts);
    if (skip >= n) return q;
    q.row0 = (uint32_t)f0 + skip;
    q.drafts = min(n - skip, a.block);
    q.ctx = min(min(ctx, room) + skip, room);
    q.limit = min(q.ctx + q.drafts, room);
    q.n_pages = (q.limit + KV_PAGE - 1) / KV_PAGE;
    q.n_tiles = (q.n_pages + PG_PAGES - 1) / PG_PAGES;
    q.n_rt = (q.drafts * a.group + MR - 1) / MR;
    return q;
}
// Pieces in the order (tile of rows, sequence, head), so that CTAs half a round apart read the same keys at about the same time.  A piece is
// PG_START units and one for each of its tiles, so that a CTA with parts of two pieces has less of them (8 x 16 tokens at 8k, ragged: 63 k
// clocks with one piece and 80 k with two before).  All of a warp's lanes hold the same walk.
template <uint32_t MR>
struct PgWalk {
    uint32_t at, end, per;       // units of this CTA, units a CTA (the launcher sees to it that all of them are below 2^31)
    uint32_t rt, seq, head, tile;
    PgSeq q;

    __device__ __forceinline__ void start(const PagedAttnArgs &a) {
        const uint32_t lane = threadIdx.x & 31;
        auto load = [&](uint32_t s0) { return s0 + lane < a.n_units ? pg_seq<MR>(a, s0 + lane) : PgSeq{}; };
        const PgSeq front = load(0);  // (up to 32 sequences are read once)
        uint32_t total = 0;
#pragma unroll 1
        for (uint32_t s0 = 0; s0 < a.n_units; s0 += 32) {
            const PgSeq x = s0 ? load(s0) : front;
            total += (uint32_t)warp_sum_i((int)((x.n_tiles + PG_START) * x.n_rt)) * a.pg.n_kv;
        }
        per = max((total + gridDim.x - 1) / gridDim.x, PG_LEAST);
        at = min(total, blockIdx.x * per), end = min(total, at + per);
        rt = seq = head = tile = 0;
        q = PgSeq{};
        if (at >= end) return;
        uint32_t before = 0;
#pragma unroll 1
        for (rt = 0; rt < a.row_tiles; ++rt)
#pragma unroll 1
            for (uint32_t s0 = 0; s0 < a.n_units; s0 += 32) {
                const PgSeq x = s0 ? load(s0) : front;
                const uint32_t mine = rt < x.n_rt ? (x.n_tiles + PG_START) * a.pg.n_kv : 0;
                uint32_t sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= (uint32_t)o) sum += up;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, at < before + sum);
                if (hit) {
                    const int src = __ffs(hit) - 1;
                    auto of = [&](uint32_t v) { return __shfl_sync(0xffffffffu, v, src); };
                    const uint32_t off = at - (before + of(sum - mine));
                    seq = s0 + src;
                    q = PgSeq{of(x.row0), of(x.drafts), of(x.ctx), of(x.limit), of(x.n_pages), of(x.n_tiles), of(x.n_rt)};
                    head = off / (q.n_tiles + PG_START);
                    begin(off % (q.n_tiles + PG_START));
                    return;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        at = end;
    }
    __device__ __forceinline__ void begin(uint32_t unit) {  // at unit `unit` of a piece
        tile = unit > PG_START ? unit - PG_START : 0u;
        at += unit < PG_START ? PG_START - unit : 0u;
    }
    __device__ __forceinline__ bool more() const { return at < end; }
    __device__ __forceinline__ uint32_t last() const { return min(q.n_tiles, tile + (end - at)); }  // the present piece is tiles [tile, last())
    __device__ __forceinline__ void next(const PagedAttnArgs &a) {
        const uint32_t to = last();
        at += to - tile + PG_START;
        tile = 0;
        if (at >= end || ++head < a.pg.n_kv) return;
        head = 0;
        do {
            if (++seq == a.n_units) {
                seq = 0;
                if (++rt >= a.row_tiles) {  // (not while nobody writes the lengths meanwhile)
                    at = end;
                    return;
                }
            }
            q = pg_seq<MR>(a, seq);
        } while (q.n_rt <= rt);
    }
};

// 4-bit pages (layout: pages_q4.cuh): the entries are f16 numbers exactly, so that the operand tiles are those of an f16 cache, made by warps instead of TMA.  A warp
// has a tile's keys (or values) at a time: codes and units come by cp.async into places of its own, a tile ahead, and go as f16 into the swizzled rows.
template <int HD, bool VALUE>
struct P4Tile {
    using B = Q4Block<HD>;
    static constexpr uint32_t QUADS = HD / 32, WORDS = B::BYTES / 16, BYTES = PG_PAGES * B::BYTES;  // 16 bytes of codes: 32 entries with one unit; a row's, a lane's

    // id: lane p < PG_PAGES has the number of the tile's page p, or -1 (zeros: its entries are zero).
    static __device__ __forceinline__ void request(uint32_t dst, const uint8_t *pool, uint32_t n_kv, uint32_t head, int32_t id) {
        const uint32_t lane = threadIdx.x & 31;
#pragma unroll
        for (uint32_t p = 0; p < PG_PAGES; ++p) {
            const int32_t page = __shfl_sync(0xffffffffu, id, p);
            const uint8_t *block = pool + ((uint64_t)max(page, 0) * n_kv + head) * B::BYTES;
#pragma unroll
            for (uint32_t c = lane; c < WORDS; c += 32) cp16(dst + p * B::BYTES + c * 16, block + c * 16, page >= 0);
        }
    }
    static __device__ __forceinline__ void put(uint32_t at, uint32_t x, uint32_t d, uint32_t n) {  // eight entries
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q4_field(x, 0, d, n)), "r"(q4_field(x, 1, d, n)), "r"(q4_field(x, 2, d, n)), "r"(q4_field(x, 3, d, n)) : "memory");
    }
    // A lane's words of a page are ROWS positions apart, a multiple of 8: where it reads and writes within them and how its rows are swizzled stays the same.
    // (With addresses made for every word, 8 x 16 tokens of 4 heads at 8192 took 77 us, and 67 so.)
    static constexpr uint32_t PER = QUADS * KV_PAGE / 32, ROWS = KV_PAGE / PER;
    static __device__ __forceinline__ void make(uint32_t src, uint32_t operand) {
        const uint32_t lane = threadIdx.x & 31;
        // eight lanes write two rows, or one: those of the second block of columns (head dimension 64: of the second row) have another order, so that no two
        // are in one bank
        const uint32_t r = lane / (2 * QUADS), w = B::eight(r, 2 * (lane % (2 * QUADS))), pos = VALUE ? 2 * r : lane / QUADS, q = VALUE ? w / 4 : lane % QUADS;
        const bool other = VALUE ? (HD == 128 ? (w & 8) != 0 : (r & 1) != 0) : HD == 128 && (q & 2);
        uint32_t to[4];  // by the order of its stores; values: two eights of two positions
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t row = VALUE ? pos + (e & 1) : pos, c = VALUE ? (e / 2 ^ (other ? 1 : 0)) + w : 4 * q + (other ? e ^ 2 : e);
            to[e] = operand + c / 8 * PG_BLOCK + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        }
        const uint32_t unit = B::unit(VALUE, pos, q);
#pragma unroll 1
        for (uint32_t page = 0; page < PG_PAGES; ++page, src += B::BYTES) {
            uint32_t code[PER][4], u[PER];
#pragma unroll
            for (uint32_t i = 0; i < PER; ++i) {
                lds_words(code[i], src + i * 512 + lane * 16);
                u[i] = VALUE ? lds32(src + unit + B::unit(true, i * ROWS, 0) - B::CODES) : lds16(src + unit + B::unit(false, i * ROWS, 0) - B::CODES);
            }
#pragma unroll
            for (uint32_t i = 0; i < PER; ++i) {
                const uint32_t a0 = other ? code[i][2] : code[i][0], b0 = other ? code[i][3] : code[i][1], a1 = other ? code[i][0] : code[i][2], b1 = other ? code[i][1] : code[i][3], at = i * ROWS * 128;
                if constexpr (VALUE) {
                    const uint32_t d0 = __byte_perm(u[i], u[i], 0x1010), d1 = __byte_perm(u[i], u[i], 0x3232), n0 = q4_offset(d0), n1 = q4_offset(d1);
                    put(to[0] + at, __byte_perm(a0, b0, 0x5410), d0, n0);
                    put(to[1] + at, __byte_perm(a0, b0, 0x7632), d1, n1);
                    put(to[2] + at, __byte_perm(a1, b1, 0x5410), d0, n0);
                    put(to[3] + at, __byte_perm(a1, b1, 0x7632), d1, n1);
                } else {
                    const uint32_t d = __byte_perm(u[i], u[i], 0x1010), n = q4_offset(d);
                    put(to[0] + at, a0, d, n);
                    put(to[1] + at, b0, d, n);
                    put(to[2] + at, a1, d, n);
                    put(to[3] + at, b1, d, n);
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) to[e] += KV_PAGE * 128;
        }
    }
};

template <typename T, int HD, bool WIDE, bool Q4>
__global__ void __launch_bounds__(Q4 ? P4_THREADS : PG_THREADS, 1)
pages_tree_tc5_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedAttnArgs a) {
    using P = PgPlan<HD, WIDE, Q4>;
    using TP = typename std::conditional<Q4, __half, T>::type;  // of the operands
    constexpr uint32_t KST = P::KST, VST = P::VST, G = P::G, PLACE = P::PLACE, OPERAND = P::OPERAND, ROWS = P::ROWS, NB = P::NB, MR = P::MR;
    extern __shared__ __align__(1024) uint8_t smem[];  // (no other shared memory: the operand tiles' swizzle counts on the alignment)
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar = sbase + P::BAR, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile uint32_t *abort = reinterpret_cast<volatile uint32_t *>(smem + P::BAR + PB_ABORT);
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < PG_STAGES; ++s) {
            mbar_init(bar + PB_K_FULL + 8 * s, 1);
            mbar_init(bar + PB_K_EMPTY + 8 * s, WIDE ? 2 : 1);  // the streams that read a tile
            mbar_init(bar + PB_V_FULL + 8 * s, 1);
            mbar_init(bar + PB_V_EMPTY + 8 * s, WIDE ? 2 : 1);
        }
        for (uint32_t s = 0; s < 2; ++s) {
            for (uint32_t b = 0; b < 2; ++b) {
                mbar_init(bar + PB_S_FULL + 16 * s + 8 * b, 1);
                mbar_init(bar + PB_P_FULL + 16 * s + 8 * b, 4);
            }
            mbar_init(bar + PB_PV_DONE + 8 * s, 1);
            mbar_init(bar + PB_O_FULL + 8 * s, 1);
        }
        mbar_init(bar + PB_Q_FULL, 8);
        *abort = 0u;
        *reinterpret_cast<volatile uint32_t *>(smem + P::BAR + PB_ODD) = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == PG_MMA_WARP) tmem_alloc(bar + PB_SLOT, PG_TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_release();  // (only now: a CTA of the next kernel must not take the tensor memory first, it would keep it until this grid is done)
    pdl_wait();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + P::BAR + PB_SLOT);
    PgWalk<MR> w;
    w.start(a);
    // Tiles of a stream in a piece: all of them or every other one.  With two tiles of rows the second stream may have no rows.
    auto steps_of = [&](uint32_t s, uint32_t tiles, uint32_t rows) { return WIDE ? (s == 0 || rows > PG_ROWS ? tiles : 0u) : (tiles + 1 - s) / 2; };
    auto tile_of = [&](uint32_t s, uint32_t step) { return WIDE ? step : s + 2 * step; };

    if (warp >= PG_MMA_WARP) {
        // One instruction for all warps of a warpgroup, before their roles part.  256 threads x 104 and 256 x 152 are the 512 x 128 of the launch.
        static_assert(PG_MMA_WARP % 4 == 0 && P4_THREADS == 2 * PG_SOFT, "whole warpgroups");
        if constexpr (Q4) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (Q4 && warp >= PG_TMA_WARP) {
            if constexpr (Q4) {
                auto make = [&](auto value, uint32_t mine) {
                    constexpr bool VALUE = decltype(value)::value;
                    using Tile = P4Tile<HD, VALUE>;
                    constexpr uint32_t PLACES = VALUE ? VST : KST;
                    static_assert(PLACES % P4_TURNS == 0 && G == 1, "a place is always the same warp's");
                    const uint32_t full = bar + (VALUE ? PB_V_FULL : PB_K_FULL), empty = bar + (VALUE ? PB_V_EMPTY : PB_K_EMPTY);
                    const uint8_t *pool = static_cast<const uint8_t *>(VALUE ? a.pg.v : a.pg.k);
                    uint8_t *own = smem + P::CODES + (warp - PG_TMA_WARP) * P4_AHEAD * Tile::BYTES;
                    // The warp's next tile: number `at` of all tiles, those of its places.
                    uint32_t at = mine, before = 0;  // tiles of the pieces before
                    auto request = [&](uint32_t slot) {
                        for (; w.more() && at - before >= w.last() - w.tile; w.next(a)) before += w.last() - w.tile;
                        if (w.more()) {
                            const int32_t *table = a.pg.tables + (uint64_t)(a.blocks > 1 ? w.seq / a.blocks : w.seq) * a.pg.stride;
                            const uint32_t p = (w.tile + at - before) * PG_PAGES + lane % PG_PAGES;
                            int32_t id = p < w.q.n_pages ? table[p] : -1;
                            if ((uint32_t)id >= a.pg.n_pages) id = -1;
                            Tile::request(smem_addr(own) + slot * Tile::BYTES, pool, a.pg.n_kv, w.head, id);
                        }
                        cp_commit();
                        const bool any = w.more();
                        at += P4_TURNS;
                        return any;
                    };
                    bool ok = true;
                    uint32_t end = ~0u;  // the first of the warp's tiles that there is not
#pragma unroll 1
                    for (uint32_t n = mine, slot = 0; ok; slot = slot + 1 == P4_AHEAD ? 0 : slot + 1) {
                        if (!request(slot)) end = min(end, at - P4_TURNS);
                        if (at < mine + P4_AHEAD * P4_TURNS) continue;  // (the first ones are only asked for)
                        if (n >= end) break;
                        cp_wait<P4_AHEAD - 1>();
                        __syncwarp();
                        const uint32_t st = n % PLACES, from = slot + 1 == P4_AHEAD ? 0 : slot + 1;
                        ok = mbar_wait_warp(empty + 8 * st, ((n / PLACES) & 1u) ^ 1u, abort);  // (a place that was not used yet is empty)
                        if (!ok) break;
                        Tile::make(smem_addr(own) + from * Tile::BYTES, sbase + (VALUE ? P::V : P::K) + st * PLACE);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();  // (all of the warp's rows are written, and its codes read)
                        if (lane == 0) mbar_arrive(full + 8 * st);
                        n += P4_TURNS;
                    }
                    cp_wait<0>();
                };
                const uint32_t role = warp - PG_TMA_WARP;  // (two warps only fill their warpgroup)
                if (role < P4_CODE_WARPS && (role & 1)) make(std::true_type{}, role / 2);
                else if (role < P4_CODE_WARPS) make(std::false_type{}, role / 2);
            }
        } else if (warp >= PG_TMA_WARP) {
            const bool values = warp > PG_TMA_WARP;
            const CUtensorMap *map = values ? &tm_v : &tm_k;
            const uint32_t ring = sbase + (values ? P::V : P::K), full = bar + (values ? PB_V_FULL : PB_K_FULL), empty = bar + (values ? PB_V_EMPTY : PB_K_EMPTY), places = values ? VST : KST;
            uint32_t st = 0, par = 1;  // the tile's place, and the parity of its last use: a place that was not used yet is empty
            bool ok = true;
            const uint32_t nowhere = a.pg.n_pages * a.pg.n_kv * KV_PAGE;  // the row behind the pool: reads as zero
            const uint32_t page = lane % (G * PG_PAGES), box = lane / (G * PG_PAGES), at = page / PG_PAGES * OPERAND + box * PG_BLOCK + page % PG_PAGES * (KV_PAGE * 128);  // a lane a copy
            for (; w.more() && ok; w.next(a)) {
                const int32_t *table = a.pg.tables + (uint64_t)(a.blocks > 1 ? w.seq / a.blocks : w.seq) * a.pg.stride;
                const uint32_t end = w.last();
                auto row_of = [&](uint32_t tile) {  // the first row of the lane's page of the tiles from this one on
                    const uint32_t p = tile * PG_PAGES + page;
                    const int32_t id = p < min(end * PG_PAGES, w.q.n_pages) ? table[p] : -1;
                    return (uint32_t)id < a.pg.n_pages ? ((uint32_t)id * a.pg.n_kv + w.head) * KV_PAGE : nowhere;
                };
                uint32_t y = row_of(w.tile);
                for (uint32_t i = w.tile; i < end; i += G) {
                    const uint32_t next = row_of(i + G);
                    if (!(ok = mbar_wait_warp(empty + 8 * st, par, abort))) break;
                    if (lane == 0) mbar_expect_tx(full + 8 * st, PLACE);
                    __syncwarp();
                    if (box < NB) tma_load_2d(ring + st * PLACE + at, map, (int32_t)(box * 64), (int32_t)y, full + 8 * st);
                    __syncwarp();
                    y = next;
                    if (++st == places) st = 0, par ^= 1;
                }
            }
        } else {
            constexpr uint32_t F16 = EXPONENT16<TP> == EXPONENT16<bf16> ? 0u : (1u << 7) | (1u << 10);  // the operands' format bits: zero for f16
            const uint32_t id_s = umma_idesc_bf16(PG_KEYS) & ~F16, id_o = (umma_idesc_bf16(HD) & ~F16) | UMMA_B_MN_MAJOR;
            const uint32_t s = warp - PG_MMA_WARP, ts = tmem + PG_TMEM_S + s * 2 * PG_KEYS, to = tmem + PG_TMEM_O + s * 128;
            uint32_t n = 0, turn = 0, done = 0;  // places, pieces and tiles of the stream so far
            bool ok = true;
            const uint64_t q_desc = umma_desc_sw128(sbase + (WIDE ? s * ROWS : 0u)), k_desc = umma_desc_sw128(sbase + P::K), v_desc = umma_desc_sw128_mn(sbase + P::V, PG_BLOCK);
            for (; w.more() && ok; w.next(a), ++turn) {
                const uint32_t tiles = w.last() - w.tile, steps = steps_of(s, tiles, w.q.drafts * a.group - w.rt * MR);
                ok = mbar_wait_warp(bar + PB_Q_FULL, turn & 1u, abort);  // (of every piece: a phase that is not waited for could be taken for the next one)
                if (WIDE && steps == 0)  // no rows: only says of every tile that it does not need it
                    for (uint32_t i = 0; i < (tiles + G - 1) / G && ok; ++i) {
                        const uint32_t kt = (n + i) % KST, vt = (n + i) % VST;
                        ok = mbar_wait_warp(bar + PB_K_FULL + 8 * kt, ((n + i) / KST) & 1u, abort) && mbar_wait_warp(bar + PB_V_FULL + 8 * vt, ((n + i) / VST) & 1u, abort);
                        if (ok && lane == 0) mbar_arrive(bar + PB_K_EMPTY + 8 * kt), mbar_arrive(bar + PB_V_EMPTY + 8 * vt);
                        __syncwarp();
                    }
#pragma unroll 1
                for (int step = -2; step < (int)steps && ok; ++step) {  // -2, -1: only the first scores
                    const uint32_t place = (done + step) & 1u;
                    if (step >= 0) {
                        const uint32_t i = tile_of(s, step), at = n + i / G, st = at % VST;
                        if (i % G == 0) ok = mbar_wait_warp(bar + PB_V_FULL + 8 * st, (at / VST) & 1u, abort);
                        ok = ok && mbar_wait_warp(bar + PB_P_FULL + 16 * s + 8 * place, (done + step) >> 1 & 1u, abort);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t p = ts + place * PG_KEYS;
                        const uint64_t vd = v_desc + ((st * PLACE + i % G * OPERAND) >> 4);
#pragma unroll
                        for (uint32_t kk = 0; kk < PG_KEYS / 16; ++kk) {  // the stream's first product writes, the others add; 16 positions: eight columns of values, eight of remainders
                            umma_bf16_ta_warp(to, p + kk * 16, vd + kk * 128, id_o, step || kk ? 1u : 0u);
                            umma_bf16_ta_warp(to, p + kk * 16 + 8, vd + kk * 128, id_o, 1u);
                        }
                        umma_commit_warp(bar + PB_PV_DONE + 8 * s);
                        if (i % G == G - 1 || step + 1 == (int)steps) umma_commit_warp(bar + PB_V_EMPTY + 8 * st);
                    }
                    const uint32_t next = step + 2;
                    if (next < steps) {
                        const uint32_t i = tile_of(s, next), at = n + i / G, st = at % KST;
                        if (i % G == 0) ok = mbar_wait_warp(bar + PB_K_FULL + 8 * st, (at / KST) & 1u, abort);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t kd = k_desc + ((st * PLACE + i % G * OPERAND) >> 4);
#pragma unroll
                        for (uint32_t b = 0; b < HD / 16; ++b)
                            umma_bf16_warp(ts + place * PG_KEYS, q_desc + (b / 4) * (PG_QBLOCK >> 4) + 2 * (b % 4), kd + (b / 4) * (PG_BLOCK >> 4) + 2 * (b % 4), id_s, b ? 1u : 0u);
                        umma_commit_warp(bar + PB_S_FULL + 16 * s + 8 * place);
                        if (i % G == G - 1 || next + 1 == steps) umma_commit_warp(bar + PB_K_EMPTY + 8 * st);
                    } else if (next == steps + 1 && steps > 0) {
                        umma_commit_warp(bar + PB_O_FULL + 8 * s);
                    }
                }
                n += (tiles + G - 1) / G, done += steps;
            }
        }
    } else {
        if constexpr (Q4) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        const uint32_t s = warp / 4, quad = warp % 4, r = quad * 32 + lane;
        const uint32_t magic = (65536 + a.group - 1) / a.group;  // x / group = x magic / 65536 for x below 4096, group up to 16
        float scale2 = a.scale * 1.4426950408889634f;  // weights are powers of two of the scaled score
        constexpr bool FACTORS = !std::is_same<T, TP>::value;
        const uint32_t lanes = tmem + ((quad * 32) << 16), ts = lanes + PG_TMEM_S + s * 2 * PG_KEYS, to = lanes + PG_TMEM_O;
        volatile float *xchg = reinterpret_cast<volatile float *>(smem + P::BAR + PB_TOP) + r;  // [stream][sum, maximum][row]; before, in a sum's place, its thread's factor of the scores
        volatile uint32_t *odd = reinterpret_cast<volatile uint32_t *>(smem + P::BAR + PB_ODD);
        bool ok = true;
        uint32_t used = 0, n = 0;   // tiles of the stream, places so far
        bool said = false;          // a piece that others go on with has been written down
        uint32_t both[2] = {0, 0};  // pieces with tiles of either stream (WIDE false: every warp reads both outputs)
        for (; w.more(); w.next(a)) {
            const uint32_t end = w.last(), tiles = end - w.tile, n_rows = w.q.drafts * a.group - w.rt * MR;  // rows from this tile of rows on
            const uint32_t f_row = (WIDE ? s * PG_ROWS : 0u) + r, warp_row = (WIDE ? s * PG_ROWS : 0u) + quad * 32;
            const bool live = f_row < n_rows, warm = warp_row < n_rows;  // this row, any row of the warp
            const int32_t *table = a.pg.tables + (uint64_t)(a.blocks > 1 ? w.seq / a.blocks : w.seq) * a.pg.stride;
            // ---- the queries, 16 bytes a thread and turn
            constexpr uint32_t WORDS = HD / 8, TURNS = MR * WORDS / PG_SOFT, BATCH = TURNS < 8 ? TURNS : 8;  // (all of a batch's loads before its stores)
#pragma unroll 1
            for (uint32_t t = 0; t < TURNS; t += BATCH) {
                uint4 v[BATCH];
#pragma unroll
                for (uint32_t k = 0; k < BATCH; ++k) {
                    const uint32_t i = (t + k) * PG_SOFT + threadIdx.x, row = i / WORDS, c = i % WORDS, f = w.rt * MR + row, t0 = f * magic >> 16;
                    v[k] = make_uint4(0, 0, 0, 0);
                    if (row < n_rows) v[k] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (uint64_t)(w.q.row0 + t0) * a.q_stride + (w.head * a.group + f - t0 * a.group) * HD + 8 * c));
                }
#pragma unroll
                for (uint32_t k = 0; k < BATCH; ++k) {
                    const uint32_t i = (t + k) * PG_SOFT + threadIdx.x, row = i / WORDS, c = i % WORDS;
                    if constexpr (FACTORS) {  // bfloat16 queries become f16 ones after a power of two per row has been taken out (pages_q4.cu)
                        uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w}, top = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7fffu, u[e] >> 16 & 0x7fffu));
#pragma unroll
                        for (uint32_t o = 1; o < WORDS; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const int e = top == 0 || top >= 0x7f80u ? 0 : max(-112, min(112, 14 - ((int)(top >> 7) - 127)));
                        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float2 f = unpack16(u[x], T());
                            u[x] = pack16<TP>(f.x * up, f.y * up);
                        }
                        v[k] = make_uint4(u[0], u[1], u[2], u[3]);
                        if (c == 0) {
                            volatile float *factor = reinterpret_cast<volatile float *>(smem + P::BAR + PB_TOP) + row % PG_ROWS;
                            factor[row / PG_ROWS * 2 * PG_ROWS] = __uint_as_float((uint32_t)(127 - e) << 23);
                            if (!WIDE) factor[2 * PG_ROWS] = __uint_as_float((uint32_t)(127 - e) << 23);
                        }
                    }
                    *reinterpret_cast<uint4 *>(smem + row / PG_ROWS * ROWS + c / 8 * PG_QBLOCK + row % PG_ROWS * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[k];
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar + PB_Q_FULL);
            if constexpr (FACTORS) {
                soft_sync();
                scale2 = a.scale * 1.4426950408889634f * xchg[2 * s * PG_ROWS];
            }
            uint64_t seen = 0;
            if (live && w.q.ctx < end * PG_KEYS) {
                const uint32_t token = (w.rt * MR + f_row) / a.group;
                seen = a.visible ? a.visible[w.q.row0 + token] : (2ull << token) - 1;
                if (w.q.limit - w.q.ctx < 64) seen &= (1ull << (w.q.limit - w.q.ctx)) - 1;
            }
            auto pages_of = [&](uint32_t tile) {  // whether the lane's page of the tile is there
                const uint32_t p = tile * PG_PAGES + lane % PG_PAGES;
                return tile < end && p < w.q.n_pages && (uint32_t)table[p] < a.pg.n_pages;
            };
            // ---- the tiles
            const uint32_t steps = steps_of(s, tiles, n_rows);
            float m = -INFINITY, l = 0.0f;
            bool there = pages_of(w.tile + tile_of(s, 0));
            for (uint32_t step = 0; step < steps; ++step, ++used) {
                const uint32_t i = tile_of(s, step), place = used & 1, x0 = (w.tile + i) * PG_KEYS, valid = __ballot_sync(0xffffffffu, there) & ((1u << PG_PAGES) - 1);
                const bool past = x0 + PG_KEYS > w.q.ctx;
                there = pages_of(w.tile + tile_of(s, step + 1));
                ok = ok && mbar_wait_warp(bar + PB_S_FULL + 16 * s + 8 * place, used >> 1 & 1u, abort);
                if (ok && past) ok = mbar_wait_warp(bar + PB_V_FULL + 8 * ((n + i / G) % VST), ((n + i / G) / VST) & 1u, abort);
                if (!ok) break;  // a wait was given up: nothing more is computed
                if (past) {  // values of positions past the context
                    uint8_t *v = smem + P::V + (n + i / G) % VST * PLACE + i % G * OPERAND;
                    const uint32_t from = w.q.ctx > x0 ? w.q.ctx - x0 : 0u;
                    bool bad = false;
#pragma unroll 1
                    for (uint32_t c = from * 8 + (warp % 4) * 32 + lane; c < PG_KEYS * 8; c += 128)
#pragma unroll 1
                        for (uint32_t b = 0; b < NB; ++b) {
                            uint4 *at = reinterpret_cast<uint4 *>(v + b * PG_BLOCK) + c;
                            uint32_t u[4] = {at->x, at->y, at->z, at->w};
                            if (x0 + c / 8 >= w.q.limit) {
                                *at = make_uint4(0, 0, 0, 0);
                            } else {
                                bool here = false;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    if ((u[e] & EXPONENT16<TP>) == EXPONENT16<TP>) u[e] &= 0xffff0000u, here = true;
                                    if ((u[e] >> 16 & EXPONENT16<TP>) == EXPONENT16<TP>) u[e] &= 0xffffu, here = true;
                                }
                                if (here) *at = make_uint4(u[0], u[1], u[2], u[3]), bad = true;
                            }
                        }
                    if (bad) *odd = 1u;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (warm) {
                    const uint32_t tp = ts + place * PG_KEYS;
                    tc_fence_after();
                    uint32_t u[2][32];
                    tmem_ld32(tp, u[0]);
                    tmem_ld32(tp + 32, u[1]);
                    tmem_ld_wait();
                    if (valid != (1u << PG_PAGES) - 1 || past) {
                        uint64_t bits = x0 >= w.q.ctx ? 0ull : w.q.ctx - x0 >= 64 ? ~0ull : (1ull << (w.q.ctx - x0)) - 1;  // what the row sees: context,
                        if (past) {                                                                                       // drafted token j at ctx + j
                            const int shift = (int)(w.q.ctx - x0);  // above -64 where any of them is here
                            bits |= shift >= 0 ? seen << shift : shift > -64 ? seen >> -shift : 0ull;
                        }
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            if (!(valid >> p & 1)) bits &= ~(0xffffull << (16 * p));
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            if (!(bits >> e & 1)) u[e / 32][e % 32] = 0xff800000u;
                    }
                    // weights against the maximum so far, which stays while no score is above it by more than the slack: then the output need not be
                    // rescaled, and the new maximum is not waited for
                    if (__any_sync(0xffffffffu, m == -INFINITY)) {  // a row that has seen nothing yet: its first maximum
                        float top = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 64; e += 2) top = max3(top, __uint_as_float(u[e / 32][e % 32]), __uint_as_float(u[e / 32][e % 32 + 1]));
                        if (m == -INFINITY) m = top * scale2;
                    }
                    float sum0, sum1;
#pragma unroll 1
                    for (;;) {
                        const float base = m == -INFINITY ? 0.0f : PG_RAISE<TP> - m;  // (still nothing: weights of zero)
                        float top[2] = {-INFINITY, -INFINITY};
                        sum0 = sum1 = 0.0f;
#pragma unroll
                        for (int g = 0; g < 4; ++g) {  // 16 positions
                            uint32_t v[16];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float x0 = __uint_as_float(u[g / 2][g % 2 * 16 + 2 * e]), x1 = __uint_as_float(u[g / 2][g % 2 * 16 + 2 * e + 1]);
                                float e0, e1;
                                top[e % 2] = max3(top[e % 2], x0, x1);
                                fma2(e0, e1, x0, x1, scale2, base);
                                e0 = pow2(e0), e1 = pow2(e1);
                                add2(sum0, sum1, e0, e1);
                                v[e] = pack16<TP>(e0, e1);
                                const float2 r = unpack16(v[e], TP());
                                v[8 + e] = pack16<TP>(e0 - r.x, e1 - r.y);
                            }
                            tmem_st16(tp + 16 * g, v);
                        }
                        const float now = fmaxf(top[0], top[1]) * scale2;
                        const bool grown = now > m + PG_SLACK;
                        if (!__any_sync(0xffffffffu, grown)) break;
                        if (step > 0) ok = mbar_wait_warp(bar + PB_PV_DONE + 8 * s, (used - 1) & 1u, abort);  // the product before these scores
                        tc_fence_after();
                        const float keep = grown ? pow2(m - now) : 1.0f;
                        if (grown) m = now, l *= keep;
#pragma unroll 1
                        for (uint32_t c = 0; c < HD; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(to + s * 128 + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st16(to + s * 128 + c, o);
                        }
                    }
                    l += sum0 + sum1;
                    tmem_st_wait();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar + PB_P_FULL + 16 * s + 8 * place);
            }
            n += (tiles + G - 1) / G;
            // ---- the piece is done: the streams' outputs and sums
            const bool had[2] = {true, WIDE ? n_rows > PG_ROWS : tiles > 1};
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k)
                if (had[k]) {
                    if (!WIDE || k == s) ok = ok && mbar_wait_warp(bar + PB_O_FULL + 8 * k, both[k] & 1u, abort);
                    ++both[k];
                }
            tc_fence_after();
            xchg[2 * s * PG_ROWS] = l, xchg[(2 * s + 1) * PG_ROWS] = m;
            soft_sync();
            const bool whole = w.tile == 0 && end == w.q.n_tiles;
            const uint32_t origin = w.at - w.tile, begin = blockIdx.x * w.per;  // of the piece's first tile and of this CTA, in units
            float *part_out = a.partial + (2ull * blockIdx.x + (origin > begin ? 1 : 0)) * P::PART;  // a CTA has a part of two pieces at most
            // this thread's columns of its row: all of them, or (both streams have the same rows) half of them of both outputs
            constexpr uint32_t COLS = WIDE ? HD : HD / 2;
            const uint32_t col0 = WIDE ? 0u : s * COLS;
            float f0 = 1.0f, f1 = 0.0f, sum = l, peak = m;
            if (!WIDE) {
                const float m0 = xchg[PG_ROWS], m1 = had[1] ? xchg[3 * PG_ROWS] : -INFINITY;
                peak = fmaxf(m0, m1);
                f0 = m0 == -INFINITY ? 0.0f : pow2(m0 - peak), f1 = m1 == -INFINITY ? 0.0f : pow2(m1 - peak);
                sum = xchg[0] * f0 + (had[1] ? xchg[2 * PG_ROWS] * f1 : 0.0f);
            }
            const float norm = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // nothing seen: 0; a sum that is no number stays none
            const bool special = *odd != 0u;
            const float gain = whole ? norm : 1.0f, g0 = f0 * gain, g1 = f1 * gain;
            // 16 columns at a time, a thread per row -> four lanes a row: whole sectors, by way of the queries' place, which no product reads any
            // more.  (One form for results and parts: instructions that are executed once are fetched from memory first.)
            uint8_t *stage = smem + warp * 2048;
            if (ok && warm && (!WIDE || had[s]))
#pragma unroll 1
                for (uint32_t c = 0; c < COLS; c += 16) {
                    uint32_t o0[16], o1[16];
                    tmem_ld16(to + (WIDE ? s * 128 : 0u) + col0 + c, o0);
                    if (!WIDE) tmem_ld16(to + 128 + col0 + c, o1);
                    tmem_ld_wait();
                    float x[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        x[e] = __uint_as_float(o0[e]) * g0;
                        if (!WIDE && had[1]) x[e] = fmaf(__uint_as_float(o1[e]), g1, x[e]);  // (a stream without tiles has left nothing there)
                    }
                    if (!Q4 && special && live) {  // values that are no numbers, of drafted tokens that this row sees (their weights are above zero)
#pragma unroll 1
                        for (uint32_t j = 0; j < w.q.limit - w.q.ctx; ++j) {
                            const uint32_t pos = w.q.ctx + j;
                            if (!(seen >> j & 1) || pos < w.tile * PG_KEYS || pos >= end * PG_KEYS) continue;
                            const int32_t id = table[pos / KV_PAGE];
                            if ((uint32_t)id >= a.pg.n_pages) continue;
                            const T *v = static_cast<const T *>(a.pg.v) + (((uint64_t)id * a.pg.n_kv + w.head) * KV_PAGE + pos % KV_PAGE) * HD + col0 + c;
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float y = from16(v[e]);
                                if (!(fabsf(y) <= 3.4028235e38f)) x[e] += y;
                            }
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<float4 *>(stage + lane * 64 + ((e ^ (lane >> 1 & 3)) << 4)) = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                    __syncwarp();
                    float4 y[4];
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t row = lane / 4 + 8 * k;
                        y[k] = *reinterpret_cast<const float4 *>(stage + row * 64 + (((lane & 3) ^ (row >> 1 & 3)) << 4));
                    }
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t row = warp_row + lane / 4 + 8 * k, e = col0 + c + 4 * (lane & 3);
                        if (row >= n_rows) break;
                        const uint32_t f = w.rt * MR + row, t0 = f * magic >> 16;
                        if (whole)
                            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + (uint64_t)(w.q.row0 + t0) * a.out_stride + (w.head * a.group + f - t0 * a.group) * HD + e) =
                                make_uint2(pack16<T>(y[k].x, y[k].y), pack16<T>(y[k].z, y[k].w));
                        else
                            __stcg(reinterpret_cast<float4 *>(part_out + (uint64_t)row * HD + e), y[k]);
                    }
                }
            if (whole && a.stats && live && (WIDE || s == 0)) {
                const uint32_t f = w.rt * MR + f_row, t0 = f * magic >> 16;
                a.stats[(uint64_t)(w.q.row0 + t0) * a.group * a.pg.n_kv + w.head * a.group + f - t0 * a.group] = make_float2(peak - PG_RAISE<TP>, norm);
            }
            if (!whole && live && (WIDE || s == 0)) __stcg(reinterpret_cast<float2 *>(part_out + (uint64_t)MR * HD + 2 * f_row), make_float2(peak, sum));
            if (!whole && origin >= begin && threadIdx.x == 0) {  // the piece begins here and goes on in other CTAs (one piece at most)
                a.pieces[blockIdx.x] = PagePiece{(origin + w.q.n_tiles - 1) / w.per - blockIdx.x + 1, 2 * blockIdx.x + (origin > begin ? 1u : 0u), min(n_rows, MR), w.rt * MR, w.q.row0, w.head};
                said = true;
            }
            tc_fence_before();
            soft_sync();  // outputs, sums and maxima have been read
            if (threadIdx.x == 0) *odd = 0u;
        }
        if (threadIdx.x == 0 && !said) a.pieces[blockIdx.x].parts = 0;
    }
    __syncwarp();
    if (*abort) gave_up(a.status);
    tc_fence_before();
    __syncthreads();
    if (warp == PG_MMA_WARP) tmem_dealloc(tmem, PG_TMEM_COLS);
}

// grid (CTAs of the kernel above, rows / ROWS): the parts of the piece that began in a CTA, four columns a thread.
template <typename T, int HD, uint32_t MR, bool Q4>
__global__ void __launch_bounds__(256) pages_merge_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr uint32_t VEC = HD / 4, ROWS = 256 / VEC;
    constexpr uint64_t PART = (uint64_t)MR * (HD + 2);
    pdl_release();
    pdl_wait();
    const PagePiece p = a.pieces[blockIdx.x];
    const uint32_t row = blockIdx.y * ROWS + threadIdx.x / VEC, c = threadIdx.x % VEC;
    if (p.parts == 0 || row >= p.rows) return;
    float top = -INFINITY, total = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (uint32_t k = 0; k < p.parts; ++k) {
        const float *at = a.partial + (k ? (p.slot & ~1u) + 2 * k : p.slot) * PART;
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(at + (uint64_t)MR * HD + 2 * row));
        const float4 y = __ldcg(reinterpret_cast<const float4 *>(at + (uint64_t)row * HD + 4 * c));
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;
        const float higher = fmaxf(top, ml.x), g0 = top == -INFINITY ? 0.0f : pow2(top - higher), g1 = ml.x == -INFINITY ? 0.0f : pow2(ml.x - higher);
        top = higher;
        total = fmaf(ml.y, g1, total * g0);
        x.x = fmaf(y.x, g1, x.x * g0), x.y = fmaf(y.y, g1, x.y * g0), x.z = fmaf(y.z, g1, x.z * g0), x.w = fmaf(y.w, g1, x.w * g0);
    }
    const float g = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;
    const uint32_t f = p.row + row;
    if (a.stats && c == 0) a.stats[(uint64_t)(p.token0 + f / a.group) * a.group * a.pg.n_kv + p.head * a.group + f % a.group] = make_float2(top - PG_RAISE<typename std::conditional<Q4, __half, T>::type>, g);
    *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + (uint64_t)(p.token0 + f / a.group) * a.out_stride + (uint64_t)(p.head * a.group + f % a.group) * HD + 4 * c) =
        make_uint2(pack16<T>(x.x * g, x.y * g), pack16<T>(x.z * g, x.w * g));
}

// A barrier that nothing arrives at, waited for with a short limit.
__global__ void __launch_bounds__(32) pages_wait_selftest_kernel(uint32_t *status) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ uint32_t abort;
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bar), 1);
        abort = 0u;
    }
    __syncwarp();
    const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), 0u, &abort, 256));
    if (!ok && *reinterpret_cast<volatile uint32_t *>(&abort)) gave_up(status);
}

template <typename T, int HD, bool WIDE, bool Q4>
cudaError_t launch(PagedAttnArgs a, const PageMaps &maps, int sm_count, cudaStream_t st) {
    using P = PgPlan<HD, WIDE, Q4>;
    auto kernel = pages_tree_tc5_kernel<T, HD, WIDE, Q4>;
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::BYTES); })) return e;
    const uint32_t most = std::min(a.max_drafts, a.block);  // tokens of a unit
    a.row_tiles = (most * a.group + P::MR - 1) / P::MR;
    const uint32_t ctas = std::min<uint32_t>({(uint32_t)sm_count, PG_COUNTERS, (uint32_t)(PG_PARTS / (2 * P::PART * 4))});
    static_assert(sizeof(PageMaps) == 2 * sizeof(CUtensorMap), "two maps");
    CUtensorMap tm[2];
    memcpy(tm, &maps, sizeof(tm));
    if (cudaError_t e = launch_pdl(kernel, dim3(ctas), dim3(Q4 ? P4_THREADS : PG_THREADS), P::BYTES, st, tm[0], tm[1], a)) return e;
    const uint32_t rows = std::min(P::MR, most * a.group), per = 256 / (HD / 4);
    return launch_pdl(pages_merge_kernel<T, HD, P::MR, Q4>, dim3(ctas, (rows + per - 1) / per), dim3(256), 0, st, a);
}

}  // namespace

bool make_page_maps(const PageView &pg, PageMaps *out) {
    const uint64_t rows = (uint64_t)pg.n_pages * pg.n_kv * KV_PAGE;
    if (rows + 128 > 0x7fffffffull) return false;  // coordinates have 31 bits, and a row behind the pool is asked for
    const CUtensorMapDataType type = pg.is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap tm[2];
    if (!make_map_2d(&tm[0], type, 2, pg.k, pg.dim, rows, (uint64_t)pg.dim * 2, 64, KV_PAGE, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !make_map_2d(&tm[1], type, 2, pg.v, pg.dim, rows, (uint64_t)pg.dim * 2, 64, KV_PAGE, CU_TENSOR_MAP_SWIZZLE_128B))
        return false;
    memcpy(out, tm, sizeof(tm));
    return true;
}

template <bool Q4>
static cudaError_t launch_type(const PagedAttnArgs &a, bool is_bf16, const PageMaps &maps, int sm_count, cudaStream_t st) {
    const bool wide = std::min(a.max_drafts, a.block) * a.group > PG_ROWS;
    if (is_bf16) {
        if (a.pg.dim == 64) return wide ? launch<bf16, 64, true, Q4>(a, maps, sm_count, st) : launch<bf16, 64, false, Q4>(a, maps, sm_count, st);
        return wide ? launch<bf16, 128, true, Q4>(a, maps, sm_count, st) : launch<bf16, 128, false, Q4>(a, maps, sm_count, st);
    }
    if (a.pg.dim == 64) return wide ? launch<__half, 64, true, Q4>(a, maps, sm_count, st) : launch<__half, 64, false, Q4>(a, maps, sm_count, st);
    return wide ? launch<__half, 128, true, Q4>(a, maps, sm_count, st) : launch<__half, 128, false, Q4>(a, maps, sm_count, st);
}
cudaError_t launch_pages_tree_tc5(const PagedAttnArgs &a, const PageMaps &maps, int sm_count, cudaStream_t st) { return launch_type<false>(a, a.pg.is_bf16, maps, sm_count, st); }
cudaError_t launch_pages_q4_tc5(const PagedAttnArgs &a, bool q_bf16, int sm_count, cudaStream_t st) { return launch_type<true>(a, q_bf16, PageMaps{}, sm_count, st); }

cudaError_t launch_pages_wait_selftest(uint32_t *status, cudaStream_t st) {
    pages_wait_selftest_kernel<<<1, 32, 0, st>>>(status);
    return cudaGetLastError();
}

}  // namespace ob
