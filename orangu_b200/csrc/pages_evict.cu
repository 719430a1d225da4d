// Cutting a cache down (ob_pages_evict): per layer, sequence and key/value head the first and the last positions stay, and of the others those with the
// most weight; what stays moves together, in order.  And the accepted positions of drafts in 4-bit pages, and of masses (ob_pages_keep).
//
// The choice is that of pages_select.cu, by counts in equal parts of the masses' range: a CTA per (layer, sequence, head), the words of its masses in shared
// memory where they fit.  The move goes to places that are never behind their sources (kept[j] >= j), so that a CTA that goes through a head's list
// in order may read ahead as far as it likes, and has only to have read a batch before it writes it: one barrier a batch, no copy in between.
#include <algorithm>

#include "mixers_common.cuh"
#include "pages.h"
#include "pages_pick.cuh"
#include "pages_q4.cuh"

namespace ob {

namespace {

constexpr uint32_t EV_HELD = 32768;  // words of masses in shared memory at most
constexpr uint32_t EV_DEEP = 4;  // pieces of a thread in flight

// Larger masses have larger words; what is no number has the smallest.
__device__ __forceinline__ uint32_t mass_word(float s) {
    if (s != s) return 0u;
    const uint32_t u = __float_as_uint(s + 0.0f);  // (-0 is 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
struct MassWords {
    const float *mass;
    uint32_t first, last;  // places below `first` and from `last` on are taken
    __device__ __forceinline__ uint32_t operator[](uint32_t i) const { return i < first || i >= last ? SEL_FORCED : mass_word(__ldcg(mass + i)); }
};

// grid (layers x sequences x heads)
template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) pages_evict_choose_kernel(const __grid_constant__ PagedEvictArgs a, uint32_t held) {
    extern __shared__ __align__(16) uint32_t s_words[];
    pdl_release();
    pdl_wait();
    const uint32_t seq = blockIdx.x / a.pg.n_kv % a.n_seq;
    const uint32_t n = min(a.n_pos[seq], a.pg.stride * KV_PAGE);
    int32_t *out = a.kept + (uint64_t)blockIdx.x * a.n_keep;
    if (blockIdx.x % a.pg.n_kv == 0 && blockIdx.x / a.pg.n_kv < a.n_seq && threadIdx.x == 0) a.n_left[seq] = min(n, a.n_keep);
    if (n <= a.n_keep) {
        for (uint64_t i = threadIdx.x; i < a.n_keep; i += THREADS) out[i] = i < n ? (int32_t)i : -1;  // (in 32 bits the last turn of a list of almost 2^32 would begin anew)
        return;
    }
    const MassWords words{a.mass + (uint64_t)blockIdx.x * a.mass_stride, a.keep_first, n - a.keep_last};
    uint32_t lo = 0xffffffffu, hi = 0;
    const bool fits = n <= held;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        const uint32_t w = words[i];
        if (fits) s_words[i] = w;
        if (w != SEL_FORCED) lo = min(lo, w), hi = max(hi, w);
    }
    const uint32_t want = a.n_keep - a.keep_first - a.keep_last;
    if (fits) pick<THREADS>(want, s_words, n, lo, hi, out);
    else pick<THREADS>(want, words, n, lo, hi, out);
}

// One position's key or value of a head, in pieces that a thread moves.
template <int HD>
struct Row16 {
    static constexpr uint32_t PIECES = HD / 8, BLOCK = KV_PAGE * HD * 2;
    using Word = uint4;
    static __device__ __forceinline__ Word load(const uint8_t *block, bool, uint32_t p, uint32_t i) { return *reinterpret_cast<const uint4 *>(block + p * HD * 2 + i * 16); }
    static __device__ __forceinline__ void store(uint8_t *block, bool, uint32_t p, uint32_t i, Word x) { *reinterpret_cast<uint4 *>(block + p * HD * 2 + i * 16) = x; }
};
template <int HD>
struct Row4 {  // eight entries each, then units
    using B = Q4Block<HD>;
    static constexpr uint32_t EIGHTS = HD / 8, PIECES = EIGHTS + B::GROUPS, BLOCK = B::BYTES;
    using Word = uint32_t;
    static __device__ __forceinline__ Word load(const uint8_t *block, bool value, uint32_t p, uint32_t i) {
        if (i >= EIGHTS) return *reinterpret_cast<const uint16_t *>(block + B::unit(value, p, i - EIGHTS));
        if (!value) return *reinterpret_cast<const uint32_t *>(block + B::key(p, i));
        const uint16_t *at = reinterpret_cast<const uint16_t *>(block + B::value(p, i));
        return at[0] | (uint32_t)at[2] << 16;
    }
    static __device__ __forceinline__ void store(uint8_t *block, bool value, uint32_t p, uint32_t i, Word x) {
        if (i >= EIGHTS) {
            *reinterpret_cast<uint16_t *>(block + B::unit(value, p, i - EIGHTS)) = (uint16_t)x;
        } else if (!value) {
            *reinterpret_cast<uint32_t *>(block + B::key(p, i)) = x;
        } else {
            uint16_t *at = reinterpret_cast<uint16_t *>(block + B::value(p, i));
            at[0] = (uint16_t)x, at[2] = (uint16_t)(x >> 16);
        }
    }
};

// grid (layers x sequences x heads, 3): keys, values, masses.  While a batch is copied the pages of the next one and the list of the one after are read: the three loads
// that depend on each other are under way at once.  8 sequences of up to 4100, 32 layers of 8 heads of 128, to 2048: 397 us without, 331 with (5 TB/s in pieces of 256 bytes);
// more CTAs on a multiprocessor made it slower (three quarters of the registers each: 553).
template <typename R, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) pages_evict_move_kernel(const __grid_constant__ PagedEvictArgs a) {
    pdl_release();
    pdl_wait();
    const uint32_t head = blockIdx.x % a.pg.n_kv, seq = blockIdx.x / a.pg.n_kv % a.n_seq, layer = blockIdx.x / a.pg.n_kv / a.n_seq;
    const uint32_t n = min(a.n_pos[seq], a.pg.stride * KV_PAGE);
    if (n <= a.n_keep) return;
    const int32_t *kept = a.kept + (uint64_t)blockIdx.x * a.n_keep;
    if (blockIdx.y == 2) {
        float *mass = a.mass + (uint64_t)blockIdx.x * a.mass_stride;
        uint32_t src[EV_DEEP];
        auto list = [&](uint32_t j0) {
#pragma unroll
            for (uint32_t u = 0; u < EV_DEEP; ++u) {
                const uint32_t j = j0 + u * THREADS + threadIdx.x;
                src[u] = j < a.n_keep ? (uint32_t)kept[j] : 0u;
            }
        };
        list(a.keep_first);
#pragma unroll 1
        for (uint32_t j0 = a.keep_first; j0 < a.n_keep; j0 += EV_DEEP * THREADS) {
            float x[EV_DEEP];
#pragma unroll
            for (uint32_t u = 0; u < EV_DEEP; ++u) x[u] = mass[src[u]];
            list(j0 + EV_DEEP * THREADS);
            __syncthreads();  // a batch has been read before it is written; what the next one reads lies behind it
#pragma unroll
            for (uint32_t u = 0; u < EV_DEEP; ++u) {
                const uint32_t j = j0 + u * THREADS + threadIdx.x;
                if (j < a.n_keep) mass[j] = x[u];
            }
        }
        return;
    }
    const bool value = blockIdx.y;
    uint8_t *pool = static_cast<uint8_t *>(const_cast<void *>(value ? a.pg.v : a.pg.k)) + layer * a.layer_bytes + (uint64_t)head * R::BLOCK;
    const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;
    constexpr uint32_t ROWS = EV_DEEP * THREADS / R::PIECES;  // positions of a batch
    const uint64_t page_bytes = (uint64_t)a.pg.n_kv * R::BLOCK;
    uint32_t src[EV_DEEP], now[EV_DEEP];  // of the next batch's rows, of this one's; a row that stays has itself
    int32_t ps[EV_DEEP], pd[EV_DEEP];
    auto row = [&](uint32_t u) { return (u * THREADS + threadIdx.x) / R::PIECES; };
    auto list = [&](uint32_t j0) {
#pragma unroll
        for (uint32_t u = 0; u < EV_DEEP; ++u) {
            const uint32_t r = row(u), j = j0 + r;
            src[u] = r < ROWS && j < a.n_keep ? (uint32_t)kept[j] : j;
        }
    };
    auto pages = [&](uint32_t j0) {
#pragma unroll
        for (uint32_t u = 0; u < EV_DEEP; ++u) {
            const uint32_t j = j0 + row(u);
            now[u] = src[u], ps[u] = pd[u] = -1;
            if (src[u] != j) ps[u] = table[src[u] / KV_PAGE], pd[u] = table[j / KV_PAGE];
        }
    };
    list(a.keep_first);
    pages(a.keep_first);
    list(a.keep_first + ROWS);
#pragma unroll 1
    for (uint32_t j0 = a.keep_first; j0 < a.n_keep; j0 += ROWS) {
        typename R::Word x[EV_DEEP];
        uint8_t *to[EV_DEEP];
        uint32_t at[EV_DEEP];
#pragma unroll
        for (uint32_t u = 0; u < EV_DEEP; ++u) {
            const uint32_t r = row(u), piece = u * THREADS + threadIdx.x - r * R::PIECES;
            to[u] = nullptr, at[u] = piece;
            if ((uint32_t)ps[u] >= a.pg.n_pages || (uint32_t)pd[u] >= a.pg.n_pages) continue;
            x[u] = R::load(pool + (uint32_t)ps[u] * page_bytes, value, now[u] % KV_PAGE, piece);
            to[u] = pool + (uint32_t)pd[u] * page_bytes;
        }
        pages(j0 + ROWS);
        list(j0 + 2 * ROWS);
        __syncthreads();  // a batch has been read before it is written; what the next one reads lies behind it
#pragma unroll
        for (uint32_t u = 0; u < EV_DEEP; ++u)
            if (to[u]) R::store(to[u], value, (j0 + row(u)) % KV_PAGE, at[u], x[u]);
    }
}

// Place of position x of a sequence, and of head 0 of its page: bytes, or all ones.
__device__ __forceinline__ bool kept_places(const PagedKeepArgs &a, uint32_t seq, uint32_t j, uint32_t &from, uint32_t &to) {
    const uint32_t n = min(a.n_kept[seq], a.kept_stride);
    if (j >= n) return false;
    const int32_t i = a.kept[(uint64_t)seq * a.kept_stride + j];
    const uint64_t ctx = a.n_ctx[seq], x = ctx + (uint32_t)i, y = ctx + j, room = (uint64_t)a.pg.stride * KV_PAGE;
    if ((uint32_t)i >= 64 || (uint32_t)i == j || x >= room || y >= room) return false;
    const int32_t *table = a.pg.tables + (uint64_t)seq * a.pg.stride;
    if ((uint32_t)table[x / KV_PAGE] >= a.pg.n_pages || (uint32_t)table[y / KV_PAGE] >= a.pg.n_pages) return false;
    from = (uint32_t)x, to = (uint32_t)y;
    return true;
}

// grid (sequences, layers x 2 x heads): all of a head's positions are read before the first is written.
template <int HD>
__global__ void __launch_bounds__(256) pages_keep_q4_kernel(const __grid_constant__ PagedKeepArgs a) {
    using R = Row4<HD>;
    pdl_release();
    pdl_wait();
    const uint32_t head = blockIdx.y % a.pg.n_kv, pool = blockIdx.y / a.pg.n_kv;
    const bool value = pool & 1;
    uint8_t *base = static_cast<uint8_t *>(const_cast<void *>(value ? a.pg.v : a.pg.k)) + (pool >> 1) * a.layer_bytes + (uint64_t)head * R::BLOCK;
    const uint64_t page_bytes = (uint64_t)a.pg.n_kv * R::BLOCK;
    const int32_t *table = a.pg.tables + (uint64_t)blockIdx.x * a.pg.stride;
    constexpr uint32_t TURNS = (64 * R::PIECES + 255) / 256;
    typename R::Word x[TURNS];
    uint32_t to[TURNS];
#pragma unroll
    for (uint32_t u = 0; u < TURNS; ++u) {
        const uint32_t i = u * 256 + threadIdx.x, j = i / R::PIECES;
        uint32_t from;
        if (!kept_places(a, blockIdx.x, j, from, to[u])) {
            to[u] = 0xffffffffu;
            continue;
        }
        x[u] = R::load(base + (uint32_t)table[from / KV_PAGE] * page_bytes, value, from % KV_PAGE, i - j * R::PIECES);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < TURNS; ++u) {
        const uint32_t i = u * 256 + threadIdx.x;
        if (to[u] != 0xffffffffu) R::store(base + (uint32_t)table[to[u] / KV_PAGE] * page_bytes, value, to[u] % KV_PAGE, i % R::PIECES, x[u]);
    }
}

// grid (sequences, layers x heads), a thread a position.
__global__ void __launch_bounds__(64) pages_keep_mass_kernel(const __grid_constant__ PagedKeepArgs a, float *mass, uint64_t stride, uint32_t n_seq) {
    pdl_release();
    pdl_wait();
    const uint32_t layer = blockIdx.y / a.pg.n_kv, head = blockIdx.y % a.pg.n_kv;
    float *row = mass + (((uint64_t)layer * n_seq + blockIdx.x) * a.pg.n_kv + head) * stride;
    uint32_t from, to;
    const bool moves = kept_places(a, blockIdx.x, threadIdx.x, from, to);
    const float x = moves ? row[from] : 0.0f;
    __syncthreads();
    if (moves) row[to] = x;
}

}  // namespace

cudaError_t launch_pages_evict(const PagedEvictArgs &a, uint32_t n_layer, uint32_t max_pos, bool q4, cudaStream_t st) {
    static PerDeviceOnce once;
    if (cudaError_t e = once.run([] {
            if (cudaError_t e = cudaFuncSetAttribute(pages_evict_choose_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_HELD * 4)) return e;
            return cudaFuncSetAttribute(pages_evict_choose_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_HELD * 4);
        }))
        return e;
    const uint32_t pairs = n_layer * a.n_seq * a.pg.n_kv, held = std::min({std::max(max_pos, 1u), a.pg.stride * KV_PAGE, EV_HELD});
    // Threads of the choice: 256 for short caches, many of which run at once, 1024 above.  2048 rows (32 layers of eight sequences, 8 heads of 128), the cut as a whole: of 200 positions 51 us
    // with 256 and 76 with 1024, of 600 114 and 99, of 2050 375 and 354, of 4100 828 and 673; 64 entries: of 600 74 and 82, of 1500 172 and 149.
    if (cudaError_t e = max_pos <= 1024 ? launch_pdl(pages_evict_choose_kernel<256>, dim3(pairs), dim3(256), (size_t)held * 4, st, a, held)
                                        : launch_pdl(pages_evict_choose_kernel<1024>, dim3(pairs), dim3(1024), (size_t)held * 4, st, a, held))
        return e;
    // Large CTAs for the moves where they are few: fewer batches, one after the other, of a head.  8 heads of 128, 128 rows of 4100 positions: 41 us with them and 69 with small ones, in 4 bits 53
    // and 111.  512 rows of 200: 21 and 17, 2048 rows of 1000: 162 and 188 (4 bits: 183 and 176), of 4100 619 and 673 (4 bits: 657 and 597).
    auto move = [&](auto small, auto large) {
        return pairs < 512 ? launch_pdl(large, dim3(pairs, 3), dim3(512), 0, st, a) : launch_pdl(small, dim3(pairs, 3), dim3(256), 0, st, a);
    };
    if (q4) return a.pg.dim == 64 ? move(pages_evict_move_kernel<Row4<64>, 256>, pages_evict_move_kernel<Row4<64>, 512>) : move(pages_evict_move_kernel<Row4<128>, 256>, pages_evict_move_kernel<Row4<128>, 512>);
    return a.pg.dim == 64 ? move(pages_evict_move_kernel<Row16<64>, 256>, pages_evict_move_kernel<Row16<64>, 512>) : move(pages_evict_move_kernel<Row16<128>, 256>, pages_evict_move_kernel<Row16<128>, 512>);
}
cudaError_t launch_pages_keep_q4(const PagedKeepArgs &a, uint32_t n_seq, uint32_t n_layer, cudaStream_t st) {
    return launch_pdl(a.pg.dim == 64 ? pages_keep_q4_kernel<64> : pages_keep_q4_kernel<128>, dim3(n_seq, 2 * n_layer * a.pg.n_kv), dim3(256), 0, st, a);
}
cudaError_t launch_pages_keep_mass(const PagedKeepArgs &a, uint32_t n_seq, uint32_t n_layer, float *mass, uint64_t stride, cudaStream_t st) {
    return launch_pdl(pages_keep_mass_kernel, dim3(n_seq, n_layer * a.pg.n_kv), dim3(64), 0, st, a, mass, stride, n_seq);
}

}  // namespace ob
