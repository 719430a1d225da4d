// Pages in 4 bits (layout: pages_q4.cuh): new keys and values become codes and units (ob_pages_store), and positions become rows again (ob_pages_load).
//
//   m = the entry of largest magnitude of 32 (of equal ones the negative one), d = -m / 8 made larger to 7 significant bits (and a multiple of 2^-24), c = rint(x / d) from -8 to 7
//
// so that m itself is -8 d or a little less.  No number counts as 0, and magnitudes above 7168 as 7168, which keeps d an f16 number and every entry c d one, too.
// The quotient is a product with about 1 / d and one step of Newton's, so that ties are ties.
//
// Half a warp has a key's or value's 128 entries, eight a lane (a quarter 64), the same place of several pages.  The arithmetic is the larger part of storing: 167
// instructions for eight entries, issued in 77 % of the slots (loading: 82, which wait for their loads).  Maxima are taken two at a time in the rows' type; codes are whole numbers in the low bits of a sum with 1.5 2^23, put together as
// one number of base 16 by fused multiply-adds.
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "mixers_common.cuh"
#include "pages.h"
#include "pages_q4.cuh"

namespace ob {

namespace {

__device__ __forceinline__ float2 as_float2(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
__device__ __forceinline__ float2 as_float2(uint32_t u, bf16) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {  // no number if either is none
        uint32_t d;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
};
template <> struct Pair<bf16> {
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
};
constexpr uint32_t SIGNS = 0x80008000u;

// What a group of lanes has: one head's keys or values, positions `pos`, `pos` + `step`, ... of the sequence.  P neighbouring groups have P neighbouring positions, from a
// multiple of P on.
struct PgRows {
    uint32_t head, pos, step, ctx, end;  // new positions: from ctx to end
    bool value;
    int32_t first;
    const int32_t *table;
};
template <uint32_t GROUPS, uint32_t P>
__device__ __forceinline__ PgRows rows_of(const PagedMoveArgs &a, uint32_t group) {
    PgRows r;
    constexpr uint32_t SETS = GROUPS / P;  // of a CTA
    const uint32_t per = 2 * a.pg.n_kv, i = blockIdx.x * SETS + group / P, part = i % per, seq = blockIdx.y;
    const int32_t f0 = a.first[seq], f1 = a.first[seq + 1];
    const uint32_t room = a.pg.stride * KV_PAGE;
    r.ctx = a.n_ctx[seq], r.first = f0;
    r.end = f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens || r.ctx >= room ? 0u : r.ctx + min(min((uint32_t)(f1 - f0), a.max_tokens), room - r.ctx);
    r.pos = r.ctx / P * P + i / per * P + group % P, r.step = gridDim.x * SETS / per * P;  // (the grid is made so that there is no remainder)
    r.value = part >= a.pg.n_kv, r.head = r.value ? part - a.pg.n_kv : part;
    r.table = a.pg.tables + (uint64_t)seq * a.pg.stride;
    return r;
}
__device__ __forceinline__ int32_t page_of(const PagedMoveArgs &a, const PgRows &r, uint32_t pos) {
    const int32_t id = pos >= r.ctx && pos < r.end ? r.table[pos / KV_PAGE] : -1;
    return (uint32_t)id < a.pg.n_pages ? id : -1;
}

constexpr uint32_t ST_DEEP = 2;  // rows of a lane under way

// grid (sets of P positions x heads x keys and values, sequences).  With P = 16 a page's positions of one head are a CTA's (two pages with head dimension 64), so that
// its sectors are read and written together: 32000 rows of 8 heads of 128 take 82 us to store and to load again (floor 51), with P = 1 101.  That is for few
// positions: a step of 64 sequences takes 3.5 and 5 us then, and 7 each with P = 16.
template <typename T, int HD, uint32_t P>
__global__ void __launch_bounds__(256) pages_store_kernel(const __grid_constant__ PagedMoveArgs a) {
    using B = Q4Block<HD>;
    constexpr uint32_t LANES = HD / 8, ROWS = 256 / LANES;
    pdl_release();
    pdl_wait();
    const uint32_t w = threadIdx.x % LANES;
    const PgRows r = rows_of<ROWS, P>(a, threadIdx.x / LANES);
    const T *src = static_cast<const T *>(r.value ? a.v : a.k) + (uint64_t)(uint32_t)r.first * (r.value ? a.v_stride : a.k_stride) + (uint64_t)r.head * HD + w * 8;
    const uint64_t stride = r.value ? a.v_stride : a.k_stride;
    uint8_t *pool = static_cast<uint8_t *>(const_cast<void *>(r.value ? a.pg.v : a.pg.k)) + (uint64_t)r.head * B::BYTES;
    const uint64_t page_bytes = (uint64_t)a.pg.n_kv * B::BYTES;
    constexpr uint32_t lanes = 0xffffffffu;  // (a warp's groups go on as long as one of them has rows)
    for (uint32_t pos = r.pos; __any_sync(lanes, pos < r.end); pos += ST_DEEP * r.step) {
        uint4 u[ST_DEEP];
        int32_t id[ST_DEEP];
#pragma unroll
        for (uint32_t k = 0; k < ST_DEEP; ++k) {
            const uint32_t x = pos + k * r.step;
            u[k] = make_uint4(0, 0, 0, 0);
            if (x >= r.ctx && x < r.end) u[k] = ldg128_stream(src + (x - r.ctx) * stride);
            id[k] = page_of(a, r, x);
        }
#pragma unroll
        for (uint32_t k = 0; k < ST_DEEP; ++k) {
            const uint32_t word[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
            uint32_t hi = Pair<T>::max(Pair<T>::max(word[0], word[1]), Pair<T>::max(word[2], word[3]));
            uint32_t lo = Pair<T>::max(Pair<T>::max(word[0] ^ SIGNS, word[1] ^ SIGNS), Pair<T>::max(word[2] ^ SIGNS, word[3] ^ SIGNS));
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                hi = Pair<T>::max(hi, __shfl_xor_sync(lanes, hi, o));
                lo = Pair<T>::max(lo, __shfl_xor_sync(lanes, lo, o));
            }
            const float2 hi2 = as_float2(hi, T()), lo2 = as_float2(lo, T());
            float most = fmaxf(hi2.x, hi2.y), least = fmaxf(lo2.x, lo2.y), x[8];  // the largest, and the smallest with its sign turned
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = as_float2(word[e], T());
                x[2 * e] = f.x, x[2 * e + 1] = f.y;
            }
            const bool odd = !(fmaxf(most, least) <= Q4_LARGEST) || hi2.x != hi2.x || hi2.y != hi2.y;  // no numbers, or too large ones, in these 32
            if (__any_sync(lanes, odd)) {
                most = least = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -Q4_LARGEST), Q4_LARGEST);
                    most = fmaxf(most, x[e]), least = fmaxf(least, -x[e]);
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    most = fmaxf(most, __shfl_xor_sync(lanes, most, o));
                    least = fmaxf(least, __shfl_xor_sync(lanes, least, o));
                }
            }
            const float eighth = fmaxf(most, least) * 0.125f;
            // up to 7 significant bits; below 2^-18 to a multiple of 2^-24, the steps of f16
            float d = __uint_as_float((__float_as_uint(eighth) + 0x1ffffu) & ~0x1ffffu);
            if (__builtin_expect(eighth < 0x1p-18f, 0)) d = ceilf(eighth * 0x1p24f) * 0x1p-24f;
            if (most > least) d = -d;
            const float by = d != 0.0f ? d : 1.0f;
            float inverse, c[8];
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(by));
            constexpr float MAGIC = 12582912.0f;  // 1.5 2^23: adding it rounds to whole numbers, ties to even
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // a product with about 1 / d, and what is left over (exact: 11 bits less 4 times 7) once more: a quotient of 5 bits, as one in the middle between two codes is,
                // comes out as it is, and any other is further from the middle (2^-12 of it) than it is off (2^-23)
                const float q = x[e] * inverse;
                c[e] = fminf((fmaf(fmaf(-q, by, x[e]), inverse, q) + MAGIC) - MAGIC, 7.0f);
            }
            // c + 8 in base 16: even entries in the low half, odd ones in the high half
            constexpr float EIGHTS = 8.0f * 0x1111;
            const float low = fmaf(fmaf(fmaf(c[6], 16.0f, c[4]), 16.0f, c[2]), 16.0f, c[0]) + (EIGHTS + MAGIC), high = fmaf(fmaf(fmaf(c[7], 16.0f, c[5]), 16.0f, c[3]), 16.0f, c[1]) + (EIGHTS + MAGIC);
            if (id[k] < 0) continue;
            const uint32_t p = (pos + k * r.step) % KV_PAGE;
            uint8_t *block = pool + (uint32_t)id[k] * page_bytes;
            if (r.value) {
                uint16_t *at = reinterpret_cast<uint16_t *>(block + B::value(p, w));
                at[0] = (uint16_t)__float_as_uint(low), at[2] = (uint16_t)__float_as_uint(high);
            } else {
                *reinterpret_cast<uint32_t *>(block + B::key(p, w)) = __byte_perm(__float_as_uint(low), __float_as_uint(high), 0x5410);
            }
            if (w % 4 == 0) *reinterpret_cast<__half *>(block + B::unit(r.value, p, w / 4)) = __float2half_rn(d);
        }
    }
}

constexpr uint32_t LD_DEEP = 4;
template <typename T, int HD, uint32_t P>
__global__ void __launch_bounds__(256) pages_load_kernel(const __grid_constant__ PagedMoveArgs a) {
    using B = Q4Block<HD>;
    constexpr uint32_t LANES = HD / 8, ROWS = 256 / LANES;
    pdl_release();
    pdl_wait();
    const uint32_t w = threadIdx.x % LANES;
    const PgRows r = rows_of<ROWS, P>(a, threadIdx.x / LANES);
    T *dst = static_cast<T *>(const_cast<void *>(r.value ? a.v : a.k)) + (uint64_t)(uint32_t)r.first * (r.value ? a.v_stride : a.k_stride) + (uint64_t)r.head * HD + w * 8;
    const uint64_t stride = r.value ? a.v_stride : a.k_stride;
    const uint8_t *pool = static_cast<const uint8_t *>(r.value ? a.pg.v : a.pg.k) + (uint64_t)r.head * B::BYTES;
    const uint64_t page_bytes = (uint64_t)a.pg.n_kv * B::BYTES;
    for (uint32_t pos = r.pos; pos < r.end; pos += LD_DEEP * r.step) {
        uint32_t code[LD_DEEP], unit[LD_DEEP];
        int32_t id[LD_DEEP];
#pragma unroll
        for (uint32_t k = 0; k < LD_DEEP; ++k) id[k] = page_of(a, r, pos + k * r.step);
#pragma unroll
        for (uint32_t k = 0; k < LD_DEEP; ++k) {
            const uint32_t p = (pos + k * r.step) % KV_PAGE;
            const uint8_t *block = pool + (uint32_t)max(id[k], 0) * page_bytes;
            code[k] = unit[k] = 0;
            if (id[k] < 0) continue;
            if (r.value) {
                const uint16_t *at = reinterpret_cast<const uint16_t *>(block + B::value(p, w));
                code[k] = at[0] | (uint32_t)at[2] << 16;
            } else {
                code[k] = *reinterpret_cast<const uint32_t *>(block + B::key(p, w));
            }
            unit[k] = *reinterpret_cast<const uint16_t *>(block + B::unit(r.value, p, w / 4));
        }
#pragma unroll
        for (uint32_t k = 0; k < LD_DEEP; ++k) {
            if (id[k] < 0) continue;
            const uint32_t d = unit[k] * 0x10001u, n = q4_offset(d);
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u[e] = q4_field(code[k], e, d, n);
                if constexpr (!std::is_same<T, __half>::value) {
                    const float2 f = as_float2(u[e], __half());
                    u[e] = pack2(f.x, f.y, T());
                }
            }
            __stcs(reinterpret_cast<uint4 *>(dst + (pos + k * r.step - r.ctx) * stride), make_uint4(u[0], u[1], u[2], u[3]));
        }
    }
}

}  // namespace

cudaError_t launch_pages_store(const PagedMoveArgs &a, bool is_bf16, bool load, int sm_count, cudaStream_t st) {
    // Whole rounds of (head, keys or values), and CTAs for all places (eight an SM); fewer where there are few positions.
    const bool whole = a.max_tokens >= KV_PAGE;  // pages
    const uint32_t positions = whole ? KV_PAGE : 1, sets = 256 / (a.pg.dim / 8) / positions, per = 2 * a.pg.n_kv, round = per / std::gcd(per, sets);
    const uint64_t all = (((uint64_t)(a.max_tokens - 1) / positions + whole + 1) * per + sets - 1) / sets, most = std::max<uint64_t>(1, 8ull * sm_count / a.n_seq);  // (positions that do not begin a page touch one more)
    const dim3 grid((uint32_t)((std::min(all, most) + round - 1) / round * round), a.n_seq);
    auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(256), 0, st, a); };
    auto dim = [&](auto type, auto p) {
        using T = decltype(type);
        constexpr uint32_t P = decltype(p)::value;
        if (load) return a.pg.dim == 64 ? go(pages_load_kernel<T, 64, P>) : go(pages_load_kernel<T, 128, P>);
        return a.pg.dim == 64 ? go(pages_store_kernel<T, 64, P>) : go(pages_store_kernel<T, 128, P>);
    };
    auto pick = [&](auto type) { return whole ? dim(type, std::integral_constant<uint32_t, KV_PAGE>()) : dim(type, std::integral_constant<uint32_t, 1>()); };
    return is_bf16 ? pick(bf16()) : pick(__half());
}

}  // namespace ob
