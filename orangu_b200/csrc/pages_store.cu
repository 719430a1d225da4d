// Pages in 4 bits (layout: pages_q4.cuh): new keys and values become codes and units (ob_pages_store), and positions become rows again (ob_pages_load).
//
//   m = the entry of largest magnitude of 32 (of equal ones the negative one), d = -m / 8 made larger to 7 significant bits (and a multiple of 2^-24), c = rint(x / d) from -8 to 7
//
// so that m itself is -8 d or a little less.  No number counts as 0, and magnitudes above 7168 as 7168, which keeps d an f16 number and every entry c d one, too.
// The quotient comes from a product with about 1 / d; where that lies near the middle between two codes the division is done.
//
// Half a warp has a key's or value's 128 entries, eight a lane (a quarter 64).
#include <algorithm>

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

// Where position n_ctx[seq] + j lies, if row j of the sequence is to be moved: page, position within it, row.
struct PgPlace {
    bool there;
    uint32_t page, p;
    uint64_t row;
};
__device__ __forceinline__ PgPlace place(const PagedMoveArgs &a, uint32_t seq, uint32_t j) {
    const int32_t f0 = a.first[seq], f1 = a.first[seq + 1];
    const uint64_t x = (uint64_t)a.n_ctx[seq] + j;
    PgPlace at{false, 0, (uint32_t)x % KV_PAGE, (uint64_t)(uint32_t)f0 + j};
    if (f0 < 0 || f1 <= f0 || (uint32_t)f1 > a.n_tokens || j >= (uint32_t)(f1 - f0) || j >= a.max_tokens || x >= (uint64_t)a.pg.stride * KV_PAGE) return at;
    const int32_t id = a.pg.tables[(uint64_t)seq * a.pg.stride + x / KV_PAGE];
    at.there = (uint32_t)id < a.pg.n_pages;
    at.page = (uint32_t)id;
    return at;
}

// grid (rows of all heads, keys and values / rows of a CTA, sequences).
template <typename T, int HD>
__global__ void __launch_bounds__(256) pages_store_kernel(const __grid_constant__ PagedMoveArgs a) {
    using B = Q4Block<HD>;
    constexpr uint32_t LANES = HD / 8, ROWS = 256 / LANES;
    pdl_release();
    pdl_wait();
    const uint32_t seq = blockIdx.y, w = threadIdx.x % LANES, per = 2 * a.pg.n_kv;
    const uint64_t i = (uint64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
    const uint32_t j = (uint32_t)(i / per), part = (uint32_t)(i % per), value = part / a.pg.n_kv, head = part % a.pg.n_kv;
    const PgPlace at = place(a, seq, j);
    const T *src = static_cast<const T *>(value ? a.v : a.k) + at.row * (value ? a.v_stride : a.k_stride) + (uint64_t)head * HD + w * 8;
    const uint4 u = at.there ? *reinterpret_cast<const uint4 *>(src) : make_uint4(0, 0, 0, 0);
    const uint32_t word[4] = {u.x, u.y, u.z, u.w};
    float x[8], most = 0.0f, least = 0.0f;  // (a group whose entries all have one sign: the other end stays zero)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = as_float2(word[e], T());
        x[2 * e] = f.x, x[2 * e + 1] = f.y;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -Q4_LARGEST), Q4_LARGEST);
        most = fmaxf(most, x[e]), least = fminf(least, x[e]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    const float eighth = fmaxf(most, -least) * 0.125f;
    // up to 7 significant bits; below 2^-18 to a multiple of 2^-24, the steps of f16 (a magnitude below 64 2^-24: its whole number of them)
    float d = __uint_as_float((__float_as_uint(eighth) + 0x1ffffu) & ~0x1ffffu);
    if (eighth < 0x1p-18f) d = ceilf(eighth * 0x1p24f) * 0x1p-24f;
    if (most > -least) d = -d;
    const float by = d != 0.0f ? d : 1.0f, inverse = __frcp_rn(by);
    uint32_t out = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float t = x[e] * inverse;  // off by less than 2^-20 (8 times 2^-23)
        const float near = rintf(t);
        if (fabsf(t - near) > 0.4999f) t = __fdiv_rn(x[e], by);
        const int c = max(-8, min(7, (int)rintf(t)));
        out |= (uint32_t)(c + 8) << (4 * (e >> 1) + 16 * (e & 1));
    }
    if (!at.there) return;
    uint8_t *block = static_cast<uint8_t *>(const_cast<void *>(value ? a.pg.v : a.pg.k)) + ((uint64_t)at.page * a.pg.n_kv + head) * B::BYTES;
    *reinterpret_cast<uint32_t *>(block + B::word(value, at.p, w)) = out;
    if (w % 4 == 0) *reinterpret_cast<__half *>(block + B::unit(value, at.p, w / 4)) = __float2half_rn(d);
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) pages_load_kernel(const __grid_constant__ PagedMoveArgs a) {
    using B = Q4Block<HD>;
    constexpr uint32_t LANES = HD / 8, ROWS = 256 / LANES;
    pdl_release();
    pdl_wait();
    const uint32_t seq = blockIdx.y, w = threadIdx.x % LANES, per = 2 * a.pg.n_kv;
    const uint64_t i = (uint64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
    const uint32_t j = (uint32_t)(i / per), part = (uint32_t)(i % per), value = part / a.pg.n_kv, head = part % a.pg.n_kv;
    const PgPlace at = place(a, seq, j);
    if (!at.there) return;
    const uint8_t *block = static_cast<const uint8_t *>(value ? a.pg.v : a.pg.k) + ((uint64_t)at.page * a.pg.n_kv + head) * B::BYTES;
    const uint32_t code = *reinterpret_cast<const uint32_t *>(block + B::word(value, at.p, w));
    const float d = __half2float(*reinterpret_cast<const __half *>(block + B::unit(value, at.p, w / 4)));
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = pack2((float)((int)(code >> (4 * e) & 15u) - 8) * d, (float)((int)(code >> (4 * e + 16) & 15u) - 8) * d, T());
    T *dst = static_cast<T *>(const_cast<void *>(value ? a.v : a.k)) + at.row * (value ? a.v_stride : a.k_stride) + (uint64_t)head * HD + w * 8;
    *reinterpret_cast<uint4 *>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
}

}  // namespace

cudaError_t launch_pages_store(const PagedMoveArgs &a, bool is_bf16, bool load, cudaStream_t st) {
    const uint32_t rows = 256 / (a.pg.dim / 8);
    const dim3 grid((uint32_t)(((uint64_t)a.max_tokens * 2 * a.pg.n_kv + rows - 1) / rows), a.n_seq);
    auto pick = [&](auto k64, auto k128) { return launch_pdl(a.pg.dim == 64 ? k64 : k128, grid, dim3(256), 0, st, a); };
    if (load) return is_bf16 ? pick(pages_load_kernel<bf16, 64>, pages_load_kernel<bf16, 128>) : pick(pages_load_kernel<__half, 64>, pages_load_kernel<__half, 128>);
    return is_bf16 ? pick(pages_store_kernel<bf16, 64>, pages_store_kernel<bf16, 128>) : pick(pages_store_kernel<__half, 64>, pages_store_kernel<__half, 128>);
}

}  // namespace ob
