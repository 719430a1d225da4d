// The picking half of the choice of pages (pages_select.cu): which of a row's words are the largest.  A file of its own, with nothing of CUDA's
// headers in it, so that its barriers can be checked on the CPU, too (tests/pages_pick_host.cpp).
#pragma once

namespace ob {

namespace {

constexpr uint32_t SEL_BINS = 2048;
constexpr uint32_t SEL_FORCED = 0xffffffffu;

// Sum over the warps before this one; every thread gets it.  parts: a word per warp.
template <uint32_t NW>
__device__ __forceinline__ uint32_t warps_before(uint32_t mine, uint32_t *parts) {  // mine: the warp's, on every lane
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) parts[warp] = mine;
    __syncthreads();
    const uint32_t v = lane < NW ? parts[lane] : 0u;
    return (uint32_t)warp_sum_i(lane < warp ? (int)v : 0);
}

// The places of all words above and of the `want` largest in [lo, hi], in ascending order, the first of equals: lo and hi are the smallest and the
// largest word that is not SEL_FORCED, as far as this thread has seen, and more than `want` words are not.  The whole CTA, once.
// keys: anything that keys[i] gives the word of place i of.
template <uint32_t THREADS, typename K>
__device__ __forceinline__ void pick(uint32_t want, K keys, uint32_t n, uint32_t lo, uint32_t hi, int32_t *out) {
    constexpr uint32_t NW = THREADS / 32, BINS = SEL_BINS / THREADS;  // bins of a thread
    __shared__ uint32_t s_hist[SEL_BINS], s_parts[5][32], s_pick[3];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) s_parts[0][warp] = lo, s_parts[1][warp] = hi;
    __syncthreads();  // (the words are written, too)
    lo = __reduce_min_sync(0xffffffffu, lane < NW ? s_parts[0][lane] : 0xffffffffu);
    hi = __reduce_max_sync(0xffffffffu, lane < NW ? s_parts[1][lane] : 0u);

    // ---- the border: of the words in [lo, hi], `want` are taken, of those above all
    bool all = want == 0;  // all words from lo on
    if (all) lo = hi = SEL_FORCED;
    while (!all && lo < hi) {
        const int shift = max(0, 32 - __clz(hi - lo) - 11);  // (hi - lo) >> shift is below 2048
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < SEL_BINS; i += THREADS) s_hist[i] = 0u;
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            const uint32_t k = keys[i];
            if (k >= lo && k <= hi) atomicAdd(s_hist + ((k - lo) >> shift), 1u);
        }
        __syncthreads();
        const uint32_t bin0 = SEL_BINS - 1 - threadIdx.x * BINS;  // this thread's bins: bin0, bin0 - 1, ...
        uint32_t count[BINS], mine = 0;
#pragma unroll
        for (uint32_t i = 0; i < BINS; ++i) mine += count[i] = s_hist[bin0 - i];
        uint32_t upto = mine;  // words of this warp's bins up to this thread's
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += up;
        }
        uint32_t above = warps_before<NW>(__shfl_sync(0xffffffffu, upto, 31), s_parts[2]) + upto - mine;
#pragma unroll
        for (uint32_t i = 0; i < BINS; ++i) {
            if (above < want && above + count[i] >= want) s_pick[0] = bin0 - i, s_pick[1] = want - above, s_pick[2] = count[i];
            above += count[i];
        }
        __syncthreads();
        lo += s_pick[0] << shift;
        hi = min(hi, lo + (1u << shift) - 1);
        want = s_pick[1];
        all = want == s_pick[2];
        __syncthreads();
    }
    // ---- the list: words above hi, all in [lo, hi] or the first `want` of them (which are equal then)
    const uint32_t span = (n + NW - 1) / NW, w0 = min(warp * span, n), w1 = min(w0 + span, n);  // this warp's pages
    uint32_t above = 0, equal = 0;
    auto kinds = [&](uint32_t i, bool &gt, bool &eq) {
        const uint32_t k = i < w1 ? keys[i] : 0u;
        gt = i < w1 && (all ? k >= lo : k > hi);
        eq = i < w1 && !all && k == lo;
    };
#pragma unroll 1
    for (uint32_t i = w0; i < w1; i += 32) {
        bool gt, eq;
        kinds(i + lane, gt, eq);
        above += __popc(__ballot_sync(0xffffffffu, gt)), equal += __popc(__ballot_sync(0xffffffffu, eq));
    }
    above = warps_before<NW>(above, s_parts[3]);  // (places of their own: where all words are equal no barrier lies between these and the first ones' reading)
    equal = warps_before<NW>(equal, s_parts[4]);
#pragma unroll 1
    for (uint32_t i = w0; i < w1; i += 32) {
        bool gt, eq;
        kinds(i + lane, gt, eq);
        const uint32_t g = __ballot_sync(0xffffffffu, gt), q = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
        const uint32_t ga = above + __popc(g & below), ea = equal + __popc(q & below);
        if (gt || (eq && ea < want)) out[ga + min(ea, want)] = (int32_t)(i + lane);
        above += __popc(g), equal += __popc(q);
    }
}

}  // namespace

}  // namespace ob
