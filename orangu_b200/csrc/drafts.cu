// Verification of drafted tokens (ob_drafts_verify): which of a tree's tokens are accepted, and the token after them, so that what comes out is distributed as if
// it had been drawn from the target alone.
//
// Node 0 is the last token that is certain.  At a node with target row p and draft row q its children, drawn from q, are tried in order; with c = 0 and T = 1 at first,
//   child x is accepted if u T q(x) < p(x) - c q(x);  otherwise c += T, T = sum_v max(p(v) - c q(v), 0)
// since the r-th residual max(r' - q, 0) / sum is max(p - c q, 0) / T.  Where no child is accepted the next token is the first v at which the sum of
// max(p - c q, 0) exceeds u_0 times all of it.  Without draft rows a drafted token had probability one: accepted if u T < p(x), otherwise p(x) = 0, T -= p(x).
//
// One chain of five, 128256 tokens: 12.5 us, of which three are loads that depend on each other; 64 trees of up to 16 nodes: 47 us, whose longest have
// rejected often.  16-bit rows take as long: conversions to 64 bits are the larger part of a sum.
//
// A cluster of CTAs per sequence: eight, or fewer where there are many sequences.  The numbers that the tests need, two a node, are read for all nodes at
// once; a path is then walked in shared memory, by every CTA for itself.  Rows of the vocabulary are read only where a child was rejected and for the last
// node, a part by each warp, and the parts' sums meet through distributed shared memory.  Sums are in 64 bits, so that the token does not depend on their order.
#include <cooperative_groups.h>

#include <algorithm>

#include "drafts.h"
#include "mixers_common.cuh"

namespace cg = cooperative_groups;

namespace ob {

namespace {

constexpr uint32_t DV_CTAS = 8 /* at most */, DV_THREADS = 512, DV_WARPS = DV_THREADS / 32, DV_PARTS = DV_CTAS * DV_WARPS, DV_DEEP = 4, DV_TILE = 1024;

__device__ __forceinline__ float number(float v) { return v; }
__device__ __forceinline__ float number(__half v) { return __half2float(v); }
__device__ __forceinline__ float number(bf16 v) { return __bfloat162float(v); }
// What is not a positive finite number counts as zero.
template <typename T> __device__ __forceinline__ double clean(T v) {
    const float f = number(v);
    return __float_as_uint(f) - 1u < 0x7f7fffffu ? (double)f : 0.0;
}
__device__ __forceinline__ double above(double w) { return __double2hiint(w) < 0 ? 0.0 : w; }  // max(w, 0)

// 16 bytes of a row as numbers.
template <typename T> struct Vec {
    static constexpr uint32_t N = 16 / sizeof(T);
    uint4 u;
    __device__ __forceinline__ T operator[](uint32_t i) const {
        const uint32_t w = i * sizeof(T) / 4 == 0 ? u.x : i * sizeof(T) / 4 == 1 ? u.y : i * sizeof(T) / 4 == 2 ? u.z : u.w;  // (i is known to the compiler)
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w);
        } else {
            const uint16_t h = (uint16_t)(i % 2 ? w >> 16 : w);
            return *reinterpret_cast<const T *>(&h);
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(DV_THREADS, 2) drafts_verify_kernel(const __grid_constant__ DraftsVerifyArgs a) {
    __shared__ double s_sum[2][DV_WARPS];  // of this CTA's parts, for the others; one after the other
    __shared__ double s_parts[DV_PARTS];   // of all
    __shared__ double s_tile[DV_TILE + DV_TILE / 32];  // weights of neighbouring tokens, 32 a lane
    __shared__ double s_p[DRAFTS_MOST], s_q[DRAFTS_MOST];  // of node i's token in its parent's rows
    __shared__ float s_u[DRAFTS_MOST];
    __shared__ int32_t s_parent[DRAFTS_MOST], s_token[DRAFTS_MOST], s_path[DRAFTS_MOST], s_gone[DRAFTS_MOST];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks(), n_parts = ctas * DV_WARPS, seq = blockIdx.x / ctas, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_release();
    pdl_wait();
    const int32_t f0 = a.first[seq], f1 = a.first[seq + 1];
    const bool any = f0 >= 0 && f1 > f0 && (uint32_t)f1 <= a.n_tokens;
    const uint32_t n = any ? min((uint32_t)(f1 - f0), DRAFTS_MOST) : 0u;
    const T *target = static_cast<const T *>(a.target) + (any ? (uint64_t)f0 * a.target_stride : 0ull);
    const T *draft = a.draft ? static_cast<const T *>(a.draft) + (any ? (uint64_t)f0 * a.draft_stride : 0ull) : nullptr;
    if (threadIdx.x < n) {
        const uint32_t i = threadIdx.x;
        const int32_t parent = i ? a.parent[f0 + i] : -1, token = i ? a.tokens[f0 + i] : -1;
        const bool known = parent >= 0 && (uint32_t)parent < i && (uint32_t)token < a.n_vocab;
        s_parent[i] = known ? parent : -1;
        s_token[i] = token;
        s_u[i] = a.uniform[f0 + i];
        s_p[i] = known ? clean(target[(uint64_t)parent * a.target_stride + token]) : 0.0;
        s_q[i] = known && draft ? clean(draft[(uint64_t)parent * a.draft_stride + token]) : 0.0;
    }
    __syncthreads();

    // weights of the vocabulary at a node: max(p - c q, 0), or p without the tokens that are gone
    const uint32_t span = (a.n_vocab + n_parts - 1) / n_parts, mine = rank * DV_WARPS + warp;
    uint32_t node = 0, n_path = 1, n_gone = 0;
    double c = 0.0, total = 1.0;
    bool summed = false;
    uint32_t turn = 0;
    auto weight = [&](const T *p, const T *q, uint32_t v) {
        const double x = clean(p[v]);
        if (q) return above(x - c * clean(q[v]));
        for (uint32_t i = 0; i < n_gone; ++i)
            if ((uint32_t)s_gone[i] == v) return 0.0;
        return x;
    };
    auto all_of = [&]() {  // the same order, and so the same sum, in every warp of the cluster
        double s = 0.0;
        for (uint32_t i = lane; i < n_parts; i += 32) s += s_parts[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    };
    auto sum_up = [&]() {  // parts of all CTAs in s_parts, in the order of the vocabulary
        const T *p = target + (uint64_t)node * a.target_stride, *q = draft && c > 0.0 ? draft + (uint64_t)node * a.draft_stride : nullptr;
        const uint32_t v0 = min(mine * span, a.n_vocab), v1 = min(v0 + span, a.n_vocab);
        double s = 0.0;
        auto one = [&](uint32_t v) { s += q ? above(clean(p[v]) - c * clean(q[v])) : clean(p[v]); };
        // 16 bytes a lane where both rows allow it (a whole span of them is 64 KB under way per CTA and row), single numbers elsewhere
        constexpr uint32_t N = Vec<T>::N;
        const uintptr_t pa = reinterpret_cast<uintptr_t>(p + v0), qa = q ? reinterpret_cast<uintptr_t>(q + v0) : pa;
        uint32_t from = v1, to = v1;  // what is read in vectors
        if (((pa ^ qa) & 15) == 0) {
            from = min(v1, v0 + (uint32_t)((16 - (pa & 15)) % 16 / sizeof(T)));
            to = from + (v1 - from) / N * N;
        }
        for (uint32_t v = v0 + lane; v < from; v += 32) one(v);
        for (uint32_t v = to + lane; v < v1; v += 32) one(v);
#pragma unroll 1
        for (uint32_t v = from + N * lane; v < to; v += 32 * N * DV_DEEP) {
            Vec<T> x[DV_DEEP], y[DV_DEEP];
#pragma unroll
            for (uint32_t u = 0; u < DV_DEEP; ++u) {
                x[u].u = y[u].u = make_uint4(0, 0, 0, 0);
                if (v + 32 * N * u < to) {
                    x[u].u = __ldg(reinterpret_cast<const uint4 *>(p + v + 32 * N * u));
                    if (q) y[u].u = __ldg(reinterpret_cast<const uint4 *>(q + v + 32 * N * u));
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < DV_DEEP; ++u)
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) s += q ? above(clean(x[u][i]) - c * clean(y[u][i])) : clean(x[u][i]);
        }
        for (uint32_t i = 0; i < n_gone; ++i) {  // (few, and each of them in one part only)
            const uint32_t v = (uint32_t)s_gone[i];
            if (v >= v0 && v < v1 && (v - v0) % 32 == lane) s -= clean(p[v]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) s_sum[turn][warp] = fmax(s, 0.0);
        cluster.sync();  // (between two writes of one place lies the other's sync, before which all have read this one's)
        if (threadIdx.x < n_parts) s_parts[threadIdx.x] = cluster.map_shared_rank(s_sum[turn], threadIdx.x / DV_WARPS)[threadIdx.x % DV_WARPS];
        turn ^= 1;
        __syncthreads();
        summed = true;
        return all_of();
    };
    if (threadIdx.x == 0 && n) s_path[0] = 0;
#pragma unroll 1
    for (uint32_t i = 1; i < n && n_path < a.kept_stride; ++i) {  // (a full list ends the path: what is drawn next follows its last node)
        if (s_parent[i] != (int32_t)node) continue;
        const double u = fmax((double)s_u[i], 0.0);
        double p = s_p[i];
        if (!draft)
            for (uint32_t k = 0; k < n_gone; ++k)
                if (s_gone[k] == s_token[i]) p = 0.0;
        if (draft ? u * total * s_q[i] < p - c * s_q[i] : u * total < p) {
            node = i, c = 0.0, total = 1.0, n_gone = 0, summed = false;
            __syncthreads();  // (s_gone is written again)
            if (threadIdx.x == 0) s_path[n_path] = (int32_t)i;
            ++n_path;
        } else if (draft) {
            if (total > 0.0) {
                c += total;
                total = sum_up();
            }
        } else if (p > 0.0) {
            total = fmax(total - p, 0.0);
            if (threadIdx.x == 0) s_gone[n_gone] = s_token[i];
            ++n_gone;
            summed = false;
            __syncthreads();
        }
    }
    // ---- the next token
    int32_t next = -1;
    if (n) {
        double all = 0.0;
        all = summed ? all_of() : sum_up();
        if (!(all > 0.0)) {  // nothing is left: the target's own row
            c = 0.0, n_gone = 0;
            all = sum_up();
        }
        if (all > 0.0) {
            const double r = fmax((double)s_u[0], 0.0) * all;
            // the part in which the sum passes r, each lane's parts being neighbours; rounding may leave none: the last one with anything
            constexpr uint32_t EACH = DV_PARTS / 32;
            double held[EACH], mine_sum = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < EACH; ++k) {
                const uint32_t i = lane * EACH + k;
                held[k] = i < n_parts ? s_parts[i] : 0.0;
                mine_sum += held[k];
            }
            double upto = mine_sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += x;
            }
            double start = __shfl_up_sync(0xffffffffu, upto, 1);
            if (lane == 0) start = 0.0;
            uint32_t part = 0;
            bool found = false;
#pragma unroll
            for (uint32_t k = 0; k < EACH; ++k)
                if (!found && held[k] > 0.0) {
                    part = lane * EACH + k;
                    found = start + held[k] > r;
                    if (!found) start += held[k];
                }
            const uint32_t hits = __ballot_sync(0xffffffffu, found), some = __ballot_sync(0xffffffffu, mine_sum > 0.0);
            const int src = hits ? __ffs(hits) - 1 : 31 - __clz(some);
            part = __shfl_sync(0xffffffffu, part, src), start = __shfl_sync(0xffffffffu, start, src);
            if (!hits) start = -INFINITY;  // (nothing passes r there: its last one)
            if (part / DV_WARPS == rank) {  // (alike for the whole CTA, which reads; its first warp looks for the token)
                const T *p = target + (uint64_t)node * a.target_stride, *q = draft && c > 0.0 ? draft + (uint64_t)node * a.draft_stride : nullptr;
                const uint32_t v0 = min(part * span, a.n_vocab), v1 = min(v0 + span, a.n_vocab);
                int32_t last = -1;
#pragma unroll 1
                for (uint32_t t0 = v0; t0 < v1; t0 += DV_TILE) {
                    __syncthreads();
#pragma unroll
                    for (uint32_t k = 0; k < DV_TILE / DV_THREADS; ++k) {
                        const uint32_t i = k * DV_THREADS + threadIdx.x, v = t0 + i;
                        s_tile[i / 32 * 33 + i % 32] = v < v1 ? weight(p, q, v) : 0.0;
                    }
                    __syncthreads();
                    if (warp || next >= 0) continue;
                    const double *own = s_tile + lane * 33;  // tokens t0 + 32 lane ..
                    double sum = 0.0;
#pragma unroll 8
                    for (uint32_t k = 0; k < 32; ++k) sum += own[k];
                    double upto = sum;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double x = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= (uint32_t)o) upto += x;
                    }
                    const uint32_t some = __ballot_sync(0xffffffffu, sum > 0.0), hit = __ballot_sync(0xffffffffu, sum > 0.0 && start + upto > r);
                    if (some) {
                        const int who = hit ? __ffs(hit) - 1 : 31 - __clz(some);
                        double at = __shfl_up_sync(0xffffffffu, upto, 1);
                        at = start + (lane ? at : 0.0);
                        int32_t mine_last = -1, mine_hit = -1;
                        if ((int)lane == who)
                            for (uint32_t k = 0; k < 32; ++k) {
                                if (!(own[k] > 0.0)) continue;
                                at += own[k];
                                mine_last = (int32_t)(t0 + lane * 32 + k);
                                if (hit && mine_hit < 0 && at > r) mine_hit = mine_last;
                            }
                        last = __shfl_sync(0xffffffffu, mine_last, who);
                        const int32_t h = __shfl_sync(0xffffffffu, mine_hit, who);
                        if (hit) next = h >= 0 ? h : last;
                    }
                    start += __shfl_sync(0xffffffffu, upto, 31);
                }
                if (threadIdx.x == 0) a.next[seq] = next < 0 ? last : next;
            }
        } else if (rank == 0 && threadIdx.x == 0) {
            a.next[seq] = -1;
        }
    } else if (rank == 0 && threadIdx.x == 0) {
        a.next[seq] = -1;
    }
    cluster.sync();  // (nobody's memory goes away while others may read it)
    if (rank == 0) {
        for (uint32_t j = threadIdx.x; j < a.kept_stride; j += DV_THREADS) a.kept[(uint64_t)seq * a.kept_stride + j] = n && j < n_path ? s_path[j] : -1;
        if (threadIdx.x == 0) a.n_kept[seq] = n ? n_path : 0u;
    }
}

}  // namespace

cudaError_t launch_drafts_verify(const DraftsVerifyArgs &a, uint32_t n_seq, uint32_t type, int sm_count, cudaStream_t st) {
    auto kernel = type == 0 ? drafts_verify_kernel<float> : type == 1 ? drafts_verify_kernel<__half> : drafts_verify_kernel<bf16>;
    // Two CTAs run on a multiprocessor at once; with up to twice as many, sequences that reject often still have all of them in the second round (64 trees of up to
    // 16 nodes: 46 us with eight CTAs each and 56 with four; chains of up to 8, which reject once, 22 and 17).
    uint32_t ctas = DV_CTAS;
    while (ctas > 1 && (uint64_t)n_seq * ctas > 4ull * sm_count) ctas /= 2;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = ctas, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(n_seq * ctas), cfg.blockDim = dim3(DV_THREADS), cfg.stream = st;
    cfg.attrs = at, cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace ob
