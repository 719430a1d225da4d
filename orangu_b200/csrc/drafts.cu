// Verification of drafted tokens (ob_drafts_verify): which of a tree's tokens are accepted, and the token after them, so that what comes out is distributed as if
// it had been drawn from the target alone.
//
// Node 0 is the last token that is certain.  At a node with target row p and draft row q its children, drawn from q, are tried in order; with c = 0 and T = 1 at first,
//   child x is accepted if u T q(x) < p(x) - c q(x);  otherwise c += T, T = sum_v max(p(v) - c q(v), 0)
// since the r-th residual max(r' - q, 0) / sum is max(p - c q, 0) / T.  Where no child is accepted the next token is the first v at which the sum of
// max(p - c q, 0) exceeds u_0 times all of it.  Without draft rows a drafted token had probability one: accepted if u T < p(x), otherwise p(x) = 0, T -= p(x).
//
// A cluster of CTAs per sequence: eight, or as many fewer as let all sequences run at once.  The numbers that the tests need, two a node, are read for all nodes at
// once; a path is then walked in shared memory, by every CTA for itself.  Rows of the vocabulary are read only where a child was rejected and for the last
// node, a part by each warp, and the parts' sums meet through distributed shared memory.  Sums are in 64 bits, so that the token does not depend on their order.
#include <cooperative_groups.h>

#include <algorithm>

#include "drafts.h"
#include "mixers_common.cuh"

namespace cg = cooperative_groups;

namespace ob {

namespace {

constexpr uint32_t DV_CTAS = 8 /* at most */, DV_THREADS = 512, DV_WARPS = DV_THREADS / 32, DV_PARTS = DV_CTAS * DV_WARPS, DV_DEEP = 8, DV_TILE = 1024;

__device__ __forceinline__ float number(float v) { return v; }
__device__ __forceinline__ float number(__half v) { return __half2float(v); }
__device__ __forceinline__ float number(bf16 v) { return __bfloat162float(v); }
// What is not a positive finite number counts as zero.
template <typename T> __device__ __forceinline__ double clean(T v) {
    const float f = number(v);
    return f > 0.0f && f <= 3.4028234664e38f ? (double)f : 0.0;
}

template <typename T>
__global__ void __launch_bounds__(DV_THREADS, 2) drafts_verify_kernel(const __grid_constant__ DraftsVerifyArgs a) {
    __shared__ double s_sum[DV_WARPS];     // of this CTA's parts, for the others
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
    auto weight = [&](const T *p, const T *q, uint32_t v) {
        const double x = clean(p[v]);
        if (q) return fmax(x - c * clean(q[v]), 0.0);
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
#pragma unroll 1
        for (uint32_t v = v0 + lane; v < v1; v += 32 * DV_DEEP) {
            T x[DV_DEEP], y[DV_DEEP];
#pragma unroll
            for (uint32_t u = 0; u < DV_DEEP; ++u) {
                x[u] = y[u] = T(0.0f);
                if (v + 32 * u < v1) {
                    x[u] = p[v + 32 * u];
                    if (q) y[u] = q[v + 32 * u];
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < DV_DEEP; ++u) s += q ? fmax(clean(x[u]) - c * clean(y[u]), 0.0) : clean(x[u]);
        }
        for (uint32_t i = 0; i < n_gone; ++i) {  // (few, and each of them in one part only)
            const uint32_t v = (uint32_t)s_gone[i];
            if (v >= v0 && v < v1 && (v - v0) % 32 == lane) s -= clean(p[v]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) s_sum[warp] = fmax(s, 0.0);
        cluster.sync();
        if (threadIdx.x < n_parts) s_parts[threadIdx.x] = cluster.map_shared_rank(s_sum, threadIdx.x / DV_WARPS)[threadIdx.x % DV_WARPS];
        cluster.sync();  // (all have read before anybody's sums are written again, or its memory goes away)
        summed = true;
        return all_of();
    };
    if (threadIdx.x == 0 && n) s_path[0] = 0;
#pragma unroll 1
    for (uint32_t i = 1; i < n; ++i) {
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
            if (part == mine) {
                const T *p = target + (uint64_t)node * a.target_stride, *q = draft && c > 0.0 ? draft + (uint64_t)node * a.draft_stride : nullptr;
                const uint32_t v0 = min(part * span, a.n_vocab), v1 = min(v0 + span, a.n_vocab);
                int32_t last = -1;
#pragma unroll 1
                for (uint32_t t0 = v0; t0 < v1 && next < 0; t0 += DV_TILE) {
                    __syncwarp();
#pragma unroll 8
                    for (uint32_t k = 0; k < DV_TILE / 32; ++k) {
                        const uint32_t v = t0 + k * 32 + lane;
                        s_tile[k * 33 + lane] = v < v1 ? weight(p, q, v) : 0.0;
                    }
                    __syncwarp();
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
                if (next < 0) next = last;
                if (lane == 0) a.next[seq] = next;
            }
        } else if (rank == 0 && threadIdx.x == 0) {
            a.next[seq] = -1;
        }
    } else if (rank == 0 && threadIdx.x == 0) {
        a.next[seq] = -1;
    }
    if (rank == 0) {
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < a.kept_stride; j += DV_THREADS) a.kept[(uint64_t)seq * a.kept_stride + j] = n && j < n_path ? s_path[j] : -1;
        if (threadIdx.x == 0) a.n_kept[seq] = n ? min(n_path, a.kept_stride) : 0u;
    }
}

}  // namespace

cudaError_t launch_drafts_verify(const DraftsVerifyArgs &a, uint32_t n_seq, uint32_t type, int sm_count, cudaStream_t st) {
    auto kernel = type == 0 ? drafts_verify_kernel<float> : type == 1 ? drafts_verify_kernel<__half> : drafts_verify_kernel<bf16>;
    uint32_t ctas = DV_CTAS;  // two a multiprocessor at once
    while (ctas > 1 && (uint64_t)n_seq * ctas > 2ull * sm_count) ctas /= 2;
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
