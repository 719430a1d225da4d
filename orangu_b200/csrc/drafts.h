// Verification of drafted tokens: what the entry point hands to the kernel of drafts.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ob {

constexpr uint32_t DRAFTS_MOST = 64;  // nodes of a tree

struct DraftsVerifyArgs {
    const void *target, *draft;  // [n_tokens][n_vocab] probabilities; draft may be null
    uint64_t target_stride, draft_stride;
    uint32_t n_vocab, n_tokens;
    const int32_t *tokens, *parent, *first;
    const float *uniform;
    int32_t *kept;               // [n_seq][kept_stride]
    uint32_t kept_stride;
    uint32_t *n_kept;
    int32_t *next;
};
cudaError_t launch_drafts_verify(const DraftsVerifyArgs &a, uint32_t n_seq, uint32_t type, int sm_count, cudaStream_t st);  // type: 0 f32, 1 f16, 2 bf16

}  // namespace ob
