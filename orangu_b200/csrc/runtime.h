// Host-side state shared by the runtime translation units (internal).
#pragma once

#include <cuda_runtime.h>

#include <mutex>
#include <string>
#include <vector>

#include "../../include/orangu_b200.h"
#include "common.cuh"
#include "kernels.h"

using namespace ob;

struct Scratch {  // grow-only device buffer
    void *p = nullptr;
    size_t cap = 0;
};

struct PageWorkspace {  // of a handle of cache pages (pages.cu)
    uint8_t *mem;      // on the device
    uint32_t *status;  // pinned: set by a kernel that gave up a wait
};

struct ob_ctx {
    int device = 0;
    int sm_count = 0;
    cudaStream_t stream = nullptr;
    cudaEvent_t ev0 = nullptr, ev1 = nullptr;
    std::mutex mu;
    std::string err;
    uint64_t launches = 0;
    float last_ms = 0.0f;
    Scratch sx, sy, sq, sd, ss, sh, shs, sdt, saux, saux2, saux3;
    // Cache pages of callers (pages.cu): handles that are open, all workspaces that were made for handles, and those that no handle uses.
    std::mutex pages_mu;  // of the list and what its handles have not been told; taken for moments, after `mu` where both are
    std::vector<ob_pages *> pages;
    std::vector<PageWorkspace> page_workspaces, free_page_workspaces;
};

struct ob_weight {
    ob_ctx *ctx;
    DevWeight w;
    void *mem;
    uint64_t bytes;
    WideRows wide;
};

namespace obrt {

int fail(ob_ctx *ctx, int code, const std::string &msg);
int ensure(ob_ctx *ctx, Scratch &s, size_t bytes);
bool type_supported(uint32_t t);

#define OB_CUDA(ctx, expr)                                                                                  \
    do {                                                                                                    \
        cudaError_t e__ = (expr);                                                                           \
        if (e__ != cudaSuccess) {                                                                           \
            return obrt::fail(ctx, e__ == cudaErrorMemoryAllocation ? OB_ERR_OOM : OB_ERR_CUDA,             \
                              std::string(#expr) + ": " + cudaGetErrorString(e__));                         \
        }                                                                                                   \
    } while (0)

struct Bind {  // makes the context's device current for the scope of a call
    int prev = -1;
    explicit Bind(const ob_ctx *c) {
        cudaGetDevice(&prev);
        if (prev != c->device) cudaSetDevice(c->device);
        else prev = -1;
    }
    ~Bind() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

bool pages_gave_up(ob_ctx *ctx);  // whether a call on one of the context's handles of cache pages gave up a wait since this was last asked
void close_pages(ob_ctx *ctx);    // before the context goes: its handles of cache pages refuse every call from then on

// Uploads (a slice of) a GGUF matrix and re-lays it for the kernels; see DevWeight.
int make_weight(ob_ctx *ctx, const uint8_t *raw, uint64_t row_bytes, uint32_t type, uint32_t in_dim, uint32_t out_dim, uint32_t row0,
                uint32_t n_rows, uint32_t col0, uint32_t n_cols, ob_weight **out);

}  // namespace obrt
