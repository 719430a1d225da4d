// Operators over the pages of a cache that the caller holds (include/orangu_b200.h, ob_pages_*): what the entry points of
// pages.cu hand to the kernels of pages_attention.cu, pages_tc5.cu and pages_select.cu.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace ob {

constexpr uint32_t PG_MAX_DRAFTS = 64;   // drafted tokens of a sequence: a bit each
constexpr uint32_t PG_MAX_GROUP = 16;    // query heads of a key/value head
// Drafted tokens times heads of a key/value head: up to here mma.sync tiles of 16 rows, above tcgen05 tiles of 128.  Both at 16 rows, head
// dimension 128: 16.4 and 18.4 us for one sequence of 512, 45.1 and 51.2 for 32 of 1024, 195 and 223 for 32 of 8192; 64: 14.3 and 16.4, 30.7 and
// 43.0, 119 and 166.  More rows would read all pages once per 16.
constexpr uint32_t PG_FEW_ROWS = 16;
constexpr float PG_SLACK = 8.0f;         // growth of a row's maximum (powers of two) that is put up with before its output is rescaled
// Weights are made 2^PG_RAISE times as large, in numerator and denominator alike.  An f16 weight has steps of 2^-24 at best: of the running maximum's
// weight as 1, those below 2^-25 would vanish and those below 2^-14 lose bits, raised they are off by 2^-32.  (131,000 positions of 2^-21 behind one of 1:
// the result was off by 31 to 129 half steps of f16, now by 0.4 to 2; the rest is the sums'.)  With the slack the largest is 2^15, of f16's 2^16.  bf16
// has the range of fp32.
template <typename T> constexpr float PG_RAISE = 0.0f;
template <> inline constexpr float PG_RAISE<__half> = 7.0f;
constexpr uint32_t PG_PAGES = 4;         // pages of a tile of the tcgen05 kernel
constexpr uint32_t PG_START = 6;         // what the start and end of a piece cost there, in tiles
constexpr size_t PG_WORKSPACE = 64u << 20;  // partial results of the splits, behind the counters
constexpr uint32_t PG_COUNTERS = 4096;   // arrival counters, zero between launches
struct alignas(32) PagePiece {  // rows whose parts several CTAs have left (pages_tc5.cu), for the kernel that adds them up
    uint32_t parts, slot;       // 0: none; place of the first part, the others are at every other one from the next even place on
    uint32_t rows, row, token0, head;  // rows row .. row + rows - 1 of the sequence that begins at token0
};
constexpr size_t PG_PARTIAL = PG_WORKSPACE - PG_COUNTERS * (4 + sizeof(PagePiece));

// One layer's pages and the tables of the sequences.
struct PageView {
    const void *k, *v;  // [n_pages][n_kv][KV_PAGE][dim], f16 or bf16
    bool is_bf16;
    uint32_t n_pages, n_kv, dim;
    const int32_t *tables;
    uint32_t n_seq, stride;
};

struct PagedAttnArgs {
    PageView pg;
    const void *q;   // [token or row][n_kv * group][dim], q_stride elements apart
    void *out;
    uint64_t q_stride, out_stride;
    uint32_t group, n_units;  // n_units: sequences (tree) or rows (list)
    float scale;
    // tree
    const int32_t *first;     // [n_units + 1]
    const uint32_t *n_ctx;    // [n_units]
    const uint64_t *visible;  // [n_tokens]
    uint32_t n_tokens, max_drafts, max_ctx;
    // list
    const int32_t *list;      // [n_units][n_kv][n_list]
    const uint32_t *n_pos;    // [n_units]
    const int32_t *row_seq;   // [n_units] or null: row r is of sequence r
    uint32_t n_list;
    // workspace
    uint32_t *counters;
    PagePiece *pieces;
    float *partial;
    uint32_t *status;  // pinned host memory: 1 when a bounded wait ran out and the outputs are not valid
    // filled in by the launcher
    uint32_t row_tiles;
};
// With `tree`, max_drafts * group is at most PG_FEW_ROWS.
cudaError_t launch_pages_attention(const PagedAttnArgs &a, bool tree, int sm_count, cudaStream_t st);

// Tensor maps of one layer's keys and values (two CUtensorMap, made once per handle and layer).
struct alignas(64) PageMaps {
    uint8_t bytes[256];
};
bool make_page_maps(const PageView &pg, PageMaps *out);  // false: the pool has too many rows for them
cudaError_t launch_pages_tree_tc5(const PagedAttnArgs &a, const PageMaps &maps, int sm_count, cudaStream_t st);
cudaError_t launch_pages_wait_selftest(uint32_t *status, cudaStream_t st);  // a warp whose wait runs out, and then ends as that kernel does

struct PagedSelectArgs {
    PageView pg;
    const int8_t *codes;   // [n_pages][n_kv][2][dim]: largest, smallest
    const float *scales;   // [n_pages][n_kv]
    const void *q;
    uint64_t q_stride;
    uint32_t group, n_rows;
    const uint32_t *n_pos;
    const int32_t *row_seq;
    uint32_t max_pos, n_select, keep_first, keep_last;
    int32_t *selected;     // [n_rows][n_kv][n_select]
    uint32_t *keys;        // workspace, PG_KEYS_BYTES
};
constexpr size_t PG_KEYS_BYTES = PG_PARTIAL;    // (one of the two uses at a time)
constexpr uint32_t PG_SELECT_PAGES = 131072;    // most pages of a row
cudaError_t launch_pages_select(const PagedSelectArgs &a, int sm_count, cudaStream_t st, uint32_t *launches);

}  // namespace ob
