// Operators over the pages of a cache that the caller holds (include/orangu_b200.h, ob_pages_*): what the entry points of
// pages.cu hand to the kernels of pages_attention.cu, pages_tc5.cu, pages_select.cu, pages_q4.cu, pages_store.cu, pages_mass.cu and pages_evict.cu.
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
// The same over 4-bit pages, there in units of tokens that have up to 16 rows, each of which reads the pages for itself.  Both at 32 and 48 rows, f16 queries, 8 heads of 128: one sequence of
// 2048 16.5 and 18.6, 18.6 and 18.6 us; eight of 2048 28.9 and 30.8, 37.0 and 30.9; 32 of 2048 73.9 and 79.6, 101 and 82; eight of 8192 68.5 and 64.3, 94.3 and 65.4; with 64
// entries 45.2 and 57.5, 61.6 and 57.2.
constexpr uint32_t P4_FEW_ROWS = 32;
// Shares of a CTA from which on all are even (PA_MORE).  4-bit pages, bfloat16 rows, 8 heads of 128: 32 sequences of 2 to 8 k 59.6 us, and 67.7 with pieces that all begin a CTA; one of
// 4000 12.4 us, and 15.7 with even shares, two of 1000 with four tokens 14.5 and 20.7 (eight of 2000 16.5 and 14.8).
constexpr uint32_t PG_APART = 64;
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
constexpr size_t PG_STATS = 16u << 20;      // of these, at the end: a maximum and the inverse of a sum per (token, head), where weights are added up per position
constexpr size_t PG_PARTS = PG_PARTIAL - PG_STATS;

// One layer's pages and the tables of the sequences.
struct PageView {
    const void *k, *v;  // [n_pages][n_kv][KV_PAGE][dim], f16 or bf16, or [n_pages][n_kv] blocks in 4 bits (pages_q4.cuh)
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
    uint32_t n_tokens, max_drafts, max_ctx;  // visible may be null: a token sees those before it and itself
    uint32_t block, blocks;   // tokens of a unit, units of a sequence (n_units: all of them); several with visible == null, or (mma.sync) over 4-bit pages
    float2 *stats;            // [n_tokens][n_kv * group] or null: a row's maximum and the inverse of its sum, so that a weight is 2^(score - maximum) times that
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
    uint32_t apart;    // mma.sync forms: shares of this many pages and more are even, whatever pieces begin in their middle
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

// 4-bit pages: units of tokens that have at most PG_FEW_ROWS, and of up to PG_MAX_DRAFTS tokens.
cudaError_t launch_pages_q4_attention(const PagedAttnArgs &a, bool q_bf16, int sm_count, cudaStream_t st);
cudaError_t launch_pages_q4_tc5(const PagedAttnArgs &a, bool q_bf16, int sm_count, cudaStream_t st);
// After an attention with `stats`, whose units are of n_seq sequences: [n_seq][n_kv][mass_stride].
cudaError_t launch_pages_mass(const PagedAttnArgs &a, bool q_bf16, bool q4, uint32_t n_seq, float *mass, uint64_t mass_stride, int sm_count, cudaStream_t st);

// Rows a key/value head up to which the first of the two is taken.  Both at 64 and 128 rows over f16 pages, 16 sequences of 2000, attention among it: 71.4 and 72.4 us, 93.3 and 77.6.
// Where bfloat16 queries have to become f16 ones for every tile it is more, and depends on the sequences, too: 256 and 512 rows over 4-bit pages, one sequence of 12,000: 108 and 101,
// 181 and 160; four of 12,000: 202 and 256, 388 and 457; 2000 rows, one sequence: 627 and 366.
constexpr uint32_t PG_MASS_ROWS = 96, P4_MASS_ROWS_BF16 = 256;
cudaError_t launch_pages_mass_tc5(const PagedAttnArgs &a, bool q_bf16, bool q4, uint32_t n_seq, float *mass, uint64_t mass_stride, int sm_count, cudaStream_t st);

struct PagedMoveArgs {  // rows into 4-bit pages, or out of them
    PageView pg;
    const void *k, *v;  // [n_tokens][n_kv][dim], strides in elements
    uint64_t k_stride, v_stride;
    const int32_t *first;
    const uint32_t *n_ctx;
    uint32_t n_seq, n_tokens, max_tokens;
};
cudaError_t launch_pages_store(const PagedMoveArgs &a, bool is_bf16, bool load, int sm_count, cudaStream_t st);

struct PagedEvictArgs {
    PageView pg;             // of layer 0
    uint64_t layer_bytes;
    uint32_t n_seq;
    const uint32_t *n_pos;
    float *mass;             // [n_layer][n_seq][n_kv][mass_stride]
    uint64_t mass_stride;
    uint32_t n_keep, keep_first, keep_last;
    int32_t *kept;           // [n_layer][n_seq][n_kv][n_keep]
    uint32_t *n_left;
};
cudaError_t launch_pages_evict(const PagedEvictArgs &a, uint32_t n_layer, uint32_t max_pos, bool q4, cudaStream_t st);

struct PagedKeepArgs {
    PageView pg;             // of layer 0
    uint64_t layer_bytes;
    const uint32_t *n_ctx;
    const int32_t *kept;
    uint32_t kept_stride;
    const uint32_t *n_kept;
};
cudaError_t launch_pages_keep_q4(const PagedKeepArgs &a, uint32_t n_seq, uint32_t n_layer, cudaStream_t st);
cudaError_t launch_pages_keep_mass(const PagedKeepArgs &a, uint32_t n_seq, uint32_t n_layer, float *mass, uint64_t stride, cudaStream_t st);

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
