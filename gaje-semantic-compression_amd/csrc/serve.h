// Launch interface of the serving operators: attention over packed prompts, over a
// paged KV cache and over a shared prefix (serve_attn.hip), and the cache's pages
// (kv_pages.hip).  serve.cpp holds the C entry points and their checks.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "gaje_hip.h"

namespace gaje {

// Where the rows of a launch and their keys are.  Keys of a packed call are the
// sequence's own rows; those of a paged one are reached through a table.
struct ServeAttnParams {
    int32_t dtype;
    const void *q, *k, *v;  // k, v: packed rows, or one layer of the page pools
    int64_t ldq, ldk, ldv;  // elements between rows
    void *out;
    int64_t ldo;
    const int32_t *seq_off;  // [n_seq + 1], null: row s is sequence s
    int64_t n_seq, T;
    int32_t n_head, n_head_kv, head_dim;
    float scale;
    // paged
    const int32_t *table;  // null: packed
    const int32_t *len;
    int64_t max_pages, n_pages;
    int32_t page_shift;
    // shared prefix: positions 0..prefix_len-1 through prefix_table
    // (one row per sequence, seq_off null)
    const int32_t *prefix_table;  // null: none
    int64_t prefix_len;
    // parts of each row's own keys, [T][n_head], and partial results: [n_part][T][n_head] (maximum, sum) and [n_part][T][n_head][head_dim]
    int32_t *parts;
    float2 *part_ml;
    float *part_o;
};

// Bytes of the partial results of a launch (0: it needs none).
int64_t serve_attn_workspace(const ServeAttnParams &p);
int launch_serve_attn(const ServeAttnParams &p, void *workspace, hipStream_t s);

int64_t kv_update_workspace(const gaje_hip_kv_pages &c);
int launch_kv_update(const gaje_hip_kv_pages &c, const int32_t *source, const int32_t *add, int32_t *new_table,
                     int32_t *new_len, int32_t *new_ref, int32_t *status, void *workspace, hipStream_t s);
int launch_kv_compact(const gaje_hip_kv_pages &c, int32_t *new_table, int32_t *new_ref, int32_t *n_live,
                      void *workspace, hipStream_t s);
int launch_kv_append(const gaje_hip_kv_pages &c, int64_t layer, int source_dtype, const void *k, int64_t ldk,
                     const void *v, int64_t ldv, const int32_t *seq_off, int64_t T, hipStream_t s);

}  // namespace gaje
