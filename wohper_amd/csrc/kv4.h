// The paged 4-bit attention cache: arguments and launches of kv4.hip, which
// is a translation unit of its own (its templates compile beside the rest).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv4_index.h"

#define WH_KV_SPLIT_REQUESTS 256u  // requests of a call whose keys are cut up: each wave adds them up
#define WH_KV_MAX_REQUESTS 4096u  // requests of one plan: three prefix sums of them lie in LDS

// One step's plan (wh_kv_plan_async): device arrays as in the header.
struct wh_kv_plan_args {
    const uint32_t *old_lens, *new_lens, *free_in, *free_count;
    uint32_t *tables, *free_out, *free_count_out, *starts, *slots, *positions;
    uint64_t table_stride;
    uint32_t n, shift, n_pages, max_tokens;
    uint32_t* ticket;  // arrivals of the launch, 0 between launches
    uint32_t* status;
};
hipError_t wh_kv_plan_launch(const wh_kv_plan_args& a, hipStream_t stream);

// Codes and scales of one plane (keys, or values) of a cache.
struct wh_kv4_plane {
    uint8_t* codes;
    uint8_t* scales;
};
struct wh_kv4_shape {
    uint32_t n_pages, shift, kv_heads, head_dim;  // page_size = 1 << shift
};
// Rows in (wh_kv4_write_async) or out (wh_kv4_read_async) of one or two planes.
struct wh_kv4_rows_args {
    wh_kv4_plane plane[2];
    void* rows[2];       // [n] rows of kv_heads * head_dim values
    uint64_t stride[2];  // values between rows
    wh_kv4_shape s;
    const uint32_t* slots;
    uint32_t n, planes;
    uint32_t* status;
};
hipError_t wh_kv4_write_launch(const wh_kv4_rows_args& a, bool bf16, hipStream_t stream);
hipError_t wh_kv4_read_launch(const wh_kv4_rows_args& a, bool bf16, hipStream_t stream);

struct wh_kv4_attn_args {
    wh_kv4_plane k, v;
    wh_kv4_shape s;
    const void* q;
    void* out;
    uint64_t q_stride, out_stride;
    const uint32_t *starts, *lens, *tables;
    uint64_t table_stride;
    const float* sink;
    float* part;        // [unit][kv head][rows][head_dim + 2]: normalised outputs, sums of weights (kv_put_sum)
    uint32_t n_tokens, n_requests, group, window, first;
    uint32_t n_tiles;     // slots or tiles, at most
    uint32_t units;       // workgroups of a key head, at most; > n_tiles: their keys are cut up
    uint32_t min_runs;    // runs of 64 keys that a part of a tile has at least
    bool wide;            // tiles of 64 (f32: 32) rows instead of 16
    float scale_log2;   // scale * log2(e)
    uint32_t* status;
};
// How a call is cut up: by sizes the host knows.
struct wh_kv4_attn_plan {
    uint32_t n_tiles, units, min_runs;
    bool wide;
    size_t part_bytes;  // scratch for partial results, 0 for one split
};
wh_kv4_attn_plan wh_kv4_attn_plan_of(const wh_kv4_attn_args& a, bool bf16, size_t max_len);
hipError_t wh_kv4_setup();  // once for each device, before the first launch there
hipError_t wh_kv4_attn_launch(const wh_kv4_attn_args& a, bool bf16, bool latent, hipStream_t stream);
