// 8-bit rows and their products with resident FP8 weights: arguments and
// launches of fp8_rows.hip, a translation unit of its own.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define WH_ROWS_NONE 0xFFFFFFFFu     // a route to no expert, a slot of no row
#define WH_ROWS_MAX_GROUPS 1024u     // experts of a grouped product or a plan

#define WH_ROWS_TICKETS 16u          // counters that a context's products share

// 8-bit rows in device memory (wh_fp8_rows).
struct wh_rows8 {
    uint8_t* codes;
    uint64_t stride;
    uint8_t* scales;
    uint64_t scale_stride;
};

// Rows to 8 bits and back: n rows of `blocks` blocks of 128 columns.
struct wh_rows_quant_args {
    const void* x;   // SwiGLU: the gate rows
    const void* up;  // SwiGLU: the up rows, else null
    uint64_t x_stride;
    uint32_t n, blocks;
    float limit;
    wh_rows8 out;
};
hipError_t wh_rows_quant_launch(const wh_rows_quant_args& a, bool bf16, hipStream_t stream);

struct wh_rows_read_args {
    wh_rows8 in;
    void* out;
    uint64_t out_stride;
    uint32_t n, blocks;
};
hipError_t wh_rows_read_launch(const wh_rows_read_args& a, bool bf16, hipStream_t stream);

// A product: listed row j of group g (starts[g] <= j < starts[g + 1]; without
// starts one group of n rows) is x row rows[j] (without rows: j), and meets
// weight rows row_start + g * out_rows + [0, out_rows).
struct wh_rows_mm_args {
    const uint8_t* w;    // the store's lane layout
    const void* w_scales;
    wh_rows8 x;
    const uint32_t *rows, *starts;
    void* y;
    uint64_t y_stride, row_start;
    uint32_t n, n_x, n_groups, out_rows;
    uint32_t cols;       // a multiple of 128
    uint32_t row_block;  // weight rows that share a scale
    uint32_t scale_f32;  // scales are f32, else UE8M0 bytes
    uint32_t special;    // weight codes 0x7F / 0xFF are there, +-480
    uint32_t odd_scale;  // UE8M0 scale bytes 0 or 255 are there
    float* part;         // the plan's part_bytes
    uint32_t* tickets;   // [WH_ROWS_TICKETS], 0 between launches
};
// How a product is done: by sizes that the host knows.
struct wh_rows_mm_plan {
    enum kind_t { kAny, kThin, kTile, kHalf, kTall } kind;
    uint32_t splits, per;  // ranges that its columns are cut into, and blocks of each
    uint32_t threads;
    uint64_t tiles;        // at most, of the kernel's
    uint64_t grid;         // workgroups for each range
    size_t part_bytes;     // scratch for the ranges' parts
};
wh_rows_mm_plan wh_rows_mm_plan_of(const wh_rows_mm_args& a, bool bf16);
hipError_t wh_rows_mm_launch(const wh_rows_mm_args& a, const wh_rows_mm_plan& p, bool bf16, hipStream_t stream);
hipError_t wh_rows_setup();  // once for each device, before the first launch there

// The store's lane layout of a tensor that is on the device, and which of its
// codes and scales the matrix instructions read otherwise: *flags gets bit 0
// for codes 0x7F / 0xFF, bit 1 for UE8M0 bytes 0 / 255.
hipError_t wh_rows_store_launch(const uint8_t* weight, uint8_t* out, uint64_t rows, uint32_t cols, uint32_t* flags,
                                hipStream_t stream);
hipError_t wh_rows_scales_launch(const uint8_t* scales, uint64_t n, uint32_t* flags, hipStream_t stream);

// Expert lists of npos * topk routes.
struct wh_expert_plan_args {
    const uint32_t* ids;
    uint32_t *starts, *rows, *slots;
    uint32_t* counts;  // scratch [chunks + 1][n_groups, padded to 4], where there is more than one chunk
    uint32_t n, topk, n_groups;
};
size_t wh_expert_plan_scratch(size_t n, size_t n_groups);
hipError_t wh_expert_plan_launch(const wh_expert_plan_args& a, hipStream_t stream);

struct wh_expert_combine_args {
    const void* y;
    uint64_t y_stride, out_stride, add_stride;
    const uint32_t* slots;
    const float* weights;
    const float* add;
    float* out;
    uint32_t n_rows, npos, topk, hidden;
};
hipError_t wh_expert_combine_launch(const wh_expert_combine_args& a, bool bf16, hipStream_t stream);
