// Where the paged 4-bit cache's kernels read and write: pages, rows, tiles of
// query rows and their keys.  Host and device, so that every bound can be
// tested without a GPU.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define WH_KV_HD __host__ __device__ __forceinline__
#else
#define WH_KV_HD static inline
#endif

#define WH_KV_NONE 0xffffffffu  // a slot or page that is none

// f(i) for a thread's share of n things: first, first + step, ..; 64 bits, since a
// cache may have 2^32 - 2 pages, past which a step would start over.
template <class F>
WH_KV_HD void wh_kv_share(uint64_t first, uint64_t step, uint64_t n, F f) {
    for (uint64_t i = first; i < n; i += step) f((uint32_t)i);
}

// Line of a row in a plane: codes start at line * head_dim / 2, scale bytes at
// line * head_dim / 32.
WH_KV_HD uint64_t wh_kv4_line(uint32_t page, uint32_t head, uint32_t row, uint32_t kv_heads, uint32_t shift) {
    return ((((uint64_t)page * kv_heads) + head) << shift) + row;
}

// Rows of a call that one launch takes, of `pieces` work-items each (at most 65535
// heads of 64): 2^31 items, well below the 2^32 of a grid dimension.
WH_KV_HD uint64_t wh_kv4_rows_of_launch(uint64_t n, uint64_t pieces) {
    const uint64_t most = (1ull << 31) / pieces;
    return n < most ? n : most;
}

// A slot's page, or false when the slot is none or behind the cache.
WH_KV_HD bool wh_kv4_slot_page(uint32_t slot, uint32_t shift, uint32_t n_pages, uint32_t* page, uint32_t* row) {
    *page = slot >> shift;
    *row = slot & ((1u << shift) - 1u);
    return slot != WH_KV_NONE && *page < n_pages;
}

// A tile of `kRows` flattened (token, head of the group) rows of one request.
struct wh_kv4_tile {
    uint32_t request, row0, rows, n_q;  // first row of the request's n_q * group and how many
    uint32_t token0;                    // the request's first row of q and out
    int32_t len;                        // its cached rows
    uint32_t first, from, end;          // its rows see keys [0, first) and [from, end) at most
    uint32_t first_runs, lo, runs;      // runs of 64 keys that hold those: first_runs from key 0, the others from lo
    bool ok;                            // holds rows
};

// First tile slot of request b, whose first token is `start`: at least as many
// slots before request b + 1's as b has tiles, and not falling with b, so that a
// search for the last one at or before a slot finds its request without a sum
// over the others.  Where a token fills whole tiles there is none between.
WH_KV_HD uint64_t wh_kv4_tile_base(uint32_t start, uint32_t group, uint32_t b, uint32_t tile_rows) {
    return (uint64_t)start * group / tile_rows + (group % tile_rows ? b : 0);
}

// Tile slots of a call.
WH_KV_HD uint64_t wh_kv4_tile_slots(uint64_t n_tokens, uint64_t n_requests, uint32_t group, uint32_t tile_rows) {
    return n_tokens * group / tile_rows + (group % tile_rows ? n_requests : 0);
}

// Slot x of request b with tokens [s0, s1) (both at most n_tokens) and len
// cached rows, of which a table row holds at most cap < 2^31.
WH_KV_HD wh_kv4_tile wh_kv4_tile_of(uint64_t x, uint32_t b, uint32_t s0, uint32_t s1, uint32_t len, uint32_t cap,
                                    uint32_t group, uint32_t window, uint32_t first, uint32_t tile_rows) {
    wh_kv4_tile r;
    r.request = b;
    r.token0 = s0;
    r.n_q = s1 > s0 ? s1 - s0 : 0;
    const uint64_t base = wh_kv4_tile_base(s0, group, b, tile_rows);
    const uint64_t row0 = x >= base ? (x - base) * tile_rows : 0, all = (uint64_t)r.n_q * group;
    r.ok = x >= base && row0 < all;
    r.row0 = r.ok ? (uint32_t)row0 : 0;
    r.rows = r.ok ? (uint32_t)(all - row0 < tile_rows ? all - row0 : tile_rows) : 0;
    r.len = (int32_t)(len < cap ? len : cap);
    r.first = r.from = r.end = r.first_runs = r.lo = r.runs = 0;
    if (!r.ok) return r;
    // positions of the first and the last row; negative where there are more tokens than rows
    const int64_t p0 = (int64_t)r.len - r.n_q + r.row0 / group;
    const int64_t p1 = (int64_t)r.len - r.n_q + (r.row0 + r.rows - 1) / group;
    if (p1 < 0) return r;
    const int64_t from = window && p0 + 1 > (int64_t)window ? p0 + 1 - (int64_t)window : 0;
    r.from = (uint32_t)from;
    r.end = (uint32_t)(p1 + 1);
    r.lo = r.from & ~63u;
    r.first = first < r.from ? first : r.from;
    r.first_runs = r.first < r.lo ? (r.first + 63) / 64 : r.lo / 64;
    r.runs = r.first_runs + (r.end - r.lo + 63) / 64;
    return r;
}

// First key of run x, a multiple of 64: where a page has 64 rows or more, a run
// lies in one, and some row sees a key of it.
WH_KV_HD uint32_t wh_kv4_run(const wh_kv4_tile& t, uint32_t x) { return x < t.first_runs ? 64 * x : t.lo + 64 * (x - t.first_runs); }

// A key of a run that some row may see: `key` itself or, where no row does, one
// that stands in for it.  Keys that no row sees need not have pages.
WH_KV_HD uint32_t wh_kv4_seen(const wh_kv4_tile& t, uint32_t key0, uint32_t key) {
    const uint32_t low = key0 < t.lo ? t.first - 1 : t.from, high = key0 < t.lo ? t.first - 1 : t.end - 1;
    const uint32_t in = key < low ? low : key < high ? key : high;
    return key < t.first ? key : in;
}

// How a call whose tiles are fewer than its workgroups cuts up their keys.  Of
// request b, n_q tokens on len rows: tiles, and at most how many runs each has.
WH_KV_HD uint32_t wh_kv4_tiles(uint32_t n_q, uint32_t group, uint32_t tile_rows) {
    return (uint32_t)(((uint64_t)n_q * group + tile_rows - 1) / tile_rows);
}
WH_KV_HD uint32_t wh_kv4_runs(uint32_t n_q, uint32_t len, uint32_t cap, uint32_t window, uint32_t first) {
    const uint64_t keys = len < cap ? len : cap, all = (keys + 63) / 64;
    if (!window) return (uint32_t)all;
    const uint64_t seen = ((uint64_t)first + 63) / 64 + ((uint64_t)window + n_q + 125) / 64;  // from a multiple of 64
    return (uint32_t)(seen < all ? seen : all);
}
// Workgroups of a tile of so many runs: one, and its part of the `units` that
// are more than there are tiles (by all their runs, `sum`), rounded down: all
// tiles together have max(units, tiles) at most.  No less than min_runs each.
// The quotient of whole numbers below 2^53 is rounded to the nearest double, which
// does not reach a whole number that it is less than (by 1 / sum at least).
WH_KV_HD uint32_t wh_kv4_splits(uint32_t runs, uint64_t sum, uint64_t tiles, uint32_t units, uint32_t min_runs) {
    const uint32_t most = runs / min_runs;
    if (units <= tiles || !sum || most <= 1) return 1;
    const double share = (double)((uint64_t)runs * (units - (uint32_t)tiles)) / (double)sum;
    return share + 1.0 < (double)most ? 1 + (uint32_t)share : most;
}
// And runs of each of those when they share alike: so many that at most `splits` have any.
WH_KV_HD uint32_t wh_kv4_even(uint32_t runs, uint32_t splits) {
    return splits <= 1 ? 0x7fffffffu : (runs + splits - 1) / splits;
}
