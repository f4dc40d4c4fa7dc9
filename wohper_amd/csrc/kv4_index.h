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

// Line of a row in a plane: codes start at line * head_dim / 2, scale bytes at
// line * head_dim / 32.
WH_KV_HD uint64_t wh_kv4_line(uint32_t page, uint32_t head, uint32_t row, uint32_t kv_heads, uint32_t shift) {
    return ((((uint64_t)page * kv_heads) + head) << shift) + row;
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
    uint32_t n_first, lo, n_keys;       // keys [0, n_first) and [lo, lo + n_keys - n_first)
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
    r.n_first = r.lo = r.n_keys = 0;
    if (!r.ok) return r;
    // positions of the first and the last row; negative where there are more tokens than rows
    const int64_t p0 = (int64_t)r.len - r.n_q + r.row0 / group;
    const int64_t p1 = (int64_t)r.len - r.n_q + (r.row0 + r.rows - 1) / group;
    if (p1 < 0) return r;
    const int64_t from = window && p0 + 1 > (int64_t)window ? p0 + 1 - (int64_t)window : 0;
    r.lo = (uint32_t)from;
    r.n_first = first < r.lo ? first : r.lo;
    r.n_keys = r.n_first + (uint32_t)(p1 + 1 - from);
    return r;
}

// The v-th key of a tile, v < n_keys.
WH_KV_HD uint32_t wh_kv4_key(const wh_kv4_tile& t, uint32_t v) { return v < t.n_first ? v : v - t.n_first + t.lo; }

// Whether a token at position pos (negative: none) sees a key.
WH_KV_HD bool wh_kv4_sees(int32_t pos, uint32_t key, uint32_t window, uint32_t first) {
    return (int64_t)key <= pos && (!window || key < first || (int64_t)key + window > pos);
}

// How a call whose tiles are fewer than its workgroups cuts up their keys.  Of
// request b, n_q tokens on len rows: tiles, and at most how many blocks of
// `block` keys each sees.
WH_KV_HD uint32_t wh_kv4_tiles(uint32_t n_q, uint32_t group, uint32_t tile_rows) {
    return (uint32_t)(((uint64_t)n_q * group + tile_rows - 1) / tile_rows);
}
WH_KV_HD uint32_t wh_kv4_blocks(uint32_t n_q, uint32_t len, uint32_t cap, uint32_t window, uint32_t first, uint32_t block) {
    uint64_t keys = len < cap ? len : cap;
    if (window && keys > (uint64_t)window + first + n_q) keys = (uint64_t)window + first + n_q;
    return (uint32_t)((keys + block - 1) / block);
}
// Workgroups of a tile of `blocks` blocks: one, and its part of the `units` that
// are more than there are tiles (by all their blocks, `sum`), rounded down: all
// tiles together have max(units, tiles) at most.  No less than min_blocks each.
// The quotient of whole numbers below 2^53 is rounded to the nearest double, which
// does not reach a whole number that it is less than (by 1 / sum at least).
WH_KV_HD uint32_t wh_kv4_splits(uint32_t blocks, uint64_t sum, uint64_t tiles, uint32_t units, uint32_t min_blocks) {
    const uint32_t most = blocks / min_blocks;
    if (units <= tiles || !sum || most <= 1) return 1;
    const double share = (double)((uint64_t)blocks * (units - (uint32_t)tiles)) / (double)sum;
    return share + 1.0 < (double)most ? 1 + (uint32_t)share : most;
}
// And blocks of each of those when they share alike: so many that at most `splits` have any.
WH_KV_HD uint32_t wh_kv4_even(uint32_t blocks, uint32_t splits) {
    return splits <= 1 ? 0x7fffffffu : (blocks + splits - 1) / splits;
}
