// Host driver for the address arithmetic of the paged 4-bit cache
// (wohper_amd/csrc/kv4_index.h): random calls, half of them with garbage in
// the arrays that live on the device, checked against counting by hand.
// Prints nothing and returns 0 when every row is taken once, every key is the
// one it should be and nothing leaves its buffer.  Built and run by
// tests/test_kv4_host.py.
//   usage: kv4_index ITERATIONS
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "kv4_index.h"

namespace {

uint64_t g_state = 0x9e3779b97f4a7c15ull;

uint64_t next() {  // xorshift64*
    g_state ^= g_state >> 12;
    g_state ^= g_state << 25;
    g_state ^= g_state >> 27;
    return g_state * 0x2545f4914f6cdd1dull;
}
uint32_t upto(uint32_t n) { return (uint32_t)((next() >> 20) % ((uint64_t)n + 1)); }

#define CHECK(x)                                                          \
    do {                                                                  \
        if (!(x)) {                                                       \
            std::printf("line %d, iteration %d: %s\n", __LINE__, it, #x); \
            return 1;                                                     \
        }                                                                 \
    } while (0)

}  // namespace

int main(int argc, char** argv) {
    if (argc != 2) return 2;
    const int n = std::atoi(argv[1]);
    for (int it = 0; it < n; ++it) {
        const bool garbage = it & 1;
        const uint32_t tile_rows = 16u << upto(2), shift = upto(8), group = it % 7 == 2 ? 16u << upto(3) : 1 + upto(it % 3 ? 8 : 70);
        const uint32_t requests = 1 + upto(it % 5 ? 6 : 150), n_tokens = upto(60);
        const uint32_t table_stride = upto(30), n_pages = 1 + upto(40), kv_heads = 1 + upto(3);
        const uint32_t window = upto(1) ? 0 : 1 + upto(it % 8 ? 20 : 300), first = upto(it % 4 ? 6 : 200);
        std::vector<uint32_t> starts(requests + 1), lens(requests);
        for (auto& s : starts) s = garbage && upto(1) ? (uint32_t)next() : upto(n_tokens);
        std::sort(starts.begin(), starts.end());
        if (garbage && upto(1)) std::swap(starts[0], starts[requests]);
        if (!garbage) starts[0] = 0;
        const uint32_t cap = (uint32_t)std::min<uint64_t>((uint64_t)table_stride << shift, 0x7fffffff);
        for (auto& l : lens) l = garbage && upto(1) ? (uint32_t)next() : upto(cap);
        auto start = [&](uint32_t b) { return std::min(starts[b], n_tokens); };
        std::vector<int> taken((size_t)n_tokens * group);
        const uint64_t slots = wh_kv4_tile_slots(n_tokens, requests, group, tile_rows);
        for (uint64_t x = 0; x < slots; ++x) {
            // any request a search may end at
            uint32_t b = 0;
            if (garbage) b = upto(requests - 1);
            else
                while (b + 1 < requests && wh_kv4_tile_base(start(b + 1), group, b + 1, tile_rows) <= x) ++b;
            const wh_kv4_tile t = wh_kv4_tile_of(x, b, start(b), start(b + 1), lens[b], cap, group, window, first, tile_rows);
            if (!t.ok) {
                CHECK(t.runs == 0 && t.rows == 0);
                continue;
            }
            CHECK(t.rows >= 1 && t.rows <= tile_rows && (uint64_t)t.row0 + t.rows <= (uint64_t)t.n_q * group);
            std::set<uint32_t> want;
            for (uint32_t r = 0; r < t.rows; ++r) {
                const uint32_t flat = t.row0 + r, tok = flat / group;
                CHECK(t.token0 + tok < n_tokens);
                if (!garbage) ++taken[(size_t)(t.token0 + tok) * group + flat % group];
                const int64_t pos = (int64_t)t.len - t.n_q + tok;
                for (int64_t j = 0; j <= pos; ++j) {
                    const bool sees = !window || j > pos - (int64_t)window || j < first;
                    if (sees) want.insert((uint32_t)j);
                }
            }
            std::set<uint32_t> got;
            for (uint32_t run = 0; run < t.runs; ++run) {
                const uint32_t key0 = wh_kv4_run(t, run);
                CHECK(key0 % 64 == 0);
                for (uint32_t key = key0; key < key0 + 64; ++key) {
                    const uint32_t some = wh_kv4_seen(t, key0, key);
                    CHECK(some >= key0 && some < key0 + 64 && some < cap && (some >> shift) < table_stride);
                    if (some != key) continue;
                    CHECK(got.insert(key).second);  // each once
                    const uint32_t page = upto(n_pages - 1), head = upto(kv_heads - 1), row = key & ((1u << shift) - 1u);
                    CHECK(wh_kv4_line(page, head, row, kv_heads, shift) < ((uint64_t)n_pages * kv_heads << shift));
                }
            }
            for (uint32_t j : want) CHECK(got.count(j));
            CHECK(t.runs <= wh_kv4_runs(t.n_q, lens[b], cap, window, first));
        }
        uint64_t tiles = 0, blocks = 0;
        for (uint32_t b = 0; b < requests; ++b) {
            const uint32_t n_q = start(b + 1) > start(b) ? start(b + 1) - start(b) : 0, k = wh_kv4_tiles(n_q, group, tile_rows);
            tiles += k;
            blocks += (uint64_t)k * wh_kv4_runs(n_q, lens[b], cap, window, first);
        }
        if (!garbage) CHECK(tiles <= slots);
        for (uint32_t units : {1u, 7u, 64u, 300u}) {
            const uint32_t least = 1 + upto(6);
            uint64_t used = 0;
            for (uint32_t b = 0; b < requests; ++b) {
                const uint32_t n_q = start(b + 1) > start(b) ? start(b + 1) - start(b) : 0;
                const uint32_t k = wh_kv4_runs(n_q, lens[b], cap, window, first), splits = wh_kv4_splits(k, blocks, tiles, units, least);
                const uint32_t chunk = wh_kv4_even(k, splits);
                CHECK(splits >= 1 && (splits == 1 || splits * least <= k));
                CHECK((uint64_t)splits * chunk >= k);
                used += (uint64_t)wh_kv4_tiles(n_q, group, tile_rows) * splits;
            }
            CHECK(used <= std::max<uint64_t>(units, tiles));
        }
        if (!garbage) {
            std::vector<int> all((size_t)n_tokens * group);
            for (uint32_t i = 0; i < start(requests) * group; ++i) all[i] = 1;
            CHECK(taken == all);
        }
        for (int k = 0; k < 8; ++k) {
            const uint32_t slot = k == 0 ? WH_KV_NONE : garbage ? (uint32_t)next() : upto((n_pages + 2) << shift);
            uint32_t page, row;
            const bool ok = wh_kv4_slot_page(slot, shift, n_pages, &page, &row);
            CHECK(ok == (slot != WH_KV_NONE && (uint64_t)slot < ((uint64_t)n_pages << shift)));
            if (ok) CHECK(wh_kv4_line(page, kv_heads - 1, row, kv_heads, shift) < ((uint64_t)n_pages * kv_heads << shift));
        }
    }
    // a cache whose codes pass 32 bits
    int it = -1;
    CHECK(wh_kv4_line(0xfffffffe >> 6, 7, 63, 8, 6) == ((uint64_t)(0xfffffffe >> 6) * 8 + 7) * 64 + 63);
    return 0;
}
