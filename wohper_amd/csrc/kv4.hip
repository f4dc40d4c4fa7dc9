// The paged 4-bit attention cache (gfx950): plans, rows in and out, attention.
//
// A row of head_dim values is held as E2M1 codes, two a byte (low nibble: the
// even dim), with one UE8M0 scale byte for every 32 dims: value = grid[code] *
// 2^(byte - 127), grid {0, .5, 1, 1.5, 2, 3, 4, 6} and its negatives.  This
// grid is the hardware's conversion, not the weights' (whose second magnitude
// is 0.125): a cache is rounded here, so nothing fixes it to a checkpoint's
// bytes.  Byte 0 stands for 0.0 and 255 for NaN.
#include "kv4.h"

#include <algorithm>
#include <type_traits>

#include "wh_device.h"

namespace {

typedef _Float16 wh_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 wh_h8 __attribute__((ext_vector_type(8)));
typedef int wh_i8 __attribute__((ext_vector_type(8)));
typedef int wh_i2 __attribute__((ext_vector_type(2)));
typedef uint32_t wh_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t wh_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float kv_bits(uint32_t u) { return __uint_as_float(u); }

// ------------------------------------------------------------------- plan

// Sum over this lane and those before it: within rows of 16, then over the rows.
template <int kFrom, int kRows>
__device__ __forceinline__ uint64_t kv_scan_step(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kFrom, kRows, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), kFrom, kRows, 0xf, false);
    return v + ((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint64_t kv_scan(uint64_t v) {
    v = kv_scan_step<0x111, 0xf>(v);  // 1, 2, 4, 8 lanes before
    v = kv_scan_step<0x112, 0xf>(v);
    v = kv_scan_step<0x114, 0xf>(v);
    v = kv_scan_step<0x118, 0xf>(v);
    v = kv_scan_step<0x142, 0xa>(v);  // the end of the row before
    return kv_scan_step<0x143, 0xc>(v);  // the end of the first half
}
__device__ __forceinline__ uint64_t kv_lane(uint64_t v, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

// Last indexes i with prefix[i] <= x (prefix ascending, prefix[0] = 0 <= x), kN
// searches in step.
template <int kN>
__device__ __forceinline__ void kv_find(const uint32_t* prefix, uint32_t n, const uint32_t (&x)[kN], uint32_t (&at)[kN]) {
#pragma unroll
    for (int i = 0; i < kN; ++i) at[i] = 0;  // the answer is in [at, at + n)
    while (n > 1) {
        const uint32_t half = n >> 1;
#pragma unroll
        for (int i = 0; i < kN; ++i) at[i] += prefix[at[i] + half] <= x[i] ? half : 0;
        n -= half;
    }
}
__device__ __forceinline__ uint32_t kv_find(const uint32_t* prefix, uint32_t n, uint32_t x) {
    const uint32_t xs[1] = {x};
    uint32_t at[1];
    kv_find<1>(prefix, n, xs, at);
    return at[0];
}

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kPlanStage = 8192;  // table entries given back that lie in LDS
constexpr size_t plan_lds(uint32_t n) { return (4 * ((size_t)n + 1) + kPlanStage) * sizeof(uint32_t); }

// Every workgroup adds up all requests (three prefix sums of n <= 4096 numbers
// in LDS: new tokens, pages taken, table entries given back) and then fills its share
// of the outputs, so a plan is one launch whose workgroups wait for nobody.  A
// page that a request takes is worked out where it is needed (its table entry,
// each slot on it) instead of being read back from another workgroup's store.
// Entries given back that are no pages (behind a window, and given back before)
// are not numbered: a workgroup that finds one counts the pages of every request
// that shrinks and lays all of them out on the stack, each for itself, as the
// same values.
// Bound by latency: the prefix sums and one chain of dependent loads (7.5 us for
// 64 requests, 12.6 for 512).
__global__ void __launch_bounds__(kPlanThreads) k_kv_plan(wh_kv_plan_args a) {
    extern __shared__ __align__(16) uint32_t lds[];
    uint32_t* const tok = lds;                  // [n + 1]
    uint32_t* const take = tok + a.n + 1;       // [n + 1]
    uint32_t* const give = take + a.n + 1;      // [n + 1]
    uint32_t* const kept = give + a.n + 1;      // [n + 1] pages of a request after the step
    uint32_t* const stage = kept + a.n + 1;     // [kPlanStage]
    __shared__ uint64_t wave_sum[3][kPlanThreads / 64];
    __shared__ uint32_t bad;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t count_in = *a.free_count, mask = (1u << a.shift) - 1u;
    if (t == 0) bad = 0;
    __syncthreads();
    constexpr uint32_t kPer = WH_KV_MAX_REQUESTS / kPlanThreads;
    const uint32_t per = (a.n + kPlanThreads - 1) / kPlanThreads, b0 = t * per;
    auto pages = [&](uint64_t len) { return (len + mask) >> a.shift; };
    uint64_t mine[kPer][3], run[3] = {0, 0, 0};
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
        const uint32_t b = b0 + k;
#pragma unroll
        for (int s = 0; s < 3; ++s) mine[k][s] = run[s];
        if (k < per && b < a.n) {
            const uint64_t o = a.old_lens[b], w = a.new_lens[b];
            const uint64_t po = pages(o), pw = pages(w);
            kept[b] = (uint32_t)pw;
            if (po > a.table_stride || pw > a.table_stride) bad = 1;
            run[0] += w > o ? w - o : 0;
            run[1] += pw > po ? pw - po : 0;
            run[2] += po > pw ? po - pw : 0;
        }
    }
    // the sums over all threads, and of each request's share those before it
    uint64_t total[3];
    auto prefix = [&](auto from) {
        constexpr int kFrom = decltype(from)::value;
        uint64_t incl[3];
#pragma unroll
        for (int s = kFrom; s < 3; ++s) {
            incl[s] = kv_scan(run[s]);
            if (lane == 63) wave_sum[s][wave] = incl[s];
        }
        __syncthreads();
#pragma unroll
        for (int s = kFrom; s < 3; ++s) {
            const uint64_t sum = lane < kPlanThreads / 64 ? wave_sum[s][lane] : 0, upto = kv_scan(sum);
            const uint64_t all = kv_lane(upto, 63), before = kv_lane(upto - sum, wave);
            total[s] = all;
            uint32_t* const dst = s == 0 ? tok : s == 1 ? take : give;
            const uint64_t base = before + incl[s] - run[s];
#pragma unroll
            for (uint32_t k = 0; k < kPer; ++k)
                if (k < per && b0 + k < a.n) dst[b0 + k] = (uint32_t)(base + mine[k][s]);
            if (t == 0) dst[a.n] = (uint32_t)all;
        }
        __syncthreads();
    };
    prefix(std::integral_constant<int, 0>());
    const bool narrow = bad || total[0] > a.max_tokens;
    auto entry = [&](uint32_t j) {  // the j-th table entry given back
        const uint32_t b = kv_find(give, a.n, j);
        return a.tables[b * a.table_stride + kept[b] + (j - give[b])];
    };
    bool odd = false;  // whether some of them are no pages
    const bool staged = total[2] <= kPlanStage;
    if (!narrow && staged) {
        const uint32_t n = (uint32_t)total[2];
        for (uint32_t j0 = t; j0 < n; j0 += 4 * kPlanThreads) {
            uint32_t j[4], b[4], page[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) j[i] = min(j0 + i * kPlanThreads, n - 1);
            kv_find<4>(give, a.n, j, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) page[i] = a.tables[b[i] * a.table_stride + kept[b[i]] + (j[i] - give[b[i]])];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                stage[j[i]] = page[i];
                odd |= page[i] >= a.n_pages;
            }
        }
    } else if (!narrow && total[2] <= 0xffffffffu) {
        for (uint64_t j = t; j < total[2]; j += kPlanThreads) odd |= entry((uint32_t)j) >= a.n_pages;
    }
    const bool holes = total[2] && __syncthreads_or(odd);
    if (holes) {
        // pages of each request, counted by a wave, in the place of its entries
        for (uint32_t b = wave; b < a.n; b += kPlanThreads / 64) {
            const uint32_t po = (uint32_t)pages(a.old_lens[b]), pw = kept[b];
            uint32_t n = 0;
            for (uint64_t i = pw; i < po; i += 64) {
                const uint32_t page = i + lane < po ? a.tables[b * a.table_stride + i + lane] : WH_KV_NONE;
                if (page >= a.n_pages && page != WH_KV_NONE && blockIdx.x == 0) atomicOr(a.status, WH_ST_NOT_RESIDENT);
                n += (uint32_t)__popcll(__ballot(page < a.n_pages));
            }
            if (lane == 0) give[b] = n;
        }
        __syncthreads();
        run[2] = 0;
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            mine[k][2] = run[2];
            if (k < per && b0 + k < a.n) run[2] += give[b0 + k];
        }
        prefix(std::integral_constant<int, 2>());
    }
    // a plan that does not fit is none: nothing is taken, given or numbered
    const bool empty = count_in > a.n_pages || count_in + total[2] > a.n_pages || total[1] > count_in + total[2];
    const bool ok = !narrow && !empty;
    const uint32_t n_tok = ok ? (uint32_t)total[0] : 0, n_take = ok ? (uint32_t)total[1] : 0,
                   n_give = ok ? (uint32_t)total[2] : 0;
    const uint32_t top = count_in + n_give;
    if (holes && ok) {
        for (uint32_t b = wave; b < a.n; b += kPlanThreads / 64) {
            const uint32_t po = (uint32_t)pages(a.old_lens[b]), pw = kept[b];
            uint32_t to = count_in + give[b];
            for (uint64_t i = pw; i < po; i += 64) {
                const uint32_t page = i + lane < po ? a.tables[b * a.table_stride + i + lane] : WH_KV_NONE;
                const uint64_t real = __ballot(page < a.n_pages);
                if (page < a.n_pages) a.free_out[to + (uint32_t)__popcll(real & ((1ull << lane) - 1))] = page;
                to += (uint32_t)__popcll(real);
            }
        }
        __syncthreads();
    }
    auto given = [&](uint32_t j) { return holes ? a.free_out[count_in + j] : staged ? stage[j] : entry(j); };  // the j-th page given back
    auto taken = [&](uint32_t k) {  // the k-th page off the stack
        const uint32_t at = top - 1 - k;
        return at < count_in ? a.free_in[at] : given(at - count_in);
    };
    auto share = [&](uint32_t n, auto f) { wh_kv_share(blockIdx.x * kPlanThreads + t, gridDim.x * kPlanThreads, n, f); };
    share(a.max_tokens, [&](uint32_t i) {
        uint32_t slot = WH_KV_NONE, pos = 0;
        if (i < n_tok) {
            const uint32_t b = kv_find(tok, a.n, i);
            const uint32_t old = a.old_lens[b];
            pos = old + (i - tok[b]);
            const uint32_t po = (uint32_t)pages(old), pi = pos >> a.shift;
            const uint32_t page = pi < po ? a.tables[b * a.table_stride + pi] : taken(take[b] + (pi - po));
            if (page < a.n_pages) slot = (page << a.shift) + (pos & mask);
            else atomicOr(a.status, WH_ST_NOT_RESIDENT);
        }
        a.slots[i] = slot;
        a.positions[i] = pos;
    });
    share(n_take, [&](uint32_t k) {
        const uint32_t b = kv_find(take, a.n, k);
        a.tables[b * a.table_stride + (uint32_t)pages(a.old_lens[b]) + (k - take[b])] = taken(k);
    });
    if (!holes) share(n_give, [&](uint32_t j) { a.free_out[count_in + j] = given(j); });
    if (a.free_out != a.free_in) share(min(count_in, a.n_pages), [&](uint32_t k) { a.free_out[k] = a.free_in[k]; });
    share(a.n + 1, [&](uint32_t b) { a.starts[b] = ok ? tok[b] : 0; });
    if (t == 0 && blockIdx.x == 0 && !ok) atomicOr(a.status, narrow ? WH_ST_KV_NARROW : WH_ST_KV_PAGES);
    // free_count_out may be free_count: it is written once every workgroup has read it
    if (t == 0) {
        const uint32_t left = top - n_take;
        if (gridDim.x == 1) *a.free_count_out = left;
        else if (atomicAdd(a.ticket, 1u) == gridDim.x - 1) {
            *a.free_count_out = left;
            *a.ticket = 0;
        }
    }
}

// ------------------------------------------------------------- rows in, out

// Max over groups of 2, 4 or 8 lanes next to each other, in all of them.
template <int kN>
__device__ __forceinline__ uint32_t kv_near_max(uint32_t v) {
    auto with = [&](uint32_t other) { v = max(v, other); };
    with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));                  // lanes 1 0 3 2 of a quad
    if constexpr (kN >= 4) with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));   // 2 3 0 1
    if constexpr (kN >= 8) with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));  // 7 - lane of eight
    return v;
}

// Where 8 values of a row lie in a plane: piece of 8 within the row of a slot.
struct wh_kv4_at {
    uint64_t code;   // dword index
    uint64_t scale;  // byte index
    bool ok;
};
__device__ __forceinline__ wh_kv4_at kv_at(const wh_kv4_rows_args& a, uint32_t slot, uint32_t piece) {
    const uint32_t pieces = a.s.head_dim / 8, head = piece / pieces, p = piece - head * pieces;
    uint32_t page, row;
    wh_kv4_at r;
    r.ok = wh_kv4_slot_page(slot, a.s.shift, a.s.n_pages, &page, &row);
    if (slot != WH_KV_NONE && !r.ok && p == 0) atomicOr(a.status, WH_ST_NOT_RESIDENT);
    const uint64_t line = wh_kv4_line(page, head, row, a.s.kv_heads, a.s.shift);
    r.code = line * pieces + p;
    r.scale = line * (pieces / 4) + p / 4;
    return r;
}

// Rounds rows into the cache.  A lane takes 8 values, four lanes a group of 32:
// the group's largest magnitude (its bits, so an infinity or NaN shows) gives
// the least power of two under which it is at most 6, the conversion
// instruction rounds to nearest, ties to even.  A group that holds an infinity
// or NaN has codes 0 and byte 255.  Bound by memory, 4.53 bytes in and out for
// an f32 value, 2.53 for bf16: keys and values of 20011 tokens, 8 heads of 128 in
// bf16, 53.6 us, 78 % of the rate of a large copy.
template <bool kBf16>
__global__ void __launch_bounds__(256) k_kv4_write(wh_kv4_rows_args a) {
    const uint32_t pl = blockIdx.y, per = a.s.kv_heads * (a.s.head_dim / 8);
    const uint64_t unit = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (unit >= (uint64_t)a.n * per) return;  // whole quads: per is a multiple of 4
    const uint32_t i = (uint32_t)(unit / per), piece = (uint32_t)(unit - (uint64_t)i * per);
    const wh_kv4_at at = kv_at(a, a.slots[i], piece);
    if (!at.ok) return;
    float v[8];
    if constexpr (kBf16) {
        const wh_u4 w = *(const wh_u4*)((const uint16_t*)a.rows[pl] + i * a.stride[pl] + piece * 8);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = kv_bits(w[k] << 16);
            v[2 * k + 1] = kv_bits(w[k] & 0xffff0000u);
        }
    } else {
        const wh_f4* p = (const wh_f4*)((const float*)a.rows[pl] + i * a.stride[pl] + piece * 8);
        const wh_f4 x = p[0], y = p[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = x[k];
            v[4 + k] = y[k];
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
    top = kv_near_max<4>(top);
    // 1.m * 2^(E - 127) <= 6 * 2^e = 1.5 * 2^(e + 2): e = E - 129, one more when 1.m > 1.5
    const uint32_t exp = top >> 23;
    uint32_t byte = exp < 3 ? 1 : exp - 2 + ((top & 0x7fffffu) > 0x400000u);
    const bool bad = top >= 0x7f800000u;
    const float scale = kv_bits(byte << 23);
    uint32_t c = 0;
    if (!bad) {
        if (byte == 253) {  // 4 * 2^126 is past f32: 3 * 2^126 is the largest finite value
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = fminf(fmaxf(v[k], -3.0f * scale), 3.0f * scale);
        }
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    }
    if (top == 0) byte = 0;
    ((uint32_t*)a.plane[pl].codes)[at.code] = c;
    if ((piece & 3) == 0) a.plane[pl].scales[at.scale] = (uint8_t)(bad ? 255 : byte);
}

// The values that rows of the cache stand for.  Exact in f32 and in bf16: a
// code has two significant bits.  Bound by memory: 50021 rows of 512 to f32 31.2
// us, 75 % of the rate of a large copy.
template <bool kBf16>
__global__ void __launch_bounds__(256) k_kv4_read(wh_kv4_rows_args a) {
    const uint32_t pl = blockIdx.y, per = a.s.kv_heads * (a.s.head_dim / 8);
    const uint64_t unit = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (unit >= (uint64_t)a.n * per) return;
    const uint32_t i = (uint32_t)(unit / per), piece = (uint32_t)(unit - (uint64_t)i * per);
    const wh_kv4_at at = kv_at(a, a.slots[i], piece);
    if (!at.ok) return;
    const uint32_t byte = a.plane[pl].scales[at.scale];
    const uint32_t codes = ((const uint32_t*)a.plane[pl].codes)[at.code], c = byte ? codes : 0;
    const float scale = kv_bits(byte << 23);  // of 0 the conversion makes 2^-127, of 255 NaN
    wh_f2 v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
    if constexpr (kBf16) {
        wh_u4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = (__float_as_uint(v[k].x) >> 16) | (__float_as_uint(v[k].y) & 0xffff0000u);
        *(wh_u4*)((uint16_t*)a.rows[pl] + i * a.stride[pl] + piece * 8) = w;
    } else {
        wh_f4* p = (wh_f4*)((float*)a.rows[pl] + i * a.stride[pl] + piece * 8);
        p[0] = (wh_f4){v[0].x, v[0].y, v[1].x, v[1].y};
        p[1] = (wh_f4){v[2].x, v[2].y, v[3].x, v[3].y};
    }
}

// -------------------------------------------------------------- attention
//
// A request's queries are rows (token, head of the group) of one key head,
// flattened; a workgroup takes a tile of them and a part of the keys that any of
// them sees, and adds weights and values in one pass with the running maximum.
// Softmax in powers of two: w = 2^(s * scale * log2(e) - m).
//
// Numbers.  Scores, bf16: the codes as they lie and the query as two E4M3 parts
// with a power of two for every 32 values (together 2^-9 of a value, and 8 u of
// the largest of the 32), in the scaled matrix instruction; products are exact in
// its f32 sums.  f32: keys decoded to f16 against their row's largest scale byte
// (exact down to 2^-23 of that, kKeyNear; what lies further apart kv_plain_part
// takes, as below) and the query as two f16 parts, the second times 2^10: 22 bits,
// and 2^-48 of its largest value, which is 2^-24 of that of a group of 32 dims up to
// 2^24 below (kQueryNear).  Outputs:
// values are f16 against their row's largest scale byte, exact down to 2^-23 of it,
// and that byte's power of two goes into the weight.  Weights are f16, times 2^8,
// against a reference of each query row: the largest score plus value exponent of
// the keys that this row sees.  So what a row does not see, or sees with no weight,
// takes no bits from it.  bf16 calls take one f16 (11 bits, one more than a bf16
// output keeps beside its sign), f32 calls two.  Sums of weights and of products
// and references are f32.
//
// f16 ends 2^-33 below the reference.  A group of 32 dims that lies as high as its
// row keeps 2^-33 of its largest term, one that lies 2^9 below it 2^-24, which is
// what an f32 sum rounds a term by too; bf16 calls, whose outputs round by 2^-9, allow
// 2^12.  Values past that (kNear), or whose powers of two are too far from 1 for f32
// sums of weights under such references (kLow, kHigh), are left to kv_plain_part,
// which takes the workgroup's part in f32.  That takes five (one short list) to thirty
// times as long (a chunk of 384 tokens, all of whose tiles see such a row).

#define kMinusInf (-__builtin_inff())
constexpr float kMaxFloat = 3.402823466e38f;
constexpr float kMinusBig = -kMaxFloat;  // the reference of no key: finite, so that differences are, and below every score
// Weights are held times 2^kUp: f16 keeps small ones.  A row's reference is raised
// to its largest score once a weight is past f16, 2^8 above: with 2^5 the prompts of
// k_kv4_attn_packed took 290 us for 243.  Rows raise theirs by themselves: that
// another one does changes nothing in a row's rounding.
constexpr float kUp = 8.0f;
constexpr float kMost = 65504.0f;
constexpr uint32_t kApart = 0xffffffffu;  // past every run
constexpr int kKeyNear = 23;              // f32: a key group's scale byte is at most so far below its row's
constexpr int kQueryNear = 24;            // f32: a query's group's exponent is at most so far below the row's
constexpr float kLowPart = 1024.0f;       // f32: what a query's second f16 part is multiplied by
template <bool kF32>
constexpr int kNear = kF32 ? 9 : 12;      // a value group's scale byte is at most so far below its row's
constexpr uint32_t kLow = 127 - 40, kHigh = 127 + 40;  // and the row's in here

// The tile of slot x: a search over the requests, 64 candidates a step.
template <int kRows>
__device__ __forceinline__ wh_kv4_tile kv_tile(const wh_kv4_attn_args& a, uint32_t x) {
    const uint32_t lane = threadIdx.x & 63;
    auto start = [&](uint32_t b) { return min(a.starts[b], a.n_tokens); };
    uint32_t lo = 0, n = a.n_requests;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, b = lo + lane * step;
        const bool le = lane * step < n && wh_kv4_tile_base(start(b), a.group, b, kRows) <= x;
        const uint32_t hits = (uint32_t)__popcll(__ballot(le)), k = hits ? hits - 1 : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const uint32_t s0 = __builtin_amdgcn_readfirstlane(start(lo)), s1 = __builtin_amdgcn_readfirstlane(start(lo + 1));
    const uint32_t len = __builtin_amdgcn_readfirstlane(a.lens[lo]);
    const uint32_t cap = (uint32_t)min(a.table_stride << a.s.shift, (uint64_t)0x7fffffff);
    const wh_kv4_tile r = wh_kv4_tile_of(x, lo, s0, s1, len, cap, a.group, a.window, a.first, kRows);
    if (r.ok && len > cap && threadIdx.x == 0) atomicOr(a.status, WH_ST_NOT_RESIDENT);
    return r;
}

// What a workgroup does: a tile of one key head, and which of its blocks of
// keys.  Key heads lie next to each other in the grid, so that of eight each
// has an XCD's L2 to itself.
struct wh_kv4_place {
    wh_kv4_tile tile;
    uint32_t head, unit;    // unit: where a partial result goes
    uint32_t chunk, split;  // blocks [split * chunk, ...)
};

// Where there are more workgroups than tiles, the requests' lengths decide how
// many share one: every wave adds up all requests (at most WH_KV_SPLIT_REQUESTS)
// and finds its own by the running sum.  by_tile: x counts tiles, and the place
// is their first unit.
template <int kRows>
__device__ __forceinline__ wh_kv4_place kv_place(const wh_kv4_attn_args& a, bool by_tile) {
    wh_kv4_place r;
    const uint32_t x = blockIdx.x / a.s.kv_heads;
    r.head = blockIdx.x % a.s.kv_heads;
    r.unit = x;
    r.split = 0;
    r.chunk = 0x7fffffffu;
    if (a.units <= a.n_tiles) {
        r.tile = kv_tile<kRows>(a, a.n_tiles - 1 - x);  // a prompt's last tiles, which see the most keys, first
        return r;
    }
    const uint32_t lane = threadIdx.x & 63, cap = (uint32_t)min(a.table_stride << a.s.shift, (uint64_t)0x7fffffff);
    auto start = [&](uint32_t b) { return min(a.starts[b], a.n_tokens); };
    uint32_t s0, s1, len, tiles, blocks;  // of this lane's request
    auto request = [&](uint32_t b) {
        const bool ok = b < a.n_requests;
        s0 = ok ? start(b) : 0;
        s1 = ok ? start(b + 1) : 0;
        len = ok ? a.lens[b] : 0;
        const uint32_t n_q = s1 > s0 ? s1 - s0 : 0;
        tiles = wh_kv4_tiles(n_q, a.group, kRows);
        blocks = wh_kv4_runs(n_q, len, cap, a.window, a.first);
    };
    uint64_t sum_tiles = 0, sum_blocks = 0;
    for (uint32_t b = 0; b < a.n_requests; b += 64) {
        request(b + lane);
        sum_tiles += tiles;
        sum_blocks += (uint64_t)tiles * blocks;
    }
    sum_tiles = kv_lane(kv_scan(sum_tiles), 63);
    sum_blocks = kv_lane(kv_scan(sum_blocks), 63);
    uint32_t tile0 = 0, unit0 = 0;  // of the requests before these 64
    r.tile = wh_kv4_tile_of(0, 0, 0, 0, 0, 0, a.group, 0, 0, kRows);  // none
    for (uint32_t b = 0; b < a.n_requests; b += 64) {
        if (a.n_requests > 64) request(b + lane);
        const uint32_t splits = wh_kv4_splits(blocks, sum_blocks, sum_tiles, a.units, a.min_runs);
        // tiles below, their units above
        const uint64_t mine = (uint64_t)(tiles * splits) << 32 | tiles, sum = kv_scan(mine), past = sum - mine;
        const uint64_t hit = __ballot((by_tile ? tile0 + (uint32_t)sum : unit0 + (uint32_t)(sum >> 32)) > x);
        if (hit) {
            const uint32_t src = (uint32_t)__ffsll((unsigned long long)hit) - 1;
            const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)splits, src);
            const uint64_t all_before = kv_lane(past, src);
            const uint32_t before = by_tile ? (uint32_t)all_before : (uint32_t)(all_before >> 32);
            const uint32_t at = x - (by_tile ? tile0 : unit0) - before, local = by_tile ? at : at / n;
            r.chunk = wh_kv4_even((uint32_t)__builtin_amdgcn_readlane((int)blocks, src), n);
            if (by_tile) r.unit = unit0 + (uint32_t)(all_before >> 32) + at * n;
            r.split = by_tile ? 0 : at - local * n;
            const uint32_t q = b + src, from = (uint32_t)__builtin_amdgcn_readlane((int)s0, src);
            const uint32_t rows = (uint32_t)__builtin_amdgcn_readlane((int)len, src);
            r.tile = wh_kv4_tile_of(wh_kv4_tile_base(from, a.group, q, kRows) + local, q, from,
                                    (uint32_t)__builtin_amdgcn_readlane((int)s1, src), rows, cap, a.group, a.window, a.first, kRows);
            if (rows > cap && threadIdx.x == 0) atomicOr(a.status, WH_ST_NOT_RESIDENT);
            break;
        }
        const uint64_t last = kv_lane(sum, 63);
        tile0 += (uint32_t)last;
        unit0 += (uint32_t)(last >> 32);
    }
    // wave-uniform: in scalar registers from here
    r.tile.request = __builtin_amdgcn_readfirstlane(r.tile.request);
    r.tile.row0 = __builtin_amdgcn_readfirstlane(r.tile.row0);
    r.tile.rows = __builtin_amdgcn_readfirstlane(r.tile.rows);
    r.tile.n_q = __builtin_amdgcn_readfirstlane(r.tile.n_q);
    r.tile.token0 = __builtin_amdgcn_readfirstlane(r.tile.token0);
    r.tile.len = __builtin_amdgcn_readfirstlane(r.tile.len);
    r.tile.first = __builtin_amdgcn_readfirstlane(r.tile.first);
    r.tile.from = __builtin_amdgcn_readfirstlane(r.tile.from);
    r.tile.end = __builtin_amdgcn_readfirstlane(r.tile.end);
    r.tile.first_runs = __builtin_amdgcn_readfirstlane(r.tile.first_runs);
    r.tile.lo = __builtin_amdgcn_readfirstlane(r.tile.lo);
    r.tile.runs = __builtin_amdgcn_readfirstlane(r.tile.runs);
    r.tile.ok = __builtin_amdgcn_readfirstlane((int)r.tile.ok) != 0;
    r.unit = __builtin_amdgcn_readfirstlane(r.unit);
    r.split = __builtin_amdgcn_readfirstlane(r.split);
    r.chunk = __builtin_amdgcn_readfirstlane(r.chunk);
    return r;
}

// -inf for the keys key + 16 b + i that position pos (-1: none) does not see.  A
// branch (the empty asm) and not a part of what every run does: the compiler
// would otherwise compare for all of them.
template <int kN>
__device__ __forceinline__ void kv_mask(wh_f4 (&s)[kN], int32_t pos, uint32_t key, uint32_t window, uint32_t first) {
    asm volatile("");
    const int32_t past = pos - (int32_t)key;  // the last offset that is not past pos
#pragma unroll
    for (int b = 0; b < kN; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[b][i] = 16 * b + i <= past ? s[b][i] : kMinusInf;
    if (window) {
        const int32_t near = past - (int32_t)window, early = (int32_t)first - (int32_t)key;
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[b][i] = ((16 * b + i > near) | (16 * b + i < early)) ? s[b][i] : kMinusInf;
    }
}

// max over the bytes of w
__device__ __forceinline__ uint32_t kv_max_bytes(uint32_t w) {
    const uint32_t m = max(w & 0xff, (w >> 8) & 0xff);
    return max(max(m, (w >> 16) & 0xff), w >> 24);
}

// Eight codes times 2^(relative scale) as f16, exact.
__device__ __forceinline__ wh_h8 kv_decode(uint32_t c, float scale) {
    union {
        wh_h2 h[4];
        wh_h8 v;
    } u;
    u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0);
    u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1);
    u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2);
    u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3);
    return u.v;
}

__device__ __forceinline__ void kv_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A barrier that orders LDS only: loads in flight go on.
__device__ __forceinline__ void kv_lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Raw rows of a lane: key lane % 16 of kN blocks of 16, of each 128 dims the 32
// that are chunk g (of 64 the 32 that are chunk g % 2), and all its scale bytes.
template <int HD, int kN>
struct wh_kv4_raw {
    static constexpr int kPieces = HD >= 128 ? HD / 128 : 1;
    uint32_t c[kN][kPieces][4];
    uint32_t s[kN][kPieces];
};

template <int HD, int kN>
__device__ __forceinline__ void kv_load(wh_kv4_raw<HD, kN>& r, int half, const wh_kv4_plane& p, uint64_t line, uint32_t g) {
    const uint8_t* const c = p.codes + line * (HD / 2) + 16 * (HD == 64 ? g & 1 : g);
#pragma unroll
    for (int j = 0; j < r.kPieces; ++j) {
        const wh_u4 w = *(const wh_u4*)(c + 64 * j);
#pragma unroll
        for (int k = 0; k < 4; ++k) r.c[half][j][k] = w[k];
    }
    const uint8_t* const s = p.scales + line * (HD / 32);
    if constexpr (HD == 64) r.s[half][0] = *(const uint16_t*)s;
    else if constexpr (HD == 128) r.s[half][0] = *(const uint32_t*)s;
    else if constexpr (HD == 256) {
        const wh_u2 w = *(const wh_u2*)s;
        r.s[half][0] = w[0];
        r.s[half][1] = w[1];
    } else {
        const wh_u4 w = *(const wh_u4*)s;
#pragma unroll
        for (int k = 0; k < 4; ++k) r.s[half][k] = w[k];
    }
}
// The largest scale byte of a raw row.
template <int HD, int kN>
__device__ __forceinline__ uint32_t kv_top_byte(const wh_kv4_raw<HD, kN>& r, int half) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < r.kPieces; ++k) m = max(m, kv_max_bytes(r.s[half][k]));
    return m;
}

// Scale bytes of a lane's pieces, piece j in byte j.
template <int HD, int kN>
__device__ __forceinline__ uint32_t kv_piece_scales(const wh_kv4_raw<HD, kN>& r, int half, uint32_t g) {
    const uint32_t pick = g | (4 + g) << 8;
    if constexpr (HD == 64) return (r.s[half][0] >> (8 * (g & 1))) & 0xff;
    if constexpr (HD == 128) return (r.s[half][0] >> (8 * g)) & 0xff;
    if constexpr (HD == 256) return __builtin_amdgcn_perm(r.s[half][1], r.s[half][0], pick) & 0xffff;
    if constexpr (HD == 512)
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(r.s[half][3], r.s[half][2], pick),
                                     __builtin_amdgcn_perm(r.s[half][1], r.s[half][0], pick), 0x05040100u);
    return 0;
}

// Scale of piece j relative to the row's largest byte: 2^0 at most, so that
// decoded values are finite whatever the bytes are.
template <int HD, int kN>
__device__ __forceinline__ float kv_rel(const wh_kv4_raw<HD, kN>& r, int half, int j, uint32_t g, uint32_t top) {
    const uint32_t b = HD == 64 ? (r.s[half][0] >> (8 * (g & 1))) & 0xff : (r.s[half][j] >> (8 * g)) & 0xff;
    return kv_bits((uint32_t)max((int)b - (int)top + 127, 0) << 23);
}

// 2^(byte - 127) of a key row, or NaN where it or its value row holds one: the
// score is NaN then, and with it the weight, in the rows that see the key.
__device__ __forceinline__ float kv_key_scale(uint32_t ktop, uint32_t vtop) {
    return ktop == 255 || vtop == 255 ? kv_bits(0x7fc00000u) : kv_bits(ktop << 23);
}
// The exponent byte that a value row's weights take, from its largest scale byte
// (0: a row of zeros; 255: NaN, whose weights are NaN or 0).
__device__ __forceinline__ uint32_t kv_value_top(uint32_t top) { return min(max(top, kLow), kHigh); }
// A value group's scale against that: a power of two of at most 1, as f16, and 0
// from 2^-15 on (kNear is less).
__device__ __forceinline__ _Float16 kv_value_rel(uint32_t b, uint32_t vexp) {
    union {
        uint16_t u;
        _Float16 h;
    } x;
    x.u = (uint16_t)((min(max((int)b - (int)vexp, -15), 0) + 15) << 10);
    return x.h;
}
// The same of a key row's group, in f32.
__device__ __forceinline__ bool kv_key_odd(uint32_t b, uint32_t top) { return (int)top - (int)b > kKeyNear; }
// Whether a group of a value row (top: its largest byte) is to be looked at: not held
// by f16 products, or NaN, or zeros.
template <bool kF32>
__device__ __forceinline__ bool kv_value_odd(uint32_t b, uint32_t top, uint32_t vexp) {
    return ((int)b - (int)vexp < -kNear<kF32>) | (vexp != top);
}

// First dim of a lane's eight in step s of the product with keys.
template <int HD>
__device__ __forceinline__ int kv_dim(int s, uint32_t g) {
    return HD >= 128 ? 32 * (4 * (s >> 2) + (int)g) + 8 * (s & 3) : 32 * ((int)g & 1) + 16 * ((int)g >> 1) + 8 * s;
}

// Max over groups of sixteen lanes, in all of them.
__device__ __forceinline__ uint32_t kv_row_max(uint32_t v) {
    v = kv_near_max<8>(v);
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));  // 15 - lane
}
// Max over the wave, in all lanes.
__device__ __forceinline__ uint32_t kv_wave_max(uint32_t v) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    v = kv_row_max(v);
    u2 p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p[0], p[1]);
    p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(p[0], p[1]);
}

// Queries in f32: the waves share a tile's rows, sixteen lanes a row, and leave
// each in LDS as two f16 parts against its largest exponent.
template <int HD, int kRows, int kWaves>
struct wh_kv4_query {
    static constexpr int kLd = HD + 8;                        // f16 between rows
    static constexpr int kEach = kRows / kWaves / 4;          // rows of a lane
    static constexpr int kBytes = 2 * kRows * kLd * 2;
    wh_u4 raw[kEach][HD / 64];

    __device__ __forceinline__ static uint32_t row(int i, uint32_t wave, uint32_t lane) { return 4 * (kEach * wave + i) + (lane >> 4); }

    // at(row): the row's first value
    template <class At>
    __device__ __forceinline__ void load(uint32_t wave, uint32_t lane, At at) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float* const p = at(row(i, wave, lane)) + 4 * (lane & 15);
#pragma unroll
            for (int k = 0; k < HD / 64; ++k) raw[i][k] = *(const wh_u4*)(p + 64 * k);
        }
    }

    // factor[row]: what a sum of products with the row is to be multiplied by,
    // `scale` included.  Sums are below 2^26: whether that takes finite ones past
    // f32 before the key's power of two brings them back, or is subnormal itself;
    // or a group of 32 dims lies too far below the row's largest value.
    __device__ __forceinline__ bool put(uint32_t wave, uint32_t lane, _Float16* lds, float* factor, float scale) const {
        bool far = false;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            // the largest of each group of 32 dims, eight lanes, and of the row
            uint32_t top = 0, low = 0x7fffffffu;
#pragma unroll
            for (int k = 0; k < HD / 64; ++k) {
                uint32_t group = 0;
#pragma unroll
                for (int n = 0; n < 4; ++n) group = max(group, raw[i][k][n] & 0x7fffffffu);
                group = kv_near_max<8>(group);
                top = max(top, group);
                low = min(low, group - 1);  // zeros are of no size
            }
            top = kv_row_max(top);
            far |= top < 0x7f800000u && (int)(top >> 23) - (int)((low + 1) >> 23) > kQueryNear;
            const int e = max((int)(top >> 23), 27);  // of the largest; 2^-100 at least, so that the factor is finite
            const float up = kv_bits((uint32_t)(127 + 13 + 127 - e) << 23);
            const uint32_t r = row(i, wave, lane);
            _Float16* const dst = lds + r * kLd + 4 * (lane & 15);
#pragma unroll
            for (int k = 0; k < HD / 64; ++k) {
                union {
                    _Float16 h[4];
                    wh_u2 u;
                } hi, lo;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float x = kv_bits(raw[i][k][n]) * up;
                    hi.h[n] = (_Float16)x;
                    lo.h[n] = (_Float16)((x - (float)hi.h[n]) * kLowPart);
                }
                *(wh_u2*)(dst + 64 * k) = hi.u;
                *(wh_u2*)(dst + kRows * kLd + 64 * k) = lo.u;
            }
            const float c = scale * kv_bits((uint32_t)(e - 13) << 23), size = fabsf(c);
            if ((lane & 15) == 0) factor[r] = c;
            far |= e < 255 && scale != 0.0f && !(size >= 0x1p-126f && size < 0x1p102f);
        }
        return far;
    }

    // A lane's operands: the parts of a row's dims kv_dim(step, g) ..
    __device__ __forceinline__ static void get(wh_h8 (&q)[HD / 32][2], const _Float16* lds, uint32_t row, uint32_t g) {
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
#pragma unroll
            for (int p = 0; p < 2; ++p) q[s][p] = *(const wh_h8*)(lds + (p * kRows + row) * kLd + kv_dim<HD>(s, g));
    }
};

// Four output values at `at`, in the type of the call.
template <bool kF32>
__device__ __forceinline__ void kv_store(void* out, uint64_t at, const wh_f4& x) {
    if constexpr (kF32) {
        *(wh_f4*)((float*)out + at) = x;
    } else {
        union {
            __bf16 b[4];
            wh_u2 u;
        } y;
#pragma unroll
        for (int k = 0; k < 4; ++k) y.b[k] = (__bf16)x[k];
        *(wh_u2*)((uint16_t*)out + at) = y.u;
    }
}

// A lane's 32 of 128 bf16 values of a query as two E4M3 parts: dims 16g .. of
// the first half and of the second, where the instruction wants 8-bit values (it
// takes 4-bit ones and all scales as 32g ..).  Returns the first part's scale
// byte for dims 32g .. (the second's is 4 less), 255 where one is not finite.
__device__ __forceinline__ uint32_t kv_query_e4m3(const wh_u4 (&raw)[2][2], uint32_t flip, wh_i8& hi, wh_i8& lo) {
    int e[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t w = raw[h][i][k];
                top = max(top, max((w << 16) & 0x7fffffffu, w & 0x7fff0000u));
            }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));  // the other 16 of the 32
        e[h] = max((int)(top >> 23), 11);  // the second part's byte is 11 less
        const float up = kv_bits((uint32_t)(127 + 127 + 7 - min(e[h], 254)) << 23);  // the largest to [2^7, 2^8)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int a = 0, b = 0;
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t w = raw[h][i >> 1][2 * (i & 1) + (k >> 1)] ^ flip;
                x[k] = kv_bits(k & 1 ? w & 0xffff0000u : w << 16) * up;
            }
            a = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], a, false);
            a = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], a, true);
            const wh_f2 u = __builtin_amdgcn_cvt_pk_f32_fp8(a, false), v = __builtin_amdgcn_cvt_pk_f32_fp8(a, true);
            b = __builtin_amdgcn_cvt_pk_fp8_f32((x[0] - u.x) * 16.0f, (x[1] - u.y) * 16.0f, b, false);
            b = __builtin_amdgcn_cvt_pk_fp8_f32((x[2] - v.x) * 16.0f, (x[3] - v.y) * 16.0f, b, true);
            hi[4 * h + i] = a;
            lo[4 * h + i] = b;
        }
    }
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, from = (lane & 15) + 32 * (g & 1);
    const int e0 = __shfl(e[0], (int)from, 64), e1 = __shfl(e[1], (int)from, 64), w = g < 2 ? e0 : e1;
    return w == 255 ? 255u : (uint32_t)(w - 7);
}

// Max and sum over the four lanes of a row (lane % 16), in all of them.
__device__ __forceinline__ float kv_max_groups(float v) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    u2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
// Sum over the wave, in all lanes.
__device__ __forceinline__ float kv_wave_sum(float v) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k, 64);
    return v;
}
__device__ __forceinline__ float kv_sum_groups(float v) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    u2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// A power of two's exponent.
__device__ __forceinline__ int kv_exponent(float power) { return (int)(__float_as_uint(power) >> 23) - 127; }

// A part's sum of weights, l * 2^m, as a power of two and a factor in [.5, 1): by
// it parts are compared, since references include the values' exponents.
__device__ __forceinline__ void kv_put_sum(float* to, float m, float l) {
    to[0] = m + (float)__builtin_amdgcn_frexp_expf(l);
    to[1] = __builtin_amdgcn_frexp_mantf(l);
}

// A workgroup's part of a tile in plain f32: for values, or in f32 calls queries and
// keys, that f16 products do not hold (above).  A wave takes up to eight rows, a lane
// a key of their scores and HD / 64 dims of their outputs.  Outputs are kept divided
// by the sum of weights so far, so they stay within the values' size whatever that
// is.  Bound by instruction issue: HD products a row and key, without the matrix
// instructions.
template <int HD, bool kF32, bool kLatent, int kRows, int kWaves>
__device__ __forceinline__ void kv_plain_part(const wh_kv4_attn_args& a, const wh_kv4_place& place, uint32_t wave) {
    constexpr int kPer = HD / 64;  // dims of a lane
    constexpr int kMany = kRows / kWaves < 8 ? kRows / kWaves : 8;
    const uint32_t lane = threadIdx.x & 63, kvh = place.head, pmask = (1u << a.s.shift) - 1u;
    const wh_kv4_tile& tile = place.tile;
    const uint32_t run0 = place.split ? place.split * place.chunk : 0, run1 = min(tile.runs, run0 + place.chunk);
    const bool whole = place.chunk >= tile.runs;
    const uint32_t* const table = a.tables + tile.request * a.table_stride;
    bool bad = false;
    for (uint32_t first = kMany * wave; first < tile.rows; first += kMany * kWaves) {
        uint64_t at_q[kMany];
        int32_t pos[kMany];
        float m[kMany], l[kMany], o[kMany][kPer];
#pragma unroll
        for (int r = 0; r < kMany; ++r) {
            const uint32_t flat = tile.row0 + min(first + r, tile.rows - 1), tok = flat / a.group;
            pos[r] = tile.len - (int32_t)tile.n_q + (int32_t)tok;
            at_q[r] = (uint64_t)(tile.token0 + tok) * a.q_stride + (uint64_t)(kvh * a.group + (flat - tok * a.group)) * HD;
            m[r] = kMinusBig;
            l[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[r][i] = 0.0f;
        }
        for (uint32_t run = run0; run < run1; ++run) {
            const uint32_t key0 = wh_kv4_run(tile, run), key = key0 + lane;
            const bool some = wh_kv4_seen(tile, key0, key) == key;
            const uint32_t page = table[wh_kv4_seen(tile, key0, key) >> a.s.shift];
            const bool out = page >= a.s.n_pages;
            bad |= out;
            const uint64_t line = wh_kv4_line(out ? 0 : page, kvh, key & pmask, a.s.kv_heads, a.s.shift);
            float s[kMany];
#pragma unroll
            for (int r = 0; r < kMany; ++r) s[r] = 0.0f;
            uint32_t n0 = 0;
            asm volatile("" : "+s"(n0));  // queries are not to be held over the runs: there are no registers
#pragma unroll 1
            for (uint32_t n = n0; n < HD / 32; ++n) {
                const uint32_t byte = a.k.scales[line * (HD / 32) + n];
                const float scale = kv_bits(byte << 23);
                wh_u4 codes = *(const wh_u4*)(a.k.codes + line * (HD / 2) + 16 * n);
                if (byte == 0) codes = (wh_u4){0, 0, 0, 0};
                float k[32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const wh_f2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 0),
                                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 1),
                                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 2),
                                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], scale, 3)};
#pragma unroll
                    for (int e = 0; e < 8; ++e) k[8 * i + e] = e & 1 ? v[e >> 1].y : v[e >> 1].x;
                }
#pragma unroll
                for (int r = 0; r < kMany; ++r) {
                    __builtin_amdgcn_sched_barrier(0);  // nor all rows' at once
                    // sixteen bytes that all lanes read
                    if constexpr (kF32) {
#pragma unroll
                        for (int h = 0; h < 8; ++h) {
                            const wh_f4 q = *(const wh_f4*)((const float*)a.q + at_q[r] + 32 * n + 4 * h);
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[r] = fmaf(q[e], k[4 * h + e], s[r]);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const wh_u4 q = *(const wh_u4*)((const uint16_t*)a.q + at_q[r] + 32 * n + 8 * h);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                s[r] = fmaf(kv_bits(e & 1 ? q[e >> 1] & 0xffff0000u : q[e >> 1] << 16), k[8 * h + e], s[r]);
                        }
                    }
                }
            }
            bool nan = false;  // a value row that holds NaN makes all of the output NaN
            if constexpr (!kLatent)
#pragma unroll 1
                for (int n = 0; n < HD / 32; ++n) nan |= a.v.scales[line * (HD / 32) + n] == 255;
            float p[kMany];
#pragma unroll
            for (int r = 0; r < kMany; ++r) {
                const bool sees = (int64_t)key <= pos[r] && (!a.window || (int64_t)key > (int64_t)pos[r] - a.window || key < a.first);
                const float x = !sees ? kMinusInf : nan ? kv_bits(0x7fc00000u) : s[r] * a.scale_log2;
                const float to = fmaxf(m[r], wh_wave_max(x)), f = l[r] * __builtin_amdgcn_exp2f(m[r] - to), w = __builtin_amdgcn_exp2f(x - to);
                l[r] = f + kv_wave_sum(w);
                m[r] = to;
                const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
                p[r] = w * inv;
#pragma unroll
                for (int i = 0; i < kPer; ++i) o[r][i] *= f * inv;
            }
            const uint64_t seen = __ballot(some);
#pragma unroll 8
            for (int j = 0; j < 64; ++j) {
                const uint64_t at = kv_lane(line, j);
                const uint8_t* const codes = a.v.codes + at * (HD / 2) + lane * kPer / 2;
                uint32_t code;
                if constexpr (kPer == 8) code = *(const uint32_t*)codes;
                else if constexpr (kPer == 4) code = *(const uint16_t*)codes;
                else code = *codes;
                uint32_t byte = a.v.scales[at * (HD / 32) + lane * kPer / 32];
                // finite for the rows that do not see it: their weight is 0
                if (!(seen >> j & 1) || byte == 255) byte = 0;
                if (byte == 0) code = 0;
                const float scale = kv_bits(byte << 23);
                float v[kPer];
                if constexpr (kPer == 1) {
                    const wh_f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0);
                    v[0] = lane & 1 ? x.y : x.x;
                } else {
                    wh_static_for<kPer / 2>([&](auto ic) {
                        constexpr int i = decltype(ic)::value;
                        const wh_f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, i);
                        v[2 * i] = x.x;
                        v[2 * i + 1] = x.y;
                    });
                }
#pragma unroll
                for (int i = 0; i < kPer; ++i) v[i] = fminf(fmaxf(v[i], -kMaxFloat), kMaxFloat);
#pragma unroll
                for (int r = 0; r < kMany; ++r) {
                    const float pj = kv_bits((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(p[r]), j));
#pragma unroll
                    for (int i = 0; i < kPer; ++i) o[r][i] = fmaf(pj, v[i], o[r][i]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kMany; ++r) {
            const uint32_t row = first + r;
            if (row >= tile.rows) continue;
            const uint32_t flat = tile.row0 + row, tok = flat / a.group, head = kvh * a.group + (flat - tok * a.group);
            float* const part = a.part + (((uint64_t)place.unit * a.s.kv_heads + kvh) * kRows + row) * (HD + 2);
            float f = 1.0f;
            if (whole && a.sink && l[r] > 0.0f) f = l[r] / (l[r] + __builtin_amdgcn_exp2f(a.sink[head] * 1.44269504088896340736f - m[r]));
            const uint64_t at = (uint64_t)(tile.token0 + tok) * a.out_stride + (uint64_t)head * HD + lane * kPer;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (!whole) part[lane * kPer + i] = o[r][i];
                else if constexpr (kF32) ((float*)a.out)[at + i] = o[r][i] * f;
                else ((__bf16*)a.out)[at + i] = (__bf16)(o[r][i] * f);
            }
            if (!whole && lane == 0) kv_put_sum(part + HD, m[r], l[r]);
        }
    }
    if (bad) atomicOr(a.status, WH_ST_NOT_RESIDENT);
}

// Four waves share a tile of 16 rows; wave w takes the blocks of 64 keys w, w +
// 4, ... of the workgroup's run with a softmax of its own, and the four are
// joined at the end: no barrier between waves before that.  Scores are formed as
// [key][row]: lane (row, g) holds the keys 16 b + 4 g + i of four blocks b.  The
// value rows' codes go through the wave's own LDS as they lie and come back
// transposed, sixteen keys of one dim a lane (the 4-bit transposing read), whose
// source rows are chosen to be just these keys: a lane's weights are the operand
// of the product with the values as they are.  A key's codes are decoded for 16 rows
// at most, which keeps every unit short of full: 32 tokens, up to 8192 keys, 8 heads
// on each of 8 key heads of 128, bf16: 57 us and 6 for the join, 3.4 TB/s of cache (a
// copy: 4.9), vector instructions 43 % and matrix ones 8 % of the cycles, waves
// waiting for 35 % of theirs; 96 windows, 4 heads a key head, f32: 41 us.  Up to 128
// dims two waves a SIMD with all registers as vector ones: one a SIMD, which puts
// accumulators aside, takes 58.6 us in all instead of 56.5 and 41.5 instead of 40.4.
template <int HD, bool kF32>
struct wh_kv4_narrow {
    static constexpr bool kDirect = !kF32;                   // scores on codes as they lie
    static constexpr int kParts = kF32 ? 2 : 1;
    static constexpr int kPieces = HD / 128 ? HD / 128 : 1;
    static constexpr int kHold = HD >= 256 ? 2 : 4;          // blocks of 16 keys whose rows are held at once
    static constexpr int kRow = HD / 2;                      // bytes of a row's codes
    static constexpr int kGroups = HD / 32, kRel = 72;       // f16 between groups of value scales
    static constexpr int kAtRel = 64 * kRow;                 // byte offsets in a wave's LDS
    static constexpr int kAtKeys = kAtRel + kGroups * kRel * 2;
    static constexpr int kAtPow = kAtKeys + (kDirect ? 0 : 64 * 4);
    static constexpr int kWave = kAtPow + 64 * 4;
    static constexpr size_t kLds = 4 * (size_t)kWave > 2 * 64 * (size_t)HD ? 4 * (size_t)kWave : 2 * 64 * (size_t)HD;
    using Query = wh_kv4_query<HD, 16, 4>;  // f32: as parts in LDS before the first block
    static_assert(!kF32 || (size_t)Query::kBytes <= kLds, "queries fit");
};

template <int HD, bool kF32, bool kLatent>
__global__ void __launch_bounds__(256, HD <= 128 ? 2 : 1) k_kv4_attn(wh_kv4_attn_args a) {
    using W = wh_kv4_narrow<HD, kF32>;
    constexpr int kParts = W::kParts, kHold = W::kHold, kPieces = W::kPieces;
    constexpr bool kDirect = W::kDirect;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float wave_m[4][16], wave_l[4][16], row_c[kF32 ? 16 : 1];
    __shared__ uint32_t wave_apart[4];
    const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, r16 = lane & 15, g = lane >> 4;
    const wh_kv4_place place = kv_place<16>(a, false);
    const uint32_t kvh = place.head;
    const wh_kv4_tile tile = place.tile;
    if (!tile.ok) return;
    const uint32_t blocks = tile.runs;
    const uint32_t blk0 = place.split ? place.split * place.chunk : 0, blk1 = min(blocks, blk0 + place.chunk);
    if (place.split && blk0 >= blocks) return;
    const bool whole = place.chunk >= blocks;

    // this lane's row
    const uint32_t flat = tile.row0 + min(r16, tile.rows - 1), tok = flat / a.group;
    const uint32_t head = kvh * a.group + (flat - tok * a.group);
    const bool live = r16 < tile.rows;
    const uint32_t token = tile.token0 + tok;
    const int32_t pos = live ? tile.len - (int32_t)tile.n_q + (int32_t)tok : -1;
    const int32_t pos_lo = tile.len - (int32_t)tile.n_q + (int32_t)(tile.row0 / a.group);
    const int32_t pos_hi = tile.len - (int32_t)tile.n_q + (int32_t)((tile.row0 + tile.rows - 1) / a.group);

    // rows are requested kHold blocks of 16 ahead, their pages twice that
    const uint32_t* const table = a.tables + tile.request * a.table_stride;
    const uint32_t pmask = (1u << a.s.shift) - 1u;
    wh_kv4_raw<HD, kHold> kr, vr;
    uint32_t page[kHold];
    bool bad = false;
    // n counts parts of kHold blocks of 16
    constexpr uint32_t kParts64 = 4 / kHold;
    auto run_of = [&](uint32_t n) { return wh_kv4_run(tile, min(n / kParts64, blk1 - 1)); };
    auto key_of = [&](uint32_t n, int h) { return run_of(n) + 16 * (kHold * (n % kParts64) + h) + r16; };
    // the part after part n of this wave
    auto after = [&](uint32_t n) { return n % kParts64 == kParts64 - 1 ? n + 1 + 3 * kParts64 : n + 1; };
    auto request_pages = [&](uint32_t n) {
#pragma unroll
        for (int h = 0; h < kHold; ++h) page[h] = table[wh_kv4_seen(tile, run_of(n), key_of(n, h)) >> a.s.shift];
    };
    auto request = [&](uint32_t n) {
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
            const bool out = page[h] >= a.s.n_pages;
            bad |= out;
            const uint64_t line = wh_kv4_line(out ? 0 : page[h], kvh, key_of(n, h) & pmask, a.s.kv_heads, a.s.shift);
            kv_load(kr, h, a.k, line, g);
            if constexpr (!kLatent) kv_load(vr, h, a.v, line, g);
        }
        request_pages(after(n));
    };
    const uint32_t part0 = (blk0 + wave) * kParts64;
    const bool any = blk0 + wave < blk1;
    if (any) request_pages(part0);

    // the row's query
    bool apart = false;  // what f16 products do not hold
    wh_h8 qd[kDirect ? 1 : HD / 32][kParts];
    wh_i8 qx[kDirect ? kPieces : 1][2];
    uint32_t q_scale = 0;
    float c;  // a score is its sum times this (and its key's power of two, unless direct)
    {
        if constexpr (kDirect) {
            const uint16_t* const p = (const uint16_t*)a.q + (uint64_t)token * a.q_stride + (uint64_t)head * HD + 16 * g;
            wh_u4 raw[kPieces][2][2];
#pragma unroll
            for (int j = 0; j < kPieces; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    raw[j][i >> 1][i & 1] = HD == 64 && i >= 2 ? (wh_u4){0, 0, 0, 0} : *(const wh_u4*)(p + 128 * j + 64 * (i >> 1) + 8 * (i & 1));
            if (any) request(part0);
#pragma unroll
            for (int j = 0; j < kPieces; ++j)
                q_scale |= kv_query_e4m3(raw[j], a.scale_log2 < 0.0f ? 0x80008000u : 0u, qx[j][0], qx[j][1]) << (8 * j);
            c = fmaxf(fabsf(a.scale_log2), 1.0e-37f);
        } else {
            typename W::Query query;
            query.load(wave, lane, [&](uint32_t r) {
                const uint32_t f = tile.row0 + min(r, tile.rows - 1), n = f / a.group;
                return (const float*)a.q + (uint64_t)(tile.token0 + n) * a.q_stride + (uint64_t)(kvh * a.group + f - n * a.group) * HD;
            });
            if (any) request(part0);
            apart = query.put(wave, lane, (_Float16*)smem, row_c, a.scale_log2);
            kv_lds_barrier();
            W::Query::get(qd, (const _Float16*)smem, r16, g);
            c = row_c[r16];
            kv_lds_barrier();
        }
    }

    wh_f4 acc[HD / 16];  // [dim 16 f + 4g + i][row]
#pragma unroll
    for (int f = 0; f < HD / 16; ++f) acc[f] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};
    float m = kMinusBig, l = 0.0f;  // of the row, in all its lanes: the reference, and this lane's sum of weights

    uint8_t* const mine = smem + wave * W::kWave;
    _Float16* const rel = (_Float16*)(mine + W::kAtRel);  // [group][16 g + 4 b + i of key 16 b + 4 g + i]
    float* const key_s = (float*)(mine + W::kAtKeys);     // powers of two of keys
    float* const pow_s = (float*)(mine + W::kAtPow);      // and of value rows
    // 16-byte chunk c of key's row lies at chunk c ^ swizzle: neither the rows that a store
    // meets (b fixed) nor those of a transposed read (g fixed) share banks
    auto swizzle = [](uint32_t key) {
        const uint32_t i = key & 3, b = ((key >> 4) + (key >> 2)) & 3;
        return HD == 512 ? i | b << 2 : HD == 256 ? i >> 1 | b << 1 : HD == 128 ? b : b & 1;
    };
    const uint32_t tkey = 16 * (r16 >> 2) + 4 * g + (r16 & 3);  // this lane's source row of a transposed read

    uint32_t end = blk1;  // 0 once the values are apart: not a second way out, which costs registers
    for (uint32_t blk = blk0 + wave; blk < end; blk += 4) {
        wh_f4 s[4];
        const uint32_t key0 = wh_kv4_run(tile, blk);
        kv_wave_order();
        wh_static_for<(int)kParts64>([&](auto pc) {
            constexpr int part = decltype(pc)::value;
#pragma unroll
            for (int h = 0; h < kHold; ++h) {
                const int b = kHold * part + h;
                const uint32_t key = 16 * b + r16, at = 16 * (r16 >> 2) + 4 * b + (r16 & 3);
                const auto& raw_v = kLatent ? kr : vr;
                const uint32_t kbytes = kDirect ? kv_piece_scales(kr, h, g) : kv_top_byte(kr, h);
                const uint32_t vbytes = kLatent && kDirect ? kbytes : kv_piece_scales(raw_v, h, g);
                const uint32_t vtop = kLatent && !kDirect ? kbytes : kv_top_byte(raw_v, h), vexp = kv_value_top(vtop);
                // value scales, and the powers of two of keys and value rows
                bool odd = false;
                const uint32_t kpieces = kDirect ? kbytes : kv_piece_scales(kr, h, g);
                if constexpr (!kLatent) {  // a latent row's groups are values too, and kNear is less
#pragma unroll
                    for (int j = 0; j < kPieces; ++j) {
                        const uint32_t b = (kpieces >> (8 * j)) & 0xff;
                        odd |= kDirect ? b == 0 : kv_key_odd(b, kbytes);
                    }
                }
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    const uint32_t e = (vbytes >> (8 * j)) & 0xff;
                    odd |= kv_value_odd<kF32>(e, vtop, vexp);
                    if (HD > 64 || g < 2) rel[(4 * j + g) * W::kRel + at] = kv_value_rel(e, vexp);
                }
                const uint64_t odds = __ballot(odd);
                if (__builtin_expect(odds != 0, 0)) {
                    bool far = false;  // a group of a row without NaN, not zeros
#pragma unroll
                    for (int j = 0; j < kPieces; ++j) {
                        const uint32_t kb = (kpieces >> (8 * j)) & 0xff, vb = (vbytes >> (8 * j)) & 0xff;
                        if constexpr (kDirect)  // the instruction takes a byte of 0 as 2^-127
#pragma unroll
                            for (int k = 0; k < 4; ++k) kr.c[h][j][k] = kb ? kr.c[h][j][k] : 0;
                        far |= vb != 0 && vtop != 255 && kv_value_odd<kF32>(vb, vtop, vexp);
                        if constexpr (!kDirect && !kLatent) far |= kb != 0 && kbytes != 255 && kv_key_odd(kb, kbytes);
                    }
                    apart |= far && wh_kv4_seen(tile, key0, key0 + key) == key0 + key;
                }
                if (g == 0) {
                    pow_s[key] = kv_bits(vexp << 23);
                    if constexpr (!kDirect) key_s[key] = kv_key_scale(kbytes, vtop);
                }
                // the value row's codes
                uint8_t* const row = mine + key * W::kRow;
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    const uint32_t* const cw = kLatent ? kr.c[h][j] : vr.c[h][j];
                    if (HD > 64 || g < 2) *(wh_u4*)(row + 16 * ((4 * j + g) ^ swizzle(key))) = (wh_u4){cw[0], cw[1], cw[2], cw[3]};
                }
                // scores
                s[b] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (kDirect) {
                    wh_static_for<kPieces>([&](auto jc) {
                        constexpr int j = decltype(jc)::value;
                        wh_i8 x;
                        x[0] = kr.c[h][j][0], x[1] = kr.c[h][j][1], x[2] = kr.c[h][j][2], x[3] = kr.c[h][j][3];
                        x[4] = x[5] = x[6] = x[7] = 0;
#pragma unroll
                        for (int p = 1; p >= 0; --p)
                            s[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, qx[j][p], s[b], 4, 0, j, kbytes, j,
                                                                                    q_scale - (p ? 0x04040404u : 0u));
                    });
                } else {
                    wh_f4 s_low = s[b];  // of the second parts
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) {
                        const int j = k / 4, w = k - j * 4;
                        const uint32_t codes = HD == 64 && g >= 2 ? kr.c[h][j][w + 2] : kr.c[h][j][w];
                        const wh_h8 x = kv_decode(codes, kv_rel(kr, h, j, g, kbytes));
                        s_low = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qd[k][kParts - 1], s_low, 0, 0, 0);
                        s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qd[k][0], s[b], 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[b][i] = fmaf(s_low[i], 1.0f / kLowPart, s[b][i]);
                }
                // direct: a value row that holds NaN beside keys that do not
                if constexpr (kDirect && !kLatent) {
                    if (__builtin_expect(odds != 0, 0)) {
                        const uint64_t hit = __ballot(vtop == 255);  // bit r16: key 16 b + r16, by every g
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (hit >> (4 * g + i) & 1) s[b][i] = kv_bits(0x7fc00000u);
                    }
                }
            }
            // the next rows come into the registers of these: not before they are used
#pragma unroll
            for (int h = 0; h < kHold; ++h) asm volatile("" : "+v"(s[kHold * part + h])::"memory");
            request(after(blk * kParts64 + part));
        });
        kv_wave_order();
        // -inf where the row does not see a key
        if constexpr (!kDirect) {
#pragma unroll
            for (int b = 0; b < 4; ++b) s[b] *= *(const wh_f4*)&key_s[16 * b + 4 * g] * c;
        }
        const bool all = (int32_t)key0 + 63 <= pos_lo && tile.rows == 16 && (!a.window || (int64_t)key0 + a.window > pos_hi);
        if (!all) kv_mask(s, pos, key0 + 4 * g, a.window, a.first);
        wh_h8 ph[2], pl[2];
        float add, most;
        auto weights = [&] {
            const float up = kUp - m;
            add = most = 0.0f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const wh_f4 power = *(const wh_f4*)&pow_s[16 * b + 4 * g];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = __builtin_amdgcn_exp2f(kDirect ? fmaf(s[b][i], c, up) : s[b][i] + up), x = w * power[i];
                    add += w;
                    most = fmaxf(most, x);
                    const int n = 4 * (b & 1) + i;
                    ph[b >> 1][n] = (_Float16)x;
                    if constexpr (kF32) pl[b >> 1][n] = (_Float16)(x - (float)ph[b >> 1][n]);
                }
            }
        };
        weights();
        if (__ballot(most > kMost)) {  // rows with such a weight take their largest score plus exponent as the reference
            float top = kMinusInf;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    top = fmaxf(top, s[b][i] * (kDirect ? c : 1.0f) + (float)kv_exponent(pow_s[16 * b + 4 * g + i]));
            top = kv_max_groups(top);
            const float to = kv_max_groups(most) > kMost ? fmaxf(m, top) : m, f = __builtin_amdgcn_exp2f(m - to);
            l *= f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) acc[i] *= f;
            m = to;
            weights();
        }
        l += add;
        if (__ballot(apart)) end = 0;
        // values: 16 dims a step, keys of half h in blocks 2 h and 2 h + 1
        wh_h8 rv[2];
#pragma unroll
        for (int f = 0; f < HD / 16; ++f) {
            if (f % 2 == 0) {
                const _Float16* const rp = rel + (f >> 1) * W::kRel + 16 * g;
                rv[0] = *(const wh_h8*)rp;
                rv[1] = *(const wh_h8*)(rp + 8);
            }
            const uint8_t* const src = mine + tkey * W::kRow + 16 * ((f >> 1) ^ swizzle(tkey)) + 8 * (f & 1);
            const wh_i2 codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) wh_i2*)src);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const wh_h8 x = kv_decode((uint32_t)codes[h], 1.0f) * rv[h];
                if constexpr (kF32) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl[h], acc[f], 0, 0, 0);
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph[h], acc[f], 0, 0, 0);
            }
        }
    }
    if (bad) atomicOr(a.status, WH_ST_NOT_RESIDENT);

    // join the four waves: 2 and 3 into 0 and 1, then 1 into 0
    l = kv_sum_groups(l);
    if (g == 0) {
        wave_m[wave][r16] = m;
        wave_l[wave][r16] = l;
    }
    const bool wave_is_apart = __ballot(apart) != 0;
    if (lane == 0) wave_apart[wave] = wave_is_apart;
    kv_lds_barrier();
    if (__builtin_expect(wave_apart[0] | wave_apart[1] | wave_apart[2] | wave_apart[3], 0)) {
        kv_plain_part<HD, kF32, kLatent, 16, 4>(a, place, wave);
        return;
    }
    float M = wave_m[0][r16], L = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, wave_m[w][r16]);
#pragma unroll
    for (int w = 0; w < 4; ++w) L += wave_l[w][r16] * __builtin_amdgcn_exp2f(wave_m[w][r16] - M);
    const float f0 = __builtin_amdgcn_exp2f(m - M);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) acc[i] *= f0;
    wh_f4* const o = (wh_f4*)smem;  // [wave of a pair][block of dims][lane]
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= (uint32_t)half && wave < 2 * (uint32_t)half) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) o[((wave - half) * (HD / 16) + i) * 64 + lane] = acc[i];
        }
        kv_lds_barrier();
        if (wave < (uint32_t)half) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) acc[i] += o[(wave * (HD / 16) + i) * 64 + lane];
        }
        kv_lds_barrier();
    }
    if (wave || !live) return;
    float denom = L;
    if (whole && a.sink) denom += __builtin_amdgcn_exp2f(a.sink[head] * 1.44269504088896340736f - M + kUp);
    const float inv = denom == 0.0f ? 0.0f : 1.0f / denom;
    float* const part = a.part + (((uint64_t)place.unit * a.s.kv_heads + kvh) * 16 + r16) * (HD + 2);
#pragma unroll
    for (int f = 0; f < HD / 16; ++f) {
        const uint32_t d = 16 * f + 4 * g;
        const wh_f4 x = acc[f] * inv;
        if (!whole) {
            *(wh_f2*)(part + d) = (wh_f2){x[0], x[1]};
            *(wh_f2*)(part + d + 2) = (wh_f2){x[2], x[3]};
        } else {
            kv_store<kF32>(a.out, (uint64_t)token * a.out_stride + (uint64_t)head * HD + d, x);
        }
    }
    if (!whole && g == 0) kv_put_sum(part + HD, M - kUp, L);
}

// A tile of 64 rows (32 in f32, whose queries and weights are two parts) for
// the calls that have them.  Eight waves bring a run of 64 keys' codes into LDS
// once, as they lie, and the powers of two beside them.  Wave (kq, rq) scores its
// keys against 16 rows, whose queries stay in its registers, and leaves their
// weights in LDS; for the run before it adds up its share of the dims for all
// rows: the codes are read transposed, sixteen keys of one dim a lane (the 4-bit
// transposing read), decoded to small f16 numbers and multiplied by their powers
// of two.  The two work on neighbouring runs at once, so one barrier a run is
// enough and the matrix work of one covers the loads and exponentials of the
// other.  Weights are taken against a row's reference as it is; only a run with a
// weight past f16 joins the waves' maxima and makes its weights again.
//
// Four waves up to 128 dims, three a SIMD (prompts of up to 2500 tokens, 4 heads
// on each of 8 key heads of 128, bf16: 247 us; with tiles in the order of their
// tokens 267 and, with two waves a SIMD, 305), eight above, where one workgroup takes
// a CU's registers.  In those prompts vector instructions take 67 % of the cycles,
// matrix ones 27 %, LDS 47 %, and waves wait for 27 % of theirs: instruction issue is
// what is fullest.  Not so at 512 dims: a chunk of 384 tokens, 64 heads on one key
// head, up to 2676 keys, bf16: 169 us, 0.73 PFLOP/s, vector instructions 38 % and
// matrix ones 28 %, waves waiting for a third of their cycles, and 384 workgroups
// are one and a half rounds; 12 tokens there, up to 40000 keys: 62 us and 11 for the
// join, the same shares; 3 requests of 5 tokens, f32: 34 us and 7 for the join.
template <int HD, bool kF32, bool kLatent>
struct wh_kv4_packed {
    static constexpr int kRows = kF32 ? 32 : 64, kBlocks = kRows / 16;
    static constexpr int kWaves = HD >= 256 ? 8 : 4, kThreads = 64 * kWaves, kPerSimd = HD >= 256 ? 2 : 3;
    static constexpr int kParts = kF32 ? 2 : 1;
    static constexpr int kRowGroups = kBlocks, kKeyGroups = kWaves / kRowGroups;
    static constexpr int kKeyBlocks = 4 / kKeyGroups;    // blocks of 16 keys a wave scores
    static constexpr int kPieces = HD >= 128 ? HD / 128 : 1;
    static constexpr int kGroups = HD / 32;
    static constexpr int kDims = HD / 16 / kWaves;       // blocks of 16 dims whose outputs a wave adds up
    static constexpr bool kBoth = HD >= 128 || kLatent;  // a lane brings chunks of keys and of values
    static constexpr int kMine = HD >= 256 ? HD / 256 : 1;  // 16-byte chunks, each a group of 32 dims, that a lane brings
    static constexpr int kLanes = kGroups / kMine;       // lanes of a row
    static constexpr int kBring = kLanes;                // waves that bring a plane's 64 rows
    static constexpr int kRow = HD / 2;                  // bytes of a row's codes
    static constexpr int kCodes = 64 * kRow;             // bytes of a run's codes
    static constexpr int kKeyBufs = kLatent ? 3 : 2;     // latent codes are values one run later
    static constexpr int kRel = 72;                      // f16 between groups of value scales
    static constexpr int kPl = 72;                       // f16 between rows of weights
    static constexpr int kAtValues = kKeyBufs * kCodes;                       // byte offsets in LDS
    static constexpr int kAtScales = kAtValues + (kLatent ? 0 : 3 * kCodes);  // [2][g][key] dwords
    static constexpr int kAtKeys = kAtScales + 2 * 4 * 64 * 4;                // f32: [2][key] power of two of keys
    static constexpr int kAtPow = kAtKeys + (kF32 ? 2 * 64 * 4 : 0);          // [2][key] power of two of value rows
    static constexpr int kAtRel = kAtPow + 2 * 64 * 4;                        // [3][group][key] f16
    static constexpr int kAtWeights = kAtRel + 3 * kGroups * kRel * 2;        // [2][part][row][key] f16
    static constexpr int kEnd = kAtWeights + 2 * kParts * kRows * kPl * 2;
    // f32: queries lie as parts in LDS before the first run.  At 512 dims registers do not hold all of them (what
    // the compiler moves to memory instead waits for the rows in flight): the last kFromLds steps' second parts
    // stay there, behind the rest, and are read again each run.
    using Query = wh_kv4_query<HD, kRows, kF32 ? kWaves : 4>;
    static constexpr int kFromLds = kF32 && HD == 512 ? kLatent ? 4 : 8 : 0;
    static constexpr int kAtQuery = kFromLds ? kEnd - Query::kBytes / 2 : 0;
    static constexpr size_t kLds = kFromLds ? kEnd + Query::kBytes / 2 : kEnd;
    static_assert(!kF32 || (size_t)(kAtQuery + Query::kBytes) <= kLds, "queries fit");
};

template <int HD, bool kF32, bool kLatent>
__global__ void __launch_bounds__((wh_kv4_packed<HD, kF32, kLatent>::kThreads), (wh_kv4_packed<HD, kF32, kLatent>::kPerSimd)) k_kv4_attn_packed(wh_kv4_attn_args a) {
    using W = wh_kv4_packed<HD, kF32, kLatent>;
    constexpr int kBlocks = W::kBlocks, kRows = W::kRows, kDims = W::kDims, kPieces = W::kPieces, kParts = W::kParts;
    constexpr int kKeyBlocks = W::kKeyBlocks, kWaves = W::kWaves;
    const wh_kv4_place place = kv_place<W::kRows>(a, false);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float wave_m[W::kKeyGroups][kRows], wave_l[W::kKeyGroups][kRows], row_m[kRows], row_c[kF32 ? kRows : 1];
    __shared__ int32_t row_pos[kRows];
    __shared__ uint32_t raise[2];
    __shared__ uint64_t nan_keys[3];
    const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, r16 = lane & 15, g = lane >> 4;
    const uint32_t kvh = place.head, kq = wave % W::kKeyGroups, rq = wave / W::kKeyGroups;
    const wh_kv4_tile tile = place.tile;
    if (!tile.ok) return;
    const uint32_t runs = tile.runs;
    const uint32_t run0 = place.split ? place.split * place.chunk : 0, run1 = min(runs, run0 + place.chunk);
    if (place.split && run0 >= runs) return;
    const bool whole = place.chunk >= runs;
    if (t < 2) raise[t] = 0;
    if (t < 3) nan_keys[t] = 0;
    if (t < kRows) row_m[t] = kMinusBig;

    // 16-byte chunk c of a row lies at chunk c ^ swizzle(row): 16 rows of one chunk are on all banks
    auto swizzle = [](uint32_t key) {
        return HD == 512 ? key & 15 : HD == 256 ? (key >> 1) & 7 : HD == 128 ? (key >> 2) & 3 : (key >> 3) & 1;
    };

    // this lane's key of a run, and its chunks: of the key and the value row, or
    // (short rows apart) of keys in the first waves, of values in the next
    const bool brings = wave < W::kBring * (W::kBoth ? 1u : 2u);
    const bool has_values = W::kBoth ? brings : brings && wave >= W::kBring, has_keys = W::kBoth ? brings : wave < W::kBring;
    const uint32_t* const table = a.tables + tile.request * a.table_stride;
    const uint32_t pmask = (1u << a.s.shift) - 1u;
    const uint32_t my_key = 64 / W::kLanes * (wave % W::kBring) + lane / W::kLanes, my_chunk = W::kMine * (lane % W::kLanes);
    bool bad = false;
    uint32_t page = 0;
    constexpr bool kTwo = W::kBoth && !kLatent;  // chunks of values are held beside those of keys
    wh_u4 kc[W::kMine], vc[kTwo ? W::kMine : 1];
    uint32_t kb = 0, vb = 0;  // their scale bytes
    auto run_at = [&](uint32_t run) { return wh_kv4_run(tile, min(run, run1 - 1)); };
    auto request_page = [&](uint32_t run) {
        if (W::kBring < kWaves && !brings) return;
        const uint32_t key0 = run_at(run);
        page = table[wh_kv4_seen(tile, key0, key0 + my_key) >> a.s.shift];
    };
    auto request_of = [&](const wh_kv4_plane& p, uint64_t line, wh_u4* c, uint32_t& b) {
        const uint8_t* const src = p.codes + line * (HD / 2) + 16 * my_chunk;
#pragma unroll
        for (int i = 0; i < W::kMine; ++i) c[i] = *(const wh_u4*)(src + 16 * i);
        const uint8_t* const sc = p.scales + line * (HD / 32) + my_chunk;
        b = W::kMine == 2 ? *(const uint16_t*)sc : *sc;
    };
    auto request = [&](uint32_t run) {
        if (W::kBring < kWaves && !brings) return;
        const bool out = page >= a.s.n_pages;
        bad |= out;
        const uint64_t line = wh_kv4_line(out ? 0 : page, kvh, (run_at(run) + my_key) & pmask, a.s.kv_heads, a.s.shift);
        request_of(W::kBoth || has_keys ? a.k : a.v, line, kc, kb);
        if constexpr (kTwo) request_of(a.v, line, vc, vb);
        request_page(run + 1);
    };
    auto value_bytes = [&] { return kTwo ? vb : kb; };
    // a row's largest byte, from its lanes
    auto row_top = [&](uint32_t b) { return kv_near_max<W::kLanes>(W::kMine == 2 ? max(b & 0xff, b >> 8) : b); };
    // rows of a run to LDS; now: the run that the workgroup is at
    auto stage = [&](uint32_t run, uint32_t now) {
        if (W::kBring < kWaves && !brings) return;
        uint32_t ktop = 0, vtop = 0;
        bool odd = false;
        if constexpr (kF32) ktop = row_top(kb);
        if (W::kBoth || has_keys) {
            if constexpr (!kF32)  // the instruction takes a byte of 0 as 2^-127
#pragma unroll
                for (int i = 0; i < W::kMine; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) kc[i][k] = (kb >> (8 * i)) & 0xff ? kc[i][k] : 0;
            uint8_t* const kd = smem + run % W::kKeyBufs * W::kCodes + my_key * W::kRow;
#pragma unroll
            for (int i = 0; i < W::kMine; ++i) *(wh_u4*)(kd + 16 * ((my_chunk + i) ^ swizzle(my_key))) = kc[i];
            uint8_t* const sc = smem + W::kAtScales + (run & 1) * 1024;
#pragma unroll
            for (int i = 0; i < W::kMine; ++i) {
                const uint32_t n = my_chunk + i, b = (kb >> (8 * i)) & 0xff;
                // f32: against the row's largest, so that decoded values are finite f16 whatever the bytes are
                sc[((n & 3) * 64 + my_key) * 4 + (n >> 2)] = (uint8_t)(kF32 ? (uint32_t)max((int)b - (int)ktop + 127, 0) : b);
            }
            if constexpr (kF32) {
                if (my_chunk == 0) ((float*)(smem + W::kAtKeys))[(run & 1) * 64 + my_key] = kv_key_scale(ktop, 0);
            }
            if constexpr (kF32 && !kLatent)  // a latent row's groups are values too, and kNear is less
#pragma unroll
                for (int i = 0; i < W::kMine; ++i) odd |= kv_key_odd((kb >> (8 * i)) & 0xff, ktop);
        }
        if (W::kBoth || has_values) {
            const uint32_t bytes = value_bytes();
            vtop = kTwo || !kF32 ? row_top(bytes) : ktop;
            const uint32_t vexp = kv_value_top(vtop);
            _Float16* const rel = (_Float16*)(smem + W::kAtRel) + run % 3 * (W::kGroups * W::kRel);
#pragma unroll
            for (int i = 0; i < W::kMine; ++i) {
                const uint32_t b = (bytes >> (8 * i)) & 0xff;
                rel[(my_chunk + i) * W::kRel + my_key] = kv_value_rel(b, vexp);
                odd |= kv_value_odd<kF32>(b, vtop, vexp);
            }
            ((float*)(smem + W::kAtPow))[(run & 1) * 64 + my_key] = kv_bits(vexp << 23);
            if constexpr (!kLatent) {
                uint8_t* const vd = smem + W::kAtValues + run % 3 * W::kCodes + my_key * W::kRow;
#pragma unroll
                for (int i = 0; i < W::kMine; ++i) *(wh_u4*)(vd + 16 * ((my_chunk + i) ^ swizzle(my_key))) = kTwo ? vc[kTwo ? i : 0] : kc[i];
            }
        }
        if (__builtin_expect(__ballot(odd) != 0, 0)) {
            asm volatile("");
            bool far = false;  // a group of a row without NaN, not zeros
#pragma unroll
            for (int i = 0; i < W::kMine; ++i) {
                const uint32_t k = (kb >> (8 * i)) & 0xff, v = (value_bytes() >> (8 * i)) & 0xff;
                if (W::kBoth || has_keys) {
                    if constexpr (kF32 && !kLatent) far |= k != 0 && ktop != 255 && kv_key_odd(k, ktop);
                }
                if (W::kBoth || has_values) far |= v != 0 && vtop != 255 && kv_value_odd<kF32>(v, vtop, kv_value_top(vtop));
            }
            const uint32_t key0 = run_at(run);  // the last run's once more: so too its keys
            if (wh_kv4_seen(tile, key0, key0 + my_key) == key0 + my_key) {  // some row may see this lane's key
                if (far) atomicMax(&raise[now & 1], kApart);
                if constexpr (!kLatent)
                    if (vtop == 255) atomicOr((unsigned long long*)&nan_keys[run % 3], 1ull << my_key);
            }
        }
    };

    if (run0 < run1) request_page(run0);
    // the query of row r16 of block rq
    wh_i8 qx[kF32 ? 1 : kPieces][2];
    wh_h8 qd[kF32 ? HD / 32 : 1][kParts];
    bool apart = false;  // f32: what f16 products do not hold
    uint32_t q_scale = 0;
    float c;  // scores are sums times this
    float l = 0.0f;
    const uint32_t row0 = 16 * rq + r16;
    {
        const uint32_t flat = tile.row0 + min(row0, tile.rows - 1), tok = flat / a.group;
        if constexpr (kF32) {
            typename W::Query query;
            query.load(wave, lane, [&](uint32_t r) {
                const uint32_t f = tile.row0 + min(r, tile.rows - 1), n = f / a.group;
                return (const float*)a.q + (uint64_t)(tile.token0 + n) * a.q_stride + (uint64_t)(kvh * a.group + f - n * a.group) * HD;
            });
            if (run0 < run1) request(run0);
            apart = query.put(wave, lane, (_Float16*)(smem + W::kAtQuery), row_c, a.scale_log2);
            kv_lds_barrier();
            W::Query::get(qd, (const _Float16*)(smem + W::kAtQuery), row0, g);
            c = row_c[row0];
            kv_lds_barrier();
        } else {
            const uint64_t at = (uint64_t)(tile.token0 + tok) * a.q_stride + (uint64_t)(kvh * a.group + flat - tok * a.group) * HD;
            const uint16_t* const p = (const uint16_t*)a.q + at + 16 * g;
            wh_u4 raw[kPieces][2][2];
#pragma unroll
            for (int j = 0; j < kPieces; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    raw[j][i >> 1][i & 1] = HD == 64 && i >= 2 ? (wh_u4){0, 0, 0, 0} : *(const wh_u4*)(p + 128 * j + 64 * (i >> 1) + 8 * (i & 1));
            if (run0 < run1) request(run0);
#pragma unroll
            for (int j = 0; j < kPieces; ++j)
                q_scale |= kv_query_e4m3(raw[j], a.scale_log2 < 0.0f ? 0x80008000u : 0u, qx[j][0], qx[j][1]) << (8 * j);
            c = fmaxf(fabsf(a.scale_log2), 1.0e-37f);  // above 0, which would hide what is masked; the sign is the query's
        }
        row_pos[row0] = row0 < tile.rows ? tile.len - (int32_t)tile.n_q + (int32_t)tok : -1;
    }
    const int32_t pos_lo = tile.len - (int32_t)tile.n_q + (int32_t)(tile.row0 / a.group);
    const int32_t pos_hi = tile.len - (int32_t)tile.n_q + (int32_t)((tile.row0 + tile.rows - 1) / a.group);

    const uint32_t dim0 = kDims * wave;
    wh_f4 acc[kDims][kBlocks];  // [dim 16 (dim0 + f) + 4g + i][row 16 b + r16]
#pragma unroll
    for (int f = 0; f < kDims; ++f)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[f][b] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};

    // what the first run finds in place of an earlier one's: no weights, and finite value scales
    for (uint32_t i = 16 * t; i < W::kEnd - W::kAtRel; i += 16 * W::kThreads) *(wh_u4*)(smem + W::kAtRel + i) = (wh_u4){0, 0, 0, 0};
    kv_lds_barrier();
    if (run0 < run1) {
        stage(run0, run0);
        if (kF32 && apart) atomicMax(&raise[run0 & 1], kApart);
    }
    kv_lds_barrier();

    // outputs of the run whose weights lie at `run` modulo 2, its values and their scales modulo 3: 16 dims a step
    wh_h8 w[2][kBlocks][kParts];
    auto read_weights = [&](uint32_t run) {
        const _Float16* const pb =
            (const _Float16*)(smem + W::kAtWeights) + (run & 1) * (kParts * kRows * W::kPl) + r16 * W::kPl + 16 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int p = 0; p < kParts; ++p) w[h][b][p] = *(const wh_h8*)(pb + p * (kRows * W::kPl) + 16 * b * W::kPl + 8 * h);
    };
    wh_h8 rel[2];
    auto values_step = [&](uint32_t run, int f) {
        const uint32_t block = dim0 + f, key = 16 * g + r16;  // of the transposed read
        if (f % 2 == 0) {
            const _Float16* const rp =
                (const _Float16*)(smem + W::kAtRel) + run % 3 * (W::kGroups * W::kRel) + (block >> 1) * W::kRel + 16 * g;
            rel[0] = *(const wh_h8*)rp;
            rel[1] = *(const wh_h8*)(rp + 8);
        }
        const uint8_t* const src = smem + (kLatent ? 0 : W::kAtValues) + run % 3 * W::kCodes + key * W::kRow +
                                   16 * ((block >> 1) ^ swizzle(key)) + 8 * (block & 1);
        const wh_i2 codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) wh_i2*)src);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const wh_h8 x = kv_decode((uint32_t)codes[h], 1.0f) * rel[h];
#pragma unroll
            for (int p = kParts - 1; p >= 0; --p)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) acc[f][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w[h][b][p], acc[f][b], 0, 0, 0);
        }
    };

    uint32_t end = run1;  // 0 once the values are apart: not a second way out, which costs registers
    for (uint32_t run = run0; run < end; ++run) {
        const uint32_t at = run & 1;
        request(run + 1);
        if constexpr (!kLatent)
            if (t == 0) nan_keys[(run + 2) % 3] = 0;
        // scores
        wh_f4 s[kKeyBlocks];
        uint32_t scale[kKeyBlocks];
        const uint8_t* const krow = smem + run % W::kKeyBufs * W::kCodes + (16 * kKeyBlocks * kq + r16) * W::kRow;
        const uint8_t* const krow_s =
            smem + W::kAtScales + at * 1024 + ((HD == 64 ? g & 1 : g) * 64 + 16 * kKeyBlocks * kq + r16) * 4;
        const uint32_t flip = swizzle(r16);  // of all this lane's keys
#pragma unroll
        for (int i = 0; i < kKeyBlocks; ++i) {
            scale[i] = *(const uint32_t*)(krow_s + 64 * i);
            s[i] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};
        }
        if constexpr (kF32) {
            wh_f4 s_low[kKeyBlocks];  // of the second parts: a chain of products of its own
#pragma unroll
            for (int i = 0; i < kKeyBlocks; ++i) s_low[i] = s[i];
            // keys decoded against their row's power of two
            const _Float16* const low = (const _Float16*)(smem + W::kEnd) + row0 * W::Query::kLd;
#pragma unroll
            for (int j = 0; j < kPieces; ++j)
#pragma unroll
                for (int i = 0; i < kKeyBlocks; ++i) {
                    const float against = kv_bits((scale[i] >> (8 * j) & 0xff) << 23);
                    uint32_t v[4];
                    if constexpr (HD == 64) {
                        const wh_u2 u = *(const wh_u2*)(krow + 16 * ((g & 1) ^ flip) + 8 * (g >> 1) + i * 16 * W::kRow);
                        v[0] = u[0], v[1] = u[1];
                    } else {
                        const wh_u4 u = *(const wh_u4*)(krow + 16 * ((4 * j + g) ^ flip) + i * 16 * W::kRow);
                        v[0] = u[0], v[1] = u[1], v[2] = u[2], v[3] = u[3];
                    }
#pragma unroll
                    for (int k = 0; k < (HD == 64 ? 2 : 4); ++k) {
                        const wh_h8 x = kv_decode(v[k], against);
#pragma unroll
                        for (int p = kParts - 1; p >= 0; --p) {
                            constexpr int kSteps = HD / 32;
                            const int step = 4 * j + k;
                            const wh_h8 y = p == 1 && step >= kSteps - W::kFromLds
                                                ? *(const wh_h8*)(low + kv_dim<HD>(step, g))
                                                : qd[step][p];
                            wh_f4& to = p ? s_low[i] : s[i];
                            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, to, 0, 0, 0);
                        }
                    }
                }
#pragma unroll
            for (int i = 0; i < kKeyBlocks; ++i)
            {
                const wh_f4 k_scale = *(const wh_f4*)(smem + W::kAtKeys + (at * 64 + 16 * (kKeyBlocks * kq + i) + 4 * g) * 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) s[i][k] = fmaf(s_low[i][k], 1.0f / kLowPart, s[i][k]) * c * k_scale[k];
            }
        } else {
            // codes as they lie, which takes scales by 32 dims
            wh_static_for<kPieces>([&](auto jc) {
                constexpr int j = decltype(jc)::value;
                wh_i8 x[kKeyBlocks];
#pragma unroll
                for (int i = 0; i < kKeyBlocks; ++i) {
                    const wh_u4 v = *(const wh_u4*)(krow + 16 * ((HD == 64 ? g & 1 : 4 * j + g) ^ flip) + i * 16 * W::kRow);
                    // 64 dims: the other 64 of the product are zeros of the query
                    x[i][0] = v[0], x[i][1] = v[1], x[i][2] = v[2], x[i][3] = v[3];
                    x[i][4] = x[i][5] = x[i][6] = x[i][7] = 0;
                }
#pragma unroll
                for (int p = 1; p >= 0; --p)
#pragma unroll
                    for (int i = 0; i < kKeyBlocks; ++i)
                        s[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[i], qx[j][p], s[i], 4, 0, j, scale[i], j,
                                                                                q_scale - (p ? 0x04040404u : 0u));
            });
        }
        read_weights(run + 1);
        // -inf where a row does not see this lane's keys
        const uint32_t key0 = wh_kv4_run(tile, run);
        const bool all = (int32_t)key0 + 63 <= pos_lo && tile.rows == kRows && (!a.window || (int64_t)key0 + a.window > pos_hi);
        if (!all) kv_mask(s, row_pos[row0], key0 + 16 * kKeyBlocks * kq + 4 * g, a.window, a.first);
        if constexpr (!kLatent) {
            const uint64_t nan = nan_keys[run % 3];
            if (__builtin_expect(nan != 0, 0)) {
                const uint64_t mine = nan >> (16 * kKeyBlocks * kq + 4 * g);
#pragma unroll
                for (int i = 0; i < 4 * kKeyBlocks; ++i)
                    if ((mine >> (16 * (i >> 2) + (i & 3)) & 1) && s[i >> 2][i & 3] != kMinusInf)
                        s[i >> 2][i & 3] = kv_bits(0x7fc00000u);
            }
        }
        const float* const power_of = (const float*)(smem + W::kAtPow) + at * 64 + 16 * kKeyBlocks * kq + 4 * g;
        wh_f4 power[kKeyBlocks];
#pragma unroll
        for (int i = 0; i < kKeyBlocks; ++i) power[i] = *(const wh_f4*)(power_of + 16 * i);
#pragma unroll
        for (int f = 0; f < kDims; ++f) values_step(run + 2, f);
        const float m0 = row_m[row0];
        float add, most;
        auto weights = [&](float m) {
            const float up = kUp - m;
            add = most = 0.0f;
            _Float16* const pw =
                (_Float16*)(smem + W::kAtWeights) + at * (kParts * kRows * W::kPl) + row0 * W::kPl + 16 * kKeyBlocks * kq + 4 * g;
#pragma unroll
            for (int i = 0; i < kKeyBlocks; ++i) {
                float e[4];
                union {
                    _Float16 h[4];
                    wh_u2 u;
                } hi, lo;
#pragma unroll
                for (int k = 0; k < 4; ++k) e[k] = __builtin_amdgcn_exp2f(kF32 ? s[i][k] + up : fmaf(s[i][k], c, up));
                add += (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    e[k] *= power[i][k];
                    most = fmaxf(most, e[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    hi.h[k] = (_Float16)e[k];
                    if constexpr (kF32) lo.h[k] = (_Float16)(e[k] - (float)hi.h[k]);
                }
                *(wh_u2*)(pw + 16 * i) = hi.u;
                if constexpr (kF32) *(wh_u2*)(pw + kRows * W::kPl + 16 * i) = lo.u;
            }
        };
        stage(run + 1, run);
        weights(m0);
        if (__ballot(most > kMost) && lane == 0) atomicMax(&raise[at], run + 1);
        kv_lds_barrier();
        const uint32_t raises = __builtin_amdgcn_readfirstlane(raise[at]);
        if (__builtin_expect(raises > run, 0)) {  // the whole workgroup
            if (raises == kApart) end = 0;
            // rows with such a weight take their largest score plus exponent as the reference
            float top = kMinusInf;
#pragma unroll
            for (int i = 0; i < kKeyBlocks; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    top = fmaxf(top, s[i][k] * (kF32 ? 1.0f : c) + (float)kv_exponent(power[i][k]));
            top = kv_max_groups(top);
            if (!(kv_max_groups(most) > kMost)) top = kMinusBig;
            if (g == 0) wave_m[kq][row0] = top;
            kv_lds_barrier();
            auto raised = [&](uint32_t row) {
                float m = row_m[row];
#pragma unroll
                for (int i = 0; i < W::kKeyGroups; ++i) m = fmaxf(m, wave_m[i][row]);
                return m;
            };
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const uint32_t row = 16 * b + r16;
                const float f = __builtin_amdgcn_exp2f(row_m[row] - raised(row));
#pragma unroll
                for (int k = 0; k < kDims; ++k) acc[k][b] *= f;
            }
            const float m = raised(row0);
            l *= __builtin_amdgcn_exp2f(row_m[row0] - m);
            weights(m);
            kv_lds_barrier();
            if (kq == 0 && g == 0) row_m[row0] = m;
            kv_lds_barrier();
        }
        l += add;
    }
    if (bad) atomicOr(a.status, WH_ST_NOT_RESIDENT);
    if (__builtin_expect(end < run1, 0)) {
        kv_plain_part<HD, kF32, kLatent, kRows, kWaves>(a, place, wave);
        return;
    }
    if (run0 < run1) {
        read_weights(run1 + 1);
#pragma unroll
        for (int f = 0; f < kDims; ++f) values_step(run1 + 2, f);
    }

    l = kv_sum_groups(l);
    if (g == 0) wave_l[kq][row0] = l;
    kv_lds_barrier();
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const uint32_t r = 16 * b + r16;
        if (r >= tile.rows) continue;
        const uint32_t flat = tile.row0 + r, tok = flat / a.group, head = kvh * a.group + (flat - tok * a.group);
        const float M = row_m[r];
        float L = 0.0f;
#pragma unroll
        for (int i = 0; i < W::kKeyGroups; ++i) L += wave_l[i][r];
        float denom = L;
        if (whole && a.sink) denom += __builtin_amdgcn_exp2f(a.sink[head] * 1.44269504088896340736f - M + kUp);
        const float inv = denom == 0.0f ? 0.0f : 1.0f / denom;
        float* const part = a.part + (((uint64_t)place.unit * a.s.kv_heads + kvh) * kRows + r) * (HD + 2);
        const uint64_t at = (uint64_t)(tile.token0 + tok) * a.out_stride + (uint64_t)head * HD;
#pragma unroll
        for (int f = 0; f < kDims; ++f) {
            const uint32_t d = 16 * (dim0 + f) + 4 * g;
            const wh_f4 y = acc[f][b] * inv;
            if (!whole) {
                *(wh_f2*)(part + d) = (wh_f2){y[0], y[1]};
                *(wh_f2*)(part + d + 2) = (wh_f2){y[2], y[3]};
            } else {
                kv_store<kF32>(a.out, at + d, y);
            }
        }
        if (!whole && dim0 == 0 && g == 0) kv_put_sum(part + HD, M - kUp, L);
    }
}

// Joins the workgroups of a tile: outputs weighted by their sums of weights, and
// the sink.  A wave a row, four rows a workgroup.  Bound by latency (lengths, the
// parts' maxima, the parts): 6 us for 4 parts of 256 tiles of 16 rows of 128, 11 us
// for 33 MB of 22 parts of 12 tiles of 64 rows of 512.
template <int HD, bool kF32, int kRows>
__global__ void __launch_bounds__(256) k_kv4_join(wh_kv4_attn_args a) {
    constexpr int kPer = HD >= 256 ? 4 : HD / 64;  // values of a lane next to each other
    const uint32_t lane = threadIdx.x & 63, row = 4 * blockIdx.y + (threadIdx.x >> 6);
    const wh_kv4_place place = kv_place<kRows>(a, true);
    const wh_kv4_tile& tile = place.tile;
    const uint32_t blocks = tile.runs, kvh = place.head;
    if (!tile.ok || row >= tile.rows || blocks <= place.chunk) return;
    const uint32_t n = (blocks + place.chunk - 1) / place.chunk;
    const uint32_t flat = tile.row0 + row, tok = flat / a.group, head = kvh * a.group + (flat - tok * a.group);
    const uint64_t next = (uint64_t)a.s.kv_heads * kRows * (HD + 2);
    const float* const part = a.part + (((uint64_t)place.unit * a.s.kv_heads + kvh) * kRows + row) * (HD + 2);
    float M = kMinusBig, L = 0.0f;
    for (uint32_t k = lane; k < n; k += 64) M = fmaxf(M, part[k * next + HD]);
    M = wh_wave_max(M);
    for (uint32_t k = lane; k < n; k += 64) L += part[k * next + HD + 1] * __builtin_amdgcn_exp2f(part[k * next + HD] - M);
    L = kv_wave_sum(L);
    if (a.sink) L += __builtin_amdgcn_exp2f(a.sink[head] * 1.44269504088896340736f - M);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // before the sum, which then stays within the parts' size
    float x[HD / 64];
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) x[i] = 0.0f;
#pragma unroll 4
    for (uint32_t k = 0; k < n; ++k) {
        const float* const p = part + k * next;
        const float w = p[HD + 1] * __builtin_amdgcn_exp2f(p[HD] - M) * inv;
#pragma unroll
        for (int i = 0; i < HD / 64; i += 2)
            if constexpr (kPer >= 2) {
                const wh_f2 u = *(const wh_f2*)(p + 64 * kPer * (i / kPer) + kPer * lane + i % kPer);
                x[i] += u[0] * w;
                x[i + 1] += u[1] * w;
            } else {
                x[i] += p[lane] * w;
            }
    }
    const uint64_t at = (uint64_t)(tile.token0 + tok) * a.out_stride + (uint64_t)head * HD;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        const uint64_t d = at + 64 * kPer * (i / kPer) + kPer * lane + i % kPer;
        if constexpr (kF32) ((float*)a.out)[d] = x[i];
        else ((__bf16*)a.out)[d] = (__bf16)x[i];
    }
}

template <int HD, bool kF32, bool kLatent>
hipError_t attn_launch_of(const wh_kv4_attn_args& a, hipStream_t stream) {
    const bool split = a.units > a.n_tiles;
    const dim3 grid((split ? a.units : a.n_tiles) * a.s.kv_heads);
    constexpr bool kAlways = kF32 && HD == 512;  // wide, as wh_kv4_attn_plan_of has it
    if (kAlways || a.wide) {
        using W = wh_kv4_packed<HD, kF32, kLatent>;
        k_kv4_attn_packed<HD, kF32, kLatent><<<grid, W::kThreads, W::kLds, stream>>>(a);
        if (split)
            k_kv4_join<HD, kF32, W::kRows><<<dim3(a.n_tiles * a.s.kv_heads, W::kRows / 4), 256, 0, stream>>>(a);
        return hipGetLastError();
    }
    if constexpr (!kAlways) {
        k_kv4_attn<HD, kF32, kLatent><<<grid, 256, wh_kv4_narrow<HD, kF32>::kLds, stream>>>(a);
        if (split) k_kv4_join<HD, kF32, 16><<<dim3(a.n_tiles * a.s.kv_heads, 4), 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

// Dynamic LDS above the default.
template <int HD, bool kF32, bool kLatent>
hipError_t attn_setup_of() {
    const hipError_t e = hipFuncSetAttribute((const void*)k_kv4_attn_packed<HD, kF32, kLatent>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)wh_kv4_packed<HD, kF32, kLatent>::kLds);
    if constexpr (!(kF32 && HD == 512))
        if (e == hipSuccess)
            return hipFuncSetAttribute((const void*)k_kv4_attn<HD, kF32, kLatent>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)wh_kv4_narrow<HD, kF32>::kLds);
    return e;
}
template <int HD>
hipError_t attn_setup_hd() {
    for (const hipError_t e : {attn_setup_of<HD, false, false>(), attn_setup_of<HD, false, true>(), attn_setup_of<HD, true, false>(),
                               attn_setup_of<HD, true, true>()})
        if (e != hipSuccess) return e;
    return hipSuccess;
}

template <int HD>
hipError_t attn_launch_hd(const wh_kv4_attn_args& a, bool bf16, bool latent, hipStream_t stream) {
    if (bf16) return latent ? attn_launch_of<HD, false, true>(a, stream) : attn_launch_of<HD, false, false>(a, stream);
    return latent ? attn_launch_of<HD, true, true>(a, stream) : attn_launch_of<HD, true, false>(a, stream);
}

}  // namespace

hipError_t wh_kv4_setup() {
    if (const hipError_t e = hipFuncSetAttribute((const void*)k_kv_plan, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)plan_lds(WH_KV_MAX_REQUESTS));
        e != hipSuccess)
        return e;
    for (const hipError_t e : {attn_setup_hd<64>(), attn_setup_hd<128>(), attn_setup_hd<256>(), attn_setup_hd<512>()})
        if (e != hipSuccess) return e;
    return hipSuccess;
}

hipError_t wh_kv_plan_launch(const wh_kv_plan_args& a, hipStream_t stream) {
    const uint64_t copy = a.free_out != a.free_in ? a.n_pages : 0;
    const uint64_t items = std::max<uint64_t>(std::max<uint64_t>(a.max_tokens, copy), 1);
    const uint32_t grid = (uint32_t)std::min<uint64_t>((items + 4 * kPlanThreads - 1) / (4 * kPlanThreads), 256);
    k_kv_plan<<<grid, kPlanThreads, plan_lds(a.n), stream>>>(a);
    return hipGetLastError();
}

namespace {
// Launches for all rows of a call; launch(grid, a) takes some.
template <class F>
hipError_t kv_rows_launch(wh_kv4_rows_args a, bool bf16, F launch) {
    const uint64_t pieces = (uint64_t)a.s.kv_heads * (a.s.head_dim / 8);
    for (uint64_t left = a.n; left;) {
        a.n = (uint32_t)wh_kv4_rows_of_launch(left, pieces);
        launch(dim3((uint32_t)((a.n * pieces + 255) / 256), a.planes), a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        left -= a.n;
        a.slots += a.n;
        for (uint32_t p = 0; p < a.planes; ++p) a.rows[p] = (uint8_t*)a.rows[p] + a.n * a.stride[p] * (bf16 ? 2 : 4);
    }
    return hipSuccess;
}
}  // namespace

hipError_t wh_kv4_write_launch(const wh_kv4_rows_args& a, bool bf16, hipStream_t stream) {
    return kv_rows_launch(a, bf16, [&](dim3 grid, const wh_kv4_rows_args& b) {
        if (bf16) k_kv4_write<true><<<grid, 256, 0, stream>>>(b);
        else k_kv4_write<false><<<grid, 256, 0, stream>>>(b);
    });
}

hipError_t wh_kv4_read_launch(const wh_kv4_rows_args& a, bool bf16, hipStream_t stream) {
    return kv_rows_launch(a, bf16, [&](dim3 grid, const wh_kv4_rows_args& b) {
        if (bf16) k_kv4_read<true><<<grid, 256, 0, stream>>>(b);
        else k_kv4_read<false><<<grid, 256, 0, stream>>>(b);
    });
}

// Wide tiles, of 64 rows (f32: 32), against narrow ones of 16, whose product wastes
// less where a request has few rows and whose waves wait for nobody; by the rows
// (tokens x heads of a key head) that requests have on average.  us, 16 requests of
// one token and up to 6000 keys, narrow against wide:
//  - f32, 512 dims: always wide (the narrow kernel, which is not kept, took 40 to 73
//    for 8 to 64 rows, this one 30 to 45);
//  - from 256 dims on: over 16 rows.  bf16, 4 key heads of 256: 16 rows 33 and 53, 24
//    rows 59 and 53, 64 rows 74 and 54; f32: 39 and 55, 70 and 55, 97 and 95; bf16,
//    one of 512: 35 and 33, 36 and 35, 50 and 40;
//  - up to 128 dims: bf16 over 48 rows, f32 over 64.  bf16, 8 key heads of 128: 16
//    rows 29 and 51, 32 rows 45 and 54, 48 rows 54 and 56, 64 rows 60 and 54; f32: 16
//    rows 35 and 53, 24 rows 56 and 54, 32 rows 55 and 54, 48 rows 77 and 98, 64 rows
//    79 and 88.  4 prompts of 2000 tokens, 4 rows a token: bf16 297 and 143, f32 363
//    and 275.
// Rows alone do not tell short prompts, where there are few tiles and few keys to
// cut up.  16 of 20 to 40 tokens, 8 rows each, up to 1000 rows before them, narrow
// against the wide tiles that they get: bf16, 8 key heads of 128: 60 and 74, 4 of 64:
// 30 and 48; f32, 4 of 64: 36 and 51; but 8 of 128 in f32: 73 and 65, 4 of 256: 88
// and 57 in bf16, 101 and 73 in f32.  Nor does an average tell one prompt among
// single tokens, all of which get its tiles.
//
// With few tiles their keys are cut up.  Workgroups aimed at: those that the chip
// holds at once; twice as many where that is less than four a tile, since whole
// parts of requests of different lengths do not come out even (32 requests of up to
// 8192 keys, 8 key heads of 128: 73, 61, 59 and 67 us for one, one and a half, two
// and four rounds; 16 of up to 6000 with two wide tiles each, f32: 103, 98, 94 and
// 107); none where two rounds are less than three a tile (96 windows of 1024 keys, 8
// key heads: 40 us a workgroup a tile, 55 cut up in two rounds, 67 in four).
wh_kv4_attn_plan wh_kv4_attn_plan_of(const wh_kv4_attn_args& a, bool bf16, size_t max_len) {
    wh_kv4_attn_plan p{};
    const uint64_t rows = (uint64_t)a.n_tokens * a.group;
    const uint32_t wide_rows = bf16 ? 64 : 32;
    const uint32_t narrow_rows = a.s.head_dim >= 512 && !bf16 ? 0 : a.s.head_dim >= 256 ? 16 : bf16 ? 48 : 64;
    p.wide = rows > (uint64_t)a.n_requests * narrow_rows;
    const uint32_t tile_rows = p.wide ? wide_rows : 16;
    p.n_tiles = (uint32_t)wh_kv4_tile_slots(a.n_tokens, a.n_requests, a.group, tile_rows);
    uint64_t keys = max_len;
    if (a.window) keys = std::min<uint64_t>(keys, (uint64_t)a.window + a.first + a.n_tokens);
    const uint32_t resident = (p.wide ? a.s.head_dim >= 256 ? 256 : 768 : a.s.head_dim >= 256 ? 256 : 512) / a.s.kv_heads;
    p.min_runs = 2;  // a workgroup's start and end cost as much
    const uint64_t busy = std::max<uint64_t>(rows / tile_rows, a.n_requests);  // tiles, where every request has rows
    p.units = resident < 4 * busy ? 2 * resident : resident;
    if (p.units < 3 * busy || a.n_requests > WH_KV_SPLIT_REQUESTS || keys <= 64 * (2 * p.min_runs - 1)) p.units = 0;
    p.units = std::max(p.units, p.n_tiles);
    if (p.units > p.n_tiles) p.part_bytes = (size_t)p.units * a.s.kv_heads * tile_rows * (a.s.head_dim + 2) * sizeof(float);
    return p;
}

hipError_t wh_kv4_attn_launch(const wh_kv4_attn_args& a, bool bf16, bool latent, hipStream_t stream) {
    switch (a.s.head_dim) {
        case 64: return attn_launch_hd<64>(a, bf16, latent, stream);
        case 128: return attn_launch_hd<128>(a, bf16, latent, stream);
        case 256: return attn_launch_hd<256>(a, bf16, latent, stream);
        default: return attn_launch_hd<512>(a, bf16, latent, stream);
    }
}
