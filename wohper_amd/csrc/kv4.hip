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

#include "wh_device.h"

namespace {

typedef _Float16 wh_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 wh_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 wh_h8 __attribute__((ext_vector_type(8)));
typedef short wh_s4 __attribute__((ext_vector_type(4)));
typedef __fp16 wh_hh4 __attribute__((ext_vector_type(4)));
typedef uint32_t wh_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t wh_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float kv_bits(uint32_t u) { return __uint_as_float(u); }

// ------------------------------------------------------------------- plan

__device__ __forceinline__ uint64_t kv_shfl_up64(uint64_t v, uint32_t d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d, 64), hi = __shfl_up((uint32_t)(v >> 32), d, 64);
    return ((uint64_t)hi << 32) | lo;
}

// Last index i with prefix[i] <= x (prefix ascending, prefix[0] = 0 <= x).
__device__ __forceinline__ uint32_t kv_find(const uint32_t* prefix, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;  // prefix[lo] <= x, answer in [lo, hi)
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (prefix[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

constexpr uint32_t kPlanThreads = 1024;

// Every workgroup adds up all requests (three prefix sums of n <= 4096 numbers
// in LDS: new tokens, pages taken, pages given back) and then fills its share
// of the outputs, so a plan is one launch whose workgroups wait for nobody.  A
// page that a request takes is worked out where it is needed (its table entry,
// each slot on it) instead of being read back from another workgroup's store.
// Bound by latency: the prefix sums and one chain of dependent loads.
__global__ void __launch_bounds__(kPlanThreads) k_kv_plan(wh_kv_plan_args a) {
    extern __shared__ __align__(16) uint32_t lds[];
    uint32_t* const tok = lds;                  // [n + 1]
    uint32_t* const take = tok + a.n + 1;       // [n + 1]
    uint32_t* const give = take + a.n + 1;      // [n + 1]
    __shared__ uint64_t wave_sum[3][kPlanThreads / 64];
    __shared__ uint32_t bad;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const uint32_t count_in = *a.free_count, mask = (1u << a.shift) - 1u;
    if (t == 0) bad = 0;
    __syncthreads();
    constexpr uint32_t kPer = WH_KV_MAX_REQUESTS / kPlanThreads;
    const uint32_t per = (a.n + kPlanThreads - 1) / kPlanThreads, b0 = t * per;
    uint64_t mine[kPer][3], run[3] = {0, 0, 0};
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
        const uint32_t b = b0 + k;
#pragma unroll
        for (int s = 0; s < 3; ++s) mine[k][s] = run[s];
        if (k < per && b < a.n) {
            const uint64_t o = a.old_lens[b], w = a.new_lens[b];
            const uint64_t po = (o + mask) >> a.shift, pw = (w + mask) >> a.shift;
            if (po > a.table_stride || pw > a.table_stride) bad = 1;
            run[0] += w > o ? w - o : 0;
            run[1] += pw > po ? pw - po : 0;
            run[2] += po > pw ? po - pw : 0;
        }
    }
    uint64_t incl[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        uint64_t v = run[s];
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint64_t u = kv_shfl_up64(v, d);
            if (lane >= d) v += u;
        }
        incl[s] = v;
        if (lane == 63) wave_sum[s][wave] = v;
    }
    __syncthreads();
    uint64_t total[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        uint64_t before = 0, all = 0;
        for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) before += wave_sum[s][w];
            all += wave_sum[s][w];
        }
        total[s] = all;
        uint32_t* const dst = s == 0 ? tok : s == 1 ? take : give;
        const uint64_t base = before + incl[s] - run[s];
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
            if (k < per && b0 + k < a.n) dst[b0 + k] = (uint32_t)(base + mine[k][s]);
        if (t == 0) dst[a.n] = (uint32_t)all;
    }
    __syncthreads();
    // a plan that does not fit is none: nothing is taken, given or numbered
    const bool narrow = bad || total[0] > a.max_tokens;
    const bool empty = count_in > a.n_pages || count_in + total[2] > a.n_pages || total[1] > count_in + total[2];
    const bool ok = !narrow && !empty;
    const uint32_t n_tok = ok ? (uint32_t)total[0] : 0, n_take = ok ? (uint32_t)total[1] : 0,
                   n_give = ok ? (uint32_t)total[2] : 0;
    const uint32_t top = count_in + n_give;
    const uint32_t first = blockIdx.x * kPlanThreads + t, step = gridDim.x * kPlanThreads;
    auto given = [&](uint32_t j) {  // the j-th page given back
        const uint32_t b = kv_find(give, a.n, j);
        const uint32_t at = (uint32_t)(((uint64_t)a.new_lens[b] + mask) >> a.shift) + (j - give[b]);
        return a.tables[b * a.table_stride + at];
    };
    auto taken = [&](uint32_t k) {  // the k-th page off the stack
        const uint32_t at = top - 1 - k;
        return at < count_in ? a.free_in[at] : given(at - count_in);
    };
    for (uint32_t i = first; i < a.max_tokens; i += step) {
        uint32_t slot = WH_KV_NONE, pos = 0;
        if (i < n_tok) {
            const uint32_t b = kv_find(tok, a.n, i);
            const uint32_t old = a.old_lens[b];
            pos = old + (i - tok[b]);
            const uint32_t po = (uint32_t)(((uint64_t)old + mask) >> a.shift), pi = pos >> a.shift;
            const uint32_t page = pi < po ? a.tables[b * a.table_stride + pi] : taken(take[b] + (pi - po));
            if (page < a.n_pages) slot = (page << a.shift) + (pos & mask);
            else atomicOr(a.status, WH_ST_NOT_RESIDENT);
        }
        a.slots[i] = slot;
        a.positions[i] = pos;
    }
    for (uint32_t k = first; k < n_take; k += step) {
        const uint32_t b = kv_find(take, a.n, k);
        const uint32_t po = (uint32_t)(((uint64_t)a.old_lens[b] + mask) >> a.shift);
        a.tables[b * a.table_stride + po + (k - take[b])] = taken(k);
    }
    for (uint32_t j = first; j < n_give; j += step) a.free_out[count_in + j] = given(j);
    if (a.free_out != a.free_in)
        for (uint32_t k = first; k < min(count_in, a.n_pages); k += step) a.free_out[k] = a.free_in[k];
    for (uint32_t b = first; b <= a.n; b += step) a.starts[b] = ok ? tok[b] : 0;
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

__device__ __forceinline__ uint32_t kv_quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, false));
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
// or NaN has codes 0 and byte 255.  Bound by memory: 4.27 bytes in and out for
// an f32 value's 4.
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
    top = kv_quad_max(top);
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
// code has two significant bits.
template <bool kBf16>
__global__ void __launch_bounds__(256) k_kv4_read(wh_kv4_rows_args a) {
    const uint32_t pl = blockIdx.y, per = a.s.kv_heads * (a.s.head_dim / 8);
    const uint64_t unit = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (unit >= (uint64_t)a.n * per) return;
    const uint32_t i = (uint32_t)(unit / per), piece = (uint32_t)(unit - (uint64_t)i * per);
    const wh_kv4_at at = kv_at(a, a.slots[i], piece);
    if (!at.ok) return;
    const uint32_t c = ((const uint32_t*)a.plane[pl].codes)[at.code];
    const uint32_t byte = a.plane[pl].scales[at.scale];
    const float scale = kv_bits(byte << 23);  // 0 -> 0.0; 255 -> the conversion gives NaN
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
// flattened; a workgroup takes a tile of 16 of them and a run of the keys that
// any of them sees, and adds weights and values in one pass with the running
// maximum.  Softmax in powers of two: w = 2^(s * scale * log2(e) - m).
//
// Numbers: both factors of every product go to f16 matrix instructions, whose
// products are exact in their f32 sums.  A cached row is taken relative to its
// largest scale byte (code * 2^(byte - largest): exact in f16 down to 2^-23 of
// that, below which f32 would lose it too), the power of two returns to the
// score in f32.  A query row is scaled by a power of two so that its largest
// value is 2^13..2^14: a bf16 query is exact in one f16 unless 2^-28 of that,
// an f32 query takes two (22 bits, and 2^-38 of the largest).  A weight times
// its value row's power of two is rounded to one f16 (11 bits, one more than
// a bf16 output keeps beside its sign) or, for f32, split into two.  Maxima,
// sums of weights and outputs are f32.

constexpr float kMinusBig = -1.0e30f;  // the maximum of no key: finite, so that differences are
constexpr float kUp = 10.0f;           // weights are held times 2^10: f16 keeps small ones
constexpr float kSlack = 5.0f;         // the maximum is raised once a score is 2^5 above it

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

// Blocks of 32 keys of one split.
__device__ __forceinline__ uint32_t kv_split_blocks(const wh_kv4_attn_args& a, uint32_t n_keys) {
    return wh_kv4_per_split(n_keys, 32, a.splits, a.min_blocks);
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

template <int HD>
struct wh_kv4_dims {
    static constexpr int kSteps = HD / 32;                // products of 32 dims
    static constexpr int kPieces = HD >= 128 ? HD / 128 : 1;  // loads a lane makes of a row
    static constexpr int kWords = HD >= 128 ? 4 : 2;      // dwords of a load: 32 (16) dims
    static constexpr int kScaleWords = HD >= 128 ? HD / 128 : 1;
    static constexpr int kLd = HD + 16;                   // f16 between rows of a staged block: 16 rows of a
                                                          // transposed read start 32 bytes apart modulo 256
    static constexpr int kStage = 32 * kLd * 2;           // bytes of a wave's block
};

// Raw rows of a lane: key lane % 16 of two blocks of 16.
template <int HD>
struct wh_kv4_raw {
    uint32_t c[2][wh_kv4_dims<HD>::kPieces][wh_kv4_dims<HD>::kWords];
    uint32_t s[2][wh_kv4_dims<HD>::kScaleWords];
};

template <int HD>
__device__ __forceinline__ void kv_load(wh_kv4_raw<HD>& r, int half, const wh_kv4_plane& p, uint64_t line, uint32_t g) {
    using D = wh_kv4_dims<HD>;
    const uint8_t* c = p.codes + line * (HD / 2) + g * (4 * D::kWords);
#pragma unroll
    for (int j = 0; j < D::kPieces; ++j) {
        if constexpr (D::kWords == 4) {
            const wh_u4 w = *(const wh_u4*)(c + 64 * j);
#pragma unroll
            for (int k = 0; k < 4; ++k) r.c[half][j][k] = w[k];
        } else {
            const wh_u2 w = *(const wh_u2*)c;
            r.c[half][j][0] = w[0];
            r.c[half][j][1] = w[1];
        }
    }
    const uint8_t* s = p.scales + line * (HD / 32);
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
template <int HD>
__device__ __forceinline__ uint32_t kv_top_byte(const wh_kv4_raw<HD>& r, int half) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < wh_kv4_dims<HD>::kScaleWords; ++k) m = max(m, kv_max_bytes(r.s[half][k]));
    return m;
}

// Scale of piece j relative to the row's largest byte; 0 where the row is none or holds NaN.
template <int HD>
__device__ __forceinline__ float kv_rel(const wh_kv4_raw<HD>& r, int half, int j, uint32_t g, uint32_t top, bool dead) {
    const uint32_t b = HD == 64 ? (r.s[half][0] >> (8 * (g >> 1))) & 0xff : (r.s[half][j] >> (8 * g)) & 0xff;
    const int e = (int)b - (int)top + 127;
    return dead ? 0.0f : kv_bits((uint32_t)max(e, 0) << 23);
}

// Four waves share a tile of 16 rows; wave w takes the blocks of 32 keys w,
// w + 4, ... of the workgroup's run with a softmax of its own, and the four
// are joined at the end.  Scores are formed as [key][row], so a lane's eight
// weights of a row are already the operand of the product with the values,
// whose rows pass through the wave's own LDS for the transposed read: no
// barrier between waves before the end.
template <int HD, bool kF32, bool kLatent>
__global__ void __launch_bounds__(256) k_kv4_attn(wh_kv4_attn_args a) {
    using D = wh_kv4_dims<HD>;
    constexpr int kParts = kF32 ? 2 : 1;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(16) float key_scale[4][2][32];  // [wave][keys', values'][key]
    __shared__ float row_m[4][16], row_l[4][16];
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63, r16 = lane & 15, g = lane >> 4;
    const uint32_t kvh = blockIdx.y;
    const wh_kv4_tile tile = kv_tile<16>(a, blockIdx.x);
    if (!tile.ok) return;
    const uint32_t per = kv_split_blocks(a, tile.n_keys), blocks = (tile.n_keys + 31) / 32;
    const uint32_t blk0 = blockIdx.z * per, blk1 = min(blocks, blk0 + per);
    if (blockIdx.z && blk0 >= blocks) return;
    const bool whole = per >= blocks;  // the only split: the result is final

    // this lane's row
    const uint32_t rr = min(r16, tile.rows - 1), flat = tile.row0 + rr, tok = flat / a.group;
    const uint32_t head = kvh * a.group + (flat - tok * a.group);
    const bool live = r16 < tile.rows && tile.token0 + tok < a.n_tokens;
    const uint32_t token = min(tile.token0 + tok, a.n_tokens - 1);
    const int32_t pos = live ? tile.len - (int32_t)tile.n_q + (int32_t)tok : -1;

    // the row's query, scaled, in one or two f16 parts
    wh_h8 q[D::kSteps][kParts];
    float c_row;  // score = c_row * key scale * sum
    {
        auto dim = [&](int s) { return HD >= 128 ? 32 * (4 * (s >> 2) + (int)g) + 8 * (s & 3) : 16 * (int)g + 8 * s; };
        const uint64_t at = (uint64_t)token * a.q_stride + (uint64_t)head * HD;
        uint32_t top = 0;
        float v[D::kSteps][8];
#pragma unroll
        for (int s = 0; s < D::kSteps; ++s) {
            if constexpr (kF32) {
                const wh_f4* p = (const wh_f4*)((const float*)a.q + at + dim(s));
                const wh_f4 x = p[0], y = p[1];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[s][k] = x[k];
                    v[s][4 + k] = y[k];
                }
            } else {
                const wh_u4 w = *(const wh_u4*)((const uint16_t*)a.q + at + dim(s));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[s][2 * k] = kv_bits(w[k] << 16);
                    v[s][2 * k + 1] = kv_bits(w[k] & 0xffff0000u);
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[s][k]) & 0x7fffffffu);
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
        const int e = max((int)(top >> 23), 27);  // of the largest; 2^-100 at least, so that the factor is finite
        const float up = kv_bits((uint32_t)(127 + 13 + 127 - e) << 23);
        c_row = a.scale_log2 * kv_bits((uint32_t)max(e - 13, 1) << 23);
#pragma unroll
        for (int s = 0; s < D::kSteps; ++s)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float x = v[s][k] * up;
                q[s][0][k] = (_Float16)x;
                if constexpr (kF32) q[s][1][k] = (_Float16)(x - (float)q[s][0][k]);
            }
    }

    wh_f4 acc[HD / 16];  // [dim 4g + i][row] of 16 dims each, times 2^(127 - ref)
#pragma unroll
    for (int f = 0; f < HD / 16; ++f) acc[f] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};
    float m = kMinusBig, l = 0.0f;
    int ref = 0;  // values are taken relative to this scale byte

    const uint32_t* const table = a.tables + tile.request * a.table_stride;
    const uint32_t pmask = (1u << a.s.shift) - 1u;
    wh_kv4_raw<HD> kr, vr;
    bool there[2];
    auto request = [&](uint32_t blk) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t v = blk * 32 + 16 * h + r16;
            there[h] = blk < blk1 && v < tile.n_keys;
            const uint32_t key = there[h] ? wh_kv4_key(tile, v) : 0;
            uint32_t page = there[h] ? table[key >> a.s.shift] : 0;
            if (page >= a.s.n_pages) {
                atomicOr(a.status, WH_ST_NOT_RESIDENT);
                there[h] = false;
                page = 0;
            }
            const uint64_t line = wh_kv4_line(page, kvh, key & pmask, a.s.kv_heads, a.s.shift);
            kv_load<HD>(kr, h, a.k, line, g);
            if constexpr (!kLatent) kv_load<HD>(vr, h, a.v, line, g);
        }
    };
    _Float16* const stage = (_Float16*)(smem + wave * D::kStage);
    auto put = [&](int h, int j, int w, const wh_h8& x) {
        const int d = HD >= 128 ? 32 * (4 * j + (int)g) + 8 * w : 16 * (int)g + 8 * w;
        *(wh_h8*)(stage + (16 * h + r16) * D::kLd + d) = x;
    };

    for (uint32_t blk = blk0 + wave; blk < blk1; blk += 4) {
        request(blk);
        uint32_t ktop[2], vtop[2];
        bool dead[2], vdead[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            ktop[h] = kv_top_byte<HD>(kr, h);
            dead[h] = !there[h] || ktop[h] == 255;
            if constexpr (kLatent) {
                vtop[h] = ktop[h];
                vdead[h] = dead[h];
            } else {
                vtop[h] = kv_top_byte<HD>(vr, h);
                vdead[h] = !there[h] || vtop[h] == 255;
            }
        }
        // a value row above the reference: raise it, with room, and scale what is there
        const bool above = (!vdead[0] && (int)vtop[0] > ref) || (!vdead[1] && (int)vtop[1] > ref);
        if (__ballot(above)) {
            int top = max(vdead[0] ? 0 : (int)vtop[0], vdead[1] ? 0 : (int)vtop[1]);
            for (int off = 8; off >= 1; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
            const int to = min(top + 3, 254);
            const float f = kv_bits((uint32_t)max(ref - to + 127, 0) << 23);
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) acc[i] *= f;
            ref = to;
        }
        kv_wave_order();
        if (g == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float nan = kv_bits(0x7fc00000u);
                key_scale[wave][0][16 * h + r16] = ktop[h] == 255 ? nan : kv_bits(ktop[h] << 23);
                key_scale[wave][1][16 * h + r16] =
                    vtop[h] == 255 ? nan : kv_bits((uint32_t)max((int)vtop[h] - ref + 127, 0) << 23);
            }
        }
        wh_f4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s[h] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < D::kPieces; ++j) {
                const float rel = kv_rel<HD>(kr, h, j, g, ktop[h], dead[h]);
#pragma unroll
                for (int w = 0; w < D::kWords; ++w) {
                    const wh_h8 x = kv_decode(kr.c[h][j][w], rel);
                    if constexpr (kF32) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[j * D::kWords + w][1], s[h], 0, 0, 0);
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[j * D::kWords + w][0], s[h], 0, 0, 0);
                    if constexpr (kLatent) put(h, j, w, x);
                }
            }
            if constexpr (!kLatent) {
#pragma unroll
                for (int j = 0; j < D::kPieces; ++j) {
                    const float rel = kv_rel<HD>(vr, h, j, g, vtop[h], vdead[h]);
#pragma unroll
                    for (int w = 0; w < D::kWords; ++w) put(h, j, w, kv_decode(vr.c[h][j][w], rel));
                }
            }
        }
        kv_wave_order();
        // weights of keys 4g + i of each half, row r16
        float p[2][4], top = kMinusBig;
        bool seen[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const wh_f4 ks = *(const wh_f4*)&key_scale[wave][0][16 * h + 4 * g];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = blk * 32 + 16 * h + 4 * g + i;
                seen[h][i] = v < tile.n_keys && wh_kv4_sees(pos, wh_kv4_key(tile, v), a.window, a.first);
                p[h][i] = s[h][i] * (ks[i] * c_row);
                top = fmaxf(top, seen[h][i] ? p[h][i] : kMinusBig);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__ballot(top > m + kSlack)) {
            const float to = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - to);
            l *= f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) acc[i] *= f;
            m = to;
        }
        wh_h8 ph, pl;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const wh_f4 vs = *(const wh_f4*)&key_scale[wave][1][16 * h + 4 * g];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = seen[h][i] ? __builtin_amdgcn_exp2f(p[h][i] - m + kUp) : 0.0f;
                l += w;
                const float x = seen[h][i] ? w * vs[i] : 0.0f;
                ph[4 * h + i] = (_Float16)x;
                if constexpr (kF32) pl[4 * h + i] = (_Float16)(x - (float)ph[4 * h + i]);
            }
        }
        // values: lane row = dim r16 of 16, keys 4g + i of each half
#pragma unroll
        for (int f = 0; f < HD / 16; ++f) {
            union {
                wh_s4 s[2];
                wh_h8 v;
            } x;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                x.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) wh_s4*)(stage + (16 * h + 4 * g + (r16 >> 2)) * D::kLd + 16 * f +
                                                               4 * (r16 & 3)));
            if constexpr (kF32) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v, pl, acc[f], 0, 0, 0);
            acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v, ph, acc[f], 0, 0, 0);
        }
    }

    // join the four waves
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
        row_m[wave][r16] = m;
        row_l[wave][r16] = l;
    }
    __syncthreads();
    constexpr int kOld = HD + 4;  // floats between rows of a wave's outputs
    float* const o = (float*)smem;
    float mm = row_m[0][r16];
#pragma unroll
    for (int w = 1; w < 4; ++w) mm = fmaxf(mm, row_m[w][r16]);
    {
        const float f = __builtin_amdgcn_exp2f(m - mm) * kv_bits((uint32_t)ref << 23);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) *(wh_f4*)(o + (wave * 16 + r16) * kOld + 16 * i + 4 * g) = acc[i] * f;
    }
    __syncthreads();
    // 16 threads a row
    const uint32_t row = t >> 4, d0 = (t & 15) * 4;
    float M = row_m[0][row], L = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, row_m[w][row]);
#pragma unroll
    for (int w = 0; w < 4; ++w) L += row_l[w][row] * __builtin_amdgcn_exp2f(row_m[w][row] - M);
    const uint32_t rflat = tile.row0 + row, rtok = rflat / a.group, rhead = kvh * a.group + (rflat - rtok * a.group);
    if (row >= tile.rows || tile.token0 + rtok >= a.n_tokens) return;
    float denom = L;
    if (whole && a.sink) denom += __builtin_amdgcn_exp2f(a.sink[rhead] * 1.44269504088896340736f - M + kUp);
    const float inv = denom == 0.0f ? 0.0f : 1.0f / denom;
    float* const part = a.part + ((((uint64_t)blockIdx.x * a.s.kv_heads + kvh) * a.splits + blockIdx.z) * 16 + row) * (HD + 2);
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        const uint32_t d = 64 * i + d0;
        wh_f4 x = *(const wh_f4*)(o + row * kOld + d);
#pragma unroll
        for (int w = 1; w < 4; ++w) x += *(const wh_f4*)(o + (w * 16 + row) * kOld + d);
        x *= inv;
        if (!whole) {
            *(wh_f2*)(part + d) = (wh_f2){x[0], x[1]};
            *(wh_f2*)(part + d + 2) = (wh_f2){x[2], x[3]};
        } else if constexpr (kF32) {
            *(wh_f4*)((float*)a.out + (uint64_t)(tile.token0 + rtok) * a.out_stride + (uint64_t)rhead * HD + d) = x;
        } else {
            union {
                __bf16 b[4];
                wh_u2 u;
            } y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y.b[k] = (__bf16)x[k];
            *(wh_u2*)((uint16_t*)a.out + (uint64_t)(tile.token0 + rtok) * a.out_stride + (uint64_t)rhead * HD + d) = y.u;
        }
    }
    if (!whole && (t & 15) == 0) {
        part[HD] = M;
        part[HD + 1] = L;
    }
}

// Joins the splits of a tile: outputs weighted by their sums of weights, and
// the sink.  16 threads a row.
template <int HD, bool kF32>
__global__ void __launch_bounds__(256) k_kv4_join(wh_kv4_attn_args a) {
    const uint32_t t = threadIdx.x, kvh = blockIdx.y;
    const wh_kv4_tile tile = kv_tile<16>(a, blockIdx.x);
    if (!tile.ok) return;
    const uint32_t per = kv_split_blocks(a, tile.n_keys), blocks = (tile.n_keys + 31) / 32;
    if (per >= blocks) return;
    const uint32_t n = (blocks + per - 1) / per;
    const uint32_t row = t >> 4, d0 = (t & 15) * 4;
    const uint32_t flat = tile.row0 + row, tok = flat / a.group, head = kvh * a.group + (flat - tok * a.group);
    if (row >= tile.rows || tile.token0 + tok >= a.n_tokens) return;
    const float* const part = a.part + (((uint64_t)blockIdx.x * a.s.kv_heads + kvh) * a.splits * 16 + row) * (HD + 2);
    constexpr uint64_t kNext = 16 * (HD + 2);
    float M = kMinusBig, L = 0.0f;
    for (uint32_t k = 0; k < n; ++k) M = fmaxf(M, part[k * kNext + HD]);
    wh_f4 x[HD / 64];
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) x[i] = (wh_f4){0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k = 0; k < n; ++k) {
        const float* const p = part + k * kNext;
        const float w = p[HD + 1] * __builtin_amdgcn_exp2f(p[HD] - M);
        L += w;
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
            const wh_f2 u = *(const wh_f2*)(p + 64 * i + d0), v = *(const wh_f2*)(p + 64 * i + d0 + 2);
            x[i] += (wh_f4){u[0], u[1], v[0], v[1]} * w;
        }
    }
    if (a.sink) L += __builtin_amdgcn_exp2f(a.sink[head] * 1.44269504088896340736f - M + kUp);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const uint64_t at = (uint64_t)(tile.token0 + tok) * a.out_stride + (uint64_t)head * HD;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        const wh_f4 y = x[i] * inv;
        if constexpr (kF32) {
            *(wh_f4*)((float*)a.out + at + 64 * i + d0) = y;
        } else {
            union {
                __bf16 b[4];
                wh_u2 u;
            } z;
#pragma unroll
            for (int k = 0; k < 4; ++k) z.b[k] = (__bf16)y[k];
            *(wh_u2*)((uint16_t*)a.out + at + 64 * i + d0) = z.u;
        }
    }
}

template <int HD, bool kF32, bool kLatent>
hipError_t attn_launch_of(const wh_kv4_attn_args& a, hipStream_t stream) {
    constexpr size_t lds = 4 * (size_t)wh_kv4_dims<HD>::kStage;
    static const hipError_t set = hipFuncSetAttribute((const void*)k_kv4_attn<HD, kF32, kLatent>,
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (set != hipSuccess) return set;
    k_kv4_attn<HD, kF32, kLatent><<<dim3(a.n_tiles, a.s.kv_heads, a.splits), 256, lds, stream>>>(a);
    if (a.splits > 1) k_kv4_join<HD, kF32><<<dim3(a.n_tiles, a.s.kv_heads), 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <int HD>
hipError_t attn_launch_hd(const wh_kv4_attn_args& a, bool bf16, bool latent, hipStream_t stream) {
    if (bf16) return latent ? attn_launch_of<HD, false, true>(a, stream) : attn_launch_of<HD, false, false>(a, stream);
    return latent ? attn_launch_of<HD, true, true>(a, stream) : attn_launch_of<HD, true, false>(a, stream);
}

}  // namespace

hipError_t wh_kv_plan_launch(const wh_kv_plan_args& a, hipStream_t stream) {
    const size_t lds = 3 * ((size_t)a.n + 1) * sizeof(uint32_t);
    const uint64_t copy = a.free_out != a.free_in ? a.n_pages : 0;
    const uint64_t items = std::max<uint64_t>(std::max<uint64_t>(a.max_tokens, copy), 1);
    const uint32_t grid = (uint32_t)std::min<uint64_t>((items + 4 * kPlanThreads - 1) / (4 * kPlanThreads), 256);
    k_kv_plan<<<grid, kPlanThreads, lds, stream>>>(a);
    return hipGetLastError();
}

hipError_t wh_kv4_write_launch(const wh_kv4_rows_args& a, bool bf16, hipStream_t stream) {
    const uint64_t units = (uint64_t)a.n * a.s.kv_heads * (a.s.head_dim / 8);
    const dim3 grid((uint32_t)((units + 255) / 256), a.planes);
    if (bf16) k_kv4_write<true><<<grid, 256, 0, stream>>>(a);
    else k_kv4_write<false><<<grid, 256, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t wh_kv4_read_launch(const wh_kv4_rows_args& a, bool bf16, hipStream_t stream) {
    const uint64_t units = (uint64_t)a.n * a.s.kv_heads * (a.s.head_dim / 8);
    const dim3 grid((uint32_t)((units + 255) / 256), a.planes);
    if (bf16) k_kv4_read<true><<<grid, 256, 0, stream>>>(a);
    else k_kv4_read<false><<<grid, 256, 0, stream>>>(a);
    return hipGetLastError();
}

wh_kv4_attn_plan wh_kv4_attn_plan_of(const wh_kv4_attn_args& a, bool bf16, bool latent, size_t max_len) {
    (void)bf16;
    (void)latent;
    wh_kv4_attn_plan p{};
    p.n_tiles = (uint32_t)((uint64_t)a.n_tokens * a.group / 16 + a.n_requests);
    const uint64_t wgs = (uint64_t)p.n_tiles * a.s.kv_heads;
    uint64_t keys = max_len;
    if (a.window) keys = std::min<uint64_t>(keys, (uint64_t)a.window + a.first + a.n_tokens);
    const uint64_t want = (512 + wgs - 1) / wgs, most = (keys + 127) / 128;
    p.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(want, std::min<uint64_t>(most, 64)));
    p.min_blocks = 4;
    if (p.splits > 1) p.part_bytes = wgs * p.splits * 16 * (a.s.head_dim + 2) * sizeof(float);
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
