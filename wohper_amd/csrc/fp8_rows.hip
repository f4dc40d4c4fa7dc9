// 8-bit rows (gfx950): activations to E4M3 codes and back, their products with
// resident FP8 weights, plain and grouped by expert, expert lists from routes
// and the sum over a position's experts.
//
// A row holds one code a column and one UE8M0 scale byte for every 128 columns:
// value = code * 2^(byte - 127).  Inside a block of 128 the codes lie in the
// weight store's lane order (byte 16 l + i is column 16 (i % 8) + 8 (i / 8) + l,
// kernels.h), so a product multiplies both sides' bytes as they lie: which
// column a byte is does not matter to a sum over the whole block.
#include "fp8_rows.h"

#include <algorithm>
#include <atomic>
#include <cmath>

#include "wh_device.h"

namespace {

typedef uint32_t wh_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t wh_u4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kNone = WH_ROWS_NONE;

// Largest over a row of 16 lanes, in all of them.
__device__ __forceinline__ uint32_t rows_max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, false));  // rotated by 8, 4, 2, 1
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, false));
}

// A row's scale byte, as the matrix instructions read it: 255 is NaN, 0 is 2^-127.
__device__ __forceinline__ float rows_scale(uint32_t byte) {
    return __uint_as_float(byte == 255 ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
}

// ------------------------------------------------------------------- rows

// Bytes [8] of the lanes 2 s + h (s < 8) of a row of 16 as an 8 x 8 matrix each for h = 0
// and 1, transposed: byte l of lane 2 s + h goes to byte s of lane 2 l + h.  Three
// exchanges of half of what a lane holds, with the lanes 8, 4 and 2 away.
__device__ __forceinline__ wh_u2 rows_transpose(wh_u2 v) {
    const uint32_t lane = threadIdx.x;
    {
        const bool hi = lane & 8;
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(hi ? v.x : v.y), 0x128, 0xf, 0xf, false);
        if (hi) v.x = got;
        else v.y = got;
    }
    {
        const bool hi = lane & 4;
        const uint32_t give = __builtin_amdgcn_perm(v.y, v.x, hi ? 0x05040100u : 0x07060302u);
        const uint32_t got = (uint32_t)__builtin_amdgcn_ds_swizzle((int)give, 0x101f);  // lane ^ 4
        v = hi ? wh_u2{__builtin_amdgcn_perm(v.x, got, 0x07060100u), __builtin_amdgcn_perm(v.y, got, 0x07060302u)}
               : wh_u2{__builtin_amdgcn_perm(got, v.x, 0x05040100u), __builtin_amdgcn_perm(got, v.y, 0x07060100u)};
    }
    {
        const bool hi = lane & 2;
        const uint32_t give = __builtin_amdgcn_perm(v.y, v.x, hi ? 0x06040200u : 0x07050301u);
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0x4e, 0xf, 0xf, false);  // lane ^ 2
        v = hi ? wh_u2{__builtin_amdgcn_perm(v.x, got, 0x07010500u), __builtin_amdgcn_perm(v.y, got, 0x07030502u)}
               : wh_u2{__builtin_amdgcn_perm(got, v.x, 0x05020400u), __builtin_amdgcn_perm(got, v.y, 0x07020600u)};
    }
    return v;
}

// Eight values from p on.  Rows may begin at any value: the hardware takes a 16-byte load
// at any address.
template <bool kBf16>
__device__ __forceinline__ void rows_load8(const void* p, uint64_t at, float (&v)[8]) {
    if constexpr (kBf16) {
        uint16_t w[8];
        __builtin_memcpy(w, (const uint16_t*)p + at, sizeof(w));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float((uint32_t)w[i] << 16);
    } else {
        __builtin_memcpy(v, (const float*)p + at, sizeof(v));
    }
}

// exp(-x), x >= 0 or NaN, within 3 units of 2^-24: a power of two of the product with
// log2(e) in two pieces, whose rest goes in by the first terms of its series.  The
// instruction has no results below 2^-126, where expf has.
__device__ __forceinline__ void rows_exp(const float (&x)[8], float (&z)[8]) {
    constexpr float kHi = -1.44269502f, kLo = -1.92596299e-8f, kLn2 = 0.693147182f;
    float most = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, x[i]);
    if (most < 87.0f) {  // fmaxf passes over NaN, which both ways keep
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = x[i] * kHi, rest = fmaf(x[i], kLo, fmaf(x[i], kHi, -t)), p = __builtin_amdgcn_exp2f(t);
            z[i] = fmaf(p, rest * kLn2, p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = expf(-x[i]);
    }
}

// Rows to 8 bits.  Sixteen lanes take a block of 128 columns, lane q columns 8 q .. 8 q + 7;
// their codes change places so that lane q has the store's bytes 8 q .. 8 q + 7.  The scale
// is the least power of two, 2^-126 at least, under which the block's largest finite
// magnitude is at most 448: from its bits, since 448 is 1.75 * 2^8.  Values times its
// inverse are exact (or round to code 0), so each code is rounded once, to nearest even.
// Infinities and NaN become NaN and do not count for the scale.
// Bound by memory: 8192 x 4096 in bf16 there and back 41 us (52 with a lane's columns 16
// apart, which needs no exchange but loads of two bytes), 24001 x 2048 behind SwiGLU there
// and back 80.6 us, both 4.9 TB/s, the rate of a large copy.
template <bool kBf16, bool kSwiglu>
__global__ void __launch_bounds__(256) k_rows_quant(wh_rows_quant_args a) {
    const uint64_t unit = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const uint32_t q = threadIdx.x & 15;
    const uint64_t row = unit / a.blocks;
    const uint32_t block = (uint32_t)(unit - row * a.blocks);
    if (row >= a.n) return;  // all sixteen lanes
    const uint64_t at = row * a.x_stride + block * 128u + 8 * q;
    float v[8];
    rows_load8<kBf16>(a.x, at, v);
    if constexpr (kSwiglu) {
        float u[8], x[8], z[8];
        rows_load8<kBf16>(a.up, at, u);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            // NaN stays NaN through both clamps
            v[i] = v[i] > a.limit ? a.limit : v[i];
            u[i] = u[i] > a.limit ? a.limit : u[i] < -a.limit ? -a.limit : u[i];
            x[i] = fabsf(v[i]);
        }
        rows_exp(x, z);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            // 1 / (1 + z), between 1/2 and 1: an estimate within 2^-23 and a step of Newton's
            const float d = 1.0f + z[i], r = __builtin_amdgcn_rcpf(d), s = fmaf(fmaf(-d, r, 1.0f), r, r);
            v[i] = v[i] * ((v[i] < 0.0f ? z[i] : 1.0f) * s) * u[i];
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    uint32_t bad = 0;
    if (top >= 0x7f800000u) {  // these become NaN's code on code 0
        top = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
            if (b < 0x7f800000u) top = max(top, b);
            else v[i] = 0.0f, bad |= 1u << i;
        }
    }
    top = rows_max16(top);
    int e = (int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, -126);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    wh_u2 codes;
    codes.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    codes.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, (int)codes.x, true);
    codes.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
    codes.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, (int)codes.y, true);
    if (bad) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (bad >> i & 1) codes.x |= 0x7fu << 8 * i;
            if (bad >> (4 + i) & 1) codes.y |= 0x7fu << 8 * i;
        }
    }
    *(wh_u2*)(a.out.codes + row * a.out.stride + block * 128u + 8 * q) = rows_transpose(codes);
    if (q == 0) a.out.scales[row * a.out.scale_stride + block] = top ? (uint8_t)(e + 127) : 0;
}

// 8-bit rows as the values they stand for: the same lanes the other way.
template <bool kBf16>
__global__ void __launch_bounds__(256) k_rows_read(wh_rows_read_args a) {
    const uint64_t unit = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const uint32_t q = threadIdx.x & 15;
    const uint64_t row = unit / a.blocks;
    const uint32_t block = (uint32_t)(unit - row * a.blocks);
    if (row >= a.n) return;  // all sixteen lanes
    const wh_u2 codes = rows_transpose(*(const wh_u2*)(a.in.codes + row * a.in.stride + block * 128u + 8 * q));
    const float scale = rows_scale(a.in.scales[row * a.in.scale_stride + block]);
    const uint64_t at = row * a.out_stride + block * 128u + 8 * q;
    const wh_f2 p[4] = {wh_fp8x2<false, false>(codes.x), wh_fp8x2<false, true>(codes.x), wh_fp8x2<false, false>(codes.y),
                        wh_fp8x2<false, true>(codes.y)};
    if constexpr (kBf16) {
        __bf16 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (__bf16)((i & 1 ? p[i / 2].y : p[i / 2].x) * scale);
        __builtin_memcpy((__bf16*)a.out + at, o, sizeof(o));
    } else {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (i & 1 ? p[i / 2].y : p[i / 2].x) * scale;
        __builtin_memcpy((float*)a.out + at, o, sizeof(o));
    }
}

// --------------------------------------------------------------- products

// The t-th tile of at most kRows listed rows [r0, r1) of one group g.  With
// groups, tiles are numbered group by group: every wave adds up the groups' tiles
// 64 at a time.  False behind the last tile.  Starts that do not ascend, or pass
// n, are cut off.
template <uint32_t kRows>
__device__ __forceinline__ bool rows_tile(const wh_rows_mm_args& a, uint32_t t, uint32_t& g, uint32_t& r0, uint32_t& r1) {
    if (!a.starts) {
        g = 0;
        r0 = t * kRows;
        r1 = min(a.n, r0 + kRows);
        return r0 < a.n;
    }
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t base = 0; base < a.n_groups; base += 64) {
        const uint32_t at = base + lane;
        uint32_t s = 0, e = 0;
        if (at < a.n_groups) {
            s = min(a.starts[at], a.n);
            e = max(s, min(a.starts[at + 1], a.n));
        }
        const uint32_t tiles = (e - s + kRows - 1) / kRows;
        uint32_t upto = tiles;
#pragma unroll
        for (uint32_t off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(upto, off, 64);
            if (lane >= off) upto += y;
        }
        const uint64_t past = __ballot(before + upto > t);
        if (past) {
            const uint32_t first = (uint32_t)__builtin_ctzll(past);
            const uint32_t own = __shfl(before + upto - tiles, first, 64);
            g = base + first;
            r0 = __shfl(s, first, 64) + (t - own) * kRows;
            r1 = min(__shfl(e, first, 64), r0 + kRows);
            return true;
        }
        before += __shfl(upto, 63, 64);
    }
    return false;
}

// Most tiles of `rows` listed rows that a call can have.
__host__ __device__ __forceinline__ uint64_t rows_tiles(const wh_rows_mm_args& a, uint32_t rows) {
    const uint64_t full = ((uint64_t)a.n + rows - 1) / rows;
    // each group may end in a tile that is not full, and has at least a row then
    return a.starts ? full + (a.n_groups < a.n ? a.n_groups : a.n) : full;
}

// Scale of weight row `row` in block b as mantissa * 2^exponent, so that its
// product with a row's power of two leaves f32's range only where the result does.
__device__ __forceinline__ float rows_w_scale(const wh_rows_mm_args& a, uint64_t row, uint32_t b, int* e) {
    const uint64_t at = row / a.row_block * (a.cols / 128u) + b;
    *e = 0;
    if (a.scale_f32) {
        const float s = ((const float*)a.w_scales)[at];
        if (!(fabsf(s) <= 3.4028235e38f)) return s;
        return frexpf(s, e);
    }
    const uint32_t byte = ((const uint8_t*)a.w_scales)[at];
    if (byte == 0 || byte == 255) return wh_ue8m0(byte);
    *e = (int)byte - 127;
    return 1.0f;
}

template <bool kBf16>
__device__ __forceinline__ void rows_put(const wh_rows_mm_args& a, uint64_t row, uint32_t col, float v) {
    if constexpr (kBf16) ((__bf16*)a.y)[row * a.y_stride + col] = (__bf16)v;
    else ((float*)a.y)[row * a.y_stride + col] = v;
}

// Any product: 16 x 16 outputs a workgroup, one a thread, the block's values of
// both sides decoded into LDS.  For what the matrix instructions read otherwise or
// do not take: weight codes 0x7F / 0xFF (+-480 here, NaN there) and scales shared
// by a number of rows that is no multiple of 16, and for sizes whose tiles there are more
// than a launch has threads for.  A workgroup here takes further tiles where they are more
// than a grid has workgroups, so it takes any sizes, whatever the weight's codes.  Bound by LDS reads and vector products: 5 x 4096 x 8192
// in f32 95 us, 4096 x 4096 x 8192 25 ms.
constexpr uint32_t kAnyRows = 16;
template <bool kBf16>
__device__ __forceinline__ void rows_any(const wh_rows_mm_args& a, float (*xs)[132], float (*ws)[132], uint32_t g, uint32_t r0,
                                         uint32_t r1, uint32_t c0) {
    const uint32_t t = threadIdx.x, lane16 = t & 15, row16 = t >> 4;
    const uint64_t w0 = a.row_start + (uint64_t)g * a.out_rows;
    // staging: thread (row16, lane16) brings 8 codes of row row16 of both sides
    uint32_t src = 0;
    bool have = r0 + row16 < r1;
    if (have) {
        src = a.rows ? a.rows[r0 + row16] : r0 + row16;
        have = src < a.n_x;
    }
    const bool have_w = c0 + row16 < a.out_rows;
    const uint64_t w_row = w0 + c0 + row16, my_w = w0 + min(c0 + lane16, a.out_rows - 1);
    float acc = 0.0f;
    for (uint32_t b = 0; b < a.cols / 128u; ++b) {
        wh_u2 xc = {0, 0}, wc = {0, 0};
        if (have) xc = *(const wh_u2*)(a.x.codes + (uint64_t)src * a.x.stride + b * 128u + 8 * lane16);
        if (have_w) wc = *(const wh_u2*)(a.w + w_row * a.cols + b * 128u + 8 * lane16);
        __syncthreads();
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t xw = h ? xc.y : xc.x, ww = h ? wc.y : wc.x;
            const wh_f2 x0 = wh_fp8x2<false, false>(xw), x1 = wh_fp8x2<false, true>(xw);
            const wh_f2 w0v = wh_fp8x2<true, false>(ww), w1v = wh_fp8x2<true, true>(ww);
            float* const xd = &xs[row16][8 * lane16 + 4 * h];
            float* const wd = &ws[row16][8 * lane16 + 4 * h];
            xd[0] = x0.x, xd[1] = x0.y, xd[2] = x1.x, xd[3] = x1.y;
            wd[0] = w0v.x, wd[1] = w0v.y, wd[2] = w1v.x, wd[3] = w1v.y;
        }
        __syncthreads();
        float sum = 0.0f;
        for (uint32_t k = 0; k < 128; ++k) sum = fmaf(xs[row16][k], ws[lane16][k], sum);
        int e = 0;
        const float m = rows_w_scale(a, my_w, b, &e);
        if (have) {
            const int byte = a.x.scales[(uint64_t)src * a.x.scale_stride + b];
            acc += byte == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(sum * m, byte - 127 + e);
        }
    }
    if (r0 + row16 < r1 && c0 + lane16 < a.out_rows) rows_put<kBf16>(a, r0 + row16, c0 + lane16, acc);
}

template <bool kBf16>
__global__ void __launch_bounds__(256) k_rows_mm_any(wh_rows_mm_args a) {
    __shared__ float xs[kAnyRows][132], ws[16][132];
    const uint32_t n_cols = (a.out_rows + 15) / 16;
    const uint64_t tiles = rows_tiles(a, kAnyRows) * n_cols;
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        uint32_t g = 0, r0 = 0, r1 = 0;
        if (!rows_tile<kAnyRows>(a, (uint32_t)(tile / n_cols), g, r0, r1)) return;
        rows_any<kBf16>(a, xs, ws, g, r0, r1, (uint32_t)(tile % n_cols) * 16);
    }
}

// ------------------------------------------------- matrix instructions
//
// Weights are the first operand and x rows the second, so a lane of a 16 x 16
// result holds four consecutive columns of one y row.  A lane brings 32 bytes of a
// 128-byte block, its 16-byte chunks q and 4 + q (q = lane / 16): which columns
// those are is the same for both sides.
//
// bf16 results take the 8-bit instruction with both scales as its block scales.
// It aligns the products of eight bytes to the largest of them, keeps 13 bits under
// it and adds that to the f32 sum, so an f32 result would be 2e-5 to 6e-5 off (of the
// results' norm, rows of 4096; 1.01 * 2^-10 of the products' magnitudes where all is lost
// that can be): a hundredth of what rounding to bf16 does, and a hundred times what an
// f32 sum does.  4096 x 4096 x 8192: 1.2 percent of the results are the neighbour of the
// correctly rounded bf16, 2.3e-4 of the norm beside the 1.7e-3 of rounding itself, and
// three times as fast as on f16 instructions.  So f32 results decode both sides to f16, which holds every E4M3
// value, and add a block up in the f16 instruction (8e-8 to 4e-7 off), scaled
// after it.

typedef int wh_i8 __attribute__((ext_vector_type(8)));
typedef _Float16 wh_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 wh_h8 __attribute__((ext_vector_type(8)));

struct rows_frag {
    wh_u4 a, b;
};

__device__ __forceinline__ wh_i8 rows_codes(const rows_frag& f) {
    return wh_i8{(int)f.a.x, (int)f.a.y, (int)f.a.z, (int)f.a.w, (int)f.b.x, (int)f.b.y, (int)f.b.z, (int)f.b.w};
}

// Eight codes as f16.
__device__ __forceinline__ wh_h8 rows_f16(uint32_t lo, uint32_t hi) {
    const wh_h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const wh_h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const wh_h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const wh_h2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return wh_h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
struct rows_f16x4 {
    wh_h8 v[4];
};
__device__ __forceinline__ rows_f16x4 rows_decode(const rows_frag& f) {
    return rows_f16x4{{rows_f16(f.a.x, f.a.y), rows_f16(f.a.z, f.a.w), rows_f16(f.b.x, f.b.y), rows_f16(f.b.z, f.b.w)}};
}

// acc + (block of codes) * 2^e * m.
__device__ __forceinline__ wh_f4 rows_scaled(wh_f4 acc, wh_f4 block, int e, float m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(ldexpf(block[i], e), m, acc[i]);
    return acc;
}

// A weight scale's bits, and they as the byte of a power of two and a factor: 1 for
// ordinary UE8M0 bytes, else in [1, 2), or the scale itself where it is no normal number.
// 0 goes with the least power of two and infinity with the largest, so that neither the
// largest nor the smallest rows leave f32's range before they meet it, where the product
// would be NaN.
__device__ __forceinline__ uint32_t rows_scale_bits(const wh_rows_mm_args& a, uint64_t at) {
    return a.scale_f32 ? ((const uint32_t*)a.w_scales)[at] : ((const uint8_t*)a.w_scales)[at];
}
__device__ __forceinline__ uint32_t rows_split_bits(const wh_rows_mm_args& a, uint32_t u, float* m) {
    *m = 1.0f;
    if (!a.scale_f32) {
        if (u != 0 && u != 255) return u;
        *m = wh_ue8m0(u);
        return u ? 254 : 0;
    }
    const float s = __uint_as_float(u);
    const uint32_t e = u >> 23 & 0xff;
    if (e == 255) {
        *m = s;
        return 254;
    }
    if (e == 0) {  // 0 too
        *m = s * 1.70141183460469231732e38f;  // 2^127
        return 0;
    }
    *m = __uint_as_float((u & 0x807fffffu) | 0x3f800000u);
    return e;
}
__device__ __forceinline__ uint32_t rows_split_scale(const wh_rows_mm_args& a, uint64_t at, float* m) {
    return rows_split_bits(a, rows_scale_bits(a, at), m);
}

// Four values to any address: the hardware takes stores of 8 and 16 bytes there.
template <bool kBf16>
__device__ __forceinline__ void rows_put4(const wh_rows_mm_args& a, uint64_t row, uint32_t col, wh_f4 v) {
    if (col + 4 <= a.out_rows) {
        if constexpr (kBf16) {
            const __bf16 b[4] = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
            __builtin_memcpy((__bf16*)a.y + row * a.y_stride + col, b, sizeof(b));
        } else {
            __builtin_memcpy((float*)a.y + row * a.y_stride + col, &v, sizeof(v));
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (col + i < a.out_rows) rows_put<kBf16>(a, row, col + i, v[i]);
}

// The x row of listed row j, and whether it is one.
__device__ __forceinline__ uint32_t rows_source(const wh_rows_mm_args& a, uint32_t j, bool* is) {
    const uint32_t r = a.rows ? a.rows[j] : j;
    *is = r < a.n_x;
    return *is ? r : 0;
}

// Few rows a group: bound by the weights' bytes.  A wave takes 16 kNt weight rows and one
// of ks_n ranges of their columns for up to 16 kMt x rows, straight from memory into
// registers; the waves of the same weight rows join in LDS.  Blocks come kU at a time, all
// their loads before the first product; a range's blocks lie side by side, so that one
// word holds a row's scales of four.  Registers for two workgroups a CU: 84 rows over 64
// lists of 4096 x 4096, 43 of them not empty, in f32 145 to 157 us (with one workgroup
// 226), 4.6 to 5.0 TB/s, where a large read reaches 6.2.
// x is read again for each 16 kNt weight rows: 16 x 8192 x 8192 in bf16 18.8 us with one, 16.1
// (4.2 TB/s) with two; 5 x 4096 x 8192 in f32 9.4 us, 3.6 TB/s with the launch.  The f32
// form with two spills 5 or 6 registers, two reloaded in the loop over 64 rows.
constexpr uint32_t kThinWaves = 8;
template <int kMt, int kNt, bool kBf16, bool kMant>
__device__ __forceinline__ void rows_thin(const wh_rows_mm_args& a, float (*part)[64][4], uint32_t ks_n, uint32_t g, uint32_t j0,
                                          uint32_t j1, uint32_t c0) {
    // blocks whose weights, and whose x, are asked for at once
    constexpr int kU = kMt * kNt == 1 ? 4 : kMt * kNt == 2 && (kBf16 || kNt == 2) ? 2 : 1, kW = kNt == 2 || kMt == 4 ? kU : 4;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t ks = wave & (ks_n - 1), l16 = lane & 15, q = lane >> 4;
    const uint32_t blocks = a.cols / 128u, col0 = c0 + 16 * kNt * (wave / ks_n);
    const bool works = col0 < a.out_rows;
    wh_f4 acc[kNt][kMt];
    const uint8_t *xp[kMt], *xs[kMt];
    uint32_t src[kMt];
    bool nan[kMt];
#pragma unroll
    for (int t = 0; t < kMt; ++t) {
        const uint32_t j = min(j0 + 16 * t + l16, j1 - 1);
        src[t] = a.rows ? a.rows[j] : j;
        nan[t] = false;
#pragma unroll
        for (int i = 0; i < kNt; ++i) acc[i][t] = wh_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // this wave's blocks, 64 at most
    const uint32_t len = (blocks + ks_n - 1) / ks_n, first = min(ks * len, blocks), mine = works ? min(len, blocks - first) : 0;
    if (mine) {
        const uint64_t w_row = a.row_start + (uint64_t)g * a.out_rows + col0;
        const uint8_t* wp[kNt];
        uint32_t bits[kNt], wb[kNt];
        float wm[kNt];
#pragma unroll
        for (int i = 0; i < kNt; ++i) {
            wp[i] = a.w + (w_row + min(16 * i + l16, a.out_rows - 1 - col0)) * a.cols + 16 * q;
            // scales of this wave's blocks, one a lane: 16 rows share one
            bits[i] = rows_scale_bits(a, (w_row + min(16u * i, a.out_rows - 1 - col0)) / a.row_block * blocks +
                                             min(first + lane, blocks - 1));
        }
        for (uint32_t i0 = 0; i0 < mine; i0 += kW) {
            rows_frag w[kW][kNt];
            uint32_t x0[kMt], x1[kMt];  // the words of the rows' scales that hold these blocks'
#pragma unroll
            for (int u = 0; u < kW; ++u) {
                const uint32_t b = first + min(i0 + u, mine - 1);
#pragma unroll
                for (int i = 0; i < kNt; ++i) {
                    w[u][i].a = *(const wh_u4*)(wp[i] + b * 128u);
                    w[u][i].b = *(const wh_u4*)(wp[i] + b * 128u + 64);
                }
            }
            if (i0 == 0) {  // the first weights are under way: what lists and scales say
#pragma unroll
                for (int i = 0; i < kNt; ++i) wb[i] = rows_split_bits(a, bits[i], &wm[i]);
#pragma unroll
                for (int t = 0; t < kMt; ++t) {
                    const uint32_t r = src[t] < a.n_x ? src[t] : 0;
                    xp[t] = a.x.codes + (uint64_t)r * a.x.stride + 16 * q;
                    xs[t] = a.x.scales + (uint64_t)r * a.x.scale_stride;
                }
            }
            const uint32_t b0 = first + i0, word = b0 / 4, at = b0 & 3;
#pragma unroll
            for (int v = 0; v < kW; v += kU) {
                rows_frag x[kU][kMt];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const uint32_t b = first + min(i0 + v + u, mine - 1);
#pragma unroll
                    for (int t = 0; t < kMt; ++t) {
                        x[u][t].a = *(const wh_u4*)(xp[t] + b * 128u);
                        x[u][t].b = *(const wh_u4*)(xp[t] + b * 128u + 64);
                    }
                }
                if (v == 0) {
#pragma unroll
                    for (int t = 0; t < kMt; ++t) {
                        x0[t] = ((const uint32_t*)xs[t])[word];
                        x1[t] = 0;
                    }
                    if (at + kW > 4) {
#pragma unroll
                        for (int t = 0; t < kMt; ++t) x1[t] = ((const uint32_t*)xs[t])[min(word + 1, (blocks - 1) / 4)];
                    }
                }
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    if (i0 + v + u < mine) {
                        uint32_t xb[kMt];
#pragma unroll
                        for (int t = 0; t < kMt; ++t) xb[t] = __builtin_amdgcn_alignbyte(x1[t], x0[t], at) >> 8 * (v + u) & 0xff;
#pragma unroll
                        for (int i = 0; i < kNt; ++i) {
                            const int byte = __builtin_amdgcn_readlane((int)wb[i], i0 + v + u);
                            const float m = kMant ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wm[i]), i0 + v + u)) : 1.0f;
                            if constexpr (kBf16) {
                                const wh_i8 wc = rows_codes(w[v + u][i]);
#pragma unroll
                                for (int t = 0; t < kMt; ++t) {
                                    const wh_f4 from = kMant ? wh_f4{0.0f, 0.0f, 0.0f, 0.0f} : acc[i][t];
                                    const wh_f4 s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                                        wc, rows_codes(x[u][t]), from, 0, 0, 0, byte, 0, (int)xb[t]);
                                    if constexpr (kMant) {
#pragma unroll
                                        for (int k = 0; k < 4; ++k) acc[i][t][k] = fmaf(s[k], m, acc[i][t][k]);
                                    } else {
                                        acc[i][t] = s;
                                    }
                                }
                            } else {
                                const rows_f16x4 wv = rows_decode(w[v + u][i]);
#pragma unroll
                                for (int t = 0; t < kMt; ++t) {
                                    const rows_f16x4 xv = rows_decode(x[u][t]);
                                    wh_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                    for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv.v[j], xv.v[j], s, 0, 0, 0);
                                    acc[i][t] = rows_scaled(acc[i][t], s, (int)xb[t] + byte - 254, m);
                                    nan[t] |= xb[t] == 255;
                                }
                            }
                        }
                    }
                }
            }
        }
        if constexpr (!kBf16) {
#pragma unroll
            for (int t = 0; t < kMt; ++t)
#pragma unroll
                for (int i = 0; i < kNt; ++i)
                    if (nan[t]) acc[i][t] = wh_f4{1.0f, 1.0f, 1.0f, 1.0f} * __uint_as_float(0x7fc00000u);
        }
    }
    if (ks_n > 1) {
        __syncthreads();  // the parts of the rows before have been read
#pragma unroll
        for (int t = 0; t < kMt; ++t)
#pragma unroll
            for (int i = 0; i < kNt; ++i) *(wh_f4*)part[(wave * kMt + t) * kNt + i][lane] = acc[i][t];
        __syncthreads();
    }
    if (!works) return;
#pragma unroll
    for (int t = 0; t < kMt; ++t) {
        const uint32_t j = j0 + 16 * t + l16;
#pragma unroll
        for (int i = 0; i < kNt; ++i) {
            if (((t * kNt + i) & (ks_n - 1)) != ks) continue;
            wh_f4 v = acc[i][t];
            if (ks_n > 1) {
                const uint32_t at = ((wave - ks) * kMt + t) * kNt + i;
                v = *(const wh_f4*)part[at][lane];
                for (uint32_t s = 1; s < ks_n; ++s) v += *(const wh_f4*)part[at + s * kMt * kNt][lane];
            }
            const uint32_t col = col0 + 16 * i + 4 * q;
            if (j < j1 && col < a.out_rows) rows_put4<kBf16>(a, j, col, src[t] < a.n_x ? v : wh_f4{0.0f, 0.0f, 0.0f, 0.0f});
        }
    }
}

// kNt: blocks of 16 weight rows a wave.
template <bool kBf16, bool kMant, int kNt>
__global__ void __launch_bounds__(64 * kThinWaves, 4) k_rows_mm_thin(wh_rows_mm_args a, uint32_t ks_n) {
    __shared__ __align__(16) float part[kThinWaves * 4][64][4];
    const uint32_t g = blockIdx.y, step = 16 * (kThinWaves / ks_n), c0 = blockIdx.x * step * kNt;
    uint32_t j0 = 0, j1 = a.n;
    if (a.starts) {
        j0 = min(a.starts[g], a.n);
        j1 = min(a.starts[g + 1], a.n);
    }
    while (j0 < j1) {
        const uint32_t left = j1 - j0;
        if (left <= 16) {
            rows_thin<1, kNt, kBf16, kMant>(a, part, ks_n, g, j0, j1, c0);
            return;
        }
        if (left <= 32) {
            rows_thin<2, kNt, kBf16, kMant>(a, part, ks_n, g, j0, j1, c0);
            return;
        }
        for (int i = 0; i < kNt; ++i) rows_thin<4, 1, kBf16, kMant>(a, part, ks_n, g, j0, j1, c0 + i * step);
        j0 += 64;
    }
}

// Values between rows of a part.
__host__ __device__ __forceinline__ uint32_t rows_part_stride(const wh_rows_mm_args& a) { return (a.out_rows + 3) / 4 * 4; }

// LDS byte address of a pointer into __shared__ memory.
__device__ __forceinline__ uint32_t rows_lds(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}
// One 16-byte load a lane straight into LDS: lane l's bytes land at lds + 16 l.  The
// compiler does not see them, so its own waits do not empty the queue: rows_arrived
// waits for them.
__device__ __forceinline__ void rows_dma(const uint8_t* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void rows_dma(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
// All of this wave's loads have landed and its LDS reads are done, and every wave's.
__device__ __forceinline__ void rows_arrived() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The same for all but the last kLeft of this wave's loads.
template <int kLeft>
__device__ __forceinline__ void rows_arrived_but() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

// Tiles of at most kM listed rows [r0, r1) of one group g and kN columns from c0 on.
// They are numbered group by group, in bands of kBand tiles of rows, columns outside
// rows, and every XCD (workgroup id mod 8) takes a run of consecutive ones, so that those
// in flight on one L2 share rows and weights.
constexpr uint32_t kBand = 8;
template <uint32_t kM, uint32_t kN>
struct rows_tiling {
    const wh_rows_mm_args& a;
    uint32_t n_tiles;     // of columns
    uint64_t total, per;  // tiles, and of them an XCD's
    struct lane_group {
        uint32_t s, e, tiles, upto;  // rows [s, e), their tiles, and all tiles up to it of these 64 groups
    };

    // This lane's group of the 64 from base on.  64 bits over all groups: starts that do not
    // ascend may count rows more than once.
    __device__ __forceinline__ lane_group groups(uint32_t base) const {
        const uint32_t lane = threadIdx.x & 63, at = base + lane;
        lane_group l = {0, 0, 0, 0};
        if (at < a.n_groups) {
            l.s = min(a.starts[at], a.n);
            l.e = max(l.s, min(a.starts[at + 1], a.n));
        }
        l.tiles = l.upto = (l.e - l.s + kM - 1) / kM;
#pragma unroll
        for (uint32_t off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(l.upto, off, 64);
            if (lane >= off) l.upto += y;
        }
        return l;
    }
    __device__ __forceinline__ explicit rows_tiling(const wh_rows_mm_args& args) : a(args), n_tiles((args.out_rows + kN - 1) / kN), total(0) {
        if (!a.starts) total = (a.n + kM - 1) / kM;
        for (uint32_t base = 0; a.starts && base < a.n_groups; base += 64) {
            total += (uint32_t)__builtin_amdgcn_readlane((int)groups(base).upto, 63);
        }
        total *= n_tiles;
        per = (total + 7) / 8;
    }
    __device__ __forceinline__ uint64_t count(uint32_t xcd) const { return xcd * per >= total ? 0 : min(per, total - xcd * per); }
    // The t-th tile of an XCD, t < count.
    __device__ __forceinline__ void at(uint32_t xcd, uint64_t t, uint32_t& g, uint32_t& r0, uint32_t& r1, uint32_t& c0) const {
        t += xcd * per;
        g = r0 = r1 = c0 = 0;
        // tile `own` of a group of `mine` tiles of rows [start, end), fewer than 2^32 tiles
        // with their columns, since its y rows are in memory
        auto place = [&](uint32_t own, uint32_t mine, uint32_t start, uint32_t end) {
            const uint32_t band = own / (kBand * n_tiles), in = own % (kBand * n_tiles), high = min(kBand, mine - band * kBand);
            r0 = start + (band * kBand + in % high) * kM;
            r1 = min(end, r0 + kM);
            c0 = in / high * kN;
        };
        if (!a.starts) return place((uint32_t)t, (a.n + kM - 1) / kM, 0, a.n);
        for (uint32_t base = 0; base < a.n_groups; base += 64) {
            const lane_group l = groups(base);
            const uint64_t past = __ballot((uint64_t)l.upto * n_tiles > t);
            if (past) {
                const uint32_t lead = (uint32_t)__builtin_ctzll(past);
                const uint32_t mine = __builtin_amdgcn_readlane((int)l.tiles, lead);
                const uint64_t own = t - (uint64_t)((uint32_t)__builtin_amdgcn_readlane((int)l.upto, lead) - mine) * n_tiles;
                g = base + lead;
                place(__builtin_amdgcn_readfirstlane((int)own), mine, __builtin_amdgcn_readlane((int)l.s, lead),
                      __builtin_amdgcn_readlane((int)l.e, lead));
                return;
            }
            t -= (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)l.upto, 63) * n_tiles;
        }
    }
};

// Many rows a group: tiles of kM x kN outputs in LDS.  Both sides' blocks of 128 bytes
// go straight from memory into LDS, one step ahead, 16-byte chunk c of row r at place
// c ^ (r % 8), so that the 16-byte reads of a column of chunks hit all banks.  Scales lie
// in LDS too, kScaleBlocks blocks at a time, four rows' bytes (16 apart) in a word,
// as the scaled instruction takes them.
constexpr uint32_t kScaleBlocks = 64;
template <int kMt, int kNt, int kWm, int kWn>
struct rows_tile_shape {
    static constexpr uint32_t kM = 16 * kMt * kWm, kN = 16 * kNt * kWn, kThreads = 64 * kWm * kWn;
    static constexpr uint32_t kStage = (kM + kN) * 128, kXs = 2 * kStage, kWs = kXs + kScaleBlocks * kM;
    static constexpr uint32_t kWm0 = kWs + kScaleBlocks * kN / 16, kNan = kWm0 + kScaleBlocks * kN / 4, kLds = kNan + kM;
};

// Brings the scales of blocks [b0, b0 + kScaleBlocks) below b1 into LDS (b0 a multiple
// of 4); a block behind the last gets bytes 0, whose product of 2^-254 with any sum of
// codes is 0.  One row a thread, its words all in flight.  kHalf: place r is row
// r / 128 * 64 + r % 64.
template <class S, bool kNanFlags, bool kHalf = false>
__device__ __forceinline__ void rows_tile_scales(const wh_rows_mm_args& a, uint8_t* lds, uint32_t b0, uint32_t b1, uint32_t r0,
                                                 uint32_t r1, uint32_t w0, uint32_t c0) {
    const uint32_t blocks = a.cols / 128u, count = min(kScaleBlocks, b1 - b0);
    constexpr uint32_t kParts = S::kThreads / S::kM, kWords = kScaleBlocks / 4 / kParts;
    const uint32_t r = threadIdx.x % S::kM, from = threadIdx.x / S::kM * kWords;
    bool is;
    const uint32_t src = rows_source(a, min(r0 + (kHalf ? r / 128 * 64 + r % 64 : r), r1 - 1), &is);
    const uint32_t* const xs = (const uint32_t*)(a.x.scales + (uint64_t)src * a.x.scale_stride + b0);
    uint32_t v[kWords];
#pragma unroll
    for (uint32_t k = 0; k < kWords; ++k) v[k] = 4 * (from + k) < count ? xs[from + k] : 0;
    constexpr uint32_t kTiles = S::kN / 16, kStep = S::kThreads / kTiles, kEach = kScaleBlocks / kStep;
    const uint32_t t = threadIdx.x % kTiles, k0 = threadIdx.x / kTiles;
    const uint32_t row = (w0 + min(c0 + 16 * t, a.out_rows - 1)) / a.row_block;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t k = k0 + i * kStep;
        float m = 1.0f;
        const uint32_t byte = k < count ? rows_split_scale(a, (uint64_t)row * blocks + b0 + k, &m) : 0;
        lds[S::kWs + k * kTiles + t] = (uint8_t)byte;
        if (a.scale_f32 || a.odd_scale) *(float*)(lds + S::kWm0 + 4 * (k * kTiles + t)) = m;
    }
    uint8_t* const to = lds + S::kXs + r / 64 * 64 + r % 16 * 4 + r % 64 / 16;
    bool nan = false;
#pragma unroll
    for (uint32_t k = 0; k < kWords; ++k) {
        const uint32_t b = 4 * (from + k);
        if (b < count && count - b < 4) v[k] &= (1u << 8 * (count - b)) - 1;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t byte = v[k] >> 8 * j & 0xff;
            to[(b + j) * S::kM] = (uint8_t)byte;
            if (kNanFlags) nan |= byte == 255;
        }
    }
    if (kNanFlags && nan) lds[S::kNan + r] = 1;
}

// Where there are few tiles, their columns are cut into gridDim.y ranges of `per` blocks (a
// multiple of 4), whose parts go to a.part in f32 and k_rows_join adds up: 128 x 4096 x
// 4096 in bf16 24.6 us whole, 18 in four ranges.  f32 results are bound by the vector
// instructions beside the matrix ones, two a product for decoding and two for scales, and
// by the power that the f16 instructions draw: 4096 x 4096 x 4096 138 us, 1.0 PFLOP/s (a
// library's f16 product 1.46), 165 behind idle time, when clocks are low; 333 x 32768 x
// 1024 with f32 scales 34.  Applying both scales as one factor saves 4 to 10 percent, but
// loses bits where its power of two leaves f32's range.
template <bool kBf16, bool kMant>
__global__ void __launch_bounds__(256, 2) k_rows_mm_tile(wh_rows_mm_args a, uint32_t per) {
    constexpr int kMt = 4, kNt = 4, kWm = 2, kWn = 2;
    typedef rows_tile_shape<kMt, kNt, kWm, kWn> S;
    static_assert(kMt == 4 && kNt == 4, "a word of scale bytes is four tiles");
    extern __shared__ __align__(128) uint8_t tile_lds[];
    uint8_t* const lds = tile_lds;
    uint32_t g = 0, r0 = 0, r1 = 0, c0 = 0;
    const rows_tiling<S::kM, S::kN> tiles(a);
    if (blockIdx.x / 8 >= tiles.count(blockIdx.x & 7)) return;
    tiles.at(blockIdx.x & 7, blockIdx.x / 8, g, r0, r1, c0);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t l16 = lane & 15, q = lane >> 4, wm = wave % kWm, wn = wave / kWm;
    const uint32_t first = blockIdx.y * per, end = min(a.cols / 128u, first + per);
    const uint64_t w0 = a.row_start + (uint64_t)g * a.out_rows;
    constexpr uint32_t kWaves = kWm * kWn, kXd = S::kM / 8 / kWaves, kWd = S::kN / 8 / kWaves;
    // this wave's loads: eight rows each, a lane one chunk
    const uint8_t* xp[kXd];
    uint32_t wo[kWd];
    const uint32_t chunk = 16 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (uint32_t i = 0; i < kXd; ++i) {
        bool is;
        const uint32_t src = rows_source(a, min(r0 + (wave + i * kWaves) * 8 + (lane >> 3), r1 - 1), &is);
        xp[i] = a.x.codes + (uint64_t)src * a.x.stride + chunk;
    }
    const uint8_t* wp = a.w + (w0 + c0) * a.cols;
#pragma unroll
    for (uint32_t i = 0; i < kWd; ++i)
        wo[i] = min((wave + i * kWaves) * 8 + (lane >> 3), a.out_rows - 1 - c0) * a.cols + chunk;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(rows_lds(lds));
    auto bring = [&](uint32_t b) {
        const uint32_t to = lds0 + (b - first) % 2 * S::kStage + wave * 1024;
#pragma unroll
        for (uint32_t i = 0; i < kXd; ++i) rows_dma(xp[i] + b * 128u, to + i * kWaves * 1024);
#pragma unroll
        for (uint32_t i = 0; i < kWd; ++i) rows_dma(wp + b * 128u, wo[i], to + S::kM * 128 + i * kWaves * 1024);
    };
    if constexpr (!kBf16) {
        for (uint32_t i = threadIdx.x; i < S::kM; i += S::kThreads) lds[S::kNan + i] = 0;
    }
    wh_f4 acc[kNt][kMt];
#pragma unroll
    for (int i = 0; i < kNt; ++i)
#pragma unroll
        for (int t = 0; t < kMt; ++t) acc[i][t] = wh_f4{0.0f, 0.0f, 0.0f, 0.0f};
    bring(first);
    const uint32_t at = l16 * 128 + ((q ^ (l16 & 7)) << 4);  // the lane's first chunk in a tile of 16 rows
    for (uint32_t b = first; b < end; ++b) {
        const uint32_t k = (b - first) % kScaleBlocks;
        if (k == 0) {
            __syncthreads();
            rows_tile_scales<S, !kBf16>(a, lds, b, end, r0, r1, (uint32_t)w0, c0);
        }
        rows_arrived();
        if (b + 1 < end) bring(b + 1);
        const uint8_t* const stage = lds + (b - first) % 2 * S::kStage;
        const uint8_t* const xt = stage + wm * (16 * kMt * 128);
        const uint8_t* const wt = stage + S::kM * 128 + wn * (16 * kNt * 128);
        const uint32_t xb = *(const uint32_t*)(lds + S::kXs + ((k * (S::kM / 64) + wm) * 16 + l16) * 4);
        const uint32_t wb = *(const uint32_t*)(lds + S::kWs + (k * (S::kN / 64) + wn) * 4);
        wh_f4 m = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (kMant) m = *(const wh_f4*)(lds + S::kWm0 + (k * (S::kN / 64) + wn) * 16);
        auto frag = [&](const uint8_t* p, int i) {
            rows_frag f;
            f.a = *(const wh_u4*)(p + i * 2048 + at);
            f.b = *(const wh_u4*)(p + i * 2048 + (at ^ 64));
            return f;
        };
        if constexpr (kBf16) {
            wh_i8 x[kMt];
#pragma unroll
            for (int t = 0; t < kMt; ++t) x[t] = rows_codes(frag(xt, t));
            wh_static_for<kNt>([&](auto iv) {
                constexpr int i = decltype(iv)::value;
                const wh_i8 w = rows_codes(frag(wt, i));
                wh_static_for<kMt>([&](auto tv) {
                    constexpr int t = decltype(tv)::value;
                    if constexpr (kMant) {
                        const wh_f4 s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                            w, x[t], wh_f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, i, (int)wb, t, (int)xb);
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][t][j] = fmaf(s[j], m[i], acc[i][t][j]);
                    } else {
                        acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x[t], acc[i][t], 0, 0, i, (int)wb, t, (int)xb);
                    }
                });
            });
        } else {
            rows_f16x4 w[kNt];
#pragma unroll
            for (int i = 0; i < kNt; ++i) w[i] = rows_decode(frag(wt, i));
#pragma unroll
            for (int t = 0; t < kMt; ++t) {
                const rows_f16x4 x = rows_decode(frag(xt, t));
                wh_f4 s[kNt];
#pragma unroll
                for (int i = 0; i < kNt; ++i) s[i] = wh_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < kNt; ++i) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[i].v[j], x.v[j], s[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < kNt; ++i)
                    acc[i][t] = rows_scaled(acc[i][t], s[i], (int)(xb >> 8 * t & 0xff) + (int)(wb >> 8 * i & 0xff) - 254, m[i]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kMt; ++t) {
        const uint32_t r = wm * 16 * kMt + 16 * t + l16, j = r0 + r;
        if (j >= r1) continue;
        bool is = true;
        if (a.rows) rows_source(a, j, &is);
        bool nan = false;
        if constexpr (!kBf16) nan = lds[S::kNan + r];
#pragma unroll
        for (int i = 0; i < kNt; ++i) {
            wh_f4 v = acc[i][t];
            if (nan) v = wh_f4{1.0f, 1.0f, 1.0f, 1.0f} * __uint_as_float(0x7fc00000u);
            if (!is) v = wh_f4{0.0f, 0.0f, 0.0f, 0.0f};
            const uint32_t col = c0 + (wn * kNt + i) * 16 + 4 * q;
            if (col >= a.out_rows) continue;
            if (gridDim.y > 1) *(wh_f4*)(a.part + (blockIdx.y * (uint64_t)a.n + j) * rows_part_stride(a) + col) = v;
            else rows_put4<kBf16>(a, j, col, v);
        }
    }
}

// Adds up the parts of listed rows, in order, four columns a thread.
template <bool kBf16>
__global__ void __launch_bounds__(256) k_rows_join(wh_rows_mm_args a, uint32_t splits) {
    const uint32_t units = rows_part_stride(a) / 4;
    const uint64_t u = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint64_t j = u / units;
    const uint32_t col = (uint32_t)(u - j * units) * 4;
    if (j >= a.n || (a.starts && (j < a.starts[0] || j >= a.starts[a.n_groups]))) return;
    const float* p = a.part + j * rows_part_stride(a) + col;
    wh_f4 v = *(const wh_f4*)p;
    for (uint32_t s = 1; s < splits; ++s) v += *(const wh_f4*)(p + s * (uint64_t)a.n * rows_part_stride(a));
    rows_put4<kBf16>(a, j, col, v);
}

// Tiles of 256 x 256 for bf16 results, four waves of 128 x 128, where there are enough
// of them (and no factors of scales, which would take results through vector registers).
// A block's 64 products a wave go in quarters of four by four tiles, in the
// order (w0 x0) (w0 x1) (w1 x1) (w1 x0), the next block's with x0 and x1 changed over:
// so each half of the operands dies in time to take the next block's behind products
// that do not need it, and 128 registers hold both blocks.  In LDS the halves of a block
// are free, and filled with the block after the next, as soon as every wave has read
// them: the first ones a block before the end, the others half a block later, so loads
// run a whole block ahead and come evenly.
// kHalf: a tile of 128 rows, 64 a wave: x0 alone, in two sets of registers.
template <bool kHalf>
__device__ __forceinline__ void rows_big(const wh_rows_mm_args& a, uint8_t* lds, uint32_t g, uint32_t r0, uint32_t r1, uint32_t c0) {
    typedef rows_tile_shape<8, 8, 2, 2> S;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t l16 = lane & 15, q = lane >> 4, wm = wave & 1, wn = wave >> 1, blocks = a.cols / 128u;
    const uint64_t w0 = a.row_start + (uint64_t)g * a.out_rows;
    constexpr int kXt = kHalf ? 4 : 8;                   // tiles of 16 rows a wave
    constexpr uint32_t kLoads = kHalf ? 12 : 16;         // of a wave for a block
    // this wave's loads: eight rows each, a lane one chunk; half h of a side is 64 of each
    // wave's 128 places
    auto place = [&](uint32_t h, uint32_t j) {
        const uint32_t e = wave + 4 * j;
        return 8 * (e % 8) + 128 * (e / 8) + 64 * h;
    };
    const uint8_t* xp[kXt];
    uint32_t wo[8];
    const uint32_t chunk = 16 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t at = place(i / 4, i % 4), row = (kHalf ? at / 128 * 64 + at % 64 : at) + (lane >> 3);
        if (i < kXt) {
            bool is;
            const uint32_t src = rows_source(a, min(r0 + row, r1 - 1), &is);
            xp[i] = a.x.codes + (uint64_t)src * a.x.stride + chunk;
        }
        wo[i] = min(at + (lane >> 3), a.out_rows - 1 - c0) * a.cols + chunk;
    }
    const uint8_t* const wp = a.w + (w0 + c0) * a.cols;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(rows_lds(lds));
    wh_f4 acc[8][kXt];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int t = 0; t < kXt; ++t) acc[i][t] = wh_f4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t at = l16 * 128 + ((q ^ (l16 & 7)) << 4);
    const uint32_t xt = wm * 16384 + at, wt = 32768 + wn * 16384 + at;
    // load j of 8 of x half xh and weight half wh of block b into a buffer
    auto bring = [&](uint32_t b, uint32_t buffer, uint32_t xh, uint32_t wh, uint32_t j) {
        if (j < 4) rows_dma(xp[4 * xh + j] + b * 128u, lds0 + buffer + place(xh, j) * 128);
        else rows_dma(wp + b * 128u, wo[4 * wh + j - 4], lds0 + buffer + 32768 + place(wh, j - 4) * 128);
    };
    // half h of an operand of 16 rows
    auto half = [&](wh_i8& to, uint32_t off, int h) {
        const wh_u4 v = *(const wh_u4*)(lds + (off ^ 64 * h));
#pragma unroll
        for (int j = 0; j < 4; ++j) to[4 * h + j] = (int)v[j];
    };
    wh_i8 x[8], w[8];
    uint32_t xb[2][2], wb[2][2];  // scale bytes of the halves, of even and odd blocks
    auto scales = [&](auto bv, uint32_t k) {
        constexpr int kB = decltype(bv)::value;
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            wb[kB][h] = *(const uint32_t*)(lds + S::kWs + k * 16 + wn * 8 + 4 * h);
            xb[kB][h] = kHalf && h ? 0 : *(const uint32_t*)(lds + S::kXs + ((k * 4 + wm * 2 + h) * 16 + l16) * 4);
        }
    };
    // the 16 products of weight half kW and x half kX (kHalf: set kX), f(n) behind the n-th
    auto quarter = [&](auto bv, auto wv, auto xv, auto&& f) {
        constexpr int kB = decltype(bv)::value, kW = decltype(wv)::value, kX = decltype(xv)::value;
        wh_static_for<16>([&](auto nv) {
            constexpr int n = decltype(nv)::value, i = 4 * kW + n / 4, t = n % 4, at_t = kHalf ? t : 4 * kX + t;
            acc[i][at_t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i], x[4 * kX + t], acc[i][at_t], 0, 0, n / 4,
                                                                            (int)wb[kB][kW], t, (int)xb[kB][kHalf ? 0 : kX]);
            f(nv);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    using std::integral_constant;
    constexpr integral_constant<int, 0> first;
    constexpr integral_constant<int, 1> last;
    wh_static_for<2>([&](auto bv) {
        constexpr int kB = decltype(bv)::value;
        const uint32_t b = min((uint32_t)kB, blocks - 1);
        wh_static_for<8>([&](auto iv) { bring(b, kB * S::kStage, kHalf ? 0 : kB, 0, decltype(iv)::value); });
        wh_static_for<8>([&](auto iv) {
            constexpr int j = decltype(iv)::value;
            if constexpr (!kHalf || j >= 4) bring(b, kB * S::kStage, 1 - kB, 1, j);
        });
    });
    // block b of buffer kB, first with x half kB (kHalf: in x set kB).  There is always a
    // next block and one after it: behind the last they are the last again, and not used,
    // or (blocks go in pairs) multiplied by scales of 0.  Loads and 16-byte LDS reads are
    // spread over the products: a CU takes one load of 64 lanes in 16 cycles, one read in 8.
    auto step = [&](auto bv, uint32_t b, uint32_t k) {
        constexpr int kB = decltype(bv)::value;
        constexpr integral_constant<int, 1 - kB> other;
        constexpr uint32_t here = kB * S::kStage, next = S::kStage - here;
        const uint32_t after = min(b + 2, blocks - 1);
        rows_arrived_but<kLoads>();  // every wave has b's first halves in registers, its second halves are there
        if constexpr (kHalf) {
            quarter(bv, first, bv, [&](auto nv) {
                constexpr int n = decltype(nv)::value;
                if constexpr (n % 2 == 1) bring(after, here, 0, 0, n / 2);
                if constexpr (n % 2 == 0) half(w[n / 4 + 4], here + wt + (n / 4 + 4) * 2048, n / 2 % 2);
            });
            rows_arrived_but<kLoads>();  // every wave has all of b in registers, b + 1's x and first half are there
            quarter(bv, last, bv, [&](auto nv) {
                constexpr int n = decltype(nv)::value;
                if constexpr (n % 4 == 3) bring(after, here, 0, 1, 4 + n / 4);
                if constexpr (n < 8) half(x[4 * (1 - kB) + n / 2], next + xt + n / 2 * 2048, n % 2);
                else half(w[(n - 8) / 2], next + wt + (n - 8) / 2 * 2048, n % 2);
                if constexpr (n == 12) scales(other, (k + 1) % kScaleBlocks);  // behind a chunk's last: read again
            });
            return;
        }
        quarter(bv, first, bv, [&](auto nv) {
            constexpr int n = decltype(nv)::value, t = 4 * (1 - kB) + n / 2;
            if constexpr (n % 4 == 3) bring(after, here, kB, 0, n / 4);
            if constexpr (n < 8) half(x[t], here + xt + t % 8 * 2048, n % 2);
            else if constexpr (n % 2 == 0) half(w[n / 4 + 2], here + wt + (n / 4 + 2) * 2048, n / 2 % 2);
        });
        quarter(bv, first, other, [&](auto nv) {
            constexpr int n = decltype(nv)::value;
            if constexpr (n % 4 == 3) bring(after, here, kB, 0, 4 + n / 4);
            if constexpr (n < 8 && n % 2 == 0) half(w[n / 4 + 6], here + wt + (n / 4 + 6) * 2048, n / 2 % 2);
        });
        rows_arrived_but<kLoads>();  // every wave has all of b in registers, b + 1's first halves are there
        quarter(bv, last, other, [&](auto nv) {
            constexpr int n = decltype(nv)::value;
            if constexpr (n % 4 == 3) bring(after, here, 1 - kB, 1, n / 4);
            if constexpr (n % 2 == 0) half(w[n / 4], next + wt + n / 4 * 2048, n / 2 % 2);
        });
        quarter(bv, last, bv, [&](auto nv) {
            constexpr int n = decltype(nv)::value, t = 4 * (1 - kB) + n / 2;
            if constexpr (n % 4 == 3) bring(after, here, 1 - kB, 1, 4 + n / 4);
            if constexpr (n < 8) half(x[t], next + xt + t % 8 * 2048, n % 2);
            if constexpr (n == 8) scales(other, (k + 1) % kScaleBlocks);  // behind a chunk's last: read again
        });
    };
    for (uint32_t b0 = 0; b0 < blocks; b0 += kScaleBlocks) {
        rows_tile_scales<S, false, kHalf>(a, lds, b0, blocks, r0, r1, (uint32_t)w0, c0);
        rows_arrived_but<kLoads>();
        // the first block's (a later chunk's are there already)
        scales(first, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                half(x[i], xt + i * 2048, h);
                half(w[i], wt + i * 2048, h);
            }
        const uint32_t count = min(kScaleBlocks, blocks - b0);
        for (uint32_t k = 0; k < count; k += 2) {
            step(first, b0 + k, k);
            step(last, b0 + k + 1, k + 1);
        }
    }
    rows_arrived();  // also the loads behind the last block
    // through LDS, so that rows go out in whole lines and by a short loop
    constexpr uint32_t kPitch = 2 * S::kN + 16;
    static_assert(kPitch * S::kM <= S::kLds, "a tile of results");
#pragma unroll
    for (int t = 0; t < kXt; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            typedef __bf16 b4 __attribute__((ext_vector_type(4)));
            const wh_f4 v = acc[i][t];
            *(b4*)(lds + (wm * 16 * kXt + 16 * t + l16) * kPitch + ((wn * 8 + i) * 16 + 4 * q) * 2) =
                b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        }
    __syncthreads();
#pragma unroll 4
    for (uint32_t u = threadIdx.x; u < 32 * kXt * S::kN / 8; u += S::kThreads) {
        const uint32_t r = u / (S::kN / 8), col = c0 + u % (S::kN / 8) * 8, j = r0 + r;
        if (j >= r1 || col >= a.out_rows) continue;
        wh_u4 v = *(const wh_u4*)(lds + r * kPitch + (col - c0) * 2);
        bool is = true;
        if (a.rows) rows_source(a, j, &is);
        if (!is) v = wh_u4{0, 0, 0, 0};
        uint16_t* const to = (uint16_t*)a.y + (uint64_t)j * a.y_stride + col;
        if (col + 8 <= a.out_rows) {
            __builtin_memcpy(to, &v, sizeof(v));
        } else {
            for (uint32_t e = 0; e < 8 && col + e < a.out_rows; ++e) to[e] = (uint16_t)(v[e / 2] >> 16 * (e & 1));
        }
    }
}

// kTall: tiles of 256 rows, those with at most 128 as half tiles; else of 128.  A
// workgroup a CU takes its XCD's tiles until there are none left (half tiles take half
// as long), then other XCDs': the first by its id, the next from a counter that it asks a
// tile ahead.  tickets: [8] tiles taken, workgroups done; 0 between launches.
// 4096 x 4096 x 8192 99 us, 2.8 PFLOP/s, where the clock falls under the matrix
// instructions' power (a library's 8-bit product there 3.0); 21000 rows over 64 uneven
// lists of 4096 x 4096 425 us, 1.7: 18 percent of the tiles' rows are empty, 12 percent of
// the time is the last tiles', and a tile's beginning and end take 9 us beside 46 of
// products.  kTall takes all 512 registers and spills 20 vector and 118 scalar ones, 84
// bytes of scratch, outside the loop over blocks.
template <bool kTall>
__global__ void __launch_bounds__(256, 1) k_rows_mm_big(wh_rows_mm_args a) {
    extern __shared__ __align__(128) uint8_t tile_lds[];
    __shared__ uint32_t upcoming[2];  // the next tile's XCD (8: none) and number
    const rows_tiling<kTall ? 256 : 128, 256> tiles(a);
    const uint32_t mates = gridDim.x / 8, lane = threadIdx.x & 63;
    const bool once = tiles.total <= gridDim.x;  // then nobody takes a second one (XCDs have equal shares)
    uint32_t xcd = blockIdx.x & 7;
    uint64_t t = blockIdx.x / 8;
    if (once && t >= tiles.count(xcd)) return;
    while (xcd < 8) {
        uint32_t taken = 0;
        if (!once && threadIdx.x == 0) taken = atomicAdd(&a.tickets[xcd], 1u);
        if (t < tiles.count(xcd)) {
            uint32_t g, r0, r1, c0;
            tiles.at(xcd, t, g, r0, r1, c0);
            if (kTall && r1 - r0 > 128) rows_big<false>(a, tile_lds, g, r0, r1, c0);
            else rows_big<true>(a, tile_lds, g, r0, r1, c0);
        }
        if (once) return;
        if (threadIdx.x < 64) {  // one wave's view of who has tiles left
            uint32_t x = xcd;
            uint64_t n = (uint64_t)mates + (uint32_t)__builtin_amdgcn_readfirstlane((int)taken);
            while (x < 8 && n >= tiles.count(x)) {
                const uint32_t other = (x + 1 + lane) & 7;
                const uint32_t is = __hip_atomic_load(&a.tickets[other], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const uint64_t left = __ballot(lane < 8 && (uint64_t)mates + is < tiles.count(other));
                if (!left) {
                    x = 8;
                } else {
                    x = (x + 1 + (uint32_t)__builtin_ctzll(left)) & 7;
                    if (lane == 0) taken = atomicAdd(&a.tickets[x], 1u);
                    n = (uint64_t)mates + (uint32_t)__builtin_amdgcn_readfirstlane((int)taken);
                }
            }
            if (lane == 0) {
                upcoming[0] = x;
                upcoming[1] = (uint32_t)n;
            }
        }
        __syncthreads();
        xcd = __builtin_amdgcn_readfirstlane((int)upcoming[0]);
        t = (uint32_t)__builtin_amdgcn_readfirstlane((int)upcoming[1]);
        __syncthreads();
    }
    if (threadIdx.x == 0 && atomicAdd(&a.tickets[8], 1u) == gridDim.x - 1) {
        for (uint32_t i = 0; i < 9; ++i) a.tickets[i] = 0;
    }
}

// The waves that share weight rows in the thin kernel: as many as leave each four
// blocks of columns, whose loads are in flight together, and more where there would be
// at most 128 workgroups: 60 x 600 x 1280 in f32 12.7 -> 6.0 us, 1 x 1817 x 1792 6.9 -> 4.8.
uint32_t rows_thin_split(const wh_rows_mm_args& a) {
    const uint32_t blocks = a.cols / 128u;
    const uint64_t tiles = (uint64_t)std::min(a.n_groups, a.n) * ((a.out_rows + 15) / 16);
    uint32_t ks = 1;
    while (ks < kThinWaves && 2 * ks <= blocks && (blocks >= 8 * ks || tiles * ks <= 128 * kThinWaves)) ks *= 2;
    return ks;
}
// Blocks of 16 weight rows a wave: two where that leaves a workgroup for every CU and there
// are rows enough that reading them half as often counts.  8192 x 4096 with 4, 8 and 16 rows
// in bf16 8.1, 8.9 and 10.3 us with one, 7.7, 8.0 and 8.8 with two; with 8 and 16 in f32 9.2
// and 10.7, 9.4 and 10.1.  Lists gain nothing: 16 of 2048 x 8192 with 4 rows each 58.6, 57.7.
uint32_t rows_thin_tiles(const wh_rows_mm_args& a, bool bf16) {
    const uint64_t waves = (uint64_t)((a.out_rows + 15) / 16) * rows_thin_split(a);
    return a.n_groups == 1 && a.n >= (bf16 ? 4 : 12) && waves >= 2 * 256 * kThinWaves ? 2 : 1;
}

// Whether the matrix instructions take a call: every 16 rows of a tile share a
// scale, and codes mean the same.
bool rows_mm_matrix(const wh_rows_mm_args& a) {
    return !a.special && a.row_block % 16 == 0 && a.row_start % 16 == 0 && (a.out_rows % 16 == 0 || a.n_groups == 1);
}

// ------------------------------------------------------------------ store

// Row-major codes into the store's order, and whether one is 0x7F or 0xFF.
__global__ void __launch_bounds__(256) k_rows_store(const uint8_t* in, uint8_t* out, uint64_t blocks, uint32_t* flags) {
    const uint64_t unit = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const uint32_t q = threadIdx.x & 15;
    if (unit >= blocks) return;  // all sixteen lanes
    uint8_t c[8];
    __builtin_memcpy(c, in + unit * 128 + 8 * q, sizeof(c));
    uint32_t special = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) special |= (c[i] & 0x7fu) == 0x7fu;
    wh_u2 v;
    __builtin_memcpy(&v, c, sizeof(v));
    *(wh_u2*)(out + unit * 128 + 8 * q) = rows_transpose(v);
    if (special) atomicOr(flags, 1u);
}

__global__ void __launch_bounds__(256) k_rows_scales(const uint8_t* scales, uint64_t n, uint32_t* flags) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n && (scales[i] == 0 || scales[i] == 255)) atomicOr(flags, 2u);
}

// ------------------------------------------------------------ expert lists

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// Routes of a workgroup, a chunk: a wave takes `turns` times 64 consecutive ones.
__host__ __device__ constexpr uint32_t plan_chunk(uint32_t turns) { return kPlanThreads * turns; }

// Counts of a chunk: four experts a load.
__host__ __device__ constexpr uint32_t plan_padded(uint32_t n_groups) { return (n_groups + 3) / 4 * 4; }

// What a wave's lanes have stored to LDS is there for its other lanes.
__device__ __forceinline__ void plan_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Lanes with this lane's id (< 2^bits).
__device__ __forceinline__ uint64_t plan_same(uint32_t id, uint32_t bits) {
    uint64_t same = ~0ull;
    for (uint32_t b = 0; b < bits; ++b) {
        const bool set = id >> b & 1;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
    }
    return same;
}

// How many routes of each expert a chunk has.
__global__ void __launch_bounds__(kPlanThreads) k_expert_count(wh_expert_plan_args a, uint32_t chunk) {
    __shared__ uint32_t count[WH_ROWS_MAX_GROUPS];
    const uint32_t padded = plan_padded(a.n_groups);
    for (uint32_t e = threadIdx.x; e < padded; e += kPlanThreads) count[e] = 0;
    __syncthreads();
    const uint32_t from = blockIdx.x * chunk, to = min(a.n, from + chunk);
    for (uint32_t i = from + threadIdx.x; i < to; i += kPlanThreads) {
        const uint32_t id = a.ids[i];
        if (id < a.n_groups) atomicAdd(&count[id], 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < padded; e += kPlanThreads) a.counts[(uint64_t)blockIdx.x * padded + e] = count[e];
}

// The counts of each expert become those of the chunks before, and the sum of all in a row
// behind the last.  A workgroup takes 16 experts, a thread a run of chunks of one.
constexpr uint32_t kSumExperts = 16, kSumRuns = 64;
__global__ void __launch_bounds__(kSumExperts* kSumRuns) k_expert_sum(wh_expert_plan_args a, uint32_t chunks) {
    __shared__ uint32_t run_sum[kSumRuns][kSumExperts];
    const uint32_t padded = plan_padded(a.n_groups), in = threadIdx.x % kSumExperts, run = threadIdx.x / kSumExperts;
    const uint32_t e = blockIdx.x * kSumExperts + in, len = (chunks + kSumRuns - 1) / kSumRuns;
    const uint32_t from = min(run * len, chunks), to = e < padded ? min(from + len, chunks) : from;
    uint32_t* const at = a.counts + e;
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t c = from; c < to; ++c) sum += at[(uint64_t)c * padded];
    run_sum[run][in] = sum;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t r = 0; r < run; ++r) before += run_sum[r][in];
    if (run == kSumRuns - 1 && e < padded) at[(uint64_t)chunks * padded] = before + sum;
#pragma unroll 8
    for (uint32_t c = from; c < to; ++c) {
        const uint32_t v = at[(uint64_t)c * padded];
        at[(uint64_t)c * padded] = before;
        before += v;
    }
}

// Expert lists: a counting sort that keeps the order of routes.  A workgroup takes a
// chunk of routes, a wave consecutive ones 64 at a time; lanes of the same expert find
// each other by ballots over the id's bits, so a route's place is the expert's start, its
// routes of chunks and waves before, of this wave so far, and of lanes before.  With one
// chunk this is the only launch.  kSummed: k_expert_sum has added the chunks' counts up.
template <uint32_t kTurns, bool kSummed>
__global__ void __launch_bounds__(kPlanThreads) k_expert_place(wh_expert_plan_args a, uint32_t chunks, uint32_t bits) {
    extern __shared__ uint32_t lds[];
    uint32_t* const at = lds;  // [kPlanWaves][n_groups]: counts, then next places of a wave
    __shared__ uint32_t wave_sum[kPlanWaves], all_of[WH_ROWS_MAX_GROUPS], before_of[WH_ROWS_MAX_GROUPS], listed;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, E = a.n_groups;
    for (uint32_t i = t; i < kPlanWaves * E; i += kPlanThreads) at[i] = 0;
    if (t < E) {
        const uint32_t padded = plan_padded(E);
        all_of[t] = kSummed ? a.counts[(uint64_t)chunks * padded + t] : 0;
        before_of[t] = kSummed ? a.counts[(uint64_t)blockIdx.x * padded + t] : 0;
    }
    const uint32_t from = blockIdx.x * plan_chunk(kTurns) + wave * 64 * kTurns;
    uint32_t id[kTurns];
    uint64_t same[kTurns];
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
        const uint32_t i = from + 64 * k + lane;
        id[k] = i < a.n ? a.ids[i] : kNone;
    }
    __syncthreads();
    // all chunks' routes of four experts a lane, and those before this chunk: the chunks
    // are dealt out to waves, or to as many waves together as hold all experts
    if (!kSummed && chunks > 1) {
        const uint32_t fours = plan_padded(E) / 4;
        uint32_t shift = 6;
        while (1u << shift < fours) ++shift;
        const uint32_t four = t & ((1u << shift) - 1), parts = kPlanThreads >> shift;
        wh_u4 all = {0, 0, 0, 0}, before = {0, 0, 0, 0};
        if (four < fours) {
#pragma unroll 4
            for (uint32_t c = __builtin_amdgcn_readfirstlane(t >> shift); c < chunks; c += parts) {
                const wh_u4 v = ((const wh_u4*)a.counts)[(uint64_t)c * fours + four];
                all += v;
                if (c < blockIdx.x) before += v;
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (all[j]) atomicAdd(&all_of[4 * four + j], all[j]);
            if (before[j]) atomicAdd(&before_of[4 * four + j], before[j]);
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
        if (id[k] >= E) id[k] = E;  // no expert: a number of its own, E < 2^bits
        same[k] = plan_same(id[k], bits);
        const bool leads = __builtin_ctzll(same[k]) == lane;
        if (leads && id[k] < E) at[wave * E + id[k]] += (uint32_t)__popcll(same[k]);
        plan_wave_sync();
    }
    __syncthreads();
    // waves that have experts: their starts, and each wave's first place in them
    const bool has = wave * 64 < E;
    uint32_t all = 0, upto = 0;
    if (has) {
        if (t < E) {
            if (chunks == 1) {
#pragma unroll
                for (uint32_t w = 0; w < kPlanWaves; ++w) all += at[w * E + t];
            } else {
                all = all_of[t];
            }
        }
        upto = all;
        for (uint32_t off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(upto, off, 64);
            if (lane >= off) upto += y;
        }
        if (lane == 63) wave_sum[wave] = upto;
    }
    __syncthreads();
    if (has) {
        for (uint32_t w = 0; w < wave; ++w) upto += wave_sum[w];
        if (t < E) {
            const uint32_t start = upto - all;
            uint32_t next = start + before_of[t];
#pragma unroll
            for (uint32_t w = 0; w < kPlanWaves; ++w) {
                const uint32_t v = at[w * E + t];
                at[w * E + t] = next;
                next += v;
            }
            if (blockIdx.x == 0) a.starts[t] = start;
            if (t == E - 1) {
                listed = upto;
                if (blockIdx.x == 0) a.starts[E] = upto;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
        const uint32_t i = from + 64 * k + lane;
        const bool some = id[k] < E;
        uint32_t place = kNone;
        if (some) place = at[wave * E + id[k]] + (uint32_t)__popcll(same[k] & ((1ull << lane) - 1));
        plan_wave_sync();
        if (some && __builtin_ctzll(same[k]) == lane) at[wave * E + id[k]] += (uint32_t)__popcll(same[k]);
        plan_wave_sync();
        if (i < a.n) {
            a.slots[i] = place;
            if (some) a.rows[place] = i / a.topk;
            if (i >= listed) a.rows[i] = kNone;  // behind the lists
        }
    }
}

// A position's weighted sum over its experts' rows, four columns a thread, its
// routes in order; rows of no slot are passed over.  Bound by memory: 4000 positions of 6
// rows of 4096 in bf16 50.5 us, 4.7 TB/s.
template <bool kBf16>
__global__ void __launch_bounds__(256) k_expert_combine(wh_expert_combine_args a, uint32_t units) {
    const uint32_t p = blockIdx.x / units, col = ((blockIdx.x % units) * 256 + threadIdx.x) * 4;
    if (col >= a.hidden) return;
    wh_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k = 0; k < a.topk; ++k) {
        const uint32_t slot = a.slots[(uint64_t)p * a.topk + k];
        if (slot >= a.n_rows) continue;
        const float w = a.weights[(uint64_t)p * a.topk + k];
        wh_f4 v;
        if constexpr (kBf16) {
            const wh_u2 b = *(const wh_u2*)((const uint16_t*)a.y + slot * a.y_stride + col);
            v = wh_f4{__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                      __uint_as_float(b.y & 0xffff0000u)};
        } else {
            v = *(const wh_f4*)((const float*)a.y + slot * a.y_stride + col);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(v[j], w, acc[j]);
    }
    if (a.add) {
        const wh_f4 s = *(const wh_f4*)(a.add + p * a.add_stride + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += s[j];
    }
    *(wh_f4*)(a.out + p * a.out_stride + col) = acc;
}

// A grid has less than 2^32 threads.
constexpr uint64_t kMaxGrid256 = 0xffffffull;

}  // namespace

// ------------------------------------------------------------------- host

constexpr size_t plan_lds(uint32_t n_groups) { return kPlanWaves * (size_t)n_groups * sizeof(uint32_t); }

std::atomic<uint32_t> g_workgroups{256};  // a multiple of 8, one a CU: devices of one machine are alike

hipError_t wh_rows_setup() {
    int device = 0, cus = 0;
    if (hipGetDevice(&device) == hipSuccess &&
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) == hipSuccess && cus >= 8)
        g_workgroups = (uint32_t)cus / 8 * 8;
    hipError_t e = hipSuccess;
    auto tile = [&](const void* f, size_t lds) {
        if (e == hipSuccess) e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    };
    tile((const void*)k_expert_place<1, false>, plan_lds(WH_ROWS_MAX_GROUPS));
    tile((const void*)k_expert_place<2, false>, plan_lds(WH_ROWS_MAX_GROUPS));
    tile((const void*)k_expert_place<4, false>, plan_lds(WH_ROWS_MAX_GROUPS));
    tile((const void*)k_expert_place<4, true>, plan_lds(WH_ROWS_MAX_GROUPS));
    constexpr size_t lds = rows_tile_shape<4, 4, 2, 2>::kLds;
    tile((const void*)k_rows_mm_tile<true, true>, lds);
    tile((const void*)k_rows_mm_tile<true, false>, lds);
    tile((const void*)k_rows_mm_tile<false, true>, lds);
    tile((const void*)k_rows_mm_tile<false, false>, lds);
    constexpr size_t big = rows_tile_shape<8, 8, 2, 2>::kLds;
    tile((const void*)k_rows_mm_big<true>, big);
    tile((const void*)k_rows_mm_big<false>, big);
    return e;
}

hipError_t wh_rows_quant_launch(const wh_rows_quant_args& a, bool bf16, hipStream_t stream) {
    const uint64_t grid = ((uint64_t)a.n * a.blocks + 15) / 16;
    if (grid > kMaxGrid256) return hipErrorInvalidValue;
    if (a.up) {
        if (bf16) k_rows_quant<true, true><<<(unsigned)grid, 256, 0, stream>>>(a);
        else k_rows_quant<false, true><<<(unsigned)grid, 256, 0, stream>>>(a);
    } else {
        if (bf16) k_rows_quant<true, false><<<(unsigned)grid, 256, 0, stream>>>(a);
        else k_rows_quant<false, false><<<(unsigned)grid, 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

hipError_t wh_rows_read_launch(const wh_rows_read_args& a, bool bf16, hipStream_t stream) {
    const uint64_t grid = ((uint64_t)a.n * a.blocks + 15) / 16;
    if (grid > kMaxGrid256) return hipErrorInvalidValue;
    if (bf16) k_rows_read<true><<<(unsigned)grid, 256, 0, stream>>>(a);
    else k_rows_read<false><<<(unsigned)grid, 256, 0, stream>>>(a);
    return hipGetLastError();
}

// Which kernel takes a product, and how many ranges its columns are cut into: the least
// of these estimates of its time in us, fitted to 400 measured calls (one MI355X; 1 to
// 4096 rows, 1 to 64 groups, weights from 1408 x 512 to 32768 x 1024 and 4096 x 8192; call
// after call on the same weight, which the Infinity Cache holds up to 256 MB: from memory
// one of 4096 x 4096 takes 1 to 6 us more).
//  - thin: a wave's block of columns takes 0.8, 1.05 and 3 us for up to 16, 32 and 64
//    rows (with groups of uneven lists 0.55 and 0.045 a row), workgroups in rounds of 256:
//    4096 x 4096 with 16, 64 and 128 rows 7.2, 15.6 and 29, where tiles take 23 to 25, cut
//    up 13 to 18; 64 groups with 4, 16 and 32 rows each in f32 228, 343 and 505, tiles 281,
//    299 and 309;
//  - tile: a block 0.56 us in bf16 (0.95 with factors of scales), 1.1 in f32, in rounds of
//    256 workgroups; ranges divide that and add a launch and their parts' bytes: 4096 x
//    4096 with 128 rows in 1, 2 and 4 ranges 24.6, 19.9 and 18.1, with 1024 27, 34 and 48;
//  - half and tall tiles (bf16): 5 and 9 us, and 0.85 and 1.45 a block, by rounds that need
//    not be whole, since workgroups take tiles until there are none: 4096 x 4096 with
//    1024, 2048 and 4096 rows 28, 35 and 71 in half tiles, 44, 49 and 59 in tall ones, 27, 40
//    and 80 in tiles of 128.
wh_rows_mm_plan wh_rows_mm_plan_of(const wh_rows_mm_args& a, bool bf16) {
    const uint32_t blocks = a.cols / 128u;
    const bool mant = a.scale_f32 || a.odd_scale;
    wh_rows_mm_plan p{wh_rows_mm_plan::kAny, 1, blocks, 256, 0, 0, 0};
    const double groups = std::min(a.n_groups, a.n), rows = a.n / groups;
    // tiles, of groups that end in a tile half full on average
    auto tiles = [&](double m, uint32_t n) {
        return (a.n_groups == 1 ? std::ceil(a.n / m) : std::max(groups, a.n / m + groups / 2)) * ((a.out_rows + n - 1) / n);
    };
    auto most = [&](uint32_t m, uint32_t n) { return rows_tiles(a, m) * ((a.out_rows + n - 1) / n); };
    if (rows_mm_matrix(a)) {
        const uint32_t each = 16 * (kThinWaves / rows_thin_split(a));
        const double left = rows - 64 * std::floor(rows / 64);
        const double chunk = a.n_groups > 1 ? 0.55 + 0.045 * rows
                                            : 3.0 * std::floor(rows / 64) + (left == 0 ? 0 : left <= 16 ? 0.8 : left <= 32 ? 1.05 : 3.0);
        double best = 3.5 + std::max(1.0, groups * ((a.out_rows + each - 1) / each) / 256) *
                                std::ceil((double)blocks / rows_thin_split(a)) * chunk;
        p.kind = wh_rows_mm_plan::kThin;
        auto offer = [&](double us, wh_rows_mm_plan::kind_t kind, uint32_t splits, uint32_t per) {
            if (us >= best) return;
            best = us;
            p.kind = kind;
            p.splits = splits;
            p.per = per;
        };
        const double block = bf16 ? (mant ? 0.95 : 0.56) : 1.1, n_tiles = tiles(128, 128);
        for (uint32_t want = 1; want <= 16; want *= 2) {
            uint32_t per = blocks, splits = 1;
            if (want > 1) {  // ranges of a multiple of 4 blocks, whose scales lie in whole words
                per = (blocks + want * 4 - 1) / (want * 4) * 4;
                splits = (blocks + per - 1) / per;
                if (splits == 1) continue;
            }
            const double join = splits == 1 ? 0 : 3 + 8.0 * splits * a.n * a.out_rows / 6.5e6;
            offer(7 + std::max(1.0, n_tiles * splits / 256) * per * block + join, wh_rows_mm_plan::kTile, splits, per);
        }
        if (bf16 && !mant) {
            const double half = tiles(128, 256) / 256, tall = (tiles(256, 256) - (a.n_groups == 1 ? 0 : 0.2 * groups * ((a.out_rows + 255) / 256))) / 256;
            const double uneven = a.n_groups > 1 ? 1.15 : 1.0;
            offer(uneven * (5 + std::max(1.0, half > 1 ? half + 0.25 : half) * (5 + blocks * (0.5 + 0.35 * std::min(1.0, half)))),
                  wh_rows_mm_plan::kHalf, 1, blocks);
            offer(uneven * (4 + std::max(1.0, tall > 1 ? tall + 0.25 : tall) * (9 + blocks * (0.9 + 0.55 * std::min(1.0, tall)))),
                  wh_rows_mm_plan::kTall, 1, blocks);
        }
    }
    auto size = [&] {
        switch (p.kind) {
            case wh_rows_mm_plan::kAny: p.grid = std::min(p.tiles = most(kAnyRows, 16), kMaxGrid256); break;
            case wh_rows_mm_plan::kThin: {
                p.threads = 64 * kThinWaves;
                const uint32_t each = 16 * (kThinWaves / rows_thin_split(a)) * rows_thin_tiles(a, bf16);
                p.grid = p.tiles = (uint64_t)((a.out_rows + each - 1) / each) * a.n_groups;
                break;
            }
            case wh_rows_mm_plan::kTile: p.grid = ((p.tiles = most(128, 128)) + 7) / 8 * 8; break;
            case wh_rows_mm_plan::kHalf: p.grid = std::min<uint64_t>(((p.tiles = most(128, 256)) + 7) / 8 * 8, g_workgroups.load()); break;
            case wh_rows_mm_plan::kTall: p.grid = std::min<uint64_t>(((p.tiles = most(256, 256)) + 7) / 8 * 8, g_workgroups.load()); break;
        }
    };
    size();
    if (p.grid * p.threads * p.splits > 0xffffffffull) {  // a grid's threads: the vector kernel takes any number of tiles
        p.kind = wh_rows_mm_plan::kAny;
        p.splits = 1;
        p.per = blocks;
        p.threads = 256;
        size();
    }
    if (p.splits > 1) p.part_bytes = (size_t)p.splits * a.n * rows_part_stride(a) * sizeof(float);
    return p;
}

hipError_t wh_rows_mm_launch(const wh_rows_mm_args& a, const wh_rows_mm_plan& p, bool bf16, hipStream_t stream) {
    const bool mant = a.scale_f32 || a.odd_scale;
    const uint32_t grid = (uint32_t)p.grid;
    constexpr size_t small = rows_tile_shape<4, 4, 2, 2>::kLds, big = rows_tile_shape<8, 8, 2, 2>::kLds;
    auto go = [&](size_t lds, auto kern) { kern<<<grid, p.threads, lds, stream>>>(a); };
    switch (p.kind) {
        case wh_rows_mm_plan::kAny:
            if (bf16) go(0, k_rows_mm_any<true>);
            else go(0, k_rows_mm_any<false>);
            break;
        case wh_rows_mm_plan::kThin: {
            const uint32_t ks = rows_thin_split(a);
            auto thin = [&](auto kern) { kern<<<dim3(grid / a.n_groups, a.n_groups), p.threads, 0, stream>>>(a, ks); };
            auto of = [&](auto nt) {
                constexpr int kNt = decltype(nt)::value;
                if (bf16) {
                    if (mant) thin(k_rows_mm_thin<true, true, kNt>);
                    else thin(k_rows_mm_thin<true, false, kNt>);
                } else {
                    if (mant) thin(k_rows_mm_thin<false, true, kNt>);
                    else thin(k_rows_mm_thin<false, false, kNt>);
                }
            };
            if (rows_thin_tiles(a, bf16) > 1) of(std::integral_constant<int, 2>{});
            else of(std::integral_constant<int, 1>{});
            break;
        }
        case wh_rows_mm_plan::kTile: {
            auto tile = [&](auto kern) { kern<<<dim3(grid, p.splits), p.threads, small, stream>>>(a, p.per); };
            if (bf16) {
                if (mant) tile(k_rows_mm_tile<true, true>);
                else tile(k_rows_mm_tile<true, false>);
            } else {
                if (mant) tile(k_rows_mm_tile<false, true>);
                else tile(k_rows_mm_tile<false, false>);
            }
            if (p.splits > 1) {
                const hipError_t e = hipGetLastError();
                if (e != hipSuccess) return e;
                const uint32_t join = (uint32_t)(((uint64_t)a.n * (rows_part_stride(a) / 4) + 255) / 256);
                if (bf16) k_rows_join<true><<<join, 256, 0, stream>>>(a, p.splits);
                else k_rows_join<false><<<join, 256, 0, stream>>>(a, p.splits);
            }
            break;
        }
        case wh_rows_mm_plan::kHalf: go(big, k_rows_mm_big<false>); break;
        case wh_rows_mm_plan::kTall: go(big, k_rows_mm_big<true>); break;
    }
    return hipGetLastError();
}

hipError_t wh_rows_store_launch(const uint8_t* weight, uint8_t* out, uint64_t rows, uint32_t cols, uint32_t* flags,
                                hipStream_t stream) {
    // pieces of rows whose grids are within a launch's limits
    const uint64_t per = std::max<uint64_t>(1, (kMaxGrid256 * 16) / (cols / 128u));
    for (uint64_t r = 0; r < rows; r += per) {
        const uint64_t blocks = std::min(per, rows - r) * (cols / 128u);
        k_rows_store<<<(unsigned)((blocks + 15) / 16), 256, 0, stream>>>(weight + r * cols, out + r * cols, blocks, flags);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t wh_rows_scales_launch(const uint8_t* scales, uint64_t n, uint32_t* flags, hipStream_t stream) {
    const uint64_t per = kMaxGrid256 * 256;
    for (uint64_t i = 0; i < n; i += per) {
        const uint64_t m = std::min(per, n - i);
        k_rows_scales<<<(unsigned)((m + 255) / 256), 256, 0, stream>>>(scales + i, m, flags);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// How many times 64 routes a wave takes: as few as make one launch of up to 4096 routes (96
// once 3.7 us, four times 5.5; 1800 twice 4.7, in two launches 6.4), then once (12000 routes
// over 256 experts 6.8 us, four times 9.8) until every workgroup would sum the counts of
// too many chunks: over 256 experts 98304 routes once 9.0 us, twice 9.2, four times 11.0;
// 262144 13.1, 11.4 and 12.4; 1048576 53, 24 and 20.
static uint32_t plan_turns(size_t n, size_t n_groups) {
    if (n <= plan_chunk(4)) return n <= plan_chunk(1) ? 1 : n <= plan_chunk(2) ? 2 : 4;
    const size_t counts = n * std::max<size_t>(n_groups, 256);  // a wave sums at least 256 a chunk
    return counts <= 1u << 25 ? 1 : counts <= 1u << 27 ? 2 : 4;
}

// From how many chunks on a launch of its own adds their counts up, which every workgroup
// does for itself below: that grows with the square of the routes.  1048576 routes (256
// chunks) over 8, 256 and 1024 experts 12.8, 18.8 and 23.4 us, without it 14.3, 20.1 and
// 39.4; 67108864 353, 584 and 843 us, without it 7.7, 11.4 and 44 ms.
constexpr uint32_t kPlanSummed = 256;

size_t wh_expert_plan_scratch(size_t n, size_t n_groups) {
    const size_t chunk = plan_chunk(plan_turns(n, n_groups)), chunks = (n + chunk - 1) / chunk;
    return chunks > 1 ? (chunks + 1) * plan_padded((uint32_t)n_groups) * sizeof(uint32_t) : 0;
}

hipError_t wh_expert_plan_launch(const wh_expert_plan_args& a, hipStream_t stream) {
    const uint32_t turns = plan_turns(a.n, a.n_groups), chunk = plan_chunk(turns), chunks = std::max(1u, (a.n + chunk - 1) / chunk);
    uint32_t bits = 1;
    while ((a.n_groups >> bits) != 0) ++bits;
    if (chunks > 1) {
        k_expert_count<<<chunks, kPlanThreads, 0, stream>>>(a, chunk);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const size_t lds = plan_lds(a.n_groups);
    if (turns == 4 && chunks >= kPlanSummed) {
        k_expert_sum<<<(plan_padded(a.n_groups) + kSumExperts - 1) / kSumExperts, kSumExperts * kSumRuns, 0, stream>>>(a, chunks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        k_expert_place<4, true><<<chunks, kPlanThreads, lds, stream>>>(a, chunks, bits);
    } else if (turns == 4) {
        k_expert_place<4, false><<<chunks, kPlanThreads, lds, stream>>>(a, chunks, bits);
    } else if (turns == 2) {
        k_expert_place<2, false><<<chunks, kPlanThreads, lds, stream>>>(a, chunks, bits);
    } else {
        k_expert_place<1, false><<<chunks, kPlanThreads, lds, stream>>>(a, chunks, bits);
    }
    return hipGetLastError();
}

hipError_t wh_expert_combine_launch(const wh_expert_combine_args& a, bool bf16, hipStream_t stream) {
    const uint32_t units = (a.hidden / 4 + 255) / 256;
    const uint64_t grid = (uint64_t)a.npos * units;
    if (grid > kMaxGrid256) return hipErrorInvalidValue;
    if (bf16) k_expert_combine<true><<<(unsigned)grid, 256, 0, stream>>>(a, units);
    else k_expert_combine<false><<<(unsigned)grid, 256, 0, stream>>>(a, units);
    return hipGetLastError();
}
