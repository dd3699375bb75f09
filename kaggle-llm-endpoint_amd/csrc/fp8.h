// Block-scaled fp8 on gfx950: the e4m3 row quantiser and the argument block that the fp8 products share.
//
// A row of activations is held as e4m3 values with one f32 scale per group of 128 columns, a weight matrix as e4m3
// values with one f32 scale per 128 x 128 block (the layout of fp8 checkpoints, checkpoint.py:202).  A product is
//   y[b, o] = sum_c xs[b, c] * ws[o / 128, c] * sum_{i in group c} xq[b, i] * wq[o, i]
// and a group is exactly one 16x16x128 matrix instruction: the inner sum is one instruction's f32 result, which is
// then scaled and added in f32.
#pragma once
#include "common.h"

namespace mi {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Group = 128;                   // columns per scale; rows and columns per weight scale
constexpr int kFp8MaxGroups = 512;               // K / 128: the weight scales of a tile's blocks are kept in LDS
constexpr int kFp8MinExp = -100;                 // least scale of a row's group: 2^-100
constexpr uint32_t kFp8Out = 0x80000000u;        // a buffer offset past every range: reads zero
constexpr int kFp8Word3 = 0x00020000;            // gfx9 buffer descriptor word 3 (32-bit data format)

__host__ __device__ inline int fp8_groups(int n) { return (n + kFp8Group - 1) / kFp8Group; }

// Exponent e of a group's scale 2^e from the bits of a = max |x|: the least e with a <= 448 * 2^e.  448 = 1.75 * 2^8, so
// e = exponent(a) - 8, one more if a's mantissa is past 1.75 (the carry of the addition).  A power of two, so that
// x / s is exact and each value is rounded once; a float format loses nothing by it but the range below its smallest
// normal value, and an f32 rounding in the last bit of a never moves the values.
__device__ __forceinline__ int fp8_exponent(uint32_t abits) {
    return max((int)((abits + 0x1fffffu) >> 23) - 135, kFp8MinExp);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A group's sum is scaled by xs * ws.  xs is 2^-100 to 2^120, ws any f32, and as it stands their product may leave f32 where
// the scaled sum does not: 2^120 times 2^8 is infinite, times a sum of 0 NaN.  So a row of weight blocks is computed with
// its scales times 2^-n and its sums are multiplied by 2^n in the end, n by the largest of them: 0 from 2^-26 to below
// 2^7, where xs * ws is a normal f32 (a checkpoint's scales are there, and keep their products and bits), otherwise what
// brings the largest there.  Next to that one, a scale below 2^-26 of its size may still meet an xs with which the product
// is subnormal: an error of at most 2^(n - 125) in its group's term.  (With an infinite scale the row has no finite output.)
__device__ __forceinline__ int fp8_scale_shift(float largest) {
    const int e = __builtin_amdgcn_frexp_expf(largest) - 1;          // 2^e <= largest < 2^(e + 1)
    return !(largest > 0.0f && largest < INFINITY) ? 0 : e > 6 ? e - 6 : e < -26 ? e + 26 : 0;
}
// n of a wavefront's scales, m the largest magnitude among a lane's.
__device__ __forceinline__ int fp8_wave_shift(float m) {
    if (__ballot(m >= 0x1p7f) == 0 && __ballot(m >= 0x1p-26f) != 0) return 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    return __builtin_amdgcn_readfirstlane(fp8_scale_shift(m));
}

// Two values to e4m3 (nearest even), in the low or high half of `old`; |a|, |b| <= 448 or NaN.
template <bool HI>
__device__ __forceinline__ int fp8_pack2(float a, float b, int old) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, HI);
}
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    return (uint32_t)fp8_pack2<true>(c, d, fp8_pack2<false>(a, b, 0));
}

__device__ __forceinline__ bool f32_bits_finite(uint32_t u) { return (u & 0x7fffffffu) < 0x7f800000u; }

// Infinities become NaN (e4m3 has no infinity; past 448 the conversion would otherwise be free to saturate).
__device__ __forceinline__ float fp8_inf_to_nan(float v) {
    return f32_bits_finite(__float_as_uint(v)) ? v : __uint_as_float(0x7fc00000u);
}

// silu(min(g, L)) * clip(u, -L, L) with comparisons that keep a NaN (fminf and fmaxf would return the limit).
__device__ __forceinline__ float fp8_swiglu(float g, float u, float limit) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
    return silu_f32(g) * u;
}

// The fp8 product of one 16 x 16 x 128 tile: a = 32 bytes of weight row (lane & 15), b = 32 bytes of token (lane & 15),
// both for the columns that lane >> 4 holds; the result's lane (i, q) has rows 4 q .. 4 q + 3 of token i.  (All-zero scale
// operands select the unscaled instruction.)
//
// Its arithmetic, measured: the 8 products of 8 consecutive bytes are added on a grid of 2^-13 of the largest one's power
// of two, what is below is cut; those sums are added in f32.  On normal values that is 1.3e-5 of the result (root mean
// square), the same for the 16x16x32 fp8 instruction: a hundredth of a bf16 rounding of the result.
__device__ __forceinline__ f32x4 fp8_mfma(i32x8 a, i32x8 b) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);
}

// The same product with every sum in f32: both operands converted to bf16, which holds e4m3 exactly, and four
// 16x16x32 bf16 instructions, at half the rate and with 16 conversions an operand.  Taken for gate and up where memory
// bounds the launch: their results are quantised again, and of a value next to a rounding border the last bits decide a
// whole step of e4m3.  (One token through MLPs of 1360 / 592: 0.0023 of the result with the fp8 instruction on average,
// 0.0081 at worst, against the definition; 0.0017, a bf16 rounding, with this.)
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8_t fp8_to_bf16(int lo, int hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return (bf16x8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <bool EXACT>
__device__ __forceinline__ f32x4 fp8_product(i32x8 a, i32x8 b) {
    if constexpr (!EXACT) {
        return fp8_mfma(a, b);
    } else {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; k += 2)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_to_bf16(a[k], a[k + 1]), fp8_to_bf16(b[k], b[k + 1]), c, 0, 0, 0);
        return c;
    }
}

// One product's operands.  Rows r of the activations: row r of xq, or row tok_row[r] (-1: a row of zeros).  With
// blk_expert, block r / tm uses expert blk_expert[r / tm] of E, and blocks >= *n_blocks have no product.
struct Fp8Gemm {
    const uint8_t *xq;          // e4m3 [x_rows, K]
    const float *xs;            // f32 [x_rows, K / 128]
    const uint8_t *wq[2];       // e4m3 [E, R, K]
    const float *ws[2];         // f32 [E, R / 128, K / 128]
    const int32_t *tok_row;     // [rows] or NULL
    const int32_t *live;        // [rows] or NULL: < 0 marks rows without a token, the last ones of their block
    const int32_t *blk_expert;  // [rows / tm] or NULL
    const int32_t *n_blocks;    // [1] (with blk_expert)
    int x_rows;                 // rows of xq (bounds tok_row)
    int rows, tm;
    int E, R, K;
    uint16_t *y_bf16;           // [rows, R], either may be NULL
    float *y_f32;
};

}  // namespace mi
