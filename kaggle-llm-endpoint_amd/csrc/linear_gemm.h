// bf16 products on gfx950 with an epilogue, and the two products of their gradients:
//   C[t, o] = sum_k a[o, k] b[t, k],   y = act(C + bias) + residual
// in f32, rounded once.  Forward a is the weight [n_out, n_in] and b the rows [B, n_in]; the gradients take an operand whose
// contraction index is the slow one ([k, o] in memory) as it lies: its fragments are read from LDS transposed.
#pragma once
#include <type_traits>

#include "common.h"

namespace mi {

typedef __bf16 lin_bf16x8 __attribute__((ext_vector_type(8)));
typedef short lin_s16x4 __attribute__((ext_vector_type(4)));
typedef short lin_s16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kLinOut = 0x80000000u;        // a buffer offset past every range: reads zero
constexpr int kLinWord3 = 0x00020000;            // gfx9 buffer descriptor word 3 (32-bit data format)
constexpr int kLinCols = 64;                     // contraction columns per stage
constexpr int kLinNear = 8;                      // token tiles of a weight tile that run next to each other

struct LinGemm {
    const uint16_t *a, *b;      // [R, K] and [rows, K], or (slow) [K, R] and [K, rows]
    long long lda, ldb;         // row strides in memory, multiples of 8
    int R, rows;
    int K;                      // contraction length (fast operands: a multiple of 8)
    int Ks;                     // of slow operands: rows from Ks on count as zero
    // ---- epilogue
    const uint16_t *bias;       // bf16 [R] or NULL
    int act;                    // MI_ACT_*
    const void *res;            // [rows, R] of y's type, or NULL
    int f32;                    // y and res are f32, else bf16
    void *y;                    // [rows, R]
    float *z;                   // C + bias [rows, ldz], ldz a multiple of 8 that holds R, or NULL
    long long ldz;
    // ---- tiled launches
    int nw, nb, S;              // weight tiles, token tiles, splits of K
    float *part;                // S > 1: f32 [S, rows, lin_part_ld(R)]
};

// Columns of a row of split sums: whole groups of four.
__host__ __device__ constexpr int lin_part_ld(int R) { return (R + 3) & ~3; }

// ------------------------------------------------------------------------------------------------ activations
// e^x and 1 / x by the plain instructions: 1 ulp each, besides |x| 2^-24 for the rounding of x log2(e).
__device__ __forceinline__ float lin_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float lin_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + lin_exp(-z)); }
__device__ __forceinline__ float gelu_inner2(float z) {                  // 2 sqrt(2 / pi) (z + 0.044715 z^3)
    return 1.5957691216057308f * fmaf(0.044715f * z * z, z, z);
}
// The normal distribution's Phi(z), and e = e^(-z^2 / 2): Phi(-x) = (c1 t + .. + c8 t^8) e^(-x^2 / 2) for x >= 0 with
// t = 1 / (1 + 0.305 x), which runs from 1 to 0.  The c are fitted (least largest relative error) to e^(x^2 / 2) Phi(-x) for x
// up to 14, past which e is 0: off by 9.4e-8 of it, 4.3e-7 with f32 steps.  So the tail is right relative to itself, besides
// 1.25 z^2 2^-24 from the rounding of e's argument (2e-6 at z = -5, where a fit of erf to 1e-7 is off by 2e-3).  In a product of
// 2048 x 6144 x 6144 the activation takes 2 us; erff, of three times the instructions, took 17.
__device__ __forceinline__ float normal_cdf(float z, float &e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.305f, fabsf(z), 1.0f));
    float a = fmaf(0.0366991997f, t, -0.15298835f);
    a = fmaf(a, t, 0.185716964f);
    a = fmaf(a, t, -0.037976883f);
    a = fmaf(a, t, 0.121021707f);
    a = fmaf(a, t, 0.103420858f);
    a = fmaf(a, t, 0.122466818f);
    a = fmaf(a, t, 0.121639733f) * t;
    e = __builtin_amdgcn_exp2f(z * z * -0.7213475204444817f);            // log2(e) / 2
    const float tail = a * e;
    return z < 0.0f ? tail : 1.0f - tail;
}
template <int ACT>
__device__ __forceinline__ float lin_act(float z) {
    if constexpr (ACT == MI_ACT_SILU) return z * lin_sigmoid(z);
    if constexpr (ACT == MI_ACT_GELU) {
        float e;
        return z * normal_cdf(z, e);
    }
    if constexpr (ACT == MI_ACT_GELU_TANH) return z * lin_sigmoid(gelu_inner2(z));   // (1 + tanh(u)) / 2 = sigmoid(2 u)
    if constexpr (ACT == MI_ACT_RELU) return z < 0.0f ? 0.0f : z;        // (a NaN stays)
    return z;
}
// The derivative; far out it is 0 or 1 to f32, and the factors below may be no numbers.
__device__ __forceinline__ float lin_act_grad(float z, int act) {
    const float far = z > 0.0f ? 1.0f : 0.0f;
    switch (act) {
        case MI_ACT_SILU: {
            const float s = lin_sigmoid(z);
            return fabsf(z) > 120.0f ? far : s * fmaf(z, lin_sigmoid(-z), 1.0f);
        }
        case MI_ACT_GELU: {
            float e;
            const float c = normal_cdf(z, e);
            return fabsf(z) > 30.0f ? far : fmaf(z * 0.3989422804014327f, e, c);
        }
        case MI_ACT_GELU_TANH: {
            const float s = lin_sigmoid(gelu_inner2(z)), r = lin_sigmoid(-gelu_inner2(z));
            return fabsf(z) > 30.0f ? far : s + z * s * r * 1.5957691216057308f * fmaf(0.134145f * z, z, 1.0f);
        }
        case MI_ACT_RELU: return z != z ? z : far;
        default: return 1.0f;
    }
}
// f(act) with the activation as a constant.
template <class F>
__device__ __forceinline__ void lin_with_act(int act, F f) {
    using std::integral_constant;
    switch (act) {
        case MI_ACT_SILU: return f(integral_constant<int, MI_ACT_SILU>{});
        case MI_ACT_GELU: return f(integral_constant<int, MI_ACT_GELU>{});
        case MI_ACT_GELU_TANH: return f(integral_constant<int, MI_ACT_GELU_TANH>{});
        case MI_ACT_RELU: return f(integral_constant<int, MI_ACT_RELU>{});
        default: return f(integral_constant<int, MI_ACT_NONE>{});
    }
}

// ------------------------------------------------------------------------------------------------ epilogue
__device__ __forceinline__ f32x4 lin_bf16x4(uint2 u) {
    return (f32x4){__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                   __uint_as_float(u.y & 0xffff0000u)};
}
// To nearest even, by the conversion instruction (two values each).
__device__ __forceinline__ uint2 lin_pack4(f32x4 v) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint2, __builtin_convertvector(v, bf16x4));
}

// Whether four consecutive outputs are one access each of y, the residual and the bias.
__device__ __forceinline__ bool lin_quads(const LinGemm &p) {
    const int m = p.f32 ? 15 : 7;
    return (p.R & 3) == 0 && (((uintptr_t)p.y | (uintptr_t)p.res) & m) == 0 && ((uintptr_t)p.bias & 7) == 0;
}

// Outputs o[r] .. o[r] + 3 (multiples of 4) of N places of one row from their sums: whole accesses.  Places past R are
// computed from the row's last ones and not stored, so that no branch surrounds a load.
template <int ACT, int N>
__device__ __forceinline__ void lin_out_quads(const LinGemm &p, int row, const int (&o)[N], const uint2 (&bias)[N],
                                              f32x4 (&v)[N]) {
    const bool in = row < p.rows;
    const size_t at = (size_t)min(row, p.rows - 1) * p.R;
    f32x4 res[N];
    if (p.res) {
        if (p.f32) {
#pragma unroll
            for (int r = 0; r < N; ++r) res[r] = *(const f32x4 *)((const float *)p.res + at + min(o[r], p.R - 4));
        } else {
            uint2 u[N];
#pragma unroll
            for (int r = 0; r < N; ++r) u[r] = *(const uint2 *)((const uint16_t *)p.res + at + min(o[r], p.R - 4));
#pragma unroll
            for (int r = 0; r < N; ++r) res[r] = lin_bf16x4(u[r]);
        }
    }
    if (p.bias) {
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] += lin_bf16x4(bias[r]);
    }
    if (p.z) {
#pragma unroll
        for (int r = 0; r < N; ++r)
            if (in && o[r] < p.R) *(f32x4 *)(p.z + (size_t)row * p.ldz + o[r]) = v[r];
    }
#pragma unroll
    for (int r = 0; r < N; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[r][j] = lin_act<ACT>(v[r][j]);
    if (p.res) {
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] += res[r];
    }
#pragma unroll
    for (int r = 0; r < N; ++r) {
        if (!in || o[r] >= p.R) continue;
        if (p.f32) *(f32x4 *)((float *)p.y + at + o[r]) = v[r];
        else *(uint2 *)((uint16_t *)p.y + at + o[r]) = lin_pack4(v[r]);
    }
}

// The same for four outputs of a row, value by value, before and after the activation.
__device__ __forceinline__ void lin_single_before(const LinGemm &p, int row, int o, f32x4 &v) {
    if (row >= p.rows) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (o + j >= p.R) continue;
        if (p.bias) v[j] += bf16_to_f32(p.bias[o + j]);
        if (p.z) p.z[(size_t)row * p.ldz + o + j] = v[j];
    }
}
__device__ __forceinline__ void lin_single_after(const LinGemm &p, int row, int o, f32x4 v) {
    if (row >= p.rows) return;
    const size_t at = (size_t)row * p.R + o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (o + j >= p.R) continue;
        if (p.f32) {
            if (p.res) v[j] += ((const float *)p.res)[at + j];
            ((float *)p.y)[at + j] = v[j];
        } else {
            if (p.res) v[j] += bf16_to_f32(((const uint16_t *)p.res)[at + j]);
            ((uint16_t *)p.y)[at + j] = (uint16_t)f32_to_bf16_rne(v[j]);
        }
    }
}

// Outputs o .. o + 3 of one row.
__device__ __forceinline__ void lin_out(const LinGemm &p, int row, int o, f32x4 v) {
    if (o >= p.R) return;
    if (lin_quads(p)) {
        lin_with_act(p.act, [&](auto act) __attribute__((always_inline)) {
            const int at[1] = {o};
            const uint2 bias[1] = {p.bias ? *(const uint2 *)(p.bias + o) : make_uint2(0, 0)};
            f32x4 w[1] = {v};
            lin_out_quads<decltype(act)::value, 1>(p, row, at, bias, w);
        });
        return;
    }
    lin_single_before(p, row, o, v);
    lin_with_act(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lin_act<decltype(act)::value>(v[j]);
    });
    lin_single_after(p, row, o, v);
}

// ------------------------------------------------------------------------------------------------ tiled product
__device__ __forceinline__ void lin_lds_load(__amdgpu_buffer_rsrc_t r, uint4 *dst, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 16, (int)voff, 0, 0, 0);
}

// One word of a line into a place in LDS that nobody reads: the line comes into L2.
template <int AT>
__device__ __forceinline__ void lin_lds_touch(__amdgpu_buffer_rsrc_t r, uint4 *dst, int voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 4, voff, AT, 0, 0);
}

// A slow operand's row k of a stage: the 32-byte piece u (16 columns) sits at u ^ lin_swizzle(k), so that the 16 pieces of
// one column tile that a transposed read takes (rows 8 q + 0 .. 3 of each q, or + 4 .. 7) lie on different banks.
__host__ __device__ constexpr int lin_swizzle(int k) { return (k & 3) | ((k >> 1) & 12); }

// One operand's share of a stage: T rows (fast) or columns (slow) of it, 64 deep; its loads and its fragments.
// Fast: LDS row r is 128 bytes, 16-byte chunk c of it at c ^ (r & 7).  Slow: LDS row k is T columns.
template <int T, int W, bool SLOW>
struct LinOperand {
    static constexpr int N = T / 8 / W;          // 1 KB loads of a wavefront and stage
    static_assert(T % (8 * W) == 0 && (!SLOW || (T & (T - 1)) == 0), "");
    const char *base;           // of the tile, stage 0
    long long advance;          // bytes from stage to stage
    uint32_t voff[N];
    int kat;                    // first contraction index of load 0 within the stage
    int frag;                   // byte of this lane's part of fragment 0
    uint32_t touch_at;          // the line that this lane reads ahead

    __device__ __forceinline__ void init(const uint16_t *m, long long ld, int first, int count, int wave, int lane,
                                         int tile0) {
        const int i = lane & 15, q = lane >> 4;
        if constexpr (SLOW) {
            constexpr int C = T / 8;             // 16-byte chunks of a row
            base = (const char *)(m + first);
            advance = 2 * kLinCols * ld;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int at = 64 * (j * W + wave) + lane, k = at / C, pos = at % C;
                const int chunk = (((pos >> 1) ^ (lin_swizzle(k) & (C / 2 - 1))) << 1) | (pos & 1);
                if (j == 0) kat = k;
                voff[j] = first + 8 * chunk < ((count + 7) & ~7) ? (uint32_t)(2 * (k * ld + 8 * chunk)) : kLinOut;
            }
            const int k = 8 * q + (i >> 2);
            frag = (k * T * 2 + (i & 3) * 8) ^ (((lin_swizzle(k) & (C / 2 - 1)) ^ (tile0 / 16)) * 32);
        } else {
            base = (const char *)(m + (size_t)first * ld);
            advance = 2 * kLinCols;
            kat = 8 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int r = 8 * (j * W + wave) + (lane >> 3);
                voff[j] = (uint32_t)(2 * (min(r, count - 1 - first) * ld + kat));
            }
            frag = (tile0 + i) * 128 + (q ^ (i & 7)) * 16;
        }
    }
    // load j of stage g into the operand's part of a buffer; k: the first contraction index past the operand
    __device__ __forceinline__ void load(uint4 *lds, int g, int k, int wave, int j) const {
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc((void *)(base + g * advance), (short)0, 0x7fffffff, kLinWord3);
        lin_lds_load(r, lds + 64 * (j * W + wave), voff[j] | (g * kLinCols + kat + (SLOW ? j * (512 * W / T) : 0) >= k ? kLinOut : 0u));
    }
    // Reading ahead (of a fast operand): this lane takes row n's line of a stage, 128 bytes, if n is below T.
    __device__ __forceinline__ void touch_init(long long ld, int first, int count, int n) {
        static_assert(!SLOW, "");
        touch_at = n < T && first + n < count ? (uint32_t)(2 * n * ld) : kLinOut;
    }
    // both halves of the line, as far as the row reaches (k: the first column behind it)
    __device__ __forceinline__ void touch(uint4 *lds, int g, int k) const {
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc((void *)(base + g * advance), (short)0, 0x7fffffff, kLinWord3);
        lin_lds_touch<0>(r, lds, (int)(touch_at | (g * kLinCols >= k ? kLinOut : 0u)));
        lin_lds_touch<64>(r, lds, (int)(touch_at | (g * kLinCols + kLinCols / 2 >= k ? kLinOut : 0u)));
    }
    // fragment of the 16 rows (columns) tile0 + 16 r, contraction indexes 32 half + 8 q .. + 7
    __device__ __forceinline__ lin_bf16x8 read(const uint4 *lds, int r, int half) const {
        if constexpr (SLOW) {
            typedef __attribute__((address_space(3))) lin_s16x4 piece;
            piece *p = (piece *)((__attribute__((address_space(3))) const char *)lds + (frag ^ (32 * r)) + half * 64 * T);
            const lin_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
            const lin_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p + T);
            return __builtin_bit_cast(lin_bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return __builtin_bit_cast(lin_bf16x8, lds[((frag ^ (64 * half)) >> 4) + 128 * r]);
        }
    }
};

// A workgroup computes TW weight rows x TT rows, its wavefronts WM x WN of them, 64 columns a stage, NST stages in LDS.
//
// What bounds it: of 8 wavefronts of 128 x 64 outputs a stage takes 1.27 us of which the matrix instructions are 0.85 (at 2.4
// GHz); 24 KB of fragments a wavefront keep LDS about as busy as they keep the matrix cores, then memory under load, tiles
// that do not fill the last round, and the ends (7 to 9 stages' time).  8192^3 in 790 us (1.39 PFLOP/s), its gradients' products in
// 810 and 800; a library's product, without an epilogue, takes 740, 820 and 940.  4096 x 6144 x 6144 260, 265, 285 (290, 325, 350).
//
// The tiles of 192 x 256 and 256 x 256 hold 96 and 128 sums a lane and spill: 207, and 480 / 152 / 121 (forward, dx, dW) registers,
// almost all of them in the epilogue, which has every activation, whole accesses and the value-by-value form in one kernel; the
// loop has one reload, of the dW form.
//
// Measured and not kept: 4 wavefronts of 128 x 128 (the accumulators and two sets of fragments do not fit), 2 x 2 wavefronts for
// 256 x 128 (20 % slower), 128 x 128 with 2 stages and 2 workgroups a CU (10 to 40 % slower than with 4 stages and one), or
// with 4 wavefronts instead of 8 (517 x 6144 x 6144 57 us instead of 50).
template <int TW, int TT, int WM, int WN, int NST, bool SLOWA, bool SLOWB>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) lin_gemm_kernel(LinGemm p) {
    constexpr int W = WM * WN, RT = TW / WM / 16, CT = TT / WN / 16, ROWS = TW + TT;
    constexpr bool AHEAD = TW == 192;
    constexpr int TOUCHES = AHEAD ? 2 : 0;       // loads of a stage that read ahead
    __shared__ uint4 buf0[ROWS * 8], buf1[ROWS * 8], buf2[NST > 2 ? ROWS * 8 : 1], buf3[NST > 3 ? ROWS * 8 : 1];
    __shared__ uint4 sink[AHEAD ? 16 * W : 1];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // An XCD's workgroups (ids equal modulo 8) take one contiguous piece of the work: kLinNear token tiles of a weight tile,
    // then of the next, so that its CUs meet each other's loads in its L2.
    const long long total = (long long)p.nb * p.nw * p.S;
    const int xcd = blockIdx.x & 7;
    const long long at = total * xcd / 8 + (blockIdx.x >> 3);
    if (at >= total * (xcd + 1) / 8) return;     // the whole workgroup
    const long long per = (long long)kLinNear * p.nw * p.S;
    const int pr = (int)(at / per), in = (int)(at - pr * per);
    const int width = min(kLinNear, p.nb - kLinNear * pr);
    const int tb = kLinNear * pr + in % width, ws = in / width, wt = ws % p.nw, split = ws / p.nw;
    const int row0 = tb * TT, o0 = wt * TW;
    const int steps = (p.K + kLinCols - 1) / kLinCols;
    const int t0 = (int)((long long)split * steps / p.S), t1 = (int)((long long)(split + 1) * steps / p.S);

    LinOperand<TW, W, SLOWA> A;
    LinOperand<TT, W, SLOWB> B;
    A.init(p.a, p.lda, o0, p.R, wave, lane, wm * (TW / WM));
    B.init(p.b, p.ldb, row0, p.rows, wave, lane, wn * (TT / WN));
    constexpr int PER = A.N + B.N;
    const int kend = t1 * kLinCols, ka = min(SLOWA ? p.Ks : p.K, kend), kb = min(SLOWB ? p.Ks : p.K, kend);
    // The columns are summed in a cycle that starts at another place for every XCD: with all of them at the same columns of
    // rows 12 KB apart, memory answers more slowly (4096 x 6144 x 6144, tiles of 256 x 256: 325 us from the first column on,
    // 299 so).
    const int start = xcd * 3 % 8 * (t1 - t0) / 8;
    auto stage_at = [&](int g) __attribute__((always_inline)) { return g + start - (g + start >= t1 ? t1 - t0 : 0); };
    auto load_piece = [&](uint4 *buf, int g, int j) __attribute__((always_inline)) {
        if (j < A.N) A.load(buf, stage_at(g), g < t1 ? ka : 0, wave, j);
        else B.load(buf + 8 * TW, stage_at(g), g < t1 ? kb : 0, wave, j - A.N);
    };
    // A stage's loads have a step to come back, less than memory takes.  So 3 stages ahead of its use a stage's lines are
    // brought into L2, each by one of the workgroups that share them, both 64-byte halves (one word of a line brings half of it).
    // 253 us instead of 295 of 4096 x 6144 x 6144 in these tiles (where 256 x 128 without it take 258, and are chosen), 135 instead
    // of 150 of 2048.  Tiles of 256 x 256 have no registers for it.
    if constexpr (AHEAD) {
        const int line = wave * 64 + lane;
        const bool mine = ((line ^ (int)(blockIdx.x >> 3)) & (kLinNear - 1)) == 0;
        A.touch_init(p.lda, o0, p.R, mine && line < TW ? line : TW);
        B.touch_init(p.ldb, row0, p.rows, mine && line >= TW ? line - TW : TT);
    }
    auto touch = [&](int g) __attribute__((always_inline)) {
        if constexpr (AHEAD) {
            uint4 *const to = sink + 16 * wave;
            if (wave * 64 < TW) {
                A.touch(to, stage_at(g), g < t1 ? ka : 0);
            } else {
                B.touch(to, stage_at(g), g < t1 ? kb : 0);
            }
        }
    };

    f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // A stage is two halves of 32 columns.  While one half's fragments are multiplied the next one's are read; the only
    // barrier of a stage is where its last fragment has been read: then the next stage must have landed, and this one's
    // buffer may be filled again.  The order below is the order of the instructions.
    lin_bf16x8 fa[2][RT], fb[2][CT];
    constexpr int READS = RT + CT, BAR = RT > 4 ? RT - 2 : RT - 1;
    auto read = [&](const uint4 *buf, int half, int n) __attribute__((always_inline)) {
        if (n < CT) fb[half][n] = B.read(buf + 8 * TW, n, half);
        else fa[half][n - CT] = A.read(buf, n - CT, half);
    };
    auto multiply = [&](int half, int r) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
            acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[half][r], fb[half][t], acc[r][t], 0, 0, 0);
    };
    auto step = [&](uint4 *buf, const uint4 *nbuf, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if (r < BAR) {
#pragma unroll
                for (int n = r * READS / BAR; n < (r + 1) * READS / BAR; ++n) read(buf, 1, n);
            }
            if (r == BAR) {
                vm_wait<(NST - 2) * PER + TOUCHES>();
                lds_barrier();
            }
            __builtin_amdgcn_sched_barrier(0);
            multiply(0, r);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int n = r * READS / RT; n < (r + 1) * READS / RT; ++n) read(nbuf, 0, n);
#pragma unroll
            for (int j = r * PER / RT; j < (r + 1) * PER / RT; ++j) load_piece(buf, g + NST, j);
            __builtin_amdgcn_sched_barrier(0);
            multiply(1, r);
            __builtin_amdgcn_sched_barrier(0);
        }
        touch(g + NST + 1);
    };
    uint4 *const bufs[4] = {buf0, buf1, buf2, buf3};
#pragma unroll
    for (int st = 0; st < NST; ++st)
#pragma unroll
        for (int j = 0; j < PER; ++j) load_piece(bufs[st], t0 + st, j);
    touch(t0 + NST);
    vm_wait<(NST - 1) * PER + TOUCHES>();
    lds_barrier();
#pragma unroll
    for (int n = 0; n < READS; ++n) read(buf0, 0, n);
    int g = t0;
    for (; g + NST <= t1; g += NST) {            // no branch between the steps
#pragma unroll
        for (int st = 0; st < NST; ++st) step(bufs[st], bufs[(st + 1) % NST], g + st);
    }
#pragma unroll
    for (int st = 0; st < NST - 1; ++st)
        if (g + st < t1) step(bufs[st], bufs[(st + 1) % NST], g + st);
    vm_wait<0>();

    // lane (i, q) holds outputs 4 q .. 4 q + 3 of each row tile for row 16 t + i
    auto row_of = [&](int t) { return row0 + wn * (TT / WN) + 16 * t + i; };
    auto out_of = [&](int r) { return o0 + wm * (TW / WM) + 16 * r + 4 * q; };
    if (p.S > 1) {
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            if (row_of(t) >= p.rows) continue;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int ld = lin_part_ld(p.R);
                if (out_of(r) < p.R) *(f32x4 *)(p.part + ((size_t)split * p.rows + row_of(t)) * ld + out_of(r)) = acc[r][t];
            }
        }
        return;
    }
    if (!lin_quads(p)) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) lin_single_before(p, row_of(t), out_of(r), acc[r][t]);
        if constexpr (!SLOWA) lin_with_act(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[r][t][j] = lin_act<decltype(act)::value>(acc[r][t][j]);
        });
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) lin_single_after(p, row_of(t), out_of(r), acc[r][t]);
        return;
    }
    int o[RT];
    uint2 bias[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        o[r] = out_of(r);
        bias[r] = p.bias ? *(const uint2 *)(p.bias + min(o[r], p.R - 4)) : make_uint2(0, 0);
    }
    // (of the gradients' products nothing but y: the struct's other members are not set)
    auto out = [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            f32x4 v[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) v[r] = acc[r][t];
            lin_out_quads<decltype(act)::value, RT>(p, row_of(t), o, bias, v);
        }
    };
    if constexpr (SLOWA) out(std::integral_constant<int, MI_ACT_NONE>{});
    else lin_with_act(p.act, out);
}

// The tiles (k_linear.hip, one unit each): launches a product of them.
int lin_launch_128_64(LinGemm p, bool slow_a, bool slow_b, hipStream_t st);
int lin_launch_128_128(LinGemm p, bool slow_a, bool slow_b, hipStream_t st);
int lin_launch_256_128(LinGemm p, bool slow_a, bool slow_b, hipStream_t st);
int lin_launch_256_256(LinGemm p, bool slow_a, bool slow_b, hipStream_t st);
int lin_launch_192_256(LinGemm p, bool slow_a, bool slow_b, hipStream_t st);     // two fast operands only

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 rows: the weights are streamed once, from memory into the matrix instructions' registers.  A workgroup takes 16
// weight rows, its W wavefronts every W-th piece of 32 U columns; their sums meet in LDS.  One row through 6144 x 6144 takes
// 17.5 us, 4.3 TB/s (a copy reaches 5.1); 8 or 16 wavefronts, or two row tiles for each, took 0 to 2 us more.
template <int W, int U>
__global__ void __launch_bounds__(64 * W) lin_stream_kernel(LinGemm p) {
    __shared__ f32x4 red[W][64];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int o0 = blockIdx.x * 16;
    const __amdgpu_buffer_rsrc_t ra =
        __builtin_amdgcn_make_buffer_rsrc((void *)(p.a + (size_t)o0 * p.lda), (short)0, 0x7fffffff, kLinWord3);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void *)p.b, (short)0, 0x7fffffff, kLinWord3);
    // rows past the last one read it again: their outputs are not stored
    const uint32_t va = (uint32_t)(2 * (min(i, p.R - 1 - o0) * p.lda + 8 * q));
    const uint32_t vb = (uint32_t)(2 * (min(i, p.rows - 1) * p.ldb + 8 * q));
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    lin_bf16x8 fa[2][U], fb[2][U];
    auto load = [&](int s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (g * U + u) * 32;
            const uint32_t out = k + 8 * q >= p.K ? kLinOut : 0u;
            fa[s][u] = __builtin_bit_cast(lin_bf16x8, __builtin_amdgcn_raw_buffer_load_b128(ra, (int)(va | out), 2 * k, 0));
            fb[s][u] = __builtin_bit_cast(lin_bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rb, (int)(vb | out), 2 * k, 0));
        }
    };
    auto multiply = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[s][u], fb[s][u], acc, 0, 0, 0);
    };
    const int pieces = (p.K + 32 * U - 1) / (32 * U);
    load(0, wave);
    for (int g = wave; g < pieces; g += 2 * W) { // pieces past the end read zeros
        load(1, g + W);
        multiply(0);
        load(0, g + 2 * W);
        multiply(1);
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    f32x4 v = red[0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w][lane];
    if (i < p.rows) lin_out(p, i, o0 + 4 * q, v);
}

}  // namespace mi
