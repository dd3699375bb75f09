// Block-scaled fp8 product (fp8.h) for few rows: the weights stream from memory into registers once.
//
// A workgroup owns 16 RW outputs (of each of two matrices, PAIR) for up to 16 NT rows; its W wavefronts split the groups of
// 128 columns, each holds U groups' weights in flight, quantises its own part of the activations in registers (a group of a
// row is 32 values in each of 4 lanes: two exchanges give its maximum) and multiplies with one instruction per group and
// tile; the W sums are added through LDS in wavefront order.
//
// Memory bounds it: one token's 8 experts of 6144 / 2048 take 38 us for gate and up (201 MB, 5.3 TB/s) and 22 us for down
// (101 MB), a 6144 x 6144 matrix one row 9.5 us (4.0 TB/s, most of the rest its start; 11.5 if none of it is in the
// last-level cache).  The rows are quantised once in each workgroup, which costs no pass over memory and, with several row
// tiles to serve, no time that the stream does not cover.
//
// Scales that need a shift (fp8_scale_shift) are found as they go by, and the wavefront's groups are then taken a second
// time.  (Its scales looked through beforehand, from loads ahead of the ring's, cost one row's MLP 0.8 us of 17, this 0.5.)
#pragma once
#include "fp8.h"

namespace mi {

constexpr int kFp8TileSlots = 16;                // slots that a workgroup's one token tile holds

struct Fp8Stream {
    const void *x;              // bf16, f32 or e4m3 [x_rows, K] (XD)
    const float *xs;            // XD == MI_X_FP8: its scales
    const uint8_t *wq[2];       // e4m3 [E, R, K]; PAIR: gate, up
    const float *ws[2];
    const int32_t *idx;         // expert of every slot (SLOTS)
    int rows;                   // rows of x and y; SLOTS: slots, at most kFp8TileSlots
    int div;                    // SLOTS: slot s reads row s / div of x
    int E, R, K;
    float limit;                // PAIR
    uint16_t *y_bf16;           // [rows, R]
    float *y_f32;               // [rows, R]; PAIR: h
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// A lane's 32 columns of one group: 16-byte chunks q and q + 4 of the e4m3 row (columns 16 q .. and 64 + 16 q ..).
template <int XD>
struct Fp8X {
    static constexpr int N = XD == MI_X_BF16 ? 4 : XD == MI_X_F32 ? 8 : 2;     // 16-byte loads
    uint4 v[N];
    float s;                                                                  // XD == MI_X_FP8
};

template <int XD>
__device__ __forceinline__ void fp8_x_load(Fp8X<XD> &f, __amdgpu_buffer_rsrc_t rx, __amdgpu_buffer_rsrc_t rs,
                                           uint32_t voff, uint32_t soff, uint32_t past0, uint32_t past1, uint32_t end,
                                           int g) {
    constexpr int ES = XD == MI_X_BF16 ? 2 : XD == MI_X_F32 ? 4 : 1, H = Fp8X<XD>::N / 2;
#pragma unroll
    for (int j = 0; j < 2 * H; ++j)
        f.v[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                               rx, (int)((voff | (j < H ? past0 : past1)) + (j / H) * 64 * ES + (j % H) * 16),
                                               g * kFp8Group * ES, 0));
    if (XD == MI_X_FP8) f.s = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, (int)(soff | end), 4 * g, 0));
}

// The group's e4m3 values and the row's scale; every lane of the wavefront calls it.
template <int XD>
__device__ __forceinline__ i32x8 fp8_x_quantize(const Fp8X<XD> &f, float &scale) {
    i32x8 o;
    if constexpr (XD == MI_X_FP8) {
        o = (i32x8){(int)f.v[0].x, (int)f.v[0].y, (int)f.v[0].z, (int)f.v[0].w,
                    (int)f.v[1].x, (int)f.v[1].y, (int)f.v[1].z, (int)f.v[1].w};
        scale = f.s;
    } else {
        uint32_t u[4 * Fp8X<XD>::N];
#pragma unroll
        for (int j = 0; j < Fp8X<XD>::N; ++j) {
            u[4 * j] = f.v[j].x, u[4 * j + 1] = f.v[j].y;
            u[4 * j + 2] = f.v[j].z, u[4 * j + 3] = f.v[j].w;
        }
        uint32_t a = 0;
        if constexpr (XD == MI_X_BF16) {
            u16x2 m = {0, 0};
#pragma unroll
            for (int j = 0; j < 16; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u[j] & 0x7fff7fffu));
            a = (uint32_t)max(m.x, m.y) << 16;
        } else {
            float m = 0.0f;                      // (a NaN never wins)
#pragma unroll
            for (int j = 0; j < 32; ++j) m = fmaxf(m, fabsf(__uint_as_float(u[j])));
            a = __float_as_uint(m);
        }
        a = max(a, (uint32_t)__shfl_xor((int)a, 16, 64));
        a = max(a, (uint32_t)__shfl_xor((int)a, 32, 64));
        const float s = exp2_int(fp8_exponent(a));
        // an infinity or NaN: every output of the row is NaN whatever the other values are
        scale = a >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : s;
#pragma unroll
        for (int j = 0; j < 8; ++j) {            // 4 values a word; the conversion divides by the power of two itself
            s16x2 w = {0, 0};
            if constexpr (XD == MI_X_BF16) {
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, u[2 * j]), s, false);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, u[2 * j + 1]), s, true);
            } else {
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, __uint_as_float(u[4 * j]), __uint_as_float(u[4 * j + 1]),
                                                             s, false);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, __uint_as_float(u[4 * j + 2]),
                                                             __uint_as_float(u[4 * j + 3]), s, true);
            }
            o[j] = __builtin_bit_cast(int, w);
        }
    }
    return o;
}

template <int XD, int NT, int RW, bool PAIR, bool SLOTS, int W, int U, int OCC>
__global__ void __launch_bounds__(64 * W, OCC) fp8_stream_kernel(Fp8Stream a) {
    constexpr int M = PAIR ? 2 : 1, TILES = M * RW * NT;
    static_assert(!SLOTS || NT == 1, "a slot tile is 16 slots");
    __shared__ f32x4 red[W][TILES][64];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int KB = fp8_groups(a.K), RB = fp8_groups(a.R);
    const int o0 = blockIdx.x * 16 * RW;

    int e = 0, row[NT];                          // this lane's rows of y (-1: none)
    if constexpr (SLOTS) {
        // the slots of this slot's expert; the first one's workgroups take them all, the others' end
        const int slot = blockIdx.y;
        const int e0 = lane < a.rows ? a.idx[lane] : -1;
        e = __builtin_amdgcn_readfirstlane(a.idx[slot]);
        if (e < 0 || e >= a.E) return;           // the whole workgroup: a slot without an expert has no product
        uint64_t m = __ballot(e0 == e);
        if (m & ((1ull << slot) - 1)) return;
        row[0] = -1;
        for (int j = 0; m; ++j, m &= m - 1)
            if (j == i) row[0] = __ffsll((unsigned long long)m) - 1;
    } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) row[t] = 16 * t + i < a.rows ? 16 * t + i : -1;
    }

    constexpr int ES = XD == MI_X_BF16 ? 2 : XD == MI_X_F32 ? 4 : 1;
    __amdgpu_buffer_rsrc_t rw[M];
    __amdgpu_buffer_rsrc_t rws[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        rw[m] = __builtin_amdgcn_make_buffer_rsrc((void *)(a.wq[m] + ((size_t)e * a.R + o0) * a.K), (short)0, 0x7fffffff,
                                                  kFp8Word3);
        rws[m] = __builtin_amdgcn_make_buffer_rsrc((void *)(a.ws[m] + ((size_t)e * RB + o0 / kFp8Group) * KB), (short)0,
                                                   0x7fffffff, kFp8Word3);
    }
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void *)a.x, (short)0, 0x7fffffff, kFp8Word3);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)a.xs, (short)0, 0x7fffffff, kFp8Word3);
    uint32_t wo[RW], xo[NT], so[NT];
#pragma unroll
    for (int r = 0; r < RW; ++r) wo[r] = (uint32_t)min(16 * r + i, a.R - 1 - o0) * (uint32_t)a.K + 16 * q;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t xr = (uint32_t)(SLOTS ? max(row[t], 0) / a.div : max(row[t], 0));
        xo[t] = row[t] < 0 ? kFp8Out : (xr * (uint32_t)a.K + 16 * q) * ES;
        so[t] = row[t] < 0 ? kFp8Out : xr * (uint32_t)KB * 4u;
    }
    const int g0 = wave * KB / W, g1 = (wave + 1) * KB / W;

    uint4 wv[U][M][RW][2];
    float wsv[U][M];                             // the blocks' scales, in the ring of loads like the rest
    Fp8X<XD> xv[U][NT];
    auto load = [&](int u, int g) __attribute__((always_inline)) {
        const int col = g * kFp8Group + 16 * q;
        const uint32_t end = g >= g1 ? kFp8Out : 0u;
        const uint32_t p0 = g >= g1 || col >= a.K ? kFp8Out : 0u, p1 = g >= g1 || col + 64 >= a.K ? kFp8Out : 0u;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            wsv[u][m] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rws[m], (int)end, 4 * g, 0));
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    wv[u][m][r][c] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                                                   rw[m], (int)((wo[r] | (c ? p1 : p0)) + 64 * c), g * kFp8Group, 0));
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) fp8_x_load<XD>(xv[u][t], rx, rs, xo[t], so[t], p0, p1, end, g);
    };
    f32x4 acc[M][RW][NT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[m][r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    };
    // the group in place u of the ring, its weight scales as given
    auto add = [&](int u, const float (&ws)[M]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float xs;
            const i32x8 b = fp8_x_quantize<XD>(xv[u][t], xs);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const float sc = xs * ws[m];
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    const uint4 c0 = wv[u][m][r][0], c1 = wv[u][m][r][1];
                    const f32x4 v = fp8_product<PAIR>((i32x8){(int)c0.x, (int)c0.y, (int)c0.z, (int)c0.w,
                                                     (int)c1.x, (int)c1.y, (int)c1.z, (int)c1.w}, b);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[m][r][t][j] = fmaf(v[j], sc, acc[m][r][t][j]);
                }
            }
        }
    };
    clear();
    float big[M] = {};                           // the largest scale (fp8_scale_shift)
#pragma unroll
    for (int u = 0; u < U; ++u) {
        load(u, g0 + u);
        __builtin_amdgcn_sched_barrier(0);       // the ring's order is the order of the waits
    }
    for (int g = g0; g < g1; g += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // past the last group everything reads zero and adds zero
            add(u, wsv[u]);
#pragma unroll
            for (int m = 0; m < M; ++m) big[m] = fmaxf(big[m], fabsf(wsv[u][m]));
            __builtin_amdgcn_sched_barrier(0);
            load(u, g + u + U);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    int shift[M], any = 0;
#pragma unroll
    for (int m = 0; m < M; ++m) any |= shift[m] = fp8_wave_shift(big[m]);
    if (any) {                                   // again, one group at a time, with this wavefront's scales shifted
        clear();
#pragma unroll 1
        for (int g = g0; g < g1; ++g) {
            load(0, g);
            float ws[M];
#pragma unroll
            for (int m = 0; m < M; ++m) ws[m] = ldexpf(wsv[0][m], -shift[m]);
            add(0, ws);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[m][r][t][j] = ldexpf(acc[m][r][t][j], shift[m]);
    }

#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < RW; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) red[wave][(m * RW + r) * NT + t][lane] = acc[m][r][t];
    __syncthreads();
    // wavefront w finishes tile (r, t) = w (gate and up of it together)
    for (int n = wave; n < RW * NT; n += W) {
        f32x4 v[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            v[m] = red[0][m * RW * NT + n][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) {
                const f32x4 o = red[w][m * RW * NT + n][lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[m][j] += o[j];
            }
        }
        int rr = row[0];
#pragma unroll
        for (int t = 1; t < NT; ++t)
            if (n % NT == t) rr = row[t];
        if (rr < 0) continue;
        const int o = o0 + 16 * (n / NT) + 4 * q;
        if constexpr (PAIR) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[0][j] = fp8_swiglu(v[0][j], v[M - 1][j], a.limit);
        }
        const bool quads = (a.R & 3) == 0;
        if (a.y_f32) {
            float *f = a.y_f32 + (size_t)rr * a.R + o;
            if (quads && ((uintptr_t)a.y_f32 & 15) == 0) {
                if (o < a.R) *(f32x4 *)f = v[0];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (o + j < a.R) f[j] = v[0][j];
            }
        }
        if (a.y_bf16) {
            uint16_t *y = a.y_bf16 + (size_t)rr * a.R + o;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (o + j < a.R) y[j] = (uint16_t)f32_to_bf16_rne(v[0][j]);
        }
    }
}

}  // namespace mi
