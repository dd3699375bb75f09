// bf16 products on gfx950 with an epilogue, and the two products of their gradients:
//   C[t, o] = sum_k a[o, k] b[t, k],   y = act(C + bias) + residual
// in f32, rounded once.  Forward a is the weight [n_out, n_in] and b the rows [B, n_in]; the gradients take an operand whose
// contraction index is the slow one ([k, o] in memory) as it lies: its fragments are read from LDS transposed.
#pragma once
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
    uint16_t *z;                // bf16(C + bias) [rows, ldz], ldz a multiple of 8 that holds R, or NULL
    long long ldz;
    // ---- tiled launches
    int nw, nb, S;              // weight tiles, token tiles, splits of K
    float *part;                // S > 1: f32 [S, rows, R]
};

// ------------------------------------------------------------------------------------------------ activations
__device__ __forceinline__ float lin_sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }
__device__ __forceinline__ float gelu_inner2(float z) {                  // 2 sqrt(2 / pi) (z + 0.044715 z^3)
    return 1.5957691216057308f * fmaf(0.044715f * z * z, z, z);
}
__device__ __forceinline__ float lin_act(float z, int act) {
    switch (act) {
        case MI_ACT_SILU: return z * lin_sigmoid(z);
        case MI_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.7071067811865476f));
        case MI_ACT_GELU_TANH: return z * lin_sigmoid(gelu_inner2(z));   // (1 + tanh(u)) / 2 = sigmoid(2 u)
        case MI_ACT_RELU: return z < 0.0f ? 0.0f : z;                    // (a NaN stays)
        default: return z;
    }
}
// The derivative; past |z| = 30 it is 0 or 1 to f32, and the factors below may be no numbers.
__device__ __forceinline__ float lin_act_grad(float z, int act) {
    if (act != MI_ACT_NONE && fabsf(z) > 30.0f && act != MI_ACT_SILU) return z > 0.0f ? 1.0f : 0.0f;
    switch (act) {
        case MI_ACT_SILU: {
            if (fabsf(z) > 120.0f) return z > 0.0f ? 1.0f : 0.0f;
            const float s = lin_sigmoid(z);
            return s * fmaf(z, lin_sigmoid(-z), 1.0f);
        }
        case MI_ACT_GELU:
            return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), 0.5f * (1.0f + erff(z * 0.7071067811865476f)));
        case MI_ACT_GELU_TANH: {
            const float s = lin_sigmoid(gelu_inner2(z));
            return s + z * s * (1.0f - s) * 1.5957691216057308f * fmaf(0.134145f * z, z, 1.0f);
        }
        case MI_ACT_RELU: return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
        default: return 1.0f;
    }
}

// ------------------------------------------------------------------------------------------------ epilogue
// Which accesses of four consecutive outputs are whole ones.
struct LinQuads {
    bool y, res, bias;
    __device__ __forceinline__ explicit LinQuads(const LinGemm &p) {
        const bool q = (p.R & 3) == 0;
        const int m = p.f32 ? 15 : 7;
        y = q && ((uintptr_t)p.y & m) == 0;
        res = q && ((uintptr_t)p.res & m) == 0;
        bias = q && ((uintptr_t)p.bias & 7) == 0;
    }
};

__device__ __forceinline__ f32x4 lin_bf16x4(uint2 u) {
    return (f32x4){__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                   __uint_as_float(u.y & 0xffff0000u)};
}
__device__ __forceinline__ uint2 lin_pack4(f32x4 v) {
    return make_uint2(f32_to_bf16_rne(v[0]) | (f32_to_bf16_rne(v[1]) << 16),
                      f32_to_bf16_rne(v[2]) | (f32_to_bf16_rne(v[3]) << 16));
}

// Outputs o .. o + 3 (o a multiple of 4) of one row from their sums.
__device__ __forceinline__ void lin_out(const LinGemm &p, const LinQuads &quad, int row, int o, f32x4 v) {
    if (o >= p.R) return;
    const int n = min(4, p.R - o);
    const size_t at = (size_t)row * p.R + o;
    if (p.bias) {
        if (quad.bias) {
            const f32x4 b = lin_bf16x4(*(const uint2 *)(p.bias + o));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) v[j] += bf16_to_f32(p.bias[o + j]);
        }
    }
    if (p.z) *(uint2 *)(p.z + (size_t)row * p.ldz + o) = lin_pack4(v);
    if (p.act) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lin_act(v[j], p.act);
    }
    if (p.f32) {
        float *y = (float *)p.y + at;
        const float *r = (const float *)p.res + at;
        if (p.res) {
            if (quad.res) {
                const float4 u = *(const float4 *)r;
                v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < n) v[j] += r[j];
            }
        }
        if (quad.y) {
            *(f32x4 *)y = v;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) y[j] = v[j];
        }
    } else {
        uint16_t *y = (uint16_t *)p.y + at;
        const uint16_t *r = (const uint16_t *)p.res + at;
        if (p.res) {
            if (quad.res) {
                const f32x4 u = lin_bf16x4(*(const uint2 *)r);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += u[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < n) v[j] += bf16_to_f32(r[j]);
            }
        }
        if (quad.y) {
            *(uint2 *)y = lin_pack4(v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) y[j] = (uint16_t)f32_to_bf16_rne(v[j]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ tiled product
__device__ __forceinline__ void lin_lds_load(__amdgpu_buffer_rsrc_t r, uint4 *dst, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 16, (int)voff, 0, 0, 0);
}

// A slow operand's row k of a stage: the 32-byte piece u (16 columns) sits at u ^ lin_swizzle(k), so that the 16 pieces of
// one column tile that a transposed read takes (rows 8 q + 0 .. 3 of each q, or + 4 .. 7) lie on different banks.
__host__ __device__ constexpr int lin_swizzle(int k) { return (k & 3) | ((k >> 1) & 12); }

// One operand's share of a stage: T rows (fast) or columns (slow) of it, 64 deep; its loads and its fragments.
// Fast: LDS row r is 128 bytes, 16-byte chunk c of it at c ^ (r & 7).  Slow: LDS row k is T columns.
template <int T, int W, bool SLOW>
struct LinOperand {
    static constexpr int N = T / 8 / W;          // 1 KB loads of a wavefront and stage
    static_assert(T % (8 * W) == 0, "");
    const char *base;           // of the tile, stage 0
    long long advance;          // bytes from stage to stage
    uint32_t voff[N];
    int kat;                    // first contraction index of load 0 within the stage
    int frag;                   // byte of this lane's part of fragment 0

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

template <int TW, int TT, int WM, int WN, int NST, bool SLOWA, bool SLOWB>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) lin_gemm_kernel(LinGemm p) {
    constexpr int W = WM * WN, RT = TW / WM / 16, CT = TT / WN / 16, ROWS = TW + TT;
    __shared__ uint4 buf0[ROWS * 8], buf1[ROWS * 8], buf2[NST > 2 ? ROWS * 8 : 1], buf3[NST > 3 ? ROWS * 8 : 1];
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
    auto load_piece = [&](uint4 *buf, int g, int j) __attribute__((always_inline)) {
        if (j < A.N) A.load(buf, g, ka, wave, j);
        else B.load(buf + 8 * TW, g, kb, wave, j - A.N);
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
                vm_wait<(NST - 2) * PER>();
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
    };
    uint4 *const bufs[4] = {buf0, buf1, buf2, buf3};
#pragma unroll
    for (int st = 0; st < NST; ++st)
#pragma unroll
        for (int j = 0; j < PER; ++j) load_piece(bufs[st], t0 + st, j);
    vm_wait<(NST - 1) * PER>();
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
    const LinQuads quad(p);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int row = row0 + wn * (TT / WN) + 16 * t + i;
        if (row >= p.rows) continue;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int o = o0 + wm * (TW / WM) + 16 * r + 4 * q;
            if (p.S == 1) {
                lin_out(p, quad, row, o, acc[r][t]);
            } else if (o < p.R) {
                float *f = p.part + ((size_t)split * p.rows + row) * p.R + o;
                if ((p.R & 3) == 0) {
                    *(f32x4 *)f = acc[r][t];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (o + j < p.R) f[j] = acc[r][t][j];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 NT rows: the weights are streamed once, from memory into the matrix instructions' registers.  A workgroup takes
// 16 RW weight rows, its W wavefronts every W-th piece of 32 U columns; their sums meet in LDS.
template <int NT, int RW, int W, int U>
__global__ void __launch_bounds__(64 * W) lin_stream_kernel(LinGemm p) {
    __shared__ f32x4 red[W][RW * NT][64];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int o0 = blockIdx.x * 16 * RW;
    const __amdgpu_buffer_rsrc_t ra =
        __builtin_amdgcn_make_buffer_rsrc((void *)(p.a + (size_t)o0 * p.lda), (short)0, 0x7fffffff, kLinWord3);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void *)p.b, (short)0, 0x7fffffff, kLinWord3);
    uint32_t va[RW], vb[NT];
#pragma unroll
    for (int r = 0; r < RW; ++r) va[r] = (uint32_t)(2 * (min(16 * r + i, p.R - 1 - o0) * p.lda + 8 * q));
#pragma unroll
    for (int t = 0; t < NT; ++t) vb[t] = (uint32_t)(2 * (min(16 * t + i, p.rows - 1) * p.ldb + 8 * q));
    f32x4 acc[RW][NT];
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    lin_bf16x8 fa[2][RW][U], fb[2][NT][U];
    auto load = [&](int s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (g * U + u) * 32;
            const uint32_t out = k + 8 * q >= p.K ? kLinOut : 0u;
#pragma unroll
            for (int r = 0; r < RW; ++r)
                fa[s][r][u] = __builtin_bit_cast(lin_bf16x8, __builtin_amdgcn_raw_buffer_load_b128(ra, (int)(va[r] | out), 2 * k, 0));
#pragma unroll
            for (int t = 0; t < NT; ++t)
                fb[s][t][u] = __builtin_bit_cast(lin_bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rb, (int)(vb[t] | out), 2 * k, 0));
        }
    };
    auto multiply = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[s][r][u], fb[s][t][u], acc[r][t], 0, 0, 0);
    };
    const int pieces = (p.K + 32 * U - 1) / (32 * U);
    load(0, wave);
    for (int g = wave; g < pieces; g += 2 * W) { // pieces past the end read zeros
        load(1, g + W);
        multiply(0);
        load(0, g + 2 * W);
        multiply(1);
    }
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) red[wave][r * NT + t][lane] = acc[r][t];
    __syncthreads();
    const LinQuads quad(p);
    for (int n = wave; n < RW * NT; n += W) {
        f32x4 v = red[0][n][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w][n][lane];
        const int row = 16 * (n % NT) + i;
        if (row < p.rows) lin_out(p, quad, row, o0 + 16 * (n / NT) + 4 * q, v);
    }
}

}  // namespace mi
