// Tiled block-scaled fp8 product (fp8.h) for many rows, dense or of sorted rows by expert.
#pragma once
#include "fp8.h"

namespace mi {

constexpr int kFp8MaxGroups = 1024;              // K / 128: the weight scales of a tile's blocks are kept in LDS

// Memory to LDS without registers: lane l's 16 (4) bytes to dst + 16 l (4 l).
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t r, uint4 *dst, uint32_t voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 16, (int)voff, soff, 0, 0);
}
__device__ __forceinline__ void lds_load4(__amdgpu_buffer_rsrc_t r, float *dst, uint32_t voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 4, (int)voff, soff, 0, 0);
}

struct Fp8Tiled {
    Fp8Gemm g;
    int nw;                     // weight tiles
    int nb;                     // token tiles (grouped: at most; *g.n_blocks are used)
    int S;                      // splits of K
    float limit;                // PAIR
    uint8_t *hq;                // PAIR: e4m3 [rows, R] and its scales
    float *hs;
    float *part[2];             // S > 1: f32 [S, rows, R] (PAIR: of gate and of up)
};

template <int TW, int TT, int WM, int WN, int NST, bool PAIR>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) fp8_gemm_kernel(Fp8Tiled p) {
    constexpr int W = WM * WN, RT = TW / WM / 16, CT = TT / WN / 16;
    constexpr int WL = TW / 8 / W, TL = TT / 8 >= W ? TT / 8 / W : 1;      // 1 KB loads per wavefront and stage
    constexpr int ROWS = TW + TT;
    static_assert(TW % (8 * W) == 0 && CT >= 1 && CT <= 4 && (!PAIR || (TW == 256 && RT % 2 == 0 && 16 % W == 0)), "");
    __shared__ uint4 buf0[ROWS * 8], buf1[ROWS * 8], buf2[NST > 2 ? ROWS * 8 : 1], buf3[NST > 3 ? ROWS * 8 : 1];
    __shared__ float sx0[W * 64], sx1[W * 64], sx2[NST > 2 ? W * 64 : 1], sx3[NST > 3 ? W * 64 : 1];
    __shared__ float sw[2][kFp8MaxGroups];
    const Fp8Gemm &a = p.g;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int KB = fp8_groups(a.K), RB = fp8_groups(a.R);

    // an XCD's workgroups (ids equal modulo 8) take one contiguous piece of the work, two token tiles of a weight tile
    // next to each other: they meet its weights in that XCD's L2
    const int nb = a.n_blocks ? min(max(*a.n_blocks, 0), p.nb) : p.nb;
    const long long total = (long long)nb * p.nw * p.S;
    const int xcd = blockIdx.x & 7, li = blockIdx.x >> 3;
    const long long first = total * xcd / 8, at = first + li;
    if (at >= total * (xcd + 1) / 8) return;
    const int per2 = 2 * p.nw * p.S;
    const int pr = (int)(at / per2), in2 = (int)(at - (long long)pr * per2);
    const int width = min(2, nb - 2 * pr);
    const int tb = 2 * pr + in2 % width, ws = in2 / width, wt = ws % p.nw, split = ws / p.nw;

    const int row0 = tb * TT;                    // first row of the token tile
    const int o0 = wt * (PAIR ? TW / 2 : TW);    // first output of the weight tile
    int e = 0;
    if (a.blk_expert) {
        e = a.blk_expert[tb];
        if (e < 0 || e >= a.E) return;           // the whole workgroup
    }
    const int t0 = split * KB / p.S, t1 = (split + 1) * KB / p.S;

    // ---- loads: instruction j of a wavefront fills 8 LDS rows of 128 bytes; 16-byte slot c of row r holds chunk
    // c ^ (r & 7) of the row, so that the fragment reads below spread over the banks
    const int col = 16 * ((lane & 7) ^ (lane >> 3));
    uint32_t voff[WL + TL];
    __amdgpu_buffer_rsrc_t rw[2], rx, rs;
#pragma unroll
    for (int j = 0; j < WL; ++j) {
        const int r = 8 * (j * W + wave) + (lane >> 3);
        voff[j] = (uint32_t)min(PAIR ? r & (TW / 2 - 1) : r, a.R - 1 - o0) * (uint32_t)a.K + col;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
        rw[m] = __builtin_amdgcn_make_buffer_rsrc((void *)(a.wq[PAIR ? m : 0] + ((size_t)e * a.R + o0) * a.K), (short)0,
                                                  0x7fffffff, kFp8Word3);
    rx = __builtin_amdgcn_make_buffer_rsrc((void *)a.xq, (short)0, 0x7fffffff, kFp8Word3);
    rs = __builtin_amdgcn_make_buffer_rsrc((void *)a.xs, (short)0, 0x7fffffff, kFp8Word3);
    auto token = [&](int r) {                    // row r of the tile: its row of xq, -1 for none
        int tok = row0 + r;
        if (tok >= a.rows) return -1;
        if (a.tok_row) tok = a.tok_row[tok];
        return tok < a.x_rows ? tok : -1;
    };
#pragma unroll
    for (int j = 0; j < TL; ++j) {
        const int tok = token(8 * ((j * W + wave) % (TT / 8)) + (lane >> 3));
        voff[WL + j] = tok < 0 ? kFp8Out : (uint32_t)tok * (uint32_t)a.K + col;
    }
    const int stok = token(wn * CT * 16 + lane % (CT * 16));
    const uint32_t soff = stok < 0 ? kFp8Out : (uint32_t)stok * (uint32_t)KB * 4u;
    // weight scales of the tile's one or two blocks
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float *s = a.ws[PAIR ? m : 0] + ((size_t)e * RB + min(o0 / kFp8Group + (PAIR ? 0 : m), RB - 1)) * KB;
        for (int g = tid; g < KB; g += 64 * W) sw[m][g] = s[g];
    }
    __syncthreads();

    auto load = [&](uint4 *buf, float *sx, int g) __attribute__((always_inline)) {
        const uint32_t past = g >= t1 || g * kFp8Group + col >= a.K ? kFp8Out : 0u;
        const int so = g * kFp8Group;
#pragma unroll
        for (int j = 0; j < WL; ++j) lds_load16(rw[PAIR ? (j * W) / 16 : 0], buf + 64 * (j * W + wave), voff[j] | past, so);
#pragma unroll
        for (int j = 0; j < TL; ++j)
            lds_load16(rx, buf + 8 * TW + 64 * ((j * W + wave) % (TT / 8)), voff[WL + j] | past, so);
        lds_load4(rs, sx + 64 * wave, g >= t1 ? kFp8Out : soff, 4 * g);
    };

    f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto wrow = [&](int r) {                     // LDS row of row tile r; PAIR: gate tiles, then the same rows of up
        return PAIR ? (r / (RT / 2)) * (TW / 2) + wm * (TW / 2 / WM) + (r % (RT / 2)) * 16 : wm * (TW / WM) + 16 * r;
    };
    const int c0 = q ^ (i & 7), c1 = c0 ^ 4;
    auto frag = [&](const uint4 *buf, int row) __attribute__((always_inline)) {
        const uint4 u = buf[(row + i) * 8 + c0], v = buf[(row + i) * 8 + c1];
        return (i32x8){(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w};
    };
    auto compute = [&](const uint4 *buf, const float *sx, int g) __attribute__((always_inline)) {
        i32x8 b[CT];
        float s[2][CT];
        const int m0 = PAIR ? 0 : TW == 128 ? 0 : wm * 2 / WM;
        const float w0 = sw[m0][g], w1 = PAIR ? sw[1][g] : 0.0f;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            b[t] = frag(buf, TW + wn * CT * 16 + 16 * t);
            const float x = sx[64 * wave + 16 * t + i];
            s[0][t] = x * w0;
            s[1][t] = PAIR ? x * w1 : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const i32x8 w = frag(buf, wrow(r));
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const f32x4 v = fp8_mfma(w, b[t]);
                const float sc = s[PAIR ? r / (RT / 2) : 0][t];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][t][j] = fmaf(v[j], sc, acc[r][t][j]);
            }
        }
    };
    constexpr int PER = WL + TL + 1;             // loads per wavefront and stage
    uint4 *const bufs[4] = {buf0, buf1, buf2, buf3};
    float *const sxs[4] = {sx0, sx1, sx2, sx3};
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) load(bufs[s], sxs[s], t0 + s);
    for (int t = t0; t < t1; t += NST) {
#pragma unroll
        for (int s = 0; s < NST; ++s) {
            // stage t + s has landed (the later ones stay in flight) for every wavefront, and every wavefront is done
            // with the buffer that the next loads overwrite
            vm_wait<(NST - 2) * PER>();
            lds_barrier();
            load(bufs[(s + NST - 1) % NST], sxs[(s + NST - 1) % NST], t + s + NST - 1);
            if (t + s < t1) compute(bufs[s], sxs[s], t + s);
        }
    }
    vm_wait<0>();

    // ---- lane (i, q) holds outputs 4 q .. 4 q + 3 of each row tile for row 16 t + i
    if constexpr (PAIR) {
        if (p.S == 1) {
            // h of a token's 128 outputs: the maximum over this wavefront's, then over the wavefronts of the token
            float *red = sx0;                    // [WM][TT]: loads into it have landed, every wavefront is past the loop
            __syncthreads();
            uint32_t am[CT];
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                am[t] = 0;
#pragma unroll
                for (int r = 0; r < RT / 2; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int o = o0 + wrow(r) + 4 * q + j;
                        const float h = o < a.R ? fp8_swiglu(acc[r][t][j], acc[RT / 2 + r][t][j], p.limit) : 0.0f;
                        acc[r][t][j] = h;
                        const uint32_t u = __float_as_uint(h) & 0x7fffffffu;
                        am[t] = max(am[t], u < 0x7f800000u ? u : 0u);
                    }
                am[t] = max(am[t], (uint32_t)__shfl_xor((int)am[t], 16, 64));
                am[t] = max(am[t], (uint32_t)__shfl_xor((int)am[t], 32, 64));
                if (q == 0) red[wm * TT + wn * CT * 16 + 16 * t + i] = __uint_as_float(am[t]);
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const int c = wn * CT * 16 + 16 * t + i, row = row0 + c;
                uint32_t m = 0;
#pragma unroll
                for (int k = 0; k < WM; ++k) m = max(m, __float_as_uint(red[k * TT + c]));
                const int ex = fp8_exponent(m);
                const float inv = exp2_int(-ex);
                if (row >= a.rows) continue;
                if (wm == 0 && q == 0) p.hs[(size_t)row * RB + o0 / kFp8Group] = exp2_int(ex);
#pragma unroll
                for (int r = 0; r < RT / 2; ++r) {
                    const int o = o0 + wrow(r) + 4 * q;
                    if (o < a.R)                 // R % 16 == 0
                        *(uint32_t *)(p.hq + (size_t)row * a.R + o) =
                            fp8_pack4(fp8_inf_to_nan(acc[r][t][0]) * inv, fp8_inf_to_nan(acc[r][t][1]) * inv,
                                      fp8_inf_to_nan(acc[r][t][2]) * inv, fp8_inf_to_nan(acc[r][t][3]) * inv);
                }
            }
            return;
        }
    }
    const bool quads = (a.R & 3) == 0;           // rows of outputs start at whole groups of four
    const bool b8 = quads && ((uintptr_t)a.y_bf16 & 7) == 0, f16 = quads && ((uintptr_t)a.y_f32 & 15) == 0;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int row = row0 + wn * CT * 16 + 16 * t + i;
        if (row >= a.rows) continue;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int m = PAIR ? r / (RT / 2) : 0;
            const int o = o0 + (PAIR ? wrow(r) - m * (TW / 2) : wrow(r)) + 4 * q;
            const f32x4 v = acc[r][t];
            float *f = p.S > 1 ? p.part[m] + (size_t)split * a.rows * a.R : a.y_f32;
            if (f) {
                f += (size_t)row * a.R + o;
                if (f16 || (p.S > 1 && quads)) {
                    if (o < a.R) *(f32x4 *)f = v;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (o + j < a.R) f[j] = v[j];
                }
            }
            if (a.y_bf16 && p.S == 1) {
                uint16_t *y = a.y_bf16 + (size_t)row * a.R + o;
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = f32_to_bf16_rne(v[j]);
                if (b8) {
                    if (o < a.R) *(uint2 *)y = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (o + j < a.R) y[j] = (uint16_t)h[j];
                }
            }
        }
    }
}

}  // namespace mi
