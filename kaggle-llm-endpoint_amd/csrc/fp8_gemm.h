// Tiled block-scaled fp8 product (fp8.h) for many rows, dense or of sorted rows by expert; PAIR: of gate and up, with
// h = swiglu quantised again in the epilogue.
//
// A workgroup computes TW weight rows x TT tokens, its wavefronts WM x WN of them, one group of 128 columns a step: NST
// stages of both operands are in LDS, filled from memory without registers, and a step is RT x CT matrix instructions a
// wavefront.  An instruction's operands come from LDS as whole fragments (weights in use for CT instructions, tokens for
// the whole step), its result is scaled and added by 4 fused multiply-adds.
//
// What bounds it: a step of 256 x 256 would take 72 % of its time without its loads and 50 %, about that of its matrix
// instructions, with neither loads nor barriers.  The loads mostly wait for memory under load, which takes longer to answer
// than the stages in flight last: weights that already are in the last-level cache save up to a third.  4096 x 6144 x 6144
// takes 198 us (1.56 PFLOP/s; a library's product with one scale for the whole tensor takes 123), the routed layer's 2.4 GB
// of weights for 200 tokens in 8 slots each 500 us (4.9 TB/s).
//
// Measured and not kept: touching lines two or three stages ahead from the same wavefronts (loads return in order, so they
// are waited for as well: 3 to 13 % slower), two 128 x 128 workgroups per CU (20 % faster at 768 rows, up to 15 % slower at
// 900 to 3000), higher priority around the matrix instructions, loads spread over the whole step, 2, 4 or 16 in
// kFp8Near (within 2 %).
#pragma once
#include <type_traits>

#include "fp8.h"

namespace mi {

constexpr int kFp8Near = 8;                      // token tiles of a weight tile that run next to each other
constexpr int kFp8AheadLoads = 4;                // lines in flight of a lane that reads ahead
constexpr int kFp8AheadRows = 512;               // weight rows that one workgroup reads ahead

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
    int skip;                   // rows without a token are not written (else: zeros)
    int ahead;                  // workgroups of an XCD that only read its weights, ahead of the others
    float limit;                // PAIR
    uint8_t *hq;                // PAIR: e4m3 [rows, R] and its scales
    float *hs;
    float *part[2];             // S > 1: f32 [S, rows, R] (PAIR: of gate and of up)
};

template <int TW, int TT, int WM, int WN, int NST, bool PAIR, bool EXACT>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) fp8_gemm_kernel(Fp8Tiled p) {
    constexpr int W = WM * WN, RT = TW / WM / 16, CT = TT / WN / 16;
    constexpr int WL = TW / 8 / W, TL = TT / 8 >= W ? TT / 8 / W : 1;      // 1 KB loads per wavefront and stage
    constexpr int ROWS = TW + TT;
    static_assert(TW % (8 * W) == 0 && (CT == 1 || CT == 2 || CT == 4), "");
    static_assert(!PAIR || (TW == 256 && RT % 2 == 0 && 16 % W == 0), "");
    __shared__ uint4 buf0[ROWS * 8], buf1[ROWS * 8], buf2[NST > 2 ? ROWS * 8 : 1], buf3[NST > 3 ? ROWS * 8 : 1];
    __shared__ float sx0[W * 64], sx1[W * 64], sx2[NST > 2 ? W * 64 : 1], sx3[NST > 3 ? W * 64 : 1];
    __shared__ float sw[2][kFp8MaxGroups + 1];     // (a step reads one group ahead)
    const Fp8Gemm &a = p.g;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int KB = fp8_groups(a.K), RB = fp8_groups(a.R);

    // An XCD's workgroups (ids equal modulo 8) take one contiguous piece of the work: kFp8Near token tiles of a weight
    // tile, then of the next.  Its 32 CUs then work on about 8 token tiles x 4 weight tiles at a time and meet each other's
    // loads in that XCD's L2; the blocks of one expert are next to each other and share its weights.
    const int nb = a.n_blocks ? min(max(*a.n_blocks, 0), p.nb) : p.nb;
    const long long total = (long long)nb * p.nw * p.S;
    const int xcd = blockIdx.x & 7, li = blockIdx.x >> 3;
    const long long first = total * xcd / 8, at = first + li, end = total * (xcd + 1) / 8;
    // the zeros of one 256-output piece of a block that has no product
    auto zero = [&](int blk, int w) {
        const int o1 = w * TW;
        for (int r = wave; r < TT && blk * TT + r < a.rows; r += W)
            for (int o = o1 + lane; o < min(o1 + TW, a.R); o += 64) {
                const size_t n = (size_t)(blk * TT + r) * a.R + o;
                if (a.y_f32) a.y_f32[n] = 0.0f;
                if (a.y_bf16) a.y_bf16[n] = 0;
            }
    };
    if (p.ahead && li >= (int)((total + 7) / 8)) {
        // An idle CU reads the XCD's weights into its L2 in the order of their use, one word of each 128-byte line, so that
        // the CUs at work find them there: a stage's loads have one to three steps to come back, less than a read of HBM
        // takes under load.  (nb <= kFp8Near: the XCD's items are all token tiles of some weight tiles.)
        // One CU reads about 90 bytes a ns, 512 rows in 0.7 us a group: with more than that for each it would end last.
        const int lo = (int)(first / nb), tiles = (int)((end - 1) / nb) - lo + 1;
        const int rows = min(tiles * TW, p.ahead * kFp8AheadRows);
        const int lines = rows * ((KB + p.S - 1) / p.S), step = p.ahead * 64 * W;
        for (int l = (li - (int)((total + 7) / 8)) * 64 * W + tid; l < lines; l += kFp8AheadLoads * step) {
            uint32_t v[kFp8AheadLoads];
#pragma unroll
            for (int k = 0; k < kFp8AheadLoads; ++k) {
                const int n = min(l + k * step, lines - 1), r = n % rows, item = lo + r / TW;
                const int m = PAIR ? r % TW / (TW / 2) : 0;
                const int o = item % p.nw * (PAIR ? TW / 2 : TW) + r % (PAIR ? TW / 2 : TW);
                const int g = item / p.nw * KB / p.S + n / rows;
                v[k] = *(const uint32_t *)(a.wq[m] + (size_t)min(o, a.R - 1) * a.K + min(g * kFp8Group, a.K - 16));
            }
#pragma unroll
            for (int k = 0; k < kFp8AheadLoads; ++k) asm volatile("" ::"v"(v[k]));    // (the loads stay)
        }
        return;
    }
    if (at >= end) {
        // this workgroup has none: the blocks behind the last one in use are dealt out to those that every XCD has over
        const int over = (int)(gridDim.x >> 3) - (int)((total + 7) / 8), z = (int)(at - end);
        if (PAIR || p.skip || !a.blk_expert || z >= over) return;
        const long long dead = (long long)(p.nb - nb) * p.nw;
        for (long long d = z * 8 + xcd; d < dead; d += over * 8) zero(nb + (int)(d / p.nw), (int)(d % p.nw));
        return;
    }
    const int per = kFp8Near * p.nw * p.S;
    const int pr = (int)(at / per), in = (int)(at - (long long)pr * per);
    const int width = min(kFp8Near, nb - kFp8Near * pr);
    const int tb = kFp8Near * pr + in % width, ws = in / width, wt = ws % p.nw, split = ws / p.nw;

    const int row0 = tb * TT;                    // first row of the token tile
    const int o0 = wt * (PAIR ? TW / 2 : TW);    // first output of the weight tile
    int e = 0;
    if (a.blk_expert) {
        e = a.blk_expert[tb];
        if (e < 0 || e >= a.E) {                 // the whole workgroup
            if (!PAIR && !p.skip) zero(tb, wt);
            return;
        }
    }
    const int t0 = split * KB / p.S, t1 = (split + 1) * KB / p.S;

    // token tile t of wavefront column wn is rows 16 (t WN + wn) ..: dealt out in turn, so that a block with fewer rows
    // takes as many steps less of every wavefront.  Rows are filled from the front (live says which are).
    int used = min(TT, a.rows - row0);
    if (a.live) {
        int n = 0;
        for (int r = lane; r < TT; r += 64)
            if (row0 + r < a.rows && a.live[row0 + r] >= 0) n = r + 1;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) n = max(n, __shfl_xor(n, m, 64));
        used = __builtin_amdgcn_readfirstlane(n);
    }
    const int ct = (used + 16 * WN - 1) / (16 * WN);
    auto trow = [&](int t) { return 16 * (t * WN + wn); };

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
        if (tok >= a.rows || (a.live && a.live[tok] < 0)) return -1;
        if (a.tok_row) tok = a.tok_row[tok];
        return tok < a.x_rows ? tok : -1;
    };
#pragma unroll
    for (int j = 0; j < TL; ++j) {
        const int tok = token(8 * ((j * W + wave) % (TT / 8)) + (lane >> 3));
        voff[WL + j] = tok < 0 ? kFp8Out : (uint32_t)tok * (uint32_t)a.K + col;
    }
    const int stok = token(trow(lane / 16 % CT) + i);
    const uint32_t soff = stok < 0 ? kFp8Out : (uint32_t)stok * (uint32_t)KB * 4u;
    // weight scales of the tile's one or two blocks
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float *s = a.ws[PAIR ? m : 0] + ((size_t)e * RB + min(o0 / kFp8Group + (PAIR ? 0 : m), RB - 1)) * KB;
        for (int g = tid; g < KB; g += 64 * W) sw[m][g] = s[g];
    }
    __syncthreads();

    constexpr int PER = WL + TL + 1;             // loads per wavefront and stage
    auto past = [&](int g) __attribute__((always_inline)) {
        return g >= t1 || g * kFp8Group + col >= a.K ? kFp8Out : 0u;
    };
    auto load_piece = [&](uint4 *buf, float *sx, int g, uint32_t pst, int j) __attribute__((always_inline)) {
        if (j < WL)
            lds_load16(rw[PAIR ? (j * W) / 16 : 0], buf + 64 * (j * W + wave), voff[j] | pst, g * kFp8Group);
        else if (j < WL + TL)
            lds_load16(rx, buf + 8 * TW + 64 * (((j - WL) * W + wave) % (TT / 8)), voff[j] | pst, g * kFp8Group);
        else
            lds_load4(rs, sx + 64 * wave, g >= t1 ? kFp8Out : soff, 4 * g);
    };

    f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int shift[2] = {0, 0};                       // of the scales (fp8_scale_shift); PAIR: of gate's and up's
    auto wrow = [&](int r) {                     // LDS row of row tile r; PAIR: gate tiles, then the same rows of up
        return PAIR ? (r / (RT / 2)) * (TW / 2) + wm * (TW / 2 / WM) + (r % (RT / 2)) * 16 : wm * (TW / WM) + 16 * r;
    };
    const int c0 = q ^ (i & 7), c1 = c0 ^ 4;
    auto frag = [&](const uint4 *buf, int row) __attribute__((always_inline)) {
        const uint4 u = buf[(row + i) * 8 + c0], v = buf[(row + i) * 8 + c1];
        return (i32x8){(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w};
    };
    // One matrix instruction after the other, n = r CU + t, each behind the scaling of the result two instructions
    // older, which is done by then; weights are read from LDS WD row tiles ahead (one where registers are short), the
    // next stage's tokens where this stage's are used last.  The order below is the order of the instructions: left
    // alone the compiler puts each result's use right behind its instruction and waits for it.
    //
    // The only barrier of a stage is where its last fragment has been read: then the next stage must have landed (the
    // later ones stay in flight), and this one's buffer may be overwritten.
    auto main_loop = [&](auto cu) __attribute__((always_inline)) {
        constexpr int CU = decltype(cu)::value, N = RT * CU, LAG = 2, WD = RT * CU > 16 ? 1 : 2, BAR = RT - WD;
        static_assert(RT % 4 == 0, "the rings w and v start every step at 0");
        i32x8 b[CU], w[4];
        f32x4 v[4];
        float x[CU], w0, w1, s[PAIR ? 2 : 1][CU], last[LAG];
        const int own = PAIR || TW == 128 ? 0 : wm * 2 / WM;         // the block whose scales this wavefront uses first
        auto add = [&](int n, float sc) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n / CU][n % CU][j] = fmaf(v[n & 3][j], sc, acc[n / CU][n % CU][j]);
        };
        auto read_x = [&](const uint4 *buf, const float *sx, int t) __attribute__((always_inline)) {
            b[t] = frag(buf, TW + trow(t));
            x[t] = sx[64 * wave + 16 * t + i];
        };
        auto read_sw = [&](int g) __attribute__((always_inline)) {
            w0 = sw[own][g];
            if (PAIR) w1 = sw[1][g];
        };
        // stage g in buf; the next stage in nbuf; buf takes stage g + NST
        auto step = [&](uint4 *buf, float *sx, const uint4 *nbuf, const float *nsx, int g) __attribute__((always_inline)) {
            const uint32_t pst = past(g + NST);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if (r == BAR) {
                    vm_wait<(NST - 2) * PER>();
                    lds_barrier();
                }
                w[(r + WD) & 3] = r + WD < RT ? frag(buf, wrow(r + WD)) : frag(nbuf, wrow(r + WD - RT));
                if (r >= BAR) {
#pragma unroll
                    for (int j = (r - BAR) * PER / (RT - BAR); j < (r - BAR + 1) * PER / (RT - BAR); ++j)
                        load_piece(buf, sx, g + NST, pst, j);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < CU; ++t) {
                    const int n = r * CU + t;
                    if (r == 0) {
                        if (t == 0) {
                            w0 = ldexpf(w0, -shift[0]);
                            if (PAIR) w1 = ldexpf(w1, -shift[1]);
                        }
                        s[0][t] = x[t] * w0;
                        if (PAIR) s[PAIR ? 1 : 0][t] = x[t] * w1;
                    }
                    if (n < LAG) add(N - LAG + n, last[n]);
                    else add(n - LAG, s[PAIR ? (n - LAG) / CU / (RT / 2) : 0][(n - LAG) % CU]);
                    v[n & 3] = fp8_product<EXACT>(w[r & 3], b[t]);
                    if (r == RT - 1) read_x(nbuf, nsx, t);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            read_sw(g + 1);
#pragma unroll
            for (int k = 0; k < LAG; ++k) last[k] = s[PAIR ? 1 : 0][(N - LAG + k) % CU];
        };
        uint4 *const bufs[4] = {buf0, buf1, buf2, buf3};
        float *const sxs[4] = {sx0, sx1, sx2, sx3};
#pragma unroll
        for (int st = 0; st < NST; ++st)
#pragma unroll
            for (int j = 0; j < PER; ++j) load_piece(bufs[st], sxs[st], t0 + st, past(t0 + st), j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < (PAIR ? 2 : 1); ++m) {   // while the first stages are on their way
            float big = 0.0f;
            for (int g = lane; g < KB; g += 64) big = fmaxf(big, fabsf(sw[PAIR ? m : own][g]));
            shift[m] = fp8_wave_shift(big);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < LAG; ++k) last[k] = 0.0f;
        vm_wait<(NST - 1) * PER>();
        lds_barrier();
#pragma unroll
        for (int t = 0; t < CU; ++t) read_x(buf0, sx0, t);
        read_sw(t0);
        w[0] = frag(buf0, wrow(0));
        if (WD > 1) w[1] = frag(buf0, wrow(1));
        int g = t0;
        for (; g + NST <= t1; g += NST) {            // no branch between the steps
#pragma unroll
            for (int st = 0; st < NST; ++st)
                step(bufs[st], sxs[st], bufs[(st + 1) % NST], sxs[(st + 1) % NST], g + st);
        }
#pragma unroll
        for (int st = 0; st < NST - 1; ++st)
            if (g + st < t1) step(bufs[st], sxs[st], bufs[(st + 1) % NST], sxs[(st + 1) % NST], g + st);
#pragma unroll
        for (int k = 0; k < LAG; ++k) add(N - LAG + k, last[k]);
    };
    if (CT == 4 && ct >= 4) main_loop(std::integral_constant<int, CT >= 4 ? 4 : 1>{});
    else if (CT == 4 && ct == 3) main_loop(std::integral_constant<int, CT >= 4 ? 3 : 1>{});
    else if (CT >= 2 && ct >= 2) main_loop(std::integral_constant<int, CT >= 2 ? 2 : 1>{});
    else main_loop(std::integral_constant<int, 1>{});
    vm_wait<0>();
    if (shift[0] | shift[1]) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][t][j] = ldexpf(acc[r][t][j], shift[PAIR ? r / (RT / 2) : 0]);
    }

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
                if (q == 0) red[wm * TT + trow(t) + i] = __uint_as_float(am[t]);
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const int c = trow(t) + i, row = row0 + c;
                uint32_t m = 0;
#pragma unroll
                for (int k = 0; k < WM; ++k) m = max(m, __float_as_uint(red[k * TT + c]));
                const int ex = fp8_exponent(m);
                const float inv = exp2_int(-ex);
                if (row >= a.rows || (p.skip && a.live[row] < 0)) continue;
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
        const int row = row0 + trow(t) + i;
        if (row >= a.rows) continue;
        const bool dead = a.live && a.live[row] < 0;
        if (dead && p.skip) continue;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int m = PAIR ? r / (RT / 2) : 0;
            const int o = o0 + (PAIR ? wrow(r) - m * (TW / 2) : wrow(r)) + 4 * q;
            const f32x4 v = dead ? (f32x4){0.f, 0.f, 0.f, 0.f} : acc[r][t];   // (0 times a NaN weight is not 0)
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
