// Products over bf16 weights with bias, activation and residual, for one row to many, and their gradients
// (linear_gemm.h), behind the C ABI.
#include <algorithm>

#include "linear_gemm.h"
#include "rows8.h"
#include "tuning.h"

namespace mi {

// The split sums of a product, added in split order, then its epilogue: four outputs a thread, eight splits' loads at once (one
// after the other they took 7 us for 37 rows).
__global__ void __launch_bounds__(256) lin_reduce_kernel(LinGemm p) {
    const int quads = lin_part_ld(p.R) / 4;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= (long long)p.rows * quads) return;
    const size_t n = (size_t)p.rows * quads;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.S; s0 += 8) {
        f32x4 u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = ((const f32x4 *)p.part)[min(s0 + j, p.S - 1) * n + at];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (s0 + j < p.S) v += u[j];
    }
    const int row = (int)(at / quads);
    lin_out(p, row, 4 * (int)(at - (long long)row * quads), v);
}

// dz = dy act'(z), rounded to bf16 for the products, whose matrix instructions take bf16 (each term off by at most 2^-8 of
// itself; dx and dW of 2048 x 6144 x 6144 behind gelu come out 0.00233 of their 2-norm off instead of the 0.00166 of their own
// rounding; a second product with what the rounding leaves would double their time), in rows of ldz columns whose last ones
// are zeros, and each workgroup's sums of dz (before their rounding) over its rows, for the bias.  A workgroup takes 256 columns, 32
// lanes of 8, and rows blockIdx.y * 8 + .., 8 at a time.
struct LinDz {
    const void *dy;             // [B, N]
    int f32, act, B, N;
    const float *z;             // [B, ldz] (act)
    long long ldz;
    uint16_t *dz;               // [B, ldz] or NULL
    float *part;                // [gridDim.y, N] or NULL
};
__global__ void __launch_bounds__(256) lin_dz_kernel(LinDz p) {
    __shared__ float sum[8][256];
    const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
    const int c = blockIdx.x * 256 + 8 * lane;
    const bool whole = p.N % 8 == 0 && ((uintptr_t)p.dy & 15) == 0;
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
    if (c < p.N) {
        for (int row = blockIdx.y * 8 + sub; row < p.B; row += gridDim.y * 8) {
            const size_t at = (size_t)row * p.N + c;
            Row8<MI_X_F32> g;
            if (whole) {
                if (p.f32) {
                    g.load(p.dy, at);
                } else {
                    Row8<MI_X_BF16> b;
                    b.load(p.dy, at);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g.v[j] = b.v[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    g.v[j] = c + j >= p.N ? 0.0f : p.f32 ? ((const float *)p.dy)[at + j] : bf16_to_f32(((const uint16_t *)p.dy)[at + j]);
            }
            if (p.act) {
                Row8<MI_X_F32> z;
                z.load(p.z, (size_t)row * p.ldz + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) g.v[j] = c + j >= p.N ? 0.0f : g.v[j] * lin_act_grad(z.v[j], p.act);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += g.v[j];
            if (p.dz) {
                Row8<MI_X_BF16> o;
#pragma unroll
                for (int j = 0; j < 8; ++j) o.v[j] = g.v[j];
                o.store(p.dz, (size_t)row * p.ldz + c);
            }
        }
    }
    if (!p.part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[sub][8 * lane + j] = acc[j];
    __syncthreads();
    const int o = blockIdx.x * 256 + threadIdx.x;
    if (o >= p.N) return;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sum[k][threadIdx.x];
    p.part[(size_t)blockIdx.y * p.N + o] = v;
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kLinMaxCols = 1 << 16;             // n_in, n_out
constexpr int kLinMaxRows = 1 << 20;
constexpr int kLinCus = 256;
constexpr int kLinStreamRows = 16;              // rows of one matrix instruction
constexpr long long kLinStreamWeights = 1 << 24;

static bool lin_shape_ok(int n_in, int n_out) {
    return n_in > 0 && n_in % 8 == 0 && n_in <= kLinMaxCols && n_out > 0 && n_out <= kLinMaxCols;
}
static size_t lin_up(size_t n) { return (n + 255) & ~(size_t)255; }
static bool lin_aligned(const void *a, int n) { return ((uintptr_t)a & (n - 1)) == 0; }
static int lin_ok() { return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH; }

struct LinPlan {
    int tw, tt, S;
};
constexpr int kLinMaxSplits = 8;
constexpr size_t kLinSplitTiles = 512;           // 128 x 128 pieces of all splits' sums together, at most

// Floats of split sums of a product of R outputs and any number of rows.
static size_t lin_split_floats(int R) {
    const size_t n = (size_t)(R + 127) / 128;
    return std::max<size_t>(kLinSplitTiles / n, 1) * 128 * lin_part_ld(R);
}

// The tile and the splits of the contraction: the pair of least estimated time.  A stage of 64 columns of a tile takes `one`
// us in a launch of at most one workgroup per CU, `more` in each round of `slots` workgroups otherwise, its start and epilogue
// as much as `ends` stages; a split adds a launch and a pass over its sums.  The times are those of operands from memory:
// 6144 x 6144, 37 / 48 / 128 / 256 / 517 / 2048 / 4096 rows take 15 (of 2051 outputs), 22.5, 29, 42, 50, 130 and 258 us with
// the tiles that this chooses; all with 256 x 256 would take 140 to 158 up to 2048 rows and 285.  3000 / 4096 / 6000 rows take
// 225 / 258 / 394 with 256 x 128 (chosen for the first two) and 246 / 255 / 379 with 192 x 256 (for the last).
static LinPlan lin_plan(int rows, int R, int K, bool fast) {
    struct Tile {
        int tw, tt, slots;
        float one, more;
        int ends;
    };
    static const Tile tiles[] = {{128, 64, 2 * kLinCus, 0.50f, 0.70f, 8}, {128, 128, kLinCus, 0.48f, 0.54f, 8},
                                 {256, 128, kLinCus, 0.74f, 0.83f, 9}, {256, 256, kLinCus, 1.52f, 1.38f, 8},
                                 {192, 256, kLinCus, 1.31f, 1.27f, 7}};
    const int steps = (K + kLinCols - 1) / kLinCols;
    const int tw = tuning(kTuneLinTw, 0), tt = tuning(kTuneLinTt, 0), fs = tuning(kTuneLinS, 0);
    LinPlan best{128, 128, 1};
    float least = 1e30f;
    for (const Tile &c : tiles) {
        if ((c.tw == 192 && !fast) || (tw && c.tw != tw) || (tt && c.tt != tt)) continue;
        const long long n = (long long)((R + c.tw - 1) / c.tw) * ((rows + c.tt - 1) / c.tt);
        // a forced count of splits is taken as far as the columns, the slots and the workspace hold it: the tile stays
        int most = std::max(std::min(fs ? std::min(fs, kLinMaxSplits) : kLinMaxSplits, steps), 1);
        while (most > 1 && (n * most > c.slots || (size_t)most * rows * lin_part_ld(R) > lin_split_floats(R))) --most;
        for (int S = fs ? most : 1; S <= most; ++S) {
            const long long wgs = n * S;
            const float step = wgs <= kLinCus ? c.one : (float)((wgs + c.slots - 1) / c.slots) * c.more;
            const float us = step * ((steps + S - 1) / S + c.ends) +
                             (S > 1 ? 3.0f + (float)((double)S * rows * R * 8 / 3.5e6) : 0.0f);
            if (us < least) least = us, best = LinPlan{c.tw, c.tt, S};
        }
    }
    return best;
}

static int lin_launch(LinGemm p, bool slow_a, bool slow_b, float *part, hipStream_t st) {
    const LinPlan pl = lin_plan(p.rows, p.R, p.K, !slow_a && !slow_b);
    p.S = pl.S;
    p.part = part;
    int rc;
    if (pl.tw == 192) rc = lin_launch_192_256(p, slow_a, slow_b, st);
    else if (pl.tt == 256) rc = lin_launch_256_256(p, slow_a, slow_b, st);
    else if (pl.tw == 256) rc = lin_launch_256_128(p, slow_a, slow_b, st);
    else if (pl.tt == 128) rc = lin_launch_128_128(p, slow_a, slow_b, st);
    else rc = lin_launch_128_64(p, slow_a, slow_b, st);
    if (rc != MI_OK || p.S == 1) return rc;
    const long long n = (long long)p.rows * ((p.R + 3) / 4);
    hipLaunchKernelGGL(lin_reduce_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
    return lin_ok();
}

// Whether a product of B rows streams the weights: every workgroup reads all rows again, which costs more the more they are
// (6144 x 6144: 1 / 4 / 8 / 16 rows 18 / 20 / 22 / 27 us, tiled with 4 splits 20 to 21; 2051 outputs of 6144 columns: 16 rows
// 14.4, tiled 19.3; 2048 x 2048: 5.3 and 8.8).
static bool lin_streams(int B, int K, int R) {
    return B <= tuning(kTuneLinStream, B <= 4 || (long long)K * R <= kLinStreamWeights ? kLinStreamRows : 0) &&
           B <= kLinStreamRows;
}

static int lin_check(int B, int n_in, int n_out, int64_t x_stride, int act) {
    if (B <= 0 || B > kLinMaxRows) return MI_ERR_TOKENS;
    if (!lin_shape_ok(n_in, n_out)) return MI_ERR_SHAPE;
    if (x_stride < n_in || x_stride % 8 || x_stride > (1 << 20)) return MI_ERR_ARG;
    return act >= MI_ACT_NONE && act <= MI_ACT_RELU ? MI_OK : MI_ERR_ARG;
}

static long long lin_pad(int n) { return (n + 7) & ~7; }
// Workgroups along the rows of lin_dz_kernel.
static int lin_dz_wgs(int B) { return std::min((B + 7) / 8, 64); }

}  // namespace mi

using namespace mi;

extern "C" size_t mi_bf16_linear_workspace(int32_t B, int32_t n_in, int32_t n_out) {
    if (lin_check(B, n_in, n_out, n_in, 0) != MI_OK || lin_streams(B, n_in, n_out)) return 0;
    return lin_up(lin_split_floats(n_out) * sizeof(float));
}

extern "C" int mi_bf16_linear(const uint16_t *x, int64_t x_stride, int32_t B, const uint16_t *wT, int32_t n_in, int32_t n_out,
                              const uint16_t *bias, int32_t act, const void *residual, int32_t y_dtype, void *y, float *z,
                              void *workspace, size_t workspace_bytes, void *stream) {
    if (!x || !wT || !y) return MI_ERR_NULL;
    const int rc = lin_check(B, n_in, n_out, x_stride, act);
    if (rc != MI_OK) return rc;
    if (y_dtype != MI_X_BF16 && y_dtype != MI_X_F32) return MI_ERR_ARG;
    const int el = y_dtype == MI_X_F32 ? 4 : 2;
    if (!lin_aligned(x, 16) || !lin_aligned(wT, 16) || !lin_aligned(bias, 2) || !lin_aligned(residual, el) ||
        !lin_aligned(y, el) || !lin_aligned(z, 16) || !lin_aligned(workspace, 16))
        return MI_ERR_ARG;
    const size_t need = mi_bf16_linear_workspace(B, n_in, n_out);
    if (need && (!workspace || workspace_bytes < need)) return MI_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    LinGemm p = {};
    p.a = wT, p.lda = n_in;
    p.b = x, p.ldb = x_stride;
    p.R = n_out, p.rows = B, p.K = p.Ks = n_in;
    p.bias = bias, p.act = act, p.res = residual;
    p.f32 = y_dtype == MI_X_F32;
    p.y = y, p.z = z, p.ldz = lin_pad(n_out);
    if (lin_streams(B, n_in, n_out)) {
        hipLaunchKernelGGL((lin_stream_kernel<4, 4>), dim3((n_out + 15) / 16), dim3(256), 0, st, p);
        return lin_ok();
    }
    return lin_launch(p, false, false, (float *)workspace, st);
}

extern "C" size_t mi_bf16_linear_grad_workspace(int32_t B, int32_t n_in, int32_t n_out) {
    if (lin_check(B, n_in, n_out, n_in, 0) != MI_OK) return 0;
    return lin_up((size_t)B * lin_pad(n_out) * 2) + lin_up((size_t)lin_dz_wgs(B) * n_out * sizeof(float)) +
           lin_up(lin_split_floats(n_in) * sizeof(float));
}

extern "C" int mi_bf16_linear_grad(const void *dy, int32_t dy_dtype, const float *z, int32_t act, const uint16_t *x,
                                   int64_t x_stride, int32_t B, const uint16_t *wT, int32_t n_in, int32_t n_out, uint16_t *dx,
                                   uint16_t *dw, uint16_t *dbias, void *workspace, size_t workspace_bytes, void *stream) {
    if (!dy || (act && !z) || (dx && !wT) || (dw && !x) || (!dx && !dw && !dbias)) return MI_ERR_NULL;
    int rc = lin_check(B, n_in, n_out, dw ? x_stride : n_in, act);
    if (rc != MI_OK) return rc;
    if (dy_dtype != MI_X_BF16 && dy_dtype != MI_X_F32) return MI_ERR_ARG;
    if (!lin_aligned(dy, dy_dtype == MI_X_F32 ? 4 : 2) || !lin_aligned(z, 16) || !lin_aligned(x, 16) || !lin_aligned(wT, 16) ||
        !lin_aligned(dx, 2) || !lin_aligned(dw, 2) || !lin_aligned(dbias, 2) || !lin_aligned(workspace, 16))
        return MI_ERR_ARG;
    if (!workspace || workspace_bytes < mi_bf16_linear_grad_workspace(B, n_in, n_out)) return MI_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    uint16_t *dz = (uint16_t *)ws;
    ws += lin_up((size_t)B * lin_pad(n_out) * 2);
    float *sums = (float *)ws;
    ws += lin_up((size_t)lin_dz_wgs(B) * n_out * sizeof(float));
    float *part = (float *)ws;
    // dy itself where it is dz already, in rows that the products can load
    const bool as_is = act == MI_ACT_NONE && dy_dtype == MI_X_BF16 && n_out % 8 == 0 && lin_aligned(dy, 16);
    if (!as_is || dbias) {
        const LinDz d = {dy, dy_dtype == MI_X_F32, act, B, n_out, z, lin_pad(n_out), as_is || !(dx || dw) ? nullptr : dz,
                         dbias ? sums : nullptr};
        const int n = lin_dz_wgs(B);
        hipLaunchKernelGGL(lin_dz_kernel, dim3((n_out + 255) / 256, n), dim3(256), 0, st, d);
        if ((rc = lin_ok()) != MI_OK) return rc;
        if (dbias) {
            hipLaunchKernelGGL(column_sums_kernel, dim3((n_out + 31) / 32), dim3(256), 0, st, sums, n, n_out, 0, (void *)dbias);
            if ((rc = lin_ok()) != MI_OK) return rc;
        }
    }
    LinGemm p = {};
    p.b = as_is ? (const uint16_t *)dy : dz;
    p.ldb = lin_pad(n_out);
    p.R = n_in;
    if (dx) {                                    // dx[t, k] = sum_n dz[t, n] w[n, k]
        p.a = wT, p.lda = n_in;
        p.rows = B, p.K = (int)lin_pad(n_out), p.Ks = n_out;
        p.y = dx;
        if ((rc = lin_launch(p, true, false, part, st)) != MI_OK) return rc;
    }
    if (dw) {                                    // dw[n, k] = sum_t dz[t, n] x[t, k]
        p.a = x, p.lda = x_stride;
        p.rows = n_out, p.K = p.Ks = B;
        p.y = dw;
        if ((rc = lin_launch(p, true, true, part, st)) != MI_OK) return rc;
    }
    return MI_OK;
}
