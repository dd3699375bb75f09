// Block-scaled fp8 products (fp8.h) behind the C ABI: rows to e4m3, the dense product, the MLP, the experts' products
// over sorted rows and the whole routed layer.
#include <algorithm>

#include "fp8.h"

namespace mi {

// ------------------------------------------------------------------------------------------------ rows to e4m3
// Eight consecutive values of a lane, as f32.
template <int XD>
__device__ __forceinline__ void load8(const void *x, size_t at, float v[8]) {
    if constexpr (XD == MI_X_BF16) {
        const uint4 u = *(const uint4 *)((const uint16_t *)x + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
        const float4 a = *(const float4 *)((const float *)x + at), b = *(const float4 *)((const float *)x + at + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
}

// A group of 128 columns is 16 lanes of 8 values: its maximum is 4 exchanges, its loads and stores are contiguous.
// Whole groups of lanes run or return together (the grid's tail), so the exchanges stay within live lanes.
template <int XD>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const void *__restrict__ x, int n, int K, long long stride,
                                                           uint8_t *__restrict__ q, float *__restrict__ s) {
    const int KB = fp8_groups(K);
    const long long gi = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
    if (gi >= (long long)n * KB) return;
    const int row = (int)(gi / KB), c = (int)(gi - (long long)row * KB);
    const int col = c * kFp8Group + (threadIdx.x & 15) * 8;
    const bool in = col < K;                     // K % 16 == 0: a lane's values are all inside or all past the row
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (in) load8<XD>(x, (size_t)row * stride + col, v);
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
        a = max(a, b < 0x7f800000u ? b : 0u);    // the finite values' maximum
        v[j] = fp8_inf_to_nan(v[j]);
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) a = max(a, (uint32_t)__shfl_xor((int)a, m, 64));
    const int e = fp8_exponent(a);
    const float inv = exp2_int(-e);
    if (in) {
        uint2 o;
        o.x = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        o.y = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *(uint2 *)(q + (size_t)row * K + col) = o;
    }
    if ((threadIdx.x & 15) == 0) s[(size_t)row * KB + c] = exp2_int(e);
}

// h = silu(min(g, L)) * clip(u, -L, L) in f32, quantised as above: one wavefront per row and group, two values a lane.
__global__ void __launch_bounds__(64) fp8_swiglu_kernel(const float *__restrict__ g, const float *__restrict__ u,
                                                        int I, float limit, uint8_t *__restrict__ q,
                                                        float *__restrict__ s) {
    const int row = blockIdx.x, c = blockIdx.y, lane = threadIdx.x;
    const int col = c * kFp8Group + 2 * lane;
    float h0 = 0.0f, h1 = 0.0f;
    if (col < I) {
        const float2 gv = *(const float2 *)(g + (size_t)row * I + col), uv = *(const float2 *)(u + (size_t)row * I + col);
        h0 = fp8_swiglu(gv.x, uv.x, limit);
        h1 = fp8_swiglu(gv.y, uv.y, limit);
    }
    const uint32_t b0 = __float_as_uint(h0) & 0x7fffffffu, b1 = __float_as_uint(h1) & 0x7fffffffu;
    uint32_t a = max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) a = max(a, (uint32_t)__shfl_xor((int)a, m, 64));
    const int e = fp8_exponent(a);
    const float inv = exp2_int(-e);
    if (col < I)
        *(uint16_t *)(q + (size_t)row * I + col) =
            (uint16_t)fp8_pack2<false>(fp8_inf_to_nan(h0) * inv, fp8_inf_to_nan(h1) * inv, 0);
    if (lane == 0) s[(size_t)row * fp8_groups(I) + c] = exp2_int(e);
}

// ------------------------------------------------------------------------------------------------ the product
// One wavefront per 16 output columns x 16 rows.
__global__ void __launch_bounds__(64) fp8_tile_kernel(Fp8Gemm a) {
    const int lane = threadIdx.x, i = lane & 15, q = lane >> 4;
    const int o0 = blockIdx.y * 16, r0 = blockIdx.x * 16;
    const int KB = fp8_groups(a.K), RB = fp8_groups(a.R);
    int e = 0;
    bool live = true;
    if (a.blk_expert) {
        const int blk = r0 / a.tm;
        e = a.blk_expert[blk];
        live = blk < *a.n_blocks && e >= 0 && e < a.E;
        if (!live) e = 0;
    }
    const int row = r0 + i;
    int tok = row < a.rows ? (a.tok_row ? a.tok_row[row] : row) : -1;
    if (tok >= a.x_rows) tok = -1;
    const int o = min(o0 + i, a.R - 1);
    const uint8_t *w = a.wq[0] + ((size_t)e * a.R + o) * a.K;
    const float *ws = a.ws[0] + ((size_t)e * RB + o0 / kFp8Group) * KB;
    const uint8_t *x = a.xq + (size_t)max(tok, 0) * a.K;
    const float *xs = a.xs + (size_t)max(tok, 0) * KB;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        for (int g = 0; g < KB; ++g) {
            uint4 wf[2] = {}, xf[2] = {};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = g * kFp8Group + 16 * (q + 4 * c);
                if (col < a.K) {
                    wf[c] = *(const uint4 *)(w + col);
                    if (tok >= 0) xf[c] = *(const uint4 *)(x + col);
                }
            }
            const i32x8 wv = {(int)wf[0].x, (int)wf[0].y, (int)wf[0].z, (int)wf[0].w,
                              (int)wf[1].x, (int)wf[1].y, (int)wf[1].z, (int)wf[1].w};
            const i32x8 xv = {(int)xf[0].x, (int)xf[0].y, (int)xf[0].z, (int)xf[0].w,
                              (int)xf[1].x, (int)xf[1].y, (int)xf[1].z, (int)xf[1].w};
            const f32x4 p = fp8_mfma(wv, xv);
            const float sc = (tok >= 0 ? xs[g] : 0.0f) * ws[g];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = fmaf(p[j], sc, acc[j]);
        }
    }
    if (row >= a.rows) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int oo = o0 + 4 * q + j;
        if (oo >= a.R) break;
        if (a.y_f32) a.y_f32[(size_t)row * a.R + oo] = acc[j];
        if (a.y_bf16) a.y_bf16[(size_t)row * a.R + oo] = (uint16_t)f32_to_bf16_rne(acc[j]);
    }
}

// out[t] = sum_j w[t, j] * y[row_slot[t, j]], f32, in column order.
__global__ void __launch_bounds__(256) fp8_combine_kernel(const float *__restrict__ y, const int32_t *__restrict__ row_slot,
                                                          const float *__restrict__ w, int T, int k, int D,
                                                          float *out_f32, uint16_t *out_bf16) {
    const int t = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
    if (c >= D) return;
    float acc = 0.0f;
    for (int j = 0; j < k; ++j) {
        const int r = row_slot[(size_t)t * k + j];
        if (r >= 0) acc = fmaf(w[(size_t)t * k + j], y[(size_t)r * D + c], acc);
    }
    if (out_f32) out_f32[(size_t)t * D + c] = acc;
    if (out_bf16) out_bf16[(size_t)t * D + c] = (uint16_t)f32_to_bf16_rne(acc);
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kFp8MaxCols = 1 << 17;             // K, R: 32-bit offsets within a tile of 256 rows
constexpr int kFp8MaxRows = 1 << 22;             // rows of activations
constexpr int kFp8MoeTm = 16;

static bool fp8_cols_ok(int K) { return K > 0 && K % 16 == 0 && K <= kFp8MaxCols; }
static bool fp8_rows_ok(int R) { return R > 0 && R <= kFp8MaxCols; }
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
static bool aligned4(const void *p) { return ((uintptr_t)p & 3) == 0; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static bool fp8_x_dtype_ok(int d) { return d == MI_X_BF16 || d == MI_X_F32 || d == MI_X_FP8; }

// Bytes of n quantised rows of K columns: values, then scales.
static size_t fp8_row_bytes(size_t n, int K) { return up256(n * K) + up256(n * fp8_groups(K) * sizeof(float)); }

static int fp8_launch_quantize(const void *x, int x_dtype, int n, int K, long long stride, uint8_t *q, float *s,
                               hipStream_t st) {
    const long long threads = (long long)n * fp8_groups(K) * 16;
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (x_dtype == MI_X_BF16)
        hipLaunchKernelGGL(fp8_quantize_kernel<MI_X_BF16>, grid, dim3(256), 0, st, x, n, K, stride, q, s);
    else
        hipLaunchKernelGGL(fp8_quantize_kernel<MI_X_F32>, grid, dim3(256), 0, st, x, n, K, stride, q, s);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

static int fp8_launch_gemm(const Fp8Gemm &a, hipStream_t st) {
    hipLaunchKernelGGL(fp8_tile_kernel, dim3((a.rows + 15) / 16, (a.R + 15) / 16), dim3(64), 0, st, a);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

static int fp8_launch_swiglu(const float *g, const float *u, int rows, int I, float limit, uint8_t *q, float *s,
                             hipStream_t st) {
    hipLaunchKernelGGL(fp8_swiglu_kernel, dim3(rows, fp8_groups(I)), dim3(64), 0, st, g, u, I, limit, q, s);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

// A workspace cut into pieces of whole 256 bytes.
struct Fp8Cut {
    uint8_t *p;
    size_t used = 0;
    template <class T>
    T *take(size_t n) {
        T *r = p ? (T *)(p + used) : nullptr;
        used += up256(n * sizeof(T));
        return r;
    }
};

// The activations of a call as e4m3 rows: the caller's own, or quantised into the workspace first.
static int fp8_rows_of(const void *x, int x_dtype, const float *xs, int n, int K, Fp8Cut &c, Fp8Gemm &a,
                       hipStream_t st) {
    if (x_dtype == MI_X_FP8) {
        a.xq = (const uint8_t *)x;
        a.xs = xs;
        return MI_OK;
    }
    uint8_t *q = c.take<uint8_t>((size_t)n * K);
    float *s = c.take<float>((size_t)n * fp8_groups(K));
    a.xq = q;
    a.xs = s;
    return fp8_launch_quantize(x, x_dtype, n, K, K, q, s, st);
}

static int fp8_check_x(const void *x, int x_dtype, const float *xs, int rows, int K) {
    if (!x || (x_dtype == MI_X_FP8 && !xs)) return MI_ERR_NULL;
    if (!fp8_x_dtype_ok(x_dtype)) return MI_ERR_ARG;
    if (rows <= 0 || rows > kFp8MaxRows) return MI_ERR_TOKENS;
    if (!fp8_cols_ok(K)) return MI_ERR_SHAPE;
    if ((long long)rows * K >= (1ll << 31)) return MI_ERR_TOKENS;
    if (!aligned16(x) || !aligned4(xs)) return MI_ERR_ARG;
    return MI_OK;
}

static int fp8_check_w(const uint8_t *q, const float *s, int E, int R, int K) {
    if (!q || !s) return MI_ERR_NULL;
    if (E <= 0 || E > kMaxExperts || !fp8_rows_ok(R) || !fp8_cols_ok(K)) return MI_ERR_SHAPE;
    if (!aligned16(q) || !aligned4(s)) return MI_ERR_ARG;
    return MI_OK;
}

static bool fp8_y_ok(const uint16_t *b, const float *f) { return ((uintptr_t)b & 1) == 0 && aligned4(f); }

}  // namespace mi

using namespace mi;

extern "C" int mi_fp8_quantize(const void *x, int32_t x_dtype, int32_t n, int32_t K, int64_t x_stride, uint8_t *q,
                               float *s, void *stream) {
    if (!x || !q || !s) return MI_ERR_NULL;
    if (x_dtype != MI_X_BF16 && x_dtype != MI_X_F32) return MI_ERR_ARG;
    if (n <= 0 || n > kFp8MaxRows) return MI_ERR_TOKENS;
    if (!fp8_cols_ok(K)) return MI_ERR_SHAPE;
    if (x_stride < K || x_stride % 8 || x_stride > (1ll << 40)) return MI_ERR_ARG;
    if (!aligned16(x) || !aligned16(q) || !aligned4(s)) return MI_ERR_ARG;
    return fp8_launch_quantize(x, x_dtype, n, K, x_stride, q, s, (hipStream_t)stream);
}

extern "C" size_t mi_fp8_project_workspace(int32_t B, int32_t n_in, int32_t n_out) {
    if (B <= 0 || B > kFp8MaxRows || !fp8_cols_ok(n_in) || !fp8_rows_ok(n_out) || (long long)B * n_in >= (1ll << 31))
        return 0;
    return fp8_row_bytes(B, n_in);
}

extern "C" int mi_fp8_project(const void *x, int32_t x_dtype, const float *xs, int32_t B, const uint8_t *wq,
                              const float *ws, int32_t n_in, int32_t n_out, uint16_t *y_bf16, float *y_f32,
                              void *workspace, size_t workspace_bytes, void *stream) {
    int rc = fp8_check_x(x, x_dtype, xs, B, n_in);
    if (rc == MI_OK) rc = fp8_check_w(wq, ws, 1, n_out, n_in);
    if (rc != MI_OK) return rc;
    if (!y_bf16 && !y_f32) return MI_ERR_NULL;
    if (!fp8_y_ok(y_bf16, y_f32)) return MI_ERR_ARG;
    if (!workspace || workspace_bytes < mi_fp8_project_workspace(B, n_in, n_out)) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    Fp8Cut c{(uint8_t *)workspace};
    Fp8Gemm a = {};
    rc = fp8_rows_of(x, x_dtype, xs, B, n_in, c, a, st);
    if (rc != MI_OK) return rc;
    a.wq[0] = wq, a.ws[0] = ws;
    a.x_rows = a.rows = B;
    a.E = 1, a.R = n_out, a.K = n_in;
    a.y_bf16 = y_bf16, a.y_f32 = y_f32;
    return fp8_launch_gemm(a, st);
}

extern "C" size_t mi_fp8_mlp_workspace(int32_t B, int32_t D, int32_t I) {
    if (B <= 0 || B > kFp8MaxRows || !fp8_cols_ok(D) || !fp8_cols_ok(I) || (long long)B * std::max(D, I) >= (1ll << 31))
        return 0;
    return fp8_row_bytes(B, D) + fp8_row_bytes(B, I) + 2 * up256((size_t)B * I * sizeof(float));
}

extern "C" int mi_fp8_mlp(const void *x, int32_t x_dtype, const float *xs, int32_t B, int32_t D, int32_t I,
                          const uint8_t *gate_q, const float *gate_s, const uint8_t *up_q, const float *up_s,
                          const uint8_t *down_q, const float *down_s, float limit, uint16_t *y_bf16, float *y_f32,
                          void *workspace, size_t workspace_bytes, void *stream) {
    int rc = fp8_check_x(x, x_dtype, xs, B, D);
    if (rc == MI_OK) rc = fp8_check_w(gate_q, gate_s, 1, I, D);
    if (rc == MI_OK) rc = fp8_check_w(up_q, up_s, 1, I, D);
    if (rc == MI_OK) rc = fp8_check_w(down_q, down_s, 1, D, I);
    if (rc != MI_OK) return rc;
    if (!y_bf16 && !y_f32) return MI_ERR_NULL;
    if (!(limit > 0.0f) || !fp8_y_ok(y_bf16, y_f32)) return MI_ERR_ARG;
    if ((long long)B * I >= (1ll << 31)) return MI_ERR_TOKENS;
    if (!workspace || workspace_bytes < mi_fp8_mlp_workspace(B, D, I)) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    Fp8Cut c{(uint8_t *)workspace};
    Fp8Gemm a = {};
    rc = fp8_rows_of(x, x_dtype, xs, B, D, c, a, st);
    if (rc != MI_OK) return rc;
    float *g = c.take<float>((size_t)B * I), *u = c.take<float>((size_t)B * I);
    uint8_t *hq = c.take<uint8_t>((size_t)B * I);
    float *hs = c.take<float>((size_t)B * fp8_groups(I));
    a.x_rows = a.rows = B;
    a.E = 1, a.R = I, a.K = D;
    a.wq[0] = gate_q, a.ws[0] = gate_s, a.y_f32 = g;
    if ((rc = fp8_launch_gemm(a, st)) != MI_OK) return rc;
    a.wq[0] = up_q, a.ws[0] = up_s, a.y_f32 = u;
    if ((rc = fp8_launch_gemm(a, st)) != MI_OK) return rc;
    if ((rc = fp8_launch_swiglu(g, u, B, I, limit, hq, hs, st)) != MI_OK) return rc;
    a.xq = hq, a.xs = hs;
    a.R = D, a.K = I;
    a.wq[0] = down_q, a.ws[0] = down_s, a.y_bf16 = y_bf16, a.y_f32 = y_f32;
    return fp8_launch_gemm(a, st);
}

extern "C" size_t mi_fp8_grouped_workspace(int32_t rows, int32_t K, int32_t R) {
    if (rows <= 0 || rows > kFp8MaxRows || !fp8_cols_ok(K) || !fp8_rows_ok(R) || (long long)rows * K >= (1ll << 31))
        return 0;
    return fp8_row_bytes(rows, K);
}

extern "C" int mi_fp8_grouped(const void *x, int32_t x_dtype, const float *xs, int32_t n_blk, int32_t tm,
                              const int32_t *blk_expert, const int32_t *n_blocks, const uint8_t *wq, const float *ws,
                              int32_t E, int32_t K, int32_t R, uint16_t *y_bf16, float *y_f32, void *workspace,
                              size_t workspace_bytes, void *stream) {
    if (tm != 16 && tm != 32 && tm != 64 && tm != 128) return MI_ERR_ARG;
    if (n_blk <= 0 || n_blk > kFp8MaxRows / tm) return MI_ERR_TOKENS;
    const int rows = n_blk * tm;
    int rc = fp8_check_x(x, x_dtype, xs, rows, K);
    if (rc == MI_OK) rc = fp8_check_w(wq, ws, E, R, K);
    if (rc != MI_OK) return rc;
    if (!blk_expert || !n_blocks || (!y_bf16 && !y_f32)) return MI_ERR_NULL;
    if (!aligned4(blk_expert) || !aligned4(n_blocks) || !fp8_y_ok(y_bf16, y_f32)) return MI_ERR_ARG;
    if (!workspace || workspace_bytes < mi_fp8_grouped_workspace(rows, K, R)) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    Fp8Cut c{(uint8_t *)workspace};
    Fp8Gemm a = {};
    rc = fp8_rows_of(x, x_dtype, xs, rows, K, c, a, st);
    if (rc != MI_OK) return rc;
    a.wq[0] = wq, a.ws[0] = ws;
    a.blk_expert = blk_expert, a.n_blocks = n_blocks;
    a.x_rows = a.rows = rows;
    a.tm = tm;
    a.E = E, a.R = R, a.K = K;
    a.y_bf16 = y_bf16, a.y_f32 = y_f32;
    return fp8_launch_gemm(a, st);
}

namespace mi {

struct Fp8MoeCut {
    int rows, blocks;
    uint8_t *xq, *hq;
    float *xs, *hs, *g, *u, *y, *w_row;
    int32_t *blk_expert, *n_blocks, *tok_row, *row_slot;
    size_t bytes;
};

static Fp8MoeCut fp8_moe_cut(uint8_t *base, int T, int k, int E, int D, int I) {
    Fp8MoeCut m;
    const int S = T * k, tm = kFp8MoeTm;
    m.blocks = (S + tm - 1) / tm + E;
    m.rows = m.blocks * tm;
    Fp8Cut c{base};
    m.xq = c.take<uint8_t>((size_t)T * D);
    m.xs = c.take<float>((size_t)T * fp8_groups(D));
    m.blk_expert = c.take<int32_t>(m.blocks);
    m.n_blocks = c.take<int32_t>(1);
    m.tok_row = c.take<int32_t>(m.rows);
    m.w_row = c.take<float>(m.rows);
    m.row_slot = c.take<int32_t>(S);
    m.g = c.take<float>((size_t)m.rows * I);
    m.u = c.take<float>((size_t)m.rows * I);
    m.hq = c.take<uint8_t>((size_t)m.rows * I);
    m.hs = c.take<float>((size_t)m.rows * fp8_groups(I));
    m.y = c.take<float>((size_t)m.rows * D);
    m.bytes = c.used;
    return m;
}

static int fp8_moe_check(int T, int k, int E, int D, int I) {
    if (T <= 0 || k <= 0 || (long long)T * k > kFp8MaxRows || (long long)T * D >= (1ll << 31)) return MI_ERR_TOKENS;
    if (E <= 0 || E > kMaxExperts || !fp8_cols_ok(D) || !fp8_cols_ok(I)) return MI_ERR_SHAPE;
    const long long rows = (((long long)T * k + kFp8MoeTm - 1) / kFp8MoeTm + E) * kFp8MoeTm;
    return rows * I < (1ll << 31) ? MI_OK : MI_ERR_TOKENS;
}

}  // namespace mi

extern "C" size_t mi_fp8_moe_workspace(int32_t T, int32_t k, int32_t E, int32_t D, int32_t I) {
    return fp8_moe_check(T, k, E, D, I) == MI_OK ? fp8_moe_cut(nullptr, T, k, E, D, I).bytes : 0;
}

extern "C" int mi_fp8_moe(const uint8_t *gate_q, const float *gate_s, const uint8_t *up_q, const float *up_s,
                          const uint8_t *down_q, const float *down_s, int32_t E, int32_t D, int32_t I, const void *x,
                          int32_t x_dtype, int32_t T, int32_t k, const int32_t *idx, const float *w, float limit,
                          float *out_f32, uint16_t *out_bf16, void *workspace, size_t workspace_bytes, void *stream) {
    if (!x || !idx || !w || (!out_f32 && !out_bf16)) return MI_ERR_NULL;
    if (x_dtype != MI_X_BF16 && x_dtype != MI_X_F32) return MI_ERR_ARG;
    int rc = fp8_moe_check(T, k, E, D, I);
    if (rc == MI_OK) rc = fp8_check_w(gate_q, gate_s, E, I, D);
    if (rc == MI_OK) rc = fp8_check_w(up_q, up_s, E, I, D);
    if (rc == MI_OK) rc = fp8_check_w(down_q, down_s, E, D, I);
    if (rc != MI_OK) return rc;
    if (!(limit > 0.0f) || !aligned16(x) || !aligned4(idx) || !aligned4(w) || !fp8_y_ok(out_bf16, out_f32)) return MI_ERR_ARG;
    const Fp8MoeCut m = fp8_moe_cut((uint8_t *)workspace, T, k, E, D, I);
    if (!workspace || workspace_bytes < m.bytes) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if ((rc = fp8_launch_quantize(x, x_dtype, T, D, D, m.xq, m.xs, st)) != MI_OK) return rc;
    rc = mi_ragged_plan(idx, w, T, k, E, kFp8MoeTm, m.blk_expert, m.n_blocks, m.tok_row, m.w_row, m.row_slot, stream);
    if (rc != MI_OK) return rc;
    Fp8Gemm a = {};
    a.xq = m.xq, a.xs = m.xs;
    a.tok_row = m.tok_row, a.blk_expert = m.blk_expert, a.n_blocks = m.n_blocks;
    a.x_rows = T, a.rows = m.rows, a.tm = kFp8MoeTm;
    a.E = E, a.R = I, a.K = D;
    a.wq[0] = gate_q, a.ws[0] = gate_s, a.y_f32 = m.g;
    if ((rc = fp8_launch_gemm(a, st)) != MI_OK) return rc;
    a.wq[0] = up_q, a.ws[0] = up_s, a.y_f32 = m.u;
    if ((rc = fp8_launch_gemm(a, st)) != MI_OK) return rc;
    if ((rc = fp8_launch_swiglu(m.g, m.u, m.rows, I, limit, m.hq, m.hs, st)) != MI_OK) return rc;
    a.xq = m.hq, a.xs = m.hs;
    a.tok_row = nullptr, a.x_rows = m.rows;
    a.R = D, a.K = I;
    a.wq[0] = down_q, a.ws[0] = down_s, a.y_f32 = m.y;
    if ((rc = fp8_launch_gemm(a, st)) != MI_OK) return rc;
    hipLaunchKernelGGL(fp8_combine_kernel, dim3(T, (D + 255) / 256), dim3(256), 0, st, m.y, m.row_slot, w, T, k, D,
                       out_f32, out_bf16);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}
