// Root-mean-square norm of rows, with the residual's addition before it and the e4m3 rows of fp8.h behind it, and its
// gradients.
//   s = round_t(x + residual)                   the stream, held in its type t (s = x without a residual)
//   r = f32(1 / sqrt(mean(s^2) + eps))          the squares added in 64 bits
//   y = (s r) w                                 two products, each rounded to f32
// and y to t, or to e4m3 with a power-of-two scale per 128 columns as fp8_quantize does it.
//   with g = dy w and n = s r:  ds = r (g - n mean(g n)) + dstream,  dx = dresidual = ds,  dw = sum_t dy n
//
// The sum of squares is added in 64 bits so that r is the same f32 whatever the order of the additions (but where the sum
// lies within 2^-50 of a rounding border): a value next to a border of e4m3, or a group's maximum next to a power of two,
// falls on the same side in every implementation.  It costs nothing: the launches are bound by memory.
//
// One pass: a row is loaded once and stays in registers between its sum and its outputs.  LANES lanes take a row, NV times 8
// consecutive values each.  Bound by memory: 4099 rows of 6144 bf16 values with a residual to stream and e4m3 in 38 us (4.6
// TB/s), to stream and bf16 in 42 (4.8; a copy reaches 5.1).
#include <algorithm>

#include "fp8.h"
#include "rows8.h"

namespace mi {

constexpr int kNormMaxCols = 1 << 15;            // 1024 lanes of 32 values
constexpr int kNormMaxRows = 1 << 22;

struct NormFwd {
    const void *x, *res, *w;    // res may be NULL
    int w_f32;
    long long x_stride, res_stride;
    int T, D;
    double eps;
    void *y, *stream;           // either may be NULL (stream: with res only)
    float *r;                   // [T] or NULL
    uint8_t *q;                 // with qs, or both NULL
    float *qs;
};

__device__ __forceinline__ void load8_of(Row8<MI_X_F32> &v, const void *p, bool f32, size_t at) {
    if (f32) {
        v.load(p, at);
    } else {
        Row8<MI_X_BF16> b;
        b.load(p, at);
#pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = b.v[i];
    }
}

// The sum of v over a row's LANES lanes, in every one of them; red: a double (float) per wavefront of the workgroup.
template <int LANES, class F>
__device__ __forceinline__ F row_sum(F v, F *red) {
#pragma unroll
    for (int m = 1; m < (LANES < 64 ? LANES : 64); m <<= 1) v += __shfl_xor(v, m, 64);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int k = 0; k < LANES / 64; ++k) v += red[k];
    }
    return v;
}

template <int XD, int LANES, int NV>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) rms_norm_kernel(NormFwd p) {
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
    __shared__ double red[LANES > 64 ? LANES / 64 : 1];
    const int row = blockIdx.x * ROWS + threadIdx.x / LANES, lane = threadIdx.x % LANES;
    if (LANES <= 64 && row >= p.T) return;       // a row's lanes leave together
    Row8<XD> v[NV];
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * LANES + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k].v[i] = 0.0f;
        if (c < p.D) v[k].load(p.x, (size_t)row * p.x_stride + c);
    }
    if (p.res) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LANES + lane) * 8;
            if (c >= p.D) continue;
            Row8<XD> a;
            a.load(p.res, (size_t)row * p.res_stride + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[k].v[i] += a.v[i];
                if (XD == MI_X_BF16) v[k].v[i] = round_bf16(v[k].v[i]);
            }
            if (p.stream) v[k].store(p.stream, (size_t)row * p.D + c);
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fma((double)v[k].v[i], (double)v[k].v[i], sum);
    sum = row_sum<LANES>(sum, red);
    const float r = (float)(1.0 / sqrt(sum / p.D + p.eps));
    if (p.r && lane == 0) p.r[row] = r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * LANES + lane) * 8;
        const bool in = c < p.D;
        Row8<MI_X_F32> w;
        if (in) load8_of(w, p.w, p.w_f32, c);
        Row8<XD> y;
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y.v[i] = in ? (v[k].v[i] * r) * w.v[i] : 0.0f;
            const uint32_t b = __float_as_uint(y.v[i]) & 0x7fffffffu;
            a = max(a, b < 0x7f800000u ? b : 0u);
        }
        if (p.y && in) y.store(p.y, (size_t)row * p.D + c);
        if (p.q) {
            // a group of 128 columns is 16 lanes (of which none or all exchange: they share their row)
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) a = max(a, (uint32_t)__shfl_xor((int)a, m, 64));
            const int e = fp8_exponent(a);
            const float inv = exp2_int(-e);
            if (!in) continue;
            uint2 o;
            o.x = fp8_pack4(fp8_inf_to_nan(y.v[0]) * inv, fp8_inf_to_nan(y.v[1]) * inv, fp8_inf_to_nan(y.v[2]) * inv,
                            fp8_inf_to_nan(y.v[3]) * inv);
            o.y = fp8_pack4(fp8_inf_to_nan(y.v[4]) * inv, fp8_inf_to_nan(y.v[5]) * inv, fp8_inf_to_nan(y.v[6]) * inv,
                            fp8_inf_to_nan(y.v[7]) * inv);
            *(uint2 *)(p.q + (size_t)row * p.D + c) = o;
            if ((lane & 15) == 0) p.qs[(size_t)row * fp8_groups(p.D) + c / kFp8Group] = exp2_int(e);
        }
    }
}

struct NormBwd {
    const void *dy, *s, *ds_in, *w;      // ds_in (the stream's gradient) may be NULL
    int w_f32;
    const float *r;
    long long s_stride;
    int T, D, n_wg;
    void *dx;
    float *part;                // [n_wg, D]: each workgroup's sum of dy n, or NULL
};

// A row's share of a lane as it lies in memory.
template <int XD, int NV>
struct RawRow {
    Row8<XD> v[NV];
    uint4 u[NV];
    __device__ __forceinline__ void load(const void *p, size_t row, int lanes, int lane, int D) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * lanes + lane) * 8;
            if constexpr (XD == MI_X_BF16) {
                u[k] = c < D ? *(const uint4 *)((const uint16_t *)p + row + c) : make_uint4(0, 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k].v[i] = 0.0f;
                if (c < D) v[k].load(p, row + c);
            }
        }
    }
    __device__ __forceinline__ Row8<XD> get(int k) const {
        if constexpr (XD != MI_X_BF16) return v[k];
        const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
        Row8<XD> r;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            r.v[2 * j] = __uint_as_float(w[j] << 16);
            r.v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
        return r;
    }
};

// A workgroup takes rows blockIdx.x, blockIdx.x + n_wg, ...; its columns' share of dw stays in registers over them.  (One
// row at a time by its ROWS parts, so that a lane's columns are the same for all.)  The next row is loaded while this one is
// summed, up to 256 lanes: 4096 rows of 6144 bf16 values in 45 us, 4.5 TB/s (without 55).  f32 rows past 6144 columns then take
// 273 registers, one workgroup a CU at a time, and are no slower for it: 4096 of 8192 in 117 us with the sums of dw, 4.6 TB/s
// (bf16 65 us, 4.1).  1024 lanes have registers for a row only, and past 16384 columns spill 14 (f32 12) of them.
template <int XD, int LANES, int NV>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) rms_norm_grad_kernel(NormBwd p) {
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
    constexpr bool PIPE = LANES <= 256;
    __shared__ float red[2][LANES > 64 ? LANES / 64 : 1];
    __shared__ float sum[ROWS > 1 ? ROWS * LANES * 8 : 1];
    const int part = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    float acc[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[k][i] = 0.0f;
    const float inv_d = 1.0f / (float)p.D;
    int flip = 0;
    RawRow<XD, NV> rg, rn, rd;
    float next_r = 0.0f;
    auto load = [&](int row) __attribute__((always_inline)) {
        rg.load(p.dy, (size_t)row * p.D, LANES, lane, p.D);
        rn.load(p.s, (size_t)row * p.s_stride, LANES, lane, p.D);
        if (PIPE && p.ds_in) rd.load(p.ds_in, (size_t)row * p.D, LANES, lane, p.D);
        next_r = p.r[row];
    };
    const int first = blockIdx.x * ROWS + part, step = p.n_wg * ROWS;
    if (PIPE && first < p.T) load(first);
    for (int row = first; row < p.T; row += step, flip ^= 1) {
        if (!PIPE) load(row);
        Row8<XD> g[NV], n[NV], d[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            g[k] = rg.get(k), n[k] = rn.get(k);
            if (PIPE && p.ds_in) d[k] = rd.get(k);
            else d[k] = {};
        }
        const float r = next_r;
        if (PIPE && row + step < p.T) load(row + step);
        float dot = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LANES + lane) * 8;
            if (c >= p.D) continue;
            Row8<MI_X_F32> w;
            load8_of(w, p.w, p.w_f32, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[k].v[i] *= r;
                acc[k][i] = fmaf(g[k].v[i], n[k].v[i], acc[k][i]);
                g[k].v[i] *= w.v[i];
                dot = fmaf(g[k].v[i], n[k].v[i], dot);
            }
        }
        // (two buffers in turn: a wavefront may be a row ahead of the one that still reads)
        const float mean = row_sum<LANES>(dot, red[flip]) * inv_d;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * LANES + lane) * 8;
            if (c >= p.D) continue;
            if (!PIPE && p.ds_in) d[k].load(p.ds_in, (size_t)row * p.D + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[k].v[i] = fmaf(r, fmaf(-mean, n[k].v[i], g[k].v[i]), d[k].v[i]);
            d[k].store(p.dx, (size_t)row * p.D + c);
        }
    }
    if (!p.part) return;
    if constexpr (ROWS > 1) {
        // the parts' sums, 8 columns of a lane at a time
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[(part * 8 + i) * LANES + lane] = acc[k][i];
            __syncthreads();
            const int c = (k * LANES + lane) * 8;
            if (part == 0 && c < p.D) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float a = acc[k][i];
                    for (int q = 1; q < ROWS; ++q) a += sum[(q * 8 + i) * LANES + lane];
                    acc[k][i] = a;
                }
            }
        }
        if (part) return;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * LANES + lane) * 8;
        if (c >= p.D) continue;
        float *o = p.part + (size_t)blockIdx.x * p.D + c;
        *(float4 *)o = make_float4(acc[k][0], acc[k][1], acc[k][2], acc[k][3]);
        *(float4 *)(o + 4) = make_float4(acc[k][4], acc[k][5], acc[k][6], acc[k][7]);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// f(lanes, values / 8) of the least number of values that holds a row.
template <class F>
static int norm_shape(int D, F f) {
    using std::integral_constant;
#define MI_NORM(L, N) \
    if (D <= 8 * L * N) return f(integral_constant<int, L>{}, integral_constant<int, N>{});
    MI_NORM(16, 1) MI_NORM(64, 1) MI_NORM(64, 2) MI_NORM(256, 1) MI_NORM(256, 2) MI_NORM(256, 3) MI_NORM(256, 4)
    MI_NORM(1024, 2) MI_NORM(1024, 4)
#undef MI_NORM
    return MI_ERR_SHAPE;
}

static int norm_check(int dtype, int w_dtype, int T, int D) {
    if ((dtype != MI_X_BF16 && dtype != MI_X_F32) || (w_dtype != MI_X_BF16 && w_dtype != MI_X_F32)) return MI_ERR_ARG;
    if (T <= 0 || T > kNormMaxRows) return MI_ERR_TOKENS;
    return D > 0 && D % 8 == 0 && D <= kNormMaxCols ? MI_OK : MI_ERR_SHAPE;
}
static bool norm_stride_ok(long long stride, int D) { return stride >= D && stride % 8 == 0 && stride <= (1ll << 40); }
static bool norm_aligned(const void *a, const void *b, const void *c = nullptr) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}

// Workgroups of the gradient: two for each CU, one of 1024 lanes (4096 rows of 6144 / 2048, 2000 of 16384 with 256 / 512 / 768
// workgroups: 66 / 54 / 62, 28 / 22.5 / 23, 61 / 66 / 72 us, their sums of dw in it).
static int norm_grad_wgs(int T, int D) { return std::min(T, D > 8192 ? 256 : 512); }

}  // namespace mi

using namespace mi;

extern "C" int mi_rms_norm(const void *x, int32_t dtype, int64_t x_stride, const void *residual, int64_t residual_stride,
                           const void *w, int32_t w_dtype, int32_t T, int32_t D, double eps, void *y, void *stream_out,
                           float *rstd, uint8_t *q, float *qs, void *stream) {
    if (!x || !w || (!y && !q) || (stream_out && !residual) || (!q != !qs)) return MI_ERR_NULL;
    const int rc = norm_check(dtype, w_dtype, T, D);
    if (rc != MI_OK) return rc;
    if (q && D % 16) return MI_ERR_SHAPE;
    if (!norm_stride_ok(x_stride, D) || (residual && !norm_stride_ok(residual_stride, D))) return MI_ERR_ARG;
    if (!(eps >= 0.0) || eps > 1e30) return MI_ERR_ARG;
    if (!norm_aligned(x, residual, w) || !norm_aligned(y, stream_out, q) || ((uintptr_t)rstd & 3) || ((uintptr_t)qs & 3))
        return MI_ERR_ARG;
    const NormFwd p = {x, residual, w, w_dtype == MI_X_F32, x_stride, residual_stride, T, D, eps, y, stream_out, rstd, q, qs};
    return norm_shape(D, [&](auto lanes, auto nv) {
        constexpr int L = decltype(lanes)::value, N = decltype(nv)::value, ROWS = L < 256 ? 256 / L : 1;
        if (L >= 256 && (long long)T * L >= (1ll << 32)) return (int)MI_ERR_TOKENS;      // a grid's threads
        auto kern = dtype == MI_X_BF16 ? rms_norm_kernel<MI_X_BF16, L, N> : rms_norm_kernel<MI_X_F32, L, N>;
        hipLaunchKernelGGL(kern, dim3((T + ROWS - 1) / ROWS), dim3(L < 256 ? 256 : L), 0, (hipStream_t)stream, p);
        return hipGetLastError() == hipSuccess ? (int)MI_OK : (int)MI_ERR_LAUNCH;
    });
}

extern "C" size_t mi_rms_norm_grad_workspace(int32_t T, int32_t D) {
    return norm_check(MI_X_BF16, MI_X_BF16, T, D) == MI_OK ? (size_t)norm_grad_wgs(T, D) * D * sizeof(float) : 0;
}

extern "C" int mi_rms_norm_grad(const void *dy, const void *s, int32_t dtype, int64_t s_stride, const void *dstream,
                                const void *w, int32_t w_dtype, const float *rstd, int32_t T, int32_t D, void *dx,
                                void *dw, void *workspace, size_t workspace_bytes, void *stream) {
    if (!dy || !s || !w || !rstd || !dx) return MI_ERR_NULL;
    const int rc = norm_check(dtype, w_dtype, T, D);
    if (rc != MI_OK) return rc;
    if (!norm_stride_ok(s_stride, D)) return MI_ERR_ARG;
    if (!norm_aligned(dy, s, dstream) || !norm_aligned(w, dx, dw) || ((uintptr_t)rstd & 3)) return MI_ERR_ARG;
    if (dw && (!workspace || workspace_bytes < mi_rms_norm_grad_workspace(T, D))) return MI_ERR_WORKSPACE;
    if (!norm_aligned(workspace, nullptr)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    float *part = dw ? (float *)workspace : nullptr;
    int n = 0;
    const int launched = norm_shape(D, [&](auto lanes, auto nv) {
        constexpr int L = decltype(lanes)::value, N = decltype(nv)::value, ROWS = L < 256 ? 256 / L : 1;
        n = norm_grad_wgs((T + ROWS - 1) / ROWS, D);
        const NormBwd p = {dy, s, dstream, w, w_dtype == MI_X_F32, rstd, s_stride, T, D, n, dx, part};
        auto kern = dtype == MI_X_BF16 ? rms_norm_grad_kernel<MI_X_BF16, L, N> : rms_norm_grad_kernel<MI_X_F32, L, N>;
        hipLaunchKernelGGL(kern, dim3(n), dim3(L < 256 ? 256 : L), 0, st, p);
        return hipGetLastError() == hipSuccess ? (int)MI_OK : (int)MI_ERR_LAUNCH;
    });
    if (launched != MI_OK || !dw) return launched;
    hipLaunchKernelGGL(column_sums_kernel, dim3((D + 31) / 32), dim3(256), 0, st, part, n, D, (int)(w_dtype == MI_X_F32), dw);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}
