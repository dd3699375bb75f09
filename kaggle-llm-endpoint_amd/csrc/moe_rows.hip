// Tokens into expert order and back, and the gradients of both, over the layout of ragged_plan_kernel
// (pallas_moe.py:564-592): S = T k slots, slot (t, j) has sorted row row_slot[t, j] (-1: none), padding rows have
// tok_row -1.
//   dispatch        xs[row_slot[t, j]] = x[t], 0 on all other rows           its gradient is combine with weights 1
//   combine         out[t] = sum_j w[t, j] y[row_slot[t, j]]                 f32, in column order, rounded once
//   combine_grad    dy[row_slot[t, j]] = w[t, j] dout[t], 0 on all others;    dw[t, j] = <dout[t], y[row_slot[t, j]]>
// No atomics: every output element has one writer and a fixed order of summation.  Rows and tokens outside the
// buffers count as none.
#include "common.h"

namespace mi {

constexpr int kMoeRowsMax = 1 << 22;

// Eight consecutive elements of a row.
template <int XD>
struct Row8 {
    float v[8];
    __device__ __forceinline__ void load(const void *p, size_t at) {
        if constexpr (XD == MI_X_BF16) {
            const uint4 u = *(const uint4 *)((const uint16_t *)p + at);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        } else {
            const float4 a = *(const float4 *)((const float *)p + at), b = *(const float4 *)((const float *)p + at + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    }
    __device__ __forceinline__ void store(void *p, size_t at) const {
        if constexpr (XD == MI_X_BF16) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16_rne(v[2 * j]) | (f32_to_bf16_rne(v[2 * j + 1]) << 16);
            *(uint4 *)((uint16_t *)p + at) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *(float4 *)((float *)p + at) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4 *)((float *)p + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
};

constexpr int kPadRows = 16;                     // rows that one of the padding workgroups looks at: 16 lanes each

// Zeros for the rows that no slot of their token names (padding has no token), kPadRows a workgroup: 16 lanes look through
// a row's slots, its wavefront writes its zeros.  (With the rows that the tokens' own workgroups write these are all
// rows, also where a caller has taken slots out of the plan: row_slot -1.)
template <int XD>
__device__ __forceinline__ void zero_padding(const int32_t *__restrict__ tok_row, const int32_t *__restrict__ row_slot,
                                             int blk, int T, int k, int D, int rows, void *out) {
    const Row8<XD> zero = {};
    const int tid = threadIdx.x, row = blk * kPadRows + tid / 16;
    const int t = row < rows ? tok_row[row] : -1;
    bool named = false;
    if (t >= 0 && t < T)
        for (int j = tid % 16; j < k; j += 16) named |= row_slot[(size_t)t * k + j] == row;
    const uint64_t m = __ballot(named);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = blk * kPadRows + tid / 64 * 4 + j;
        if (r >= rows || ((m >> (16 * j)) & 0xffff)) continue;
        for (int c = (tid & 63) * 8; c < D; c += 512) zero.store(out, (size_t)r * D + c);
    }
}

// A token is read once and stored to its k rows (by row, reading tok_row's token, took 122 us instead of 93 for
// 4096 tokens of 6144 bf16 values in 8 rows each: the token's row comes from memory again where its rows are far apart).
// Workgroups 0 .. T - 1: one token each; the others zero the rows without a slot.
template <int XD>
__global__ void __launch_bounds__(256) moe_dispatch_kernel(const void *__restrict__ x, const int32_t *__restrict__ row_slot,
                                                           const int32_t *__restrict__ tok_row, int T, int k, int D,
                                                           int rows, void *__restrict__ xs) {
    const int t = blockIdx.x;
    if (t >= T) {
        zero_padding<XD>(tok_row, row_slot, t - T, T, k, D, rows, xs);
        return;
    }
    for (int c = threadIdx.x * 8; c < D; c += 2048) {
        Row8<XD> v;
        v.load(x, (size_t)t * D + c);
        for (int j0 = 0; j0 < k; j0 += 8) {
            int r[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = j0 + j < k ? row_slot[(size_t)t * k + j0 + j] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (r[j] >= 0 && r[j] < rows) v.store(xs, (size_t)r[j] * D + c);
        }
    }
}

// A workgroup per token; the rows of eight slots are loaded before the first is added.
template <int XD>
__global__ void __launch_bounds__(256) moe_combine_kernel(const void *__restrict__ y, const int32_t *__restrict__ row_slot,
                                                          const float *__restrict__ w, int k, int D, int rows,
                                                          void *__restrict__ out) {
    const int t = blockIdx.x;
    for (int c = threadIdx.x * 8; c < D; c += 2048) {
        Row8<XD> acc = {};
        for (int j0 = 0; j0 < k; j0 += 8) {
            Row8<XD> v[8];
            float wt[8];
            bool in[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // (no branch around the loads: a slot without a row loads row 0 and adds nothing, whatever that holds)
                const size_t s = (size_t)t * k + min(j0 + j, k - 1);
                const int r = row_slot[s];
                in[j] = j0 + j < k && r >= 0 && r < rows;
                wt[j] = w ? w[s] : 1.0f;
                v[j].load(y, (size_t)(in[j] ? r : 0) * D + c);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc.v[i] = in[j] ? fmaf(wt[j], v[j].v[i], acc.v[i]) : acc.v[i];
        }
        acc.store(out, (size_t)t * D + c);
    }
}

// DW: the gradient of w too, which y is read for.  The first workgroups zero the rows without a slot, the others take one token each (302 us forward and backward of 4096
// tokens with the zeros last, 297 with them first; dispatch takes 101 and 105: last there).
template <int XD, bool DW>
__global__ void __launch_bounds__(256) moe_combine_grad_kernel(const void *__restrict__ dout, const void *__restrict__ y,
                                                               const int32_t *__restrict__ row_slot,
                                                               const int32_t *__restrict__ tok_row,
                                                               const float *__restrict__ w, int T, int k, int D,
                                                               int rows, void *__restrict__ dy, float *__restrict__ dw) {
    __shared__ float part[4];
    const int pads = (rows + kPadRows - 1) / kPadRows, t = (int)blockIdx.x - pads;
    if (t < 0) {
        zero_padding<XD>(tok_row, row_slot, blockIdx.x, T, k, D, rows, dy);
        return;
    }
    for (int j = 0; j < k; ++j) {
        const int r = row_slot[(size_t)t * k + j];
        float dot = 0.0f;
        if (r >= 0 && r < rows) {
            const float wt = w[(size_t)t * k + j];
            for (int c = threadIdx.x * 8; c < D; c += 2048) {
                Row8<XD> g, v;
                g.load(dout, (size_t)t * D + c);
                if constexpr (DW) v.load(y, (size_t)r * D + c);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (DW) dot = fmaf(g.v[i], v.v[i], dot);
                    g.v[i] *= wt;
                }
                g.store(dy, (size_t)r * D + c);
            }
        }
        if constexpr (!DW) continue;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) dot += __shfl_xor(dot, m, 64);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
        __syncthreads();
        if (threadIdx.x == 0) dw[(size_t)t * k + j] = part[0] + part[1] + part[2] + part[3];
        __syncthreads();
    }
}

static int moe_rows_check(int dtype, int T, int k, int D, int rows) {
    if (dtype != MI_X_BF16 && dtype != MI_X_F32) return MI_ERR_ARG;
    if (T <= 0 || k <= 0 || (long long)T * k > kMoeRowsMax || rows <= 0 || rows > 2 * kMoeRowsMax) return MI_ERR_TOKENS;
    if (D <= 0 || D % 8 || D > (1 << 17)) return MI_ERR_SHAPE;
    return MI_OK;
}
static bool moe_rows_aligned(const void *a, const void *b, const void *c = nullptr) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}
static bool words_aligned(const void *a, const void *b = nullptr, const void *c = nullptr) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0;
}

}  // namespace mi

using namespace mi;

extern "C" int mi_moe_dispatch(const void *x, int32_t dtype, int32_t T, int32_t k, int32_t D, const int32_t *row_slot,
                               const int32_t *tok_row, int32_t rows, void *xs, void *stream) {
    if (!x || !row_slot || !tok_row || !xs) return MI_ERR_NULL;
    const int rc = moe_rows_check(dtype, T, k, D, rows);
    if (rc != MI_OK) return rc;
    if (!moe_rows_aligned(x, xs) || !words_aligned(row_slot, tok_row)) return MI_ERR_ARG;
    auto kern = dtype == MI_X_BF16 ? moe_dispatch_kernel<MI_X_BF16> : moe_dispatch_kernel<MI_X_F32>;
    hipLaunchKernelGGL(kern, dim3(T + (rows + kPadRows - 1) / kPadRows), dim3(256), 0, (hipStream_t)stream, x, row_slot,
                       tok_row, T, k, D, rows, xs);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

extern "C" int mi_moe_combine(const void *y, int32_t dtype, int32_t T, int32_t k, int32_t D, const int32_t *row_slot,
                              const float *w, int32_t rows, void *out, void *stream) {
    if (!y || !row_slot || !out) return MI_ERR_NULL;
    const int rc = moe_rows_check(dtype, T, k, D, rows);
    if (rc != MI_OK) return rc;
    if (!moe_rows_aligned(y, out) || !words_aligned(row_slot, w)) return MI_ERR_ARG;
    auto kern = dtype == MI_X_BF16 ? moe_combine_kernel<MI_X_BF16> : moe_combine_kernel<MI_X_F32>;
    hipLaunchKernelGGL(kern, dim3(T), dim3(256), 0, (hipStream_t)stream, y, row_slot, w, k, D, rows, out);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

extern "C" int mi_moe_combine_grad(const void *dout, const void *y, int32_t dtype, int32_t T, int32_t k, int32_t D,
                                   const int32_t *row_slot, const int32_t *tok_row, const float *w, int32_t rows,
                                   void *dy, float *dw, void *stream) {
    if (!dout || (dw && !y) || !row_slot || !tok_row || !w || !dy) return MI_ERR_NULL;
    const int rc = moe_rows_check(dtype, T, k, D, rows);
    if (rc != MI_OK) return rc;
    if (!moe_rows_aligned(dout, y, dy) || !words_aligned(row_slot, tok_row, w) || !words_aligned(dw)) return MI_ERR_ARG;
    auto kern = dtype == MI_X_BF16 ? dw ? moe_combine_grad_kernel<MI_X_BF16, true> : moe_combine_grad_kernel<MI_X_BF16, false>
                                   : dw ? moe_combine_grad_kernel<MI_X_F32, true> : moe_combine_grad_kernel<MI_X_F32, false>;
    hipLaunchKernelGGL(kern, dim3(T + (rows + kPadRows - 1) / kPadRows), dim3(256), 0, (hipStream_t)stream, dout, y,
                       row_slot, tok_row, w, T, k, D,
                       rows, dy, dw);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}
