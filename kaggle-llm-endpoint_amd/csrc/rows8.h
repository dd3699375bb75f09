// Rows of bf16 or f32 values: eight consecutive elements as f32, one 16-byte access (two for f32), and sums of columns.
#pragma once
#include "common.h"

namespace mi {

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

// Sums over the n rows of part [n, D]: in order within 8 pieces, then the pieces; 32 columns a workgroup.
static __global__ void __launch_bounds__(256) column_sums_kernel(const float *__restrict__ part, int n, int D, int f32, void *out) {
    __shared__ float sum[8][32];
    const int lane = threadIdx.x & 31, piece = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float a = 0.0f;
    if (c < D)
        for (int k0 = piece; k0 < n; k0 += 64) { // eight loads at once
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k0 + 8 * j < n ? part[(size_t)(k0 + 8 * j) * D + c] : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) a += v[j];
        }
    sum[piece][lane] = a;
    __syncthreads();
    if (piece || c >= D) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) a += sum[k][lane];
    if (f32)
        ((float *)out)[c] = a;
    else
        ((uint16_t *)out)[c] = (uint16_t)f32_to_bf16_rne(a);
}

}  // namespace mi
