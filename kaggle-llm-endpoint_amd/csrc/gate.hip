// Routing from a router's logits: scores, balancing bias, groups of experts, the k largest choices, renormalised weights,
// and the gradient of the logits.  (route.hip has the reference's sigmoid router, from hidden states.)
//   s = sigmoid(l) or softmax(l);  c = s + bias, -inf where l is;  of n_group groups the topk_group with the largest sum of
//   their 1 or 2 largest c stay;  idx = the k largest c, equal ones by the lower id;  w = s[idx] / (sum + 1e-20) scaling
//
// A choice is a key: c as a double whose lowest 10 bits hold the id, so that one maximum finds the largest c and among
// equal ones the lowest id.  c has to be exact to the 42 bits that are left, since the order of the choices is whole
// numbers that a router's f32 scores decide otherwise about once in 10^5 choices: the scores behind choices are made in 64
// bits (2^-47, by the series of e^r).  Without a bias, or groups, the logits order the experts as they are.
//
// LPR lanes take a row (4 rows a wavefront where E <= 256), a lane PER consecutive experts, no lane's experts in two groups.
// A round of the selection is a lane's maximum, 4 rotations within 16 lanes (and 2 exchanges for 64) and the removal of the
// winner: about 4 PER + 16 instructions.
#include <math.h>

#include "common.h"

namespace mi {

constexpr int kGateMaxE = 1024;
constexpr int kGateMaxK = 32;
constexpr int kGateMaxT = 1 << 22;
constexpr uint32_t kGateNone = 0xffefffffu;      // high word of a key that is out: below every f32

struct GateArgs {
    const void *logits;
    long long stride;
    const float *bias;          // [E] or NULL
    int T, E, k, scores, n_group, topk_group, group_top, norm;
    float scaling;
    int32_t *idx;               // [T, k]
    float *w;                   // [T, k]; gradient: dw
    void *dlogits;              // gradient: [T, E]
};

// (The plain instruction: fmax would also quiet each operand first, in an instruction of its own.  A rotation may not read
// its result within two wait states, which the compiler keeps for instructions of its own only: key_max_then_rotate.)
__device__ __forceinline__ double key_max(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double key_max_then_rotate(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// f over the LPR lanes of a row, in every one of them.
template <int N>
__device__ __forceinline__ int row_ror(int v) { return __builtin_amdgcn_update_dpp(v, v, 0x120 + N, 0xf, 0xf, false); }
template <int N, class T>
__device__ __forceinline__ T rotated(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint2 u = __builtin_bit_cast(uint2, v);
        return __builtin_bit_cast(T, make_uint2((uint32_t)row_ror<N>((int)u.x), (uint32_t)row_ror<N>((int)u.y)));
    } else {
        return __builtin_bit_cast(T, row_ror<N>(__builtin_bit_cast(int, v)));
    }
}
template <int LPR, class T, class F>
__device__ __forceinline__ T over_row(T v, F f) {
    v = f(v, rotated<8>(v));
    v = f(v, rotated<4>(v));
    v = f(v, rotated<2>(v));
    v = f(v, rotated<1>(v));
    if constexpr (LPR == 64) {
        v = f(v, __shfl_xor(v, 16, 64));
        v = f(v, __shfl_xor(v, 32, 64));
    }
    return v;
}

// e^x for x <= 0: 2^n times the series of e^r, |r| <= ln 2 / 2, whose first term left out is below 2^-47.
__device__ __forceinline__ double exp_neg(double x) {
    x = x < -1100.0 ? -1100.0 : x;                           // (0 from there on; a NaN stays one)
    const double shifted = fma(x, 1.4426950408889634, 0x1.8p52);        // n, to nearest, in the lowest bits
    const double n = shifted - 0x1.8p52;
    const double r = fma(n, -1.9082149292705877e-10, fma(n, -0.6931471803691238, x));
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)__builtin_bit_cast(uint2, shifted).x);
}
// 1 / x for x in [1, 2^11]: the instruction's 2^-14 or better, squared twice.
__device__ __forceinline__ double reciprocal(double x) {
    double y = __builtin_amdgcn_rcp(x);
    y = fma(y, fma(-x, y, 1.0), y);
    return fma(y, fma(-x, y, 1.0), y);
}
__device__ __forceinline__ double sigmoid64(double l) {
    const double e = exp_neg(-fabs(l));
    return (l < 0.0 ? e : 1.0) * reciprocal(1.0 + e);
}
__device__ __forceinline__ float sigmoid32(float l) {
    const float e = expf(-fabsf(l));
    return (l < 0.0f ? e : 1.0f) / (1.0f + e);
}

__device__ __forceinline__ double gate_key(double c, int id, bool none) {
    // the minimum makes +inf and NaN the largest double, the sum -0 to 0
    const uint2 u = __builtin_bit_cast(uint2, fmin(c + 0.0, 0x1.fffffffffffffp1023));
    const uint32_t flip = (uint32_t)((int)u.y >> 31);                    // all ones below 0: the lower id is the larger key
    return __builtin_bit_cast(double, make_uint2((u.x & ~1023u) | ((1023u - (uint32_t)id) ^ (flip & 1023u)), none ? kGateNone : u.y));
}
__device__ __forceinline__ bool gate_out(double key) { return key < -0x1p1000; }
__device__ __forceinline__ int gate_id(double key) {
    const uint2 u = __builtin_bit_cast(uint2, key);
    return gate_out(key) ? -1 : (int)((int)u.y < 0 ? u.x & 1023u : 1023u - (u.x & 1023u));
}
__device__ __forceinline__ double gate_drop(double key, bool drop) {
    const uint2 u = __builtin_bit_cast(uint2, key);
    return __builtin_bit_cast(double, make_uint2(u.x, drop ? kGateNone : u.y));
}

__device__ __forceinline__ double without_id(double key) {
    const uint2 u = __builtin_bit_cast(uint2, key);
    return __builtin_bit_cast(double, make_uint2(u.x & ~1023u, u.y));
}

template <int XD>
__device__ __forceinline__ float gate_load(const void *p, size_t at) {
    if constexpr (XD == MI_X_BF16)
        return bf16_to_f32(((const uint16_t *)p)[at]);
    else
        return ((const float *)p)[at];
}

// A row's share of a lane: experts id0 .. id0 + n - 1.
template <int LPR>
struct GateLane {
    int row, lane, group, id0, n;
    __device__ __forceinline__ GateLane(const GateArgs &p) {
        row = (int)((blockIdx.x * 256ll + threadIdx.x) / LPR);
        lane = threadIdx.x % LPR;
        const int lanes = LPR / p.n_group, size = p.E / p.n_group;       // of a group
        const int per = (size + lanes - 1) / lanes, in = lane % lanes;
        group = lane / lanes;
        id0 = group * size + in * per;
        n = max(0, min(per, size - in * per));
    }
};

// The row's logits: -inf behind the lane's share.  16-byte loads where they fit.
template <int XD, int PER>
__device__ __forceinline__ void gate_logits(const GateArgs &p, int row, int id0, int n, float (&l)[PER]) {
    constexpr int V = XD == MI_X_BF16 ? 8 : 4;
    const char *base = (const char *)p.logits + ((size_t)row * p.stride + id0) * (XD == MI_X_BF16 ? 2 : 4);
    if (PER % V == 0 && __ballot(n != PER || ((uintptr_t)base & 15)) == 0) {
#pragma unroll
        for (int j = 0; j < PER / V; ++j) {
            const uint4 u = ((const uint4 *)base)[j];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (XD == MI_X_BF16) {
                    l[8 * j + 2 * i] = __uint_as_float(w[i] << 16);
                    l[8 * j + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                } else {
                    l[4 * j + i] = __uint_as_float(w[i]);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = j < n ? gate_load<XD>(base, j) : -INFINITY;
}

// 1 / (the sum of e^(l - m) over the row), m the row's maximum: 0 for a row without an expert.
template <int LPR, int PER>
__device__ __forceinline__ float softmax32(const float (&l)[PER], float &m) {
    m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) m = fmaxf(m, l[j]);
    m = over_row<LPR>(m, [](float a, float b) { return fmaxf(a, b); });
    if (m == -INFINITY) {
        m = 0.0f;                                // (e^(-inf) = 0 for each)
        float any = 0.0f;                        // NaN where all are NaN or -inf and one is NaN
#pragma unroll
        for (int j = 0; j < PER; ++j) any += l[j] != l[j] ? l[j] : 0.0f;
        return over_row<LPR>(any, [](float a, float b) { return a + b; });
    }
    float z = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) z += expf(l[j] - m);
    return 1.0f / over_row<LPR>(z, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ float add(float a, float b) { return a + b; }

template <int XD, int LPR, int PER>
__global__ void __launch_bounds__(256) moe_gate_kernel(GateArgs p) {
    const GateLane<LPR> at(p);
    if (at.row >= p.T) return;                   // a row's lanes leave together
    const int lane = at.lane;
    float l[PER];
    gate_logits<XD, PER>(p, at.row, at.id0, at.n, l);
    double key[PER];
    float m = 0.0f, iz = 0.0f;                   // of a softmax
    if (p.scores == MI_GATE_SOFTMAX) iz = softmax32<LPR, PER>(l, m);
    const bool soft = p.scores == MI_GATE_SOFTMAX;
    if (p.bias || p.n_group > 1) {
        double c[PER];
        if (soft) {
            double z = 0.0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                c[j] = exp_neg((double)l[j] - (double)m);
                z += c[j];
            }
            z = reciprocal(over_row<LPR>(z, [](double a, double b) { return a + b; }));
#pragma unroll
            for (int j = 0; j < PER; ++j) c[j] *= z;
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) c[j] = sigmoid64((double)l[j]);
        }
        if (p.bias) {
            const float *b = p.bias + at.id0;
            if (__ballot(at.n != PER || ((uintptr_t)b & 15)) == 0) {
#pragma unroll
                for (int j = 0; j < PER; j += 4) {
                    const float4 u = *(const float4 *)(b + j);
                    c[j] += (double)u.x, c[j + 1] += (double)u.y, c[j + 2] += (double)u.z, c[j + 3] += (double)u.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j) c[j] += j < at.n ? (double)b[j] : 0.0;
            }
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            key[j] = gate_key(c[j], min(at.id0 + j, kGateMaxE - 1), l[j] == -INFINITY || c[j] == -INFINITY);
        }
    }
    if (p.n_group > 1) {
        // the lane's two largest, then its group's, by exchanges with the lanes of the group
        double a = key[0], b = __builtin_bit_cast(double, make_uint2(0u, kGateNone));
#pragma unroll
        for (int j = 1; j < PER; ++j) {
            const double lo = a < key[j] ? a : key[j];
            a = key_max(a, key[j]);
            b = key_max(b, lo);
        }
        const int lanes = LPR / p.n_group;
        for (int d = 1; d < lanes; d <<= 1) {
            const double oa = __shfl_xor(a, d, 64), ob = __shfl_xor(b, d, 64);
            const double lo = a < oa ? a : oa;
            a = key_max(a, oa);
            b = key_max(key_max(b, ob), lo);
        }
        // the groups' places: a group stays if fewer than topk_group are better
        double g = without_id(a);
        if (p.group_top == 2 && !gate_out(b)) g += without_id(b);
        g = gate_key(g, at.group, gate_out(a));
        int better = 0;
        for (int q = 0; q < p.n_group; ++q) {
            const double o = __shfl(g, (threadIdx.x & 63) / LPR * LPR + q * lanes, 64);
            better += o > g || (gate_out(g) && (!gate_out(o) || q < at.group));
        }
        const bool drop = better >= p.topk_group;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (!p.bias) key[j] = gate_key((double)l[j], min(at.id0 + j, kGateMaxE - 1), l[j] == -INFINITY);
            key[j] = gate_drop(key[j], drop);
        }
    } else if (!p.bias) {
#pragma unroll
        for (int j = 0; j < PER; ++j) key[j] = gate_key((double)l[j], min(at.id0 + j, kGateMaxE - 1), l[j] == -INFINITY);
    }

    int id[2] = {-1, -1};                        // of slots lane and 16 + lane (lane % 16)
    for (int r = 0; r < p.k; ++r) {
        double best = key[0];
#pragma unroll
        for (int j = 1; j < PER - 1; ++j) best = key_max(best, key[j]);
        best = key_max_then_rotate(best, key[PER - 1]);
        best = over_row<LPR>(best, key_max_then_rotate);
        const int e = gate_id(best);
        if ((lane & 15) == (r & 15)) id[r >> 4] = e;
#pragma unroll
        for (int j = 0; j < PER; ++j) key[j] = gate_drop(key[j], key[j] == best);
    }
    // a slot's score from its logit again, its weight from the sum over the slots
    float s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float x = id[h] >= 0 ? gate_load<XD>(p.logits, (size_t)at.row * p.stride + id[h]) : 0.0f;
        s[h] = id[h] < 0 ? 0.0f : soft ? expf(x - m) * iz : sigmoid32(x);
    }
    float sum = s[0] + s[1];
    sum = over_row<16>(sum, add);                // (every 16 lanes hold all slots)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = 16 * h + lane;
        if (lane >= 16 || r >= p.k) continue;
        p.idx[(size_t)at.row * p.k + r] = id[h];
        p.w[(size_t)at.row * p.k + r] = (p.norm ? s[h] / (sum + 1e-20f) : s[h]) * p.scaling;
    }
}

// With S = sum of the slots' s, A = sum of dw s (times scaling): ds = dw scaling, or renormalised (dw scaling - A / S') / S',
// S' = S + 1e-20; then dl = ds s (1 - s) (sigmoid) or s (ds - sum ds s) over all experts (softmax).
template <int XD, int LPR, int PER>
__global__ void __launch_bounds__(256) moe_gate_grad_kernel(GateArgs p) {
    __shared__ float row_dl[256 / LPR][LPR * PER];
    const GateLane<LPR> at(p);
    const int lane = at.lane;
    const bool live = at.row < p.T, soft = p.scores == MI_GATE_SOFTMAX;
    const int row = min(at.row, p.T - 1);
    float l[PER], m = 0.0f, iz = 0.0f;
    if (soft) {
        gate_logits<XD, PER>(p, row, at.id0, at.n, l);
        iz = softmax32<LPR, PER>(l, m);
    }
    int id[2];
    float s[2], f[2], g[2], sum = 0.0f, a = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = 16 * h + (lane & 15);
        id[h] = r < p.k ? p.idx[(size_t)row * p.k + r] : -1;
        if (id[h] >= p.E) id[h] = -1;
        const float x = id[h] >= 0 ? gate_load<XD>(p.logits, (size_t)row * p.stride + id[h]) : 0.0f;
        s[h] = id[h] < 0 ? 0.0f : soft ? expf(x - m) * iz : sigmoid32(x);
        f[h] = soft ? 1.0f : sigmoid32(-x);
        g[h] = id[h] < 0 ? 0.0f : p.w[(size_t)row * p.k + r] * p.scaling;
        sum += s[h];
        a = fmaf(g[h], s[h], a);
    }
    sum = over_row<16>(sum, add) + 1e-20f;
    a = over_row<16>(a, add);
    if (p.norm) {
        const float mean = a / sum;
#pragma unroll
        for (int h = 0; h < 2; ++h) g[h] = (g[h] - mean) / sum;
        a = mean * (1e-20f / sum);               // sum of ds s: (A - A S / S') / S'
    }
    float *dl = row_dl[threadIdx.x / LPR];
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (j < at.n) dl[at.id0 + j] = soft ? -a * (expf(l[j] - m) * iz) : 0.0f;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (lane < 16 && id[h] >= 0) dl[id[h]] = s[h] * f[h] * (soft ? g[h] - a : g[h]);
    __syncthreads();
    if (!live) return;
    for (int e = lane; e < p.E; e += LPR) {
        const size_t o = (size_t)row * p.E + e;
        if constexpr (XD == MI_X_BF16)
            ((uint16_t *)p.dlogits)[o] = (uint16_t)f32_to_bf16_rne(dl[e]);
        else
            ((float *)p.dlogits)[o] = dl[e];
    }
}

// ------------------------------------------------------------------------------------------------ host side
static int gate_check(int dtype, long long stride, int T, int E, int k, int scores, int norm, float scaling) {
    if (dtype != MI_X_BF16 && dtype != MI_X_F32) return MI_ERR_ARG;
    if (T <= 0 || T > kGateMaxT) return MI_ERR_TOKENS;
    if (E <= 0 || E > kGateMaxE || stride < E || stride > (1ll << 40)) return MI_ERR_SHAPE;
    if (k <= 0 || k > kGateMaxK || k > E) return MI_ERR_ARG;
    if ((scores != MI_GATE_SIGMOID && scores != MI_GATE_SOFTMAX) || (norm != 0 && norm != 1) || !isfinite(scaling))
        return MI_ERR_ARG;
    return MI_OK;
}
static bool gate_aligned(const void *logits, int dtype, const void *a, const void *b, const void *c = nullptr) {
    return ((uintptr_t)logits & (dtype == MI_X_BF16 ? 1 : 3)) == 0 && (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0;
}

// f(lanes of a row, experts of a lane): 16 lanes unless that would be more than 16 experts, or groups, for each.
template <class F>
static int gate_shape(int E, int n_group, F f) {
    using std::integral_constant;
    const int size = E / n_group, lanes = n_group <= 16 ? 16 / n_group : 0;
    const int per = lanes ? (size + lanes - 1) / lanes : 1 << 20;
    if (per <= 4) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    if (per <= 8) return f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    if (per <= 16) return f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
    if ((size + 64 / n_group - 1) / (64 / n_group) <= 8) return f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

}  // namespace mi

using namespace mi;

extern "C" int mi_moe_gate(const void *logits, int32_t dtype, int64_t stride, const float *bias, int32_t T, int32_t E,
                           int32_t k, int32_t scores, int32_t n_group, int32_t topk_group, int32_t group_top,
                           int32_t norm_topk, float scaling, int32_t *idx, float *w, void *stream) {
    if (!logits || !idx || !w) return MI_ERR_NULL;
    const int rc = gate_check(dtype, stride, T, E, k, scores, norm_topk, scaling);
    if (rc != MI_OK) return rc;
    if (n_group < 1 || n_group > 32 || (n_group & (n_group - 1)) || E % n_group || topk_group < 1 || topk_group > n_group)
        return MI_ERR_ARG;
    if ((group_top != 1 && group_top != 2) || k > E / n_group * topk_group) return MI_ERR_ARG;
    if (!gate_aligned(logits, dtype, bias, idx, w)) return MI_ERR_ARG;
    const GateArgs p = {logits, stride, bias, T, E, k, scores, n_group, topk_group, group_top, norm_topk, scaling, idx, w, nullptr};
    return gate_shape(E, n_group, [&](auto lanes, auto per) {
        constexpr int L = decltype(lanes)::value, N = decltype(per)::value;
        auto kern = dtype == MI_X_BF16 ? moe_gate_kernel<MI_X_BF16, L, N> : moe_gate_kernel<MI_X_F32, L, N>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(((long long)T * L + 255) / 256)), dim3(256), 0, (hipStream_t)stream, p);
        return hipGetLastError() == hipSuccess ? (int)MI_OK : (int)MI_ERR_LAUNCH;
    });
}

extern "C" int mi_moe_gate_grad(const void *logits, int32_t dtype, int64_t stride, const int32_t *idx, const float *dw,
                                int32_t T, int32_t E, int32_t k, int32_t scores, int32_t norm_topk, float scaling,
                                void *dlogits, void *stream) {
    if (!logits || !idx || !dw || !dlogits) return MI_ERR_NULL;
    const int rc = gate_check(dtype, stride, T, E, k, scores, norm_topk, scaling);
    if (rc != MI_OK) return rc;
    if (!gate_aligned(logits, dtype, idx, dw) || !gate_aligned(dlogits, dtype, nullptr, nullptr)) return MI_ERR_ARG;
    const GateArgs p = {logits, stride, nullptr, T, E, k, scores, 1, 1, 1, norm_topk, scaling, (int32_t *)idx, (float *)dw, dlogits};
    return gate_shape(E, 1, [&](auto lanes, auto per) {
        constexpr int L = decltype(lanes)::value, N = decltype(per)::value;
        auto kern = dtype == MI_X_BF16 ? moe_gate_grad_kernel<MI_X_BF16, L, N> : moe_gate_grad_kernel<MI_X_F32, L, N>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(((long long)T * L + 255) / 256)), dim3(256), 0, (hipStream_t)stream, p);
        return hipGetLastError() == hipSuccess ? (int)MI_OK : (int)MI_ERR_LAUNCH;
    });
}
