// Block-scaled fp8 products (fp8.h) behind the C ABI: rows to e4m3, the dense product, the MLP, the experts' products
// over sorted rows and the whole routed layer.
#include <algorithm>

#include "fp8_gemm.h"
#include "fp8_stream.h"
#include "tuning.h"

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

// A group of 128 columns is 16 lanes of 8 values: its maximum is 4 exchanges, its loads and stores are contiguous.  One
// pass, bound by memory: 4099 rows of 6144 bf16 values in 15 us (76 MB, 5.0 TB/s; a copy reaches 4.9).
// Whole groups of lanes run or return together (the grid's tail), so the exchanges stay within live lanes.  gi: the
// group of this lane, over all rows.
template <int XD>
__device__ __forceinline__ void fp8_quantize_group(const void *__restrict__ x, long long gi, int n, int K,
                                                   long long stride, const int32_t *__restrict__ live,
                                                   uint8_t *__restrict__ q, float *__restrict__ s) {
    const int KB = fp8_groups(K);
    if (gi >= (long long)n * KB) return;
    const int row = (int)(gi / KB), c = (int)(gi - (long long)row * KB);
    if (live && live[row] < 0) return;           // (the same for the group's 16 lanes)
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

template <int XD>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const void *__restrict__ x, int n, int K, long long stride,
                                                           const int32_t *__restrict__ live, uint8_t *__restrict__ q,
                                                           float *__restrict__ s) {
    fp8_quantize_group<XD>(x, ((long long)blockIdx.x * 256 + threadIdx.x) >> 4, n, K, stride, live, q, s);
}

// What the tiled routed layer needs first, in one launch: workgroup 0 gives every slot a row (its expert's blocks of tm
// rows; rows without a slot get token -1), the others quantise the tokens.  Within an expert the rows are dealt out by LDS
// atomics: their order is the run's, but a row's result does not depend on its place, so the layer's bits do not either.
struct Fp8Prepare {
    const void *x;
    uint8_t *xq;
    float *xs;
    const int32_t *idx;         // [T, k]
    int32_t *blk_expert, *n_blocks, *tok_row, *row_slot;
    int T, k, D, E, tm;
};
constexpr int kFp8PrepareThreads = 1024;

template <int XD>
__global__ void __launch_bounds__(kFp8PrepareThreads) fp8_prepare_kernel(Fp8Prepare p) {
    __shared__ int cnt[kMaxExperts], base[kMaxExperts], wsum[kFp8PrepareThreads / 64], total;
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        fp8_quantize_group<XD>(p.x, ((long long)(blockIdx.x - 1) * kFp8PrepareThreads + tid) >> 4, p.T, p.D, p.D, nullptr,
                               p.xq, p.xs);
        return;
    }
    const int S = p.T * p.k;
    cnt[tid] = 0;                                // kMaxExperts == threads
    __syncthreads();
    // eight slots at a time, every load issued before its count; a slot's place in its expert waits in row_slot
    for (int s0 = tid; s0 < S; s0 += 8 * kFp8PrepareThreads) {
        int e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = s0 + j * kFp8PrepareThreads;
            e[j] = s < S ? p.idx[s] : -1;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = s0 + j * kFp8PrepareThreads;
            if (s < S) p.row_slot[s] = e[j] >= 0 && e[j] < p.E ? atomicAdd(&cnt[e[j]], 1) : -1;
        }
    }
    __syncthreads();
    const int n = cnt[tid], nb = (n + p.tm - 1) / p.tm;
    int incl = nb;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d, 64);
        if ((tid & 63) >= d) incl += o;
    }
    if ((tid & 63) == 63) wsum[tid >> 6] = incl;
    __syncthreads();
    for (int w = 0; w < tid >> 6; ++w) incl += wsum[w];
    base[tid] = (incl - nb) * p.tm;
    if (tid == kFp8PrepareThreads - 1) *p.n_blocks = incl;
    for (int b = incl - nb; b < incl; ++b) p.blk_expert[b] = tid;
    if (tid == kFp8PrepareThreads - 1) total = incl;
    __syncthreads();
    for (int r = tid; r < total * p.tm; r += kFp8PrepareThreads) {      // rows behind an expert's last
        const int e = p.blk_expert[r / p.tm];
        if (r - base[e] >= cnt[e]) p.tok_row[r] = -1;
    }
    for (int s0 = tid; s0 < S; s0 += 8 * kFp8PrepareThreads) {
        int e[8], at[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = s0 + j * kFp8PrepareThreads;
            e[j] = s < S ? p.idx[s] : -1;
            at[j] = s < S ? p.row_slot[s] : -1;  // this thread's own store above
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = s0 + j * kFp8PrepareThreads;
            if (at[j] < 0) continue;
            const int row = base[e[j]] + at[j];
            p.row_slot[s] = row;
            p.tok_row[row] = s / p.k;
        }
    }
}
static_assert(kMaxExperts == kFp8PrepareThreads, "one thread per expert");

// The split sums of gate and up added in split order, then h = silu(min(g, L)) * clip(u, -L, L) in f32, quantised as
// above: one wavefront per row and group, two values a lane.
__global__ void __launch_bounds__(64) fp8_swiglu_kernel(const float *__restrict__ g, const float *__restrict__ u, int S,
                                                        int rows, int I, float limit, uint8_t *__restrict__ q,
                                                        float *__restrict__ s) {
    const int row = blockIdx.x, c = blockIdx.y, lane = threadIdx.x;
    const int col = c * kFp8Group + 2 * lane;
    float h0 = 0.0f, h1 = 0.0f;
    if (col < I) {
        float2 gv = {0.f, 0.f}, uv = {0.f, 0.f};
        for (int k = 0; k < S; ++k) {
            const size_t at = ((size_t)k * rows + row) * I + col;
            const float2 a = *(const float2 *)(g + at), b = *(const float2 *)(u + at);
            gv.x += a.x, gv.y += a.y;
            uv.x += b.x, uv.y += b.y;
        }
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

// The split sums of a product, added in split order.
__global__ void __launch_bounds__(256) fp8_reduce_kernel(const float *__restrict__ part, int S, long long n,
                                                         uint16_t *y_bf16, float *y_f32) {
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    float v = part[at];
    for (int k = 1; k < S; ++k) v += part[k * n + at];
    if (y_f32) y_f32[at] = v;
    if (y_bf16) y_bf16[at] = (uint16_t)f32_to_bf16_rne(v);
}

// out[t] = sum_j w[t, j] * y[r(t, j)], f32, in column order: r the slot's sorted row, or (row_slot NULL) the slot itself.
// Four outputs a thread, the rows of eight slots loaded before the first is added (D % 16 == 0).
__global__ void __launch_bounds__(256) fp8_combine_kernel(const float *__restrict__ y, const int32_t *__restrict__ row_slot,
                                                          const int32_t *__restrict__ idx, int E,
                                                          const float *__restrict__ w, int k, int D, float *out_f32,
                                                          uint16_t *out_bf16) {
    const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (c >= D) return;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < k; j0 += 8) {
        float4 v[8];
        float wt[8];
        bool in[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = t * k + min(j0 + j, k - 1), e = idx[s];
            const int r = j0 + j >= k || e < 0 || e >= E ? -1 : row_slot ? row_slot[s] : s;
            // (no branch around the loads: a slot without a row loads row 0 and adds nothing, whatever that holds)
            in[j] = r >= 0;
            wt[j] = w[s];
            v[j] = *(const float4 *)(y + (size_t)max(r, 0) * D + c);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            acc[0] = in[j] ? fmaf(wt[j], v[j].x, acc[0]) : acc[0];
            acc[1] = in[j] ? fmaf(wt[j], v[j].y, acc[1]) : acc[1];
            acc[2] = in[j] ? fmaf(wt[j], v[j].z, acc[2]) : acc[2];
            acc[3] = in[j] ? fmaf(wt[j], v[j].w, acc[3]) : acc[3];
        }
    }
    const size_t at = (size_t)t * D + c;
    if (out_f32) {
        if (((uintptr_t)out_f32 & 15) == 0) {
            *(float4 *)(out_f32 + at) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out_f32[at + j] = acc[j];
        }
    }
    if (out_bf16) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = f32_to_bf16_rne(acc[j]);
        if (((uintptr_t)out_bf16 & 7) == 0) {
            *(uint2 *)(out_bf16 + at) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out_bf16[at + j] = (uint16_t)h[j];
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kFp8MaxCols = 1 << 16;             // K, R: a tile's weight scales in LDS
constexpr int kFp8MaxRows = 1 << 22;             // rows of activations

static bool fp8_cols_ok(int K) { return K > 0 && K % 16 == 0 && K <= kFp8MaxCols; }
static bool fp8_rows_ok(int R) { return R > 0 && R <= kFp8MaxCols; }
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
static bool aligned4(const void *p) { return ((uintptr_t)p & 3) == 0; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static bool fp8_x_dtype_ok(int d) { return d == MI_X_BF16 || d == MI_X_F32 || d == MI_X_FP8; }

// Bytes of n quantised rows of K columns: values, then scales.
static size_t fp8_row_bytes(size_t n, int K) { return up256(n * K) + up256(n * fp8_groups(K) * sizeof(float)); }

static int fp8_launch_quantize(const void *x, int x_dtype, int n, int K, long long stride, const int32_t *live,
                               uint8_t *q, float *s, hipStream_t st) {
    const long long threads = (long long)n * fp8_groups(K) * 16;
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (x_dtype == MI_X_BF16)
        hipLaunchKernelGGL(fp8_quantize_kernel<MI_X_BF16>, grid, dim3(256), 0, st, x, n, K, stride, live, q, s);
    else
        hipLaunchKernelGGL(fp8_quantize_kernel<MI_X_F32>, grid, dim3(256), 0, st, x, n, K, stride, live, q, s);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

constexpr int kFp8Cus = 256;
// Idle workgroups of an XCD that read weights ahead.  6144 x 6144, 40 / 64 / 128 / 300 / 768 rows: 22.9 / 24.7 / 25.4 / 37 /
// 72 us with none, 16.3 / 18.1 / 21.4 / 32.7 / 53 with up to 8 of idle CUs; sharing CUs with the others (where a CU takes two
// workgroups) 40 and 300 rows took 20.5 and 37.5, all idle CUs instead of 8 up to 2 us more.  Nothing is gained or lost where
// the weights are in the last-level cache.
constexpr int kFp8Ahead = 8;

// ---- the tiled product.  Tiles: 256 weight rows (128 where a dense product has few tiles) x tt tokens.
template <int TW, int TT, int WM, int WN, int NST, bool PAIR, bool EXACT = false>
static int fp8_launch_tiled(Fp8Tiled p, hipStream_t st) {
    p.nw = (p.g.R + (PAIR ? TW / 2 : TW) - 1) / (PAIR ? TW / 2 : TW);
    p.nb = (p.g.rows + TT - 1) / TT;
    // ids equal modulo 8 share an XCD and a piece of at most ceil(total / 8) workgroups
    // (one more for each XCD where there may be blocks without a product, to write their zeros)
    const long long total = (long long)p.nb * p.nw * p.S;
    long long grid = (total + 7) / 8 * 8 + (p.g.blk_expert && !p.skip ? 8 : 0);
    // of a dense product, up to kFp8Ahead idle CUs of an XCD
    constexpr int kSlots = kFp8Cus * (163840 / (NST * (128 * (TW + TT) + 256 * WM * WN) + 8 * kFp8MaxGroups + 8));
    static_assert(kSlots == kFp8Cus || kSlots == 2 * kFp8Cus, "workgroups per CU");
    const long long slots = grid < kFp8Cus ? kFp8Cus : kSlots;
    if (!p.g.blk_expert && p.nb <= kFp8Near && grid < slots) p.ahead = std::min(kFp8Ahead, (int)(slots - grid) / 8);
    grid += 8 * p.ahead;
    if (grid >= (1ll << 31) / (64 * WM * WN)) return MI_ERR_TOKENS;
    hipLaunchKernelGGL((fp8_gemm_kernel<TW, TT, WM, WN, NST, PAIR, EXACT>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, st, p);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

constexpr int kFp8ExactRows = 128;               // rows of a dense gate/up product up to which its sums are in f32
template <bool PAIR>
static int fp8_tiled(const Fp8Tiled &p, int tw, int tt, bool exact, hipStream_t st) {
    if constexpr (!PAIR) {
        if (tw == 128) return tt == 64 ? fp8_launch_tiled<128, 64, 2, 2, 3, false>(p, st)
                                       : fp8_launch_tiled<128, 128, 2, 2, 4, false>(p, st);
    }
    switch (tt) {
        case 16: return fp8_launch_tiled<256, 16, 4, 1, 4, PAIR, PAIR>(p, st);
        case 32: return fp8_launch_tiled<256, 32, 4, 1, 4, PAIR, PAIR>(p, st);
        case 64:
            if constexpr (PAIR)
                if (exact) return fp8_launch_tiled<256, 64, 4, 1, 3, true, true>(p, st);
            return fp8_launch_tiled<256, 64, 4, 1, 3, PAIR>(p, st);
        case 128:
            if constexpr (PAIR)
                if (exact) return fp8_launch_tiled<256, 128, 4, 2, 3, true, true>(p, st);
            return fp8_launch_tiled<256, 128, 4, 2, 3, PAIR>(p, st);
        default: return fp8_launch_tiled<256, 256, 2, 4, 2, PAIR>(p, st);
    }
}

// The tile and the splits of K of a dense product of B rows: the pair of least estimated time.  A group of 128 columns of a
// tile takes `one` us in a launch of at most one workgroup per CU and `more` for each round of `slots` workgroups otherwise;
// a split adds a launch and a pass over its partial sums, and only fills CUs of the first round.  The times are those of
// weights from memory, 40 to 4096 rows at 6144 x 6144, 2048 x 6144 and 6144 x 2048 with all tiles and splits: over these 45
// the choice takes 1.1 % more than the best of all on average, 10 % at worst.  (6144 x 6144, 100 / 517 / 1024 / 2048 rows:
// 20.6 us with 128 x 64 in two splits, 36.4 with 128 x 128, 52 with 256 x 128, 86 with 256 x 256; the best of the other
// tiles take 22.1 / 44 / 78 / 126.)
struct Fp8Plan {
    int tw, tt, S;
};
constexpr int kFp8SplitTiles = 512;              // tiles x splits at most

// Floats of split sums that any B up to the given one may need.
static size_t fp8_split_floats(int R, bool pair) {
    const size_t n = (size_t)(R + 127) / 128;    // tiles of 128 outputs per token tile
    return std::max<size_t>(kFp8SplitTiles / n, 1) * 64 * R * (pair ? 2 : 1);
}

// A token tile that the tiled kernels have.
static int fp8_tile_of(int tt) { return tt <= 16 ? 16 : tt <= 32 ? 32 : tt <= 64 ? 64 : tt <= 128 ? 128 : 256; }

static Fp8Plan fp8_plan(int B, int R, int K, bool pair) {
    struct Tile {
        int tw, tt, slots;
        float one, more, ends;             // ends: a tile's start and epilogue, in groups
    };
    static const Tile dense[] = {{128, 64, 2 * kFp8Cus, 0.46f, 1.02f, 1}, {128, 128, kFp8Cus, 0.72f, 0.82f, 1},
                                 {256, 64, kFp8Cus, 0.76f, 0.85f, 1}, {256, 128, kFp8Cus, 1.02f, 1.36f, 1},
                                 {256, 256, kFp8Cus, 1.60f, 1.86f, 4}};
    static const Tile gate_up[] = {{256, 32, kFp8Cus, 0.90f, 0.95f, 1}, {256, 64, kFp8Cus, 0.76f, 0.85f, 1},
                                   {256, 128, kFp8Cus, 1.02f, 1.36f, 1}, {256, 256, kFp8Cus, 1.60f, 1.86f, 4}};
    const Tile *c = pair ? gate_up : dense;
    const int n = pair ? 4 : 5, KB = fp8_groups(K);
    const int tw = tuning(kTuneF8Tw, 0), tt = tuning(kTuneF8Tt, 0), fs = tuning(kTuneF8S, 0);
    Fp8Plan best{c[0].tw, c[0].tt, 1};
    float least = 1e30f;
    for (int i = 0; i < n; ++i) {
        if ((tw && !pair && c[i].tw != tw) || (tt && c[i].tt != tt)) continue;
        const int w = pair ? c[i].tw / 2 : c[i].tw;
        const long long tiles = (long long)((R + w - 1) / w) * ((B + c[i].tt - 1) / c[i].tt);
        for (int S = 1; S <= std::min(8, KB); ++S) {
            const double floats = (double)S * B * R * (pair ? 2 : 1);
            if (S > 1 && (tiles * S > c[i].slots || floats > (double)fp8_split_floats(R, pair))) break;
            if (fs && S != fs) continue;
            const long long n_wg = tiles * S, left = n_wg % c[i].slots;
            const bool light = c[i].slots > kFp8Cus && left <= kFp8Cus;          // the last round has one per CU
            const float step = n_wg <= kFp8Cus ? c[i].one
                                               : n_wg / c[i].slots * c[i].more + (!left ? 0.0f : light ? c[i].one : c[i].more);
            const float us = step * ((KB + S - 1) / S + c[i].ends) + (S > 1 ? 3.0f + (float)(floats * 8 / 3.5e6) : 0.0f);
            if (us < least) least = us, best = Fp8Plan{c[i].tw, c[i].tt, S};
        }
    }
    return best;
}

static int fp8_launch_dense(Fp8Gemm a, float *part, hipStream_t st) {
    const Fp8Plan pl = fp8_plan(a.rows, a.R, a.K, false);
    Fp8Tiled p = {};
    p.g = a;
    p.S = pl.S;
    p.part[0] = part;
    int rc = fp8_tiled<false>(p, pl.tw, pl.tt, false, st);
    if (rc != MI_OK || pl.S == 1) return rc;
    const long long n = (long long)a.rows * a.R;
    hipLaunchKernelGGL(fp8_reduce_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, pl.S, n, a.y_bf16,
                       a.y_f32);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

// gate and up of a dense MLP -> h as e4m3 rows.
static int fp8_launch_dense_pair(Fp8Gemm a, float limit, uint8_t *hq, float *hs, float *part, hipStream_t st) {
    const Fp8Plan pl = fp8_plan(a.rows, a.R, a.K, true);
    Fp8Tiled p = {};
    p.g = a;
    p.S = pl.S;
    p.limit = limit, p.hq = hq, p.hs = hs;
    p.part[0] = part, p.part[1] = part + (size_t)pl.S * a.rows * a.R;
    int rc = fp8_tiled<true>(p, 256, pl.tt, a.rows <= kFp8ExactRows, st);
    if (rc != MI_OK || pl.S == 1) return rc;
    hipLaunchKernelGGL(fp8_swiglu_kernel, dim3(a.rows, fp8_groups(a.R)), dim3(64), 0, st, p.part[0], p.part[1], pl.S,
                       a.rows, a.R, limit, hq, hs);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

// ---- the streaming product
// Rows that the dense streaming kernels take.  6144 x 6144: 24 / 32 bf16 rows streamed 18.0 / 20.1 us, 40 tiled 18.5; an MLP of
// 6144 / 2048: 32 rows streamed 32.5, 33 tiled 34.1.
constexpr int kFp8StreamRows = 32;

template <int XD, int NT, int RW, bool PAIR, bool SLOTS, int W, int U, int OCC>
static int fp8_launch_stream_as(const Fp8Stream &a, hipStream_t st) {
    const dim3 grid((a.R + 16 * RW - 1) / (16 * RW), SLOTS ? a.rows : 1);
    hipLaunchKernelGGL((fp8_stream_kernel<XD, NT, RW, PAIR, SLOTS, W, U, OCC>), grid, dim3(64 * W), 0, st, a);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

// Two row tiles a wavefront halve the reads of x, one gives twice the workgroups: two where that leaves half the CUs a
// workgroup each (6144 x 6144: 1 / 16 / 32 rows take 12.6 / 19.9 / 30.9 us with one, 11.5 / 14.3 / 19.8 with two; 2048
// x 6144: 16 / 32 rows 11.3 / 16.4 with one, 13.5 / 19.4 with two).
template <int XD, bool PAIR>
static int fp8_stream_dense_as(const Fp8Stream &a, hipStream_t st) {
    constexpr int U = XD == MI_X_F32 ? 1 : 2;
    if (a.R / 32 >= kFp8Cus / 2)
        return a.rows > 16 ? fp8_launch_stream_as<XD, 2, 2, PAIR, false, 4, U, 2>(a, st)
                           : fp8_launch_stream_as<XD, 1, 2, PAIR, false, 4, 2, PAIR ? 2 : 3>(a, st);
    return a.rows > 16 ? fp8_launch_stream_as<XD, 2, 1, PAIR, false, 4, U, 2>(a, st)
                       : fp8_launch_stream_as<XD, 1, 1, PAIR, false, 4, XD == MI_X_F32 ? 2 : 3, 3>(a, st);
}

template <bool PAIR>
static int fp8_stream_dense(const Fp8Stream &a, int xd, hipStream_t st) {
    return xd == MI_X_BF16 ? fp8_stream_dense_as<MI_X_BF16, PAIR>(a, st)
         : xd == MI_X_F32 ? fp8_stream_dense_as<MI_X_F32, PAIR>(a, st) : fp8_stream_dense_as<MI_X_FP8, PAIR>(a, st);
}

// Of the routed layer, more row tiles a wavefront where that leaves enough workgroups: the rows that a workgroup quantises
// serve them all.  Whole calls at 6144 / 2048: 8 slots 68 us with one row tile of gate and up and four of down, 65 with two
// and four, 73 with one and two; 2 slots 25, 30 and 26.
static int fp8_stream_gate_up(const Fp8Stream &a, int xd, hipStream_t st) {
    const bool two = (long long)(a.R / 32) * a.rows >= kFp8Cus;
    if (xd == MI_X_F32)
        return two ? fp8_launch_stream_as<MI_X_F32, 1, 2, true, true, 4, 1, 2>(a, st)
                   : fp8_launch_stream_as<MI_X_F32, 1, 1, true, true, 4, 2, 3>(a, st);
    return two ? fp8_launch_stream_as<MI_X_BF16, 1, 2, true, true, 4, 2, 2>(a, st)
               : fp8_launch_stream_as<MI_X_BF16, 1, 1, true, true, 4, 3, 3>(a, st);
}
static int fp8_stream_down(const Fp8Stream &a, hipStream_t st) {
    return (long long)(a.R / 64) * a.rows >= kFp8Cus / 2
               ? fp8_launch_stream_as<MI_X_F32, 1, 4, false, true, 4, 1, 3>(a, st)
               : fp8_launch_stream_as<MI_X_F32, 1, 2, false, true, 4, 2, 3>(a, st);
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
    return fp8_launch_quantize(x, x_dtype, n, K, K, a.live, q, s, st);
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
    if ((long long)n * fp8_groups(K) >= (1ll << 28)) return MI_ERR_TOKENS;         // 16 threads each: a grid's 2^32
    if (x_stride < K || x_stride % 8 || x_stride > (1ll << 40)) return MI_ERR_ARG;
    if (!aligned16(x) || !aligned16(q) || !aligned4(s)) return MI_ERR_ARG;
    return fp8_launch_quantize(x, x_dtype, n, K, x_stride, nullptr, q, s, (hipStream_t)stream);
}

extern "C" size_t mi_fp8_project_workspace(int32_t B, int32_t n_in, int32_t n_out) {
    if (B <= 0 || B > kFp8MaxRows || !fp8_cols_ok(n_in) || !fp8_rows_ok(n_out) || (long long)B * n_in >= (1ll << 31))
        return 0;
    return B <= kFp8StreamRows ? 0 : fp8_row_bytes(B, n_in) + up256(fp8_split_floats(n_out, false) * sizeof(float));
}

extern "C" int mi_fp8_project(const void *x, int32_t x_dtype, const float *xs, int32_t B, const uint8_t *wq,
                              const float *ws, int32_t n_in, int32_t n_out, uint16_t *y_bf16, float *y_f32,
                              void *workspace, size_t workspace_bytes, void *stream) {
    int rc = fp8_check_x(x, x_dtype, xs, B, n_in);
    if (rc == MI_OK) rc = fp8_check_w(wq, ws, 1, n_out, n_in);
    if (rc != MI_OK) return rc;
    if (!y_bf16 && !y_f32) return MI_ERR_NULL;
    if (!fp8_y_ok(y_bf16, y_f32)) return MI_ERR_ARG;
    const size_t need = mi_fp8_project_workspace(B, n_in, n_out);
    if (need && (!workspace || workspace_bytes < need)) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (B <= kFp8StreamRows) {
        Fp8Stream f = {};
        f.x = x, f.xs = xs;
        f.wq[0] = wq, f.ws[0] = ws;
        f.rows = B;
        f.E = 1, f.R = n_out, f.K = n_in;
        f.y_bf16 = y_bf16, f.y_f32 = y_f32;
        return fp8_stream_dense<false>(f, x_dtype, st);
    }
    Fp8Cut c{(uint8_t *)workspace};
    Fp8Gemm a = {};
    rc = fp8_rows_of(x, x_dtype, xs, B, n_in, c, a, st);
    if (rc != MI_OK) return rc;
    a.wq[0] = wq, a.ws[0] = ws;
    a.x_rows = a.rows = B;
    a.E = 1, a.R = n_out, a.K = n_in;
    a.y_bf16 = y_bf16, a.y_f32 = y_f32;
    return fp8_launch_dense(a, c.take<float>(fp8_split_floats(n_out, false)), st);
}

extern "C" size_t mi_fp8_mlp_workspace(int32_t B, int32_t D, int32_t I) {
    if (B <= 0 || B > kFp8MaxRows || !fp8_cols_ok(D) || !fp8_cols_ok(I) || (long long)B * std::max(D, I) >= (1ll << 31))
        return 0;
    const size_t few = up256((size_t)std::min(B, kFp8StreamRows) * I * sizeof(float));
    if (B <= kFp8StreamRows) return few;
    return std::max(few, fp8_row_bytes(B, D) + fp8_row_bytes(B, I) +
                             up256(std::max(fp8_split_floats(I, true), fp8_split_floats(D, false)) * sizeof(float)));
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
    if (B <= kFp8StreamRows) {
        float *h = c.take<float>((size_t)B * I);
        Fp8Stream f = {};
        f.x = x, f.xs = xs;
        f.wq[0] = gate_q, f.ws[0] = gate_s, f.wq[1] = up_q, f.ws[1] = up_s;
        f.rows = B;
        f.E = 1, f.R = I, f.K = D;
        f.limit = limit;
        f.y_f32 = h;
        if ((rc = fp8_stream_dense<true>(f, x_dtype, st)) != MI_OK) return rc;
        f.x = h, f.xs = nullptr;
        f.wq[0] = down_q, f.ws[0] = down_s;
        f.R = D, f.K = I;
        f.y_bf16 = y_bf16, f.y_f32 = y_f32;
        return fp8_stream_dense<false>(f, MI_X_F32, st);
    }
    Fp8Gemm a = {};
    rc = fp8_rows_of(x, x_dtype, xs, B, D, c, a, st);
    if (rc != MI_OK) return rc;
    uint8_t *hq = c.take<uint8_t>((size_t)B * I);
    float *hs = c.take<float>((size_t)B * fp8_groups(I));
    float *part = c.take<float>(std::max(fp8_split_floats(I, true), fp8_split_floats(D, false)));
    a.x_rows = a.rows = B;
    a.E = 1, a.R = I, a.K = D;
    a.wq[0] = gate_q, a.ws[0] = gate_s, a.wq[1] = up_q, a.ws[1] = up_s;
    if ((rc = fp8_launch_dense_pair(a, limit, hq, hs, part, st)) != MI_OK) return rc;
    a.xq = hq, a.xs = hs;
    a.R = D, a.K = I;
    a.wq[0] = down_q, a.ws[0] = down_s, a.y_bf16 = y_bf16, a.y_f32 = y_f32;
    return fp8_launch_dense(a, part, st);
}

extern "C" size_t mi_fp8_grouped_workspace(int32_t rows, int32_t K, int32_t R) {
    if (rows <= 0 || rows > kFp8MaxRows || !fp8_cols_ok(K) || !fp8_rows_ok(R) || (long long)rows * K >= (1ll << 31))
        return 0;
    return fp8_row_bytes(rows, K);
}

extern "C" int mi_fp8_grouped(const void *x, int32_t x_dtype, const float *xs, int32_t n_blk, int32_t tm,
                              const int32_t *blk_expert, const int32_t *n_blocks, const int32_t *tok_row,
                              const uint8_t *wq, const float *ws, int32_t E, int32_t K, int32_t R, uint16_t *y_bf16,
                              float *y_f32, void *workspace,
                              size_t workspace_bytes, void *stream) {
    if (tm != 16 && tm != 32 && tm != 64 && tm != 128) return MI_ERR_ARG;
    if (n_blk <= 0 || n_blk > kFp8MaxRows / tm) return MI_ERR_TOKENS;
    const int rows = n_blk * tm;
    int rc = fp8_check_x(x, x_dtype, xs, rows, K);
    if (rc == MI_OK) rc = fp8_check_w(wq, ws, E, R, K);
    if (rc != MI_OK) return rc;
    if (!blk_expert || !n_blocks || (!y_bf16 && !y_f32)) return MI_ERR_NULL;
    if (!aligned4(blk_expert) || !aligned4(n_blocks) || !aligned4(tok_row) || !fp8_y_ok(y_bf16, y_f32)) return MI_ERR_ARG;
    if (!workspace || workspace_bytes < mi_fp8_grouped_workspace(rows, K, R)) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    Fp8Cut c{(uint8_t *)workspace};
    Fp8Gemm a = {};
    a.live = tok_row;
    rc = fp8_rows_of(x, x_dtype, xs, rows, K, c, a, st);
    if (rc != MI_OK) return rc;
    a.wq[0] = wq, a.ws[0] = ws;
    a.blk_expert = blk_expert, a.n_blocks = n_blocks;
    a.x_rows = a.rows = rows;
    a.tm = tm;
    a.E = E, a.R = R, a.K = K;
    a.y_bf16 = y_bf16, a.y_f32 = y_f32;
    Fp8Tiled p = {};
    p.g = a;
    p.S = 1;
    return fp8_tiled<false>(p, 256, tm, false, st);
}

namespace mi {

// A call of a few slots streams each expert's weights, without a plan (6144 / 2048, one and two tokens in 8 slots each: 65
// and 113 us, sorted 78 and 124; 12 slots 87 to 90 and 98 to 105).  A larger one sorts its slots by expert and takes the
// tiled product, its blocks the smaller the fewer rows an expert has (64 experts, top-8, 48 / 96 / 200 / 512 / 1999 tokens:
// 443 / 463 / 500 / 585 / 1170 us with 16 / 32 / 64 / 128 / 256 rows; half the rows 6 to 20 % more from 96 tokens on, twice
// as many 2 to 14 % more).
constexpr int kFp8StreamSlots = kFp8TileSlots;
static bool fp8_moe_streams(int S) { return S <= std::min(tuning(kTuneF8Stream, kFp8StreamSlots), kFp8TileSlots); }
static int fp8_moe_tile(int S, int E) {
    const int per = S / E;
    return fp8_tile_of(tuning(kTuneF8Tm, per <= 8 ? 16 : per <= 18 ? 32 : per <= 40 ? 64 : per <= 96 ? 128 : 256));
}

struct Fp8MoeCut {
    int rows, blocks, tm;
    uint8_t *xq, *hq;
    float *xs, *hs, *h, *y;
    int32_t *blk_expert, *n_blocks, *tok_row, *row_slot;
    size_t bytes;
};

static Fp8MoeCut fp8_moe_cut_stream(uint8_t *base, int S, int D, int I) {
    Fp8MoeCut m = {};
    Fp8Cut c{base};
    m.h = c.take<float>((size_t)S * I);
    m.y = c.take<float>((size_t)S * D);
    m.bytes = c.used;
    return m;
}

static Fp8MoeCut fp8_moe_cut(uint8_t *base, int T, int k, int E, int D, int I) {
    Fp8MoeCut m = {};
    const int S = T * k;
    m.tm = fp8_moe_tile(S, E);
    m.blocks = (S + m.tm - 1) / m.tm + E;
    m.rows = m.blocks * m.tm;
    Fp8Cut c{base};
    m.xq = c.take<uint8_t>((size_t)T * D);
    m.xs = c.take<float>((size_t)T * fp8_groups(D));
    m.blk_expert = c.take<int32_t>(m.blocks);
    m.n_blocks = c.take<int32_t>(1);
    m.tok_row = c.take<int32_t>(m.rows);
    m.row_slot = c.take<int32_t>(S);
    m.hq = c.take<uint8_t>((size_t)m.rows * I);
    m.hs = c.take<float>((size_t)m.rows * fp8_groups(I));
    m.y = c.take<float>((size_t)m.rows * D);
    m.bytes = c.used;
    return m;
}

static int fp8_moe_check(int T, int k, int E, int D, int I) {
    if (T <= 0 || k <= 0 || (long long)T * k > kFp8MaxRows || (long long)T * D >= (1ll << 31)) return MI_ERR_TOKENS;
    if (E <= 0 || E > kMaxExperts || !fp8_cols_ok(D) || !fp8_cols_ok(I)) return MI_ERR_SHAPE;
    const long long rows = ((long long)T * k / 256 + 1 + E) * 256;
    return rows * I < (1ll << 31) ? MI_OK : MI_ERR_TOKENS;
}

// Enough for every smaller T too: the streaming form's slots besides the tiled form's rows, which grow with T.
static size_t fp8_moe_bytes(int T, int k, int E, int D, int I) {
    const int S = T * k;
    const size_t few = fp8_moe_cut_stream(nullptr, std::min(S, kFp8TileSlots), D, I).bytes;
    return fp8_moe_streams(S) ? few : std::max(few, fp8_moe_cut(nullptr, T, k, E, D, I).bytes);
}

}  // namespace mi

extern "C" size_t mi_fp8_moe_workspace(int32_t T, int32_t k, int32_t E, int32_t D, int32_t I) {
    return fp8_moe_check(T, k, E, D, I) == MI_OK ? fp8_moe_bytes(T, k, E, D, I) : 0;
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
    if (!workspace || workspace_bytes < fp8_moe_bytes(T, k, E, D, I)) return MI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MI_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    const int S = T * k;
    Fp8MoeCut m;
    if (fp8_moe_streams(S)) {
        m = fp8_moe_cut_stream((uint8_t *)workspace, S, D, I);
        Fp8Stream f = {};
        f.x = x;
        f.wq[0] = gate_q, f.ws[0] = gate_s, f.wq[1] = up_q, f.ws[1] = up_s;
        f.idx = idx;
        f.rows = S, f.div = k;
        f.E = E, f.R = I, f.K = D;
        f.limit = limit;
        f.y_f32 = m.h;
        rc = fp8_stream_gate_up(f, x_dtype, st);
        if (rc != MI_OK) return rc;
        f.x = m.h;
        f.wq[0] = down_q, f.ws[0] = down_s;
        f.div = 1;
        f.R = D, f.K = I;
        f.y_f32 = m.y;
        if ((rc = fp8_stream_down(f, st)) != MI_OK) return rc;
    } else {
        m = fp8_moe_cut((uint8_t *)workspace, T, k, E, D, I);
        const Fp8Prepare f = {x, m.xq, m.xs, idx, m.blk_expert, m.n_blocks, m.tok_row, m.row_slot, T, k, D, E, m.tm};
        const dim3 grid((unsigned)(1 + ((long long)T * fp8_groups(D) * 16 + kFp8PrepareThreads - 1) / kFp8PrepareThreads));
        if (x_dtype == MI_X_BF16)
            hipLaunchKernelGGL(fp8_prepare_kernel<MI_X_BF16>, grid, dim3(kFp8PrepareThreads), 0, st, f);
        else
            hipLaunchKernelGGL(fp8_prepare_kernel<MI_X_F32>, grid, dim3(kFp8PrepareThreads), 0, st, f);
        if (hipGetLastError() != hipSuccess) return MI_ERR_LAUNCH;
        Fp8Tiled p = {};
        Fp8Gemm &a = p.g;
        a.xq = m.xq, a.xs = m.xs;
        a.tok_row = a.live = m.tok_row, a.blk_expert = m.blk_expert, a.n_blocks = m.n_blocks;
        a.x_rows = T, a.rows = m.rows, a.tm = m.tm;
        a.E = E, a.R = I, a.K = D;
        a.wq[0] = gate_q, a.ws[0] = gate_s, a.wq[1] = up_q, a.ws[1] = up_s;
        p.S = 1;
        p.skip = 1;
        p.limit = limit, p.hq = m.hq, p.hs = m.hs;
        if ((rc = fp8_tiled<true>(p, 256, m.tm, true, st)) != MI_OK) return rc;
        a.xq = m.hq, a.xs = m.hs;
        a.tok_row = nullptr, a.x_rows = m.rows;
        a.R = D, a.K = I;
        a.wq[0] = down_q, a.ws[0] = down_s, a.y_f32 = m.y;
        if ((rc = fp8_tiled<false>(p, 256, m.tm, false, st)) != MI_OK) return rc;
    }
    hipLaunchKernelGGL(fp8_combine_kernel, dim3(T, (D + 1023) / 1024), dim3(256), 0, st, m.y, m.row_slot, idx, E, w, k, D,
                       out_f32, out_bf16);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}
