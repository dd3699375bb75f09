// The tiled products of linear_gemm.h, one unit per tile (MI_LIN_TILE: weight rows * 1000 + rows).
#include "linear_gemm.h"

namespace mi {

// FAST: for a product of two fast operands only.
template <int TW, int TT, int WM, int WN, int NST, bool FAST = false>
static int lin_launch_tile(LinGemm p, bool slow_a, bool slow_b, hipStream_t st) {
    p.nw = (p.R + TW - 1) / TW;
    p.nb = (p.rows + TT - 1) / TT;
    const long long total = (long long)p.nw * p.nb * p.S, grid = (total + 7) / 8 * 8;
    if (grid >= (1ll << 31) / (64 * WM * WN)) return MI_ERR_TOKENS;
    auto kern = lin_gemm_kernel<TW, TT, WM, WN, NST, false, false>;
    if constexpr (!FAST) {
        if (slow_b) kern = lin_gemm_kernel<TW, TT, WM, WN, NST, true, true>;
        else if (slow_a) kern = lin_gemm_kernel<TW, TT, WM, WN, NST, true, false>;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * WM * WN), 0, st, p);
    return hipGetLastError() == hipSuccess ? MI_OK : MI_ERR_LAUNCH;
}

#if MI_LIN_TILE == 128064
int lin_launch_128_64(LinGemm p, bool sa, bool sb, hipStream_t st) { return lin_launch_tile<128, 64, 2, 2, 3>(p, sa, sb, st); }
#elif MI_LIN_TILE == 128128
int lin_launch_128_128(LinGemm p, bool sa, bool sb, hipStream_t st) { return lin_launch_tile<128, 128, 2, 4, 4>(p, sa, sb, st); }
#elif MI_LIN_TILE == 256128
int lin_launch_256_128(LinGemm p, bool sa, bool sb, hipStream_t st) { return lin_launch_tile<256, 128, 4, 2, 3>(p, sa, sb, st); }
#elif MI_LIN_TILE == 256256
int lin_launch_256_256(LinGemm p, bool sa, bool sb, hipStream_t st) { return lin_launch_tile<256, 256, 2, 4, 2>(p, sa, sb, st); }
#elif MI_LIN_TILE == 192256
int lin_launch_192_256(LinGemm p, bool sa, bool sb, hipStream_t st) {
    return sa || sb ? MI_ERR_ARG : lin_launch_tile<192, 256, 2, 4, 2, true>(p, sa, sb, st);
}
#endif

}  // namespace mi
