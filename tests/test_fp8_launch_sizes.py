"""CPU: fp8_quantize refuses, before a launch, what a grid of 2^32 threads does not cover."""
import ctypes

P = ctypes.c_void_p


def test_quantize_past_a_grid(pkg):
    call = lambda n, K: pkg._lib.lib().mi_fp8_quantize(P(0x10000), 0, n, K, K, P(0x20000), P(0x30000), None)
    for n, K in ((1 << 22, 8192), (1 << 22, 65536), (1 << 20, 32768)):
        assert call(n, K) == 4, (n, K)                     # MI_ERR_TOKENS
