"""GPU: rows to e4m3 past 2^31 values and past 2^32 bytes of input: the last rows are those of a smaller call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,K,dtype", [((1 << 19) + 5, 4112, torch.bfloat16), ((1 << 22) - 3, 528, torch.float32)])
def test_quantize_past_32_bits(pkg, gpu, n, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.empty((n, K), dtype=dtype, device="cuda")
    for r in range(0, n, 1 << 18):
        m = min(1 << 18, n - r)
        x[r:r + m] = torch.randn((m, K), device="cuda", generator=g)
    q, s = pkg.fp8_quantize(x)
    for r in (0, (1 << 31) // K - 1, n // 2, n - 300):
        wq, ws = pkg.fp8_quantize(x[r:r + 300].clone())
        assert torch.equal(q[r:r + 300].view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s[r:r + 300], ws)
