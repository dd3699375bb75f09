"""GPU: bf16_linear's activations relative to their own size, where they are small."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _grid(n):
    """z from -12.5 to 8 as the exact sum of two bf16 values (16 bits of it), and rows of 64 columns that hold them."""
    z = torch.linspace(-12.5, 8.0, n, dtype=torch.float64, device="cuda")
    x = torch.zeros((n, 64), dtype=BF16, device="cuda")
    x[:, 0] = z.to(BF16)
    x[:, 1] = (z - x[:, 0].double()).to(BF16)
    return x, x[:, 0].double() + x[:, 1].double()


def _want(z, act):
    """The activation in 64 bits without a difference in its tail, and how many roundings f32 may be off."""
    if act == "silu":
        # e^-z: its argument's rounding and the factor's, 1.5 |z|; the sum, the reciprocal, e^x and the product
        return z * torch.sigmoid(z), 16 + 2 * z.abs()
    if act == "gelu":
        # e^(-z^2 / 2): three roundings of at most half a step of z^2 / 2, one of them the factor's (1.25 z^2); the fit 7.2,
        # its reciprocal 2, e^x 2, three products, and 1 - tail
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0)), 20 + 1.5 * z * z
    u = 2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
    # e^-u: four roundings of u and two of the argument; the rest as silu
    return z * torch.sigmoid(u), 16 + 6 * u.abs()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("n,n_out", [(16, 8), (16, 5), (4001, 8), (4001, 5), (700, 1000)])
def test_tails(pkg, gpu, act, n, n_out):
    """Streamed and tiled calls, whole groups of outputs and single ones."""
    x, z = _grid(n)
    w = torch.zeros((n_out, 64), dtype=BF16, device="cuda")
    w[:, :2] = 1.0
    want, steps = _want(z, act)
    for dtype, half in ((F32, 2.0 ** -24), (BF16, 2.0 ** -8)):
        y = pkg.bf16_linear(x, pkg.Bf16Leaf(w), act=act, dtype=dtype).double()
        err = 2.0 ** -24 * steps * want.abs()
        # (the least normal f32 times |z|: what the exponential and the reciprocal may flush)
        bad = (y - want[:, None]).abs() - (err * (1 + half) + half * want.abs() + 1e-36)[:, None]
        assert bool((bad <= 0).all()), (act, dtype, float(z[bad.amax(1).argmax()]), float((y[:, 0] / want).sub(1).abs().max()))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_tails_of_split_sums(pkg, gpu, act):
    x, z = _grid(300)
    x = torch.cat([x, torch.zeros((300, 512 - 64), dtype=BF16, device="cuda")], 1)
    w = torch.zeros((40, 512), dtype=BF16, device="cuda")
    w[:, :2] = 1.0
    want, steps = _want(z, act)
    with pkg.tuning(LIN_S=4, LIN_STREAM=0):
        y = pkg.bf16_linear(x, pkg.Bf16Leaf(w), act=act, dtype=F32).double()
    assert bool(((y - want[:, None]).abs() <= (2.0 ** -24 * (1 + steps) * want.abs() + 1e-36)[:, None]).all())
