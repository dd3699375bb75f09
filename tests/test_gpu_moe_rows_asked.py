"""GPU: the gradients of moe_combine one at a time: what is asked for is the same, bit for bit, as when both are."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k,tm,D", [(1, 4, 2, 16, 8), (6, 4, 2, 16, 64), (130, 16, 5, 40, 520)])
def test_values_of_what_is_asked(pkg, gpu, T, E, k, tm, D, dtype):
    rng = np.random.default_rng(T)
    idx = torch.from_numpy(rng.integers(0, E, (T, k)).astype(np.int32)).cuda()
    w = torch.from_numpy(rng.standard_normal((T, k)).astype(np.float32)).cuda()
    plan = pkg.ragged_plan(idx, w, E, tm)
    y = torch.randn((plan["tok_row"].numel(), D), device="cuda").to(dtype)
    gout = torch.randn((T, D), device="cuda").to(dtype)

    def grads(ask_y, ask_w):
        a, b = y.clone().requires_grad_(ask_y), w.clone().requires_grad_(ask_w)
        out = pkg.moe_combine(a, plan, b)
        return out, dict(zip([n for n, ask in (("y", ask_y), ("w", ask_w)) if ask],
                             torch.autograd.grad(out, [t for t, ask in ((a, ask_y), (b, ask_w)) if ask], gout)))

    out, both = grads(True, True)
    rows = plan["row_slot"].long()
    want_w = (gout.double()[:, None] * y.double()[rows]).sum(-1)
    assert (both["w"].double() - want_w).abs().max() <= (D + 1) * 2.0 ** -24 * float(
        (gout.double()[:, None] * y.double()[rows]).abs().sum(-1).max())
    want_y = torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    want_y[rows.reshape(-1)] = (w.double()[..., None] * gout.double()[:, None]).reshape(-1, D)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0           # one rounding to bf16 of the f32 product
    assert ((both["y"].double() - want_y).abs() <= (half + 2.0 ** -24 * (1 + half)) * want_y.abs()).all()
    for ask in ("y", "w"):
        alone, one = grads(ask == "y", ask == "w")
        assert torch.equal(alone, out) and list(one) == [ask] and torch.equal(one[ask], both[ask])


def test_no_tokens_have_no_plan(pkg, gpu):
    """ragged_plan refuses a call without tokens, and so do the rows that go by a plan of none."""
    idx, w = torch.zeros((0, 2), dtype=torch.int32, device="cuda"), torch.zeros((0, 2), device="cuda")
    with pytest.raises(pkg._lib.MiError):
        pkg.ragged_plan(idx, w, 4, 16)
    plan = {"tok_row": torch.full((64,), -1, dtype=torch.int32, device="cuda"), "row_slot": idx}
    with pytest.raises(pkg._lib.MiError):
        pkg.moe_dispatch(torch.zeros((0, 32), device="cuda"), plan)
    with pytest.raises(pkg._lib.MiError):
        pkg.moe_combine(torch.zeros((64, 32), device="cuda"), plan, w)
