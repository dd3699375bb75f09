"""GPU: forced tiles and splits of bf16_linear are those that run: more splits than a call can have are as many as it can."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
TILES = [(128, 64), (128, 128), (256, 128), (256, 256), (192, 256)]


def _rand(shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g).to(BF16)


@pytest.mark.parametrize("tw,tt", TILES)
def test_more_splits_than_columns(pkg, gpu, tw, tt):
    """136 columns are three pieces of 64: 8 splits are 3, whose sums have other last bits than one."""
    x, leaf = _rand((530, 136), 1), pkg.Bf16Leaf(_rand((772, 136), 2))
    got = {}
    for S in (1, 3, 8):
        with pkg.tuning(LIN_TW=tw, LIN_TT=tt, LIN_S=S, LIN_STREAM=0):
            got[S] = pkg.bf16_linear(x, leaf, dtype=F32)
    assert torch.equal(got[8], got[3]) and not torch.equal(got[3], got[1])


@pytest.mark.parametrize("tw,tt", TILES[:4])
def test_more_splits_than_the_gradients_have(pkg, gpu, tw, tt):
    """dx sums over 448 outputs (7 pieces), dw over 448 rows."""
    x, w, gy = _rand((448, 712), 1), _rand((448, 712), 2), _rand((448, 448), 3)
    got = {}
    for S in (7, 8):
        with pkg.tuning(LIN_TW=tw, LIN_TT=tt, LIN_S=S, LIN_STREAM=0):
            a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
            got[S] = torch.autograd.grad(pkg.bf16_linear(a, pkg.Bf16Leaf(b)), [a, b], gy)
    assert all(torch.equal(p, q) for p, q in zip(got[7], got[8]))


def test_forced_tiles_stay(pkg, gpu):
    """2000 x 1024 x 2000 fills the CUs: one split of the small tiles, two of the others (the workspace).  The tiles' workgroups
    stand on different XCDs, which start at different columns, so that no two tiles give the same last bits."""
    x, leaf = _rand((2000, 1024), 1), pkg.Bf16Leaf(_rand((2000, 1024), 2))

    def run(tw, tt, S):
        with pkg.tuning(LIN_TW=tw, LIN_TT=tt, LIN_S=S):
            return pkg.bf16_linear(x, leaf, dtype=F32)

    got = [run(tw, tt, 8) for tw, tt in TILES]
    for (tw, tt), y in zip(TILES, got):
        assert torch.equal(y, run(tw, tt, 1 if tw == 128 else 2)), (tw, tt)
    assert not any(torch.equal(got[a], got[b]) for a in range(5) for b in range(a))
