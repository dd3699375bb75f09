"""GPU: the block-scaled fp8 products over the whole range of f32 scales.  A group's sum times its two scales is what
counts: their product alone may leave f32 (2^120 times 2^8) where the scaled sum is an ordinary number or 0."""
import numpy as np
import pytest
import torch

from oracle import fp8 as of8

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
LIMIT = 4.0
ROWS = [1, 9, 20, 40, 130, 300]          # streamed with one and two token tiles, tiled with and without splits


def _leaf(pkg, bits, s):
    return pkg.Fp8Leaf(torch.from_numpy(bits).cuda().view(F8), torch.from_numpy(np.ascontiguousarray(s)).cuda())


def _forms(pkg, x, leaf):
    """The f32 output of every form of activations that x has."""
    outs = [pkg.fp8_project(a, leaf, want_f32=True)[1] for a in (x, x.float(), pkg.fp8_quantize(x))]
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
    return outs[0].double().cpu().numpy()


@pytest.mark.parametrize("B", ROWS)
def test_largest_activations_times_large_scales(pkg, gpu, B):
    """2^127 * (2^-9 * 2^9) = 2^127, beside a group of 2^127 whose weights are 0 with scales up to the largest power."""
    K, R = 400, 300
    x = torch.zeros((B, K), dtype=torch.bfloat16, device="cuda")
    x[:, 133] = 2.0 ** 127
    x[:, 256:384] = -2.0 ** 127
    bits = np.zeros((R, K), np.uint8)
    bits[:, 133] = 0x01                                    # 2^-9
    for top in (2.0 ** 9, 2.0 ** 60, 2.0 ** 127):
        s = np.ones((3, 4), np.float32)
        s[:, 1], s[:, 2] = 2.0 ** 9, top
        assert (_forms(pkg, x, _leaf(pkg, bits, s)) == 2.0 ** 127).all()


@pytest.mark.parametrize("B", ROWS)
def test_products_of_powers_of_two(pkg, gpu, B):
    """x = 2^a in one column, weights 1 with scales 2^b from the smallest f32 to the largest power, another b in every
    block of rows, smaller scales in the other groups: 2^(a + b), exactly, wherever that is a normal f32."""
    K, R = 400, 300
    bits = np.full((R, K), 0x38, np.uint8)                 # 1.0
    for three in ((-149, 0, 127), (-140, 7, 100), (-126, 6, 60), (-100, -26, 8), (-27, -60, 20)):
        b = np.repeat(three, 128)[:R].astype(np.float64)
        s = np.zeros((3, 4), np.float32)
        s[:, 1] = 2.0 ** np.array(three, np.float64)
        s[:, 3] = s[:, 1] * 2.0 ** -4
        leaf = _leaf(pkg, bits, s)
        for a in (-109, -60, -9, 0, 33, 90, 127):
            x = torch.zeros((B, K), dtype=torch.bfloat16, device="cuda")
            x[:, 128 + B % 128] = 2.0 ** a
            keep = (a + b >= -126) & (a + b <= 127)
            got = _forms(pkg, x, leaf)
            assert (got[:, keep] == 2.0 ** (a + b[keep])).all(), (three, a)
            assert (got[:, a + b > 127] == np.inf).all() and (np.abs(got[:, a + b < -126]) <= 2.0 ** -126).all()


@pytest.mark.parametrize("B", ROWS)
def test_blocks_of_rows_far_apart(pkg, gpu, B):
    """Random values, the blocks of rows 2^-90, 1 and 2^70 times as large: within the bound of each."""
    rng = np.random.default_rng(B)
    K, R = 528, 384
    bits, s = of8.random_weights(rng, R, K)
    s *= np.array([2.0 ** -90, 1.0, 2.0 ** 70], np.float32)[:, None]
    x = torch.from_numpy(rng.standard_normal((B, K)).astype(np.float32)).to(torch.bfloat16).cuda()
    want, bound = of8.project(of8.rows_dense(*of8.quantize(x.double().cpu().numpy())), of8.weights_dense(bits, s))
    assert np.all(np.abs(_forms(pkg, x, _leaf(pkg, bits, s)) - want) <= bound)


def _poisoned(rng, raw, x):
    """Weights whose second group of columns is 0 with a scale of 2^90, and activations that are 2^125 there."""
    y = x.clone()
    y[:, 128:256] = 2.0 ** 125
    out = []
    for bits, s in raw:
        bits, s = bits.copy(), s.copy()
        bits[..., 128:256] = 0
        s[..., 1] = 2.0 ** 90
        out.append((bits, s))
    return out, y


def _plain(raw):
    """The same with ordinary scales."""
    out = []
    for bits, s in raw:
        s = s.copy()
        s[..., 1] = 1.0
        out.append((bits, s))
    return out


@pytest.mark.parametrize("B", ROWS)
def test_mlp_powers_of_two_cancel(pkg, gpu, B):
    """Scales of gate and up 2^40 times as large with activations 2^-40 times as large: the same bits; scales of down
    2^70 times as large: 2^70 times the output; a group of zero weights with a large scale adds nothing."""
    rng = np.random.default_rng(B)
    D, I = 528, 400
    raw = [of8.random_weights(rng, R, K, 0.05) for R, K in ((I, D), (I, D), (D, I))]
    x = torch.from_numpy(rng.standard_normal((B, D)).astype(np.float32)).to(torch.bfloat16).cuda()
    call = lambda x, raw: pkg.fp8_mlp(x, *[_leaf(pkg, *r) for r in raw], LIMIT, want_f32=True)[1]
    want = call(x, raw)
    assert (want != 0).any()
    for n in (40, -40):
        up = [(b, s * np.float32(2.0 ** n)) for b, s in raw[:2]]
        assert torch.equal(call(x * 2.0 ** -n, up + raw[2:]), want)
    for n in (70, -70):
        assert torch.equal(call(x, raw[:2] + [(raw[2][0], raw[2][1] * np.float32(2.0 ** n))]), want * 2.0 ** n)
    bad, xp = _poisoned(rng, raw[:2], x)
    x0 = x.clone()
    x0[:, 128:256] = 0.0
    assert torch.equal(call(xp, bad + raw[2:]), call(x0, _plain(bad) + raw[2:]))


@pytest.mark.parametrize("T,tm", [(1, 16), (3, 16), (40, 32), (300, 64), (300, 128)])
def test_experts_with_far_scales(pkg, gpu, T, tm):
    """The experts' products and the routed layer, one expert's scales 2^60 times as large: bits and magnitudes follow,
    and a group of zero weights with a large scale adds nothing."""
    rng = np.random.default_rng(T + tm)
    E, k, D, I = 4, 2, 400, 272
    raw = [of8.random_weights(rng, R, K, 0.05, E) for R, K in ((I, D), (I, D), (D, I))]
    x = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(torch.bfloat16).cuda()
    idx = torch.from_numpy(np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)).cuda()
    w = torch.ones((T, k), device="cuda")
    plan = pkg.ragged_plan(idx, w, E, tm)
    far = raw[0][1].copy()
    far[2] *= np.float32(2.0 ** 60)
    xs = pkg.moe_dispatch(x, plan)
    want = pkg.fp8_grouped(xs, plan, _leaf(pkg, *raw[0]), want_f32=True)[1]
    got = pkg.fp8_grouped(xs, plan, _leaf(pkg, raw[0][0], far), want_f32=True)[1]
    expert = plan["blk_expert"].repeat_interleave(tm)
    assert torch.equal(got, want * torch.where(expert == 2, 2.0 ** 60, 1.0)[:, None])

    call = lambda x, raw: pkg.fp8_moe(*[_leaf(pkg, *r) for r in raw], x, idx, w, LIMIT)[0]
    bad, xp = _poisoned(rng, raw[:2], x)
    x0 = x.clone()
    x0[:, 128:256] = 0.0
    base = call(x0, _plain(bad) + raw[2:])
    assert torch.isfinite(base).all() and (base != 0).any()
    assert torch.equal(call(xp, bad + raw[2:]), base)
    down = (raw[2][0], raw[2][1] * np.float32(2.0 ** 60))
    assert torch.equal(call(x, raw[:2] + [down]), call(x, raw) * 2.0 ** 60)
