"""GPU: the block-scaled fp8 products against the 64-bit oracle.  Quantised values and scales have to be equal; f32
outputs within the oracle's bound for f32 sums (oracle.fp8.sum_bound, and mlp's for a value next to a rounding border);
bf16 outputs within that plus one rounding (2^-8 of the value)."""
import numpy as np
import pytest
import torch

from oracle import fp8 as of8

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
LIMIT = 4.0


def _leaf(pkg, bits, s):
    return pkg.Fp8Leaf(torch.from_numpy(bits).cuda().view(F8), torch.from_numpy(s).cuda())


def _acts(rng, n, K, dtype=torch.bfloat16):
    x = rng.standard_normal((n, K)) * np.exp(rng.uniform(-3, 3, (n, 1)))
    x[:, rng.integers(0, K, max(1, K // 100))] *= 20.0
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


def _np(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _close(got, want, bound):
    got = _np(got)
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    assert over.max() <= 0, (float(over.max()), np.unravel_index(over.argmax(), over.shape), float(np.abs(want).max()))


def _check(yb, yf, want, bound):
    """Both outputs; the bf16 one rounds the f32 one."""
    _close(yf, want, bound)
    assert torch.equal(yb, yf.to(torch.bfloat16))


# ------------------------------------------------------------------------------------------------ quantize
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,K", [(1, 16), (1, 128), (3, 144), (5, 6144), (67, 1360), (1000, 592), (2, 65536)])
def test_quantize(pkg, gpu, n, K, dtype):
    x = _acts(np.random.default_rng(n + K), n, K, dtype)
    q, s = pkg.fp8_quantize(x)
    wq, ws = of8.quantize(_np(x))
    assert np.array_equal(_np(s), ws)
    assert np.array_equal(_np(q), wq)


def test_quantize_borders(pkg, gpu):
    """Group maxima on and next to 448 * 2^e, ties, zeros, the smallest and largest values, infinities and NaN."""
    rows = []
    for top in (448.0, 447.0, 449.0, 224.0, 1.75, 1.7578125, 2.0 ** -95, 2.0 ** -120, 0.0, 3.3e38, 2.0 ** -133):
        r = np.zeros(256)
        r[0] = top
        r[1:120] = top * np.linspace(-1, 1, 119)
        r[130] = -top
        rows.append(r)
    ties = np.zeros(256)
    ties[:128] = (of8.VALUES[:128].copy() + np.roll(of8.VALUES[:128], -1)) / 2
    ties[~np.isfinite(ties)] = 0
    ties[0] = 448.0
    rows.append(ties)
    odd = np.ones(256)
    odd[3], odd[4], odd[200] = np.inf, np.nan, -np.inf
    rows.append(odd)
    allnan = np.full(256, np.nan)
    rows.append(allnan)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.from_numpy(np.stack(rows).astype(np.float32)).to(dtype).cuda()
        q, s = pkg.fp8_quantize(x)
        wq, ws = of8.quantize(_np(x))
        assert np.array_equal(_np(s), ws)
        assert np.array_equal(_np(q), wq, equal_nan=True)


def test_quantize_views(pkg, gpu):
    """Strided rows, misaligned views, leading dimensions, an empty tensor, outputs given."""
    x = _acts(np.random.default_rng(5), 12, 640)
    want = pkg.fp8_quantize(x[:, 128:384].contiguous())
    for v in (x[:, 128:384], ):
        got = pkg.fp8_quantize(v)
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    for v in (x[:, 3:259], x[::2, :256], x[:, :512:2]):
        got, w2 = pkg.fp8_quantize(v), pkg.fp8_quantize(v.contiguous().clone())
        assert torch.equal(got[0].view(torch.uint8), w2[0].view(torch.uint8)) and torch.equal(got[1], w2[1])
    q3, s3 = pkg.fp8_quantize(x.view(3, 4, 640))
    q2, s2 = pkg.fp8_quantize(x)
    assert q3.shape == (3, 4, 640) and s3.shape == (3, 4, 5)
    assert torch.equal(q3.view(torch.uint8).view(12, 640), q2.view(torch.uint8)) and torch.equal(s3.view(12, 5), s2)
    q0, s0 = pkg.fp8_quantize(x[:0])
    assert q0.shape == (0, 640) and s0.shape == (0, 5)
    one = x[0].expand(4, 640)
    assert torch.equal(pkg.fp8_quantize(one)[1], s2[:1].expand(4, 5))
    out = torch.full((12, 640), 7, dtype=torch.uint8, device="cuda").view(F8)
    assert pkg.fp8_quantize(x, q=out)[0] is out and torch.equal(out.view(torch.uint8), q2.view(torch.uint8))
    with pytest.raises(ValueError, match="current device"):
        pkg.fp8_quantize(torch.zeros(2, 32))


# ------------------------------------------------------------------------------------------------ project
SHAPES = [(1, 16, 1), (1, 128, 7), (2, 144, 64), (5, 256, 130), (16, 1360, 592), (17, 592, 1360), (33, 272, 200),
          (64, 640, 256), (70, 1360, 129), (129, 768, 384), (300, 1040, 515), (1, 6144, 2048), (9, 6144, 576),
          (48, 4096, 768), (513, 2048, 640), (1100, 768, 1152)]


@pytest.mark.parametrize("B,K,R", SHAPES)
def test_project(pkg, gpu, B, K, R):
    rng = np.random.default_rng(B + K + R)
    bits, s = of8.random_weights(rng, R, K)
    leaf, x = _leaf(pkg, bits, s), _acts(rng, B, K)
    xd = of8.rows_dense(*of8.quantize(_np(x)))
    want, bound = of8.project(xd, of8.weights_dense(bits, s))
    yb, yf = pkg.fp8_project(x, leaf, want_f32=True)
    _check(yb, yf, want, bound)
    pair = pkg.fp8_project(pkg.fp8_quantize(x), leaf, want_f32=True)      # the same values: the same bits
    assert torch.equal(pair[1], yf) and torch.equal(pkg.fp8_project(x, leaf), yb)
    assert torch.equal(pkg.fp8_project(x.float(), leaf, want_f32=True)[1], yf)


@pytest.mark.parametrize("B", [1, 3, 16, 20, 40, 100, 300])
def test_project_rows_end_inside_a_group(pkg, gpu, B):
    """n_in past a whole group: the bytes behind a row (the next row: NaN codes here) add nothing to it; a NaN in a row
    of the activations or of the weights stays in that row or column."""
    rng = np.random.default_rng(B)
    for K, R in ((144, 130), (1040, 48), (16, 20)):
        bits, s = of8.random_weights(rng, R, K)
        bits[1::2] = 0x7f
        x = _acts(rng, B, K)
        if B > 1:
            x[1::2] = float("nan")
        y = _np(pkg.fp8_project(x, _leaf(pkg, bits, s), want_f32=True)[1])
        even = of8.weights_dense(bits[::2], np.repeat(s, 128, 0)[:R][::2][::64][:(R + 127) // 128]) if R <= 128 else None
        assert np.isfinite(y[::2, ::2]).all() and np.isnan(y[:, 1::2]).all()
        if B > 1:
            assert np.isnan(y[1::2]).all()
        if even is not None:
            want, bound = of8.project(of8.rows_dense(*of8.quantize(_np(x)[::2])), even)
            assert np.all(np.abs(y[::2, ::2] - want) <= bound)


@pytest.mark.parametrize("B", [1, 16, 24, 64, 257])
def test_project_extremes(pkg, gpu, B):
    """Zero rows, scales far apart, groups of largest values: sums of 128 * 448^2 and of the smallest subnormals."""
    rng = np.random.default_rng(B)
    K, R = 512, 144
    bits, s = of8.random_weights(rng, R, K)
    bits[:, :128] = 0x7e                                   # 448
    bits[:, 128:256] = 0x01                                # 2^-9
    s[:, 2] = 2.0 ** -60
    s[:, 3] = 2.0 ** 40
    x = torch.ones((B, K), device="cuda")
    x[:, 128:256] = torch.from_numpy(rng.standard_normal((B, 128)).astype(np.float32)).cuda() * 1e-30
    x[:, 256:384] *= 3e30
    x[:, 384:] *= 1e-25
    if B > 3:
        x[3] = 0.0
    want, bound = of8.project(of8.rows_dense(*of8.quantize(_np(x))), of8.weights_dense(bits, s))
    yb, yf = pkg.fp8_project(x, _leaf(pkg, bits, s), want_f32=True)
    _check(yb, yf, want, bound)
    if B > 3:
        assert (yf[3] == 0).all()


TILES = [(128, 64), (128, 128), (256, 64), (256, 128), (256, 256)]


@pytest.mark.parametrize("tw,tt", TILES)
@pytest.mark.parametrize("B,K,R", [(33, 144, 20), (64, 1040, 300), (200, 640, 515), (270, 128, 128), (530, 272, 272)])
def test_project_every_tile(pkg, gpu, tw, tt, B, K, R):
    """Every tile of the tiled product, whole and split along K, at sizes that end inside a tile, a group and a block; row
    counts that fill from one to all of a tile's parts."""
    rng = np.random.default_rng(B + K + tw + tt)
    bits, s = of8.random_weights(rng, R, K)
    leaf, x = _leaf(pkg, bits, s), _acts(rng, B, K)
    want, bound = of8.project(of8.rows_dense(*of8.quantize(_np(x))), of8.weights_dense(bits, s))
    for S in (1, 2, 5, 8):
        with pkg.tuning(F8_TW=tw, F8_TT=tt, F8_S=S):
            yb, yf = pkg.fp8_project(x, leaf, want_f32=True)
            _check(yb, yf, want, bound)
            few = max(33, B - 31)                         # fewer rows of the same tile: the same bits
            assert torch.equal(pkg.fp8_project(x[:few], leaf), yb[:few])


def test_project_outputs_and_views(pkg, gpu):
    """Outputs given, a misaligned and a strided x, no tokens, a kept workspace for a smaller batch, a column slice of
    a larger output left as it was."""
    rng = np.random.default_rng(11)
    K, R = 384, 200
    leaf = _leaf(pkg, *of8.random_weights(rng, R, K))
    x = _acts(rng, 50, K)
    want = pkg.fp8_project(x, leaf, want_f32=True)
    ws = torch.full((pkg._lib.lib().mi_fp8_project_workspace(64, K, R),), 255, dtype=torch.uint8, device="cuda")
    big = torch.full((60, R), 3.0, dtype=torch.bfloat16, device="cuda")
    yf = torch.empty((50, R), device="cuda")
    got = pkg.fp8_project(x, leaf, want_f32=True, y_bf16=big[:50], y_f32=yf, workspace=ws)
    assert got[1] is yf and torch.equal(big[:50], want[0]) and torch.equal(yf, want[1]) and (big[50:] == 3.0).all()
    flat = torch.zeros(50 * K + 8, dtype=torch.bfloat16, device="cuda")
    flat[3:3 + 50 * K] = x.view(-1)
    assert torch.equal(pkg.fp8_project(flat[3:3 + 50 * K].view(50, K), leaf), want[0])
    wide = torch.zeros((50, 2 * K), dtype=torch.bfloat16, device="cuda")
    wide[:, ::2] = x
    assert torch.equal(pkg.fp8_project(wide[:, ::2], leaf), want[0])
    assert pkg.fp8_project(x[:0], leaf).shape == (0, R)
    y1 = torch.zeros(50 * R + 1, dtype=torch.bfloat16, device="cuda")
    pkg.fp8_project(x, leaf, y_bf16=y1[1:].view(50, R))                   # rows at odd 2-byte addresses
    assert torch.equal(y1[1:].view(50, R), want[0]) and y1[0] == 0
    with pytest.raises(pkg._lib.MiError):
        pkg.fp8_project(x, leaf, workspace=ws[:64])


def test_project_scale_blocks(pkg, gpu):
    """Each 128 x 128 block uses its own scale: one block nonzero at a time."""
    K, R = 400, 300
    bits = np.full((R, K), 0x38, np.uint8)                # 1.0
    x = torch.ones((20, K), dtype=torch.bfloat16, device="cuda")
    for rb in range(3):
        for kb in range(4):
            s = np.zeros((3, 4), np.float32)
            s[rb, kb] = 1.0 + rb + 10 * kb
            y = _np(pkg.fp8_project(x, _leaf(pkg, bits, s), want_f32=True)[1])
            want = np.zeros(R)
            want[rb * 128:(rb + 1) * 128] = (min(K, (kb + 1) * 128) - kb * 128) * float(s[rb, kb])
            assert np.array_equal(y, np.broadcast_to(want, y.shape)), (rb, kb)


# ------------------------------------------------------------------------------------------------ MLP
@pytest.mark.parametrize("B,D,I", [(1, 128, 16), (1, 1360, 592), (4, 256, 144), (16, 640, 384), (19, 592, 272),
                                   (40, 768, 256), (130, 512, 400), (300, 384, 640)])
def test_mlp(pkg, gpu, B, D, I):
    rng = np.random.default_rng(B + D + I)
    raw = [of8.random_weights(rng, R, K, 0.05) for R, K in ((I, D), (I, D), (D, I))]
    x = _acts(rng, B, D)
    want, bound = of8.mlp(of8.rows_dense(*of8.quantize(_np(x))), *[of8.weights_dense(*r) for r in raw], LIMIT)
    leaves = [_leaf(pkg, *r) for r in raw]
    yb, yf = pkg.fp8_mlp(x, *leaves, LIMIT, want_f32=True)
    _check(yb, yf, want, bound)
    p = dict(zip(("gate", "up", "down"), leaves))
    assert torch.equal(pkg.mlp_partial(p, x, LIMIT), yb)
    p["up"] = {"q": leaves[1].q, "s": leaves[1].s}
    assert torch.equal(pkg.mlp_partial(p, x, LIMIT), yb)
    assert torch.equal(pkg.fp8_mlp(pkg.fp8_quantize(x), *leaves, LIMIT), yb)
    assert pkg.fp8_mlp(x[:0], *leaves, LIMIT).shape == (0, D)


@pytest.mark.parametrize("tt", [32, 64, 128, 256])
@pytest.mark.parametrize("B,D,I", [(33, 144, 16), (70, 1040, 272), (300, 512, 400)])
def test_mlp_every_tile(pkg, gpu, tt, B, D, I):
    rng = np.random.default_rng(B + D + tt)
    raw = [of8.random_weights(rng, R, K, 0.05) for R, K in ((I, D), (I, D), (D, I))]
    x = _acts(rng, B, D)
    want, bound = of8.mlp(of8.rows_dense(*of8.quantize(_np(x))), *[of8.weights_dense(*r) for r in raw], LIMIT)
    for S in (1, 3, 8):
        with pkg.tuning(F8_TT=max(tt, 64) if S == 8 else tt, F8_S=S):
            yb, yf = pkg.fp8_mlp(x, *[_leaf(pkg, *r) for r in raw], LIMIT, want_f32=True)
            _check(yb, yf, want, bound)


# ------------------------------------------------------------------------------------------------ grouped, moe
def _experts(rng, E, D, I, std=0.05):
    return [of8.random_weights(rng, R, K, std, E) for R, K in ((I, D), (I, D), (D, I))]


def _routing(rng, T, E, k, skew=False):
    logits = rng.standard_normal((T, E)) + (np.arange(E) * -0.5 if skew else 0)
    idx = np.argsort(-logits, -1)[:, :k].astype(np.int32)
    w = rng.uniform(0.01, 1, (T, k)).astype(np.float32)
    return idx, w / w.sum(-1, keepdims=True)


@pytest.mark.parametrize("T,E,k,tm,D,R", [(1, 4, 2, 16, 256, 130), (7, 8, 2, 32, 144, 64), (50, 5, 2, 64, 272, 200),
                                          (200, 6, 3, 128, 384, 256), (33, 40, 5, 16, 1360, 592)])
def test_grouped(pkg, gpu, T, E, k, tm, D, R):
    rng = np.random.default_rng(T + E + tm)
    bits, s = of8.random_weights(rng, R, D, 0.05, E)
    idx, w = _routing(rng, T, E, k, True)
    idx[0, 0] = E                                         # a slot without a row
    plan = pkg.ragged_plan(torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), E, tm)
    x = _acts(rng, T, D)
    xs = pkg.moe_dispatch(x, plan)
    yb, yf = pkg.fp8_grouped(xs, plan, _leaf(pkg, bits, s), want_f32=True)
    xd = of8.rows_dense(*of8.quantize(_np(xs)))
    blk, n = plan["blk_expert"].cpu().numpy(), int(plan["n_blocks"])
    want, bound = np.zeros((xs.shape[0], R)), np.zeros((xs.shape[0], R))
    for g in range(n):
        r = slice(g * tm, (g + 1) * tm)
        want[r], bound[r] = of8.project(xd[r], of8.weights_dense(bits[blk[g]], s[blk[g]]))
    assert n < blk.size
    _check(yb, yf, want, bound)
    assert (yf[n * tm:] == 0).all()
    pair = pkg.fp8_grouped(pkg.fp8_quantize(xs), plan, _leaf(pkg, bits, s), want_f32=True)
    assert torch.equal(pair[1], yf)


def test_grouped_plan_out_of_range(pkg, gpu):
    """Experts outside [0, E) and more blocks than there are: those blocks are zero."""
    rng = np.random.default_rng(2)
    leaf = _leaf(pkg, *of8.random_weights(rng, 100, 128, 0.05, 3))
    x = _acts(rng, 64, 128)
    plan = {"blk_expert": torch.tensor([0, -1, 3, 2], dtype=torch.int32, device="cuda"),
            "n_blocks": torch.tensor([1000], dtype=torch.int32, device="cuda"),
            "tok_row": torch.zeros(64, dtype=torch.int32, device="cuda")}
    y = pkg.fp8_grouped(x, plan, leaf, want_f32=True)[1]
    assert (y[16:48] == 0).all() and (y[:16] != 0).any() and (y[48:] != 0).any()
    plan["tok_row"][5:16] = -1                            # padding rows: zeros whatever x holds
    z = pkg.fp8_grouped(x, plan, leaf, want_f32=True)[1]
    assert (z[5:16] == 0).all() and torch.equal(z[:5], y[:5]) and torch.equal(z[48:], y[48:])
    bad = leaf.q.view(torch.uint8).clone()
    bad[0, 3] = 0x7f                                       # and whatever the weights hold
    z = pkg.fp8_grouped(x, plan, pkg.Fp8Leaf(bad.view(F8), leaf.s), want_f32=True)[1]
    assert (z[5:16] == 0).all() and torch.isnan(z[:5, 3]).all()
    plan["n_blocks"].fill_(-5)
    assert (pkg.fp8_grouped(x, plan, leaf) == 0).all()


MOE = [(1, 4, 1, 128, 16), (1, 8, 2, 256, 144), (1, 64, 8, 640, 272), (2, 8, 3, 1360, 592), (3, 40, 5, 256, 128),
       (16, 64, 8, 512, 256), (17, 16, 8, 256, 144), (40, 8, 4, 272, 400), (64, 64, 8, 384, 128), (150, 4, 2, 256, 256),
       (300, 6, 2, 512, 384), (700, 3, 2, 144, 272)]


@pytest.mark.parametrize("T,E,k,D,I", MOE)
def test_moe(pkg, gpu, T, E, k, D, I):
    rng = np.random.default_rng(T + E + D)
    raw = _experts(rng, E, D, I)
    idx, w = _routing(rng, T, E, k, skew=T % 2 == 0)
    w[0, 0] = -0.3
    if T > 2:
        idx[1, 0] = -1
        idx[2, -1] = E
        idx[T - 1] = idx[T - 1, 0]                        # one expert in every column
    x = _acts(rng, T, D)
    xd = of8.rows_dense(*of8.quantize(_np(x)))
    cache = {}

    def dense(e):
        if e not in cache:
            cache[e] = [of8.weights_dense(b[e], s[e]) for b, s in raw]
        return cache[e]

    want, bound = of8.moe(xd, idx, w, dense, LIMIT, E)
    leaves = [_leaf(pkg, *r) for r in raw]
    it, wt = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    of, ob = pkg.fp8_moe(*leaves, x, it, wt, LIMIT, want_bf16=True)
    _check(ob, of, want, bound)
    of2, ob2 = pkg.fp8_moe(*leaves, x.float(), it.long(), wt, LIMIT)      # f32 activations of the same values
    assert ob2 is None and torch.equal(of2, of)


@pytest.mark.parametrize("tm", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T,E,k,D,I", [(1, 8, 2, 256, 144), (9, 4, 2, 640, 272), (70, 3, 2, 272, 128), (230, 3, 2, 384, 400)])
def test_moe_every_block_size(pkg, gpu, tm, T, E, k, D, I):
    """Each block size of the sorted form, from one row a block to full ones."""
    rng = np.random.default_rng(T + tm + D)
    raw = _experts(rng, E, D, I)
    idx, w = _routing(rng, T, E, k, skew=True)
    if T > 2:
        idx[1, 0], idx[2, -1] = -1, E
    x = _acts(rng, T, D)
    xd = of8.rows_dense(*of8.quantize(_np(x)))
    want, bound = of8.moe(xd, idx, w, lambda e: [of8.weights_dense(b[e], s[e]) for b, s in raw], LIMIT, E)
    args = [_leaf(pkg, *r) for r in raw] + [x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), LIMIT]
    with pkg.tuning(F8_STREAM=0, F8_TM=tm):
        _close(pkg.fp8_moe(*args)[0], want, bound)


@pytest.mark.parametrize("T,k,E", [(1, 16, 3), (16, 1, 2), (8, 2, 64), (5, 3, 4), (2, 8, 1)])
def test_moe_streams_up_to_16_slots(pkg, gpu, T, k, E):
    """The streaming form up to its limit: all slots on one expert, spread ones, some without an expert."""
    rng = np.random.default_rng(T * k + E)
    D, I = 256, 144
    raw = _experts(rng, E, D, I)
    idx = rng.integers(0, E, (T, k)).astype(np.int32)
    if T * k > 3:
        idx.reshape(-1)[2] = -7
    w = rng.uniform(-1, 1, (T, k)).astype(np.float32)
    x = _acts(rng, T, D)
    want, bound = of8.moe(of8.rows_dense(*of8.quantize(_np(x))), idx, w,
                          lambda e: [of8.weights_dense(b[e], s[e]) for b, s in raw], LIMIT, E)
    for limit in (16, 0):
        with pkg.tuning(F8_STREAM=limit):
            of, _ = pkg.fp8_moe(*[_leaf(pkg, *r) for r in raw], x, torch.from_numpy(idx).cuda(),
                                torch.from_numpy(w).cuda(), LIMIT)
        _close(of, want, bound)


@pytest.mark.parametrize("T,E,k,D,I", [(1, 8, 8, 1104, 1072), (2, 8, 4, 1040, 1040), (4, 6, 2, 1296, 1040),
                                       (8, 3, 1, 1168, 1040), (1, 9, 7, 1184, 1200)])
def test_moe_streams_several_row_tiles(pkg, gpu, T, E, k, D, I):
    """Few slots of wider layers, whose wavefronts take two row tiles of gate and up and four of down; the last ones
    end inside a wavefront's."""
    test_moe(pkg, gpu, T, E, k, D, I)


def test_moe_no_live_slots(pkg, gpu):
    rng = np.random.default_rng(0)
    leaves = [_leaf(pkg, *r) for r in _experts(rng, 3, 256, 128)]
    for T in (1, 4, 200):
        idx = torch.full((T, 2), 5, dtype=torch.int32, device="cuda")
        of, ob = pkg.fp8_moe(*leaves, _acts(rng, T, 256), idx, torch.ones((T, 2), device="cuda"), LIMIT, want_bf16=True)
        assert (of == 0).all() and (ob == 0).all()
    of, _ = pkg.fp8_moe(*leaves, _acts(rng, 1, 256)[:0], idx[:0], torch.ones((0, 2), device="cuda"), LIMIT)
    assert of.shape == (0, 256)


def test_moe_nan_stays_in_its_token(pkg, gpu):
    rng = np.random.default_rng(8)
    leaves = [_leaf(pkg, *r) for r in _experts(rng, 4, 256, 144)]
    for T in (2, 20, 150):
        idx, w = _routing(rng, T, 4, 2)
        x = _acts(rng, T, 256)
        it, wt = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
        clean, _ = pkg.fp8_moe(*leaves, x, it, wt, LIMIT)
        x[1, 7] = float("inf")
        of, _ = pkg.fp8_moe(*leaves, x, it, wt, LIMIT)
        keep = torch.arange(T, device="cuda") != 1
        assert torch.equal(of[keep], clean[keep]) and torch.isnan(of[1]).any()


@pytest.mark.parametrize("T", [1, 5, 90, 400])
def test_moe_repeats_its_bits(pkg, gpu, T):
    """The same call gives the same bits, on another stream and from a kept workspace too, and leaves its inputs alone."""
    rng = np.random.default_rng(T)
    E, k, D, I = 12, 3, 640, 272
    leaves = [_leaf(pkg, *r) for r in _experts(rng, E, D, I)]
    idx, w = [torch.from_numpy(a).cuda() for a in _routing(rng, T, E, k)]
    x = _acts(rng, T, D)
    before = [t.clone() for t in (x, idx, w)]
    want, _ = pkg.fp8_moe(*leaves, x, idx, w, LIMIT)
    ws = torch.full((pkg._lib.lib().mi_fp8_moe_workspace(T + 7, k, E, D, I),), 255, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(3):
        assert torch.equal(pkg.fp8_moe(*leaves, x, idx, w, LIMIT, workspace=ws)[0], want)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.fp8_moe(*leaves, x, idx, w, LIMIT)[0]
    side.synchronize()
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(before, (x, idx, w)))


@pytest.mark.parametrize("T", [1, 16, 80, 300])
def test_graphs(pkg, gpu, T):
    """Two captured graphs of the same calls on other inputs, replayed in turn between eager work, with new inputs:
    every replay equals the eager call."""
    rng = np.random.default_rng(T)
    E, k, D, I = 6, 2, 384, 144
    raw = _experts(rng, E, D, I)
    leaves = [_leaf(pkg, *r) for r in raw]
    one = [pkg.Fp8Leaf(l.q[0], l.s[0]) for l in leaves]

    def make():
        idx, w = _routing(rng, T, E, k)
        return _acts(rng, T, D), torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()

    def run(x, idx, w):
        plan = pkg.ragged_plan(idx, w, E, 16)
        xs = pkg.moe_dispatch(x, plan)
        y = pkg.fp8_grouped(xs, plan, leaves[0])
        return (pkg.fp8_moe(*leaves, x, idx, w, LIMIT)[0], pkg.fp8_project(x, one[0]), pkg.fp8_mlp(x, *one, LIMIT),
                pkg.moe_combine(y, plan, w))

    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        ins = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*ins)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run(*ins)
        graphs.append((g, ins, outs))
    for _ in range(3):
        wants = []
        for g, ins, outs in graphs:
            new = make()
            for a, b in zip(ins, new):
                a.copy_(b)
            wants.append([t.clone() for t in run(*new)])
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, _, outs), want in zip(graphs, wants):
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("T,tm", [(1, 16), (23, 16), (150, 64)])
def test_layer_from_its_parts(pkg, gpu, T, tm):
    """A routed layer as a program runs it: router, plan, dispatch, the experts' products, combine -- against fp8_moe on
    the same routing and the oracle's bound for it.  The parts round more (rows to bf16 between the products), so the
    two differ by bf16 roundings: y and the sum are rounded once each (2^-8 of a value, of the terms' magnitudes), g, u
    and h once each before h is quantised, which moves h by at most 3 * 2^-8 of itself times the slopes of silu (under
    1.1 + |g|, |g| <= LIMIT) and, past a border, by a step of e4m3 (2^-3 of its binade): both carried through |Wd|."""
    rng = np.random.default_rng(T)
    E, k, D, I = 8, 2, 512, 256
    raw = _experts(rng, E, D, I)
    gate, up, down = [_leaf(pkg, *r) for r in raw]
    x = _acts(rng, T, D)
    rw = torch.randn((D, E), device="cuda") * 0.05
    idx, w = pkg.route(x, rw, None, k)
    plan = pkg.ragged_plan(idx, w, E, tm)
    xs = pkg.fp8_quantize(pkg.moe_dispatch(x, plan))
    g, u = pkg.fp8_grouped(xs, plan, gate).float(), pkg.fp8_grouped(xs, plan, up).float()
    h = (torch.nn.functional.silu(g.clamp_max(LIMIT)) * u.clamp(-LIMIT, LIMIT)).to(torch.bfloat16)
    out = pkg.moe_combine(pkg.fp8_grouped(h, plan, down), plan, w)
    layer, _ = pkg.fp8_moe(gate, up, down, x, idx, w, LIMIT)
    xd, ni, nw = of8.rows_dense(*of8.quantize(_np(x))), idx.cpu().numpy(), _np(w)
    want, bound = of8.moe(xd, ni, nw, lambda e: [of8.weights_dense(b[e], s[e]) for b, s in raw], LIMIT, E)
    _close(layer, want, bound)
    slack = np.zeros_like(want)
    for t in range(T):
        for j in range(k):
            wg, wu, wd = [of8.weights_dense(b[ni[t, j]], s[ni[t, j]]) for b, s in raw]
            gv, uv = np.minimum(xd[t] @ wg.T, LIMIT), np.clip(xd[t] @ wu.T, -LIMIT, LIMIT)
            hv = of8.swiglu(gv, uv, LIMIT)
            dh = 2.0 ** -8 * (1.1 * np.abs(gv) * np.abs(uv) + 2 * np.abs(hv))
            step = 2.0 ** -3 * (np.abs(hv) + dh) + np.abs(hv).max() * 2.0 ** -15
            y = np.abs(wd @ of8.rows_dense(*of8.quantize(hv[None]))[0])
            e = np.abs(wd) @ (dh + step)
            slack[t] += abs(nw[t, j]) * (e + 2.0 ** -8 * (y + e))
    slack += 2.0 ** -8 * (np.abs(want) + slack)
    _close(out, want, bound + slack)


def test_weights_past_32_bits(pkg, gpu):
    """Experts that begin past 2^32 bytes of weights: the same bits as of a leaf that holds those experts alone."""
    rng = np.random.default_rng(5)
    E, I, D = 1024, 1040, 4112                            # 4.4 GB a matrix
    at = [3, 1019, 1023]
    small = [_leaf(pkg, *r) for r in _experts(rng, 3, D, I)]
    big = []
    for q, s in small:
        bq = torch.zeros((E,) + tuple(q.shape[1:]), dtype=torch.uint8, device="cuda")
        bs = torch.ones((E,) + tuple(s.shape[1:]), device="cuda")
        for j, e in enumerate(at):
            bq[e], bs[e] = q[j].view(torch.uint8), s[j]
        big.append(pkg.Fp8Leaf(bq.view(F8), bs))
    names = torch.tensor(at, dtype=torch.int32, device="cuda")
    for T, tm in ((2, None), (40, None), (200, 64), (200, 256)):
        x = _acts(rng, T, D)
        idx = torch.from_numpy(rng.integers(0, 3, (T, 2)).astype(np.int32)).cuda()
        w = torch.rand((T, 2), device="cuda")
        with pkg.tuning(**({} if tm is None else {"F8_TM": tm})):
            got, _ = pkg.fp8_moe(*big, x, names[idx.long()], w, LIMIT)
        with pkg.tuning(F8_TM=16 if T == 40 else tm or 0) if T > 2 else pkg.tuning():
            want, _ = pkg.fp8_moe(*small, x, idx, w, LIMIT)
        assert torch.equal(got, want)


def test_outputs_past_32_bits(pkg, gpu):
    """An output of more than 2^32 values: its rows are those of a smaller call."""
    rng = np.random.default_rng(6)
    B, K, R = 65600, 16, 65536
    leaf = _leaf(pkg, *of8.random_weights(rng, R, K))
    x = _acts(rng, B, K)
    y = pkg.fp8_project(x, leaf)
    few = pkg.fp8_project(x[-300:], leaf)
    assert torch.equal(y[-300:], few) and torch.equal(y[:64], pkg.fp8_project(x[:64], leaf))
