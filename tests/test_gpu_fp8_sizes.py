"""GPU: the fp8 calls at the ends of their sizes: the longest rows (512 groups), more slots than the plan's workgroup takes in
one pass (8192), against the 64-bit oracle."""
import numpy as np
import pytest
import torch

from oracle import fp8 as of8
from tests import fp8_cases as fc

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _leaf(pkg, bits, s):
    return pkg.Fp8Leaf(torch.from_numpy(bits).cuda().view(F8), torch.from_numpy(s).cuda())


def _check(got, want, bound):
    got = got.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) - bound).max())
    assert np.median(bound) < 0.2 * np.sqrt(np.mean(want ** 2))


@pytest.mark.parametrize("B", [1, 17, 40, 150, 300])
@pytest.mark.parametrize("K,R", [(65536, 20), (65520, 130), (65424, 300)])
def test_project_longest_rows(pkg, gpu, B, K, R):
    rng = np.random.default_rng(B + R)
    bits, s = of8.random_weights(rng, R, K)
    x = fc.acts(rng, B, K)
    want, bound = of8.project(fc.values(x), of8.weights_dense(bits, s))
    leaf = _leaf(pkg, bits, s)
    got = pkg.fp8_project(x.cuda(), leaf, want_f32=True)[1]
    _check(got, want, bound)
    assert torch.equal(pkg.fp8_project(pkg.fp8_quantize(x.cuda()), leaf, want_f32=True)[1], got)


@pytest.mark.parametrize("B,D,I", [(1, 65536, 16), (33, 65520, 16), (1, 16, 65536), (20, 144, 65536), (40, 16, 65520),
                                   (200, 16, 65536)])
def test_mlp_longest_rows(pkg, gpu, B, D, I):
    x, raw, args = fc.mlp_case(B, D, I)
    if D > I:                                              # sums of 65536 values: weights that keep g and u ordinary
        raw = [(b, s * np.float32(0.02)) for b, s in raw[:2]] + raw[2:]
        args = (args[0], *[of8.weights_dense(*r) for r in raw], fc.LIMIT)
    want, bound = of8.mlp(*args, f32_gate_up=fc.mlp_sums_f32(B))
    _check(pkg.fp8_mlp(x.cuda(), *[_leaf(pkg, *r) for r in raw], fc.LIMIT, want_f32=True)[1], want, bound)


@pytest.mark.parametrize("T,E,k,D,I", [(2, 3, 2, 65536, 16), (40, 2, 1, 65520, 32)])
def test_routed_longest_rows(pkg, gpu, T, E, k, D, I):
    x, idx, w, raw, args = fc.moe_case(T, E, k, D, I)
    raw = [(b, s * np.float32(0.02)) for b, s in raw[:2]] + raw[2:]
    dense = lambda e: [of8.weights_dense(b[e], s[e]) for b, s in raw]
    want, bound = of8.moe(*args[:3], dense, *args[4:], f32_gate_up=True)
    it, wt = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    _check(pkg.fp8_moe(*[_leaf(pkg, *r) for r in raw], x.cuda(), it, wt, fc.LIMIT)[0], want, bound)
    plan = pkg.ragged_plan(it, wt, E, 16)
    y = pkg.fp8_grouped(pkg.moe_dispatch(x.cuda(), plan), plan, _leaf(pkg, *raw[0]), want_f32=True)[1]
    for t in range(T):
        for j in range(k):
            if 0 <= idx[t, j] < E:
                v, b = of8.project(args[0][t:t + 1], dense(idx[t, j])[0])
                got = y[plan["row_slot"][t, j]].double().cpu().numpy()
                assert np.all(np.abs(got - v[0]) <= b[0])


@pytest.mark.parametrize("T,E,k", [(1024, 3, 8), (1025, 1024, 8), (1100, 5, 8), (2300, 900, 8), (8500, 16, 1), (500, 64, 40)])
def test_routed_many_slots(pkg, gpu, T, E, k):
    """8192 slots, one token more, two and three passes; experts outside the range among the last."""
    rng = np.random.default_rng(T + E)
    D, I = 144, 32
    raw = [of8.random_weights(rng, R, K, 0.05, E) for R, K in ((I, D), (I, D), (D, I))]
    idx = rng.integers(0, E, (T, k)).astype(np.int32)
    idx[-1, 0], idx[-2, -1], idx[T // 2, 0] = E, -1, 1 << 30
    w = rng.uniform(0.1, 1, (T, k)).astype(np.float32)
    x = fc.acts(rng, T, D)
    cache = {}

    def dense(e):
        if e not in cache:
            cache[e] = [of8.weights_dense(b[e], s[e]) for b, s in raw]
        return cache[e]

    want, bound = of8.moe(fc.values(x), idx, w, dense, fc.LIMIT, E, f32_gate_up=fc.moe_sums_f32(T, E, k))
    call = [_leaf(pkg, *r) for r in raw] + [x.cuda(), torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), fc.LIMIT]
    got = pkg.fp8_moe(*call)[0]
    _check(got, want, bound)
    assert torch.equal(pkg.fp8_moe(*call)[0], got)
