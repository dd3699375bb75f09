"""CPU: the bounds that the MLP and routed-layer tests allow are far below the values that they check: a missing output, and
one whose h lacks its last 16 columns, are outside of them."""
import numpy as np
import pytest

from oracle import fp8 as of8
from tests import fp8_cases as fc


def _without_tail(gate, up, down):
    """Weights of an MLP whose h ends 16 columns early."""
    gate, down = gate.copy(), down.copy()
    gate[-16:], down[:, -16:] = 0.0, 0.0
    return gate, up, down


def _caught(got, want, bound):
    return float(np.mean(np.abs(got - want) > bound))


def _notices(want, bound, cut, f32):
    """Over the rows that are not zero: the median bound of a row is a small part of its values, zeros are outside of nearly
    all bounds, and a shorter h of many.  (The fp8 instruction's grid allows a row more, where gate and up go through it.)"""
    live = np.abs(want).max(1) > 0
    want, bound, cut = want[live], bound[live], cut[live]
    rows = np.median(bound, 1) / np.sqrt(np.mean(np.square(want), 1))
    assert np.median(rows) <= (0.07 if f32 else 0.2)
    assert _caught(np.zeros_like(want), want, bound) > (0.93 if f32 else 0.8)
    assert _caught(cut, want, bound) > 0.25


@pytest.mark.parametrize("B,D,I", fc.MLP)
def test_mlp_bound_notices(B, D, I):
    f32 = fc.mlp_sums_f32(B)
    _, _, args = fc.mlp_case(B, D, I)
    want, bound = of8.mlp(*args, f32_gate_up=f32)
    _notices(want, bound, of8.mlp(args[0], *_without_tail(*args[1:4]), fc.LIMIT)[0], f32)


@pytest.mark.parametrize("T,E,k,D,I", fc.MOE)
def test_moe_bound_notices(T, E, k, D, I):
    f32 = fc.moe_sums_f32(T, E, k)
    *_, args = fc.moe_case(T, E, k, D, I)
    want, bound = of8.moe(*args, f32_gate_up=f32)
    dense = args[3]
    _notices(want, bound, of8.moe(*args[:3], lambda e: _without_tail(*dense(e)), *args[4:])[0], f32)


def test_f32_bound_covers_any_order_of_an_f32_sum():
    """Each product added to an f32 sum one by one, forwards, backwards and in order of magnitude."""
    rng = np.random.default_rng(4)
    K = 1360
    xd = of8.rows_dense(*of8.quantize(rng.standard_normal((5, K))))
    wd = of8.weights_dense(*of8.random_weights(rng, 7, K))
    want, bound = of8.project(xd, wd, f32=True)
    for b in range(5):
        for o in range(7):
            p = (xd[b] * wd[o]).astype(np.float32)
            for order in (np.arange(K), np.arange(K)[::-1], np.argsort(np.abs(p)), np.argsort(p)):
                total = np.float32(0)
                for g in range(0, K, 128):                 # a sum per group, the groups' sums added
                    t = np.float32(0)
                    for v in p[order[(order >= g) & (order < g + 128)]]:
                        t = np.float32(t + v)
                    total = np.float32(total + t)
                assert abs(float(total) - want[b, o]) <= bound[b, o]
