"""Inputs, oracle values and bounds of MLP and routed-layer calls over block-scaled fp8, for the tests of the oracle's
bounds (CPU) and of the kernels against them (GPU)."""
import numpy as np
import torch

from oracle import fp8 as of8

LIMIT = 4.0
# (B, D, I); (T, E, k, D, I): one row to some hundred, widths that end inside a group, a wavefront's row tiles, a block
MLP = [(1, 128, 16), (1, 1360, 592), (4, 256, 144), (16, 640, 384), (19, 592, 272), (32, 1040, 400), (40, 768, 256),
       (128, 528, 272), (130, 128, 144), (300, 128, 208)]
MOE = [(1, 4, 1, 128, 16), (1, 64, 8, 640, 272), (2, 8, 3, 1360, 592), (3, 40, 5, 256, 128), (16, 64, 8, 512, 256),
       (17, 16, 8, 256, 144), (40, 8, 4, 272, 400), (150, 4, 2, 256, 256), (300, 6, 2, 144, 208), (700, 3, 2, 144, 272),
       (1, 8, 8, 1104, 1072), (2, 8, 4, 1040, 1040), (4, 6, 2, 1296, 1040), (8, 3, 1, 1168, 1040), (1, 9, 7, 1184, 1200)]


def mlp_sums_f32(B):
    """Whether a dense call of B rows sums gate and up in f32."""
    return B <= 128


def moe_sums_f32(T, E, k):
    """Whether a routed call does: up to 96 slots an expert, on average."""
    return T * k // E <= 96


def acts(rng, n, K):
    x = rng.standard_normal((n, K)) * np.exp(rng.uniform(-4, 0, (n, 1)))
    x[:, rng.integers(0, K, max(1, K // 100))] *= 20.0
    return torch.from_numpy(x.astype(np.float32)).to(torch.bfloat16)


def values(x):
    """What quantised rows stand for."""
    return of8.rows_dense(*of8.quantize(x.double().numpy()))


def mlp_case(B, D, I):
    """x, the raw leaves, and of8.mlp's arguments."""
    rng = np.random.default_rng(B + D + I)
    raw = [of8.random_weights(rng, R, K, 0.05) for R, K in ((I, D), (I, D), (D, I))]
    x = acts(rng, B, D)
    return x, raw, (values(x), *[of8.weights_dense(*r) for r in raw], LIMIT)


def moe_case(T, E, k, D, I):
    rng = np.random.default_rng(T + E + D)
    raw = [of8.random_weights(rng, R, K, 0.05, E) for R, K in ((I, D), (I, D), (D, I))]
    idx = np.argsort(-(rng.standard_normal((T, E)) + (np.arange(E) * -0.5 if T % 2 == 0 else 0)), -1)[:, :k].astype(np.int32)
    w = rng.uniform(0.01, 1, (T, k)).astype(np.float32)
    w[0, 0] = -0.3
    if T > 2:
        idx[1, 0], idx[2, -1] = -1, E
        idx[T - 1] = idx[T - 1, 0]
    x = acts(rng, T, D)
    cache = {}

    def dense(e):
        if e not in cache:
            cache[e] = [of8.weights_dense(b[e], s[e]) for b, s in raw]
        return cache[e]

    return x, idx, w, raw, (values(x), idx, w, dense, LIMIT, E)
