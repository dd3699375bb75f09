"""GPU: the fp8 MLP and routed layer within bounds that notice a missing part (test_oracle_fp8_bounds.py), and the calls that
sum gate and up in f32 told from those that go through the fp8 instruction."""
import numpy as np
import pytest
import torch

from oracle import fp8 as of8
from tests import fp8_cases as fc

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _leaf(pkg, bits, s):
    return pkg.Fp8Leaf(torch.from_numpy(bits).cuda().view(F8), torch.from_numpy(s).cuda())


def _check(yb, yf, want, bound):
    got = yf.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) - bound).max())
    assert torch.equal(yb, yf.to(torch.bfloat16))


@pytest.mark.parametrize("B,D,I", fc.MLP)
def test_mlp(pkg, gpu, B, D, I):
    x, raw, args = fc.mlp_case(B, D, I)
    want, bound = of8.mlp(*args, f32_gate_up=fc.mlp_sums_f32(B))
    leaves = [_leaf(pkg, *r) for r in raw]
    _check(*pkg.fp8_mlp(x.cuda(), *leaves, fc.LIMIT, want_f32=True), want, bound)
    _check(*pkg.fp8_mlp(pkg.fp8_quantize(x.cuda().float()), *leaves, fc.LIMIT, want_f32=True), want, bound)


@pytest.mark.parametrize("tt", [32, 64, 128])
@pytest.mark.parametrize("B,D,I", [c for c in fc.MLP if 32 < c[0] <= 128])
def test_mlp_every_tile(pkg, gpu, tt, B, D, I):
    x, raw, args = fc.mlp_case(B, D, I)
    want, bound = of8.mlp(*args, f32_gate_up=True)
    for S in (1, 3):
        with pkg.tuning(F8_TT=tt, F8_S=S):
            _check(*pkg.fp8_mlp(x.cuda(), *[_leaf(pkg, *r) for r in raw], fc.LIMIT, want_f32=True), want, bound)


@pytest.mark.parametrize("T,E,k,D,I", fc.MOE)
def test_moe(pkg, gpu, T, E, k, D, I):
    x, idx, w, raw, args = fc.moe_case(T, E, k, D, I)
    want, bound = of8.moe(*args, f32_gate_up=fc.moe_sums_f32(T, E, k))
    call = [_leaf(pkg, *r) for r in raw] + [x.cuda(), torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), fc.LIMIT]
    of, ob = pkg.fp8_moe(*call, want_bf16=True)
    _check(ob, of, want, bound)
    if T * k // E <= 96:
        for tm in (16, 32, 64, 128):                       # the sorted form, in every block size that sums in f32
            with pkg.tuning(F8_STREAM=0, F8_TM=tm):
                of, ob = pkg.fp8_moe(*call, want_bf16=True)
                _check(ob, of, want, bound)


# Products 2^16, seven of 4, -2^16, seven of 4: 56 in f32 (all partial sums are integers below 2^24).  The fp8 instruction adds
# eight on a grid of 2^-13 of the largest, 8, and cuts the fours.
def _cancelling(B, I):
    x = np.zeros((B, 128), np.float32)
    x[:, :16] = 2.0
    x[:, 0] = x[:, 8] = 256.0
    gate = np.zeros((I, 128), np.float32)
    gate[:, :16] = 2.0
    gate[:, 0], gate[:, 8] = 256.0, -256.0
    up = np.zeros((I, 128), np.float32)
    up[:, 0] = 2.0 ** -8                                   # u = 1
    down = np.zeros((128, I), np.float32)
    down[np.arange(I), np.arange(I)] = 1.0                 # y = h
    h = of8.swiglu(np.full((1, I), 56 * 2.0 ** -6), np.ones((1, I)), fc.LIMIT)
    want = np.zeros(128)
    want[:I] = of8.rows_dense(*of8.quantize(h))[0]
    assert want[0] > 0.5
    return torch.from_numpy(x).to(torch.bfloat16), (gate, up, down), (2.0 ** -6, 1.0, 1.0), want


def _one(pkg, w, s, E=None):
    q = torch.from_numpy(w).to(F8).cuda()
    q = q if E is None else q.view(torch.uint8).expand((E,) + q.shape).contiguous().view(F8)
    return pkg.Fp8Leaf(q, torch.full(q.shape[:-2] + (1, 1), s, device="cuda"))


@pytest.mark.parametrize("B", [1, 16, 17, 32, 33, 64, 100, 128])
def test_mlp_sums_gate_and_up_in_f32(pkg, gpu, B):
    x, ws, ss, want = _cancelling(B, 16)
    leaves = [_one(pkg, w, s) for w, s in zip(ws, ss)]
    for form in (x.cuda(), x.cuda().float(), pkg.fp8_quantize(x.cuda())):
        got = pkg.fp8_mlp(form, *leaves, fc.LIMIT, want_f32=True)[1].double().cpu().numpy()
        assert (got == want).all()


@pytest.mark.parametrize("T,k,E", [(1, 8, 8), (2, 8, 64), (16, 1, 4), (5, 4, 8), (60, 8, 16), (100, 2, 4), (96, 1, 1)])
def test_moe_sums_gate_and_up_in_f32(pkg, gpu, T, k, E):
    """Streamed calls and blocks up to 128 rows; every token's experts are the same, so out = h times the weights' sum."""
    x, ws, ss, want = _cancelling(T, 16)
    leaves = [_one(pkg, w, s, E) for w, s in zip(ws, ss)]
    idx = torch.stack([torch.randperm(max(E, k), device="cuda")[:k] % E for _ in range(T)]).to(torch.int32)
    w = torch.full((T, k), 0.5, device="cuda")
    got = pkg.fp8_moe(*leaves, x.cuda(), idx, w, fc.LIMIT)[0].double().cpu().numpy()
    assert (got == want * 0.5 * k).all()
