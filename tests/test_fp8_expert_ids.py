"""CPU: expert ids of a wider type than int32 keep being outside [0, E) when they are: none wraps into the range."""
import ctypes

import pytest
import torch

F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_ids_outside_the_range_stay_outside(pkg, monkeypatch, dtype):
    seen = []

    class Lib:
        def mi_fp8_moe_workspace(self, *a):
            return 1 << 16

        def mi_fp8_moe(self, *a):
            seen.append(list((ctypes.c_int32 * (a[11] * a[12])).from_address(a[13])))
            return 0

    monkeypatch.setattr(pkg.fp8, "lib", Lib)
    monkeypatch.setattr(pkg.fp8, "_stream_of", lambda *a: 0)
    E = 3
    leaf = lambda R, K: pkg.Fp8Leaf(torch.zeros((E, R, K)).to(F8), torch.zeros((E, -(-R // 128), -(-K // 128))))
    ids = [0, 2, -1, E, 2 ** 31 - 1, -2 ** 31]
    if dtype == torch.int64:
        ids += [2 ** 32, 2 ** 32 + 2, -2 ** 32, 2 ** 33 + 1, -2 ** 63, 2 ** 63 - 1, 1, 2 ** 31]
    idx = torch.tensor(ids, dtype=dtype).view(-1, 2)
    pkg.fp8_moe(leaf(16, 32), leaf(16, 32), leaf(32, 16), torch.zeros((idx.shape[0], 32)), idx,
                torch.ones(idx.shape), 7.0)
    assert len(seen[0]) == len(ids)
    for want, got in zip(ids, seen[0]):
        assert got == want if 0 <= want < E else not 0 <= got < E, (want, got)
