"""CPU: more rows or columns than 32 bits count reach the C entries of the norms, the gate and the linear layer as more than they
take, never as what the low 32 bits happen to say."""
import sys

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32
PAST = 1 << 32


class Launched(Exception):
    """A call that reached the library with counts it takes."""


@pytest.fixture
def entries(pkg, monkeypatch):
    """The library's entries, which launch nothing: a call past their limits (rows, columns) is refused as theirs are."""
    class Lib:
        def __getattr__(self, name):
            at, limits = {"mi_rms_norm": ((7, 8), (1 << 22, 1 << 15)), "mi_rms_norm_grad": ((8, 9), (1 << 22, 1 << 15)),
                          "mi_moe_gate": ((4, 5), (1 << 22, 1024)), "mi_moe_gate_grad": ((5, 6), (1 << 22, 1024)),
                          "mi_bf16_linear": ((2, 4, 5), (1 << 20, 1 << 16, 1 << 16)),
                          "mi_bf16_linear_grad": ((6, 8, 9), (1 << 20, 1 << 16, 1 << 16))}.get(name, (None, None))
            if at is None:                                          # the sizes of workspaces: 0 for what is refused
                def size(*a):
                    assert all(0 <= v < 1 << 31 for v in a)
                    return 0
                return size

            def call(*a):
                assert all(0 <= a[k] < 1 << 31 for k in at), (name, [a[k] for k in at])
                if any(a[k] > limit for k, limit in zip(at, limits)):
                    return 4
                raise Launched
            return call

    for fn in (pkg.rms_norm, pkg.moe_gate, pkg.bf16_linear):
        module = sys.modules[fn.__module__]
        monkeypatch.setattr(module, "lib", Lib)
        monkeypatch.setattr(module, "_stream_of", lambda *a: 0)
    return pkg


def _meta(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _calls(pkg):
    return {
        "norm rows": lambda: pkg.rms_norm(_meta(PAST + 4, 8), _meta(8)),
        "norm columns": lambda: pkg.rms_norm(_meta(2, PAST + 64), _meta(PAST + 64)),
        "norm with a gradient": lambda: pkg.rms_norm(_meta(PAST + 4, 8).requires_grad_(), _meta(8)),
        "fp8 norm rows": lambda: pkg.fp8_rms_norm(_meta(PAST + 4, 16), _meta(16), residual=_meta(PAST + 4, 16)),
        "gate rows": lambda: pkg.moe_gate(_meta(PAST + 4, 16, dtype=F32), 2),
        "gate with a gradient": lambda: pkg.moe_gate(_meta(PAST + 4, 16, dtype=F32).requires_grad_(), 2),
        "linear rows": lambda: pkg.bf16_linear(_meta(PAST + 4, 16), pkg.Bf16Leaf(_meta(24, 16))),
        "linear columns": lambda: pkg.bf16_linear(_meta(3, PAST + 16), pkg.Bf16Leaf(_meta(24, PAST + 16))),
        "linear outputs": lambda: pkg.bf16_linear(_meta(3, 16), pkg.Bf16Leaf(_meta(PAST + 24, 16))),
        "linear with a gradient": lambda: pkg.bf16_linear(_meta(PAST + 4, 16).requires_grad_(), pkg.Bf16Leaf(_meta(24, 16)), act="silu"),
    }


@pytest.mark.parametrize("name", ["norm rows", "norm columns", "norm with a gradient", "fp8 norm rows", "gate rows",
                                  "gate with a gradient", "linear rows", "linear columns", "linear outputs", "linear with a gradient"])
def test_counts_past_32_bits(entries, name):
    with pytest.raises(entries._lib.MiError):
        _calls(entries)[name]()


def test_counts_within_reach_the_library(entries):
    pkg = entries
    for call in (lambda: pkg.rms_norm(_meta(1 << 22, 8), _meta(8)), lambda: pkg.moe_gate(_meta(1 << 22, 16, dtype=F32), 2),
                 lambda: pkg.bf16_linear(_meta(1 << 20, 16), pkg.Bf16Leaf(_meta(1 << 16, 16)))):
        with pytest.raises(Launched):
            call()
