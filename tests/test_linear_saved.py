"""CPU: what bf16_linear keeps for its backward pass: z only where a gradient reads it."""
import sys

import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture
def calls(pkg, monkeypatch):
    """The z of each forward call and the z of each backward call, with a library that launches nothing."""
    seen = []

    class Lib:
        def mi_bf16_linear_workspace(self, *a):
            return 0

        def mi_bf16_linear_grad_workspace(self, *a):
            return 0

        def mi_bf16_linear(self, *a):
            seen.append(("forward", a[11] is not None))
            return 0

        def mi_bf16_linear_grad(self, *a):
            seen.append(("backward", a[2] is not None))
            return 0

    linear = sys.modules[pkg.bf16_linear.__module__]
    monkeypatch.setattr(linear, "lib", Lib)
    monkeypatch.setattr(linear, "_stream_of", lambda *a: 0)
    return seen


def _inputs():
    return dict(x=torch.zeros((5, 16), dtype=BF16), w=torch.zeros((24, 16), dtype=BF16), bias=torch.zeros(24, dtype=BF16),
                residual=torch.zeros((5, 24), dtype=BF16))


def _run(pkg, t, act):
    return pkg.bf16_linear(t["x"], pkg.Bf16Leaf(t["w"]), bias=t["bias"], act=act, residual=t["residual"])


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_only_the_residual(pkg, calls, act):
    """Frozen weights in a stream that has a gradient: dy goes through, nothing is kept or written for it."""
    t = _inputs()
    t["residual"].requires_grad_()
    y = _run(pkg, t, act)
    assert calls == [("forward", False)] and all(s is None for s in y.grad_fn.saved_tensors)
    gy = torch.ones((5, 24), dtype=BF16)
    g, = torch.autograd.grad(y, t["residual"], gy)
    assert torch.equal(g, gy) and len(calls) == 1


@pytest.mark.parametrize("name", ["x", "w", "bias"])
def test_gradients_that_read_z(pkg, calls, name):
    t = _inputs()
    t[name].requires_grad_()
    y = _run(pkg, t, "gelu")
    assert calls == [("forward", True)]
    g, = torch.autograd.grad(y, t[name], torch.ones((5, 24), dtype=BF16))
    assert g.shape == t[name].shape and calls[1:] == [("backward", True)]


def test_no_activation_keeps_none(pkg, calls):
    t = _inputs()
    t["x"].requires_grad_()
    torch.autograd.grad(_run(pkg, t, None), t["x"], torch.ones((5, 24), dtype=BF16))
    assert calls == [("forward", False), ("backward", False)]
