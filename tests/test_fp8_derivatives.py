"""CPU: forward-mode duals are refused by the fp8 and sort entry points.  A dual does not require a gradient and has a
readable address, so its tangent would otherwise be dropped without a word."""
import sys

import pytest
import torch
from torch.autograd import forward_ad

F8 = torch.float8_e4m3fn


@pytest.fixture
def host(pkg, monkeypatch):
    """The package with a library that launches nothing, so that calls go through on the CPU."""
    class Lib:
        def __getattr__(self, name):
            return (lambda *a: 1 << 16) if name.endswith("_workspace") else (lambda *a: 0)

    rows = sys.modules[pkg.moe_dispatch.__module__]
    for m in (pkg.fp8, rows):
        monkeypatch.setattr(m, "lib", Lib)
        monkeypatch.setattr(m, "_stream_of", lambda *a: 0)
    monkeypatch.setattr(rows, "_stream", lambda: 0)
    return pkg


def _leaf(pkg, R, K, E=None, s=None):
    lead = () if E is None else (E,)
    s = torch.ones(lead + (-(-R // 128), -(-K // 128))) if s is None else s
    return pkg.Fp8Leaf(torch.zeros(lead + (R, K)).to(F8), s)


def _calls(pkg):
    """name -> (input, function of it): every input that a derivative could flow through."""
    plan = {"blk_expert": torch.zeros(4, dtype=torch.int32), "n_blocks": torch.ones(1, dtype=torch.int32),
            "tok_row": torch.zeros(64, dtype=torch.int32), "row_slot": torch.zeros((5, 2), dtype=torch.int32)}
    leaf, g, d = _leaf(pkg, 100, 256), _leaf(pkg, 144, 256, 3), _leaf(pkg, 256, 144, 3)
    one = [pkg.Fp8Leaf(l.q[0], l.s[0]) for l in (g, g, d)]
    idx, w, x, xs = torch.zeros((5, 2), dtype=torch.int32), torch.ones((5, 2)), torch.ones((5, 256)), torch.ones((64, 256))
    return {
        "quantize": (x, lambda t: pkg.fp8_quantize(t)),
        "project": (x, lambda t: pkg.fp8_project(t, leaf)),
        "project of quantised rows": (torch.ones((5, 2)), lambda t: pkg.fp8_project((x.to(F8), t), leaf)),
        "weight scales": (leaf.s, lambda t: pkg.fp8_project(x, pkg.Fp8Leaf(leaf.q, t))),
        "mlp": (x, lambda t: pkg.mlp_partial(dict(zip(("gate", "up", "down"), one)), t, 7.0)),
        "grouped": (xs, lambda t: pkg.fp8_grouped(t, plan, g)),
        "moe": (x, lambda t: pkg.fp8_moe(g, g, d, t, idx, w, 7.0)),
        "routing weights": (w, lambda t: pkg.fp8_moe(g, g, d, x, idx, t, 7.0)),
        "dispatch": (x, lambda t: pkg.moe_dispatch(t, plan)),
        "combine": (xs, lambda t: pkg.moe_combine(t, plan, w)),
        "combine's weights": (w, lambda t: pkg.moe_combine(xs, plan, t)),
    }


NAMES = ["quantize", "project", "project of quantised rows", "weight scales", "mlp", "grouped", "moe", "routing weights",
         "dispatch", "combine", "combine's weights"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(host, name):
    x, f = _calls(host)[name]
    f(x)                                                    # the call itself is a good one
    with forward_ad.dual_level():
        f(x)                                                # and stays one beside duals of others
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            f(dual)                                         # no_grad() turns reverse mode off, not this
        f(forward_ad.unpack_dual(dual).primal)


def test_forward_over_reverse_is_refused(host):
    """A tangent in the gradient that arrives."""
    calls = _calls(host)
    for name in ("dispatch", "combine", "combine's weights"):
        x, f = calls[name]
        x = x.clone().requires_grad_()
        out = f(x)
        torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, g)


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(host, name):
    """torch.func's wrappers hold no memory of their own: every transform ends in an error, none in a wrong value."""
    x, f = _calls(host)[name]
    first = lambda t: (lambda y: y[0] if isinstance(y, tuple) else y)(f(t)).float()
    with pytest.raises(RuntimeError):
        torch.func.jvp(first, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: first(t).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(first)(torch.stack([x, x]))


@pytest.mark.parametrize("what", ["rows", "weights"])
def test_e4m3_values_that_require_a_gradient_are_refused(host, what):
    """``t.to(torch.float8_e4m3fn)`` records a gradient: quantised rows and weights made so are refused like scales."""
    leaf, x = _leaf(host, 100, 256), torch.ones((5, 256))
    rows = lambda t: host.fp8_project((t.to(F8), torch.ones((5, 2))), leaf)
    weights = lambda t: host.fp8_project(x, host.Fp8Leaf(t.to(F8), leaf.s))
    f, t = (rows, x) if what == "rows" else (weights, torch.ones((100, 256)))
    f(t)
    t = t.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        f(t)
    with torch.no_grad():
        f(t)
    f(t.detach())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        f(forward_ad.make_dual(t.detach(), torch.ones_like(t)))
