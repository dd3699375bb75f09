"""CPU: what moe_combine keeps for its backward pass: y only where the gradient of w needs it."""
import gc
import sys
import weakref

import pytest
import torch


@pytest.fixture
def calls(pkg, monkeypatch):
    """The calls of the backward entry point (its y and dw), with a library that launches nothing."""
    seen = []

    class Lib:
        def mi_moe_combine(self, *a):
            return 0

        def mi_moe_combine_grad(self, dout, y, *a):
            seen.append((y, a[-2]))
            return 0

    rows = sys.modules[pkg.moe_combine.__module__]
    monkeypatch.setattr(rows, "lib", Lib)
    monkeypatch.setattr(rows, "_stream_of", lambda *a: 0)
    monkeypatch.setattr(rows, "_stream", lambda: 0)
    return seen


def _plan():
    return {"tok_row": torch.zeros(64, dtype=torch.int32), "row_slot": torch.zeros((5, 2), dtype=torch.int32)}


def test_frozen_weights_leave_y_free(pkg, calls):
    """With w frozen, y may be changed in place or dropped between the two passes, as with torch's own products."""
    leaf = torch.ones((64, 32), requires_grad=True)
    y = leaf * 2.0
    out = pkg.moe_combine(y, _plan(), torch.ones((5, 2)))
    gone = weakref.ref(y)
    y.zero_()
    del y
    gc.collect()
    assert gone() is None
    g, = torch.autograd.grad(out.sum(), leaf)
    assert g.shape == leaf.shape and calls == [(None, None)]


def test_gradient_of_w_keeps_y(pkg, calls):
    leaf, w = torch.ones((64, 32), requires_grad=True), torch.ones((5, 2), requires_grad=True)
    y = leaf * 2.0
    out = pkg.moe_combine(y, _plan(), w)
    torch.autograd.grad(out.sum(), [leaf, w], retain_graph=True)
    assert calls[0][0] == y.data_ptr() and calls[0][1] is not None
    gw, = torch.autograd.grad(out.sum(), [w], retain_graph=True)
    assert gw.shape == w.shape
    y.zero_()                                              # a value that the gradient of w is made of
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), [w])


def test_refusals(pkg):
    """dw may be left out, and y with it; nothing else may."""
    import ctypes
    P = ctypes.c_void_p
    f = lambda dout=P(0x10000), y=P(0x90000), sl=P(0x60000), tr=P(0x70000), w=P(0x80000), dy=P(0x40000), dw=P(0xa0000), dt=7: \
        pkg._lib.lib().mi_moe_combine_grad(dout, y, dt, 4, 2, 64, sl, tr, w, 32, dy, dw, None)
    assert f() == 8                                        # the type comes after the pointers
    assert f(dw=None) == 8 and f(y=None, dw=None) == 8
    assert f(y=None) == 1
    for name in ("dout", "sl", "tr", "w", "dy"):
        assert f(**{name: None}) == 1 and f(**{name: None, "dw": None}) == 1
