"""CPU: what mi_rms_norm, mi_moe_gate, mi_bf16_linear and their gradients refuse, each before any launch."""
import ctypes

import pytest

P = ctypes.c_void_p
A, B, C, D, E, W = [P(0x10000 * (k + 1)) for k in range(6)]         # never dereferenced
ODD, HALF = P(0x10002), P(0x10008)
BIG = 1 << 40


@pytest.fixture(scope="module")
def abi(pkg):
    L = pkg._lib.lib()
    codes = dict(NULL=1, SHAPE=3, TOKENS=4, WORKSPACE=5, ARG=8)

    def call(fn, base, expect, **change):
        args = dict(base)
        args.update(change)
        assert getattr(L, fn)(*args.values()) == codes[expect], (fn, change)
    return call


NORM = dict(x=A, dtype=0, x_stride=64, residual=B, residual_stride=64, w=C, w_dtype=1, T=4, D=64, eps=1e-5, y=D, stream_out=E,
            rstd=W, q=None, qs=None, stream=None)
NORM_GRAD = dict(dy=A, s=B, dtype=0, s_stride=64, dstream=None, w=C, w_dtype=0, rstd=D, T=4, D=64, dx=E, dw=W, workspace=A, nbytes=BIG,
                 stream=None)
GATE = dict(logits=A, dtype=1, stride=64, bias=B, T=4, E=64, k=8, scores=0, n_group=1, topk_group=1, group_top=2, norm=1, scaling=1.0,
            idx=C, w=D, stream=None)
GATE_GRAD = dict(logits=A, dtype=1, stride=64, idx=B, dw=C, T=4, E=64, k=8, scores=0, norm=1, scaling=1.0, dlogits=D, stream=None)
LINEAR = dict(x=A, x_stride=64, B=40, w=B, n_in=64, n_out=24, bias=C, act=1, residual=D, y_dtype=0, y=E, z=W, workspace=A, nbytes=BIG,
              stream=None)
LINEAR_GRAD = dict(dy=A, dy_dtype=0, z=B, act=1, x=C, x_stride=64, B=40, w=D, n_in=64, n_out=24, dx=E, dw=W, dbias=A, workspace=B,
                   nbytes=BIG, stream=None)


def test_rms_norm(abi):
    for name in ("x", "w"):
        abi("mi_rms_norm", NORM, "NULL", **{name: None})
    abi("mi_rms_norm", NORM, "NULL", y=None)
    abi("mi_rms_norm", NORM, "NULL", residual=None)                 # a stream output without one
    abi("mi_rms_norm", NORM, "NULL", q=A)
    abi("mi_rms_norm", NORM, "NULL", qs=A)
    for name in ("dtype", "w_dtype"):
        abi("mi_rms_norm", NORM, "ARG", **{name: 2})
    for T in (0, -1, (1 << 22) + 1):
        abi("mi_rms_norm", NORM, "TOKENS", T=T)
    abi("mi_rms_norm", NORM, "TOKENS", T=1 << 22, D=8200, x_stride=8200, residual_stride=8200)     # 2^32 threads
    for d in (0, -8, 63, 32776):
        abi("mi_rms_norm", NORM, "SHAPE", D=d, x_stride=1 << 16, residual_stride=1 << 16)
    abi("mi_rms_norm", NORM, "SHAPE", D=56, q=A, qs=B)
    for name in ("x_stride", "residual_stride"):
        for v in (56, 68, -64, (1 << 40) + 8):
            abi("mi_rms_norm", NORM, "ARG", **{name: v})
    for eps in (-1e-9, float("nan"), float("inf"), 1e31):
        abi("mi_rms_norm", NORM, "ARG", eps=eps)
    for name in ("x", "residual", "w", "y", "stream_out"):
        abi("mi_rms_norm", NORM, "ARG", **{name: HALF})
    abi("mi_rms_norm", NORM, "ARG", q=HALF, qs=B)
    abi("mi_rms_norm", NORM, "ARG", q=A, qs=ODD)
    abi("mi_rms_norm", NORM, "ARG", rstd=ODD)


def test_rms_norm_grad(abi, pkg):
    for name in ("dy", "s", "w", "rstd", "dx"):
        abi("mi_rms_norm_grad", NORM_GRAD, "NULL", **{name: None})
    abi("mi_rms_norm_grad", NORM_GRAD, "TOKENS", T=0)
    abi("mi_rms_norm_grad", NORM_GRAD, "SHAPE", D=60)
    abi("mi_rms_norm_grad", NORM_GRAD, "ARG", s_stride=60)
    abi("mi_rms_norm_grad", NORM_GRAD, "ARG", dtype=3)
    for name in ("dy", "s", "dstream", "w", "dx", "dw", "workspace"):
        abi("mi_rms_norm_grad", NORM_GRAD, "ARG", **{name: HALF})
    abi("mi_rms_norm_grad", NORM_GRAD, "WORKSPACE", workspace=None)
    size = pkg._lib.lib().mi_rms_norm_grad_workspace
    abi("mi_rms_norm_grad", NORM_GRAD, "WORKSPACE", nbytes=size(4, 64) - 1)
    assert size(0, 64) == size(4, 60) == 0 < size(1, 8) <= size(2, 8) <= size(1 << 22, 8)


def test_moe_gate(abi):
    for name in ("logits", "idx", "w"):
        abi("mi_moe_gate", GATE, "NULL", **{name: None})
    for name in ("logits", "idx", "dw", "dlogits"):
        abi("mi_moe_gate_grad", GATE_GRAD, "NULL", **{name: None})
    for fn, base in (("mi_moe_gate", GATE), ("mi_moe_gate_grad", GATE_GRAD)):
        for T in (0, -3, (1 << 22) + 1):
            abi(fn, base, "TOKENS", T=T)
        for e in (0, -1, 1025):
            abi(fn, base, "SHAPE", E=e, stride=2000)
        abi(fn, base, "SHAPE", stride=63)
        for k in (0, -1, 33, 65):
            abi(fn, base, "ARG", k=k)
        for change in (dict(dtype=2), dict(scores=2), dict(norm=2), dict(scaling=float("nan")), dict(scaling=float("inf")),
                       dict(logits=ODD), dict(idx=ODD)):
            abi(fn, base, "ARG", **change)
    for change in (dict(n_group=0), dict(n_group=3), dict(n_group=64), dict(n_group=4, topk_group=5), dict(n_group=4, topk_group=0),
                   dict(n_group=16, topk_group=1), dict(group_top=0), dict(group_top=3), dict(bias=ODD), dict(w=ODD),
                   dict(E=62, n_group=4, topk_group=4)):
        abi("mi_moe_gate", GATE, "ARG", **change)
    abi("mi_moe_gate_grad", GATE_GRAD, "ARG", dlogits=ODD)
    abi("mi_moe_gate_grad", GATE_GRAD, "ARG", dw=ODD)


def test_bf16_linear(abi, pkg):
    for name in ("x", "w", "y"):
        abi("mi_bf16_linear", LINEAR, "NULL", **{name: None})
    for n in (0, -1, (1 << 20) + 1):
        abi("mi_bf16_linear", LINEAR, "TOKENS", B=n)
    for change in (dict(n_in=0), dict(n_in=60), dict(n_in=65544, x_stride=1 << 17), dict(n_out=0), dict(n_out=65537)):
        abi("mi_bf16_linear", LINEAR, "SHAPE", **change)
    for change in (dict(x_stride=56), dict(x_stride=68), dict(x_stride=(1 << 20) + 8), dict(act=5), dict(act=-1), dict(y_dtype=2),
                   dict(x=HALF), dict(w=HALF), dict(z=HALF), dict(workspace=HALF), dict(bias=P(0x10001)), dict(y=P(0x10001)),
                   dict(residual=ODD, y_dtype=1)):
        abi("mi_bf16_linear", LINEAR, "ARG", **change)
    size = pkg._lib.lib().mi_bf16_linear_workspace(40, 64, 24)
    abi("mi_bf16_linear", LINEAR, "WORKSPACE", workspace=None)
    abi("mi_bf16_linear", LINEAR, "WORKSPACE", nbytes=size - 1)


def test_bf16_linear_grad(abi, pkg):
    for change in (dict(dy=None), dict(z=None), dict(w=None), dict(x=None), dict(dx=None, dw=None, dbias=None)):
        abi("mi_bf16_linear_grad", LINEAR_GRAD, "NULL", **change)
    abi("mi_bf16_linear_grad", LINEAR_GRAD, "TOKENS", B=0)
    abi("mi_bf16_linear_grad", LINEAR_GRAD, "SHAPE", n_in=4)
    for change in (dict(x_stride=60), dict(act=9), dict(dy_dtype=2), dict(dy=P(0x10001)), dict(z=HALF), dict(x=HALF), dict(w=HALF),
                   dict(dx=P(0x10001)), dict(dw=P(0x10001)), dict(dbias=P(0x10001)), dict(workspace=HALF)):
        abi("mi_bf16_linear_grad", LINEAR_GRAD, "ARG", **change)
    size = pkg._lib.lib().mi_bf16_linear_grad_workspace(40, 64, 24)
    abi("mi_bf16_linear_grad", LINEAR_GRAD, "WORKSPACE", workspace=None)
    abi("mi_bf16_linear_grad", LINEAR_GRAD, "WORKSPACE", nbytes=size - 1)
