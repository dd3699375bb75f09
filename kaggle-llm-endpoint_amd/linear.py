"""Products over bf16 weights with bias, activation and residual in one launch, for one row to many, with gradients:

    y = bf16_linear(x, leaf)                                        a projection (bf16_project's product)
    h = bf16_linear(x, leaf, bias=b, act="silu")                    a biased, activated one
    s = bf16_linear(a, leaf, residual=s)                            back into the stream

Products of bf16 values are exact and summed in f32; bias, activation and residual follow in f32, and the result is rounded
once.  Gradients of x, the weight, the bias and the residual are recorded, first order and reverse mode only (a forward-mode
tangent is refused); for an activation the forward pass keeps the values before it, in f32 (rounded to bf16 they would cost
the gradients another such rounding), unless the residual's gradient is the only one asked for.  Sums without atomics, in an
order that the call's sizes and a row's place in it decide: equal calls give equal bits, but a row's last bits may change
with the number of rows, or between equal rows of one call.  For the products of the gradients act'(z) dy is rounded to bf16
(where it is not dy itself, in bf16).  A captured backward pass needs leaves of its own (``x.detach().requires_grad_()``
inside the capture): an eager graph that still holds the same leaves has bound their gradients to another stream.
Everything runs on the current torch (HIP) stream of the current device; outputs and workspaces must not overlap the inputs
or each other.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import INT_MAX, check, lib
from .fp8 import _DTYPES, _aligned, _no_tangent, _out, _stream_of, _workspace
from .resident import Bf16Leaf, _ptr

ACTS = {None: _lib.MI_ACT_NONE, "silu": _lib.MI_ACT_SILU, "gelu": _lib.MI_ACT_GELU, "gelu_tanh": _lib.MI_ACT_GELU_TANH,
        "relu": _lib.MI_ACT_RELU}


def _rows_of(x):
    """(x's rows at a 16-byte address, their stride): as they lie where a kernel can read them so, else a copy."""
    if not x.is_contiguous():
        stride = x.stride(0)
        if x.stride(1) == 1 and x.shape[1] <= stride <= 1 << 20 and stride % 8 == 0 and x.data_ptr() % 16 == 0:
            return x, stride
    return _aligned(x), x.shape[1]


def _linear(x, wT, bias, act, residual, dtype, y, z, workspace):
    B, K, R = min(x.shape[0], INT_MAX), min(x.shape[1], INT_MAX), min(wT.shape[0], INT_MAX)
    stream = _stream_of("bf16_linear", x, wT, bias, residual, y, z, workspace)
    x, stride = _rows_of(x)
    wT = _aligned(wT)
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    held, ws, nbytes = _workspace(workspace, lib().mi_bf16_linear_workspace(B, K, R), x.device)
    check("mi_bf16_linear", lib().mi_bf16_linear(_ptr(x), stride, B, _ptr(wT), K, R, _ptr(bias), act, _ptr(residual),
                                                 _DTYPES[dtype], _ptr(y), _ptr(z), ws, nbytes, stream))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wT, bias, residual, act, dtype):
        B, R = x.shape[0], wT.shape[0]
        y = torch.empty((B, R), dtype=dtype, device=x.device)
        # (the residual's gradient is dy: z serves the others only)
        keep = act and any(ctx.needs_input_grad[:3])
        z = torch.empty((B, -(-R // 8) * 8), dtype=torch.float32, device=x.device) if keep else None
        if B:
            _linear(x, wT, bias, act, residual, dtype, y, z, None)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, wT if ctx.needs_input_grad[0] else None, z)
        ctx.act, ctx.shape = act, (B, x.shape[1], R)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, wT, z = ctx.saved_tensors
        B, K, R = ctx.shape
        _no_tangent("bf16_linear's gradient", gy)
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dev, bf16 = gy.device, torch.bfloat16
        dx = torch.empty((B, K), dtype=bf16, device=dev) if need_x else None
        dw = torch.empty((R, K), dtype=bf16, device=dev) if need_w else None
        db = torch.empty(R, dtype=bf16, device=dev) if need_b else None
        if B == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif need_x or need_w or need_b:
            g = gy.contiguous()
            stream = _stream_of("bf16_linear's gradient", g, x, wT, z)
            stride = K
            if x is not None:
                x, stride = _rows_of(x)
            if wT is not None:
                wT = _aligned(wT)
            nbytes = lib().mi_bf16_linear_grad_workspace(B, K, R)
            ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
            check("mi_bf16_linear_grad",
                  lib().mi_bf16_linear_grad(_ptr(g), _DTYPES[g.dtype], _ptr(z), ctx.act, _ptr(x), stride, B, _ptr(wT), K, R,
                                            _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, stream))
        return dx, dw, db, gy if need_r else None, None, None


def bf16_linear(x, w, bias=None, act=None, residual=None, dtype=torch.bfloat16, y=None, workspace=None):
    """y = act(x W + bias) + residual: x bf16 [B, n_in] (B up to 2^20, n_in a multiple of 8 up to 65536; rows may be
    strided), w a Bf16Leaf (n_out up to 65536; bf16_project takes a wider vocabulary) or the reference's W bf16 [n_in, n_out],
    transposed in the call; bias bf16 [n_out]; act None, "silu", "gelu", "gelu_tanh" or "relu"; residual [B, n_out] of
    ``dtype`` -> y [B, n_out] of ``dtype`` (bf16 or f32).  ``y`` and
    ``workspace`` (uint8, mi_bf16_linear_workspace bytes, needs no initialisation) make the call allocation-free; gradients
    are recorded without them only."""
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise TypeError("bf16_linear: x must be bf16 [B, n_in], got %s %s" % (x.dtype, tuple(x.shape)))
    if act not in ACTS:
        raise ValueError("bf16_linear: act is one of %s, got %r" % (sorted(ACTS, key=str), act))
    if dtype not in _DTYPES:
        raise TypeError("bf16_linear: y is bf16 or f32, got %s" % dtype)
    wT = w.wT if isinstance(w, Bf16Leaf) else w
    if not isinstance(wT, torch.Tensor) or wT.dtype != torch.bfloat16 or wT.dim() != 2:
        raise TypeError("bf16_linear: the weight must be a Bf16Leaf or bf16 W [n_in, n_out]")
    if wT is w:
        wT = w.t().contiguous()
    (B, K), R = x.shape, wT.shape[0]
    if wT.shape[1] != K:
        raise ValueError("bf16_linear: x has %d columns, the weight takes %d" % (K, wT.shape[1]))
    if bias is not None and (bias.dtype != torch.bfloat16 or tuple(bias.shape) != (R,)):
        raise ValueError("bf16_linear: bias must be bf16 [%d]" % R)
    if residual is not None and (residual.dtype != dtype or tuple(residual.shape) != (B, R)):
        raise ValueError("bf16_linear: residual must be %s [%d, %d]" % (dtype, B, R))
    leaves = [t for t in (x, wT, bias, residual) if t is not None]
    _no_tangent("bf16_linear", *leaves)
    if torch.is_grad_enabled() and any(t.requires_grad for t in leaves):
        if y is not None or workspace is not None:
            raise RuntimeError("bf16_linear: preallocated outputs record no gradient: detach the inputs or call it under "
                               "torch.no_grad()")
        return _Linear.apply(x, wT, bias, residual, ACTS[act], dtype)
    y = _out(y, (B, R), dtype, "bf16_linear", x.device)
    if B:
        _linear(x, wT, bias, ACTS[act], residual, dtype, y, None, workspace)
    return y
