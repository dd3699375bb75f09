"""Tokens into expert order and back over the layout of ``ragged_plan`` (pallas_moe.py:564-592), the gather and the
combine around the ragged products (resident.py:153-165), with their gradients:

    plan = ragged_plan(idx, w, E, tm)
    xs   = moe_dispatch(x, plan)            [Rp, D]; the experts' products of xs give y [Rp, D]
    out  = moe_combine(y, plan, w)          [T, D]

Both record gradients (x; y and w), first order and reverse mode only (a forward-mode tangent is refused), and save no
copies: the rows a backward pass reads are the forward's own inputs (y only where w requires a gradient).  Deterministic:
no atomics, sums in f32 in column order, one rounding.  A captured backward pass needs leaves of its own
(``x.detach().requires_grad_()`` inside the capture): an eager graph that still holds the same leaves has bound their
gradients to another stream.

The products of this package have no gradient with respect to the rows (fp8_grouped refuses rows that require one), so a
gradient of x, or of y, flows through products of the caller's own between the two; that of w needs none.  A plan has at
least one token, and no two of its slots share a row.
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from .fp8 import _DTYPES, _aligned, _no_tangent, _stream_of
from .resident import _as, _ptr, _stream


def _rows_dtype(t, who):
    if t.dtype not in _DTYPES:
        raise TypeError("%s: rows are bf16 or f32, got %s" % (who, t.dtype))
    if t.dim() != 2:
        raise ValueError("%s: rows are [n, D]" % who)


def _plan_rows(plan):
    """(tok_row [Rp], row_slot [T, k]) of a plan, contiguous int32."""
    tok, slot = _as(plan["tok_row"], torch.int32), _as(plan["row_slot"], torch.int32)
    if tok.dim() != 1 or slot.dim() != 2:
        raise ValueError("a plan holds tok_row [Rp] and row_slot [T, k]")
    return tok, slot


def _dispatch(x, tok, slot):
    xs = torch.empty((tok.numel(), x.shape[1]), dtype=x.dtype, device=x.device)
    T, k = slot.shape
    check("mi_moe_dispatch", lib().mi_moe_dispatch(_ptr(x), _DTYPES[x.dtype], T, k, x.shape[1], _ptr(slot), _ptr(tok),
                                                   tok.numel(), _ptr(xs), _stream()))
    return xs


def _combine(y, slot, w):
    T, k = slot.shape
    out = torch.empty((T, y.shape[1]), dtype=y.dtype, device=y.device)
    check("mi_moe_combine", lib().mi_moe_combine(_ptr(y), _DTYPES[y.dtype], T, k, y.shape[1], _ptr(slot), _ptr(w),
                                                 y.shape[0], _ptr(out), _stream()))
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tok, slot):
        ctx.save_for_backward(slot)
        return _dispatch(x, tok, slot)

    @staticmethod
    @once_differentiable
    def backward(ctx, gxs):
        slot, = ctx.saved_tensors
        _no_tangent("moe_dispatch's gradient", gxs)
        return _combine(_aligned(gxs), slot, None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, w, tok, slot):
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, w, tok, slot)     # only dw is made of y
        return _combine(y, slot, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        y, w, tok, slot = ctx.saved_tensors
        _no_tangent("moe_combine's gradient", gout)
        gout = _aligned(gout)
        T, k = slot.shape
        rows, D = tok.numel(), gout.shape[1]
        dy = torch.empty((rows, D), dtype=gout.dtype, device=gout.device)
        dw = torch.empty_like(w) if y is not None else None
        check("mi_moe_combine_grad",
              lib().mi_moe_combine_grad(_ptr(gout), _ptr(y), _DTYPES[gout.dtype], T, k, D, _ptr(slot), _ptr(tok), _ptr(w),
                                        rows, _ptr(dy), _ptr(dw), _stream()))
        return dy, dw, None, None


def moe_dispatch(x, plan):
    """Tokens into expert order: x bf16 or f32 [T, D] (D a multiple of 8), plan = ragged_plan(idx, w, E, tm) ->
    xs [Rp, D] of x's dtype, xs[row_slot[t, j]] = x[t], zeros on all other rows (padding, and rows of slots that the
    caller has taken out: row_slot -1).  Records the gradient of x: the sum over a token's rows."""
    _rows_dtype(x, "moe_dispatch")
    _no_tangent("moe_dispatch", x)
    tok, slot = _plan_rows(plan)
    if slot.shape[0] != x.shape[0]:
        raise ValueError("moe_dispatch: the plan is of %d tokens, x has %d" % (slot.shape[0], x.shape[0]))
    _stream_of("moe_dispatch", x, tok, slot)
    x = _aligned(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, tok, slot)
    return _dispatch(x, tok, slot)


def moe_combine(y, plan, w):
    """The way back: y bf16 or f32 [Rp, D] in the plan's row order, w f32 [T, k] -> out [T, D] of y's dtype, out[t] =
    sum_j w[t, j] * y[row_slot[t, j]] in f32, in column order, rounded once; a slot without a row (an expert id outside
    [0, E), or row_slot set to -1) adds nothing.  Records the gradients of y (zeros on rows without a slot) and w."""
    _rows_dtype(y, "moe_combine")
    _no_tangent("moe_combine", y, w)
    tok, slot = _plan_rows(plan)
    if tok.numel() != y.shape[0]:
        raise ValueError("moe_combine: the plan has %d rows, y %d" % (tok.numel(), y.shape[0]))
    if w.dtype != torch.float32 or w.shape != slot.shape:
        raise ValueError("moe_combine: w must be float32 %s" % (tuple(slot.shape),))
    _stream_of("moe_combine", y, w, tok, slot)
    y, w = _aligned(y), w.contiguous()
    if (y.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(y, w, tok, slot)
    return _combine(y, slot, w)
