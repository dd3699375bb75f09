"""A router's logits to the experts of each token and their weights, with the gradient of the logits:

    idx, w = moe_gate(logits, k, scores="sigmoid", bias=b, n_group=8, topk_group=4)
    plan = ragged_plan(idx, w, E, tm); out = moe_combine(experts(moe_dispatch(x, plan)), plan, w)

``route`` is the reference's router from hidden states to the same pair, with sigmoid scores, no groups and no gradient; a
gradient of w that moe_combine returns goes on here to the logits and the router behind them.  First order and reverse mode
only (a forward-mode tangent is refused); the balancing bias only chooses and has no gradient.  Deterministic, without
atomics.  A captured backward pass needs leaves of its own (``logits.detach().requires_grad_()`` inside the capture): an
eager graph that still holds the same leaves has bound their gradients to another stream.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import INT_MAX, check, lib
from .fp8 import _DTYPES, _no_tangent, _stream_of
from .resident import _ptr

SCORES = {"sigmoid": _lib.MI_GATE_SIGMOID, "softmax": _lib.MI_GATE_SOFTMAX}


def _rows(t):
    """(t, its row stride): as it lies where its rows are, else a contiguous copy."""
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t, t.stride(0)
    return t.contiguous(), t.shape[1]


def _gate(logits, args):
    bias, k, scores, n_group, topk_group, group_top, norm, scaling = args
    T, E = logits.shape
    stream = _stream_of("moe_gate", logits, bias)
    dev = logits.device
    idx = torch.empty((T, k), dtype=torch.int32, device=dev)
    w = torch.empty((T, k), dtype=torch.float32, device=dev)
    if T:
        l, stride = _rows(logits)
        check("mi_moe_gate", lib().mi_moe_gate(l.data_ptr(), _DTYPES[l.dtype], stride, _ptr(bias), min(T, INT_MAX), E, k, scores,
                                               n_group, topk_group, group_top, norm, scaling, idx.data_ptr(), w.data_ptr(), stream))
    return idx, w


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args):
        idx, w = _gate(logits, args)
        ctx.save_for_backward(logits, idx)
        ctx.args = args
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return idx, w

    @staticmethod
    @once_differentiable
    def backward(ctx, _, gw):
        if gw is None:
            return None, None
        logits, idx = ctx.saved_tensors
        _no_tangent("moe_gate's gradient", gw)
        bias, k, scores, n_group, topk_group, group_top, norm, scaling = ctx.args
        gw = gw.contiguous()
        T, E = logits.shape
        dl = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
        stream = _stream_of("moe_gate's gradient", logits, gw)
        if T:
            l, stride = _rows(logits)
            check("mi_moe_gate_grad", lib().mi_moe_gate_grad(l.data_ptr(), _DTYPES[l.dtype], stride, idx.data_ptr(),
                                                             gw.data_ptr(), T, E, k, scores, norm, scaling, dl.data_ptr(), stream))
        return dl, None


def moe_gate(logits, k, scores="sigmoid", bias=None, n_group=1, topk_group=1, group_top=2, norm_topk=True, scaling=1.0):
    """logits bf16 or f32 [T, E] -> (idx int32 [T, k], w f32 [T, k]).  s = sigmoid(logits) or softmax(logits), the choices
    c = s + bias (f32 [E]); with ``n_group`` > 1 (a power of two, up to 32) the E / n_group consecutive experts of a group
    stay if it is one of the ``topk_group`` with the largest sum of their ``group_top`` (1 or 2) largest choices; idx = the k
    largest choices (equal ones: the lower id), w = s[idx], divided by their sum + 1e-20 with ``norm_topk``, times
    ``scaling``.  E up to 1024, k up to 32, T up to 2^22.

    An expert whose logit is -inf is out of service.  A slot that no expert is left for has id -1 and weight 0, which
    ragged_plan, fp8_moe and moe_combine take as nothing.  Choices are compared in 64 bits (within 2^-42 of each other's size
    they count as equal; without a bias the logits themselves order the experts of the groups that stay), and one that is no
    number counts as the largest.  Records the gradient of the logits."""
    kind = SCORES.get(scores)
    if kind is None:
        raise ValueError("moe_gate: scores are 'sigmoid' or 'softmax', got %r" % (scores,))
    if logits.dtype not in _DTYPES:
        raise TypeError("moe_gate: logits are bf16 or f32, got %s" % logits.dtype)
    if logits.dim() != 2:
        raise ValueError("moe_gate: logits are [T, E]")
    E = logits.shape[1]
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E,):
            raise ValueError("moe_gate: bias must be float32 [%d]" % E)
        if bias.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("moe_gate: the bias only chooses and has no gradient: detach it")
        _no_tangent("moe_gate", bias)
        bias = bias.contiguous()
    _no_tangent("moe_gate", logits)
    if not 0 < E <= 1024 or not 0 < k <= min(E, 32):
        raise ValueError("moe_gate: 1 to 1024 experts and k up to them and 32, got %d and %d" % (E, k))
    if not 1 <= n_group <= 32 or n_group & (n_group - 1) or E % n_group:
        raise ValueError("moe_gate: n_group must be a power of two up to 32 that divides %d experts, got %d" % (E, n_group))
    if not 1 <= topk_group <= n_group or k > E // n_group * topk_group:
        raise ValueError("moe_gate: %d of %d groups do not hold %d experts" % (topk_group, n_group, k))
    if group_top not in (1, 2):
        raise ValueError("moe_gate: a group counts by its 1 or 2 largest choices, got %r" % (group_top,))
    args = (bias, int(k), kind, int(n_group), int(topk_group), int(group_top), 1 if norm_topk else 0, float(scaling))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Gate.apply(logits, args)
    return _gate(logits, args)
