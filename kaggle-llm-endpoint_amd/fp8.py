"""Products over block-scaled fp8 weights: the layout of fp8 checkpoints (checkpoint.py:202), e4m3 values with one f32
scale per 128 x 128 block, contracted as fp8 on the matrix cores with activations quantised per row and 128 columns.

    q, s = fp8_quantize(x)                              rows of activations, once for several products
    y    = fp8_project(x, leaf)                         a dense projection
    y    = fp8_mlp(x, gate, up, down, limit)            mlp_partial's products (mlp_partial calls it for such leaves)
    y    = fp8_grouped(xs, plan, leaf)                  the sorted rows of a ragged_plan, each times its expert's matrix
    o, _ = fp8_moe(gate, up, down, x, idx, w, limit)    the routed experts of a layer

Products are exact and summed in f32, but for those of 8 consecutive columns, which the fp8 matrix instruction adds on a grid
of 2^-13 of the largest one: 1.3e-5 of a result (root mean square), of f32 outputs too.  Gate and up of fp8_mlp up to 128 rows
and of fp8_moe up to 96 slots an expert (T k / E) are summed in f32 throughout, since h is quantised again and a last bit may
move a value by a step of e4m3; of larger calls they are not, so that a row's result may differ, within that, with the
number of rows in its call.

Everything runs on the current torch (HIP) stream of the current device.  The weights are a checkpoint's and the
products have no gradient: an input (rows, weights, scales, routing weights) that requires one is refused while gradients are
recorded, and one that carries a forward-mode tangent always.  Outputs and workspaces must not overlap the inputs or each other.
"""
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib
from .resident import _as, _ptr

BLOCK = 128                     # columns per activation scale; rows and columns per weight scale
FP8 = torch.float8_e4m3fn


def _blocks(n):
    return -(-n // BLOCK)


class Fp8Leaf(NamedTuple):
    """Block-scaled weights on the device: q e4m3 [n_out, n_in] (or [E, n_out, n_in] of E experts), s f32
    [..., ceil(n_out / 128), ceil(n_in / 128)]; a weight is f32(q) * s of its block."""
    q: torch.Tensor
    s: torch.Tensor


def fp8_leaf(leaf, device="cuda"):
    """{"q": float8_e4m3fn [..., n_out, n_in], "s": [..., ceil(n_out / 128), ceil(n_in / 128)]}, as a checkpoint stores
    a matrix (or E of them) and its scales -> Fp8Leaf on the device."""
    q, s = (leaf["q"], leaf["s"]) if isinstance(leaf, dict) else leaf
    leaf = Fp8Leaf(q.detach().to(device).contiguous(), s.detach().to(device=device, dtype=torch.float32).contiguous())
    _leaf_dims(leaf, "fp8_leaf")
    return leaf


def _leaf_dims(leaf, who):
    """(E, n_out, n_in) of an Fp8Leaf, its types and shapes checked; E is 0 for one matrix."""
    q, s = leaf
    qs, ss = q.shape, s.shape
    n = len(qs)
    if q.dtype is not FP8 or s.dtype is not torch.float32:
        raise TypeError("%s: weights are float8_e4m3fn with float32 scales (got %s, %s)" % (who, q.dtype, s.dtype))
    if n not in (2, 3) or len(ss) != n:
        raise ValueError("%s: weights are [n_out, n_in] or [E, n_out, n_in], scales likewise" % who)
    R, K = qs[n - 2], qs[n - 1]
    E = qs[0] if n == 3 else 0
    if ss[n - 2] != -(-R // BLOCK) or ss[n - 1] != -(-K // BLOCK) or (E and ss[0] != E):
        raise ValueError("%s: scales %s do not fit weights %s: one per 128 x 128 block" % (who, tuple(ss), tuple(qs)))
    if not (q.is_contiguous() and s.is_contiguous()):
        raise ValueError("%s: weights and scales must be contiguous (fp8_leaf makes them so)" % who)
    _no_grad(who, q, s)
    return E, R, K


def _stream_of(who, *tensors):
    """The current stream; every tensor has to be on the current device, whose stream the call runs on."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError("%s: every tensor must be on the current device (cuda:%d), got one on %s" % (who, dev,
                                                                                                       t.device))
    return torch._C._cuda_getCurrentRawStream(dev)


def _no_tangent(who, *tensors):
    """A tangent would be lost without a word: a dual tensor does not require a gradient, and its address is read."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("%s has no forward-mode derivative: call it on the primal (forward_ad.unpack_dual)" % who)


def _no_grad(who, *tensors):
    if forward_ad._current_level >= 0:
        _no_tangent(who, *tensors)
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("%s has no gradient: detach its inputs or call it under torch.no_grad()" % who)


def _aligned(t):
    """t contiguous, at a 16-byte address (a copy when it is not)."""
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _out(t, shape, dtype, who, device):
    """A caller's output checked, or a new one."""
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous():
        raise ValueError("%s: an output must be a contiguous %s tensor of shape %s" % (who, dtype, tuple(shape)))
    return t


def _workspace(workspace, need, device):
    """(tensor, address, bytes) of a call's workspace: the caller's, or the call's own, since two captured calls would
    share a kept one (the caller of this holds the tensor until its launches are queued).  need 0: none (or a shape that
    the call refuses)."""
    if workspace is None:
        if need == 0:
            return None, None, 0
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif not workspace.is_contiguous():
        raise ValueError("a workspace must be contiguous: a view's elements may be more than its memory")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


_DTYPES = {torch.bfloat16: _lib.MI_X_BF16, torch.float32: _lib.MI_X_F32}


def _rows_of(x, K, who):
    """(rows, scales or None, dtype code) of a product's activations: bf16 or f32 [B, K], or fp8_quantize's pair."""
    if isinstance(x, (tuple, list)):
        q, s = x
        if q.dtype != FP8 or s.dtype != torch.float32:
            raise TypeError("%s: quantised activations are (float8_e4m3fn, float32 scales)" % who)
        if q.dim() != 2 or tuple(s.shape) != (q.shape[0], _blocks(q.shape[1])):
            raise ValueError("%s: quantised activations are q [B, n_in] with s [B, ceil(n_in / 128)]" % who)
        _no_grad(who, q, s)
        x, xs, dtype = _aligned(q), s.contiguous(), _lib.MI_X_FP8
    else:
        xs, dtype = None, _DTYPES.get(x.dtype)
        if dtype is None:
            raise TypeError("%s: activations are bf16 or f32 (or fp8_quantize's pair), got %s" % (who, x.dtype))
        if x.dim() != 2:
            raise ValueError("%s: activations are [B, n_in]" % who)
        _no_grad(who, x)
        x = _aligned(x)
    if x.shape[1] != K:
        raise ValueError("%s: activations have %d columns, the weight %d" % (who, x.shape[1], K))
    return x, xs, dtype


def fp8_quantize(x, q=None, s=None):
    """x bf16 or f32 [..., K], K a multiple of 16 -> (q float8_e4m3fn [..., K], s f32 [..., ceil(K / 128)]): per row and
    group of 128 columns s = 2^e, the least e >= -100 with max |x| <= 448 * 2^e over the group's finite values, and
    q = x / s to nearest even; infinities and NaN become NaN.  A power of two, so that x / s is exact and each value is
    rounded once.  Rows may be strided.  ``q`` and ``s``: outputs to write into."""
    dtype, shape = _DTYPES.get(x.dtype), x.shape
    if dtype is None:
        raise TypeError("fp8_quantize: x must be bf16 or f32, got %s" % x.dtype)
    if not shape:
        raise ValueError("fp8_quantize: x must have at least one dimension")
    _no_grad("fp8_quantize", x)
    K = shape[-1]
    q = _out(q, shape, FP8, "fp8_quantize", x.device)
    s = _out(s, shape[:-1] + (_blocks(K),), torch.float32, "fp8_quantize", x.device)
    size = x.numel()
    if size == 0:
        return q, s
    stream = _stream_of("fp8_quantize", x, q, s)
    n = size // K
    x2 = x if len(shape) == 2 else x.reshape(n, K)
    if x2.is_contiguous():
        stride = -(-K // 8) * 8 if n == 1 else K
        x2 = _aligned(x2)
    else:
        stride = x2.stride(0)
        if x2.stride(1) != 1 or stride < K or stride % 8 or x2.data_ptr() % 16:
            x2, stride = _aligned(x2), K
    check("mi_fp8_quantize", lib().mi_fp8_quantize(x2.data_ptr(), dtype, n, K, stride, q.data_ptr(), s.data_ptr(), stream))
    return q, s


def fp8_project(x, leaf, want_f32=False, y_bf16=None, y_f32=None, workspace=None):
    """y = x W^T over a block-scaled leaf (Fp8Leaf, [n_out, n_in], any n_out, n_in a multiple of 16): x bf16 or f32
    [B, n_in], quantised as by fp8_quantize, or that function's pair.  -> y bf16 [B, n_out]
    (and y f32 with want_f32).  Preallocated outputs and ``workspace`` (uint8, mi_fp8_project_workspace bytes, needs no
    initialisation) make the call allocation-free."""
    E, R, K = _leaf_dims(leaf, "fp8_project")
    if E:
        raise ValueError("fp8_project: the weight must be one matrix [n_out, n_in]")
    x, xs, dtype = _rows_of(x, K, "fp8_project")
    B = x.shape[0]
    yb = _out(y_bf16, (B, R), torch.bfloat16, "fp8_project", x.device)
    yf = _out(y_f32, (B, R), torch.float32, "fp8_project", x.device) if want_f32 or y_f32 is not None else None
    if B:
        stream = _stream_of("fp8_project", x, xs, leaf.q, leaf.s, yb, yf, workspace)
        held, ws, nbytes = _workspace(workspace, lib().mi_fp8_project_workspace(B, K, R), x.device)
        check("mi_fp8_project", lib().mi_fp8_project(x.data_ptr(), dtype, _ptr(xs), B, _ptr(leaf.q), _ptr(leaf.s), K, R,
                                                     _ptr(yb), _ptr(yf), ws, nbytes, stream))
    return (yb, yf) if want_f32 else yb


def _mlp_dims(gate, up, down, who):
    E, I, D = _leaf_dims(gate, who)
    if _leaf_dims(up, who) != (E, I, D) or _leaf_dims(down, who) != (E, D, I):
        raise ValueError("%s: gate and up must be [.., I, D] and down [.., D, I], got %s, %s, %s"
                         % (who, tuple(gate.q.shape), tuple(up.q.shape), tuple(down.q.shape)))
    return E, I, D


def fp8_mlp(x, gate, up, down, limit, want_f32=False, y_bf16=None, y_f32=None, workspace=None):
    """mlp_partial over block-scaled leaves (model.py:125-127): g, u = x Wg^T, x Wu^T as f32 values,
    h = silu(min(g, limit)) * clip(u, -limit, limit) (limit > 0), quantised as by fp8_quantize, y = h Wd^T.  x as for fp8_project;
    gate, up [I, D], down [D, I].  -> y bf16 [B, D] (and y f32 with want_f32).  Preallocated outputs and ``workspace``
    (mi_fp8_mlp_workspace bytes) make the call allocation-free."""
    E, I, D = _mlp_dims(gate, up, down, "fp8_mlp")
    if E:
        raise ValueError("fp8_mlp: gate, up and down are one matrix each")
    x, xs, dtype = _rows_of(x, D, "fp8_mlp")
    B = x.shape[0]
    yb = _out(y_bf16, (B, D), torch.bfloat16, "fp8_mlp", x.device)
    yf = _out(y_f32, (B, D), torch.float32, "fp8_mlp", x.device) if want_f32 or y_f32 is not None else None
    if B:
        stream = _stream_of("fp8_mlp", x, xs, *gate, *up, *down, yb, yf, workspace)
        held, ws, nbytes = _workspace(workspace, lib().mi_fp8_mlp_workspace(B, D, I), x.device)
        check("mi_fp8_mlp", lib().mi_fp8_mlp(x.data_ptr(), dtype, _ptr(xs), B, D, I, _ptr(gate.q), _ptr(gate.s),
                                             _ptr(up.q), _ptr(up.s), _ptr(down.q), _ptr(down.s), float(limit), _ptr(yb),
                                             _ptr(yf), ws, nbytes, stream))
    return (yb, yf) if want_f32 else yb


def fp8_grouped(xs, plan, leaf, want_f32=False, y_bf16=None, y_f32=None, workspace=None):
    """The sorted rows of a ragged_plan (tm 16, 32, 64 or 128), each times its expert's matrix of ``leaf`` [E, R, K]: xs
    bf16 or f32 [Rp, K] (moe_dispatch's rows) or fp8_quantize's pair -> y bf16 [Rp, R] (and y f32 with want_f32), ready
    for moe_combine.  Rows of blocks that the plan does not use, and padding rows, are zero."""
    E, R, K = _leaf_dims(leaf, "fp8_grouped")
    if not E:
        raise ValueError("fp8_grouped: the weights must be [E, R, K]")
    x, xs, dtype = _rows_of(xs, K, "fp8_grouped")
    blk, nb, tok = [_as(plan[k], torch.int32) for k in ("blk_expert", "n_blocks", "tok_row")]
    rows, G = x.shape[0], blk.numel()
    if rows != tok.numel() or nb.numel() != 1 or G == 0 or rows % G:
        raise ValueError("fp8_grouped: %d rows do not fit the plan's %d rows in %d blocks" % (rows, tok.numel(), G))
    yb = _out(y_bf16, (rows, R), torch.bfloat16, "fp8_grouped", x.device)
    yf = _out(y_f32, (rows, R), torch.float32, "fp8_grouped", x.device) if want_f32 or y_f32 is not None else None
    stream = _stream_of("fp8_grouped", x, xs, blk, nb, tok, leaf.q, leaf.s, yb, yf, workspace)
    held, ws, nbytes = _workspace(workspace, lib().mi_fp8_grouped_workspace(rows, K, R), x.device)
    check("mi_fp8_grouped", lib().mi_fp8_grouped(x.data_ptr(), dtype, _ptr(xs), G, rows // G, _ptr(blk), _ptr(nb),
                                                 _ptr(tok), _ptr(leaf.q), _ptr(leaf.s), E, K, R, _ptr(yb), _ptr(yf), ws, nbytes,
                                                 stream))
    return (yb, yf) if want_f32 else yb


def fp8_moe(gate, up, down, x, idx, w, limit, want_f32=True, want_bf16=False, out_f32=None, out_bf16=None,
            workspace=None):
    """The routed experts of one layer over block-scaled weights, for one token or a whole prompt piece: out[t] =
    sum_j w[t, j] * MLP_{idx[t, j]}(x[t]) with the MLP of fp8_mlp, whose y stays f32 until the sum is rounded.  gate, up
    [E, I, D], down [E, D, I] (Fp8Leaf); x bf16 or f32 [T, D]; idx int32 (or int64) [T, k]; w f32 [T, k] -> (out_f32 [T, D]
    or None, out_bf16 [T, D] or None).  A slot whose expert id is outside [0, E) adds nothing.  Preallocated outputs and
    ``workspace`` (mi_fp8_moe_workspace bytes) make the call allocation-free."""
    E, I, D = _mlp_dims(gate, up, down, "fp8_moe")
    if not E:
        raise ValueError("fp8_moe: gate, up and down must be [E, ..] experts")
    if isinstance(x, (tuple, list)):
        raise TypeError("fp8_moe: activations are bf16 or f32")
    x, _, dtype = _rows_of(x, D, "fp8_moe")
    if idx.dim() != 2 or w.shape != idx.shape or idx.shape[0] != x.shape[0]:
        raise ValueError("fp8_moe: idx and w must be [T, k] for the %d tokens of x" % x.shape[0])
    _no_grad("fp8_moe", w)
    if idx.dtype == torch.int64:
        idx = idx.clamp(-1, E)                    # (an id outside the range must not wrap into it)
    idx, w = _as(idx, torch.int32), _as(w, torch.float32)
    T, k = idx.shape
    of, ob = out_f32, out_bf16
    if of is not None or want_f32:
        of = _out(of, (T, D), torch.float32, "fp8_moe", x.device)
    if ob is not None or want_bf16:
        ob = _out(ob, (T, D), torch.bfloat16, "fp8_moe", x.device)
    if T:
        stream = _stream_of("fp8_moe", x, idx, w, *gate, *up, *down, of, ob, workspace)
        held, ws, nbytes = _workspace(workspace, lib().mi_fp8_moe_workspace(T, k, E, D, I), x.device)
        check("mi_fp8_moe", lib().mi_fp8_moe(_ptr(gate.q), _ptr(gate.s), _ptr(up.q), _ptr(up.s), _ptr(down.q),
                                             _ptr(down.s), E, D, I, x.data_ptr(), dtype, T, k, _ptr(idx), _ptr(w),
                                             float(limit), _ptr(of), _ptr(ob), ws, nbytes, stream))
    return of, ob
