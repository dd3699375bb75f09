"""Root-mean-square norms of rows with the residual's addition before them, in the rows' type with gradients, or straight
to the e4m3 values and scales that the fp8 products take:

    y, h = rms_norm(x, weight, eps, residual=h)                  h: the stream with x added
    (q, s), h, _ = fp8_rms_norm(x, weight, eps, residual=h)      fp8_project((q, s), leaf), fp8_mlp((q, s), ...)

The squares of a row are added in 64 bits, every later step is a rounding to f32: two calls, or another implementation of
the same steps, give the same bits.

rms_norm records its gradients (x, residual, weight), first order and reverse mode only; sums in f32 in a fixed order,
without atomics.  fp8_rms_norm has none and refuses inputs that require one.  A captured backward pass needs leaves of its
own (``x.detach().requires_grad_()`` inside the capture): an eager graph that still holds the same leaves has bound their
gradients to another stream.  Everything runs on the current torch (HIP) stream of the current device; outputs must not
overlap the inputs or each other.
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import INT_MAX, check, lib
from .fp8 import _DTYPES, FP8, _aligned, _blocks, _no_grad, _no_tangent, _out, _stream_of
from .resident import _ptr


def _rows_of(t, D):
    """(t's rows at a 16-byte address, their stride): as they lie where a kernel can read them so, else a copy."""
    if not t.is_contiguous():
        rows = t if t.dim() == 2 else t.reshape(-1, D)
        stride = rows.stride(0)
        if rows.stride(1) == 1 and stride >= D and stride % 8 == 0 and rows.data_ptr() % 16 == 0:
            return rows, stride
    return _aligned(t), D


def _checked(x, weight, eps, residual, who):
    if x.dtype not in _DTYPES:
        raise TypeError("%s: x must be bf16 or f32, got %s" % (who, x.dtype))
    if weight.dtype not in _DTYPES:
        raise TypeError("%s: weight must be bf16 or f32, got %s" % (who, weight.dtype))
    if not x.dim() or weight.shape != x.shape[-1:]:
        raise ValueError("%s: x is [..., D] and weight [D], got %s and %s" % (who, tuple(x.shape), tuple(weight.shape)))
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError("%s: residual must be %s %s as x is" % (who, x.dtype, tuple(x.shape)))
    if not 0.0 <= eps <= 1e30:
        raise ValueError("%s: eps must be a number from 0 to 1e30, got %r" % (who, eps))


def _like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _launch(x, weight, eps, residual, y, stream, rstd, q, s, hip):
    D = weight.numel()
    x, x_stride = _rows_of(x, D)
    r_stride = 0
    if residual is not None:
        residual, r_stride = _rows_of(residual, D)
    w = _aligned(weight)
    check("mi_rms_norm", lib().mi_rms_norm(x.data_ptr(), _DTYPES[x.dtype], x_stride, _ptr(residual), r_stride, w.data_ptr(),
                                           _DTYPES[w.dtype], min(x.numel() // D, INT_MAX), min(D, INT_MAX), eps, _ptr(y),
                                           _ptr(stream), _ptr(rstd), _ptr(q), _ptr(s), hip))


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        hip = _stream_of("rms_norm", x, weight, residual)
        y = _like(x)
        stream = None if residual is None else _like(x)
        rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        if x.numel():
            _launch(x, weight, eps, residual, y, stream, rstd, None, None, hip)
        ctx.save_for_backward(x if stream is None else stream, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if stream is None else (y, stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gstream=None):
        s, weight, rstd = ctx.saved_tensors
        _no_tangent("rms_norm's gradient", *[g for g in (gy, gstream) if g is not None])
        both = ctx.needs_input_grad[1]
        if gy is None:                            # y was not used
            return gstream, gstream if both else None, None, None
        D, T = weight.numel(), rstd.numel()
        dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if ctx.needs_input_grad[2] else None
        dx = torch.empty(s.shape, dtype=s.dtype, device=s.device)
        if T == 0 or D == 0:
            return dx, dx if both else None, None if dw is None else dw.zero_(), None
        gy = _aligned(gy)
        gstream = None if gstream is None else _aligned(gstream)
        s, s_stride = _rows_of(s, D)
        w = _aligned(weight)
        hip = _stream_of("rms_norm's gradient", gy, s, gstream, w)
        nbytes = lib().mi_rms_norm_grad_workspace(T, D) if dw is not None else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=s.device) if nbytes else None
        check("mi_rms_norm_grad",
              lib().mi_rms_norm_grad(_ptr(gy), _ptr(s), _DTYPES[s.dtype], s_stride, _ptr(gstream), _ptr(w), _DTYPES[w.dtype],
                                     _ptr(rstd), T, D, _ptr(dx), _ptr(dw), _ptr(ws), nbytes, hip))
        return dx, dx if both else None, dw, None


def rms_norm(x, weight, eps=1e-5, residual=None, y=None, stream=None):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last dimension: x bf16 or f32 [..., D] (D a multiple of 8, up to
    32768; up to 2^22 rows, one less where D is past 8192), weight bf16 or f32 [D] -> y as x.  With ``residual`` (as x) s = x + residual, rounded to their type, and the
    result is (y, s): s is the stream that goes on, and y the norm of what it holds.  Rows may be strided.  ``y`` and
    ``stream``: outputs to write into.  Records the gradients of x, residual (the same one) and weight; not into
    preallocated outputs."""
    _checked(x, weight, eps, residual, "rms_norm")
    _no_tangent("rms_norm", x, weight, *(() if residual is None else (residual,)))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        if y is not None or stream is not None:
            raise RuntimeError("rms_norm: preallocated outputs record no gradient: detach the inputs or call it under "
                               "torch.no_grad()")
        return _RmsNorm.apply(x, residual, weight, eps)
    if residual is None and stream is not None:
        raise ValueError("rms_norm: a stream output needs a residual")
    hip = _stream_of("rms_norm", x, weight, residual, y, stream)
    y = _like(x) if y is None else _out(y, x.shape, x.dtype, "rms_norm", x.device)
    if residual is not None:
        stream = _like(x) if stream is None else _out(stream, x.shape, x.dtype, "rms_norm", x.device)
    if x.numel():
        _launch(x, weight, eps, residual, y, stream, None, None, None, hip)
    return y if residual is None else (y, stream)


def fp8_rms_norm(x, weight, eps=1e-5, residual=None, want_y=False, q=None, s=None, y=None, stream=None):
    """rms_norm with its output as fp8_quantize's pair: -> ((q float8_e4m3fn [..., D], scales f32 [..., ceil(D / 128)]),
    stream or None, y or None), ready for the fp8 products.  D a multiple of 16.  Quantised from the f32 values of the norm,
    by fp8_quantize's rule, so each value is rounded once; with ``want_y`` (or ``y``) the norm in x's type too, for a router
    that reads the same rows.  ``q``, ``s``, ``y``, ``stream``: outputs to write into."""
    _checked(x, weight, eps, residual, "fp8_rms_norm")
    _no_grad("fp8_rms_norm", x, weight, *(() if residual is None else (residual,)))
    if residual is None and stream is not None:
        raise ValueError("fp8_rms_norm: a stream output needs a residual")
    D = x.shape[-1]
    hip = _stream_of("fp8_rms_norm", x, weight, residual, q, s, y, stream)
    q = _out(q, x.shape, FP8, "fp8_rms_norm", x.device)
    s = _out(s, x.shape[:-1] + (_blocks(D),), torch.float32, "fp8_rms_norm", x.device)
    if want_y or y is not None:
        y = _out(y, x.shape, x.dtype, "fp8_rms_norm", x.device)
    if residual is not None:
        stream = _like(x) if stream is None else _out(stream, x.shape, x.dtype, "fp8_rms_norm", x.device)
    if x.numel():
        _launch(x, weight, eps, residual, y, stream, None, q, s, hip)
    return (q, s), stream, y
