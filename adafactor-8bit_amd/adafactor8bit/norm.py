"""Root-mean-square norm with the residual's addition, its output in the input's type or in MX blocks.

An addition of this build: the norm in front of every projection of the models whose states the
optimizer holds, writing the 8-bit activations that ``mx_matmul`` reads.
"""
import torch
from torch.autograd import forward_ad

from . import _native as nat
from .mx import _DTYPE, _FMT, _RULE, _code, _launch, _new, _on_gpu, _rows, first_order, no_tangents

_DENSE = torch.contiguous_format


def _dense(t):
    return t if t.is_contiguous() and not t.is_neg() else t.resolve_neg().contiguous()


def _forward(x, residual, weight, eps, fmt, keep, rule=0):
    """(y or an MX tensor, h or None, and for a backward pass the bits below h or None, 1 / rms of each row)."""
    rows, cols = x.shape
    dev = x.device
    f = nat.MX_NONE if fmt is None else _FMT[fmt]
    y = torch.empty_like(x, memory_format=_DENSE) if fmt is None else _new(rows, cols, fmt, f, dev)
    h = torch.empty_like(residual, memory_format=_DENSE) if residual is not None else None
    low = h.new_empty((rows, (cols + 7) // 8), dtype=torch.int32) if keep and h is not None and h.element_size() == 2 else None
    rstd = x.new_empty(rows, dtype=torch.float32) if keep else None
    t = _DTYPE[x.dtype]
    _launch("a8_rms_norm", x.get_device(), t, t if h is None else _DTYPE[h.dtype], _DTYPE[weight.dtype],
            f | nat.MX_CEIL if rule else f, x.data_ptr(), x.stride(0),
            None if h is None else residual.data_ptr(), 0 if h is None else residual.stride(0), weight.data_ptr(),
            *((y.data_ptr(), None, None) if fmt is None else (None, *y._addresses()[:2])),
            None if h is None else h.data_ptr(), None if low is None else low.data_ptr(),
            None if rstd is None else rstd.data_ptr(), rows, cols, eps)
    return y, h, low, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        y, h, low, rstd = _forward(x, residual, weight, eps, None, True)
        ctx.save_for_backward(x.contiguous() if h is None else h, low, weight, rstd)
        ctx.dtype, ctx.residual = x.dtype, residual is not None
        return (y, h) if ctx.residual else y

    @staticmethod
    def gradients(ctx, dy, dh=None):
        if dy is None:   # h alone was used: its gradient, as it is
            return (None, None, None, None) if dh is None else (dh.to(ctx.dtype), dh, None, None)
        h, low, weight, rstd = ctx.saved_tensors
        rows, cols = h.shape
        dy = _dense(dy)
        dh = None if dh is None else _dense(dh)
        dx = torch.empty_like(dy)
        dr = torch.empty_like(h) if ctx.residual and h.dtype != ctx.dtype else None
        dw = ws = None
        if ctx.needs_input_grad[2]:   # a frozen weight's gradient is not summed
            dw = torch.empty_like(weight)
            ws = rstd.new_empty(nat.lib().a8_rms_norm_workspace_floats(rows, cols))
        _launch("a8_rms_norm_backward", h.get_device(), _DTYPE[ctx.dtype], _DTYPE[h.dtype], _DTYPE[weight.dtype], dy.data_ptr(),
                None if dh is None else dh.data_ptr(), h.data_ptr(),
                None if low is None else low.data_ptr(), weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                None if dr is None else dr.data_ptr(), None if dw is None else dw.data_ptr(),
                None if ws is None else ws.data_ptr(), rows, cols)
        if not ctx.residual:
            return dx, None, dw, None
        return dx, dx if dr is None else dr, dw, None

    backward = first_order("rms_norm", gradients)


def rms_norm(x, weight, eps=1e-6, residual=None, out_fmt=None, scale="floor"):
    """``h = x + residual`` (h = x without one) and ``y = h / sqrt(mean(h^2) + eps) * weight`` over the
    last dimension.  Returns y, or (y, h) with a residual.

    x is fp32, bf16 or fp16; ``weight`` [cols] and ``residual`` (x's shape) have x's type or fp32; y has
    x's type, h the residual's.  The sum enters the norm, and its gradients, before it is
    rounded to h's type (the gradients: to four bits more than a 16-bit h has, half a byte an element kept for them);
    the gradients have none themselves: ``create_graph`` is refused, as forward-mode derivatives are.  ``out_fmt``
    "mxfp8" or "mxfp4": y is an MXTensor [rows, cols] (leading dimensions flattened) for ``mx_matmul``,
    without gradients, its blocks' scales by the rule ``scale`` ("floor" or "ceil", as mx_quantize has them).
    """
    rule = _code(_RULE, scale, "scale")
    if out_fmt is not None:
        _code(_FMT, out_fmt, "out_fmt")
    shape, dtype, dev = x.shape, x.dtype, x.device
    if not shape or weight.shape != shape[-1:] or shape[-1] < 1:
        raise ValueError(f"adafactor8bit: rms_norm of x {tuple(shape)} with weight {tuple(weight.shape)}")
    if dtype not in _DTYPE:
        raise TypeError(f"adafactor8bit: rms_norm takes fp32, bf16 or fp16, got {dtype}")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise TypeError(f"adafactor8bit: rms_norm's weight is {dtype} or fp32, got {weight.dtype}")
    _on_gpu(x, "rms_norm")
    if weight.device != dev or (residual is not None and residual.device != dev):
        raise ValueError("adafactor8bit: rms_norm's operands are on one device")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"adafactor8bit: rms_norm of x {tuple(shape)} with residual {tuple(residual.shape)}")
        if residual.dtype != dtype and residual.dtype != torch.float32:
            raise TypeError(f"adafactor8bit: rms_norm's residual is {dtype} or fp32, got {residual.dtype}")
    if forward_ad._current_level >= 0:
        no_tangents("rms_norm", x, weight, residual)
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                        or (residual is not None and residual.requires_grad))
    if grad and out_fmt is not None:
        raise ValueError("adafactor8bit: rms_norm's output in MX blocks has no gradient; call it under torch.no_grad()")
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    w = _dense(weight)
    if grad:
        out = _RmsNorm.apply(x2, r2, w, eps)
        y, h = out if r2 is not None else (out, None)
    else:
        y, h, _, _ = _forward(x2, r2, w, eps, out_fmt, False, 0 if out_fmt is None else rule)
    if len(shape) != 2:
        y = y if out_fmt is not None else y.reshape(shape)
        h = None if h is None else h.reshape(shape)
    return y if residual is None else (y, h)
