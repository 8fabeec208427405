"""Microscaled (MX) matrices: blocks of 32 elements with a shared power-of-two scale, in 4 or 8
bits, their products on the matrix cores, and a linear layer made of them.

An addition of this build (the reference holds optimizer states in blocks of 8 and 4 bits; these
are the weights, activations and gradients next to it).  Formats:

    mxfp4   E2M1 codes, two a byte (0 0.5 1 1.5 2 3 4 6 and their negatives)
    mxfp8   E4M3 codes, one a byte (to 448)

A block's scale is 2^e with e = floor(log2 max|v|) - 2 or - 8 (``scale="floor"``, the formats' own
rule, under which the block's largest elements may saturate) or the next power of two where it
would saturate (``scale="ceil"``).  A block that holds a NaN or an infinity reads as NaN.
"""
import math
import operator

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _native as nat

_FMT = {"mxfp4": nat.MXFP4, "mxfp8": nat.MXFP8}
_DTYPE = {torch.float32: nat.F32, torch.bfloat16: nat.BF16, torch.float16: nat.F16}
_RULE = {"floor": 0, "ceil": 1}
_MASK64 = (1 << 64) - 1


def _code(table, key, what):
    try:
        return table[key]
    except (KeyError, TypeError):
        raise ValueError(f"adafactor8bit: {what} must be one of {', '.join(map(str, table))}, got {key!r}") from None


def _seed(seed):
    """None, or the whole number's low 64 bits."""
    if seed is None:
        return None
    try:
        return operator.index(seed) & _MASK64
    except TypeError:
        raise TypeError(f"adafactor8bit: seed must be None or a whole number, got {seed!r}") from None


def _pitch(cols):   # no shifts or masks here and in _bytes: torch.compile's symbolic sizes have none
    return (cols + 255) // 256 * 256


class MXTensor:
    """A [rows, cols] matrix in blocks of 32 along its rows.

    ``codes``: uint8 [rows, P] (mxfp8) or [rows, P / 2] (mxfp4, the even element in the low half);
    ``scales``: uint8 [rows, P / 32], byte b for 2^(b - 127) and 255 for NaN; P is ``cols`` rounded
    up to 256, and the codes beyond ``cols`` are 0.  Both on the GPU, contiguous, 16-byte aligned.
    """
    # keep: the codes and the scales, or the one buffer that holds both; f: the format's number.  Addresses are
    # read from `keep` for every call: a copy of the object, or parts whose memory was replaced, have others
    __slots__ = ("rows", "cols", "fmt", "f", "keep")

    def __init__(self, codes, scales, cols, fmt):
        f = _code(_FMT, fmt, "fmt")
        if cols < 0:
            raise ValueError(f"adafactor8bit: an MX tensor of {cols} columns")
        p = _pitch(cols)
        rows = codes.shape[0] if codes.dim() else 0
        if codes.shape != (rows, p if f else p // 2) or scales.shape != (rows, p // 32):
            raise ValueError(f"adafactor8bit: a {fmt} tensor of {cols} columns has codes [rows, {p if f else p // 2}] and "
                             f"scales [rows, {p // 32}], got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("adafactor8bit: codes and scales of an MX tensor are uint8")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("adafactor8bit: codes and scales of an MX tensor are contiguous")
        if codes.device != scales.device:
            raise ValueError("adafactor8bit: codes and scales of an MX tensor are on one device")
        self.rows, self.cols, self.fmt, self.f, self.keep = rows, cols, fmt, f, (codes, scales)

    def __reduce__(self):   # copies and pickles are made of the parts
        return MXTensor, (self.codes, self.scales, self.cols, self.fmt)

    def _addresses(self):
        """Of the codes and the scales, and the number of the GPU that they are on (-1: none)."""
        keep = self.keep
        codes = keep[0]
        at = codes.data_ptr()
        if len(keep) == 1:
            return at, at + self.rows * (_pitch(self.cols) // (2 - self.f)), codes.get_device()
        i = codes.get_device()
        return at, keep[1].data_ptr(), i if keep[1].get_device() == i else -1

    def _split(self):
        if len(self.keep) == 1:   # one buffer from _over: the codes, then the scales
            buf, p = self.keep[0], _pitch(self.cols)
            n = self.rows * (p if self.f else p // 2)
            self.keep = (buf[:n].view(self.rows, -1) if n else buf[:0].view(self.rows, p if self.f else p // 2),
                         buf[n:].view(self.rows, p // 32))
        return self.keep

    @property
    def codes(self):
        return self._split()[0]

    @property
    def scales(self):
        return self._split()[1]

    @property
    def device(self):
        return self.keep[0].device

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    def __repr__(self):
        return f"MXTensor({self.fmt}, shape={tuple(self.shape)}, device={self.device})"


def _over(buf, rows, cols, fmt, f):
    """An MX tensor over a buffer of _bytes(rows, cols, f) bytes."""
    t = object.__new__(MXTensor)
    t.rows, t.cols, t.fmt, t.f, t.keep = rows, cols, fmt, f, (buf,)
    return t


def _bytes(rows, cols, f):
    p = _pitch(cols)
    return rows * (p // (2 - f) + p // 32)


def _new(rows, cols, fmt, f, device):
    """An MX tensor to be written."""
    return _over(torch.empty(_bytes(rows, cols, f), dtype=torch.uint8, device=device), rows, cols, fmt, f)


def _on_gpu(x, what):
    if not x.is_cuda:
        raise RuntimeError(f"adafactor8bit: {what} runs on the GPU only, got a tensor on {x.device}")


def no_tangents(what, *tensors):
    """A launch that autograd does not see carries no tangent on: its result would read as a constant.  (Called
    where a dual level is entered, forward_ad._current_level >= 0.)"""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"adafactor8bit: {what} has no forward-mode derivative, got a dual tensor")


def _mx(t, what):
    if not isinstance(t, MXTensor):
        raise TypeError(f"adafactor8bit: {what} takes an MXTensor, got {type(t).__name__}")


def _not_on_gpu(t, what):
    return RuntimeError(f"adafactor8bit: {what} runs on the GPU only, got an MX tensor on {t.keep[0].device} and {t.keep[-1].device}")


_fn = {}
_jit_traces, _modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
_pre_dispatch = torch._ops.mode_stack_state_for_pre_dispatch()
_current, _stream = (getattr(torch._C, n, None) for n in ("_cuda_getDevice", "_cuda_getCurrentRawStream"))


def _launch(name, i, *args):
    """A library call on the current stream of GPU i, with that GPU current."""
    # under torch.jit.trace, make_fx or an export (the shorter questions first: 0.3 us)
    if _jit_traces() or _pre_dispatch.get(0) is not None or (_modes() and get_proxy_mode() is not None):
        raise RuntimeError(f"adafactor8bit: {name} cannot be traced: the trace would hold its output's allocation, not its launch")
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(nat.lib(), name)
    if i == _current():
        rc = fn(*args, _stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _stream(i))
    if rc:
        nat.check(rc, name)


def _rows(x):
    """x as a matrix of its last dimension's rows, whose elements are adjacent (a copy where they are not, or
    where their sign is still to be applied)."""
    if x.is_neg():
        x = x.resolve_neg()
    if x.dim() != 2:
        x = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    if x.is_contiguous():
        return x
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def _quantize(x, fmt, f, along, down, rule, seed):
    """(along the rows or None, down the columns or None) of a matrix from _rows."""
    rows, cols = x.shape
    dev = x.device
    a = _new(rows, cols, fmt, f, dev) if along else None
    d = _new(cols, rows, fmt, f, dev) if down else None
    _launch("a8_mx_quantize", x.get_device(), _DTYPE[x.dtype], f, rule, seed is not None, x.data_ptr(), rows, cols,
            x.stride(0) if rows > 1 and cols else cols, *(a._addresses()[:2] if along else (None, None)),
            *(d._addresses()[:2] if down else (None, None)), seed or 0)
    return a, d


def mx_quantize(x, fmt="mxfp8", axis=1, scale="floor", seed=None):
    """``x`` (fp32, bf16 or fp16; leading dimensions are flattened into rows) as an MX tensor.

    ``axis=1``: blocks along the rows of x.  ``axis=0``: the transpose [cols, rows], in blocks down
    x's columns (what a product over x's rows reads).  ``axis="both"``: the pair, from one reading.
    ``seed``: None rounds to the nearest code, ties to even; a whole number rounds up with the
    probability of the distance, by the optimizer's counter stream for that seed (other seeds, other
    draws; the same seed, the same codes).  An MX tensor has no gradient: an x that requires one is refused
    where gradients are recorded.
    """
    f, rule, seed = _code(_FMT, fmt, "fmt"), _code(_RULE, scale, "scale"), _seed(seed)
    if x.dim() < 1:
        raise ValueError("adafactor8bit: mx_quantize takes a tensor of at least one dimension")
    if x.dtype not in _DTYPE:
        raise TypeError(f"adafactor8bit: mx_quantize takes fp32, bf16 or fp16, got {x.dtype}")
    _on_gpu(x, "mx_quantize")
    if forward_ad._current_level >= 0:
        no_tangents("mx_quantize", x)
    if axis not in (0, 1, "both"):
        raise ValueError(f"adafactor8bit: axis must be 0, 1 or 'both', got {axis!r}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("adafactor8bit: an MX tensor has no gradient; call mx_quantize under torch.no_grad() or on x.detach()")
    a, d = _quantize(_rows(x), fmt, f, axis != 0, axis != 1, rule, seed)
    return (a, d) if axis == "both" else a if axis == 1 else d


def mx_dequantize(t, dtype=torch.bfloat16):
    """The values of an MX tensor as a contiguous [rows, cols] matrix."""
    _mx(t, "mx_dequantize")
    if dtype not in _DTYPE:
        raise TypeError(f"adafactor8bit: mx_dequantize writes fp32, bf16 or fp16, got {dtype}")
    cp, sp, i = t._addresses()
    if i < 0:
        raise _not_on_gpu(t, "mx_dequantize")
    out = t.keep[0].new_empty((t.rows, t.cols), dtype=dtype)
    _launch("a8_mx_dequantize", i, _DTYPE[dtype], t.f, out.data_ptr(), cp, sp, t.rows, t.cols)
    return out


def _matmul(a, b, out_dtype, what):
    ac, asc, i = a._addresses()
    bc, bsc, j = b._addresses()
    if i < 0 or j < 0:
        raise _not_on_gpu(a if i < 0 else b, what)
    if i != j:
        raise ValueError(f"adafactor8bit: {what}'s operands are on one device")
    m, n = a.rows, b.rows
    c = a.keep[0].new_empty((m, n), dtype=out_dtype)
    _launch("a8_mx_matmul", i, a.f, b.f, _DTYPE[out_dtype], ac, asc, bc, bsc, c.data_ptr(), m, n, a.cols)
    return c


def mx_matmul(a, b, out_dtype=torch.bfloat16):
    """``a @ b.T`` [rows of a, rows of b] of two MX tensors of the same number of columns, in any
    pairing of the formats, accumulated in fp32 and rounded once to ``out_dtype``.  (Where a side is
    in 8 bits the matrix cores cut the 64 products they add at a time at 2^-13 of the largest one's
    binade, about 1.5e-5 of a result's size for two 8-bit sides; products of 4-bit sides are exact.)"""
    _mx(a, "mx_matmul")
    _mx(b, "mx_matmul")
    _code(_DTYPE, out_dtype, "out_dtype")
    if b.cols != a.cols:
        raise ValueError(f"adafactor8bit: mx_matmul of {a.cols} and {b.cols} columns")
    return _matmul(a, b, out_dtype, "mx_matmul")


def first_order(name, gradients):
    """A Function's backward from its static ``gradients``, launches that autograd does not see: a second
    derivative would lack their part without a word, so create_graph is an error."""
    plain = gradients.__func__

    def backward(ctx, *dy):
        if torch.is_grad_enabled():
            raise RuntimeError(f"adafactor8bit: {name} cannot be differentiated twice; call without create_graph")
        if forward_ad._current_level >= 0:
            no_tangents(f"{name}'s backward pass", *dy)
        return plain(ctx, *dy)

    return staticmethod(backward)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, fmts, rule, seed):
        need_x, need_w, _, _, _ = ctx.needs_input_grad
        (act, fa), (weight, fw), _ = fmts
        xa, xd = _quantize(x, act, fa, True, need_w, rule, None)
        wa, wd = _quantize(w, weight, fw, True, need_x, rule, None)
        ctx.save_for_backward(xd.keep[0] if need_w else None, wd.keep[0] if need_x else None)
        ctx.rest = fmts, rule, seed, x.dtype, w.dtype, x.shape[1]
        return _matmul(xa, wa, x.dtype, "mx_linear")

    @staticmethod
    def gradients(ctx, dy):
        xd, wd = ctx.saved_tensors
        ((act, fa), (weight, fw), (grad, fg)), rule, seed, xt, wt, k = ctx.rest
        dy = _rows(dy)
        m, n = dy.shape
        da, dd = _quantize(dy, grad, fg, wd is not None, xd is not None, rule, seed)
        dx = _matmul(da, _over(wd, k, n, weight, fw), xt, "mx_linear") if wd is not None else None
        dw = _matmul(dd, _over(xd, k, m, act, fa), wt, "mx_linear") if xd is not None else None
        return dx, dw, None, None, None

    backward = first_order("mx_linear", gradients)


def mx_linear(x, weight, act_fmt="mxfp8", weight_fmt="mxfp4", grad_fmt="mxfp8", scale="ceil", seed=None):
    """``x @ weight.T`` in microscaled formats, with its gradients.

    ``x`` [..., k] and ``weight`` [n, k] are fp32, bf16 or fp16; the output has x's type.  Every
    product reads its operands in blocks along the summed dimension: the output from x and weight
    along k, x's gradient from dy and weight^T along n, the weight's gradient from dy^T and x^T along
    the rows.  For the backward pass only the transposed blocks are kept.  ``seed``: a whole number
    rounds dy stochastically; None rounds to nearest.  Its random bits go by an element's place, so
    pass another one in each step and in each layer: layers of one seed round alike.  ``scale`` is the
    rule of every operand; "ceil" saturates nothing, so that stochastic rounding has no bias.  The gradients
    have none themselves: ``create_graph`` is refused, and so are forward-mode derivatives. Products with an
    8-bit side have the precision that mx_matmul names, gradients of fp32 tensors among them.

    ``weight`` may be an MXTensor laid out once (serving): x is then quantised and multiplied, without
    gradients.
    """
    fmts = ((act_fmt, _code(_FMT, act_fmt, "act_fmt")), (weight_fmt, _code(_FMT, weight_fmt, "weight_fmt")),
            (grad_fmt, _code(_FMT, grad_fmt, "grad_fmt")))
    rule, seed = _code(_RULE, scale, "scale"), _seed(seed)
    if x.dim() < 1 or len(weight.shape) != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"adafactor8bit: mx_linear of x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    if x.dtype not in _DTYPE:
        raise TypeError(f"adafactor8bit: mx_linear takes fp32, bf16 or fp16, got {x.dtype}")
    _on_gpu(x, "mx_linear")
    if forward_ad._current_level >= 0:
        no_tangents("mx_linear", x, None if isinstance(weight, MXTensor) else weight)
    if weight.device != x.device:
        raise ValueError("adafactor8bit: mx_linear's operands are on one device")
    blocks = isinstance(weight, MXTensor)
    if not blocks and weight.dtype not in _DTYPE:
        raise TypeError(f"adafactor8bit: mx_linear takes fp32, bf16 or fp16 weights, got {weight.dtype}")
    if torch.is_grad_enabled() and (x.requires_grad or (not blocks and weight.requires_grad)):
        if blocks:
            raise ValueError("adafactor8bit: mx_linear with a weight in MX blocks has no backward pass")
        y = _Linear.apply(_rows(x), _rows(weight), fmts, rule, seed)
    else:   # no gradients: along the rows alone
        xa, _ = _quantize(_rows(x), *fmts[0], True, False, rule, None)
        wa = weight if blocks else _quantize(_rows(weight), *fmts[1], True, False, rule, None)[0]
        y = _matmul(xa, wa, x.dtype, "mx_linear")
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], weight.shape[0])
