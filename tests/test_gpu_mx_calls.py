"""Calls of the microscaled operators and the norm under autograd's and the tracers' modes: what has no
derivative or no graph is refused, and what a mode does not ask for is not computed."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

import adafactor8bit as a8
from adafactor8bit import mx as mxmod
from adafactor8bit import norm as normmod

pytestmark = pytest.mark.gpu


def _r(m, k, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * scale).to(dtype).cuda()


def _calls(monkeypatch):
    """The library's calls from here on, as (name, arguments)."""
    seen, real = [], mxmod._launch

    def launch(name, device, *args):
        seen.append((name, args))
        return real(name, device, *args)

    monkeypatch.setattr(mxmod, "_launch", launch)
    monkeypatch.setattr(normmod, "_launch", launch)
    return seen


def test_forward_mode_is_refused():
    """A tangent would be dropped: the result would read as one that does not depend on its input."""
    x, w, g = _r(8, 64, 1), _r(16, 64, 2), _r(1, 64, 3)[0]
    q = a8.mx_quantize(w, "mxfp4")
    with fwd.dual_level():
        d, dw, dg = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, g))
        for f in (lambda: a8.rms_norm(d, g), lambda: a8.rms_norm(x, dg), lambda: a8.rms_norm(x, g, residual=d),
                  lambda: a8.rms_norm(d, g, out_fmt="mxfp8"), lambda: a8.mx_quantize(d), lambda: a8.mx_linear(d, q),
                  lambda: a8.mx_linear(d, w), lambda: a8.mx_linear(x, dw),
                  lambda: a8.mx_linear(d.clone().requires_grad_(), w)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                f()
        assert torch.isfinite(a8.rms_norm(x, g)).all()          # without a tangent the level changes nothing
        r = x.clone().requires_grad_()
        for f in (lambda: a8.rms_norm(r, g), lambda: a8.mx_linear(r, w), lambda: a8.rms_norm(r, g, residual=r)[1]):
            y = f()
            assert torch.isfinite(torch.autograd.grad(y, r, torch.ones_like(y), retain_graph=True)[0]).all()
            with pytest.raises(RuntimeError, match="forward-mode"):   # nor does a gradient have a tangent
                torch.autograd.grad(y, r, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
    assert a8.mx_linear(x, q).shape == (8, 16)


def test_tracing_is_refused():
    """A trace would hold the outputs' allocation and not the launch that writes them."""
    x, w, g = _r(8, 64, 1), _r(16, 64, 2), _r(1, 64, 3)[0]
    q = a8.mx_quantize(w, "mxfp4")
    for f in (lambda t: a8.rms_norm(t, g), lambda t: a8.rms_norm(t, g, residual=t)[0], lambda t: a8.mx_linear(t, w),
              lambda t: a8.mx_linear(t, q), lambda t: a8.mx_dequantize(a8.mx_quantize(t))):
        want = f(x)
        for trace in (lambda: torch.jit.trace(f, (x,), check_trace=False), lambda: make_fx(f)(x),
                      lambda: make_fx(f, pre_dispatch=True)(x)):
            with pytest.raises(RuntimeError, match="trace"):
                trace()
        assert torch.equal(f(x), want)


def test_quantize_keeps_no_gradient_and_says_so():
    x = _r(8, 64, 1).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        a8.mx_quantize(x)
    want = a8.mx_quantize(x.detach(), axis="both")
    with torch.no_grad():
        got = a8.mx_quantize(x, axis="both")
    for a, b in zip(got, want):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_linear_without_gradients_quantises_along_the_rows_alone(mode, monkeypatch):
    x, w = _r(24, 96, 1, torch.bfloat16).requires_grad_(), _r(40, 96, 2, torch.bfloat16).requires_grad_()
    want = a8.mx_linear(x, w)
    assert want.requires_grad
    seen = _calls(monkeypatch)
    with mode():
        y = a8.mx_linear(x, w)
    assert torch.equal(y, want) and not y.requires_grad
    assert [n for n, _ in seen] == ["a8_mx_quantize", "a8_mx_quantize", "a8_mx_matmul"]
    assert all(a[10] is None and a[11] is None for _, a in seen[:2])   # codes and scales of the transpose


@pytest.mark.parametrize("dtype,k", [(torch.bfloat16, 300), (torch.float32, 3000), (torch.float16, 17000)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_with_a_frozen_gain_sums_no_gradient_of_it(dtype, k, residual, monkeypatch):
    x, r, w = _r(9, k, 1, dtype).requires_grad_(), _r(9, k, 2, dtype), _r(1, k, 3, dtype)[0]
    dy = _r(9, k, 4, dtype)
    first = lambda o: o[0] if residual else o  # noqa: E731
    f = lambda w: first(a8.rms_norm(x, w, residual=r if residual else None))  # noqa: E731
    want = torch.autograd.grad(f(w.clone().requires_grad_()), x, dy)[0]
    seen = _calls(monkeypatch)
    got = torch.autograd.grad(f(w), x, dy)[0]
    assert torch.equal(got, want)
    name, args = seen[-1]
    assert name == "a8_rms_norm_backward" and args[11] is None and args[12] is None   # dw and its workspace


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
def test_the_residual_alone_passes_its_gradient_through(types):
    """Where only h is used its gradient is dh itself, also in a row with infinities or NaN."""
    tx, tr = types
    x, r = _r(5, 40, 1, tx), _r(5, 40, 2, tr)
    x[0, 3], x[1, 4], r[2, 5] = float("inf"), float("nan"), -float("inf")
    x, r, w = x.requires_grad_(), r.requires_grad_(), torch.ones(40, device="cuda", dtype=tx, requires_grad=True)
    dh = _r(5, 40, 3, tr)
    _, h = a8.rms_norm(x, w, residual=r)
    gx, gr, gw = torch.autograd.grad(h, (x, r, w), dh, allow_unused=True)
    assert gx.dtype == tx and torch.equal(gx, dh.to(tx)) and torch.equal(gr, dh)
    assert gw is None or not gw.any()


@pytest.mark.parametrize("rows", [(8,), (8, 12, 5)])
def test_compiled_programs_call_the_operators(rows):
    """torch.compile runs the operators between its graphs, also where it makes sizes symbolic."""
    w, g = _r(16, 64, 2), _r(1, 64, 3)[0]
    q = a8.mx_quantize(w, "mxfp4")
    for f in (lambda t: a8.rms_norm(t * 2, g) + 1, lambda t: a8.mx_linear(t * 2, w) + 1, lambda t: a8.mx_linear(t * 2, q) + 1,
              lambda t: a8.mx_linear(t * 2, w, "mxfp4", "mxfp8", "mxfp4", seed=3) + 1,
              lambda t: a8.mx_dequantize(a8.mx_quantize(t * 2)) + 1):
        torch._dynamo.reset()
        c = torch.compile(f, backend="eager")
        for m in rows:
            x = _r(m, 64, m)
            with torch.no_grad():
                assert torch.equal(c(x), f(x))
    for f in (lambda t: a8.rms_norm(t * 2, g) + 1, lambda t: a8.mx_linear(t * 2, w) + 1):
        torch._dynamo.reset()
        c = torch.compile(f, backend="eager")
        for m in rows:
            x = _r(m, 64, m).requires_grad_()
            y, z = c(x), f(x)
            assert torch.equal(y, z)
            assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], torch.autograd.grad(z, x, torch.ones_like(z))[0])


def test_lazily_negated_views():
    """The imaginary part of a conjugate is a view with the sign still to be applied."""
    re, im = _r(6, 1, 1), _r(6, 1, 2)
    v = torch.complex(re, im).conj().imag
    assert v.is_neg() and torch.equal(v, -im)
    assert torch.equal(a8.mx_dequantize(a8.mx_quantize(v), torch.float32), a8.mx_dequantize(a8.mx_quantize(-im), torch.float32))
    one = torch.ones(1, device="cuda")
    assert torch.equal(a8.rms_norm(v, one), a8.rms_norm(-im, one))
    assert torch.equal(a8.mx_linear(v, one[None]), a8.mx_linear(-im, one[None]))
    x, g, w, dy = _r(5, 40, 3), _r(1, 40, 4)[0], _r(7, 40, 5), _r(5, 40, 6)
    neg = torch._neg_view
    assert torch.equal(a8.rms_norm(neg(x), neg(g), residual=neg(dy))[0], a8.rms_norm(-x, -g, residual=-dy)[0])
    assert torch.equal(a8.mx_linear(neg(x), neg(w)), a8.mx_linear(-x, -w))
    xr, gr, wr = (t.clone().requires_grad_() for t in (x, g, w))
    y, h = a8.rms_norm(xr, gr, residual=xr)
    for grads in ((neg(dy), neg(x)), (-dy, -x)):
        got = torch.autograd.grad((y, h), (xr, gr), grads, retain_graph=True)
        if grads[0].is_neg():
            want = got
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, dz = a8.mx_linear(xr, wr), _r(5, 7, 7)
    a, b = (torch.autograd.grad(y, (xr, wr), d, retain_graph=True) for d in (neg(dz), -dz))
    assert all(torch.equal(s, t) for s, t in zip(a, b))
