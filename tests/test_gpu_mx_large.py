"""Sizes past one grid's 2^32 - 1 work-items, which go in several launches: the rows around the first launch's
end equal the same rows by themselves."""
import numpy as np
import pytest
import torch

import adafactor8bit as a8
from oracle import mx
from oracle.sr import splitmix64

pytestmark = pytest.mark.gpu
GROUPS = (2 ** 32 - 1) // 256   # of 256 threads


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _tail(rows, cols, dtype=torch.bfloat16):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(cols)).to(dtype).cuda()


def test_norm_of_many_short_rows():
    """Norms of a row a wave: four rows a workgroup."""
    n, k = 4 * GROUPS, 16
    x = torch.zeros(n + 100, k, dtype=torch.bfloat16, device="cuda")
    x[n - 200:] = _tail(300, k)
    w = _tail(1, k)[0]
    y, h = a8.rms_norm(x, w, residual=x)
    y1, h1 = a8.rms_norm(x[n - 200:], w, residual=x[n - 200:])
    assert torch.equal(y[n - 200:], y1) and torch.equal(h[n - 200:], h1) and not y[:1000].any()
    del y, h
    q, q1 = a8.rms_norm(x, w, out_fmt="mxfp4"), a8.rms_norm(x[n - 200:], w, out_fmt="mxfp4")
    assert torch.equal(q.codes[n - 200:], q1.codes) and torch.equal(q.scales[n - 200:], q1.scales)
    del q
    xr = x.requires_grad_()
    dy = torch.zeros_like(x)
    dy[n - 200:] = _tail(300, k).flip(0)
    gx, = torch.autograd.grad(a8.rms_norm(xr, w), xr, dy)
    t = x[n - 200:].detach().clone().requires_grad_()
    g1, = torch.autograd.grad(a8.rms_norm(t, w), t, dy[n - 200:])
    assert torch.equal(gx[n - 200:], g1)


def test_quantise_many_narrow_rows(monkeypatch):
    """A row of one column is padded to 32 lanes."""
    n = GROUPS * 256 // 32
    x = torch.zeros(n + 100, 1, dtype=torch.float16, device="cuda")
    x[n - 200:] = _tail(300, 1, torch.float16)
    q, q1 = a8.mx_quantize(x, "mxfp4"), a8.mx_quantize(x[n - 200:], "mxfp4")
    assert torch.equal(q.codes[n - 200:], q1.codes) and torch.equal(q.scales[n - 200:], q1.scales)
    del q
    q = a8.mx_quantize(x, "mxfp4", seed=9)   # the random bits are those of the element's place
    i = np.arange((n - 200) * 256, (n + 100) * 256, dtype=np.uint64)
    with np.errstate(over="ignore"):
        w = splitmix64(np.uint64((9 * 0x9E3779B97F4A7C15) & (2 ** 64 - 1)) + (i >> np.uint64(2)))
    u = ((w >> (np.uint64(16) * (i & np.uint64(3)))) & np.uint64(0xFFFF)).reshape(300, 256)
    monkeypatch.setattr(mx, "draws", lambda *a: u)
    code, s = mx.quantize(x[n - 200:].double().cpu().numpy(), "mxfp4", "floor", 9)
    got = mx.values(q.codes[n - 200:].cpu().numpy(), q.scales[n - 200:].cpu().numpy(), "mxfp4", 1)
    assert np.array_equal(got, mx.values(mx.bytes_of(code, "mxfp4"), s, "mxfp4", 1))


def test_read_back_many_rows():
    n = GROUPS * 256 // 32
    codes = torch.zeros(n + 100, 128, dtype=torch.uint8, device="cuda")
    scales = torch.full((n + 100, 8), 127, dtype=torch.uint8, device="cuda")
    codes[n - 200:] = torch.randint(0, 256, (300, 128), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).cuda()
    v = a8.mx_dequantize(a8.MXTensor(codes, scales, 256, "mxfp4"))
    assert torch.equal(v[n - 200:], a8.mx_dequantize(a8.MXTensor(codes[n - 200:], scales[n - 200:], 256, "mxfp4")))
    assert not v[:1000].any() and v[n:].any()


def test_empty_contraction_of_many_outputs():
    m, n = 65540, 65540
    a = a8.mx_quantize(torch.zeros(m, 0, device="cuda"))
    torch.ones(m, n, dtype=torch.bfloat16, device="cuda")   # c gets memory that held ones, as a rule
    c = a8.mx_matmul(a, a)
    assert all(not c[i:i + 8192].any() for i in range(0, m, 8192))
