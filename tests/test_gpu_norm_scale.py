"""The scale rule of the norm's MX output: in fp32, where y is not rounded before its blocks are formed, the output
is mx_quantize's of y, bit for bit, under either rule."""
import pytest
import torch

import adafactor8bit as a8
from adafactor8bit import _native as nat

pytestmark = pytest.mark.gpu


def _r(m, k, seed):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("m,k", [(1, 1), (5, 300), (33, 1000), (4, 2048), (3, 5003), (2, 16385), (2, 40000)])
def test_norm_into_blocks_of_either_rule(fmt, m, k):
    x, r, w = _r(m, k, 1), _r(m, k, 2), _r(1, k, 3)[0]
    for res in (None, r):
        y = a8.rms_norm(x, w, residual=res)
        y = y if res is None else y[0]
        found = []
        for scale in ("floor", "ceil"):
            q = a8.rms_norm(x, w, residual=res, out_fmt=fmt, scale=scale)
            q = q if res is None else q[0]
            want = a8.mx_quantize(y, fmt, scale=scale)
            assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
            found.append(q)
        default = a8.rms_norm(x, w, out_fmt=fmt)
        assert res is not None or torch.equal(default.codes, found[0].codes)
        if m * k > 1000:   # the rules differ
            assert not torch.equal(found[0].scales, found[1].scales)


def test_serving_reproduces_the_trained_layer():
    x, r, g, w = _r(40, 512, 1), _r(40, 512, 2), _r(1, 512, 3)[0], _r(96, 512, 4)
    y, h = a8.rms_norm(x, g, residual=r)
    want = a8.mx_linear(y, w)
    y8, h8 = a8.rms_norm(x, g, residual=r, out_fmt="mxfp8", scale="ceil")
    assert torch.equal(h, h8) and torch.equal(a8.mx_matmul(y8, a8.mx_quantize(w, "mxfp4", scale="ceil"), torch.float32), want)


def test_refusals():
    x, w = _r(4, 64, 1), _r(1, 64, 2)[0]
    with pytest.raises(ValueError, match="scale"):
        a8.rms_norm(x, w, out_fmt="mxfp8", scale="up")
    n = nat.lib().a8_rms_norm
    for fmt in (2, 0x102, 0x200, -2, 0x100 - 0x200):
        assert n(0, 0, 0, fmt, 16, 1, None, 0, 16, 16, 16, 16, None, None, None, 1, 1, 1e-6, None) == -1


def test_the_example_serves_what_it_trained():
    """One rule in training and serving: a step of examples/mx_lm.py's server has the model's logits."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    try:
        import mx_lm
    finally:
        sys.path.pop(0)
    torch.manual_seed(3)
    model = mx_lm.Model().cuda()
    pairs = torch.randint(0, mx_lm.VOCAB, (16, 2)).cuda()
    with torch.no_grad():
        want = model(pairs)[:, 0]
    assert torch.equal(mx_lm.Server(model).logits(pairs[:, 0], pairs[:, 1]), want)
