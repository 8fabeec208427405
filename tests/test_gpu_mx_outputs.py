"""A product's output types against each other: the sums are the same and are rounded once, so the fp32 output
rounded to 16 bits is the 16-bit output, bit for bit."""
import pytest
import torch

import adafactor8bit as a8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fa,fb", [("mxfp8", "mxfp4"), ("mxfp4", "mxfp8"), ("mxfp4", "mxfp4"), ("mxfp8", "mxfp8")])
@pytest.mark.parametrize("m,n,k", [(33, 65, 4096), (130, 300, 4200), (256, 2048, 5632), (40, 12300, 4100), (1000, 1000, 8192),
                                   (5, 300, 4500), (700, 1500, 600), (2100, 2300, 300)])
def test_fp32_output_rounds_to_the_16_bit_one(fa, fb, m, n, k):
    g = torch.Generator().manual_seed(m + n)
    a = a8.mx_quantize(torch.randn(m, k, generator=g).cuda(), fa)
    b = a8.mx_quantize(torch.randn(n, k, generator=g).cuda(), fb)
    want = [a8.mx_matmul(a, b, t) for t in (torch.bfloat16, torch.float16)]
    for c in [a8.mx_matmul(a, b, torch.float32) for _ in range(12)]:
        for w in want:
            assert torch.equal(c.to(w.dtype), w)
