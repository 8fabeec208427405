"""Arguments of the microscaled operators that are refused before anything is computed."""
import numpy as np
import pytest
import torch

import adafactor8bit as a8
from adafactor8bit import mx


@pytest.mark.parametrize("seed", [1.5, "1", (1,), torch.tensor(0.5)])
def test_seed_is_a_whole_number(seed):
    """mx_linear uses the seed in the backward pass: it is looked at before the forward one."""
    x, w = torch.zeros(4, 64), torch.zeros(8, 64, requires_grad=True)
    with pytest.raises(TypeError, match="seed"):
        a8.mx_quantize(x, seed=seed)
    with pytest.raises(TypeError, match="seed"):
        a8.mx_linear(x, w, seed=seed)


def test_seed_of_any_integer_type():
    assert mx._seed(None) is None
    for seed in (5, np.int64(5), np.uint64(5), torch.tensor(5)):
        assert mx._seed(seed) == 5 and type(mx._seed(seed)) is int
    assert mx._seed(-1) == mx._MASK64 and mx._seed(1 << 70 | 3) == 3


def test_operands_are_mx_tensors():
    t = a8.MXTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.uint8), 64, "mxfp4")
    for bad in (torch.zeros(4, 64), None, (t.codes, t.scales)):
        with pytest.raises(TypeError, match="MXTensor"):
            a8.mx_dequantize(bad)
        with pytest.raises(TypeError, match="MXTensor"):
            a8.mx_matmul(bad, t)
        with pytest.raises(TypeError, match="MXTensor"):
            a8.mx_matmul(t, bad)


def test_weights_of_other_shapes():
    for weight in (torch.zeros(()), torch.zeros(64), torch.zeros(2, 3, 64)):
        with pytest.raises(ValueError, match="mx_linear"):
            a8.mx_linear(torch.zeros(4, 64), weight)
    with pytest.raises(ValueError, match="mx_linear"):
        a8.mx_linear(torch.zeros(()), torch.zeros(4, 64))


def test_parts_of_other_shapes():
    u8 = dict(dtype=torch.uint8)
    for codes, scales in (((), (4, 8)), ((4, 128), ()), ((512,), (4, 8)), ((4, 128, 1), (4, 8))):
        with pytest.raises(ValueError, match="codes"):
            a8.MXTensor(torch.zeros(codes, **u8), torch.zeros(scales, **u8), 64, "mxfp4")
    for cols in (-1, -300):
        with pytest.raises(ValueError):
            a8.MXTensor(torch.zeros(4, 0, **u8), torch.zeros(4, 0, **u8), cols, "mxfp4")
