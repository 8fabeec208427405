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
