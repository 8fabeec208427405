"""MXTensor objects: their copies, and the addresses that the library is given."""
import copy
import pickle

import pytest
import torch

import adafactor8bit as a8
from adafactor8bit import mx


def _parts(rows=4, cols=64, fmt="mxfp4"):
    g = torch.Generator().manual_seed(rows)
    p = -(-cols // 256) * 256
    return (torch.randint(0, 256, (rows, p if fmt == "mxfp8" else p // 2), generator=g).to(torch.uint8),
            torch.randint(0, 255, (rows, p // 32), generator=g).to(torch.uint8))


def _addresses(t):
    return t.codes.data_ptr(), t.scales.data_ptr(), -1


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("made", ["from parts", "by the operators"])
def test_copies_have_their_own_addresses(fmt, made):
    if made == "from parts":
        t = a8.MXTensor(*_parts(fmt=fmt), 64, fmt)
    else:
        t = mx._new(4, 64, fmt, mx._FMT[fmt], torch.device("cpu"))
        t.codes.copy_(_parts(fmt=fmt)[0])
        t.scales.copy_(_parts(fmt=fmt)[1])
    want = t.codes.clone(), t.scales.clone()
    assert t._addresses() == _addresses(t)
    for c in (copy.deepcopy(t), pickle.loads(pickle.dumps(t))):
        assert (c.shape, c.fmt, c.device) == (t.shape, t.fmt, t.device)
        assert c._addresses() == _addresses(c) and c._addresses()[0] != t._addresses()[0]
        assert torch.equal(c.codes, want[0]) and torch.equal(c.scales, want[1])
        c.codes.zero_()
        assert torch.equal(t.codes, want[0])
    c = copy.copy(t)
    assert c._addresses() == t._addresses() and c.codes.data_ptr() == t.codes.data_ptr()


def test_addresses_follow_the_parts():
    """Parts whose memory is replaced (a module that moves its parameters) are read where they are now."""
    codes, scales = _parts()
    t = a8.MXTensor(codes, scales, 64, "mxfp4")
    codes.data = codes.clone()
    assert t._addresses() == (codes.data_ptr(), scales.data_ptr(), -1) == _addresses(t)
