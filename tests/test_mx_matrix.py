"""What an MxMatrix keeps: the arrays it was made of, at the addresses its calls read."""
import copy
import pickle

import numpy as np
import pytest
import torch

import numkong_b200 as nk


def parts():
    return np.zeros((3, 16), np.uint8), np.full((3, 1), 127, np.uint8)


def test_parts_are_the_callers():
    codes, scales = parts()
    q = nk.MxMatrix(codes, scales, 32)
    assert q.codes is codes and q.scales is scales and (q.rows, q.depth) == (3, 32)
    codes[1, 2] = 7
    assert q.codes[1, 2] == 7


@pytest.mark.parametrize("name", ["codes", "scales", "rows", "depth"])
def test_parts_are_not_exchanged(name):
    """Calls would go on reading the old arrays."""
    q = nk.MxMatrix(*parts(), 32)
    with pytest.raises(AttributeError):
        setattr(q, name, torch.zeros(3, 16, dtype=torch.uint8))


@pytest.mark.parametrize("again", [copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q))], ids=["deepcopy", "pickle"])
@pytest.mark.parametrize("kind", ["numpy", "torch"])
def test_copies_read_their_own_parts(kind, again):
    """A copy's addresses are those of its own arrays: the original may go."""
    codes, scales = parts() if kind == "numpy" else map(torch.from_numpy, parts())
    q = again(nk.MxMatrix(codes, scales, 31))
    address = (lambda a: a.ctypes.data) if kind == "numpy" else (lambda a: a.data_ptr())
    assert q.codes is not codes and q._parts == (address(q.codes), 16, address(q.scales), 1) and (q.rows, q.depth) == (3, 31)


@pytest.mark.gpu
def test_quantised_parts_are_not_exchanged():
    q = nk.mx_quantise(np.ones((3, 32), np.float32))
    with pytest.raises(AttributeError):
        q.codes = torch.from_numpy(q.codes).cuda()
    assert q.codes.shape == (3, 16) and q.scales.shape == (3, 1)
