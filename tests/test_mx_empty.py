"""Products of 4-bit matrices without rows, columns or depth, whose tensors have no address."""
import numpy as np
import pytest
import torch

import numkong_b200 as nk


def mx(rows, depth, device):
    return nk.MxMatrix(torch.zeros(rows, (depth + 1) // 2, dtype=torch.uint8, device=device), torch.zeros(rows, (depth + 31) // 32, dtype=torch.uint8, device=device), depth)


def packed(width, depth):
    """Never read: a result without cells needs no product."""
    return nk.PackedMatrix(np.zeros(nk.lib.nkb_dots_packed_size_mxfp4(1, width, depth), np.uint8), "mxfp4", width, depth)


@pytest.mark.parametrize("cells", ["f32", "bf16"])
def test_no_rows(cells):
    q = mx(0, 64, "cpu")
    assert q.codes.data_ptr() == 0
    assert tuple(nk.dots_packed(q, packed(9, 64), out_dtype=cells).shape) == (0, 9)


def test_no_columns():
    assert tuple(nk.dots_packed(mx(3, 0, "cpu"), packed(0, 0)).shape) == (3, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_no_depth(where):
    w = nk.dots_pack(mx(9, 0, where))
    for rows in (1, 4):
        got = nk.dots_packed(mx(rows, 0, where), w)
        assert tuple(got.shape) == (rows, 9) and (got == 0).all()
    assert tuple(nk.dots_packed(mx(0, 64, where), nk.dots_pack(nk.mx_quantise(torch.randn(9, 64, device=where)))).shape) == (0, 9)
    assert nk.synchronize() == 0
