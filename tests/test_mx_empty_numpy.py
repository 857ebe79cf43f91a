"""The 4-bit and routing calls on NumPy matrices without rows, whose strides are 0: results without rows, and no GPU asked for any."""
import numpy as np

import numkong_b200 as nk


def packed(width, depth, groups=1):
    return nk.PackedMatrix(np.zeros(nk.lib.nkb_dots_packed_size_mxfp4(groups, width, depth), np.uint8), "mxfp4", width, depth, groups)


def test_no_rows():
    x = np.zeros((0, 64), np.float32)
    q = nk.mx_quantise(x)
    assert q.codes.shape == (0, 32) and q.scales.shape == (0, 2)
    assert nk.mx_dequantise(q).shape == (0, 64)
    assert nk.mx_dequantise(nk.MxMatrix(np.zeros((0, 32), np.uint8), np.zeros((0, 2), np.uint8), 64), "bf16").shape == (0, 64)
    for a in (x, q):
        assert nk.dots_packed(a, packed(5, 64)).shape == (0, 5)
        assert nk.dots_packed(a, packed(5, 64), out_dtype="bf16").shape == (0, 5)


def test_no_tokens():
    logits, ids, part = np.zeros((0, 16), np.float32), np.zeros((0, 2), np.int32), np.zeros((0, 2), np.float32)
    weights, chosen = nk.route(logits, 2, bias=np.zeros(16, np.float32), groups=4, top_groups=2)
    assert weights.shape == (0, 2) and chosen.shape == (0, 2)
    assert nk.route_gradient(part, ids, logits).shape == (0, 16)
    x = np.zeros((0, 64), np.float32)
    assert nk.experts_packed(x, ids, packed(5, 64, 4)).shape == (0, 2, 5)
    assert nk.experts_packed(x, ids, packed(5, 64, 4), weights=part).shape == (0, 5)
    assert nk.experts_packed(np.zeros((0, 2, 64), np.float32), ids, packed(5, 64, 4)).shape == (0, 2, 5)
