"""What a 4-bit or routing call on host memory leaves behind when it fails after its operands were placed: 0xFF in its outputs,
row by row at the caller's stride, and nothing in the bytes between and behind them."""
import numpy as np
import pytest
import torch

import numkong_b200 as nk
from numkong_b200 import _lib

pytestmark = pytest.mark.gpu

lib = _lib.lib
F32, BF16 = _lib.DTYPE_CODES["f32"], _lib.DTYPE_CODES["bf16"]
ROWS, DEPTH, WIDTH, EXPERTS = 4, 70, 5, 3


def p(a):
    return a.ctypes.data


class Held:
    """Room for rows of `row_bytes` bytes, `row_bytes + pad` apart, and as much again behind them."""

    def __init__(self, rows, row_bytes, pad):
        self.rows, self.row_bytes, self.stride = rows, row_bytes, row_bytes + pad
        self.bytes = np.zeros(4096, np.uint8)
        self.at = p(self.bytes)

    def spoilt(self):
        want = np.zeros_like(self.bytes)
        for r in range(self.rows):
            want[r * self.stride:r * self.stride + self.row_bytes] = 255
        return np.array_equal(self.bytes, want)


def operands():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((ROWS, DEPTH)).astype(np.float32)
    w = nk.mx_quantise(rng.standard_normal((EXPERTS * WIDTH, DEPTH)).astype(np.float32))
    return x, nk.mx_quantise(x), nk.dots_pack(nk.MxMatrix(w.codes[:WIDTH], w.scales[:WIDTH], DEPTH)), nk.dots_pack(w, groups=EXPERTS)


def calls(pad, workspace):
    """(name, call, its outputs) of every entry point; `pad` bytes between the rows of an output."""
    x, q, plain, grouped = operands()
    ids, weights = np.zeros((ROWS, 2), np.int32), np.ones((ROWS, 2), np.float32)
    logits = x[:, :16].copy()
    codes, scales = Held(ROWS, 35, pad), Held(ROWS, 3, pad)
    yield "quantise", lambda: lib.nkb_mx_quantise(p(x), F32, ROWS, DEPTH, 280, codes.at, codes.stride, scales.at, scales.stride), [codes, scales]
    for cell, code in ((4, F32), (2, BF16)):
        out = Held(ROWS, DEPTH * cell, pad)
        yield "dequantise", lambda: lib.nkb_mx_dequantise(p(q.codes), 35, p(q.scales), 3, ROWS, DEPTH, out.at, code, out.stride), [out]
        out = Held(ROWS, WIDTH * cell, pad)
        yield "product of codes", lambda: lib.nkb_dots_packed_mxfp4(p(q.codes), 35, p(q.scales), 3, p(plain.buffer), out.at, code, ROWS, WIDTH, DEPTH, out.stride, workspace), [out]
        out = Held(ROWS, WIDTH * cell, pad)
        yield "product of floats", lambda: lib.nkb_dots_packed_quantised_mxfp4(p(x), F32, 280, p(plain.buffer), out.at, code, ROWS, WIDTH, DEPTH, out.stride, workspace), [out]
        out = Held(2 * ROWS, WIDTH * cell, pad)
        yield "experts", lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 280, 0, p(ids), ROWS, 2, p(grouped.buffer), EXPERTS, WIDTH, DEPTH, None, out.at, code, out.stride, workspace), [out]
        out = Held(ROWS, WIDTH * cell, pad)
        yield "weighted experts", lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 280, 0, p(ids), ROWS, 2, p(grouped.buffer), EXPERTS, WIDTH, DEPTH, p(weights), out.at, code, out.stride, workspace), [out]
    if pad == 0:
        w, i, g = Held(ROWS, 8, 0), Held(ROWS, 8, 0), Held(ROWS, 64, 0)
        yield "route", lambda: lib.nkb_route(p(logits), F32, ROWS, 16, 64, None, 0, 1, 1, 2, 1, 1.0, w.at, i.at), [w, i]
        yield "route_gradient", lambda: lib.nkb_route_gradient(p(weights), p(ids), p(logits), F32, ROWS, 16, 64, 0, 2, 1, 1.0, g.at), [g]


@pytest.mark.parametrize("pad", [0, 4, 20])
def test_a_reported_wait_that_gave_up(pad):
    """The failure is made on the host: the error word holds what a wait that ran out would have left there."""
    for name, call, outputs in calls(pad, None):
        assert lib.nkb_test_set_error_word(0, 0x80040002) == 0
        call()
        assert "gave up" in nk.last_error(), name
        for held in outputs:
            assert held.spoilt(), name
    assert nk.synchronize() == 0


@pytest.mark.parametrize("pad", [0, 4, 20])
def test_a_refused_workspace(pad):
    room = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    for name, call, outputs in calls(pad, room.data_ptr() + 16):
        if "product" not in name and "experts" not in name:
            continue
        call()
        assert "workspace" in nk.last_error(), name
        for held in outputs:
            assert held.spoilt(), name
    assert nk.synchronize() == 0


def test_a_pack_to_a_misaligned_address():
    size = lib.nkb_dots_packed_size_mxfp4(1, WIDTH, DEPTH)
    room = torch.zeros(size + 64, dtype=torch.uint8, device="cuda")
    q = operands()[1]
    lib.nkb_dots_pack_mxfp4(p(q.codes), 35, p(q.scales), 3, 1, ROWS, DEPTH, room.data_ptr() + 8)
    assert "aligned" in nk.last_error()
    torch.cuda.synchronize()
    assert (room[8:8 + size] == 255).all() and (room[:8] == 0).all() and (room[8 + size:] == 0).all()
    assert nk.synchronize() == 0
