"""What the microscaled 4-bit and routing calls refuse, through Python and through the C ABI. No kernel is launched: every
refusal comes before the first."""
import numpy as np
import pytest

import numkong_b200 as nk
from numkong_b200 import _lib

lib = _lib.lib
F32, F16, BF16, I8 = (_lib.DTYPE_CODES[t] for t in ("f32", "f16", "bf16", "i8"))


def mx(rows, depth):
    return nk.MxMatrix(np.zeros((rows, (depth + 1) // 2), np.uint8), np.full((rows, (depth + 31) // 32), 127, np.uint8), depth)


def packed(width, depth, groups=1):
    return nk.PackedMatrix(np.zeros(lib.nkb_dots_packed_size_mxfp4(groups, width, depth), np.uint8), "mxfp4", width, depth, groups)


@pytest.mark.parametrize("codes,scales,depth", [((3, 16), (3, 1), 33), ((3, 17), (3, 1), 33), ((3, 16), (2, 1), 32), ((3, 16), (3, 2), 32), ((3, 15), (3, 1), 32)])
def test_mx_matrix_checks_its_parts(codes, scales, depth):
    with pytest.raises(ValueError):
        nk.MxMatrix(np.zeros(codes, np.uint8), np.zeros(scales, np.uint8), depth)


def test_mx_matrix_wants_bytes_and_rows():
    with pytest.raises(TypeError):
        nk.MxMatrix(np.zeros((3, 16), np.int32), np.zeros((3, 1), np.uint8), 32)
    with pytest.raises(ValueError):
        nk.MxMatrix(np.zeros((32, 3), np.uint8).T[:, ::2], np.zeros((3, 1), np.uint8), 32)
    with pytest.raises(ValueError):
        nk.MxMatrix(np.zeros(16, np.uint8), np.zeros((1, 1), np.uint8), 32)


def test_python_refusals():
    with pytest.raises(TypeError):
        nk.mx_quantise(np.zeros((3, 4), np.int8))
    with pytest.raises(TypeError):
        nk.mx_quantise(np.zeros((3, 4), np.float64))
    with pytest.raises(TypeError):
        nk.mx_dequantise(np.zeros((3, 4), np.uint8))
    with pytest.raises(TypeError):
        nk.mx_dequantise(mx(2, 32), "e4m3")
    with pytest.raises(ValueError):
        nk.dots_pack(mx(7, 32), groups=2)
    with pytest.raises(ValueError):
        nk.dots_pack(mx(7, 32), groups=0)
    with pytest.raises(ValueError):
        nk.dots_pack(np.zeros((4, 4), np.float32), groups=2)
    p = packed(5, 64)
    with pytest.raises(ValueError):
        nk.dots_packed(mx(2, 32), p)
    with pytest.raises(ValueError):
        nk.dots_packed(mx(2, 64), packed(5, 64, 2))
    with pytest.raises(TypeError):
        nk.dots_packed(np.zeros((2, 64), np.int8), p)
    with pytest.raises(TypeError):
        nk.dots_packed(mx(2, 64), p, out_dtype="f16")
    with pytest.raises(ValueError):
        nk.dots_packed(mx(2, 64), p, columns=(0, 1))
    with pytest.raises(ValueError):
        nk.dots_packed(mx(2, 64), p, out=np.zeros((2, 6), np.float32))
    with pytest.raises(TypeError):
        nk.dots_packed(mx(2, 64), p, out=np.zeros((2, 5), np.float64))
    with pytest.raises(TypeError):
        nk.angulars_packed(np.zeros((2, 64), np.float32), p)
    with pytest.raises(ValueError):
        nk.dots_packed(np.zeros((2, 64), np.float32), nk.PackedMatrix(np.zeros(1, np.uint8), "f32", 5, 64), out_dtype="bf16")


@pytest.mark.parametrize("how", [dict(top=0), dict(top=33), dict(top=17), dict(top=2, groups=3), dict(top=2, groups=0), dict(top=2, groups=4, top_groups=5),
                                 dict(top=2, groups=4, top_groups=0), dict(top=2, groups=64)], ids=str)
def test_route_refuses_in_the_library(how):
    with pytest.raises(RuntimeError):
        nk.route(np.zeros((3, 16), np.float32), **how)


def test_route_python_refusals():
    x = np.zeros((3, 16), np.float32)
    with pytest.raises(ValueError):
        nk.route(x, 2, score="relu")
    with pytest.raises(TypeError):
        nk.route(np.zeros((3, 16)), 2)
    with pytest.raises(ValueError):
        nk.route(x, 2, bias=np.zeros(15, np.float32))
    with pytest.raises(ValueError):
        nk.route(x, 2, bias=np.zeros(16))
    with pytest.raises(RuntimeError):
        nk.route(np.zeros((3, 1025), np.float32), 2)
    ids, g = np.zeros((3, 2), np.int32), np.zeros((3, 2), np.float32)
    with pytest.raises(ValueError):
        nk.route_gradient(g, ids.astype(np.int64), x)
    with pytest.raises(ValueError):
        nk.route_gradient(g[:2], ids, x)
    with pytest.raises(ValueError):
        nk.route_gradient(g, ids[:, ::2].repeat(2, 1)[:, ::-1], x)
    with pytest.raises(ValueError):
        nk.route_gradient(g, ids, x, score="relu")


def test_experts_python_refusals():
    x, ids, p = np.zeros((3, 64), np.float32), np.zeros((3, 2), np.int32), packed(5, 64, 4)
    for bad in (lambda: nk.experts_packed(x[:2], ids, p), lambda: nk.experts_packed(x, ids.astype(np.int64), p), lambda: nk.experts_packed(x[:, :32], ids, p),
                lambda: nk.experts_packed(x, ids, p, weights=np.zeros((3, 3), np.float32)), lambda: nk.experts_packed(np.zeros((3, 3, 64), np.float32), ids, p),
                lambda: nk.experts_packed(x, ids[0], p), lambda: nk.experts_packed(x, ids, p, out=np.zeros((6, 5), np.float32)),
                lambda: nk.experts_packed(x, ids, p, weights=np.zeros((3, 2), np.float32), out=np.zeros((3, 6), np.float32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nk.experts_packed(x, ids, np.zeros(3))
    with pytest.raises(TypeError):
        nk.experts_packed(x.astype(np.int8), ids, p)
    with pytest.raises(TypeError):
        nk.experts_packed(x, ids, p, out_dtype="i8")


def refused(call, *outputs):
    """The call sets the error text and fills its outputs with 0xFF."""
    call()
    assert nk.last_error()
    for out in outputs:
        assert (out.view(np.uint8) == 255).all()


def test_c_refusals_fill_their_outputs():
    x, codes, scales, c = np.zeros((4, 64), np.float32), np.zeros((4, 32), np.uint8), np.zeros((4, 2), np.uint8), np.zeros((4, 5), np.float32)
    p = lambda a: a.ctypes.data
    refused(lambda: lib.nkb_mx_quantise(p(x), I8, 4, 64, 256, p(codes), 32, p(scales), 2), codes, scales)
    codes[:], scales[:] = 0, 0
    refused(lambda: lib.nkb_mx_quantise(p(x), F32, 4, 64, 252, p(codes), 32, p(scales), 2), codes, scales)
    refused(lambda: lib.nkb_mx_quantise(None, F32, 4, 64, 256, p(codes), 32, p(scales), 2), codes, scales)
    refused(lambda: lib.nkb_mx_dequantise(p(codes), 31, p(scales), 2, 4, 64, p(x), F32, 256), x)
    blob = packed(5, 64).buffer
    refused(lambda: lib.nkb_dots_packed_mxfp4(p(codes), 32, p(scales), 2, p(blob), p(c), F32, 4, 5, 64, 20, None), c)   # a blob nobody packed
    c[:] = 0
    refused(lambda: lib.nkb_dots_packed_mxfp4(p(codes), 32, p(scales), 2, p(blob), p(c), F16, 4, 5, 64, 20, None), c[:, :0])
    refused(lambda: lib.nkb_dots_packed_mxfp4(p(codes), 32, p(scales), 2, p(blob), p(c), F32, 4, 5, 64, 22, None))
    refused(lambda: lib.nkb_dots_packed_mxfp4(None, 32, p(scales), 2, p(blob), p(c), F32, 4, 5, 64, 20, None), c)
    refused(lambda: lib.nkb_dots_packed_quantised_mxfp4(p(x), I8, 256, p(blob), p(c), F32, 4, 5, 64, 20, None), c)
    refused(lambda: lib.nkb_dots_packed_quantised_mxfp4(p(x), F32, 255, p(blob), p(c), F32, 4, 5, 64, 20, None), c)
    refused(lambda: lib.nkb_dots_pack_mxfp4(p(codes), 31, p(scales), 2, 1, 4, 64, p(blob)), blob)
    refused(lambda: lib.nkb_dots_pack_mxfp4(None, 32, p(scales), 2, 1, 4, 64, p(blob)), blob)
    logits, w, ids = np.zeros((2, 8), np.float32), np.zeros((2, 2), np.float32), np.zeros((2, 2), np.int32)
    refused(lambda: lib.nkb_route(p(logits), F32, 2, 8, 31, None, 0, 1, 1, 2, 1, 1.0, p(w), p(ids)), w, ids)
    refused(lambda: lib.nkb_route(p(logits), F32, 2, 8, 32, None, 2, 1, 1, 2, 1, 1.0, p(w), p(ids)), w, ids)
    grad = np.zeros((2, 8), np.float32)
    refused(lambda: lib.nkb_route_gradient(p(w), p(ids), p(logits), I8, 2, 8, 32, 0, 2, 1, 1.0, p(grad)), grad)
    out = np.zeros((4, 5), np.float32)
    blob = packed(5, 64, 3).buffer
    refused(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), 2, 2, p(blob), 0, 5, 64, None, p(out), F32, 20, None), out)
    refused(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), 2, 2, p(blob), 3, 5, 64, None, p(out), F32, 20, None), out)
    refused(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), 2, 2, p(blob), 2000, 5, 64, None, p(out), F32, 20, None), out)
    refused(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, None, 2, 2, p(blob), 3, 5, 64, None, p(out), F32, 20, None), out)
    refused(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), 2, 2, p(blob), 3, 5, 64, None, p(out), F32, 19, None))


def test_sizes_are_pure():
    for groups, width, depth in [(1, 1, 1), (1, 128, 256), (3, 129, 257), (64, 2048, 2048)]:
        size = lib.nkb_dots_packed_size_mxfp4(groups, width, depth)
        assert size == lib.nkb_dots_packed_size_mxfp4(groups, width, depth)
        assert size == 128 + groups * -(-width // 128) * -(-depth // 256) * 17408
    assert lib.nkb_dots_workspace_mxfp4(129, 257) == 2 * 2 * 17408
    assert lib.nkb_experts_workspace_mxfp4(4, 2, 8, 64, 256, 1) >= 8 * 17408 + 8 * 64 * 4
    assert lib.nkb_experts_workspace_mxfp4(4, 2, 8, 64, 256, 0) < lib.nkb_experts_workspace_mxfp4(4, 2, 8, 64, 256, 1)


def test_refusals_stay_inside_what_sizes_and_strides_span():
    """Rows that overlap are filled as far as the caller's stride reaches, sizes that nothing takes are not believed."""
    held = np.zeros(4096, np.uint8)
    x, codes, scales, ids = np.zeros((4, 64), np.float32), np.zeros((4, 32), np.uint8), np.zeros((4, 2), np.uint8), np.zeros((4, 1), np.int32)
    p = lambda a: a.ctypes.data
    blob, experts = packed(50, 64).buffer, packed(50, 64, 3).buffer

    def spans(call, last):
        held[:] = 0
        call()
        assert nk.last_error()
        assert (held[:last] == 255).all() and (held[last:] == 0).all()
    spans(lambda: lib.nkb_dots_packed_mxfp4(p(codes), 32, p(scales), 2, p(blob), p(held), F32, 4, 50, 64, 100, None), 3 * 100 + 200)
    spans(lambda: lib.nkb_dots_packed_mxfp4(p(codes), 32, p(scales), 2, p(blob), p(held), I8, 4, 50, 64, 50, None), 4 * 50)
    spans(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), 4, 1, p(experts), 3, 50, 64, None, p(held), F32, 100, None), 3 * 100 + 200)
    spans(lambda: lib.nkb_mx_dequantise(p(codes), 32, p(scales), 2, 4, 64, p(held), F32, 64), 3 * 64 + 256)
    spans(lambda: lib.nkb_mx_quantise(p(x), F32, 4, 64, 256, p(held), 16, p(scales), 2), 3 * 16 + 32)
    huge = 2 ** 64 - 1
    for size in (huge, 2 ** 31):
        spans(lambda: lib.nkb_dots_packed_mxfp4(p(codes), 32, p(scales), 2, p(blob), p(held), F32, size, 50, 64, 200, None), 0)
        spans(lambda: lib.nkb_dots_packed_mxfp4(None, 32, p(scales), 2, p(blob), p(held), F32, 4, size, 64, 200, None), 0)
        spans(lambda: lib.nkb_dots_pack_mxfp4(p(codes), 32, p(scales), 2, 1, size, 64, p(held)), 0)
        spans(lambda: lib.nkb_dots_pack_mxfp4(p(codes), 32, p(scales), 2, size, 4, 64, p(held)), 0)
        spans(lambda: lib.nkb_mx_quantise(p(x), F32, size, 64, 256, p(held), 32, p(scales), 2), 0)
        spans(lambda: lib.nkb_mx_dequantise(p(codes), 32, p(scales), 2, size, 64, p(held), F32, 256), 0)
        spans(lambda: lib.nkb_route(p(x), F32, size, 64, 256, None, 0, 1, 1, 2, 1, 1.0, p(held), p(ids)), 0)
        spans(lambda: lib.nkb_route(p(x), F32, 4, 64, 256, None, 0, 1, 1, size, 1, 1.0, p(held), p(ids)), 0)
        spans(lambda: lib.nkb_route_gradient(p(x), p(ids), p(x), F32, size, 64, 256, 0, 2, 1, 1.0, p(held)), 0)
        spans(lambda: lib.nkb_route_gradient(p(x), p(ids), p(x), F32, 4, size, 256, 0, 2, 1, 1.0, p(held)), 0)
        spans(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), size, 1, p(experts), 3, 50, 64, None, p(held), F32, 200, None), 0)
        spans(lambda: lib.nkb_experts_packed_mxfp4(p(x), F32, 256, 0, p(ids), 4, size, p(experts), 3, 50, 64, None, p(held), F32, 200, None), 0)


def test_no_choice_is_refused():
    with pytest.raises(ValueError):
        nk.experts_packed(np.zeros((3, 64), np.float32), np.zeros((3, 0), np.int32), packed(5, 64, 4), weights=np.zeros((3, 0), np.float32))


class DeviceArray:
    """What a library without DLPack offers for device memory."""
    shape = (3, 64)
    __cuda_array_interface__ = {"shape": (3, 64), "typestr": "<f4", "data": (256, False), "version": 3}


def test_device_arrays_without_dlpack_are_refused():
    ids = np.zeros((3, 2), np.int32)
    for call in (lambda: nk.mx_quantise(DeviceArray()), lambda: nk.route(DeviceArray(), 2), lambda: nk.experts_packed(DeviceArray(), ids, packed(5, 64, 4)),
                 lambda: nk.dots_packed(DeviceArray(), packed(5, 64)), lambda: nk.route_gradient(DeviceArray(), ids, np.zeros((3, 8), np.float32))):
        with pytest.raises(TypeError):
            call()
