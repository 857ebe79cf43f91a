"""Microscaled 4-bit floats on the device: quantisation and its reverse bit for bit against the definition, products against
64-bit sums of the exactly decoded operands."""
import numpy as np
import pytest
import torch

import _mx_reference as ref
import numkong_b200 as nk

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def wide_values(rows, depth, seed, low=-30, high=30):
    """Values whose blocks differ in scale and hit codes, midpoints and the saturated range."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, depth)) * np.exp2(rng.integers(low, high + 1, (rows, depth // 32 + 1)).repeat(32, axis=1)[:, :depth])
    halves = rng.integers(-16, 17, (rows, depth)) * 0.25  # every code and every tie when the block's scale is 1
    return np.where(rng.random((rows, 1)) < 0.3, halves, x).astype(np.float32)


def stored(x, name):
    t = torch.from_numpy(x).to(TORCH[name])
    return t, t.double().numpy()


def random_mx(rows, depth, seed, spread=8):
    """Codes of every kind with scales over 2^(2 spread)."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (rows, (depth + 1) // 2), dtype=np.uint8)
    if depth % 2:
        codes[:, -1] &= 15
    scales = rng.integers(127 - spread, 128 + spread, (rows, (depth + 31) // 32)).astype(np.uint8)
    return codes, scales


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,depth", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 255), (4, 256), (7, 257), (33, 777), (130, 1024)])
def test_quantise_is_the_definition(rows, depth, name):
    x, exact = stored(wide_values(rows, depth, rows + depth, *((-10, 8) if name == "f16" else (-30, 30))), name)
    codes, scales = ref.quantise(exact)
    q = nk.mx_quantise(x.cuda())
    assert nk.synchronize() == 0
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    want = ref.dequantise(codes, scales, depth)
    for to in ("f32", "bf16") + (("f16",) if name == "f16" else ()):
        got = nk.mx_dequantise(q, to)
        assert nk.synchronize() == 0
        assert got.dtype == TORCH[to] and np.array_equal(got.double().cpu().numpy(), want)
    if name == "f32":  # host arrays take the same path
        host = nk.mx_quantise(x.numpy())
        assert np.array_equal(host.codes, codes) and np.array_equal(host.scales, scales)
        assert np.array_equal(nk.mx_dequantise(host), want.astype(np.float32))


def test_quantise_extremes():
    big, tiny = np.float32(3.4028235e38), np.float32(1e-45)
    x = np.zeros((8, 64), np.float32)
    x[0, 0], x[0, 40] = big, -big
    x[1, 5], x[1, 33] = tiny, 2.0 ** -126
    x[2, 3] = np.inf
    x[3, 60] = np.nan
    x[4, 1], x[4, 2] = -np.inf, np.nan
    x[5, :32] = 2.0 ** -127
    x[6, :] = -0.0
    x[7, :4] = [4.0, 5.0, 7.0, -7.99]
    codes, scales = ref.quantise(x)
    q = nk.mx_quantise(torch.from_numpy(x).cuda())
    assert nk.synchronize() == 0
    assert np.array_equal(q.scales.cpu().numpy(), scales) and np.array_equal(q.codes.cpu().numpy(), codes)
    assert scales[2].tolist() == [255, 0] and scales[3, 1] == 255 and scales[5].tolist() == [0, 0]
    values = nk.mx_dequantise(q).cpu().numpy()
    assert np.isnan(values[2, :32]).all() and (values[2, 32:] == 0).all()
    assert np.array_equal(values[7, :4], [4, 4, 6, -6])  # 5 lies between 4 and 6 and goes to the even code; beyond 6 saturates


@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (8, 0), (5, 3)])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_quantise_strides_and_alignments(pad, offset, name):
    rows, depth = 37, 300
    wide = np.zeros((rows, depth + pad + offset), np.float32)
    wide[:, offset:offset + depth] = wide_values(rows, depth, 9)
    t, exact = stored(wide, name)
    q = nk.mx_quantise(t.cuda()[:, offset:offset + depth])
    assert nk.synchronize() == 0
    codes, scales = ref.quantise(exact[:, offset:offset + depth])
    assert np.array_equal(q.codes.cpu().numpy(), codes) and np.array_equal(q.scales.cpu().numpy(), scales)
    # and back out of padded codes: a view whose rows start off a four-byte boundary
    held = torch.zeros(rows, codes.shape[1] + 3, dtype=torch.uint8, device="cuda")
    held[:, 1:1 + codes.shape[1]] = q.codes
    marks = torch.zeros(rows, scales.shape[1] + 2, dtype=torch.uint8, device="cuda")
    marks[:, 2:] = q.scales
    again = nk.mx_dequantise(nk.MxMatrix(held[:, 1:1 + codes.shape[1]], marks[:, 2:], depth), name)
    assert nk.synchronize() == 0
    assert np.array_equal(again.double().cpu().numpy(), ref.dequantise(codes, scales, depth))


def test_every_byte_pair_decodes():
    """All 256 bytes of codes under all 256 scales."""
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None].repeat(16, axis=1)
    got = nk.mx_dequantise(nk.MxMatrix(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), 512)).cpu().numpy()
    want = ref.dequantise(codes, scales, 512)
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want.astype(np.float32), equal_nan=True)


SHAPES = [(1, 1, 1), (1, 8, 32), (3, 5, 31), (7, 130, 64), (128, 128, 256), (129, 257, 255), (33, 300, 257), (200, 129, 1000), (130, 513, 2500),
          (300, 640, 4096), (1, 4096, 512), (64, 1000, 300)]


def check_product(a, b, depth, got, cells):
    fa, fb = ref.dequantise(*a, depth), ref.dequantise(*b, depth)
    exact = fa @ fb.T
    assert got.shape == exact.shape
    off = np.abs(got.double().cpu().numpy() - exact)
    assert (off <= ref.product_bound(fa, fb, cells)).all(), float((off - ref.product_bound(fa, fb, cells)).max())


@pytest.mark.parametrize("cells", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, cells):
    a, b = random_mx(m, k, m + k), random_mx(n, k, n + k + 1)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    got = nk.dots_packed(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in a), k), packed, out_dtype=cells)
    assert nk.synchronize() == 0
    assert got.dtype == TORCH[cells]
    check_product(a, b, k, got, cells)


@pytest.mark.parametrize("cells", ["f32", "bf16"])
@pytest.mark.parametrize("rows_aligned", [True, False])
@pytest.mark.parametrize("m,n,k", [(2304, 2304, 256), (2400, 2100, 520), (100, 19000, 321), (1, 19001, 300), (19001, 3, 1030), (5000, 1025, 2049)])
def test_large_product(m, n, k, rows_aligned, cells):
    """Sizes that fill the GPU with 256 x 256 tiles, with whole and with ragged edges, A's rows on and off 16-byte boundaries."""
    a, b = random_mx(m, k, m + k), random_mx(n, k, n + k + 1)
    bytes_a = a[0].shape[1]
    held = np.zeros((m, -(-bytes_a // 16) * 16 + (0 if rows_aligned else 1)), np.uint8)
    held[:, :bytes_a] = a[0]
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    x = nk.MxMatrix(torch.from_numpy(held).cuda()[:, :bytes_a], torch.from_numpy(a[1]).cuda(), k)
    got = nk.dots_packed(x, packed, out_dtype=cells)
    assert nk.synchronize() == 0
    check_product(a, b, k, got, cells)
    if rows_aligned and cells == "f32":  # the same bits as a float matrix of these values quantised on the way, and as few rows alone
        assert torch.equal(nk.dots_packed(nk.mx_dequantise(x), packed), nk.dots_packed(nk.mx_quantise(nk.mx_dequantise(x)), packed))
        few = nk.MxMatrix(x.codes[m // 2:m // 2 + 3], x.scales[m // 2:m // 2 + 3], k)
        assert torch.equal(nk.dots_packed(few, packed), got[m // 2:m // 2 + 3])


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 512), (5, 128, 100), (9, 70, 255), (16, 20000, 777), (17, 300, 777), (70, 200, 321), (257, 384, 1024)])
def test_product_of_floats_quantises_first(m, n, k, name):
    x, _ = stored(wide_values(m, k, m, -6, 6), name)
    b = random_mx(n, k, n)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    x = x.cuda()
    got, two = nk.dots_packed(x, packed), nk.dots_packed(nk.mx_quantise(x), packed)
    assert nk.synchronize() == 0
    assert torch.equal(got, two)
    q = nk.mx_quantise(x)
    check_product((q.codes.cpu().numpy(), q.scales.cpu().numpy()), b, k, got, "f32")


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
def test_few_float_rows_off_their_boundaries(name):
    """Up to 16 float rows are quantised inside the product: strides and offsets of every kind, rows of infinities and NaN."""
    n, k = 200, 515
    b = random_mx(n, k, 3)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    for rows in (1, 2, 8, 13, 16):
        wide = np.zeros((rows, k + 9), np.float32)
        wide[:, 4:4 + k] = wide_values(rows, k, rows, -6, 6)
        t = stored(wide, name)[0].cuda()
        for first in (4, 3):
            x = t[:, first:first + k]
            got, two = nk.dots_packed(x, packed), nk.dots_packed(nk.mx_quantise(x), packed)
            assert nk.synchronize() == 0
            assert torch.equal(got, two)
    x = torch.ones(3, k, device="cuda", dtype=TORCH[name])
    x[1, 40], x[2, 7] = float("inf"), float("nan")
    got = nk.dots_packed(x, packed)
    assert nk.synchronize() == 0
    assert got[0].isfinite().all() and got[1].isnan().all() and got[2].isnan().all()


def test_rows_do_not_depend_on_one_another():
    """A row's bits are the same alone, among others and behind other rows."""
    k, n = 1500, 700
    a, b = random_mx(400, k, 1), random_mx(n, k, 2)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    c, s = (torch.from_numpy(v).cuda() for v in a)
    whole = nk.dots_packed(nk.MxMatrix(c, s, k), packed)
    for first, count in ((0, 1), (17, 1), (399, 1), (100, 200), (127, 2)):
        part = nk.dots_packed(nk.MxMatrix(c[first:first + count], s[first:first + count], k), packed)
        assert nk.synchronize() == 0
        assert torch.equal(part, whole[first:first + count])


def test_product_strides_and_out():
    m, n, k = 70, 133, 500
    a, b = random_mx(m, k, 4), random_mx(n, k, 5)
    held = np.zeros((m, a[0].shape[1] + 5), np.uint8)
    held[:, 3:3 + a[0].shape[1]] = a[0]
    marks = np.zeros((m, a[1].shape[1] + 1), np.uint8)
    marks[:, 1:] = a[1]
    x = nk.MxMatrix(torch.from_numpy(held).cuda()[:, 3:3 + a[0].shape[1]], torch.from_numpy(marks).cuda()[:, 1:], k)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    for cells in ("f32", "bf16"):
        wide = torch.full((m + 2, n + 3), 7.0, dtype=TORCH[cells], device="cuda")
        got = nk.dots_packed(x, packed, out=wide[1:-1, 1:1 + n], out_dtype=cells)
        assert nk.synchronize() == 0
        check_product(a, b, k, got, cells)
        assert (wide[0] == 7).all() and (wide[-1] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 1 + n:] == 7).all()


@pytest.mark.parametrize("cells", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(40, 301, 300), (3, 150, 64), (2300, 2311, 260)])
def test_product_out_at_any_offset(m, n, k, cells):
    """Result rows at every cell offset from a 16-byte boundary, what lies around them untouched."""
    a, b = random_mx(m, k, 8), random_mx(n, k, 9)
    x = nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in a), k)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    want = nk.dots_packed(x, packed, out_dtype=cells)
    check_product(a, b, k, want, cells)
    for first, pad in ((0, 1), (1, 0), (2, 3), (3, 6), (4, 2), (5, 5), (6, 1), (7, 9)):
        wide = torch.full((m + 2, first + n + pad), 7.0, dtype=TORCH[cells], device="cuda")
        got = nk.dots_packed(x, packed, out=wide[1:-1, first:first + n], out_dtype=cells)
        assert nk.synchronize() == 0
        assert torch.equal(got, want)
        assert (wide[0] == 7).all() and (wide[-1] == 7).all() and (wide[:, :first] == 7).all() and (wide[:, first + n:] == 7).all()


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("depth", [1, 2, 7, 255, 513, 1291])
def test_codes_at_any_offset(depth, offset):
    """Codes and scales whose rows begin at every byte of a word, packed and multiplied."""
    rows = 50
    a, b = random_mx(rows, depth, depth), random_mx(9, depth, depth + 1)
    def held(part):
        wide = np.full((rows, part.shape[1] + 5), 255, np.uint8)
        wide[:, offset:offset + part.shape[1]] = part
        return torch.from_numpy(wide).cuda()[:, offset:offset + part.shape[1]]
    x = nk.MxMatrix(held(a[0]), held(a[1]), depth)
    few = nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), depth)
    one, other = nk.dots_packed(x, nk.dots_pack(few)), nk.dots_packed(few, nk.dots_pack(x))
    assert nk.synchronize() == 0
    check_product(a, b, depth, one, "f32")
    assert torch.equal(one, other.T)


def test_product_on_the_host():
    m, n, k = 40, 150, 333
    a, b = random_mx(m, k, 6), random_mx(n, k, 7)
    packed = nk.dots_pack(nk.MxMatrix(*b, k))
    assert not packed.is_cuda
    got = nk.dots_packed(nk.MxMatrix(*a, k), packed)
    check_product(a, b, k, torch.from_numpy(got), "f32")
    x = np.random.default_rng(8).standard_normal((m, k)).astype(np.float32)
    got = nk.dots_packed(x, packed, out_dtype="bf16")
    assert got.dtype == np.uint16
    check_product(ref.quantise(x), b, k, torch.from_numpy(got.view(np.int16)).view(torch.bfloat16), "bf16")


def test_nan_scale_reaches_its_row_and_column_only():
    m, n, k = 20, 40, 256
    a, b = random_mx(m, k, 10), random_mx(n, k, 11)
    a[1][3, 2] = 255
    b[1][9, 0] = 255
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    got = nk.dots_packed(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in a), k), packed).cpu().numpy()
    want = np.zeros((m, n), bool)
    want[3], want[:, 9] = True, True
    assert np.array_equal(np.isnan(got), want)


def test_empty_and_zero_depth():
    packed = nk.dots_pack(nk.MxMatrix(torch.zeros(9, 0, dtype=torch.uint8, device="cuda"), torch.zeros(9, 0, dtype=torch.uint8, device="cuda"), 0))
    got = nk.dots_packed(torch.zeros(4, 0, device="cuda"), packed)
    assert got.shape == (4, 9) and (got == 0).all()
    packed = nk.dots_pack(nk.mx_quantise(torch.randn(9, 64, device="cuda")))
    assert nk.dots_packed(torch.zeros(0, 64, device="cuda"), packed).shape == (0, 9)
    assert nk.mx_quantise(torch.zeros(0, 64, device="cuda")).rows == 0


@pytest.mark.parametrize("cells", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 16, 17, 128, 129])
def test_few_rows_of_a_wide_matrix(m, cells):
    """Wide enough for CTA pairs, with rows for one of them; and one row whose result has a stride that is not used."""
    n, k = 13000, 260
    a, b = random_mx(m, k, 12), random_mx(n, k, 13)
    q = nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in a), k)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    got = nk.dots_packed(q, packed, out_dtype=cells)
    assert nk.synchronize() == 0
    check_product(a, b, k, got, cells)
    if m == 1:
        out = torch.full((n + 8,), 7.0, dtype=TORCH[cells], device="cuda")
        nk.lib.nkb_dots_packed_mxfp4(q.codes.data_ptr(), 3, q.scales.data_ptr(), 1, packed.buffer.data_ptr(), out.data_ptr(),
                                     nk.DTYPE_CODES[cells], 1, n, k, 1, None)
        assert nk.last_error() == "" and nk.synchronize() == 0
        assert torch.equal(out[:n], got[0]) and (out[n:] == 7).all()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("n,k", [(13000, 3000), (2304, 520)])
def test_every_kernel_sums_alike(n, k, name):
    """One row, few rows, rows for CTA pairs: the bits of a row are the same from each of them."""
    x = torch.randn(2304, k, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(TORCH[name])
    b = random_mx(n, k, 14)
    packed = nk.dots_pack(nk.MxMatrix(*(torch.from_numpy(v).cuda() for v in b), k))
    whole = nk.dots_packed(x, packed)
    for first, count in ((0, 1), (5, 2), (7, 3), (100, 16), (100, 17), (1000, 128), (1000, 129), (2303, 1)):
        assert torch.equal(nk.dots_packed(x[first:first + count], packed), whole[first:first + count])
        assert torch.equal(nk.dots_packed(nk.mx_quantise(x[first:first + count]), packed), whole[first:first + count])
    assert nk.synchronize() == 0
