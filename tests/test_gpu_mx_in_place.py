"""Products whose result takes the place of their float rows."""
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 40])
@pytest.mark.parametrize("size", [256, 4096, 12000])
def test_result_in_place_of_the_rows(size, rows, name):
    g = torch.Generator(device="cuda").manual_seed(size + rows)
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[name]
    packed = nk.dots_pack(nk.mx_quantise(torch.randn(size, size, generator=g, device="cuda") * size ** -0.5))
    x = torch.randn(rows, size, generator=g, device="cuda").to(dtype)
    want = nk.dots_packed(x, packed, out_dtype=name)
    for _ in range(10):
        held = x.clone()
        got = nk.dots_packed(held, packed, out=held, out_dtype=name)
        assert got is held and torch.equal(held, want)
    wide = torch.zeros(2 * rows, size, dtype=dtype, device="cuda")
    for first in range(rows + 1):  # and where the two only overlap
        wide[rows - first:2 * rows - first] = x
        if rows <= 2:
            assert torch.equal(nk.dots_packed(wide[rows - first:2 * rows - first], packed, out=wide[:rows], out_dtype=name), want)
    assert nk.synchronize() == 0


@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_experts_in_place(tokens):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    packed = nk.dots_pack(nk.mx_quantise(torch.randn(6 * 320, 320, generator=g, device="cuda")), groups=6)
    ids = torch.randint(-1, 6, (tokens, 2), generator=g, device="cuda").to(torch.int32)
    weights = torch.rand(tokens, 2, generator=g, device="cuda")
    x, h = torch.randn(tokens, 320, generator=g, device="cuda"), torch.randn(tokens, 2, 320, generator=g, device="cuda")
    sums, rows = nk.experts_packed(x, ids, packed, weights=weights), nk.experts_packed(h, ids, packed)
    assert torch.equal(nk.experts_packed(x, ids, packed, weights=weights, out=x), sums)
    assert torch.equal(nk.experts_packed(h, ids, packed, out=h), rows)
    assert nk.synchronize() == 0
