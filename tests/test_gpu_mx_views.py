"""Rows of experts' operands that have to be copied before they can be read, on a stream that torch does not know of."""
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weighted", [False, True])
def test_rows_that_do_not_fold_on_a_chosen_stream(weighted):
    """The copy is made on the chosen stream: not behind torch's own work, and not handed on while the kernels read it."""
    tokens, experts, top, n, k = 600, 5, 3, 40, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    packed = nk.dots_pack(nk.mx_quantise(torch.randn(experts * n, k, generator=g, device="cuda")), groups=experts)
    h = torch.randn(tokens, top + 1, k, generator=g, device="cuda")[:, :top]
    ids = torch.randint(0, experts, (tokens, top), generator=g, device="cuda").to(torch.int32)
    weights = torch.rand(tokens, top, generator=g, device="cuda") if weighted else None
    want = nk.experts_packed(h.contiguous(), ids, packed, weights=weights)
    out, busy = [torch.empty_like(want) for _ in range(4)], torch.randn(8192, 8192, device="cuda")
    held, side = torch.empty_like(busy), torch.cuda.Stream()
    torch.cuda.synchronize()
    nk.set_stream(side.cuda_stream)
    try:
        for o in out:
            for _ in range(2):
                torch.mm(busy, busy, out=held)
            nk.experts_packed(h, ids, packed, weights=weights, out=o)
            junk = [torch.full((tokens, top, k), 100.0, device="cuda") for _ in range(3)]
            side.synchronize()
            torch.cuda.synchronize()
            del junk
            assert torch.equal(o, want)
        assert nk.synchronize() == 0
    finally:
        nk.set_stream(0)
