"""Packed matrices in host memory with operands on a side stream of torch's, and the other way round: what is uploaded, packed or
prepared for a product is there before the product reads it, whatever the other streams are busy with."""
import numpy as np
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu

K, WIDTH = 256, 64


class Busy:
    """Some tens of milliseconds of work for a stream."""

    def __init__(self):
        self.a = torch.randn(8192, 8192, device="cuda")
        self.b = torch.empty_like(self.a)

    def keep(self, stream, times=2):
        with torch.cuda.stream(stream):
            for _ in range(times):
                torch.mm(self.a, self.a, out=self.b)


def matrices(count, experts=1, pinned=False):
    """(packed in host memory, packed on the GPU) of `count` different matrices."""
    rng = np.random.default_rng(count + experts)
    pairs = []
    for _ in range(count):
        q = nk.mx_quantise(rng.standard_normal((experts * WIDTH, K)).astype(np.float32))
        host = nk.dots_pack(q, groups=experts)
        if pinned:
            host = nk.PackedMatrix(torch.from_numpy(host.buffer).pin_memory(), "mxfp4", host.width, host.depth, experts)
        pairs.append((host, nk.dots_pack(nk.MxMatrix(torch.from_numpy(q.codes).cuda(), torch.from_numpy(q.scales).cuda(), K), groups=experts)))
    torch.cuda.synchronize()
    return pairs


@pytest.mark.parametrize("pinned", [False, True])
@pytest.mark.parametrize("count", [6, 20])  # the library keeps copies of eight
def test_matrices_in_host_memory_on_a_side_stream(count, pinned):
    pairs, busy, side = matrices(count, pinned=pinned), Busy(), torch.cuda.Stream()
    x = torch.randn(40, K, device="cuda").bfloat16()
    want = [nk.dots_packed(x, device) for _, device in pairs]
    torch.cuda.synchronize()
    nk.lib.nkb_release_caches()
    order = list(range(count))[::-1]
    got = {}
    for i in order + order:
        if i % 3 == 0:
            busy.keep(torch.cuda.default_stream())
        with torch.cuda.stream(side):
            got[i] = nk.dots_packed(x, pairs[i][0])
            side.synchronize()
        assert torch.equal(got[i].cpu(), want[i].cpu()), i
    assert nk.synchronize() == 0


def test_a_copy_just_made_serves_other_streams():
    pairs, busy = matrices(6), Busy()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    x = torch.randn(3, K, device="cuda")
    want = [nk.dots_packed(x, device) for _, device in pairs]
    torch.cuda.synchronize()
    nk.lib.nkb_release_caches()
    for i in range(5, -1, -1):
        busy.keep(torch.cuda.default_stream())
        busy.keep(streams[0])
        got = []
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(nk.dots_packed(x, pairs[i][0]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want[i]) for g in got), i
    assert nk.synchronize() == 0


def test_experts_in_host_memory_on_a_side_stream():
    pairs, busy, side = matrices(5, experts=4), Busy(), torch.cuda.Stream()
    x = torch.randn(30, K, device="cuda").bfloat16()
    ids = torch.randint(0, 4, (30, 2), device="cuda").to(torch.int32)
    want = [nk.experts_packed(x, ids, device) for _, device in pairs]
    torch.cuda.synchronize()
    nk.lib.nkb_release_caches()
    for i in range(4, -1, -1):
        busy.keep(torch.cuda.default_stream())
        with torch.cuda.stream(side):
            got = nk.experts_packed(x, ids, pairs[i][0])
            side.synchronize()
        assert torch.equal(got, want[i]), i
    assert nk.synchronize() == 0


@pytest.mark.parametrize("kind", ["numpy", "torch"])
def test_host_operands_against_a_matrix_packed_on_a_side_stream(kind):
    """The call works where the matrix lives, and after what prepares it there."""
    rng, busy, side = np.random.default_rng(3), Busy(), torch.cuda.Stream()
    x, ids = rng.standard_normal((30, K)).astype(np.float32), rng.integers(0, 4, (30, 2)).astype(np.int32)
    part = rng.random((30, 2)).astype(np.float32)
    as_given = (lambda a: a) if kind == "numpy" else torch.from_numpy
    for attempt in range(4):
        w = torch.from_numpy(rng.standard_normal((4 * WIDTH, K)).astype(np.float32)).cuda()
        torch.cuda.synchronize()
        busy.keep(side)
        with torch.cuda.stream(side):
            q = nk.mx_quantise(w)
            plain, grouped = nk.dots_pack(q), nk.dots_pack(q, groups=4)
            got = [nk.dots_packed(as_given(x), plain), nk.dots_packed(as_given(x[:1]), plain), nk.dots_packed(nk.mx_quantise(as_given(x)), plain),
                   nk.experts_packed(as_given(x), as_given(ids), grouped), nk.experts_packed(as_given(x), as_given(ids), grouped, weights=as_given(part))]
        torch.cuda.synchronize()
        xd, idsd, partd = (torch.from_numpy(a).cuda() for a in (x, ids, part))
        want = [nk.dots_packed(xd, plain), nk.dots_packed(xd[:1], plain), nk.dots_packed(nk.mx_quantise(xd), plain),
                nk.experts_packed(xd, idsd, grouped), nk.experts_packed(xd, idsd, grouped, weights=partd)]
        for g, v in zip(got, want, strict=True):
            assert np.array_equal(np.asarray(g), v.cpu().numpy()), attempt
    assert nk.synchronize() == 0
