"""Packed matrices in host memory with operands on a side stream of torch's: what is uploaded is there before the product reads it,
whatever the other streams are busy with."""
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
