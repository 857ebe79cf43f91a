"""The microscaled 4-bit and routing calls where their surroundings are not the ordinary ones: captured into graphs, on streams of the
caller's, from two threads at once, and on operands that reach past 32-bit offsets."""
import threading

import numpy as np
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu


class Layer:
    """Router product, routing, experts with and without weights, gradient: everything with operands of its own."""

    def __init__(self, seed, tokens=50, experts=12, top=3, k=320, hidden=200):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
        self.router = nk.dots_pack(nk.mx_quantise(torch.randn(experts, k, generator=g, device="cuda") * k ** -0.5))
        self.first = nk.dots_pack(nk.mx_quantise(torch.randn(experts * hidden, k, generator=g, device="cuda") * k ** -0.5), groups=experts)
        self.second = nk.dots_pack(nk.mx_quantise(torch.randn(experts * k, hidden, generator=g, device="cuda") * hidden ** -0.5), groups=experts)
        self.grad = torch.randn(tokens, top, generator=g, device="cuda")
        self.top = top
        torch.cuda.synchronize()

    def __call__(self):
        logits = nk.dots_packed(self.x, self.router)
        weights, ids = nk.route(logits, self.top, score="sigmoid")
        h = nk.experts_packed(self.x, ids, self.first, out_dtype="bf16")
        out = nk.experts_packed(torch.nn.functional.silu(h), ids, self.second, weights=weights)
        q = nk.mx_quantise(out)
        return [logits, weights, ids, h, out, q.codes, q.scales, nk.mx_dequantise(q), nk.route_gradient(self.grad, ids, logits, score="sigmoid"),
                nk.dots_packed(self.x[:1], self.router, out_dtype="bf16"), nk.dots_packed(nk.mx_quantise(self.x), self.router)]


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_two_graphs_replayed_at_once():
    layers = [Layer(1), Layer(2, tokens=700, experts=5, top=2)]
    graphs, results = [], []
    for layer in layers:
        layer()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(layer())
        graphs.append(graph)
    fresh = [torch.randn_like(layer.x) for layer in layers]
    for layer, x in zip(layers, fresh):
        layer.x.copy_(x)
    wants = [layer() for layer in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        layers[0]()  # and the same calls of the thread that captured them, on a third stream
    torch.cuda.synchronize()
    for result, want in zip(results, wants):
        assert same(result, want)
    assert nk.synchronize() == 0


def test_a_captured_call_needs_a_workspace():
    layer = Layer(3)
    q = nk.mx_quantise(layer.x)
    out = torch.zeros(50, 12, device="cuda")
    torch.cuda.synchronize()
    graph, errors = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        nk.lib.nkb_borrow_stream(torch.cuda.current_stream().cuda_stream, 1)
        try:
            nk.lib.nkb_dots_packed_mxfp4(*q._parts, layer.router.buffer.data_ptr(), out.data_ptr(), 1 << 11, 50, 12, 320, 48, None)
            errors.append(nk.last_error())
            ids = torch.zeros(50, 3, dtype=torch.int32, device="cuda")
            nk.lib.nkb_experts_packed_mxfp4(layer.x.data_ptr(), 1 << 13, 640, 0, ids.data_ptr(), 50, 3, layer.first.buffer.data_ptr(), 12, 200, 320, None,
                                            torch.empty(150, 200, device="cuda").data_ptr(), 1 << 11, 800, None)
            errors.append(nk.last_error())
        finally:
            nk.lib.nkb_borrow_stream(None, 0)
    assert len(errors) == 2 and all("workspace" in e for e in errors)


@pytest.mark.parametrize("chosen", ["torch's", "the same", "another"])
def test_streams(chosen):
    """Work behind a slow producer on a side stream; `another`: a stream that set_stream chose and torch does not know of."""
    layer = Layer(4)
    want = layer()
    torch.cuda.synchronize()
    x, h, stream = layer.x.clone(), torch.nn.functional.silu(want[3]), torch.cuda.Stream()
    big = torch.randn(8192, 8192, device="cuda")
    layer.x.zero_()
    torch.cuda.synchronize()
    if chosen == "another":
        layer.x.copy_(x)
        torch.cuda.synchronize()
        nk.set_stream(stream.cuda_stream)
        try:
            got = [nk.dots_packed(layer.x, layer.router), *nk.route(want[0], layer.top, score="sigmoid")]
            got += [nk.experts_packed(layer.x, want[2], layer.first, out_dtype="bf16"), nk.experts_packed(h, want[2], layer.second, weights=want[1])]
            stream.synchronize()
            torch.cuda.synchronize()
            assert nk.synchronize() == 0
        finally:
            nk.set_stream(0)
        assert same(got, want[:5])
        return
    if chosen == "the same":
        nk.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            for _ in range(4):
                big = torch.mm(big, big).clamp_(-1, 1)
            layer.x.copy_(x)
            got = layer()
        stream.synchronize()
        assert same(got, want)
    finally:
        nk.set_stream(0)
    assert nk.synchronize() == 0


def test_two_threads_at_once():
    layers = [Layer(5), Layer(6, tokens=300)]
    wants = [layer() for layer in layers]
    torch.cuda.synchronize()
    failures = []

    def work(layer, want):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(15):
                got = layer()
                stream.synchronize()
                if not same(got, want):
                    failures.append(layer)
    threads = [threading.Thread(target=work, args=pair) for pair in zip(layers, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    assert nk.synchronize() == 0


def test_rows_past_32_bit_offsets():
    """Every operand as columns of a wide matrix, rows 4 MB apart, over 4 GiB long."""
    rows, wide, k, n = 1100, 1 << 22, 300, 70
    held = torch.zeros(rows, wide, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)

    def spread(t, at):
        view = held[:, at:at + t.shape[1] * t.element_size()].view(t.dtype)
        view.copy_(t)
        return view
    x = torch.randn(rows, k, generator=g, device="cuda")
    q, packed = nk.mx_quantise(x), nk.dots_pack(nk.mx_quantise(torch.randn(n, k, generator=g, device="cuda")))
    far = nk.mx_quantise(spread(x, 0))
    assert torch.equal(far.codes, q.codes) and torch.equal(far.scales, q.scales)
    far = nk.MxMatrix(spread(q.codes, 4096), spread(q.scales, 8192), k)
    want = nk.dots_packed(q, packed)
    assert torch.equal(nk.dots_packed(far, packed), want)
    assert torch.equal(nk.mx_dequantise(far), nk.mx_dequantise(q))
    for cells in ("f32", "bf16"):
        out = held[:, 16384:16384 + n * 4].view(torch.float32) if cells == "f32" else held[:, 32768:32768 + n * 2].view(torch.bfloat16)
        assert torch.equal(nk.dots_packed(far, packed, out=out, out_dtype=cells), nk.dots_packed(q, packed, out_dtype=cells))
    logits = torch.randn(rows, 16, generator=g, device="cuda")
    weights, ids = nk.route(logits, 4)
    far_logits = spread(logits, 65536)
    assert same(nk.route(far_logits, 4), (weights, ids))
    assert torch.equal(nk.route_gradient(weights, ids, far_logits), nk.route_gradient(weights, ids, logits))
    experts = nk.dots_pack(nk.mx_quantise(torch.randn(16 * n, k, generator=g, device="cuda")), groups=16)
    out = held[:, 131072:131072 + n * 4].view(torch.float32)
    assert torch.equal(nk.experts_packed(spread(x, 0), ids, experts, weights=weights, out=out), nk.experts_packed(x, ids, experts, weights=weights))
    assert nk.synchronize() == 0


def test_a_packed_matrix_past_32_bit_offsets():
    """Experts whose matrices lie more than 4 GiB into the packed blob."""
    experts, n, k = 72, 8192, 16384
    g = torch.Generator(device="cuda").manual_seed(8)
    codes = torch.randint(0, 256, (experts * n, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    scales = torch.randint(120, 130, (experts * n, k // 32), generator=g, dtype=torch.uint8, device="cuda")
    packed = nk.dots_pack(nk.MxMatrix(codes, scales, k), groups=experts)
    assert packed.buffer.numel() > 1 << 32
    x = torch.randn(3, k, generator=g, device="cuda").bfloat16()
    ids = torch.tensor([[71, 0], [70, 69], [5, 71]], dtype=torch.int32, device="cuda")
    got = nk.experts_packed(x, ids, packed)
    for e in (0, 5, 69, 70, 71):
        only = nk.dots_pack(nk.MxMatrix(codes[e * n:(e + 1) * n], scales[e * n:(e + 1) * n], k))
        want = nk.dots_packed(nk.mx_quantise(x), only)
        for t, j in (ids == e).nonzero().tolist():
            assert torch.equal(got[t, j], want[t])
    assert nk.synchronize() == 0


@pytest.mark.parametrize("m,n", [(1, 64), (40, 300), (2304, 2304)])
def test_scales_of_any_size(m, n):
    """Scales from one end of their range to the other whose products are ordinary numbers: exact, each cell being one value."""
    rng = np.random.default_rng(m)
    k = 256
    a_codes, b_codes = np.zeros((m, k // 2), np.uint8), np.zeros((n, k // 2), np.uint8)
    a_codes[:, 7], b_codes[:, 7] = rng.integers(0, 16, m), rng.integers(0, 16, n)  # value 14 of each row
    a_scale, b_scale = rng.integers(0, 255, m), rng.integers(0, 255, n)
    b_scale[: n // 2] = 254 - a_scale[rng.integers(0, m, n // 2)]
    values = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6])

    def mx(codes, scale):
        return nk.MxMatrix(torch.from_numpy(codes).cuda(), torch.from_numpy(np.repeat(scale[:, None], k // 32, 1).astype(np.uint8)).cuda(), k)
    got = nk.dots_packed(mx(a_codes, a_scale), nk.dots_pack(mx(b_codes, b_scale))).double().cpu().numpy()
    assert nk.synchronize() == 0
    want = values[a_codes[:, 7], None] * np.exp2(a_scale[:, None] - 127.0) * (values[b_codes[:, 7]] * np.exp2(b_scale - 127.0))
    normal = (np.abs(want) >= 2.0 ** -126) & (np.abs(want) < 2.0 ** 127) | (want == 0)
    assert normal.any() and np.array_equal(got[normal], want[normal])
    small = np.abs(want) < 2.0 ** -126
    assert (np.abs(got[small]) <= 2.0 ** -126).all()
    large = np.abs(want) >= 2.0 ** 128
    assert np.isinf(got[large]).all() and (np.sign(got[large]) == np.sign(want[large])).all()


@pytest.mark.parametrize("m,n", [(64, 20000), (600, 20000)])
def test_waits_that_give_up(m, n):
    """The epilogue's waits run out: the error word says so once, and the next call is right."""
    k = 8192
    g = torch.Generator(device="cuda").manual_seed(m)
    q = nk.mx_quantise(torch.randn(m, k, generator=g, device="cuda"))
    packed = nk.dots_pack(nk.mx_quantise(torch.randn(n, k, generator=g, device="cuda")))
    want = nk.dots_packed(q, packed)
    assert nk.synchronize() == 0
    nk.set_wait_limit_ns(0, 20_000_000)  # every site: 20 ms
    nk.set_wait_limit_ns(4, 3_000)       # the epilogue's wait for an accumulator: 3 microseconds
    try:
        nk.dots_packed(q, packed)
        word = nk.synchronize()
    finally:
        nk.set_wait_limit_ns(0, 0)
    assert word & 0x80000000 and (word >> 16) & 0xff == 4
    assert torch.equal(nk.dots_packed(q, packed), want)
    assert nk.synchronize() == 0
