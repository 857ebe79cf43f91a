"""The experts' products on the device against 64-bit products of the exactly decoded operands, and a decoding step that runs
all the 4-bit and routing operators together."""
import numpy as np
import pytest
import torch

import _mx_reference as ref
import numkong_b200 as nk

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(tokens, experts, top, n, k, per_slot, name, seed):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((tokens, top, k) if per_slot else (tokens, k)).astype(np.float32)).to(TORCH[name])
    ids = np.stack([rng.permutation(experts)[:top] for _ in range(tokens)]).astype(np.int32) if experts >= top else rng.integers(0, experts, (tokens, top)).astype(np.int32)
    w = rng.standard_normal((experts * n, k)).astype(np.float32)
    return x, ids, w, rng


def expected(x, ids, codes, scales, n, k, weights):
    """(exact result, bound on the error of f32 cells)."""
    tokens, top = ids.shape
    flat = x.double().numpy().reshape(-1, k)
    a = ref.dequantise(*ref.quantise(flat), k)
    if x.dim() == 2:
        a = a.repeat(top, axis=0)
    b = ref.dequantise(codes, scales, k).reshape(-1, n, k)
    y, bound = np.zeros((tokens * top, n)), np.zeros((tokens * top, n))
    for s, e in enumerate(ids.reshape(-1)):
        if 0 <= e < len(b):
            y[s] = b[e] @ a[s]
            bound[s] = ref.product_bound(a[s:s + 1], b[e], "f32")[0]
    y, bound = y.reshape(tokens, top, n), bound.reshape(tokens, top, n)
    if weights is not None:
        w = np.where((ids >= 0) & (ids < len(b)), weights.astype(np.float64), 0)[:, :, None]  # slots without an expert are left out
        part = np.abs(w) * (np.abs(y) + bound)
        bound = (np.abs(w) * bound).sum(1) + (top + 1) * 2.0 ** -24 * part.sum(1)
        y = (w * y).sum(1)
    return y, bound


def run(x, ids, w, n, k, weights, cells, experts):
    q = nk.mx_quantise(torch.from_numpy(w).cuda())
    packed = nk.dots_pack(q, groups=experts)
    got = nk.experts_packed(x.cuda(), torch.from_numpy(ids).cuda(), packed, weights=None if weights is None else torch.from_numpy(weights).cuda(), out_dtype=cells)
    assert nk.synchronize() == 0
    y, bound = expected(x, ids, q.codes.cpu().numpy(), q.scales.cpu().numpy(), n, k, weights)
    assert got.shape == y.shape and got.dtype == TORCH[cells]
    if cells == "bf16":
        bound = bound + 2.0 ** -8 * (np.abs(y) + bound)
    off = np.abs(got.double().cpu().numpy() - y)
    assert (off <= bound).all(), float((off - bound).max())
    return got


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("tokens,experts,top,n,k,name,cells", [
    (1, 1, 1, 1, 1, "f32", "f32"), (1, 8, 2, 64, 100, "bf16", "f32"), (3, 4, 3, 130, 257, "f16", "bf16"), (40, 6, 2, 200, 64, "bf16", "bf16"),
    (300, 3, 2, 100, 300, "f32", "f32"), (129, 1, 1, 128, 256, "bf16", "f32"), (17, 64, 6, 96, 512, "bf16", "f32"), (513, 2, 1, 257, 33, "f32", "bf16")])
def test_experts(tokens, experts, top, n, k, name, cells, per_slot, weighted):
    x, ids, w, rng = make(tokens, experts, top, n, k, per_slot, name, tokens + n)
    weights = rng.random((tokens, top)).astype(np.float32) if weighted else None
    run(x, ids, w, n, k, weights, cells, experts)


def test_uneven_and_missing_experts():
    """All tokens on one expert, the same expert twice, experts that nobody chose, slots without an expert."""
    tokens, experts, top, n, k = 260, 5, 2, 70, 128
    x, ids, w, rng = make(tokens, experts, top, n, k, False, "bf16", 1)
    ids[:] = 3
    run(x, ids, w, n, k, None, "f32", experts)
    ids[::2, 1] = -1
    ids[7] = [-1, 99]
    ids[8] = [2147483647, -2147483648]
    for weights in (None, rng.random((tokens, top)).astype(np.float32)):
        for cells in ("f32", "bf16"):
            got = run(x, ids, w, n, k, weights, cells, experts)
            assert (got[7] == 0).all() and (got[8] == 0).all()
    if weights is not None:  # a weight of a slot without an expert is not looked at
        weights[7] = np.nan
        got = run(x, ids, w, n, k, weights, "f32", experts)
        assert (got[7] == 0).all()
    ids[:] = -1
    assert (run(x, ids, w, n, k, None, "f32", experts) == 0).all()


def test_results_repeat_bit_for_bit():
    x, ids, w, rng = make(700, 9, 3, 300, 320, False, "bf16", 2)
    weights = torch.from_numpy(rng.random((700, 3)).astype(np.float32)).cuda()
    packed = nk.dots_pack(nk.mx_quantise(torch.from_numpy(w).cuda()), groups=9)
    args = x.cuda(), torch.from_numpy(ids).cuda(), packed
    first, sums = nk.experts_packed(*args), nk.experts_packed(*args, weights=weights)
    # the same rows as a plain product with one expert's matrix
    only = nk.dots_pack(nk.mx_quantise(torch.from_numpy(w[4 * 300:5 * 300]).cuda()))
    rows = np.argwhere(ids == 4)
    assert torch.equal(first[rows[:, 0], rows[:, 1]], nk.dots_packed(args[0], only)[rows[:, 0]])
    for _ in range(5):
        assert torch.equal(nk.experts_packed(*args), first)
        assert torch.equal(nk.experts_packed(*args, weights=weights), sums)
    assert nk.synchronize() == 0


def test_rows_outside_the_result_stay():
    x, ids, w, _ = make(20, 3, 2, 33, 64, False, "f32", 3)
    packed = nk.dots_pack(nk.mx_quantise(torch.from_numpy(w).cuda()), groups=3)
    held = torch.full((22, 40), 5.0, device="cuda")
    weights = torch.rand(20, 2, device="cuda")
    got = nk.experts_packed(x.cuda(), torch.from_numpy(ids).cuda(), packed, weights=weights, out=held[1:21, 2:35])
    assert nk.synchronize() == 0
    assert torch.equal(got, nk.experts_packed(x.cuda(), torch.from_numpy(ids).cuda(), packed, weights=weights))
    assert (held[0] == 5).all() and (held[21] == 5).all() and (held[:, :2] == 5).all() and (held[:, 35:] == 5).all()


def test_experts_on_the_host():
    x, ids, w, rng = make(30, 4, 2, 50, 96, False, "f32", 4)
    weights = rng.random((30, 2)).astype(np.float32)
    packed = nk.dots_pack(nk.mx_quantise(w), groups=4)
    got = nk.experts_packed(x.numpy(), ids, packed, weights=weights)
    want = nk.experts_packed(x.cuda(), torch.from_numpy(ids).cuda(), nk.dots_pack(nk.mx_quantise(torch.from_numpy(w).cuda()), groups=4),
                             weights=torch.from_numpy(weights).cuda())
    assert np.array_equal(got, want.cpu().numpy())


def test_a_layer_of_experts_from_logits_to_sums():
    """Router product, routing, both expert layers and the weighted sum, as a program runs them."""
    tokens, experts, top, k, hidden = 90, 16, 4, 256, 320
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
    router = nk.dots_pack(nk.mx_quantise(torch.randn(experts, k, generator=g, device="cuda") * k ** -0.5))
    first = nk.dots_pack(nk.mx_quantise(torch.randn(experts * hidden, k, generator=g, device="cuda") * k ** -0.5), groups=experts)
    second_q = nk.mx_quantise(torch.randn(experts * k, hidden, generator=g, device="cuda") * hidden ** -0.5)
    second = nk.dots_pack(second_q, groups=experts)
    logits = nk.dots_packed(x, router)
    weights, ids = nk.route(logits, top, score="sigmoid")
    h = nk.experts_packed(x, ids, first, out_dtype="bf16")
    h = torch.nn.functional.silu(h.float()).bfloat16()
    out = nk.experts_packed(h, ids, second, weights=weights)
    assert nk.synchronize() == 0
    want_w, want_ids = ref.route(logits.double().cpu().numpy(), top, score="sigmoid")
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    y, bound = expected(h.cpu(), want_ids, second_q.codes.cpu().numpy(), second_q.scales.cpu().numpy(), k, hidden, weights.cpu().numpy())
    assert (np.abs(out.double().cpu().numpy() - y) <= bound).all()


@pytest.mark.parametrize("tokens,experts,top", [(9001, 5, 2), (700, 1024, 3), (18000, 1, 1)])
def test_many_slots(tokens, experts, top):
    """More slots than a pass of the order takes, experts without a slot, one expert for all."""
    x, ids, w, _ = make(tokens, experts, top, 8, 32, False, "bf16", tokens)
    ids[::7, 0] = -1
    run(x, ids, w, 8, 32, None, "f32", experts)


def test_the_workload_runs():
    from numkong_b200.workloads import run_experts
    out = run_experts(40, 6, 2, 192, 130, steps=2, warmup=1)
    assert out["workload"] == "experts" and out["ms"] > 0 and out["tokens_per_s"] > 0


@pytest.mark.parametrize("tokens,experts,top", [(256, 1, 1), (200, 1, 1), (128, 3, 2), (64, 1024, 4), (86, 40, 3), (257, 2, 1), (33, 7, 3), (1, 1024, 32)])
def test_few_slots(tokens, experts, top):
    """As many slots as are ordered and quantised in one launch, and one more: any ids, missing ones among them."""
    x, ids, w, rng = make(tokens, experts, top, 40, 300, False, "bf16", tokens + top)
    weights = rng.random((tokens, top)).astype(np.float32)
    for _ in range(2):
        run(x, ids, w, 40, 300, None, "bf16", experts)
        run(x, ids, w, 40, 300, weights, "f32", experts)
        ids = np.where(rng.random(ids.shape) < 0.4, rng.integers(-3, experts + 3, ids.shape), ids).astype(np.int32)
    ids[:] = experts - 1
    run(x, ids, w, 40, 300, None, "f32", experts)
    ids[:] = experts
    assert (run(x, ids, w, 40, 300, None, "f32", experts) == 0).all()
