"""Routing on the device: the choice bit for bit and the weights against the definition in 64 bits, gradients against the
formula and against differences."""
import numpy as np
import pytest
import torch

import _mx_reference as ref
import numkong_b200 as nk

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# Weights are computed in 64 bits (or in 32 with a handful of roundings) and stored in f32: eight half steps of the value.
WEIGHT_RTOL = 8 * 2.0 ** -24
# Gradients are differences of such products; the same eight half steps, of the largest term.
CASES = [
    dict(top=1), dict(top=8), dict(top=6, renormalise=False), dict(top=4, score="sigmoid"), dict(top=8, score="sigmoid", bias=True, groups=8, top_groups=4, scale=2.5),
    dict(top=5, bias=True), dict(top=3, groups=2, top_groups=1), dict(top=7, score="sigmoid", renormalise=False, groups=4, top_groups=3, bias=True),
    dict(top=32, bias=True, scale=0.5), dict(top=2, groups=32, top_groups=5),
]


def logits_of(tokens, experts, name, seed, spread=1.0):
    x = np.random.default_rng(seed).standard_normal((tokens, experts)).astype(np.float32) * spread
    t = torch.from_numpy(x).to(TORCH[name])
    return t, t.double().numpy()


def run(t, exact, case, bias_values):
    case = dict(case)
    bias = bias_values if case.pop("bias", False) else None
    want_w, want_ids = ref.route(exact, bias=bias, **case)
    w, ids = nk.route(t.cuda(), bias=None if bias is None else torch.from_numpy(bias).cuda(), **case)
    assert nk.synchronize() == 0
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.double().cpu().numpy()
    assert np.allclose(got, want_w, rtol=WEIGHT_RTOL, atol=1e-37)
    return want_w, want_ids


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("tokens,experts", [(1, 64), (77, 64), (33, 256), (5, 1024), (19, 96)])
def test_route(tokens, experts, case, name):
    t, exact = logits_of(tokens, experts, name, tokens + experts)
    bias = (0.05 * np.random.default_rng(3).standard_normal(experts)).astype(np.float32)
    run(t, exact, case, bias)


@pytest.mark.parametrize("experts,top", [(1, 1), (2, 2), (3, 2), (31, 31), (33, 32), (40, 7), (511, 16), (1000, 9)])
def test_route_odd_sizes(experts, top):
    t, exact = logits_of(29, experts, "f32", experts, 3.0)
    for score in ("softmax", "sigmoid"):
        run(t, exact, dict(top=top, score=score), None)
        run(t, exact, dict(top=top, score=score, bias=True, renormalise=False), np.zeros(experts, np.float32))


@pytest.mark.parametrize("tokens", [4095, 4096, 4097, 5003])
@pytest.mark.parametrize("experts,top", [(64, 6), (40, 9), (200, 20), (1000, 8), (33, 1)])
def test_many_tokens(tokens, experts, top):
    """Enough tokens that a warp works on several at once, numbers of them that fill no batch, infinities and ties among them."""
    rng = np.random.default_rng(tokens + experts)
    x = (rng.standard_normal((tokens, experts)) * 2).astype(np.float32)
    x[5, :], x[7, ::2], x[tokens - 1, 1:] = -np.inf, np.nan, -np.inf
    x[11] = 0
    g = rng.standard_normal((tokens, top)).astype(np.float32)
    for score, renormalise in (("softmax", True), ("sigmoid", True), ("softmax", False)):
        how = dict(score=score, renormalise=renormalise, scale=1.5)
        w, ids = nk.route(torch.from_numpy(x).cuda(), top, **how)
        some = np.r_[0:40, tokens // 2:tokens // 2 + 9, tokens - 9:tokens]
        want_w, want_ids = ref.route(x[some], top, **how)
        assert np.array_equal(ids.cpu().numpy()[some], want_ids)
        assert np.allclose(w.double().cpu().numpy()[some], want_w, rtol=WEIGHT_RTOL, atol=1e-37)
        grad = nk.route_gradient(torch.from_numpy(g).cuda(), ids, torch.from_numpy(x).cuda(), **how)
        assert nk.synchronize() == 0
        want = ref.route_gradient(g[some], want_ids, x[some], **how)
        size = 1.5 * np.abs(g[some]).sum(1, keepdims=True)
        assert (np.abs(grad.double().cpu().numpy()[some] - want) <= WEIGHT_RTOL * (np.abs(want) + size)).all()


def test_ties_go_to_the_lower_index():
    x = np.zeros((4, 64), np.float32)
    x[1, 50:] = 1
    x[2, ::2] = 2
    bias = np.zeros(64, np.float32)
    bias[40:44] = 0.25
    for case in (dict(top=8), dict(top=8, bias=True), dict(top=8, groups=8, top_groups=3), dict(top=8, groups=8, top_groups=3, bias=True, score="sigmoid")):
        run(torch.from_numpy(x), x, case, bias)


def test_near_ties_are_decided_in_64_bits():
    """Scores that 32 bits cannot tell apart: neighbouring f32 logits deep in the flat end of the sigmoid, and biases that
    cancel score differences to the last bits."""
    rng = np.random.default_rng(1)
    base = np.float32(9.0)
    steps = rng.permuted(np.tile(np.arange(64), (50, 1)), axis=1)
    x = base + steps.astype(np.float32) * np.spacing(base)
    run(torch.from_numpy(x), x.astype(np.float64), dict(top=8, score="sigmoid", bias=True), np.full(64, 0.125, np.float32))
    logits = rng.standard_normal((200, 64)).astype(np.float32)
    logits[:, 1::2] = logits[:, ::2] + (rng.integers(-2, 3, (200, 32)) * np.spacing(logits[:, ::2])).astype(np.float32)
    run(torch.from_numpy(logits), logits.astype(np.float64), dict(top=16, score="softmax", bias=True, groups=4, top_groups=2), np.zeros(64, np.float32))


@pytest.mark.parametrize("case", [dict(top=4), dict(top=4, renormalise=False), dict(top=4, score="sigmoid", bias=True, groups=4, top_groups=2), dict(top=4, score="sigmoid", renormalise=False)], ids=str)
def test_masked_logits(case):
    x = np.random.default_rng(5).standard_normal((9, 32)).astype(np.float32)
    x[0] = -np.inf                       # nobody
    x[1, 2:] = -np.inf                   # two
    x[2, ::3] = np.nan
    x[3] = np.nan
    x[4, 7] = np.inf
    x[5, [3, 9]] = np.inf
    x[6] = np.finfo(np.float32).min      # the type's lowest value is not a mask
    x[7, 8:] = np.finfo(np.float32).min
    x[8] = -3e38
    bias = (0.01 * np.arange(32)).astype(np.float32)
    bias[30], bias[31] = -np.inf, np.nan
    w, ids = run(torch.from_numpy(x), x, case, bias)
    assert (ids[0] == -1).all() and (ids[3] == -1).all() and (w[0] == 0).all()
    assert (ids[1] >= 0).sum() == 2


@pytest.mark.parametrize("offset,spread", [(5.0, 0.1), (-5.0, 0.1), (0.0, 30.0), (1e8, 0.0), (0.0, 1e30), (-1e-30, 0.0)])
def test_biases_of_any_size(offset, spread):
    """Biases beyond the scores' range, far from zero, all of one sign, infinite."""
    x = np.random.default_rng(11).standard_normal((40, 96)).astype(np.float32)
    bias = (offset + spread * np.random.default_rng(12).standard_normal(96)).astype(np.float32)
    for case in (dict(top=6, score="sigmoid"), dict(top=6), dict(top=5, groups=8, top_groups=3, score="sigmoid"), dict(top=5, groups=6, top_groups=2)):
        run(torch.from_numpy(x), x, dict(case, bias=True), bias)
        barred = bias.copy()
        barred[::5], barred[1] = -np.inf, np.inf
        run(torch.from_numpy(x), x, dict(case, bias=True), barred)


def test_groups_with_one_expert_left():
    x = np.random.default_rng(13).standard_normal((64, 64)).astype(np.float32)
    x[:, 1:8] = -np.inf                 # one left in the first group
    x[::2, 8:16] = -np.inf              # none in the second
    x[::3, 17:24] = np.nan
    bias = (0.3 * np.random.default_rng(14).standard_normal(64)).astype(np.float32)
    for shift in (-0.5, 0.0, 2.0):
        for score in ("softmax", "sigmoid"):
            run(torch.from_numpy(x), x, dict(top=9, groups=8, top_groups=5, score=score, bias=True), bias + np.float32(shift))
    run(torch.from_numpy(x), x, dict(top=9, groups=8, top_groups=5), None)


def test_f32_logits_that_differ_in_their_last_bits():
    """Without a bias the choice is the logits' own order, to the last bit, at every size and sign."""
    rng = np.random.default_rng(15)
    base = np.repeat(rng.standard_normal((60, 8)).astype(np.float32) * 50, 16, axis=1)
    x = base.view(np.int32) + rng.permuted(np.tile(np.arange(128, dtype=np.int32) % 16, (60, 1)), axis=1)
    x = x.view(np.float32)
    for score in ("softmax", "sigmoid"):
        run(torch.from_numpy(x), x, dict(top=20, score=score), None)


def test_scores_too_small_to_represent_renormalise():
    x = np.full((3, 16), -200, np.float32)
    x[1, 4], x[2] = -190, -1e4
    run(torch.from_numpy(x), x, dict(top=4, score="sigmoid"), None)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (7, 33, 4), (50, 64, 6), (21, 256, 8), (3, 1000, 32)])
def test_gradient(tokens, experts, top, name, renormalise, score):
    t, exact = logits_of(tokens, experts, name, 7 * experts + tokens)
    how = dict(score=score, renormalise=renormalise, scale=1.5)
    _, ids = ref.route(exact, top, **how)
    g = np.random.default_rng(2).standard_normal((tokens, top)).astype(np.float32)
    want = ref.route_gradient(g, ids, exact, **how)
    got = nk.route_gradient(torch.from_numpy(g).cuda(), torch.from_numpy(ids).cuda(), t.cuda(), **how)
    assert nk.synchronize() == 0
    got = got.double().cpu().numpy()
    size = 1.5 * np.abs(g).sum(1, keepdims=True)
    assert (np.abs(got - want) <= WEIGHT_RTOL * (np.abs(want) + size)).all()
    # the formula against differences, in 64 bits
    if experts <= 64:
        step = 1e-4
        for e in range(0, experts, 5):
            up, down = exact.copy(), exact.copy()
            up[:, e] += step
            down[:, e] -= step
            def total(x):
                s = ref.scores_of(x, score)
                p = np.take_along_axis(s, ids, 1)
                return (1.5 * g * (p / p.sum(1, keepdims=True) if renormalise else p)).sum(1)
            slope = (total(up) - total(down)) / (2 * step)
            assert np.allclose(slope, want[:, e], atol=1e-6)  # step^2 / 6 times a third derivative of at most a few


def test_gradient_odd_ids():
    """Slots without an expert, ids out of range, an expert named twice, a masked logit."""
    x = np.random.default_rng(4).standard_normal((5, 40)).astype(np.float32)
    x[2, 11] = -np.inf
    ids = np.array([[3, -1, 5], [7, 7, 2], [11, 0, 1], [40, 2, 2147483647], [-1, -1, -1]], np.int32)
    g = np.random.default_rng(6).standard_normal((5, 3)).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            how = dict(score=score, renormalise=renormalise, scale=2.0)
            want = ref.route_gradient(g, ids, x, **how)
            got = nk.route_gradient(torch.from_numpy(g).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(x).cuda(), **how)
            assert nk.synchronize() == 0
            assert (np.abs(got.double().cpu().numpy() - want) <= WEIGHT_RTOL * (np.abs(want) + 2 * np.abs(g).sum(1, keepdims=True))).all()
            assert (got[4] == 0).all()


def test_route_strides_and_host():
    x = np.random.default_rng(8).standard_normal((23, 70)).astype(np.float32)
    wide = torch.from_numpy(np.pad(x, ((0, 0), (3, 2)))).cuda()
    want = nk.route(torch.from_numpy(x).cuda(), 5)
    got = nk.route(wide[:, 3:73], 5)
    host = nk.route(x, 5)
    assert nk.synchronize() == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert np.array_equal(host[0], want[0].cpu().numpy()) and np.array_equal(host[1], want[1].cpu().numpy())
    grad = nk.route_gradient(host[0], host[1], x)
    assert np.array_equal(grad, nk.route_gradient(want[0], want[1], wide[:, 3:73]).cpu().numpy())


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("experts,top", [(2, 1), (40, 3), (300, 32)])
def test_zeros_of_either_sign_tie(experts, top, name):
    logits = torch.zeros(3, experts, dtype=TORCH[name], device="cuda")
    logits[0, ::2] = -0.0
    logits[1, 1::2] = -0.0
    _, ids = nk.route(logits, top)
    assert (ids.cpu() == torch.arange(top)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
def test_tokens_do_not_depend_on_one_another(score, renormalise):
    """The same bits for a token alone, in a batch, and beside tokens whose scores almost vanish."""
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = 3 * torch.randn(5000, 48, generator=g, device="cuda")
    logits[1::4] -= 95
    logits[2::4] += 95
    how = dict(score=score, renormalise=renormalise)
    weights, ids = nk.route(logits, 6, **how)
    incoming = torch.randn(5000, 6, generator=g, device="cuda")
    grad = nk.route_gradient(incoming, ids, logits, **how)
    for first, count in ((0, 1), (4, 1), (8, 3), (1000, 700)):
        part = logits[first:first + count]
        some, chosen = nk.route(part, 6, **how)
        assert torch.equal(some, weights[first:first + count]) and torch.equal(chosen, ids[first:first + count])
        assert torch.equal(nk.route_gradient(incoming[first:first + count], chosen, part, **how), grad[first:first + count])
    assert nk.synchronize() == 0
