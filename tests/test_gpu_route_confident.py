"""Gradients of routers that have made up their minds: one score so far above the others that what its expert's gradient is
made of nearly cancels. Every value is held to its own size, not to that of the incoming gradient."""
import numpy as np
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
# A chosen expert's gradient, with p its score's numerator, g the incoming gradients and S the sum of the numerators, is
#   p_e (sum over the chosen j of p_j (g_e - g_j), plus g_e times the others' numerators) / S^2, for sigmoids times 1 - s_e.
# Half steps of f32 (u = 2^-24) in it: an exponential two, the rounding of its argument made good for one more, so 3 for every p and for
# sums of them; p_e 3, S^2 6, the bracket's terms 3, the result's rounding 1: 13. Sigmoids: 2 for each score, 2 for 1 - s, in all 11.
# An expert that was not chosen: its p 3, the factor all of them share 3 + 6 + 1, their product 1: 14. Sixteen hold for all, of the
# sum of the terms' magnitudes; 64-bit roundings are nothing beside that.
RTOL = 16 * 2.0 ** -24
ATOL = 2.0 ** -123  # numerators below f32's normal range lose their digits


def exact(g, ids, x, score, renormalise):
    """(gradient, sum of its terms' magnitudes) by the formula above in 64 bits, which nothing cancels in but the terms themselves."""
    tokens, experts = x.shape
    out, size = np.zeros((tokens, experts)), np.zeros((tokens, experts))
    for t in range(tokens):
        here = [int(e) for e in ids[t]]
        if score == "sigmoid":
            log_p = np.where(x[t] >= 0, -np.log1p(np.exp(-np.abs(x[t]))), x[t] - np.log1p(np.exp(-np.abs(x[t]))))
            other = np.exp(np.where(x[t] >= 0, -x[t] - np.log1p(np.exp(-np.abs(x[t]))), -np.log1p(np.exp(-np.abs(x[t])))))  # 1 - s
        else:
            log_p, other = x[t], np.ones(experts)
        if renormalise:
            p = np.exp(log_p - log_p[here].max())
            total = p[here].sum()
            for j, e in enumerate(here):
                terms = np.array([p[i] * (g[t, j] - g[t, m]) for m, i in enumerate(here)])
                out[t, e] += p[e] * terms.sum() / total ** 2 * other[e]
                size[t, e] += p[e] * np.abs(terms).sum() / total ** 2 * other[e]
        else:
            p = np.exp(log_p - log_p.max())
            total = p.sum()
            distinct = sorted(set(here))
            whole = {e: sum(g[t, j] for j, i in enumerate(here) if i == e) for e in distinct}
            rest = p[[e for e in range(experts) if e not in whole]].sum()
            for e in range(experts):
                if e in whole:
                    terms = np.array([p[i] * (whole[e] - whole[i]) for i in distinct] + [whole[e] * rest])
                else:
                    terms = -np.array([p[i] * whole[i] for i in distinct])
                out[t, e], size[t, e] = p[e] * terms.sum() / total ** 2, p[e] * np.abs(terms).sum() / total ** 2
    return out, size


def check(x, ids, g, score, renormalise, scale=1.5):
    want, size = exact(scale * g.astype(np.float64), ids, x.double().numpy(), score, renormalise)
    got = nk.route_gradient(torch.from_numpy(g).cuda(), torch.from_numpy(ids).cuda(), x.cuda(), score=score, renormalise=renormalise, scale=scale)
    assert nk.synchronize() == 0
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= RTOL * size + ATOL).all(), float((off / (size + ATOL)).max() / 2.0 ** -24)


def confident(tokens, experts, gap, name, seed):
    """One logit per token `gap` above the largest of the others."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((tokens, experts)).astype(np.float32)
    x[np.arange(tokens), rng.integers(0, experts, tokens)] = x.max(1) + np.float32(gap)
    return torch.from_numpy(x).to(TORCH[name])


HOW = [("softmax", False), ("softmax", True), ("sigmoid", True)]


@pytest.mark.parametrize("score,renormalise", HOW)
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [0, 5, 10, 14, 18, 22, 30, 45, 70])
def test_one_logit_far_above_the_others(gap, name, score, renormalise):
    for tokens, experts, top in ((20, 64, 1), (20, 64, 2), (9, 40, 6), (5, 300, 20)):
        x = confident(tokens, experts, gap, name, gap + top)
        if score == "sigmoid":
            x = x - gap  # where the scores still differ by that much
        ids = np.argsort(-x.double().numpy(), axis=1, kind="stable")[:, :top].astype(np.int32)
        g = np.random.default_rng(top).standard_normal((tokens, top)).astype(np.float32)
        check(x, ids, g, score, renormalise)


@pytest.mark.parametrize("score,renormalise", HOW)
def test_any_ids_and_incoming_gradients(score, renormalise):
    """The far logit chosen last, not at all, or twice; incoming gradients that are equal, zero or far apart."""
    x = confident(8, 40, 16, "f32", 3)
    if score == "sigmoid":
        x = x - 16
    best = x.argmax(1).numpy()
    rng = np.random.default_rng(4)
    ids = np.array([rng.choice([e for e in range(40) if e != b], 3, replace=False) for b in best], np.int32)
    ids[1:3, 2] = best[1:3]
    ids[3], ids[4], ids[5, 0] = best[3], [best[4], ids[4, 1], best[4]], best[5]
    g = rng.standard_normal((8, 3)).astype(np.float32)
    g[2], g[5] = 0.75, [1e4, 1e-4, -1e4]
    g[6], g[7] = 0, [0, 1, 0]
    check(x, ids, g, score, renormalise)


@pytest.mark.parametrize("score,renormalise", HOW)
@pytest.mark.parametrize("top", [2, 9])
def test_many_tokens(top, score, renormalise):
    """Enough tokens that a warp works on several at once: the same bits as for the same tokens alone, held to the same bound."""
    x = confident(4100, 48, 17, "f32", 5)
    if score == "sigmoid":
        x = x - 17
    ids = np.argsort(-x.numpy(), axis=1, kind="stable")[:, :top].astype(np.int32)
    g = np.random.default_rng(6).standard_normal((4100, top)).astype(np.float32)
    how = dict(score=score, renormalise=renormalise, scale=1.5)
    whole = nk.route_gradient(torch.from_numpy(g).cuda(), torch.from_numpy(ids).cuda(), x.cuda(), **how)
    for first, count in ((0, 1), (100, 30), (4090, 10)):
        some = slice(first, first + count)
        alone = nk.route_gradient(torch.from_numpy(g[some]).cuda(), torch.from_numpy(ids[some]).cuda(), x[some].cuda(), **how)
        assert torch.equal(alone, whole[some])
        check(x[some], ids[some], g[some], score, renormalise)


def test_a_row_of_the_softmax_sums_to_zero():
    """Adding the same to all logits changes nothing, so a row's gradients cancel, up to their own roundings."""
    x = confident(50, 64, 12, "f32", 7)
    ids = np.argsort(-x.numpy(), axis=1, kind="stable")[:, :2].astype(np.int32)
    g = np.random.default_rng(8).standard_normal((50, 2)).astype(np.float32)
    got = nk.route_gradient(torch.from_numpy(g).cuda(), torch.from_numpy(ids).cuda(), x.cuda(), renormalise=False).double().cpu().numpy()
    assert nk.synchronize() == 0
    _, size = exact(g.astype(np.float64), ids, x.double().numpy(), "softmax", False)
    assert (np.abs(got.sum(1)) <= RTOL * size.sum(1)).all()
