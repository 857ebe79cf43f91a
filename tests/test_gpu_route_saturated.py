"""Choices among scores that 64 bits cannot tell apart: in the order of the logits, whether no bias is given or one that is the same for
all experts, and in that of the indices where biases or groups make keys of the scores."""
import numpy as np
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu

INPUTS = {
    "ones of the sigmoid": ("sigmoid", lambda rng, shape: rng.uniform(20, 90, shape)),
    "sigmoids that tie by rounding": ("sigmoid", lambda rng, shape: 24 + rng.integers(0, 200, shape) * np.spacing(np.float32(24))),
    "zeros of the softmax": ("softmax", lambda rng, shape: rng.uniform(-3000, 0, shape)),
    "logits next to nothing": ("sigmoid", lambda rng, shape: rng.standard_normal(shape) * 1e-12),
    "softmax of logits next to nothing": ("softmax", lambda rng, shape: rng.standard_normal(shape) * 1e-18),
    "some of each": ("sigmoid", lambda rng, shape: rng.standard_normal(shape) * 60),
}


@pytest.mark.parametrize("kind", INPUTS)
@pytest.mark.parametrize("tokens,experts,top", [(30, 64, 8), (4100, 64, 8), (20, 300, 20), (9, 30, 30), (5, 1000, 32)])
def test_a_bias_that_changes_nothing(tokens, experts, top, kind):
    score, make = INPUTS[kind]
    x = make(np.random.default_rng(tokens + experts), (tokens, experts)).astype(np.float32)
    x[::3, 5:9] = x[::3, 5:6]  # and equal logits
    want = np.argsort(-x, axis=1, kind="stable")[:, :top]
    logits = torch.from_numpy(x).cuda()
    weights, ids = nk.route(logits, top, score=score)
    assert np.array_equal(ids.cpu().numpy(), want)
    for value in (0.0, -0.0, 0.125, -1e8, np.inf):
        bias = torch.full((experts,), value, device="cuda")
        some, chosen = nk.route(logits, top, score=score, bias=bias)
        assert torch.equal(chosen, ids) and torch.equal(some, weights)
    barred = torch.full((experts,), -3.5, device="cuda")
    barred[::2] = -np.inf
    barred[1] = np.nan
    x[:, ::2], x[:, 1] = -np.inf, -np.inf
    assert all(torch.equal(a, b) for a, b in zip(nk.route(logits, top, score=score, bias=barred)[1:], nk.route(torch.from_numpy(x).cuda(), top, score=score)[1:]))
    assert nk.synchronize() == 0


def test_biases_make_keys():
    """Scores of 1 under two biases: those with the larger bias, each by their indices."""
    x = np.random.default_rng(1).uniform(40, 80, (40, 64)).astype(np.float32)
    bias = np.where(np.arange(64) % 3 == 0, 0.25, 0).astype(np.float32)
    want = np.argsort(-bias, kind="stable")[:30]
    _, ids = nk.route(torch.from_numpy(x).cuda(), 30, score="sigmoid", bias=torch.from_numpy(bias).cuda())
    assert nk.synchronize() == 0
    assert (ids.cpu().numpy() == want).all()


def test_groups_of_saturated_scores():
    x = np.random.default_rng(2).uniform(40, 80, (40, 64)).astype(np.float32)
    for bias in (None, torch.zeros(64, device="cuda")):
        _, ids = nk.route(torch.from_numpy(x).cuda(), 9, score="sigmoid", groups=8, top_groups=3, bias=bias)
        assert (ids.cpu().numpy() == np.arange(9)).all()
    assert nk.synchronize() == 0
