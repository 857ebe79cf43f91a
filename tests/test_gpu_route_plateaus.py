"""Choices where many experts share one logit and a few differ from it by less than 32 bits can tell: more equal ones than are chosen must
not hide a larger one behind them."""
import numpy as np
import pytest
import torch

import numkong_b200 as nk

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}


def plateau(tokens, experts, level, steps, name, seed):
    """All logits `level`, for a few experts of each token the type's next values above or below it."""
    rng = np.random.default_rng(seed)
    step = np.spacing(np.float32(level)) * (1 if name == "f32" else 2 ** 16)
    x = np.full((tokens, experts), level, np.float32)
    for t in range(tokens):
        some = rng.choice(experts, rng.integers(1, 4), replace=False)
        x[t, some] += step * rng.choice(steps, len(some)).astype(np.float32)
    return torch.from_numpy(x).to(TORCH[name])


@pytest.mark.parametrize("experts", [16, 33, 64, 100, 256, 500, 1000])
@pytest.mark.parametrize("tokens", [40, 4100])
@pytest.mark.parametrize("top", [1, 4, 9, 32])
def test_logits(tokens, experts, top):
    """Without a bias the logits' own order."""
    if top > experts:
        pytest.skip("more choices than experts")
    for score in ("softmax", "sigmoid"):
        for level in (1.0, -3.7, 25.0):
            x = plateau(tokens, experts, level, [-1, 1, 2], "f32", experts + top)
            _, ids = nk.route(x.cuda(), top, score=score)
            assert np.array_equal(ids.cpu().numpy(), np.argsort(-x.numpy(), axis=1, kind="stable")[:, :top])
    assert nk.synchronize() == 0


@pytest.mark.parametrize("experts,groups,top_groups", [(64, 1, 1), (300, 1, 1), (64, 4, 4), (96, 12, 5), (16, 16, 16)])
@pytest.mark.parametrize("name,level", [("f32", 2.0), ("bf16", 15.0), ("bf16", -300.0), ("f32", -300.0)])
@pytest.mark.parametrize("top", [1, 5, 12])
def test_keys(experts, groups, top_groups, name, level, top):
    """With a bias or groups the keys' order in 64 bits, which these scores still differ in."""
    x = plateau(60, experts, level, [-1, 1, 2], name, experts + top)
    bias = np.zeros(experts, np.float32)
    if groups == 1:
        bias[-1] = -2.0  # so that there is one, and it leaves the others' order alone
    _, ids = nk.route(x.cuda(), top, score="sigmoid", groups=groups, top_groups=top_groups, bias=torch.from_numpy(bias).cuda())
    assert nk.synchronize() == 0
    l = x.double().numpy()
    keys = np.exp(np.minimum(l, 0)) / (1 + np.exp(-np.abs(l))) + bias
    for t in range(len(l)):
        k = keys[t].copy()
        if groups > 1:
            by = -np.sort(-k.reshape(groups, -1), axis=1)[:, :2].sum(1)
            shut = np.argsort(-by, kind="stable")[top_groups:]
            k.reshape(groups, -1)[shut] = -np.inf
        assert ids[t].tolist() == np.argsort(-k, kind="stable")[:top].tolist()
