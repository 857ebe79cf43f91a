"""The 4-bit and routing operators as a program calls them, beside their plain forms in elementary torch operations.

Four operators, all of them around products with microscaled 4-bit floats (MXFP4: e2m1 values, one power-of-two scale for
every 32 of a row):

  quantise   a float matrix into 4-bit codes and scales, and the values the codes stand for
  product    C = A . B^T of two such matrices, B packed once
  route      every token's experts and their weights from its logits, and the gradient that trains the router
  experts    every token's rows of its experts' products, or their weighted sum

`own` false: the plain forms. `own` true: the calls into numkong_b200.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32
DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One decoding step of a small batch: the activations of eight sequences, rounded before a 4-bit layer.
        dict(name="quantise_step", op="quantise", rows=8, depth=4096, type="bf16"),
        # A whole prompt's activations, or the rounding of one large weight matrix after training.
        dict(name="quantise_prompt", op="quantise", rows=8192, depth=8192, type="bf16"),
        # Gradients or embeddings kept in 4 bits, whose rows end inside a block.
        dict(name="quantise_ragged", op="quantise", rows=5003, depth=777, type="f32"),
        # A single sequence's decoding step through one square layer: latency, and reading the weights.
        dict(name="product_single", op="product", m=1, n=4096, k=4096, a="bf16", out="bf16"),
        # A batch of 64 sequences through a wide layer: still the weights' bytes.
        dict(name="product_batch", op="product", m=64, n=8192, k=8192, a="bf16", out="f32"),
        # A prompt (or the all-pairs scores of 4-bit embeddings) at the size of the repository's headline product.
        dict(name="product_prompt", op="product", m=8192, n=8192, k=8192, a="mx", out="f32"),
        # Sizes that fill no tile: a cut-down vocabulary, a depth that ends inside a block.
        dict(name="product_ragged", op="product", m=1000, n=5003, k=2500, a="mx", out="bf16"),
        # A decoding step's router: 16 tokens, 256 experts in groups, balanced by a bias.
        dict(name="route_step", op="route", tokens=16, experts=256, top=8, score="sigmoid", bias=True, groups=8, top_groups=4, renormalise=True,
             scale=2.5, type="f32", gradient=False),
        # A training step of a softmax router over 64 experts: forward and gradient.
        dict(name="route_train", op="route", tokens=16384, experts=64, top=6, score="softmax", bias=False, groups=1, top_groups=1, renormalise=True,
             scale=1.0, type="bf16", gradient=True),
        # The grouped router over a long prompt, with its gradient.
        dict(name="route_prompt", op="route", tokens=16384, experts=256, top=8, score="sigmoid", bias=True, groups=8, top_groups=4, renormalise=True,
             scale=2.5, type="f32", gradient=True),
        # A decoding step's first expert layer: 32 tokens reach nearly all of 32 experts once or a few times.
        dict(name="experts_step", op="experts", tokens=32, experts=32, top=4, n=4096, k=2048, per_slot=False, weighted=False, type="bf16", out="bf16"),
        # A prompt's second expert layer: rows per token and slot, added up with the router's weights.
        dict(name="experts_prompt", op="experts", tokens=4096, experts=32, top=4, n=2048, k=2048, per_slot=True, weighted=True, type="bf16", out="f32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "route", "experts"])
    if op == "quantise":
        depth = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(1, min(16384, 8192 * 8192 // depth)))
        return dict(op=op, rows=rows, depth=depth, type=rng.choice(["f32", "bf16", "f16"]))
    if op == "product":
        n, k = _log(rng, 16, 16384), _log(rng, 32, 16384)
        m = _log(rng, 1, max(1, min(8192, 8192 ** 3 // (n * k))))
        return dict(op=op, m=m, n=n, k=k, a=rng.choice(["mx", "bf16", "f16", "f32"]), out=rng.choice(["f32", "bf16"]))
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 8 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        top = _log(rng, 1, min(16, top_groups * (experts // groups)))
        tokens = _log(rng, 1, 16384 * 256 // max(256, experts))
        return dict(op=op, tokens=tokens, experts=experts, top=top, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    top_groups=top_groups, renormalise=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), type=rng.choice(["f32", "bf16", "f16"]),
                    gradient=rng.random() < 0.5)
    experts = _log(rng, 4, 64)
    top = rng.randint(1, min(6, experts))
    n, k = _log(rng, 64, 4096), _log(rng, 64, 4096)
    while experts * n * k > 32 * 4096 * 2048:
        n, k = max(64, n // 2), max(64, k // 2 + k % 2)
    per_slot = rng.random() < 0.5
    most = 4096 * 4 * 2048 * 2048 // (n * k * top)
    tokens = _log(rng, 1, max(1, min(4096, most, 2 ** 28 // (experts * n * (top if per_slot else 1)))))
    return dict(op=op, tokens=tokens, experts=experts, top=top, n=n, k=k, per_slot=per_slot, weighted=rng.random() < 0.5,
                type=rng.choice(["f32", "bf16", "f16"]), out=rng.choice(["f32", "bf16"]))


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _activations(g, rows, cols, kind):
    """Activations as layers see them: near normal, with a few channels an order of magnitude above the rest."""
    x = torch.randn(rows, cols, generator=g, device=DEVICE)
    loud = torch.rand(cols, generator=g, device=DEVICE) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(TYPES[kind])


def _weights(g, rows, cols):
    """Weights with a spread of row norms, as codes and scales."""
    spread = torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEVICE))
    return _plain_quantise(torch.randn(rows, cols, generator=g, device=DEVICE) * spread * cols ** -0.5)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case)
    op = case["op"]
    if op == "quantise":
        s["x"] = _activations(g, case["rows"], case["depth"], case["type"])
    elif op == "product":
        x = _activations(g, case["m"], case["k"], "f32" if case["a"] == "mx" else case["a"])
        s["x"] = _plain_quantise(x) if case["a"] == "mx" else x
        s["w"] = _kept(_weights(g, case["n"], case["k"]), case["k"], 1)
    elif op == "route":
        t, e = case["tokens"], case["experts"]
        popular = 0.5 * torch.randn(1, e, generator=g, device=DEVICE)
        s["logits"] = (torch.randn(t, e, generator=g, device=DEVICE) + popular).to(TYPES[case["type"]])
        s["bias_values"] = 0.1 * torch.randn(e, generator=g, device=DEVICE) if case["bias"] else None
        s["weights_grad"] = torch.randn(t, case["top"], generator=g, device=DEVICE) if case["gradient"] else None
    else:
        t, e, j = case["tokens"], case["experts"], case["top"]
        s["x"] = _activations(g, t * j if case["per_slot"] else t, case["k"], case["type"])
        if case["per_slot"]:
            s["x"] = s["x"].view(t, j, case["k"])
        liked = torch.randn(t, e, generator=g, device=DEVICE) + 0.5 * torch.randn(1, e, generator=g, device=DEVICE)
        s["ids"] = torch.sort(liked, dim=1, descending=True).indices[:, :j].to(torch.int32).contiguous()
        part = torch.rand(t, j, generator=g, device=DEVICE) + 0.1
        s["weights"] = part / part.sum(1, keepdim=True) if case["weighted"] else None
        s["w"] = _kept(_weights(g, e * case["n"], case["k"]), case["k"], e)
    return s


def _kept(quantised, depth, groups):
    """What a program keeps of a weight matrix: the packed codes here, the plain values in the plain form."""
    if own:
        import numkong_b200 as nk
        return nk.dots_pack(nk.MxMatrix(quantised[0], quantised[1], depth), groups=groups)
    return _plain_values(quantised[0], quantised[1], depth)


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _power(e):
    """2^e exactly, for -127 <= e <= 127."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _plain_quantise(x):
    """(codes, scales): per 32 values of a row the scale 2^(floor(log2(largest)) - 2), stored as exponent + 127, and each
    value over the scale rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, above 6 to 6). Two
    codes to a byte, the even one in the low half."""
    rows, depth = x.shape
    blocks = (depth + BLOCK - 1) // BLOCK
    v = torch.zeros(rows, blocks * BLOCK, device=x.device)
    v[:, :depth] = x
    v = v.view(rows, blocks, BLOCK)
    largest = v.abs().amax(2)
    exponent = torch.where(largest > 0, torch.frexp(largest).exponent - 3, -127).clamp(-127, 127)
    r = v * _power(-exponent)[:, :, None]
    a = r.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(a / step) * step, max=6.0)
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(r).to(torch.uint8)
    code = code.view(rows, blocks * BLOCK)[:, :depth + depth % 2]
    return (code[:, 0::2] + 16 * code[:, 1::2]).contiguous(), (exponent + 127).to(torch.uint8).contiguous()


def _plain_values(codes, scales, depth):
    rows = codes.shape[0]
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    v = torch.empty(rows, codes.shape[1], 2, device=codes.device)
    v[:, :, 0] = table[(codes & 15).int()]
    v[:, :, 1] = table[(codes >> 4).int()]
    v = v.view(rows, -1)[:, :depth]
    return v * torch.repeat_interleave(_power(scales.int() - 127), BLOCK, dim=1)[:, :depth]


def _plain_scores(logits, score):
    """In 64 bits: which of two near scores is the larger decides who is chosen."""
    x = logits.double()
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    e = torch.exp(x - x.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _plain_route(s):
    t, e = s["logits"].shape
    scores = _plain_scores(s["logits"], s["score"])
    keys = scores if s["bias_values"] is None else scores + s["bias_values"].double()
    if s["groups"] > 1:
        grouped = keys.view(t, s["groups"], -1)
        best = torch.sort(grouped, dim=2, descending=True, stable=True).values[:, :, :2].sum(2)
        chosen = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        open_groups = torch.zeros(t, s["groups"], dtype=torch.bool, device=keys.device).scatter_(1, chosen, True)
        keys = torch.where(open_groups[:, :, None], grouped, -math.inf).view(t, e)
    ids = torch.sort(keys, dim=1, descending=True, stable=True).indices[:, :s["top"]]
    w = torch.gather(scores, 1, ids)
    if s["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return (w * s["scale"]).float(), ids.to(torch.int32), scores


def _plain_route_gradient(s, ids, scores):
    ids, dw = ids.long(), s["weights_grad"].double() * s["scale"]
    p = torch.gather(scores, 1, ids)
    if s["renormalise"]:
        total = p.sum(1, keepdim=True)
        dp = (dw - (dw * p).sum(1, keepdim=True) / total) / total
    else:
        dp = dw
    dscores = torch.zeros_like(scores).scatter_(1, ids, dp)
    if s["score"] == "sigmoid":
        return (dscores * scores * (1 - scores)).float()
    return (scores * (dscores - (dscores * scores).sum(1, keepdim=True))).float()


def _plain_experts(s):
    t, e, j, n, k = s["tokens"], s["experts"], s["top"], s["n"], s["k"]
    rows = s["x"].reshape(-1, k)
    a = _plain_values(*_plain_quantise(rows), k)
    every = torch.matmul(a, s["w"].T).view(a.shape[0], e, n)
    ids = s["ids"].long()
    row = torch.arange(t * j, device=a.device) if s["per_slot"] else torch.arange(t, device=a.device).repeat_interleave(j)
    y = every[row, ids.reshape(-1)].view(t, j, n)
    if s["weights"] is not None:
        y = (y * s["weights"][:, :, None]).sum(1)
    return y.to(TYPES[s["out"]])


def run(s):
    op = s["op"]
    if own:
        import numkong_b200 as nk
        if op == "quantise":
            return nk.mx_dequantise(nk.mx_quantise(s["x"]), s["type"])
        if op == "product":
            a = nk.MxMatrix(s["x"][0], s["x"][1], s["k"]) if s["a"] == "mx" else s["x"]
            return nk.dots_packed(a, s["w"], out_dtype=s["out"])
        if op == "route":
            how = dict(score=s["score"], renormalise=s["renormalise"], scale=s["scale"])
            w, ids = nk.route(s["logits"], s["top"], bias=s["bias_values"], groups=s["groups"], top_groups=s["top_groups"], **how)
            if s["weights_grad"] is None:
                return {"weights": w, "ids": ids}
            return {"weights": w, "ids": ids, "logits_grad": nk.route_gradient(s["weights_grad"], ids, s["logits"], **how)}
        return nk.experts_packed(s["x"], s["ids"], s["w"], weights=s["weights"], out_dtype=s["out"])
    if op == "quantise":
        return _plain_values(*_plain_quantise(s["x"]), s["depth"]).to(TYPES[s["type"]])
    if op == "product":
        a = _plain_values(s["x"][0], s["x"][1], s["k"]) if s["a"] == "mx" else _plain_values(*_plain_quantise(s["x"]), s["k"])
        return torch.matmul(a, s["w"].T).to(TYPES[s["out"]])
    if op == "route":
        w, ids, scores = _plain_route(s)
        if s["weights_grad"] is None:
            return {"weights": w, "ids": ids}
        return {"weights": w, "ids": ids, "logits_grad": _plain_route_gradient(s, ids, scores)}
    return _plain_experts(s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _mx_bytes(rows, depth):
    return rows * ((depth + 1) // 2 + (depth + BLOCK - 1) // BLOCK)


def work(case):
    op = case["op"]
    if op == "quantise":
        return {"bytes": 2 * case["rows"] * case["depth"] * BYTES[case["type"]] + 2 * _mx_bytes(case["rows"], case["depth"]), "flops": 0}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = _mx_bytes(m, k) if case["a"] == "mx" else m * k * BYTES[case["a"]]
        return {"bytes": a + _mx_bytes(n, k) + m * n * BYTES[case["out"]], "flops": 2 * m * n * k}
    if op == "route":
        t, e, j = case["tokens"], case["experts"], case["top"]
        forward = t * e * BYTES[case["type"]] + 8 * t * j + (4 * e if case["bias"] else 0)
        return {"bytes": forward + (4 * t * j + 4 * t * e if case["gradient"] else 0), "flops": 0}
    t, e, j, n, k = case["tokens"], case["experts"], case["top"], case["n"], case["k"]
    x = t * k * BYTES[case["type"]] * (j if case["per_slot"] else 1)
    out = t * n * BYTES[case["out"]] * (1 if case["weighted"] else j)
    return {"bytes": x + min(e, t * j) * _mx_bytes(n, k) + out + t * j * (8 if case["weighted"] else 4), "flops": 2 * t * j * n * k}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _exact_rounded(x):
    """Every value as its code stands for it, row block by row block: the nearest grid point times the block's scale."""
    rows, depth = x.shape
    out = torch.empty(rows, depth, dtype=torch.float64, device=x.device)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    middles = (grid[1:] + grid[:-1]) / 2
    powers = torch.tensor([2.0 ** e for e in range(-125, 128)], dtype=torch.float64, device=x.device)
    for first in range(0, rows, 1024):
        v = x[first:first + 1024].double()
        pad = -depth % BLOCK
        v = torch.nn.functional.pad(v, (0, pad)).unflatten(1, (-1, BLOCK))
        top = v.abs().max(dim=2, keepdim=True).values
        scale = powers[(torch.bucketize(top, powers, right=True) - 1).clamp(min=0)] / 4
        size = v.abs() / scale
        at = torch.bucketize(size, middles)
        tie = (at < 7) & (size == middles[at.clamp(max=6)]) & (at % 2 == 1)
        value = grid[at + tie.long()] * torch.sign(v) * scale
        out[first:first + 1024] = value.flatten(1)[:, :depth]
    return out


def _exact_decoded(codes, scales, depth):
    c = torch.stack([codes & 15, codes >> 4], dim=2).flatten(1)[:, :depth].long()
    e, f = (c & 7) >> 1, (c & 1).double()
    size = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2((e - 1).double()))
    block = torch.arange(depth, device=codes.device) // BLOCK
    return size * torch.where(c >= 8, -1.0, 1.0) * torch.exp2(scales.double() - 127)[:, block]


def _exact_state(case, seed):
    """The inputs of prepare() with the weights as exact values."""
    global _kept
    kept, _kept = _kept, lambda quantised, depth, groups: _exact_decoded(quantised[0], quantised[1], depth)
    try:
        return prepare(case, seed)
    finally:
        _kept = kept


def _exact_route(s):
    x = s["logits"].double().cpu().numpy()
    t, e, j = s["tokens"], s["experts"], s["top"]
    if s["score"] == "sigmoid":
        p = np.reciprocal(1.0 + np.exp(-x))
    else:
        p = np.exp(x - x.max(1)[:, None])
        p /= p.sum(1)[:, None]
    keys = p if s["bias_values"] is None else p + s["bias_values"].double().cpu().numpy()
    if s["groups"] > 1:
        size = e // s["groups"]
        by = keys.reshape(t, s["groups"], size)
        worth = -np.partition(-by, min(1, size - 1), axis=2)[:, :, :2].sum(2) if size > 1 else by[:, :, 0]
        rank = np.argsort(-worth, axis=1, kind="stable")
        shut = np.zeros((t, s["groups"]), bool)
        np.put_along_axis(shut, rank[:, s["top_groups"]:], True, axis=1)
        keys = np.where(np.repeat(shut, size, axis=1), -np.inf, keys)
    ids = np.argsort(-keys, axis=1, kind="stable")[:, :j]
    mine = np.take_along_axis(p, ids, 1)
    total = mine.sum(1)[:, None] if s["renormalise"] else 1.0
    out = {"weights": torch.from_numpy(s["scale"] * mine / total), "ids": None}
    if s["weights_grad"] is not None:
        up = s["scale"] * s["weights_grad"].double().cpu().numpy()
        if s["renormalise"]:
            up = (up - (up * mine / total).sum(1)[:, None]) / total
        grad = np.zeros((t, e))
        if s["score"] == "sigmoid":
            np.put_along_axis(grad, ids, up * mine * (1 - mine), axis=1)
        else:
            np.put_along_axis(grad, ids, up * mine, axis=1)
            grad -= p * (up * mine).sum(1)[:, None]
        out["logits_grad"] = torch.from_numpy(grad)
    return out


def exact(case, seed):
    s = _exact_state(case, seed)
    op = case["op"]
    if op == "quantise":
        return _exact_rounded(s["x"])
    if op == "product":
        a = _exact_decoded(s["x"][0], s["x"][1], case["k"]) if case["a"] == "mx" else _exact_rounded(s["x"])
        return a @ s["w"].T
    if op == "route":
        return _exact_route(s)
    t, j, n, k = case["tokens"], case["top"], case["n"], case["k"]
    x = s["x"] if case["per_slot"] else s["x"][:, None, :].expand(t, j, k)
    a = _exact_rounded(x.reshape(t * j, k))
    who = s["ids"].reshape(-1).long()
    y = torch.zeros(t * j, n, dtype=torch.float64, device=a.device)
    for e in range(case["experts"]):
        mine = torch.nonzero(who == e)[:, 0]
        y[mine] = a[mine] @ s["w"][e * n:(e + 1) * n].T
    y = y.view(t, j, n)
    return y if s["weights"] is None else torch.einsum("tj,tjn->tn", s["weights"].double(), y)
