"""Plain 64-bit implementations of the microscaled 4-bit and routing operators, for the tests."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
DECODE = np.concatenate([GRID, -GRID])


def encode_value(v):
    """Code of one value already over its scale: nearest grid point, ties to the even code, beyond 6 to 6."""
    size = abs(v)
    gap = np.abs(GRID - size)
    near = np.flatnonzero(gap == gap.min())
    code = near[0] if len(near) == 1 or near[0] % 2 == 0 else near[1]
    return int(code) + (8 if np.signbit(v) else 0)


def quantise(x):
    """(codes, scales) of a float matrix, by the definition."""
    x = np.asarray(x, dtype=np.float64)
    rows, depth = x.shape
    codes = np.zeros((rows, (depth + 1) // 2), np.uint8)
    scales = np.zeros((rows, (depth + 31) // 32), np.uint8)
    for r in range(rows):
        for b in range(scales.shape[1]):
            v = x[r, 32 * b:32 * b + 32]
            if not np.isfinite(v).all():
                scales[r, b] = 255
                continue
            top = np.abs(v).max()
            e = -127 if top == 0 else int(np.clip(np.frexp(top)[1] - 1 - 2, -127, 127))
            scales[r, b] = e + 127
            for i, value in enumerate(v):
                at = 32 * b + i
                codes[r, at // 2] |= encode_value(np.copysign(np.ldexp(abs(value), -e), value)) << (4 * (at % 2))
    return codes, scales


def dequantise(codes, scales, depth):
    both = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1)[:, :depth]
    scale = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int32) - 127))
    return DECODE[both] * np.repeat(scale, 32, axis=1)[:, :depth]


def product_bound(a, b, cells):
    """How far a product's cell may be from the exact one: a step of 64 values adds to an f32 accumulator without rounding up
    (off by at most one unit, 2^-23 of the largest partial sum, once inside the step and once on adding), bf16 cells add half a
    unit of theirs."""
    size = np.abs(a) @ np.abs(b).T
    steps = (a.shape[1] + 63) // 64
    bound = 2 * steps * 2.0 ** -23 * size
    return bound if cells == "f32" else bound + 2.0 ** -8 * (np.abs(a @ b.T) + bound)


def clean_logits(logits):
    x = np.asarray(logits, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    return np.minimum(x, np.finfo(np.float32).max)


def scores_of(logits, score):
    x = clean_logits(logits)
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "sigmoid":
            return np.where(x >= 0, 1 / (1 + np.exp(-np.maximum(x, 0))), np.exp(np.minimum(x, 0)) / (1 + np.exp(np.minimum(x, 0))))
        top = x.max(1, keepdims=True)
        e = np.where(np.isneginf(x), 0, np.exp(x - np.where(np.isneginf(top), 0, top)))
        total = e.sum(1, keepdims=True)
        return np.divide(e, total, out=np.zeros_like(e), where=total > 0)


def route(logits, top, bias=None, score="softmax", groups=1, top_groups=None, renormalise=True, scale=1.0):
    x = clean_logits(logits)
    s = scores_of(logits, score)
    tokens, experts = x.shape
    b = np.zeros(experts) if bias is None else np.minimum(np.where(np.isnan(bias), -np.inf, bias.astype(np.float64)), np.finfo(np.float32).max)
    keys = np.where(np.isneginf(x), -np.inf, (x if bias is None and groups == 1 else s + b))
    ids = np.full((tokens, top), -1, np.int32)
    weights = np.zeros((tokens, top))
    for t in range(tokens):
        k = keys[t].copy()
        if groups > 1:
            size = experts // groups
            worth = []
            for g in range(groups):
                best = sorted((v for v in k[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:2]
                worth.append(sum(best) if best else -np.inf)
            opened = sorted(range(groups), key=lambda g: (-worth[g], g))[:groups if top_groups is None else top_groups]
            for g in range(groups):
                if g not in opened:
                    k[g * size:(g + 1) * size] = -np.inf
        chosen = [e for e in sorted(range(experts), key=lambda e: (-k[e], e))[:top] if k[e] > -np.inf]
        ids[t, :len(chosen)] = chosen
        if not chosen:
            continue
        if renormalise:
            logs = np.array([-np.logaddexp(0, -x[t, e]) if score == "sigmoid" else x[t, e] for e in chosen])
            w = np.exp(logs - logs.max())
            w /= w.sum()
        else:
            w = s[t, chosen]
        weights[t, :len(chosen)] = scale * w
    return weights, ids


def route_gradient(weights_grad, ids, logits, score="softmax", renormalise=True, scale=1.0):
    x, s = clean_logits(logits), scores_of(logits, score)
    tokens, experts = x.shape
    out = np.zeros((tokens, experts))
    for t in range(tokens):
        slots = [(j, e) for j, e in enumerate(ids[t]) if 0 <= e < experts and x[t, e] > -np.inf]
        if not slots:
            continue
        g = np.array([float(weights_grad[t, j]) * scale for j, _ in slots])
        e = [e for _, e in slots]
        if renormalise:
            logs = np.array([-np.logaddexp(0, -x[t, i]) if score == "sigmoid" else x[t, i] for i in e])
            u = np.exp(logs - logs.max())
            u /= u.sum()
            d = u * (g - (g * u).sum())
            if score == "sigmoid":
                d = d * np.exp(-np.logaddexp(0, x[t, e]))
            np.add.at(out[t], e, d)
        elif score == "sigmoid":
            np.add.at(out[t], e, g * s[t, e] * np.exp(-np.logaddexp(0, x[t, e])))
        else:
            np.add.at(out[t], e, g * s[t, e])
            out[t] -= s[t] * (g * s[t, e]).sum()
    return out
