"""The 8-bit operators and the routing in 64 bits, straight from their definitions (numpy)."""
import numpy as np
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {n: torch.finfo(t).eps / 2 for n, t in DT.items()}   # of a rounding, relative to the value
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # the same below the normal numbers, absolute
F32_STEP = 2.0 ** -24


def f64(t):
    return t.detach().cpu().double().numpy()


def quantise(x):
    x = f64(x)
    bad = ~np.isfinite(x).all(1)
    a = np.abs(np.where(np.isfinite(x), x, 0)).max(1)
    a[bad] = 0
    q = np.rint(np.divide(x * 127.0, a[:, None], out=np.zeros_like(x), where=(a[:, None] > 0)))
    s = (a / 127.0).astype(np.float32)
    s[bad] = np.nan
    return q.astype(np.int8), s


def prelu(y, alpha):
    return np.where(y > 0, y, y * alpha)


def product(q, scale, w, w_scale, alpha):
    acc = q.astype(np.float64) @ w.astype(np.float64).T
    return prelu(acc * scale.astype(np.float64)[:, None] * w_scale.astype(np.float64), alpha)


def product_error(y, dtype):
    """int32 -> fp32, two scales and the slope: four roundings to 24 bits (their second-order terms covered by the 1 %), then the
    rounding to the result's type."""
    return np.abs(y) * (4.04 * F32_STEP + (0 if dtype == "f32" else 1.01 * HALF_STEP[dtype])) + LEAST[dtype] + 4 * 2.0 ** -149


def route(logits, bias, r):
    """experts, weights (float64) of every token; r: the fields of a Route."""
    x = f64(logits)
    T, E = x.shape
    size = E // r.groups
    big = np.finfo(np.float32).max
    experts, weights = np.full((T, r.top_k), -1, np.int32), np.zeros((T, r.top_k))
    b = None if bias is None else f64(bias)
    for t in range(T):
        barred = np.isnan(x[t]) | np.isneginf(x[t])
        v = np.minimum(np.where(barred, 0, x[t]), big)
        p = np.zeros(E)
        if not barred.all():
            if r.score == 1:
                with np.errstate(over="ignore"):
                    p[~barred] = 1 / (1 + np.exp(-v[~barred]))
            else:
                ex = np.exp(v[~barred] - v[~barred].max())
                p[~barred] = ex / ex.sum()
        if b is not None:
            barred = barred | np.isnan(b) | np.isneginf(b)
            worth = p + np.minimum(np.where(barred, 0, b), big)
            key = worth
        else:
            worth, key = p, v
        there = [e for e in range(E) if not barred[e]]
        if r.top_groups < r.groups:
            groups = []
            for g in range(r.groups):
                inside = [e for e in there if e // size == g]
                if inside:
                    groups.append((-(max(key[e] for e in inside) if r.group_top == 1 else sum(sorted(worth[e] for e in inside)[-2:])), g))
            kept = {g for _, g in sorted(groups)[:r.top_groups]}
            there = [e for e in there if e // size in kept]
        chosen = sorted(there, key=lambda e: (-key[e], e))[:r.top_k]
        s = p[chosen] if chosen else np.zeros(0)
        experts[t, :len(chosen)] = chosen
        weights[t, :len(chosen)] = np.float64(np.float32(r.scale)) * (s / (s.sum() + 1e-20) if r.renormalise else s)
    return experts, weights


def plan(experts, E):
    T, k = experts.shape
    offsets, rows, slots, at = np.zeros(E + 1, np.int32), np.full(T * k, -1, np.int32), np.full((T, k), -1, np.int32), 0
    for e in range(E):
        for t, j in np.argwhere(experts == e):
            rows[at], slots[t, j] = t, at
            at += 1
        offsets[e + 1] = at
    return offsets, rows, slots
