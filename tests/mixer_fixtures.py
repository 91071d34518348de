"""Plain statements of the token mixers (include/rl_mixers.h) in float64, on the
CPU, and the rounding of their element types. Written from the formulas alone."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Half a unit in the last place, relative, and the smallest absolute half step.
HALF_ULP = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}


def rounding(want, dtype):
    """The largest distance from `want` to its rounding."""
    rel, least = HALF_ULP[dtype]
    return np.abs(want) * rel + least


def as64(t):
    return t.detach().cpu().double().numpy()


def frequencies(dims, base, scaling="none", factor=1.0, original=0, fast=32.0, slow=1.0):
    """(radians a position of each pair, magnitude)."""
    if scaling == "ntk":
        base = base * factor ** (dims / (dims - 2))
    f = np.array([base ** (-2.0 * i / dims) for i in range(dims // 2)])
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        def place(turns):
            return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(place(fast)), 0), min(math.ceil(place(slow)), dims - 1)
        ramp = np.clip((np.arange(dims // 2) - low) / max(high - low, 0.001), 0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1
    return f, 1.0


def turn(x, positions, radians, magnitude, layout, sign=1.0):
    """x [rows][heads][dim] f64 with its first pairs turned."""
    y, n = x.copy(), len(radians)
    i = np.arange(n)
    a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    # Reduced before the cosine: exact for the integers and f64 radians used here to 1e-10.
    angle = np.asarray(positions, np.float64)[:, None] * radians
    c, s = magnitude * np.cos(angle)[:, None], sign * magnitude * np.sin(angle)[:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def encode(x, fmt):
    """What a cache of a format holds for f32 vectors, as f64 values: the step and
    the quotient are f32 by definition."""
    x = np.asarray(x, np.float32)
    if fmt in TYPES:
        return as64(torch.from_numpy(x.copy()).to(TYPES[fmt]))
    with np.errstate(all="ignore"):
        top = np.float32(127 if fmt == "i8" else 448)
        most = np.abs(x).max(-1, keepdims=True)
        step = (most / top).astype(np.float32)
        y = np.where(step > 0, (x / np.where(step > 0, step, 1)).astype(np.float32), np.float32(0))
        y = np.clip(y, -top, top)
        codes = np.rint(y) if fmt == "i8" else as64(torch.from_numpy(y.copy()).to(torch.float8_e4m3fn).float())
        out = (codes.astype(np.float32) * step).astype(np.float64)
    bad = ~np.isfinite(x).all(-1)
    out[bad] = np.nan
    return out


def attention(q, keys, values, scale, length, window=0):
    """One sequence: q [rows][q_heads][dim] its newest rows; keys, values
    [length][kv_heads][dim]. Returns out, lse, and per (row, head) the weighted sum
    of |values| and the largest sum of |q k|, which the error bounds need."""
    n, qh, dim = q.shape
    kv = keys.shape[1]
    out, lse = np.zeros((n, qh, dim)), np.full((n, qh), -np.inf)
    mass, size = np.zeros((n, qh, dim)), np.zeros((n, qh))
    for i in range(n):
        end = length - n + i + 1
        begin = max(0, end - window) if window else 0
        if end <= begin:
            continue
        for h in range(qh):
            k, v = keys[begin:end, h // (qh // kv)], values[begin:end, h // (qh // kv)]
            x = scale * (k @ q[i, h])
            top = x.max()
            p = np.exp(x - top)
            lse[i, h] = top + np.log(p.sum())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ v, p @ np.abs(v)
            size[i, h] = abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max()
    return out, lse, mass, size


def delta(q, k, v, g, beta, state, scale, eps):
    """One sequence, token after token: q, k [rows][key_heads][dk], v
    [rows][value_heads][dv], state [value_heads][dk][dv]; all f64."""
    state, share = state.copy(), v.shape[1] // q.shape[1]
    out = np.zeros_like(v)
    for t in range(q.shape[0]):
        for h in range(v.shape[1]):
            kt, qt = k[t, h // share], q[t, h // share]
            if eps >= 0:
                kt, qt = kt / np.sqrt(kt @ kt + eps), qt / np.sqrt(qt @ qt + eps)
            s = np.exp(g[t, h]) * state[h]
            u = beta[t, h] * (v[t, h] - kt @ s)
            state[h] = s + np.outer(kt, u)
            out[t, h] = scale * (qt @ state[h])
    return out, state
