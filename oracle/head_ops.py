"""Rotation and norm of attention heads, a paged cache and attention over it
in float64 numpy, from their formulas: the oracle of tl_rotary_*,
tl_cache_append and tl_paged_attention (include/templit_cuda.h).  No
counterpart in the reference, whose positions are a learned embedding and
whose generation keeps no cache (include/inference.h:45-97)."""
from __future__ import annotations

import numpy as np

PLAIN, LINEAR, NTK, PARTS, SMOOTH = range(5)


def frequencies(dim, base=10000.0, scaling=PLAIN, factor=1.0, original=0.0, low=1.0, high=32.0):
    """Radians a position for each pair, and the magnitude."""
    i = np.arange(dim // 2, dtype=np.float64)
    if scaling == NTK:
        return (base * factor ** (dim / (dim - 2.0))) ** (-2 * i / dim), 1.0
    f = base ** (-2 * i / dim)
    if scaling == PLAIN:
        return f, 1.0
    if scaling == LINEAR:
        return f / factor, 1.0
    if scaling == SMOOTH:
        stay = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0.0, 1.0)
        return stay * f + (1 - stay) * f / factor, 1.0

    def pair(turns):  # index whose frequency gives that many turns over the original length
        return dim * np.log(original / (2 * np.pi * turns)) / (2 * np.log(base))

    first, last = max(np.floor(pair(high)), 0.0), min(np.ceil(pair(low)), dim - 1.0)
    ramp = np.clip((i - first) / max(last - first, 1e-3), 0.0, 1.0)
    return (1 - ramp) * f + ramp * f / factor, 0.1 * np.log(factor) + 1.0


def _pairs(rotary, interleaved):
    i = np.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def turn(x, positions, radians, interleaved=False, magnitude=1.0, back=False):
    """x [..., H, D] at positions [...]; `back` applies the transpose."""
    x = np.asarray(x, np.float64)
    rotary = 2 * len(radians)
    a, b = _pairs(rotary, interleaved)
    angle = np.asarray(positions, np.float64)[..., None, None] * np.asarray(radians)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if back else 1)
    out = x.copy()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def norm(x, weight=None, eps=1e-6):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * weight


def heads(x, positions, radians, interleaved=False, magnitude=1.0, normed=False, weight=None, eps=1e-6):
    y = norm(x, weight, eps) if normed else x
    return turn(y, positions, radians, interleaved, magnitude)


def heads_gradient(x, d_out, positions, radians, interleaved=False, magnitude=1.0, normed=False, weight=None,
                   eps=1e-6):
    """(dx, dweight or None)."""
    g = turn(d_out, positions, radians, interleaved, magnitude, back=True)
    if not normed:
        return g, None
    x = np.asarray(x, np.float64)
    rms = np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = x / rms
    dw = (g * y).reshape(-1, x.shape[-1]).sum(0)
    if weight is not None:
        g = g * weight
    return (g - y * (g * y).mean(-1, keepdims=True)) / rms, dw


def attention(q, k, v, scale, causal=True, window=0):
    """q [N, Hq, D] are the last N positions of k, v [L, H, D].  Returns out,
    lse and A, the same sum over |v| (what an error of the probabilities is
    relative to).  What a row does not see is not touched."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    n, hq, d = q.shape
    length, h = k.shape[:2]
    out, lse, size = np.zeros((n, hq, d)), np.full((n, hq), -np.inf), np.zeros((n, hq, d))
    for i in range(n):
        p = length - n + i
        to = min(max(p + 1, 0), length) if causal else length
        a = max(p + 1 - window, 0) if window else 0
        if a >= to:
            continue
        for g in range(hq):
            with np.errstate(invalid="ignore", over="ignore"):
                x = (k[a:to, g // (hq // h)] @ q[i, g]) * scale
                m = x.max()
                if m == -np.inf:
                    continue
                e = np.exp(x - m)
                keep = x > -np.inf
                val = v[a:to, g // (hq // h)][keep]
                out[i, g] = e[keep] @ val / e.sum()
                size[i, g] = e[keep] @ np.abs(val) / e.sum()
                lse[i, g] = m + np.log(e.sum())
    return out, lse, size
