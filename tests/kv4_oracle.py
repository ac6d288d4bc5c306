"""numpy float64 restatement of the rotary positions, the 4-bit key / value
groups and attention, from their formulas (include/rabbit_cuda.h)."""
from __future__ import annotations

import math

import numpy as np

# names of the C dtype codes -> half a step relative to the value
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def bf16(x):
    """float32 -> the nearest bf16 (ties to even) as float32; finite values."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32)


def freqs(rot, *, scaling="none", base=10000.0, factor=1.0, low=None, high=None, ctx=None):
    """Angle per position of each pair."""
    out = []
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "bands":
            n = ctx * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (n - low) / (high - low)))
            f = keep * f + (1 - keep) * f / factor
        elif scaling == "yarn":
            a = max(0, math.floor(rot * math.log(ctx / (high * 2 * math.pi)) / (2 * math.log(base))))
            b = min(rot - 1, math.ceil(rot * math.log(ctx / (low * 2 * math.pi)) / (2 * math.log(base))))
            t = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            f = f * (1 - t) + f / factor * t
        out.append(f)
    return np.array(out)


def pair_channels(rot, layout):
    i = np.arange(rot // 2)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def rotate(x, pos, freq, layout, mag=1.0):
    """x [T, heads, head_dim] float64, pos [T]."""
    y = np.array(x, np.float64)
    a, b = pair_channels(2 * len(freq), layout)
    ang = np.asarray(pos, np.float64)[:, None, None] * freq
    c, s = mag * np.cos(ang), mag * np.sin(ang)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def hold(x):
    """x [..., head_dim] float64 as the cache holds it (code * scale), and the
    scale of each channel; a group with an infinity or NaN is NaN."""
    out, scale = np.zeros_like(x), np.zeros_like(x)
    for c in range(0, x.shape[-1], 32):
        g = x[..., c:c + 32]
        with np.errstate(invalid="ignore", over="ignore"):
            top = np.abs(g).max(-1, keepdims=True).astype(np.float32)
            bad = ~np.isfinite(top)
            s = bf16(np.where(bad, 0, top) * (np.float32(1) / np.float32(7))).astype(np.float64)
            q = np.where(s > 0, np.rint(np.where(bad, 0, g) / np.where(s > 0, s, 1)), 0)
        out[..., c:c + 32] = np.where(bad, np.nan, q * s)
        scale[..., c:c + 32] = np.where(bad, np.nan, s)
    return out, scale


def attend(q, k, v, at, window, scale):
    """One head: q [R, d] at positions at [R], k / v [n, d]. Returns out [R, d]
    and the weights [R, n]; rows that see nothing are 0."""
    n = k.shape[0]
    out, w = np.zeros((len(q), v.shape[1])), np.zeros((len(q), n))
    for r, p in enumerate(at):
        lo = max(0, p - window + 1) if window else 0
        hi = min(p + 1, n)
        if hi <= lo:
            continue
        z = k[lo:hi] @ q[r] * scale
        e = np.exp(z - z.max())
        w[r, lo:hi] = e / e.sum()
        out[r] = w[r, lo:hi] @ v[lo:hi]
    return out, w
