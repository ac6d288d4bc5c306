"""float64 restatements (numpy) of the 8-bit rows, the products, the expert routing
and the weighted sum, from their definitions."""
from __future__ import annotations

import numpy as np

BLOCK = 128


def e4m3_values() -> np.ndarray:
    """The value of each code 0..255 (NaN at 127 and 255)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c & 128, -v, v)


VALUES = e4m3_values()


def nearest_code(t: float) -> int:
    """e4m3 code of t >= 0, to nearest even, held at 448: by search over all codes."""
    held = VALUES[:127]
    d = np.abs(held - t)
    best = np.flatnonzero(d == d.min())
    return int(best[0] if len(best) == 1 else [b for b in best if b % 2 == 0][0])


def codes(x, s):
    """Codes of float64 x over the scale s (one number): of x / s, exactly: x and s are
    fp32 numbers, so the middles between codes times s are exact in 64 bits."""
    x = np.asarray(x, np.float64)
    if np.isnan(s):
        return np.full(x.shape, 127, np.uint8)
    if s == 0:
        return np.zeros(x.shape, np.uint8)
    held = VALUES[:127]
    mids = (held[1:] + held[:-1]) / 2 * float(s)
    a = np.abs(x)
    low = np.searchsorted(mids, a, "left")      # middles below |x|
    high = np.searchsorted(mids, a, "right")    # and at or below
    c = np.where(low == high, low, np.where(low % 2 == 0, low, high))  # a tie: to the even code
    return (c | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def quantise(x, block_rows=1):
    """(codes [R, C], scales) of x [R, C] (float64 holding the input type's values)."""
    R, C = x.shape
    s = np.zeros((-(-R // block_rows), -(-C // BLOCK)), np.float32)
    q = np.zeros((R, C), np.uint8)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = np.s_[i * block_rows:(i + 1) * block_rows, j * BLOCK:(j + 1) * BLOCK]
            b = x[at]
            s[i, j] = np.float32(np.abs(b).max() / 448.0) if np.isfinite(b).all() else np.nan
            q[at] = codes(b, s[i, j])
    return q, s


def dequantise(q, s, block_rows=1):
    R, C = q.shape
    s = s.astype(np.float64)
    return VALUES[q] * np.repeat(np.repeat(s, block_rows, 0)[:R], BLOCK, 1)[:, :C]


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def product(x, w):
    """x [R, K], w [G, N, K] (float64): (y, sums of |terms| of each matrix [G, R, N])."""
    parts = [x @ m.T for m in w]
    mags = np.stack([np.abs(x) @ np.abs(m).T for m in w])
    return (parts[0] if len(parts) == 1 else silu(parts[0]) * parts[1]), parts, mags


def product_bar(parts, mags, steps, half, tiny):
    """How far a computed product may be off (test_linear_gpu.py has the derivation)."""
    u = 2.0 ** -24
    e = 4 * u * (steps + 4) * mags
    if len(parts) == 1:
        y, err = parts[0], e[0]
    else:
        g, up = parts
        s = silu(g)
        y = s * up
        # |silu'| <= 1.1; exp (|g| u + 4 u of itself), 1 + exp (u) and the division (4 u); the
        # product of the two
        err = (1.1 * e[0] + (9 + np.abs(g)) * u * np.abs(s)) * (np.abs(up) + e[1]) + (np.abs(s) + 1.1 * e[0]) * e[1] + u * np.abs(y)
    return err + half * (np.abs(y) + err) + tiny


def route(scores, k, over_all):
    """ids and weights of scores [T, E] (float64)."""
    T, E = scores.shape
    ids, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        live = [e for e in range(E) if scores[t, e] > -np.inf]
        pick = sorted(live, key=lambda e: (-scores[t, e], e))[:k]
        if not pick:
            continue
        top = scores[t, pick[0]]
        part = lambda e: 1.0 if scores[t, e] == top else np.exp(scores[t, e] - top)  # noqa: E731
        total = sum(part(e) for e in (live if over_all else pick))
        for j, e in enumerate(pick):
            ids[t, j], w[t, j] = e, part(e) / total
    return ids, w


def order(ids, n_experts):
    """offsets, rows and place of ids [T, k]."""
    T, k = ids.shape
    flat = ids.reshape(-1)
    live = (flat >= 0) & (flat < n_experts)
    rows, place = np.full(T * k, -1, np.int32), np.full(T * k, -1, np.int32)
    offsets = np.zeros(n_experts + 1, np.int32)
    offsets[1:] = np.cumsum(np.bincount(flat[live], minlength=n_experts))
    pairs = np.flatnonzero(live)
    pairs = pairs[np.argsort(flat[pairs], kind="stable")]
    place[pairs] = np.arange(len(pairs))
    rows[:len(pairs)] = pairs // k
    return offsets, rows, place.reshape(T, k)


def combine(y, place, weights, base):
    """(sums, sums of |terms|) in float64."""
    out = np.zeros((place.shape[0], y.shape[1])) if base is None else base.copy()
    mag = np.abs(out)
    for t in range(place.shape[0]):
        for j, p in enumerate(place[t]):
            if 0 <= p < y.shape[0]:
                out[t] += weights[t, j] * y[p]
                mag[t] += np.abs(weights[t, j] * y[p])
    return out, mag
