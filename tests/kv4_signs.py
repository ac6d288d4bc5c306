"""Attention inputs whose result tells each cached token from every other: keys and
values are random signs that the 4-bit cache holds exactly, so a token that is lost,
seen twice or taken from a wrong place moves every channel of a row.

Keys: channel `PICK` is 7 or -7, the others zero; a query has 1 or -1 there. With
scale ln(2) / 7 a score is 1 or -1 as a power of two: weights 2 and 1 / 2. Values
are 7 or -7 in every channel."""
from __future__ import annotations

import numpy as np

PICK = 5
SCALE = float(np.log(2.0) / 7)

CASES = [
    # decoding: one granule to many per CTA, ragged ends, shared heads, every width of row
    dict(nh=8, nkv=2, hd=128, page=16, lens=[255, 1, 16, 17, 3]),
    dict(nh=4, nkv=1, hd=64, page=64, lens=[9000, 1, 0, 700]),
    dict(nh=8, nkv=8, hd=40, page=48, lens=[2300]),
    dict(nh=20, nkv=1, hd=32, page=16, lens=[600, 47]),
    dict(nh=4, nkv=2, hd=256, page=16, lens=[500, 90]),
    dict(nh=3, nkv=3, hd=160, page=16, lens=[333]),
    dict(nh=2, nkv=1, hd=96, page=32, lens=[(53 * i) % 400 for i in range(200)]),
    dict(nh=8, nkv=4, hd=8, page=16, lens=[2000, 30], window=700),
    # drafted tokens
    dict(nh=8, nkv=2, hd=128, page=32, lens=[900, 40, 3], qs=[4, 5, 7]),
    dict(nh=6, nkv=1, hd=64, page=16, lens=[3000], qs=[4], window=1000),
    # chunks
    dict(nh=16, nkv=8, hd=64, page=16, lens=[700, 90, 70], qs=[90, 90, 70]),
    dict(nh=10, nkv=10, hd=128, page=48, lens=[511, 130], qs=[130, 130], window=100),
    dict(nh=8, nkv=8, hd=96, page=64, lens=[1000], qs=[600]),
    dict(nh=4, nkv=2, hd=256, page=16, lens=[150], qs=[150]),
]


def inputs(seed, *, nh, nkv, hd, lens, qs, **_):
    """(q [rows, nh], per sequence (k [n, nkv], v [n, nkv, hd])), all of 1 and -1."""
    rng = np.random.default_rng(seed)
    sign = lambda *shape: (2 * rng.integers(0, 2, shape) - 1).astype(np.int8)
    return sign(sum(qs), nh), [(sign(n, nkv), sign(n, nkv, hd)) for n in lens]


def attend(q, k, v, p, window):
    """A row's output at position p (below 0: it sees nothing), its weights, and their sum."""
    lo, hi = max(0, p - window + 1) if window else 0, max(0, p + 1)
    w = np.zeros(len(k))
    w[lo:hi] = 2.0 ** (q * k[lo:hi])
    total = w.sum()
    return (7 * (w @ v) / total if total else np.zeros(v.shape[1])), w, total


def bar(out, half):
    """What an output may be off, given half a step of its type. The weights' powers of
    two are off by 2^-21 at most, and rounded to fp16 they are exact; a sum of at
    most 600 of them in a thread by 600 2^-24; so out by 2^-14 of itself and
    2^-19 of the values."""
    return (2.0 ** -14 + 1.01 * half) * np.abs(out) + 7 * 2.0 ** -19
