"""The 4-bit cache without a GPU: what the binding refuses itself, and the oracle
(tests/kv4_oracle.py) against its formulas written out number by number."""
from __future__ import annotations

import math

import numpy as np
import pytest

import kv4_oracle as ko
import kv4_signs as ks


def test_a_freed_rope_is_refused(rc):
    """Its handle is NULL, which in the C call means keys as they are."""
    kv = object.__new__(rc.Kv4)
    kv.handle = None
    rope = rc.Rope(64)
    rope.free()
    with pytest.raises(rc.RabbitCudaError, match="freed") as e:
        kv.append_dev(0, rc.F32, 1, 1, 1, 1, rope=rope, d_positions=1)
    assert e.value.status == rc.ERR_ARGS


# -------------------------------------------------------------------- the oracle --
def test_rotate_is_the_formula():
    rng = np.random.default_rng(1)
    for hd, rot, layout, mag in [(8, 8, "interleaved", 1.0), (12, 8, "half", 1.25), (6, 2, "half", 0.5)]:
        x, pos = rng.standard_normal((3, 2, hd)), [0, 5, -70000]
        f = [10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)]
        got = ko.rotate(x, pos, ko.freqs(rot), layout, mag)
        for t, p in enumerate(pos):
            for h in range(2):
                y = list(x[t, h])
                for i in range(rot // 2):
                    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
                    c, s = math.cos(p * f[i]), math.sin(p * f[i])
                    y[a] = mag * (x[t, h, a] * c - x[t, h, b] * s)
                    y[b] = mag * (x[t, h, b] * c + x[t, h, a] * s)
                np.testing.assert_allclose(got[t, h], y, rtol=1e-12, atol=1e-12)


def test_hold_is_the_format():
    """Groups of 32 and a shorter last one; ties go to the even code, the scale is
    max / 7 in fp32, then in bf16."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 40)) * 10.0 ** rng.integers(-20, 20, (5, 1))
    x[1, :15] = np.arange(-7, 8) * 1.0
    x[1, 15:32] = 0.5
    x[2, 32:] = 0
    held, scale = ko.hold(x)
    for r in range(5):
        for c0 in (0, 32):
            g = x[r, c0:c0 + 32]
            s = np.float32(np.abs(g).max()) * np.float32(np.float32(1) / np.float32(7))
            bits = int(s.view(np.uint32))
            low, up = bits >> 16, bits & 0xFFFF
            low += up > 0x8000 or (up == 0x8000 and low & 1)
            s = float(np.uint32(low << 16).view(np.float32))
            for c in range(len(g)):
                code = round(g[c] / s) if s else 0  # Python rounds halves to even
                assert abs(code) <= 7
                assert held[r, c0 + c] == code * s and scale[r, c0 + c] == s
    assert (held[1, :15] == np.arange(-7, 8)).all() and (held[1, 15:32] == 0).all()
    odd = np.zeros((2, 64))
    odd[0, 3], odd[1, 40] = np.inf, np.nan
    held, _ = ko.hold(odd)
    assert np.isnan(held[0, :32]).all() and (held[0, 32:] == 0).all() and np.isnan(held[1, 32:]).all()


def test_attend_is_the_formula():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((3, 4)), rng.standard_normal((9, 4)), rng.standard_normal((9, 5))
    for window in (0, 1, 4):
        out, w = ko.attend(q, k, v, [8, 3, -1], window, 0.5)
        for r, p in enumerate([8, 3, -1]):
            seen = [j for j in range(9) if j <= p and (window == 0 or j > p - window)]
            e = {j: math.exp(0.5 * sum(q[r, c] * k[j, c] for c in range(4))) for j in seen}
            total = sum(e.values())
            for c in range(5):
                want = sum(e[j] * v[j, c] for j in seen) / total if seen else 0.0
                assert out[r, c] == pytest.approx(want, rel=1e-13, abs=1e-15)
            assert [w[r, j] > 0 for j in range(9)] == [j in seen for j in range(9)]


# ------------------------------------- what the structured attention tests can see --
@pytest.mark.parametrize("half", [2.0 ** -24, 2.0 ** -11, 2.0 ** -8])
@pytest.mark.parametrize("i", range(len(ks.CASES)))
def test_every_token_lost_doubled_or_misplaced_shows(i, half):
    """In each row's result, against the bar that the GPU's output has to keep: leaving a
    token out, or a granule of 16, counting it twice, or giving it its neighbour's value,
    puts some channel past it. (A row of one token has nothing to lose it against.)"""
    c = {"window": 0, **ks.CASES[i]}
    c.setdefault("qs", [1] * len(c["lens"]))
    q, seqs = ks.inputs(i, **c)
    rng, row = np.random.default_rng(7), 0
    for (k, v), n, nq in zip(seqs, c["lens"], c["qs"]):
        rows = range(nq) if nq < 8 else rng.choice(nq, 3, replace=False)
        for r in rows if n < 3000 else rows[:1]:
            p, h = n - nq + r, int(rng.integers(c["nh"]))
            kvh = h // (c["nh"] // c["nkv"])
            out, w, total = ks.attend(q[row + r, h], k[:, kvh], v[:, kvh], p, c["window"])
            at = np.nonzero(w)[0]
            if len(at) < 2:
                continue
            limit = ks.bar(out, half)
            wv = 7 * w[:, None] * v[:, kvh]
            worst = lambda sums, totals: (np.abs(sums / totals[:, None] - out) / limit).max(1).min()
            granule = at // 16 - at[0] // 16
            gw, gv = np.zeros(granule[-1] + 1), np.zeros((granule[-1] + 1, v.shape[2]))
            np.add.at(gw, granule, w[at])
            np.add.at(gv, granule, wv[at])
            for sign in (-1, 1):
                assert worst(out * total + sign * wv[at], total + sign * w[at]) > 1.5
                if len(gw) > 1:  # a granule that is all there is weighs the same twice
                    assert worst(out * total + sign * gv, total + sign * gw) > 2
            swap = 7 * w[at[1:], None] * (v[at[:-1], kvh].astype(int) - v[at[1:], kvh])
            if c["hd"] > 8:  # of 8 signs a neighbour's may be the same
                assert worst(out * total + swap, np.full(len(at) - 1, total)) > 1.5
        row += nq
