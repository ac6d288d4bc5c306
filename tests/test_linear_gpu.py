"""GPU: 8-bit rows, products with e4m3 and 16-bit weights, expert batches, against
float64 numpy (tests/linear_oracle.py).

Tolerances, with u = 2^-24 (half a step of fp32) and h half a step of the output type:
 * quantise, route's ids, offsets, rows and places: equal.
 * a product's sum over K is a chain of `steps` tensor-core steps of 32 bytes (32 or 16
   terms) and, in e4m3, one fp32 fma a block: with each addition held to a whole fp32 step (2 u)
   of the terms' magnitudes so far, aligned and then added, it is off by at most
   4 u steps sum |x w|; the scales' product and the cluster's sums add 4 more steps. Gated,
   the errors go through silu(g) up to first order (product_bar in linear_oracle.py). Then
   the output's rounding, h |y| and half the smallest subnormal.
 * combine: k products and sums, each within u of the terms' magnitudes: (k + 2) u sum |w y|.
 * route's weights: the difference (u |s|), expf (2 u), the sum over E (log2 E + V additions,
   taken as 40) and the division: (48 + |s - top|) u.
"""
from __future__ import annotations

import numpy as np
import pytest

import linear_oracle as lo

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


@pytest.fixture(scope="module")
def torch():
    import torch

    torch.zeros(1, device="cuda")
    return torch


def types(torch, rc, name):
    return {"f32": (torch.float32, rc.F32), "f16": (torch.float16, rc.F16),
            "bf16": (torch.bfloat16, rc.BF16), "e4m3": (torch.uint8, rc.E4M3)}[name]


def f64(t):
    return t.double().cpu().numpy()


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# --------------------------------------------------------------- quantise --
def quantise(torch, rc, x, name, block_rows=1, rows=None, gap=(0, 0), offset=(0, 0)):
    """(codes, scales, q as it lies, its canary) of float64 x through the library."""
    dt, code = types(torch, rc, name)
    R, C = (len(rows) if rows is not None else x.shape[0]), x.shape[1]
    xd = torch.zeros(x.shape[0] * (C + gap[0]) + offset[0] + 8, dtype=dt, device="cuda")
    xv = xd[offset[0]:offset[0] + x.shape[0] * (C + gap[0])].view(x.shape[0], C + gap[0])
    xv[:, :C] = dev(torch, x).to(dt)
    qd = torch.full((R * (C + gap[1]) + offset[1] + 8,), 0x55, dtype=torch.uint8, device="cuda")
    qv = qd[offset[1]:offset[1] + R * (C + gap[1])].view(R, C + gap[1])
    s = torch.full((-(-R // block_rows), -(-C // 128)), 7.0, device="cuda")
    rd = dev(torch, np.asarray(rows, np.int32)) if rows is not None else None
    rc.f8_quantise_dev(code, xv.data_ptr(), qv.data_ptr(), s.data_ptr(), R, C, block_rows=block_rows,
                       d_rows=rd.data_ptr() if rows is not None else 0, x_rows=x.shape[0],
                       x_stride=C + gap[0], q_stride=C + gap[1], stream=stream(torch))
    torch.cuda.synchronize()
    assert (qv[:, C:] == 0x55).all() and (qd[:offset[1]] == 0x55).all() and (qd[-8:] == 0x55).all()
    return qv[:, :C].cpu().numpy(), s.cpu().numpy(), f64(xv[:, :C])


def same_codes(got, want):
    nan = (want[0] & 127) == 127
    np.testing.assert_array_equal((got[0] & 127) == 127, nan)
    np.testing.assert_array_equal(got[0][~nan], want[0][~nan])
    np.testing.assert_array_equal(got[1], want[1])


@pytest.mark.parametrize("name,R,C,block,gap,offset", [
    ("f32", 1, 1, 1, (0, 0), (0, 0)), ("f32", 1, 2048, 1, (0, 0), (0, 0)),
    ("bf16", 37, 300, 1, (0, 0), (0, 0)), ("f16", 5, 128, 1, (8, 8), (0, 0)),
    ("bf16", 9, 257, 1, (7, 3), (1, 1)), ("f32", 300, 129, 1, (3, 0), (1, 3)),
    ("f16", 1000, 640, 1, (0, 0), (8, 8)), ("bf16", 2100, 136, 1, (0, 0), (0, 0)),
    ("f32", 128, 128, 128, (0, 0), (0, 0)), ("bf16", 129, 257, 128, (0, 0), (0, 0)),
    ("f16", 1, 1000, 128, (0, 0), (0, 0)), ("f32", 300, 513, 128, (3, 5), (2, 1)),
    ("bf16", 255, 384, 128, (8, 8), (8, 8)),
])
def test_quantise(torch, rc, name, R, C, block, gap, offset):
    rng = np.random.default_rng(R * C)
    x = rng.standard_normal((R, C)) * np.exp(rng.uniform(-6, 6, (R, 1)))
    q, s, held = quantise(torch, rc, x, name, block, None, gap, offset)
    same_codes((q, s), lo.quantise(held, block))


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_quantise_ties_and_edges(torch, rc, name, block):
    """Quotients at and next to every middle between codes, tiny and huge scales, zeros,
    and blocks that hold an infinity or a NaN."""
    mids = (lo.VALUES[1:127] + lo.VALUES[:126]) / 2
    rows = []
    for scale in (1.0, 2.0 ** -20, 3.0, 0.7) + ((2.0 ** -140, 2.0 ** -130, 1e30, 2.0 ** -146) if name == "f32" else ()):
        for near in (0.0, 2.0 ** -23, -2.0 ** -23, 2.0 ** -8):
            b = np.concatenate([[448.0], mids * (1 + near), [0.0]]) * scale
            b[1::2] *= -1
            rows.append(np.clip(b, -60000, 60000) if name == "f16" else b)
    top = {"f32": 3.4028234e38, "f16": 65504.0, "bf16": 3.38e38}[name]
    rows += [np.zeros(128), np.full(128, -0.0), np.full(128, top), np.eye(1, 128)[0] * 2.0 ** -149]
    bad = np.linspace(-3, 3, 128)
    for v in (np.inf, -np.inf, np.nan):
        rows.append(np.where(np.arange(128) == 77, v, bad))
    x = np.stack(rows)
    if block == 128:  # each row a block: the other rows of it zero
        x = np.stack([np.eye(1, 128)[0][:, None] * 0 + r * (np.arange(128) == 5)[:, None] if np.isfinite(r).all()
                      else np.where((np.arange(128) == 5)[:, None], r, 0.0) for r in x]).reshape(-1, 128)
    q, s, held = quantise(torch, rc, x, name, block)
    same_codes((q, s), lo.quantise(held, block))


def test_quantise_many_values_exactly(torch, rc):
    """Half a million bf16 values: near ties are common among 8-bit mantissas."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1024, 512))
    q, s, held = quantise(torch, rc, x, "bf16")
    same_codes((q, s), lo.quantise(held))


def test_quantise_through_a_list(torch, rc):
    rng = np.random.default_rng(6)
    x, rows = rng.standard_normal((50, 200)), rng.integers(0, 50, 333)
    rows[[3, 100, 332]] = -1, 50, 2 ** 31 - 1
    q, s, held = quantise(torch, rc, x, "f16", rows=rows)
    ok = (rows >= 0) & (rows < 50)
    want = lo.quantise(held[np.where(ok, rows, 0)])
    same_codes((q[ok], s[ok]), (want[0][ok], want[1][ok]))
    assert (q[~ok] == 0x55).all() and (s[~ok] == 7.0).all()


# --------------------------------------------------------------- products --
class Case:
    """Operands in device memory, with garbage wherever nothing may be read from."""

    def __init__(self, torch, rc, name, R, N, K, gated=False, experts=1, seed=0, gap=0, xgap=0):
        rng = np.random.default_rng(seed + R * N + K)
        self.torch, self.rc, self.name = torch, rc, name
        self.R, self.N, self.K, self.E, self.G = R, N, K, experts, 2 if gated else 1
        dt, self.code = types(torch, rc, name)
        unit = 16 if name == "e4m3" else 8
        ws, xs = -(-K // unit) * unit + gap * unit, -(-K // unit) * unit + xgap * unit
        x = rng.standard_normal((R, K)) * np.exp(rng.uniform(-2, 2, (R, 1)))
        w = rng.standard_normal((experts, self.G, N, K)) / np.sqrt(K)
        nb = -(-K // 128)
        if name == "e4m3":
            qx, sx = lo.quantise(x)
            qw = np.zeros(w.shape, np.uint8)
            sw = np.zeros((experts, self.G, -(-N // 128), nb), np.float32)
            for e in range(experts):
                for g in range(self.G):
                    qw[e, g], sw[e, g] = lo.quantise(w[e, g], 128)
            self.x = lo.dequantise(qx, sx)
            self.w = np.stack([[lo.dequantise(qw[e, g], sw[e, g], 128) for g in range(self.G)]
                               for e in range(experts)])
            bad = 0x7F
            self.sx, self.sw = dev(torch, sx), dev(torch, sw)
            dx, dw = dev(torch, qx), dev(torch, qw)
        else:
            dx, dw = dev(torch, x).to(dt), dev(torch, w).to(dt)
            self.x, self.w = f64(dx), f64(dw)
            bad = float("nan")
        self.xd = torch.full((R + 40, xs), bad, dtype=dt, device="cuda")
        self.xd[:R, :K] = dx
        self.wd = torch.full((experts, self.G, N, ws), bad, dtype=dt, device="cuda")
        self.wd[..., :K] = dw
        self.steps = K / (32 if name == "e4m3" else 16) + nb
        self.lin = rc.Linear(self.code, N, K, self.wd.data_ptr(), n_experts=experts, gated=gated, w_stride=ws,
                             d_scale=self.sw.data_ptr() if name == "e4m3" else 0)
        self.kw = dict(x_stride=xs, **(dict(d_x_scale=self.sx.data_ptr()) if name == "e4m3" else {}))

    def out(self, name, rows, gap=0):
        dt, code = types(self.torch, self.rc, name)
        y = self.torch.full((rows + 3, self.N + gap), -777.0, dtype=dt, device="cuda")
        return y, code

    def bar(self, x, e, out):
        y, parts, mags = lo.product(x, self.w[e])
        return y, lo.product_bar(parts, mags, self.steps, HALF[out], TINY[out])

    def close(self, got, x, e, out):
        y, bar = self.bar(x, e, out)
        off = np.abs(got - y)
        assert (off <= bar).all(), f"off by {np.nanmax(off / bar):.3g} bars at {np.unravel_index(np.argmax(off / bar), off.shape)}"


DENSE = [
    # type, rows, n_out, n_in, gated, out, gaps of w, x and y
    ("f16", 1, 1, 1, False, "f32", 0, 0, 0), ("e4m3", 1, 1, 1, False, "f32", 0, 0, 0),
    ("bf16", 1, 128, 64, False, "f32", 0, 0, 0), ("e4m3", 16, 128, 128, False, "f32", 0, 0, 0),
    ("f16", 17, 129, 200, False, "f16", 1, 2, 3), ("e4m3", 17, 129, 200, False, "bf16", 2, 1, 1),
    ("bf16", 300, 257, 136, False, "bf16", 0, 0, 0), ("e4m3", 300, 257, 136, False, "f16", 0, 0, 5),
    ("e4m3", 257, 384, 1000, False, "f32", 0, 1, 0), ("f16", 33, 100, 1000, False, "f32", 0, 0, 0),
    ("bf16", 5, 130, 2000, False, "f32", 0, 0, 0), ("e4m3", 5, 130, 2000, False, "f32", 0, 0, 0),
    ("e4m3", 40, 64, 4100, False, "f32", 0, 0, 0), ("f16", 100, 64, 4100, False, "f16", 0, 0, 0),
    ("e4m3", 1, 200, 300, True, "f32", 0, 0, 0), ("bf16", 31, 129, 500, True, "bf16", 1, 1, 1),
    ("e4m3", 129, 257, 640, True, "bf16", 0, 0, 0), ("f16", 300, 130, 264, True, "f16", 0, 0, 0),
    ("e4m3", 70, 100, 3000, True, "f32", 0, 0, 0), ("bf16", 2, 70, 3000, True, "f32", 0, 0, 0),
    ("e4m3", 700, 2000, 384, False, "bf16", 0, 0, 0), ("f16", 520, 2100, 128, True, "f32", 0, 0, 0),
]


@pytest.mark.parametrize("name,R,N,K,gated,out,wg,xg,yg", DENSE)
def test_linear(torch, rc, name, R, N, K, gated, out, wg, xg, yg):
    c = Case(torch, rc, name, R, N, K, gated, gap=wg, xgap=xg)
    y, code = c.out(out, R, yg)
    c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), R, y_stride=N + yg, stream=stream(torch), **c.kw)
    c.lin.check(stream(torch))
    got = f64(y)
    c.close(got[:R, :N], c.x, 0, out)
    assert (got[R:] == got[-1, -1]).all() and (got[:, N:] == got[-1, -1]).all()


SIZES = {  # rows of each expert
    "even": [3, 3, 3, 3], "one": [40], "empty": [0, 0, 0], "holes": [0, 5, 0, 0, 130, 1, 0],
    "large": [300, 0, 260, 129, 1, 384], "ragged": [1, 17, 0, 300, 33, 16, 2, 129], "last": [0, 0, 0, 7], "many": [1, 0, 2] * 341 + [5],
}


@pytest.mark.parametrize("name,N,K,gated,out", [
    ("e4m3", 130, 300, False, "bf16"), ("e4m3", 129, 260, True, "f32"), ("f16", 64, 136, True, "f16"),
    ("bf16", 257, 72, False, "f32"),
])
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("sizes", SIZES)
def test_grouped(torch, rc, sizes, listed, name, N, K, gated, out):
    sizes = SIZES[sizes]
    if len(sizes) > 100:
        N, K = 40, 64
    first, spare = (2, 5) if len(sizes) < 100 else (0, 0)  # rows before the first expert's and after the last
    R = first + sum(sizes) + spare
    T = 23 if listed else R
    c = Case(torch, rc, name, T, N, K, gated, experts=len(sizes))
    rng = np.random.default_rng(len(sizes) + R)
    rows = rng.integers(0, T, R) if listed else np.arange(R)
    ends = first + np.concatenate([[0], np.cumsum(sizes)])
    # no row of its own: what lies outside of the experts' rows is not looked at
    rows = np.where((np.arange(R) < ends[0]) | (np.arange(R) >= ends[-1]), -5, rows)
    off, rd = dev(torch, ends.astype(np.int32)), dev(torch, rows.astype(np.int32))
    y, code = c.out(out, R)
    c.lin.grouped_dev(c.xd.data_ptr(), T, off.data_ptr(), code, y.data_ptr(), R,
                      d_rows=rd.data_ptr() if listed else 0, stream=stream(torch), **c.kw)
    c.lin.check(stream(torch))
    got = f64(y)
    for e in range(len(sizes)):
        at = np.arange(ends[e], ends[e + 1])
        if len(at):
            c.close(got[at], c.x[rows[at]], e, out)
    left = np.ones(len(got), bool)
    left[ends[0]:ends[-1]] = False
    assert (got[left] == got[-1, -1]).all()


@pytest.mark.parametrize("name", ["e4m3", "bf16"])
def test_grouped_reports_what_is_out_of_range(torch, rc, name):
    c = Case(torch, rc, name, 20, 100, 128, experts=3)
    y, code = c.out("f32", 12)
    rows = np.array([0, 5, 20, 7, -1, 19, 3, 3, 2 ** 31 - 1, -2 ** 31, 1, 2], np.int32)
    off, rd = dev(torch, np.array([0, 4, 9, 11], np.int32)), dev(torch, rows)
    call = lambda o, r: c.lin.grouped_dev(c.xd.data_ptr(), 20, o.data_ptr(), code, y.data_ptr(), 12,  # noqa: E731
                                          d_rows=r.data_ptr(), stream=stream(torch), **c.kw)
    call(off, rd)
    with pytest.raises(rc.RabbitCudaError, match="rows") as e:
        c.lin.check(stream(torch))
    assert e.value.status == rc.ERR_ARGS
    c.lin.check(stream(torch))  # reported once
    got = f64(y)
    for i, r in enumerate(rows):
        if i < 11 and 0 <= r < 20:
            c.close(got[i:i + 1], c.x[r:r + 1], 0 if i < 4 else 1 if i < 9 else 2, "f32")
        else:
            assert (got[i] == -777).all()
    y.fill_(-777)
    for ends in ([0, 4, 3, 9], [-1, 4, 5, 9], [0, 4, 9, 13], [5, 4, 3, 2]):
        bad = dev(torch, np.array(ends, np.int32))
        call(bad, rd)
        with pytest.raises(rc.RabbitCudaError, match="offsets"):
            c.lin.check(stream(torch))
        assert (y == -777).all()


@pytest.mark.parametrize("name", ["e4m3", "f16"])
@pytest.mark.parametrize("gated", [False, True])
def test_what_is_not_finite_stays_in_its_row(torch, rc, name, gated):
    """A NaN in one token's row or in one output's weights reaches no other."""
    c = Case(torch, rc, name, 50, 200, 256, gated)
    y, code = c.out("f32", 50)
    run = lambda: c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), 50, stream=stream(torch), **c.kw)  # noqa: E731
    run()
    clean = y.clone()
    nan = 0x7F if name == "e4m3" else float("nan")
    c.xd[7, 100] = nan
    c.wd[0, 0, 130, 5] = nan
    run()
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[7], bad[:50, 130] = True, True
    bad[50:] = False
    assert y[bad].isnan().all() and (y[~bad] == clean[~bad]).all()
    if name == "e4m3":
        c.sx[9, 1] = float("inf")
        c.sw[0, 0, 1, 0] = float("nan")
        run()
        bad[9], bad[:50, 128:] = True, True
        assert not y[9].isfinite().all() and y[:50, 128:].isnan().all() and (y[~bad] == clean[~bad]).all()


def test_same_bits_each_time(torch, rc):
    for name, R, N, K, gated in [("e4m3", 3, 130, 4000, False), ("bf16", 300, 700, 500, True), ("f16", 1, 64, 4096, True)]:
        c = Case(torch, rc, name, R, N, K, gated)
        outs = []
        for _ in range(20):
            y, code = c.out("f32", R)
            c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), R, stream=stream(torch), **c.kw)
            outs.append(y)
        assert all((o == outs[0]).all() for o in outs)


@pytest.mark.parametrize("name,R,N,K,out", [
    ("bf16", 3, 128, 64, "bf16"), ("e4m3", 5, 256, 2048, "f32"), ("f16", 2, 64, 2048, "f32"),
    ("bf16", 700, 3000, 256, "bf16"), ("f16", 700, 3000, 512, "f32"), ("e4m3", 700, 3000, 512, "bf16"),
])
@pytest.mark.parametrize("listed", [False, True])
def test_waits_that_run_out(torch, rc, name, R, N, K, out, listed):
    """Copies that end early end the call with a status, and the next call is whole."""
    c = Case(torch, rc, name, R, N, K)
    off, rows = dev(torch, np.array([0, R], np.int32)), dev(torch, np.arange(R, dtype=np.int32)[::-1])
    y, code = c.out(out, R)
    run = lambda: c.lin.grouped_dev(c.xd.data_ptr(), R, off.data_ptr(), code, y.data_ptr(), R,  # noqa: E731
                                    d_rows=rows.data_ptr() if listed else 0, stream=stream(torch), **c.kw)
    rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(20))
    try:
        rc.check(rc.lib().rabbit_cuda_linear_debug_withhold(c.lin.handle))
        run()
        with pytest.raises(rc.RabbitCudaError, match="wait ran out") as e:
            c.lin.check(stream(torch))
        assert e.value.status == rc.ERR_TIMEOUT
    finally:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(2000))
    run()
    c.lin.check(stream(torch))
    at = np.arange(0, R, max(1, R // 40))
    c.close(f64(y)[at], c.x[::-1][at] if listed else c.x[at], 0, out)


@pytest.mark.parametrize("name,R,N,K,gated,out", [
    ("bf16", 20, 40, 20000, False, "bf16"), ("f16", 300, 300, 17000, True, "f16"), ("e4m3", 130, 140, 20001, False, "f16"),
])
def test_long_sums(torch, rc, name, R, N, K, gated, out):
    """More channels than a 16-bit output's sum stays in tensor memory for."""
    c = Case(torch, rc, name, R, N, K, gated)
    y, code = c.out(out, R)
    c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), R, stream=stream(torch), **c.kw)
    c.lin.check(stream(torch))
    c.close(f64(y)[:R], c.x, 0, out)


@pytest.mark.parametrize("name,K,out", [("e4m3", 140, "bf16"), ("e4m3", 500, "f32"), ("f16", 100, "f16"), ("bf16", 300, "f32")])
@pytest.mark.parametrize("N,gap,shift", [(301, 0, 0), (302, 0, 0), (301, 3, 1), (304, 0, 1), (304, 4, 2), (303, 5, 0)])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_of_y_that_do_not_lie_on_16_bytes(torch, rc, name, K, out, N, gap, shift, gated):
    for R in (3, 600):  # one CTA a tile, pairs
        c = Case(torch, rc, name, R, N, K, gated)
        dt, code = types(torch, rc, out)
        flat = torch.full(((R + 1) * (N + gap) + shift,), -777.0, dtype=dt, device="cuda")
        y = flat[shift:].view(R + 1, N + gap)
        c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), R, y_stride=N + gap, stream=stream(torch), **c.kw)
        c.lin.check(stream(torch))
        got = f64(y)
        c.close(got[:R, :N], c.x, 0, out)
        assert (got[R:] == got[-1, -1]).all() and (got[:, N:] == got[-1, -1]).all() and (flat[:shift] == flat[-1]).all()


def test_elements_past_32_bits(torch, rc):
    """Rows of x and y so far apart that their last elements lie past 2^32."""
    R, N, K = 140, 40, 64
    c = Case(torch, rc, "bf16", R, N, K)
    wide = 1 << 25
    x = torch.empty(R * wide, dtype=torch.bfloat16, device="cuda").view(R, wide)
    x[:, :K] = c.xd[:R, :K]
    y = torch.empty(R * wide, dtype=torch.bfloat16, device="cuda").view(R, wide)
    c.lin.apply_dev(x.data_ptr(), rc.BF16, y.data_ptr(), R, x_stride=wide, y_stride=wide, stream=stream(torch))
    c.lin.check(stream(torch))
    c.close(f64(y[:, :N]), c.x, 0, "bf16")


def test_arguments_are_refused(torch, rc):
    c = Case(torch, rc, "e4m3", 8, 64, 128, experts=2)
    so, h, x, s, y = rc.lib(), c.lin.handle, c.xd.data_ptr(), c.sx.data_ptr(), c.out("f32", 8)[0].data_ptr()
    off = dev(torch, np.array([0, 4, 8], np.int32))
    o = off.data_ptr()
    assert so.rabbit_cuda_linear_dev(h, x, 0, s, 0, 0, y, 0, 8, None) == rc.ERR_ARGS  # two experts
    good = [h, x, 0, 8, s, 0, None, o, 0, y, 0, 8, None]
    for i, v in [(1, None), (1, x + 8), (2, 112), (2, 130), (2, -128), (3, 7), (3, 0), (4, None), (4, s + 2),
                 (5, -1), (6, o + 1), (7, None), (7, o + 2), (8, 3), (8, -1), (9, None), (9, y + 2),
                 (10, 63), (11, -1), (11, (1 << 30) + 1), (5, (1 << 30) + 1)]:
        args = list(good)
        args[i] = v
        assert so.rabbit_cuda_linear_grouped_dev(*args) == rc.ERR_ARGS, (i, v)
    assert so.rabbit_cuda_linear_grouped_dev(*good) == rc.OK
    good[11] = 0
    assert so.rabbit_cuda_linear_grouped_dev(*good) == rc.OK
    c.lin.check(stream(torch))
    with pytest.raises(rc.RabbitCudaError):
        rc.Linear(rc.F16, 64, 64, c.wd.data_ptr(), device=99)


# ------------------------------------------------------------------ route --
def route(torch, rc, scores, k, over_all=False, ids=None, stride=0):
    T, E = (scores if ids is None else ids).shape[0], (scores.shape[1] if ids is None else scores)
    sd = None
    if ids is None:
        sd = torch.full((max(T, 1), stride or E), float("nan"), device="cuda")
        sd[:T, :E] = dev(torch, scores.astype(np.float32))
    whole = lambda *s: torch.full(s, -99, dtype=torch.int32, device="cuda")  # noqa: E731
    idd = whole(T + 1, k) if ids is None else dev(torch, ids.astype(np.int32))
    w, off, rows, place = torch.full((T + 1, k), -9.0, device="cuda"), whole(E + 2), whole(T * k + 1), whole(T * k + 1)
    rc.experts_route_dev(sd.data_ptr() if ids is None else 0, T, E, k, idd.data_ptr(),
                         w.data_ptr() if ids is None else 0, off.data_ptr(), rows.data_ptr(), place.data_ptr(),
                         score_stride=stride, over_all=over_all, stream=stream(torch))
    torch.cuda.synchronize()
    assert off[-1] == -99 and rows[-1] == -99 and place[-1] == -99
    if ids is None:
        assert (idd[T] == -99).all() and (w[T] == -9).all()
    return (idd[:T].cpu().numpy(), f64(w[:T]), off[:-1].cpu().numpy(), rows[:-1].cpu().numpy(),
            place[:-1].view(T, k).cpu().numpy())


@pytest.mark.parametrize("T,E,k,over_all", [
    (1, 1, 1, False), (1, 8, 2, False), (31, 64, 8, True), (32, 64, 6, False), (33, 5, 5, True),
    (256, 33, 4, False), (257, 60, 8, True), (1000, 128, 8, False), (300, 129, 32, True),
    (64, 256, 3, False), (500, 257, 8, True), (70, 1024, 32, False), (5000, 64, 6, True), (3001, 3, 2, False),
])
def test_route(torch, rc, T, E, k, over_all):
    rng = np.random.default_rng(T * E + k)
    scores = np.round(rng.standard_normal((T, E)) * 8) / 8  # many equal ones
    scores[rng.random((T, E)) < 0.1] = -np.inf
    scores[rng.random(T) < 0.05] = -np.inf  # tokens without an expert
    scores[rng.random((T, E)) < 0.02] = np.nan
    scores[rng.random((T, E)) < 0.05] = -0.0
    scores = scores.astype(np.float32).astype(np.float64)
    ids, w, off, rows, place = route(torch, rc, scores, k, over_all, stride=E + 3)
    want, ww = lo.route(scores, k, over_all)
    np.testing.assert_array_equal(ids, want)
    bar = ww * U * (48 + 2 * 16)  # scores lie within 16 of each other
    assert (np.abs(w - ww) <= bar).all()
    for got, exact in zip((off, rows, place), lo.order(want, E)):
        np.testing.assert_array_equal(got, exact)


def test_route_of_infinite_and_far_scores(torch, rc):
    inf = np.inf
    scores = np.array([[inf, 1, inf, 0], [3e38, -3e38, 0, 3e38], [-inf, -inf, -3e38, -inf], [0, 1000, -1000, 999]])
    scores = scores.astype(np.float32).astype(np.float64)
    for over_all in (False, True):
        ids, w, *_ = route(torch, rc, scores, 3, over_all)
        want, ww = lo.route(scores, 3, over_all)
        np.testing.assert_array_equal(ids, want)
        np.testing.assert_allclose(w, ww, rtol=60 * U, atol=1e-44)


@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (40, 7, 3), (300, 64, 8), (4000, 200, 8), (100, 1024, 32), (9, 2, 1)])
def test_order_of_given_experts(torch, rc, T, E, k):
    rng = np.random.default_rng(T + E)
    ids = rng.integers(-1, E + 1, (T, k))  # padding, ids past the end, the same twice
    ids[rng.random((T, k)) < 0.02] = 2 ** 31 - 1
    _, _, off, rows, place = route(torch, rc, E, k, ids=ids)
    for got, exact in zip((off, rows, place), lo.order(ids, E)):
        np.testing.assert_array_equal(got, exact)
    _, _, off, rows, place = route(torch, rc, E, k, ids=np.full((T, k), -1))
    assert (off == 0).all() and (rows == -1).all() and (place == -1).all()


def test_route_of_no_token_writes_offsets(torch, rc):
    off = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    rc.experts_route_dev(0, 0, 8, 2, 0, 0, off.data_ptr(), 0, 0, stream=stream(torch))
    assert (off == 0).all()


# ---------------------------------------------------------------- combine --
@pytest.mark.parametrize("name,out,T,k,C,base,gap,offset", [
    ("f32", "f32", 1, 1, 1, False, 0, 0), ("f32", "f32", 1, 8, 2048, True, 0, 0),
    ("bf16", "bf16", 33, 2, 264, True, 8, 0), ("f16", "f32", 100, 6, 130, False, 0, 0),
    ("bf16", "f16", 7, 32, 96, True, 3, 0), ("f32", "bf16", 50, 3, 72, True, 0, 1),
    ("f16", "bf16", 2000, 2, 512, True, 0, 0),
])
def test_combine(torch, rc, name, out, T, k, C, base, gap, offset):
    rng = np.random.default_rng(T * C)
    dt, code = types(torch, rc, name)
    ot, ocode = types(torch, rc, out)
    P = T * k
    y = torch.full(((P + 1) * (C + gap) + offset,), float("nan"), dtype=dt, device="cuda")[offset:].view(P + 1, C + gap)
    y[:P, :C] = dev(torch, rng.standard_normal((P, C))).to(dt)
    place = rng.permutation(P).reshape(T, k).astype(np.int32)
    place[rng.random((T, k)) < 0.2] = -1
    place[rng.random((T, k)) < 0.1] = P
    w = rng.random((T, k)).astype(np.float32)
    pd, wd = dev(torch, place), dev(torch, w)
    o = torch.full(((T + 1) * (C + gap) + offset,), -5.0, dtype=ot, device="cuda")[offset:].view(T + 1, C + gap)
    b = None
    if base:  # in place for even T
        b = o if T % 2 == 0 else torch.full((T, C + gap), float("nan"), dtype=ot, device="cuda")
        b[:T, :C] = dev(torch, rng.standard_normal((T, C))).to(ot)
    exact, mag = lo.combine(f64(y[:P, :C]), place, w.astype(np.float64), f64(b[:T, :C]) if base else None)
    rc.experts_combine_dev(code, y.data_ptr(), P, pd.data_ptr(), wd.data_ptr(), T, k, C, ocode, o.data_ptr(),
                           d_base=b.data_ptr() if base else 0, y_stride=C + gap, base_stride=C + gap,
                           out_stride=C + gap, stream=stream(torch))
    got = f64(o)
    err = (k + 2) * U * mag
    assert (np.abs(got[:T, :C] - exact) <= err + HALF[out] * (np.abs(exact) + err) + TINY[out]).all()
    assert (got[T:] == -5).all() and (got[:, C:] == -5).all()


# --------------------------------------------------------------- together --
class Layer:
    """An expert layer of e4m3 weights with all its buffers, as an engine keeps them."""

    def __init__(self, torch, rc, T, H, I, E, k, seed):
        self.torch, self.rc, self.T, self.H, self.I, self.E, self.k = torch, rc, T, H, I, E, k
        gen = torch.Generator("cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.h, self.scores = normal(T, H), normal(T, E)
        P, nh, ni = T * k, -(-H // 128), -(-I // 128)
        empty = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
        whole = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.wq, self.ws = empty(E, 2, I, H), torch.zeros(E, 2, ni, nh, device="cuda")
        self.vq, self.vs = empty(E, 1, H, I), torch.zeros(E, 1, nh, ni, device="cuda")
        for q, s, n_in in ((self.wq, self.ws, H), (self.vq, self.vs, I)):
            for e in range(E):
                for g in range(q.shape[1]):
                    w = normal(q.shape[2], n_in) / n_in ** 0.5
                    rc.f8_quantise_dev(rc.F32, w.data_ptr(), q[e, g].data_ptr(), s[e, g].data_ptr(), q.shape[2],
                                       n_in, block_rows=128, stream=stream(torch))
        self.up = rc.Linear(rc.E4M3, I, H, self.wq.data_ptr(), n_experts=E, gated=True, d_scale=self.ws.data_ptr())
        self.down = rc.Linear(rc.E4M3, H, I, self.vq.data_ptr(), n_experts=E, d_scale=self.vs.data_ptr())
        self.ids, self.place, self.off, self.rows = whole(T, k), whole(T, k), whole(E + 1), whole(P)
        self.weights = torch.zeros(T, k, device="cuda")
        self.xq, self.xs = empty(T, H), torch.zeros(T, nh, device="cuda")
        self.mid, self.mq, self.ms = normal(P, I).bfloat16(), empty(P, I), torch.zeros(P, ni, device="cuda")
        self.y, self.out = normal(P, H), torch.zeros(T, H, device="cuda")

    def run(self, s):
        rc, T, H, I, E, k, P = self.rc, self.T, self.H, self.I, self.E, self.k, self.T * self.k
        rc.experts_route_dev(self.scores.data_ptr(), T, E, k, self.ids.data_ptr(), self.weights.data_ptr(),
                             self.off.data_ptr(), self.rows.data_ptr(), self.place.data_ptr(), stream=s)
        rc.f8_quantise_dev(rc.F32, self.h.data_ptr(), self.xq.data_ptr(), self.xs.data_ptr(), T, H, stream=s)
        self.up.grouped_dev(self.xq.data_ptr(), T, self.off.data_ptr(), rc.BF16, self.mid.data_ptr(), P,
                            d_rows=self.rows.data_ptr(), d_x_scale=self.xs.data_ptr(), stream=s)
        rc.f8_quantise_dev(rc.BF16, self.mid.data_ptr(), self.mq.data_ptr(), self.ms.data_ptr(), P, I, stream=s)
        self.down.grouped_dev(self.mq.data_ptr(), P, self.off.data_ptr(), rc.F32, self.y.data_ptr(), P,
                              d_x_scale=self.ms.data_ptr(), stream=s)
        rc.experts_combine_dev(rc.F32, self.y.data_ptr(), P, self.place.data_ptr(), self.weights.data_ptr(), T, k,
                               H, rc.F32, self.out.data_ptr(), d_base=self.h.data_ptr(), stream=s)

    def verify(self):
        """Each step against the oracle on what the step before it left."""
        n = lambda t: t.cpu().numpy()  # noqa: E731
        ids, w = lo.route(f64(self.scores), self.k, False)
        np.testing.assert_array_equal(n(self.ids), ids)
        off, rows, place = lo.order(ids, self.E)
        np.testing.assert_array_equal(n(self.rows), rows)
        same_codes((n(self.xq), n(self.xs)), lo.quantise(f64(self.h)))
        live = off[-1]
        same_codes((n(self.mq)[:live], n(self.ms)[:live]), lo.quantise(f64(self.mid)[:live]))
        x, m = lo.dequantise(n(self.xq), n(self.xs)), lo.dequantise(n(self.mq), n(self.ms))
        for e in range(self.E):
            at = np.arange(off[e], off[e + 1])
            if not len(at):
                continue
            for got, rows_in, q, s, out in ((self.mid, x[rows[at]], self.wq, self.ws, "bf16"),
                                            (self.y, m[at], self.vq, self.vs, "f32")):
                wd = np.stack([lo.dequantise(n(q[e, g]), n(s[e, g]), 128) for g in range(q.shape[1])])
                exact, parts, mags = lo.product(rows_in, wd)
                bar = lo.product_bar(parts, mags, wd.shape[2] / 32 + wd.shape[2] / 128 + 1, HALF[out], TINY[out])
                assert (np.abs(f64(got)[at] - exact) <= bar).all()
        exact, mag = lo.combine(f64(self.y), place, f64(self.weights), f64(self.h))
        assert (np.abs(f64(self.out) - exact) <= (self.k + 2) * U * mag + U * np.abs(exact)).all()


@pytest.mark.parametrize("T,H,I,E,k", [(1, 256, 128, 8, 2), (40, 384, 200, 16, 4), (300, 256, 264, 6, 3)])
def test_expert_layer(torch, rc, T, H, I, E, k):
    if I % 16:
        I = -(-I // 16) * 16
    layer = Layer(torch, rc, T, H, I, E, k, 1)
    layer.run(stream(torch))
    layer.up.check(stream(torch))
    layer.down.check(stream(torch))
    layer.verify()


@pytest.mark.parametrize("name", ["e4m3", "f16"])
@pytest.mark.parametrize("R", [7, 60, 200])
def test_listed_rows_split_over_k(torch, rc, name, R):
    """Few tiles and many channels: a cluster for each tile, rows gathered by either way."""
    c = Case(torch, rc, name, 50, 100, 4000)
    rows = np.random.default_rng(R).integers(0, 50, R)
    off, rd = dev(torch, np.array([0, R], np.int32)), dev(torch, rows.astype(np.int32))
    y, code = c.out("bf16", R)
    c.lin.grouped_dev(c.xd.data_ptr(), 50, off.data_ptr(), code, y.data_ptr(), R, d_rows=rd.data_ptr(),
                      stream=stream(torch), **c.kw)
    c.lin.check(stream(torch))
    c.close(f64(y)[:R], c.x[rows], 0, "bf16")


def test_expert_layers_in_graphs_and_streams(torch, rc):
    """A layer captured once and replayed with other inputs in its buffers, while another
    runs on a second stream; a second graph of the same objects."""
    a, b = Layer(torch, rc, 40, 256, 256, 8, 2, 3), Layer(torch, rc, 70, 384, 128, 5, 2, 4)
    other = torch.cuda.Stream()
    a.run(stream(torch))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for i, g in enumerate(graphs * 2):
        a.h.normal_()
        a.scores.normal_()
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(other):
            for _ in range(3):
                b.run(other.cuda_stream)
        torch.cuda.synchronize()
        a.verify()
        b.verify()
    a.up.check(stream(torch))
    b.down.check(other.cuda_stream)
