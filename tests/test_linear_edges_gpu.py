"""GPU: the products, the e4m3 rows and the expert routing at their edges: launches one right after
the other, waits that run out, sums without cancellation, far gates, against float64 numpy
(tests/linear_oracle.py; the bars of tests/test_linear_gpu.py unless said otherwise)."""
from __future__ import annotations

import numpy as np
import pytest

import linear_oracle as lo
import test_linear_gpu as base

pytestmark = pytest.mark.gpu

torch = base.torch  # the module's fixture


def test_pairs_that_follow_one_another(torch, rc):
    """Pairs of CTAs with a step or a few a tile, one launch right behind the other on two streams: what
    the last products of one launch still have to say reaches no barrier of the next."""
    cases = []
    for name, R, N, K, gated, out in [("e4m3", 600, 700, 128, False, "bf16"), ("bf16", 600, 2000, 64, False, "bf16"),
                                      ("e4m3", 520, 300, 384, True, "f32"), ("f16", 640, 2100, 200, True, "f32")]:
        c = base.Case(torch, rc, name, R, N, K, gated)
        y, code = c.out(out, R)
        cases.append((c, y, code, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(100):
        for c, y, code, _ in cases:
            s = streams[c.G - 1]
            c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), c.R, stream=s.cuda_stream, **c.kw)
    for c, y, code, out in cases:
        c.lin.check(streams[c.G - 1].cuda_stream)
        at = np.arange(0, c.R, 7)
        c.close(base.f64(y)[at], c.x[at], 0, out)
        first = y.clone()
        c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), c.R, stream=base.stream(torch), **c.kw)
        torch.cuda.synchronize()
        assert torch.equal(y, first)


@pytest.mark.parametrize("name,R,N,K,gated,out", [
    ("bf16", 700, 3000, 256, False, "bf16"), ("f16", 700, 3000, 512, False, "f32"),
    ("e4m3", 700, 3000, 512, False, "bf16"), ("e4m3", 600, 700, 2500, True, "f32"), ("f16", 600, 2000, 200, True, "f16"),
])
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("cta", [0, 1])
def test_a_pair_of_which_one_gives_up_first(torch, rc, name, R, N, K, gated, out, listed, cta):
    """One CTA of each pair copies a step less than the other. The call ends with a status, nothing of it
    is still under way then (the check would say so), and the next call is whole."""
    c = base.Case(torch, rc, name, R, N, K, gated)
    off, rows = base.dev(torch, np.array([0, R], np.int32)), base.dev(torch, np.arange(R, dtype=np.int32)[::-1])
    y, code = c.out(out, R)
    run = lambda: c.lin.grouped_dev(c.xd.data_ptr(), R, off.data_ptr(), code, y.data_ptr(), R,  # noqa: E731
                                    d_rows=rows.data_ptr() if listed else 0, stream=base.stream(torch), **c.kw)
    rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(20))
    try:
        rc.check(rc.lib().rabbit_cuda_linear_debug_withhold_cta(c.lin.handle, cta))
        run()
        with pytest.raises(rc.RabbitCudaError, match="wait ran out") as e:
            c.lin.check(base.stream(torch))
        assert e.value.status == rc.ERR_TIMEOUT and "did not end" not in str(e.value)
    finally:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(2000))
    run()
    c.lin.check(base.stream(torch))
    at = np.arange(0, R, max(1, R // 40))
    c.close(base.f64(y)[at], c.x[::-1][at] if listed else c.x[at], 0, out)


def test_two_threads_route_among_different_numbers_of_experts(torch, rc):
    """Both need more shared memory than a launch has unasked, and not the same: what the kernel may take
    belongs to the kernel, not to a call."""
    import threading

    T, k, wrong = 40, 8, []
    rng = np.random.default_rng(11)
    ids = {E: rng.integers(0, E, (T, k)).astype(np.int32) for E in (360, 700, 1024)}
    idd = {E: base.dev(torch, v) for E, v in ids.items()}
    got = {E: [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * k, T * k)] for E in ids}
    streams = {E: torch.cuda.Stream() for E in ids}
    torch.cuda.synchronize()
    start = threading.Barrier(len(ids))

    def go(E):
        off, rows, place = (t.data_ptr() for t in got[E])
        start.wait()
        for _ in range(1500):
            try:
                rc.experts_route_dev(0, T, E, k, idd[E].data_ptr(), 0, off, rows, place, stream=streams[E].cuda_stream)
            except rc.RabbitCudaError as e:
                wrong.append((E, str(e)))
                return

    threads = [threading.Thread(target=go, args=(E,)) for E in ids]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
    for E in ids:
        for t, exact in zip(got[E], lo.order(ids[E], E)):
            np.testing.assert_array_equal(t.cpu().numpy(), exact.reshape(-1))


@pytest.mark.parametrize("name,R,K", [("bf16", 7, 512), ("bf16", 99, 128), ("bf16", 700, 128),  # one CTA, pairs
                                      ("e4m3", 40, 128), ("e4m3", 99, 128), ("e4m3", 700, 128)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_far_gates(torch, rc, name, R, K, out):
    """silu(g) u where exp(-g) leaves fp32 and g exp(g) does not yet: gates down to -104, each product exact
    (one channel the gate, one the up). Bar, u = 2^-24: fp32 outputs take exp(-|g| / 2) to a step (2 u), its square and
    the gate times it twice (2 * 2 u + 2 u), 1 + its square (half of 5 u, and u), the division (4 u) and up (u): 15 u.
    bf16's: exp(-|g| / 2) to 4 u and 3/4 |g| u, so 8 u + 3/2 |g| u and 2 u above, 1 + its square at most half of 9 u,
    3/4 of |g| / (1 + e^|g|) < 0.3 and u below, the division 4 u and up u: (21 + 1.5 |g|) u, then half a step of bf16.
    Below 2^-126 fp32's smallest step, times up."""
    N = 40
    gates = np.concatenate([-np.arange(87, 104.5, 0.5), -np.arange(0, 16, 0.5), [0.25, 1, 3, 8, 40, 80, 88, 100, 120],
                            -np.arange(16, 87, 1.5)])
    if name == "e4m3":  # codes of 4 bits: the scale makes the rest
        x, w = np.zeros((R, K)), np.zeros((2, N, K))
        g = np.resize(gates, R)
        x[:, 0], x[:, 1] = 1, 1
        w[0, :, 0], w[1, :, 1] = 1, 1
        xq, one = (x * 0x38).astype(np.uint8), 0x38  # the code of 1
        c = base.Case(torch, rc, name, R, N, K, True)
        c.xd[:R, :K] = base.dev(torch, xq)
        c.wd[0, :, :, :K] = base.dev(torch, (w * one).astype(np.uint8))
        up = 2.0 ** 60
        # the token's scale is |g|, the gate's its sign, the up's 2^60 / |g| cannot be exact for each: up = |g| 2^60
        c.sx[:] = base.dev(torch, np.abs(g)[:, None].astype(np.float32))
        c.sw[:] = 0
        c.sw[0, 0], c.sw[0, 1] = -1.0, up
        g, u = -np.abs(g), np.abs(g) * up
    else:
        c = base.Case(torch, rc, name, R, N, K, True)
        g = np.resize(gates, R)
        x, w = np.zeros((R, K)), np.zeros((2, N, K))
        x[:, 0], x[:, 1] = g, 1
        w[0, :, 0], w[1, :, 1] = 1, 2.0 ** 60
        c.xd[:R, :K], c.wd[0, :, :, :K] = base.dev(torch, x).bfloat16(), base.dev(torch, w).bfloat16()
        u = np.full(R, 2.0 ** 60)
    y, code = c.out(out, R)
    c.lin.apply_dev(c.xd.data_ptr(), code, y.data_ptr(), R, stream=base.stream(torch), **c.kw)
    c.lin.check(base.stream(torch))
    want = lo.silu(g) * u
    a = np.abs(g)
    steps = 15 if out == "f32" else 21 + 1.5 * a
    bar = steps * base.U * np.abs(want) + 2.0 ** -148 * np.abs(u)
    bar = bar + base.HALF[out] * (np.abs(want) + bar)
    off = np.abs(base.f64(y)[:R] - want[:, None])
    wrong = ~(off <= bar[:, None]).all(1)
    assert not wrong.any(), list(zip(g[wrong], base.f64(y)[:R][wrong, 0], want[wrong]))[:8]


@pytest.mark.parametrize("name,R,N,K,out", [
    ("bf16", 3, 70, 14336, "f32"), ("f16", 300, 130, 14336, "f32"), ("bf16", 600, 9600, 14336, "f32"),  # pairs at last
    ("e4m3", 7, 70, 14336, "f32"), ("e4m3", 600, 3000, 14336, "f32"), ("f16", 5, 9600, 32768, "f16"),
    ("f16", 600, 9600, 4096, "f16"), ("f16", 600, 9600, 14336, "f16"), ("bf16", 600, 9600, 16384, "bf16"),
    ("bf16", 600, 9600, 8192, "f16"), ("bf16", 40, 70, 17000, "bf16"),
])
def test_sums_of_one_sign(torch, rc, name, R, N, K, out):
    """Terms of one sign, so that every partial sum counts in full. Bar, u = 2^-24: each tensor-core step (32
    bytes of channels) is off by 4 u of the sum it leaves there, which starts anew with each part of 256
    channels (e4m3: block of 128); each part's addition by u of the sum so far (e4m3: a scale's product, one more u of
    the part), the sum over a cluster's eight parts and the rest by 8 u of the whole. Summed in tensor memory
    over all channels, a step's error goes by the whole sum so far: several times this bar, and the bar for
    16-bit outputs of fewer channels."""
    rng = np.random.default_rng(R + K)
    f8 = name == "e4m3"
    dt, code = base.types(torch, rc, name)
    gen = torch.Generator("cuda").manual_seed(3)
    some = lambda *s: torch.rand(*s, generator=gen, device="cuda") * 0.35 + 0.05  # noqa: E731
    x, w = some(R, K), some(N, K)
    if f8:  # codes 0x20 .. 0x40: 2^-3 .. 2
        x, w = (torch.randint(0x20, 0x40, s, generator=gen, device="cuda", dtype=torch.uint8) for s in ((R, K), (N, K)))
        nb = K // 128
        sx, sw = some(R, nb), some(-(-N // 128), nb)
    else:
        x, w = x.to(dt), w.to(dt)
    lin = rc.Linear(code, N, K, w.data_ptr(), d_scale=sw.data_ptr() if f8 else 0)
    yt, ycode = base.types(torch, rc, out)
    y = torch.zeros(R, N, dtype=yt, device="cuda")
    lin.apply_dev(x.data_ptr(), ycode, y.data_ptr(), R, d_x_scale=sx.data_ptr() if f8 else 0, stream=base.stream(torch))
    lin.check(base.stream(torch))
    step, part = (32, 128) if f8 else (16, 256)
    if K <= {"f16": 4096, "bf16": 16384, "f32": 0}[out]:
        part = K
    pad = -K % part  # (zeros: nothing is added)
    outs = np.arange(N) if N < 200 else rng.integers(0, N, 90)
    ww = lo.VALUES[w[outs].cpu().numpy()] if f8 else base.f64(w[outs])
    for r in sorted({0, R - 1, R // 2, R // 3}):
        xx = lo.VALUES[x[r].cpu().numpy()] if f8 else base.f64(x[r])
        # [outputs, parts, steps]: sums that the tensor cores leave after each step
        held = np.pad(ww * xx, ((0, 0), (0, pad))).reshape(len(outs), -1, part // step, step).sum(-1).cumsum(-1)
        if f8:
            held = held * (base.f64(sx[r]) * base.f64(sw)[outs // 128])[..., None]
        sums = held[..., -1].cumsum(-1)
        want = sums[:, -1]
        bar = base.U * (4 * held.sum((1, 2)) + sums.sum(1) + (8 + f8) * want)
        if out != "f32":  # half of the step between the numbers around it
            bar = bar + 2.0 ** (np.floor(np.log2(want)) - (11 if out == "f16" else 8))
        off = np.abs(base.f64(y[r])[outs] - want)
        assert (off <= bar).all(), (r, (off / bar).max())


@pytest.mark.parametrize("name", ["e4m3", "f16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("listed", [False, True])
def test_what_is_not_finite_stays_in_its_row_of_many(torch, rc, name, gated, listed):
    """Tiles of 256 tokens by pairs of CTAs: NaN in a token's row, in an output's weights and in a scale
    reach no other row or output, nor the other expert."""
    R, N, K = 600, 300, 256
    c = base.Case(torch, rc, name, R, N, K, gated, experts=2)
    rows = np.random.default_rng(2).integers(0, R, R) if listed else np.arange(R)
    half = 290
    off, rd = base.dev(torch, np.array([0, half, R], np.int32)), base.dev(torch, rows.astype(np.int32))
    y, code = c.out("f32", R)

    def run():
        c.lin.grouped_dev(c.xd.data_ptr(), R, off.data_ptr(), code, y.data_ptr(), R,
                          d_rows=rd.data_ptr() if listed else 0, stream=base.stream(torch), **c.kw)
        c.lin.check(base.stream(torch))
        return y.clone()

    clean = run()
    assert clean[:R].isfinite().all()
    nan = 0x7F if name == "e4m3" else float("nan")
    some = [7, 289, 290, 511]
    for r in some:
        c.xd[int(rows[r]), 100] = nan
    c.wd[1, 0, 130, 5] = nan
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[:R][base.dev(torch, np.isin(rows, rows[some]))] = True
    bad[half:R, 130] = True
    got = run()
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])
    if name == "e4m3":
        c.sx[int(rows[33]), 1] = float("nan")
        c.sw[0, 0, 1, 0] = float("nan")
        bad[:R][base.dev(torch, rows == rows[33])] = True
        bad[:half, 128:256] = True
        got = run()
        assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


def test_blocks_of_as_many_rows_as_there_may_be(torch, rc):
    """2^31 - 1 rows of one column: the last block has 127."""
    R = 2 ** 31 - 1
    x = torch.zeros(R, dtype=torch.bfloat16, device="cuda")
    q = torch.full((R + 1,), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((2 ** 24 + 1,), 7.0, device="cuda")
    x[:3], x[-127], x[-1], x[-128] = 3.0, -2.0, 1.0, 448.0
    rc.f8_quantise_dev(rc.BF16, x.data_ptr(), q.data_ptr(), s.data_ptr(), R, 1, block_rows=128,
                       stream=base.stream(torch))
    torch.cuda.synchronize()
    for a, b, block in ((0, 128, 0), (R - 127, R, 2 ** 24 - 1), (R - 255, R - 127, 2 ** 24 - 2), (2 ** 30, 2 ** 30 + 128, 2 ** 23)):
        base.same_codes((q[a:b, None].cpu().numpy(), s[block:block + 1, None].cpu().numpy()),
                        lo.quantise(base.f64(x[a:b])[:, None], 128))
    assert q[-1] == 0x55 and s[-1] == 7.0
    assert int((q[:R] != 0).sum()) == 6
