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
