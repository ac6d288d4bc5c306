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
