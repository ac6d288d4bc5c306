"""GPU: the paged 4-bit cache and its attention at their edges: many items a
CTA, against float64 numpy (tests/kv4_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest

import test_rope_kv4_gpu as base

pytestmark = pytest.mark.gpu

torch = base.torch  # the module's fixture


@pytest.mark.parametrize("dtype,nh", [("bf16", 4), ("f32", 10)])
def test_many_items_of_all_lengths_in_a_cta(torch, rc, dtype, nh):
    """Some thirty items to a CTA, each merged by one warp while it makes the
    operands of those behind: short ones that a warp takes alone, longer ones
    that all share, ones that a run's border cuts. Twenty runs, the same bits."""
    lens = [1 + (37 * i) % 230 for i in range(1100)]
    c = base.Case(torch, rc, dtype=dtype, nh=nh, nkv=2, hd=32, page=16, lens=lens, seed=40)
    c.call()
    c.check()
    first = c.out.clone()
    for _ in range(20):
        c.out.fill_(7.0)
        c.call()
        assert torch.equal(c.out, first)
    c.kv.check(base.stream(torch))
