"""GPU: the paged 4-bit cache and its attention at their edges: many items a CTA,
waits that run out, against float64 numpy (tests/kv4_oracle.py)."""
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


@pytest.mark.parametrize("kw", [
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=16, lens=[9000, 40, 700], poison=False),
    dict(dtype="f32", nh=4, nkv=4, hd=64, page=16, lens=[255]),
    dict(dtype="f32", nh=2, nkv=1, hd=256, page=16, lens=[40] * 300),          # short items first
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=32, lens=[400, 90], qs=[5, 7]),
    dict(dtype="f16", nh=8, nkv=8, hd=64, page=16, lens=[1500], qs=[640]),     # chunks: more tiles than stages
    dict(dtype="bf16", nh=16, nkv=16, hd=128, page=16, lens=[150], qs=[300]),  # and fewer
])
def test_a_wait_that_runs_out_is_a_status(torch, rc, kw):
    """One arrival is withheld, so waits of a CTA run out: the launch ends, the check
    says so once, and the next call, with a new scratch, is right."""
    c = base.Case(torch, rc, seed=41, **kw)
    spoiled = rc.Kv4Scratch(c.kv)
    try:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_us(20000))
        rc.check(rc.lib().rabbit_cuda_kv4_debug_withhold(c.kv.handle))
        c.call(ws=spoiled)
        with pytest.raises(rc.RabbitCudaError) as e:
            c.kv.check(base.stream(torch))
        assert e.value.status == rc.ERR_TIMEOUT
    finally:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(2000))
    c.kv.check(base.stream(torch))  # said once
    c.call()
    c.check()


@pytest.mark.parametrize("order", ["page first", "slot behind"])
def test_a_timeout_is_not_hidden_by_what_is_out_of_range(torch, rc, order):
    """A scratch is spoiled after a timeout, so its status comes before the others'."""
    c = base.Case(torch, rc, dtype="bf16", nh=8, nkv=2, hd=64, page=16, lens=[3000, 40], seed=42)
    st = base.stream(torch)
    if order == "page first":
        bad = c.table.clone()
        c.table[1, 0] = 100000
        c.call()
        c.table.copy_(bad)
    try:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_us(20000))
        rc.check(rc.lib().rabbit_cuda_kv4_debug_withhold(c.kv.handle))
        c.call(ws=rc.Kv4Scratch(c.kv))
    finally:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(2000))
    if order == "slot behind":
        x = torch.zeros(1, 2, 64, device="cuda")
        s = torch.tensor([1 << 40], device="cuda")
        c.kv.append_dev(0, rc.F32, x.data_ptr(), x.data_ptr(), s.data_ptr(), 1, stream=st)
    with pytest.raises(rc.RabbitCudaError, match=order.split()[0]) as e:
        c.kv.check(st)
    assert e.value.status == rc.ERR_TIMEOUT
    c.kv.check(st)
    c.call()
    c.check()
