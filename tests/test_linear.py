"""The refusals of the 8-bit rows, the products and the expert batches that need no
GPU, and their oracle against the definitions."""
from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import linear_oracle as lo

HEADER = Path(__file__).resolve().parents[1] / "include" / "rabbit_cuda.h"
P = 4096  # an address that is aligned; nothing reads it


def test_codes_are_the_nearest():
    rng = np.random.default_rng(1)
    for s in (np.float32(1.0), np.float32(0.3), np.float32(2.0 ** -149), np.float32(1e30)):
        mids = (lo.VALUES[1:127] + lo.VALUES[:126]) / 2
        t = np.concatenate([lo.VALUES[:127], mids, rng.uniform(0, 460, 300), rng.uniform(0, 0.02, 300)])
        if s == 1.0:  # t itself is x / s
            np.testing.assert_array_equal(lo.codes(t, s), [lo.nearest_code(v) for v in t])
            np.testing.assert_array_equal(lo.codes(-t, s), [lo.nearest_code(v) | 128 for v in t])
        x = (t * float(s)).astype(np.float32).astype(np.float64)
        got = lo.VALUES[lo.codes(x, s)]
        want = np.abs(lo.VALUES[:127, None] * float(s) - np.minimum(x, 448 * float(s))).min(0)
        np.testing.assert_array_equal(np.abs(got * float(s) - np.minimum(x, 448 * float(s))), want)


def test_oracle_quantises_each_block_by_its_own_maximum():
    x = np.arange(1, 131, dtype=np.float64)[None].repeat(3, 0)
    x[1] *= 100
    q, s = lo.quantise(x)
    np.testing.assert_array_equal(s[:, 0], np.float32(x[:, 127] / 448))
    np.testing.assert_array_equal(s[:, 1], np.float32(x[:, 129] / 448))
    assert (np.abs(lo.dequantise(q, s) - x) <= x * 2.0 ** -4 + s.max() * 2.0 ** -10).all()
    q, s = lo.quantise(x, 128)
    assert s.shape == (1, 2) and s[0, 0] == np.float32(12800 / 448)


def test_oracle_orders_pairs_by_expert_and_pair():
    ids = np.array([[2, 0], [0, -1], [2, 2], [9, 0]], np.int32)
    offsets, rows, place = lo.order(ids, 3)
    assert offsets.tolist() == [0, 3, 3, 6]
    assert rows.tolist() == [0, 1, 3, 0, 2, 2, -1, -1]
    assert place.tolist() == [[3, 0], [1, -1], [4, 5], [-1, 2]]


def test_linear_desc_layout_matches_header(rc):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} rabbit_cuda_linear_desc;", text).group(1)
    fields = [f.strip(" *") for line in body.split(";") for f in line.split(",") if f.strip()]
    assert [f.split()[-1].strip("*") for f in fields] == [f for f, _ in rc.LinearDesc._fields_]


@pytest.mark.parametrize("kw", [
    dict(dtype=0), dict(dtype=4), dict(n_experts=0), dict(n_experts=1025), dict(gated=2),
    dict(n_out=0), dict(n_out=(1 << 20) + 1), dict(n_in=0), dict(n_in=(1 << 20) + 1), dict(d_w=None),
    dict(d_w=P + 8), dict(w_stride=112), dict(w_stride=130), dict(n_in=100), dict(d_scale=None),
    dict(d_scale=P + 2), dict(dtype=1), dict(w_stride=-128), dict(dtype=2, d_scale=None, w_stride=132),
    dict(n_out=1 << 20, w_stride=1 << 20),
])
def test_linear_create_refuses(rc, kw):
    d = dict(dtype=rc.E4M3, n_experts=1, gated=0, n_out=64, n_in=128, d_w=P, w_stride=0, d_scale=P)
    d.update(kw)
    desc, out = rc.LinearDesc(**d), C.c_void_p(7)
    assert rc.lib().rabbit_cuda_linear_create(C.byref(desc), 0, C.byref(out)) == rc.ERR_ARGS
    assert not out.value and rc.lib().rabbit_cuda_last_error()


def test_null_arguments_are_refused(rc):
    so, out = rc.lib(), C.c_void_p()
    desc = rc.LinearDesc(rc.E4M3, 1, 0, 64, 128, P, 0, P)
    assert so.rabbit_cuda_linear_create(None, 0, C.byref(out)) == rc.ERR_ARGS
    assert so.rabbit_cuda_linear_create(C.byref(desc), 0, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_linear_dev(None, P, 0, P, 0, 0, P, 0, 1, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_linear_grouped_dev(None, P, 0, 1, P, 0, None, P, 0, P, 0, 1, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_linear_check(None, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_linear_debug_withhold(None) == rc.ERR_ARGS
    assert so.rabbit_cuda_linear_free(None) == rc.OK


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(n_rows=-1), dict(n_cols=0), dict(n_cols=(1 << 20) + 1),
    dict(block_rows=2), dict(block_rows=0), dict(d_x=None), dict(d_q=None), dict(d_scale=None),
    dict(d_x=P + 2), dict(dtype=1, d_x=P + 1), dict(d_scale=P + 1), dict(x_stride=99), dict(q_stride=99),
    dict(n_rows=1 << 30, n_cols=300), dict(d_rows=P, x_rows=4, block_rows=128), dict(d_rows=P, x_rows=0), dict(d_rows=P + 2, x_rows=4),
])
def test_quantise_refuses(rc, kw):
    d = dict(dtype=0, d_x=P, x_stride=0, x_rows=0, d_rows=None, d_q=P, q_stride=0, d_scale=P, n_rows=4,
             n_cols=100, block_rows=1, stream=None)
    d.update(kw)
    assert rc.lib().rabbit_cuda_f8_quantise_dev(*d.values()) == rc.ERR_ARGS


def test_nothing_to_do_needs_nothing(rc):
    so = rc.lib()
    assert so.rabbit_cuda_f8_quantise_dev(0, None, 0, 0, None, None, 0, None, 0, 100, 1, None) == rc.OK
    assert so.rabbit_cuda_experts_combine_dev(0, None, 0, 0, None, None, 0, 1, 8, 0, None, 0, None, 0,
                                              None) == rc.OK


@pytest.mark.parametrize("kw", [
    dict(n_tokens=-1), dict(n_experts=0), dict(n_experts=1025), dict(k=0), dict(k=9), dict(k=33, n_experts=64),
    dict(over_all=2), dict(n_tokens=1 << 29, k=2), dict(d_ids=None), dict(d_weights=None),
    dict(d_offsets=None), dict(d_rows=None), dict(d_place=None), dict(score_stride=7),
    dict(d_scores=P + 2), dict(d_place=P + 2),
])
def test_route_refuses(rc, kw):
    d = dict(d_scores=P, score_stride=0, n_tokens=4, n_experts=8, k=2, over_all=0, d_ids=P, d_weights=P,
             d_offsets=P, d_rows=P, d_place=P, stream=None)
    d.update(kw)
    assert rc.lib().rabbit_cuda_experts_route_dev(*d.values()) == rc.ERR_ARGS


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(out_dtype=-1), dict(y_rows=-1), dict(n_tokens=-1), dict(k=0), dict(k=33), dict(n_cols=0),
    dict(d_y=None), dict(d_place=None), dict(d_weights=None), dict(d_out=None), dict(y_stride=63),
    dict(out_stride=63), dict(base_stride=63), dict(d_y=P + 2), dict(d_out=P + 2), dict(d_place=P + 1),
    dict(d_base=P, d_out=P, base_stride=64, out_stride=72), dict(n_tokens=1 << 23),
])
def test_combine_refuses(rc, kw):
    d = dict(dtype=0, d_y=P, y_stride=0, y_rows=8, d_place=P, d_weights=P, n_tokens=4, k=2, n_cols=64,
             out_dtype=0, d_base=2 * P, base_stride=0, d_out=3 * P, out_stride=0, stream=None)
    d.update(kw)
    assert rc.lib().rabbit_cuda_experts_combine_dev(*d.values()) == rc.ERR_ARGS
