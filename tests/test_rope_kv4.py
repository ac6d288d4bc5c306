"""Rotary frequencies and the refusals of the cache-side entry points that need
no GPU."""
from __future__ import annotations

import ctypes as C
import math
import re
from pathlib import Path

import numpy as np
import pytest

import kv4_oracle as ko

HEADER = Path(__file__).resolve().parents[1] / "include" / "rabbit_cuda.h"


@pytest.mark.parametrize("rot,kw", [
    (128, {}), (2, {}), (64, dict(scaling="linear", factor=4.0)),
    (64, dict(scaling="ntk", factor=8.0)), (128, dict(scaling="ntk", factor=2.0, base=500000.0)),
    (128, dict(scaling="bands", factor=8.0, low=1.0, high=4.0, ctx=8192)),
    (96, dict(scaling="bands", factor=4.0, low=2.0, high=5.0, ctx=2048)),
    (64, dict(scaling="yarn", factor=32.0, low=1.0, high=32.0, ctx=4096)),
    (256, dict(scaling="yarn", factor=4.0, low=2.0, high=16.0, ctx=100)),
])
def test_frequencies(rc, rot, kw):
    names = {"none": rc.ROPE_SCALE_NONE, "linear": rc.ROPE_SCALE_LINEAR, "ntk": rc.ROPE_SCALE_NTK,
             "bands": rc.ROPE_SCALE_BANDS, "yarn": rc.ROPE_SCALE_YARN}
    r = rc.Rope(rot, scaling=names[kw.get("scaling", "none")], base=kw.get("base", 0.0),
                factor=kw.get("factor", 0.0), low=kw.get("low", 0.0), high=kw.get("high", 0.0),
                original_ctx=kw.get("ctx", 0))
    got, mag = r.freqs()
    # a power, a division and a blend of two terms: a few 2^-53 each
    np.testing.assert_allclose(got, ko.freqs(rot, **kw), rtol=1e-13)
    yarn = kw.get("scaling") == "yarn"
    assert mag == pytest.approx(1 + 0.1 * math.log(kw["factor"]) if yarn else 1.0, rel=1e-15)
    assert rc.Rope(rot, magnitude=0.5).freqs()[1] == 0.5


@pytest.mark.parametrize("kw", [
    dict(head_dim=0), dict(head_dim=1), dict(head_dim=1025), dict(head_dim=64, rot_dim=3),
    dict(head_dim=64, rot_dim=66), dict(head_dim=1024), dict(head_dim=64, rot_dim=-2),
    dict(head_dim=63), dict(head_dim=64, layout=2), dict(head_dim=64, scaling=5),
    dict(head_dim=64, scaling=-1), dict(head_dim=64, base=1.0), dict(head_dim=64, base=-1.0),
    dict(head_dim=64, base=math.nan), dict(head_dim=64, factor=-2.0),
    dict(head_dim=64, factor=math.inf), dict(head_dim=64, magnitude=math.nan),
    dict(head_dim=64, scaling=3), dict(head_dim=64, scaling=4, original_ctx=-4),
    dict(head_dim=64, scaling=3, original_ctx=64, low=4.0, high=4.0),
    dict(head_dim=2, scaling=2, factor=2.0),
])
def test_rope_refuses(rc, kw):
    with pytest.raises(rc.RabbitCudaError) as e:
        rc.Rope(kw.pop("head_dim"), **kw)
    assert e.value.status == rc.ERR_ARGS


def test_null_arguments_are_refused(rc):
    so = rc.lib()
    r = rc.Rope(64)
    one = np.zeros(4, np.int64).ctypes.data
    out = C.c_void_p()
    assert so.rabbit_cuda_rope_create(None, C.byref(out)) == rc.ERR_ARGS
    assert so.rabbit_cuda_rope_freqs(None, None, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_rope_freqs(r.handle, None, None) == rc.OK
    assert so.rabbit_cuda_rope_dev(None, 0, one, 0, one, 0, one, 1, 1, None) == rc.ERR_ARGS
    for args in [(3, one, 0, one, 0, one, 1, 1), (-1, one, 0, one, 0, one, 1, 1),
                 (0, None, 0, one, 0, one, 1, 1), (0, one, 0, None, 0, one, 1, 1),
                 (0, one, 0, one, 0, None, 1, 1), (0, one, 0, one, 0, one, -1, 1),
                 (0, one, 0, one, 0, one, 1, 0), (0, one, 63, one + 4, 0, one, 1, 1),
                 (0, one, 0, one, 60, one, 1, 1), (0, one, 64, one, 128, one, 2, 1),
                 (0, one + 2, 0, one, 0, one, 1, 1), (1, one + 1, 0, one, 0, one, 1, 1)]:
        assert so.rabbit_cuda_rope_dev(r.handle, *args, None) == rc.ERR_ARGS, args
    assert so.rabbit_cuda_rope_dev(r.handle, 0, None, 0, None, 0, None, 0, 1, None) == rc.OK
    assert so.rabbit_cuda_kv4_create(None, 0, C.byref(out)) == rc.ERR_ARGS
    assert so.rabbit_cuda_kv4_append_dev(None, 0, 0, one, 0, one, 0, one, 1, None, None,
                                         None) == rc.ERR_ARGS
    assert so.rabbit_cuda_kv4_read_dev(None, 0, 0, one, 1, one, one, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_kv4_scratch_create(None, C.byref(out)) == rc.ERR_ARGS
    b = rc.Kv4Batch(n_seqs=1)
    assert so.rabbit_cuda_kv4_attention_dev(None, 0, None, 0, one, 0, one, 0, 1, 1, C.byref(b), 0.0,
                                            0, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_kv4_check(None, None) == rc.ERR_ARGS
    assert so.rabbit_cuda_kv4_bytes(None) == 0
    for f in (so.rabbit_cuda_rope_free, so.rabbit_cuda_kv4_free, so.rabbit_cuda_kv4_scratch_free):
        assert f(None) == rc.OK


@pytest.mark.parametrize("kw", [
    dict(n_layers=0), dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(head_dim=0), dict(head_dim=12),
    dict(head_dim=264), dict(page_size=8), dict(page_size=24), dict(page_size=2048),
    dict(n_pages=0), dict(n_pages=-1), dict(device=-1), dict(device=99), dict(n_layers=1 << 20),
])
def test_cache_refuses(rc, kw):
    base = dict(n_layers=1, n_kv_heads=1, head_dim=64, page_size=16, n_pages=1)
    with pytest.raises(rc.RabbitCudaError) as e:
        rc.Kv4(**{**base, **kw})
    assert e.value.status == rc.ERR_ARGS


@pytest.mark.parametrize("struct,cls", [("rabbit_cuda_rope_desc", "RopeDesc"),
                                        ("rabbit_cuda_kv4_desc", "Kv4Desc"),
                                        ("rabbit_cuda_kv4_batch", "Kv4Batch")])
def test_struct_layouts_match_the_header(rc, struct, cls):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % struct, text).group(1)
    names = [n.strip(" *") for d in body.split(";") if d.strip()
             for n in re.sub(r"^\s*(const\s+)?\w+\s", "", d.strip()).split(",")]
    assert names == [f for f, _ in getattr(rc, cls)._fields_]
