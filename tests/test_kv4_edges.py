"""The 4-bit cache without a GPU: what the binding refuses itself, and the oracle
(tests/kv4_oracle.py) against its formulas written out number by number."""
from __future__ import annotations

import math

import numpy as np
import pytest

import kv4_oracle as ko


def test_a_freed_rope_is_refused(rc):
    """Its handle is NULL, which in the C call means keys as they are."""
    kv = object.__new__(rc.Kv4)
    kv.handle = None
    rope = rc.Rope(64)
    rope.free()
    with pytest.raises(rc.RabbitCudaError, match="freed") as e:
        kv.append_dev(0, rc.F32, 1, 1, 1, 1, rope=rope, d_positions=1)
    assert e.value.status == rc.ERR_ARGS
