"""The refusals of the products' test hooks, which need no GPU."""
from __future__ import annotations


def test_hook_arguments_are_refused(rc):
    so = rc.lib()
    for cta in (0, 1, 2, -1):
        assert so.rabbit_cuda_linear_debug_withhold_cta(None, cta) == rc.ERR_ARGS
