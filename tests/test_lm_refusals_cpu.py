"""Calls of the attention over selected blocks that are refused before anything reaches a device."""
import ctypes as C
import math

import pytest

from test_lm_cpu import P, _good, lib  # noqa: F401


@pytest.mark.parametrize("change", [dict(heads=2050, kv_heads=2), dict(scale=math.nan), dict(scale=math.inf), dict(scale=-math.inf)])
def test_refused_groups_and_scales(lib, change):
    a = _good(**change)
    assert lib.nsparse_lm_block_attention(C.byref(a), P, P, P, P, P, P, None) == -1
    assert lib.nsparse_lm_block_attention_bwd_workspace(C.byref(a)) == -1
    assert lib.nsparse_lm_last_error_string()
