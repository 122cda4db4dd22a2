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


@pytest.mark.parametrize("change", [dict(k_rows=2 ** 31 - 4096, n_seq=1), dict(q_rows=2 ** 30, n_seq=1), dict(page_size=16, k_len=P, page_table=P, k_rows=2 ** 31)])
def test_refused_sizes(lib, change):
    a = _good(**change)
    assert lib.nsparse_lm_block_attention(C.byref(a), P, P, P, P, P, P, None) == -1


def test_refused_rows_of_tokens(lib):
    most = 2 ** 28
    assert lib.nsparse_lm_gather_tokens(0, P, P, 1, 1, most + 1, P, None) == -1
    assert lib.nsparse_lm_combine_tokens(0, P, P, P, 1, 1, most + 1, P, None) == -1
    assert lib.nsparse_lm_combine_tokens_bwd(0, P, P, P, P, 1, 1, most + 1, P, P, None) == -1
    for dtype, off in ((0, 2), (1, 1), (2, 1)):
        assert lib.nsparse_lm_gather_tokens(dtype, P + off, P, 4, 2, 8, P, None) == -3
        assert lib.nsparse_lm_combine_tokens(dtype, P, P, P, 4, 2, 8, P + off, None) == -3
        assert lib.nsparse_lm_combine_tokens_bwd(dtype, P, P + off, P, P, 4, 2, 8, P, P, None) == -3


def test_cut_page_tables():
    torch = pytest.importorskip("torch")
    from nsparse_amd import lm
    wide = torch.zeros(4, 10, dtype=torch.int32)
    n = torch.zeros(4, dtype=torch.int32)
    lm.Seqs(4, k_len=n, page_table=wide[:, :6])
    with pytest.raises(ValueError):
        lm.Seqs(4, k_len=n, page_table=wide[:, 4:])  # the last row's end is behind the tensor's
    with pytest.raises(ValueError):
        lm.Seqs(4, k_len=n, page_table=wide[:1].expand(4, 10))
