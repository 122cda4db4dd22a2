"""Calls of include/nsparse_lm.h at the edges of their sizes, as far as the host decides: what has nothing to do launches nothing."""
import ctypes as C

from test_lm_cpu import P, _good, lib  # noqa: F401


def test_means_of_a_cache_whose_sequences_have_no_pages(lib):
    """No table entry, so no block: nothing is launched (a launch would fail here without a GPU, and on one read numbers of no sequence)."""
    for last in (0, 1, 100):
        a = _good(page_size=16, k_len=P, page_table=P, table_stride=0, q_rows=1)
        assert lib.nsparse_lm_block_means(C.byref(a), P, P, last, None) == 0, lib.nsparse_lm_last_error_string()


def test_refused_gradients_with_that_of_the_log_sum_exp(lib):
    a = _good()
    ref, need = C.byref(a), lib.nsparse_lm_block_attention_bwd_workspace(C.byref(a))
    for bad in (0, 1, 2, 3, 4, 5, 6, 8, 9, 10):  # all but dlse, which may be none
        args = [P] * 12
        args[bad] = None
        assert lib.nsparse_lm_block_attention_lse_bwd(ref, *args, need, None) == -1, bad
    assert lib.nsparse_lm_block_attention_lse_bwd(ref, *[P] * 12, need - 1, None) == -4
    assert lib.nsparse_lm_block_attention_lse_bwd(ref, *[P] * 11, None, need, None) == -4


def test_scales_whose_base_2_form_overflows(lib):
    """Scores are scaled by scale log2 e: where that is infinite, scores of 0 would be no numbers."""
    size = lambda x: lib.nsparse_lm_block_attention_bwd_workspace(C.byref(_good(scale=x)))
    assert size(2.3e38) > 0 and size(-2.3e38) > 0 and size(0.0) > 0
    assert size(2.4e38) == -1 and size(-2.4e38) == -1 and size(3.4e38) == -1
