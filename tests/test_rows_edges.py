"""The row operators at the ends of their arguments (CPU)."""

import pytest

from tace_amd import _native as N


@pytest.mark.parametrize("ty", range(4))
def test_workspace_is_asked_for_wherever_one_is_needed(ty):
    """0 bytes for the form that looks through all tokens, and only for it; rows of one or two elements need few."""
    L = N.lib()
    for n in (1, 100, 1000, 2049, 4096, 4097, 70000):
        for V in (1, 2, 128, 129, 1024, 1025, 2000):
            for C in (1, 2, 3, 64):
                assert L.tace_embed_grad_work(ty, n, V, C, 1) > 0
                none = n <= 4096 and V <= 1024
                if none or not L.tace_embed_grad_grouped(n, V):
                    assert (L.tace_embed_grad_work(ty, n, V, C, 0) == 0) == none


def test_no_rows_need_no_grouping():
    """A gradient of no rows takes neither a grouping nor a workspace, whatever the table's size."""
    L = N.lib()
    for V in (0, 1, 9, 128, 129, 1024, 1025, 32640, 32641, 2 ** 31 - 8193):
        assert L.tace_embed_grad_grouped(0, V) == 0, V
        assert L.tace_embed_grad_work(0, 0, V, 4, 0) == 0
    assert L.tace_embed_grad(0, 8, None, None, None, None, 0, 5000, 4, 1.0, None, None, 0, None) < 0
    assert b"null" in L.tace_last_error()   # (the gradient itself is what is missing)
