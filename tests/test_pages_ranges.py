"""Paged history, host side: calls of more rows or entries than a grid takes are refused before
anything is launched."""
import pytest

from test_pages import FAKE, RANGE, book, lib  # noqa: F401

MOST = (1 << 24) - 1
BIG = 1 << 40


@pytest.mark.parametrize("rows", [MOST + 1, 1 << 25, 2**31 - 1])
def test_more_rows_than_a_grid_takes(lib, rows):  # noqa: F811
    b = book(kv_heads=1, head_dim=64)
    for seqs, cu, n in ((None, None, rows), (FAKE, None, rows), (None, FAKE, 4)):
        assert lib.rta_paged_append(b, 0, FAKE, 64, FAKE, 64, rows, seqs, cu, n, None) == RANGE
        assert lib.rta_paged_read(b, 0, rows, seqs, cu, n, FAKE, 64, None, 0, None) == RANGE
        for most in ((1, 5) if cu else (1,)):
            assert lib.rta_paged_attention(b, 0, FAKE, 64, rows, 1, seqs, cu, n, most, 0, 0, 0, None, FAKE, None, None, FAKE,
                                           BIG, None) == RANGE


@pytest.mark.parametrize("n", [MOST + 1, 2**31 - 1])
def test_more_entries_than_a_grid_takes(lib, n):  # noqa: F811
    b = book()
    assert lib.rta_pages_fork(b, FAKE, FAKE, n, None) == RANGE
    assert lib.rta_pages_free(b, FAKE, FAKE, FAKE, n, None) == RANGE
    assert lib.rta_pages_free(b, None, None, None, n, None) == RANGE
