"""Drafted tokens without a GPU: trees on the host."""
from __future__ import annotations


def test_lines_of_parents():
    from sparse_decode.paged import _lines
    assert _lines([]) == [] and _lines([-1, 0, 0, 1, -2, 4, -1]) == [1, 3, 5, 11, 0, 0, 64]
    assert _lines(list(range(-1, 63)))[-1] == (1 << 64) - 1
