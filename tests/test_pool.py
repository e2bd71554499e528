"""A step's plan without a GPU: what is refused, and the tests' own oracle of whose
pages it hands out and takes back."""

from __future__ import annotations

import numpy as np
import pytest

from tests import step_ref as ref
from tests.test_kv4 import last_error
from tests.test_step import plan_call, pool

NONE = ref.NONE


def test_tables_past_32_bit_sums_are_refused():
    """Lengths past the table would give back every entry: their number has to stay in 32 bits."""
    for n, width in [(1024, (1 << 21) + 1), (1024, 1 << 22), (64, (1 << 25) + 1)]:
        assert plan_call(pool(n=n, width=width)) == -1
        assert "2^31 entries" in last_error()
    # (as many as may be: the next check speaks)
    assert plan_call(pool(n=1024, width=1 << 21), rows=1 << 21) == -1 and "2^21 - 1 rows" in last_error()


def plan(table, length, free, keep, own, want, rows=40, page=16, pages=24):
    stack = np.full(pages, NONE, np.uint32)
    stack[:len(free)] = free
    return ref.plan(np.asarray(table, np.uint32), length, stack, len(free), keep, own, want, rows, page, pages)


@pytest.mark.parametrize("keep,own,length,rows,slots", [
    (20, 2, 40, 0, []),              # inside another's page 8
    (33, 2, 40, 2, [145, 146]),      # inside its own page 9
    (32, 2, 40, 2, [144, 145]),      # at the border: page 9 goes back and is the first to be taken
    (16, 2, 40, 2, [144, 145]),      # a page of its own in the place of another's
])
def test_oracle_has_no_row_in_anothers_page(keep, own, length, rows, slots):
    t, ln, _, _, start, _, slot = plan([[7, 8, 9, NONE]], [length], [1, 2, 3], [keep], [own], [2])
    assert start.tolist() == [0, rows] and slot[:rows].tolist() == slots and ln.tolist() == [keep + rows]


def test_oracle_counts_every_page_once():
    """Pages that a window has left and the caller has given back."""
    _, _, free, nf, *_ = plan([[5, NONE, NONE, 6], [NONE, 7, 8, NONE]], [60, 40], [1], [0, 0], None, [0, 0])
    assert nf.tolist() == [5, 0] and free[:5].tolist() == [1, 8, 7, 6, 5]
