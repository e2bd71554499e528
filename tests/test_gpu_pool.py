"""Whose pages a step's plan hands out and takes back (chk_kv_plan_q4): no row in a page
that is another's, every page held once."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd.abi import lib
from tests import step_ref as ref
from tests.test_gpu_step import Pool, same

pytestmark = pytest.mark.gpu

NONE = ref.NONE


def step(table, length, free, keep, own, want, rows=40, page=16, pages=24):
    """One plan of a state, compared with the rules; (table, len, free, nfree, start, pos, slot)."""
    table = np.asarray(table, np.uint32)
    stack = np.full(pages, NONE, np.uint32)
    stack[:len(free)] = free
    p = Pool(table, length, stack, len(free), page, pages, rows)
    p.plan(want, keep, own)
    got = p.state()
    same(got, ref.plan(table, length, stack, len(free), keep, own, want, rows, page, pages))
    return got


def test_no_row_in_anothers_page(have_gpu):
    """Two pages of another's, 40 tokens cut back into the second of them, behind it, to where it
    begins, and below both; and a fork that counts a last page that is not full."""
    for keep, own, length, served in [
            (20, 2, 40, False),   # token 20 would lie in page 8
            (31, 2, 40, False), (33, 2, 40, True), (32, 2, 40, True), (40, 3, 40, False), (40, 2, 40, True),
            (16, 2, 40, True),    # entry 1 is a page of its own from here on
            (1, 2, 40, False), (0, 2, 40, True), (5, 1, 5, False), (5, 0, 5, True), (NONE, 3, 40, False)]:
        t, ln, _, nf, start, pos, slot = step([[7, 8, 9, NONE]], [length], [1, 2, 3], [keep], [own], [2])
        left = min(keep, length)
        assert start.tolist() == [0, 2 if served else 0] and ln.tolist() == [left + (2 if served else 0)], (keep, own)
        kept = min(own, -(-left // 16))  # entries of another's that the sequence still begins with
        assert t[0, :kept].tolist() == [7, 8, 9][:kept]
        if served:
            assert not np.isin(slot[:2] // 16, [7, 8][:own]).any(), (keep, own, slot[:2])
        else:
            assert pos[0] == NONE and slot[0] == 2**64 - 1


def test_a_refused_sequence_takes_nothing_from_the_others(have_gpu):
    """Neither room in the row arrays nor a page; and the copied page, with a lower own, serves it."""
    table = [[7, 8, NONE], [10, NONE, NONE], [11, 12, NONE]]
    args = dict(rows=20, page=16)
    _, ln, _, nf, start, _, _ = step(table, [20, 16, 18], [1, 2], None, [2, 0, 1], [18, 17, 3], **args)
    assert start.tolist() == [0, 0, 17, 20] and ln.tolist() == [20, 33, 21] and nf.tolist() == [0, 0]
    table[0][1] = 13
    t, _, _, _, start, _, slot = step(table, [20, 16, 18], [1, 2], None, [1, 0, 1], [18, 0, 2], **args)
    assert start.tolist() == [0, 18, 18, 20] and slot[:18].tolist() == [13 * 16 + 4 + i for i in range(12)] + [2 * 16 + i for i in range(6)]


@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("n", [1, 64, 200, 1024])
def test_no_slot_names_anothers_page(have_gpu, n, page):
    """Any lengths, cuts and shares of pages that are another's."""
    rng = np.random.default_rng(n + page)
    length = rng.integers(0, 5 * page, n)
    held = -(-length // page)
    own = rng.integers(0, held + 1)
    keep = np.where(rng.random(n) < 0.5, NONE, (length * rng.random(n)).astype(np.int64))
    keep = np.where(rng.random(n) < 0.2, np.minimum(own, length // page) * page, keep)
    want = rng.integers(0, 9, n)
    pages = int(held.sum()) + 2 * n
    ids = rng.permutation(pages)
    table = np.full((n, 8), NONE, np.uint32)
    for b in range(n):
        at = held[:b].sum()
        table[b, :held[b]] = ids[at:at + held[b]]
    got = step(table, length, ids[held.sum():held.sum() + n], keep, own, want, rows=int(want.sum()), page=page, pages=pages)
    start, slot = got[4], got[6]
    refused = 0
    for b in range(n):
        theirs = table[b, :own[b]]
        s = slot[start[b]:start[b + 1]] // np.uint64(page)
        assert not np.isin(s, theirs).any(), b
        left = min(int(keep[b]), int(length[b]))
        refused += want[b] > 0 and left % page != 0 and left // page < own[b]
    assert refused or n == 1
