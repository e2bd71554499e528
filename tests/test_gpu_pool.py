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


def once(table, length, page, free, nfree, pages, shared=()):
    """Every page is in one place: an entry that a sequence holds, or free (`shared`: known to be in several)."""
    held = [int(x) for b in range(len(length)) for x in table[b, :-(-int(length[b]) // page)] if x < pages and x not in shared]
    np.testing.assert_array_equal(np.sort(held + [int(x) for x in free[:nfree]]), np.setdiff1d(np.arange(pages), list(shared)))


def release(table, length, free, nfree, b, page, window, sinks, first=0):
    """What a caller does with the pages of sequence b that no later row of it sees, on host copies."""
    low = max(int(length[b]) - window + 1, 0) // page  # the next row's window begins in this entry
    for e in range(max(-(-sinks // page), first), low):
        if table[b, e] != NONE:
            free[nfree] = table[b, e]
            table[b, e] = NONE
            nfree += 1
    return nfree


@pytest.mark.parametrize("n,page,window,sinks", [(1, 16, 30, 20), (6, 16, 40, 0), (70, 16, 16, 33), (300, 32, 100, 5)])
def test_windows_give_pages_back(have_gpu, n, page, window, sinks):
    """Sequences grow, the caller gives back what their windows have left, they end and others begin in
    their place: every page is in one place after every step, and none that is gone is handed out."""
    import torch

    rng = np.random.default_rng(n)
    width = 40
    pages = n * (-(-(window + sinks) // page) + 6)
    table, length = np.full((n, width), NONE, np.uint32), np.zeros(n, np.uint32)
    free, nfree = np.arange(pages, dtype=np.uint32), pages
    p = Pool(table, length, free, nfree, page, pages, 80 * n)
    back = served = 0
    for step in range(14):
        keep = np.where(rng.random(n) < 0.15, 0, np.maximum(length.astype(np.int64) - rng.integers(0, 3, n), 0))
        want = rng.integers(0, 70, n)
        args = [keep, None if step % 2 else np.zeros(n), want]
        p.plan(want, *args[:2])
        now = ref.plan(table, length, free, nfree, keep, None, want, 80 * n, page, pages)
        same(p.state(), now)
        table, length, free, (nfree, _), start, _, slot = now
        nfree = int(nfree)
        served += int(start[-1])
        assert np.all(slot[:start[-1]] < pages * page)
        once(table, length, page, free, nfree, pages)
        was = nfree
        for b in range(n):
            nfree = release(table, length, free, nfree, b, page, window, sinks)
        back += nfree - was
        once(table, length, page, free, nfree, pages)
        for t, a in ((p.table, table), (p.free, free), (p.nfree, np.array([nfree, 0], np.uint32))):
            t.t[64:64 + t.n].copy_(torch.from_numpy(np.ascontiguousarray(a, np.uint32).view(np.int32).ravel()))
    assert back > n and served > 100 * n ** 0.5
    p.plan(np.zeros(n), np.zeros(n))
    st = p.state()
    assert st[3].tolist() == [pages, 0] and np.all(st[0] == NONE)
    np.testing.assert_array_equal(np.sort(st[2]), np.arange(pages))


@pytest.mark.parametrize("n,width", [(1, 3000), (40, 200), (1024, 9)])
def test_many_entries_that_name_no_page(have_gpu, n, width):
    """More entries given back than threads, any of them without a page: none, some, all; and pages of
    another's before them."""
    for share in (0.0, 0.4, 1.0):
        rng = np.random.default_rng(n + int(10 * share))
        length = rng.integers((width - 2) * 16, width * 16, n)
        own = np.where(rng.random(n) < 0.3, rng.integers(0, 4, n), 0)
        pages = n * width + 50
        table = rng.permutation(pages)[:n * width].reshape(n, width).astype(np.uint32)
        lost = rng.random((n, width)) < share
        table[lost] = rng.choice([NONE, pages, pages + 7, 0xFFFFFFF0], lost.sum())
        keep = np.where(rng.random(n) < 0.6, 0, length - rng.integers(0, 40, n))
        free = np.setdiff1d(np.arange(pages), table)[:50]
        step(table, length, free, keep, own, rng.integers(0, 30, n), rows=30 * n, pages=pages)


def test_first_pages_of_anothers_and_a_gap(have_gpu):
    """A request behind another's two pages whose window has left three of its own: at its end the rest
    of its own go back, the two stay."""
    table = [[7, 8, 3, NONE, NONE, NONE, 5, 6], [7, 8, 9, NONE, NONE, NONE, NONE, NONE]]
    t, ln, free, nf, start, _, slot = step(table, [118, 40], [1, 2], [0, 40], [2, 2], [0, 20], pages=12)
    assert nf.tolist() == [4, 0] and free[:4].tolist() == [1, 2, 6, 5] and start.tolist() == [0, 0, 20]
    assert t[0].tolist() == [7, 8] + [NONE] * 6 and t[1, :4].tolist() == [7, 8, 9, 3] and slot[8] == 3 * 16
