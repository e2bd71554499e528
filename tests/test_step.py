"""A serving step's calls around the 4-bit cache without a GPU: their refusals,
the rotation's table, and the plan's rules as the tests' own oracle has them."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from tests import step_ref as ref
from tests.test_kv4 import last_error

FAKE = 1 << 20  # an aligned address that no call may reach


def pool(n=2, width=3, page=16, pages=9, **at):
    p = {k: at.get(k, FAKE) for k in ("table", "len", "free", "nfree")}
    return abi.ChkKvPool(p["table"], p["len"], p["free"], p["nfree"], n, width, page, pages)


def plan_call(p, keep=None, own=None, want=FAKE, rows=5, start=FAKE, pos=FAKE, slot=FAKE):
    return abi.lib().chk_kv_plan_q4(p and C.byref(p), keep, own, want, rows, start, pos, slot, None)


def test_bad_plans_are_refused():
    for kw, msg in [(dict(n=1025), "1024 sequences"), (dict(page=24), "power of two"), (dict(page=8), "power of two"),
                    (dict(page=1 << 21), "power of two"), (dict(pages=0), "at least one page"),
                    (dict(pages=0xFFFFFFFF), "at least one page"), (dict(width=(1 << 26) + 1), "2^30 tokens"),
                    (dict(width=0), "at least one page"), (dict(n=0), "rows without a sequence"),
                    (dict(table=None), "null table"), (dict(len=None), "null table, len"), (dict(free=None), "null"),
                    (dict(nfree=None), "null"), (dict(table=FAKE + 2), "4-byte"), (dict(nfree=FAKE + 1), "4-byte")]:
        assert plan_call(pool(**kw)) == -1
        assert msg in last_error(), (kw, last_error())
    for kw, msg in [(dict(rows=1 << 21), "2^21 - 1 rows"), (dict(want=None), "null want"), (dict(start=None), "null want or start"),
                    (dict(keep=FAKE + 2), "4-byte"), (dict(own=FAKE + 2), "4-byte"), (dict(pos=FAKE + 2), "4-byte"),
                    (dict(slot=FAKE + 4), "8-byte")]:
        assert plan_call(pool(), **kw) == -1
        assert msg in last_error(), (kw, last_error())
    assert plan_call(None) == -1 and "no pool" in last_error()
    # no sequences: nothing to do
    assert plan_call(pool(n=0, width=0, table=None, len=None, free=None, nfree=None), want=None, rows=0, start=None) == 0


def test_host_memory_is_refused():
    buf = np.zeros(1 << 14, np.uint8)
    at = (buf.ctypes.data + 255) & ~255
    assert plan_call(pool(table=at, len=at, free=at, nfree=at), want=at, start=at, pos=at, slot=at) == -1
    assert "device" in last_error()
    assert norm_call(norm(q_norm=at, k_norm=at, turn=at), pos=at, q=at, q_out=at, k=at, k_out=at) == -1
    assert "device" in last_error()


def norm(rot=32, nh=4, nkv=2, hd=128, gated=0, eps=1e-6, **at):
    return abi.ChkQkNorm(*(at.get(k, FAKE) for k in ("q_norm", "k_norm", "turn")), rot, nh, nkv, hd, gated, eps)


def norm_call(n, pos=FAKE, rows=3, q=FAKE, q_stride=512, q_out=FAKE, q_out_stride=512, k=FAKE, k_stride=256, k_out=FAKE,
              k_out_stride=256, dtype=0):
    return abi.lib().chk_qk_norm_rope(n and C.byref(n), pos, rows, q, q_stride, q_out, q_out_stride, k, k_stride, k_out,
                                      k_out_stride, dtype, None)


def test_bad_norms_are_refused():
    for kw, msg in [(dict(hd=96), "head_dim"), (dict(hd=512), "head_dim"), (dict(nh=0, nkv=0), "heads"), (dict(nh=4097), "heads"),
                    (dict(nkv=4097), "heads"), (dict(rot=3), "rot must be even"), (dict(rot=130), "rot must be even"),
                    (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                    (dict(eps=float("inf")), "eps"), (dict(q_norm=FAKE + 1), "misaligned norm"),
                    (dict(turn=None), "null or misaligned turn"), (dict(turn=FAKE + 4), "null or misaligned turn"),
                    (dict(gated=1), "q row stride shorter")]:
        assert norm_call(norm(**kw)) == -1
        assert msg in last_error(), (kw, last_error())
    for kw, msg in [(dict(rows=(1 << 25) + 1), "2^25 rows"), (dict(pos=None), "pos"), (dict(pos=FAKE + 2), "pos"),
                    (dict(q=None), "null q"), (dict(q_out=None), "null q_out"), (dict(k=None), "null k"),
                    (dict(k_out=None), "null k_out"), (dict(q=FAKE + 8), "q rows must be"), (dict(k_out=FAKE + 4), "k_out rows"),
                    (dict(q_stride=508), "q row stride"), (dict(k_out_stride=252), "k_out row stride"),
                    (dict(q_out_stride=514), "q_out rows must be"), (dict(q_out_stride=1024), "keep its stride"),
                    (dict(k_stride=512), "keep its stride"), (dict(dtype=3), "dtype")]:
        assert norm_call(norm(), **kw) == -1
        assert msg in last_error(), (kw, last_error())
    assert norm_call(norm(nh=4096, nkv=4096), rows=1 << 16) == -1 and "2^28" in last_error()
    assert norm_call(None) == -1 and "no norm" in last_error()
    # no rows: nothing to do, nothing needed
    assert norm_call(norm(), rows=0, pos=None, q=None, q_out=None, k=None, k_out=None) == 0


@pytest.mark.parametrize("theta,rot", [(1e4, 128), (1e7, 64), (1.5, 2), (5e5, 256), (1e4, 20)])
def test_turns(theta, rot):
    """theta^(-2 j / rot) / 2 pi of a turn, to 2^-60 of itself: against integers
    of 30 digits from the exponential's and logarithm's own series."""
    from decimal import Decimal, getcontext

    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    turn = (C.c_uint64 * (rot // 2))()
    assert abi.lib().chk_rope_turns(theta, rot, turn) == 0
    for j in range(rot // 2):
        want = (Decimal(theta).ln() * (Decimal(-2 * j) / Decimal(rot))).exp() / (2 * pi) * 2**64
        # the power's own error, a few of 2^-64 of it, and half a unit
        assert abs(Decimal(turn[j]) - want) <= want * Decimal(2) ** -60 + 1, j


def test_bad_turns_are_refused():
    t = (C.c_uint64 * 128)()
    for args, msg in [((1.0, 8, t), "theta"), ((0.5, 8, t), "theta"), ((float("nan"), 8, t), "theta"),
                      ((float("inf"), 8, t), "theta"), ((1e4, 7, t), "rot"), ((1e4, 258, t), "rot"), ((1e4, 8, None), "null")]:
        assert abi.lib().chk_rope_turns(*args) == -1
        assert msg in last_error()


def test_oracle_plan_of_a_hand_worked_step():
    """Two pages free and two given back: sequence 0 drops a page and takes it
    again, 1 has room, 2 takes two, 3 needs two and finds one, 4 fits in the page
    that it holds, 5 has ended and keeps the page that is another's."""
    page, pages = 16, 20
    table = np.full((6, 4), ref.NONE, np.uint32)
    table[0, :2] = [10, 11]
    table[1, 0] = 12
    table[2, 0] = 13
    table[3, 0] = 14
    table[4, 0] = 15
    table[5, :2] = [16, 17]
    free = np.zeros(pages, np.uint32)
    free[:2] = [1, 2]
    t, ln, fr, nf, start, pos, slot = ref.plan(table, [20, 3, 16, 16, 5, 31], free, 2, [14, 99, 99, 99, 99, 0],
                                               [0, 0, 0, 0, 0, 1], [3, 2, 17, 17, 1, 0], 40, page, pages)
    # the stack: 1 2, then the last sequence's page 17 (16 is another's), then 11
    assert ln.tolist() == [17, 5, 33, 16, 6, 0] and start.tolist() == [0, 3, 5, 22, 22, 23, 23]
    assert t[0].tolist() == [10, 11, ref.NONE, ref.NONE]  # 11 back and taken again
    assert t[2].tolist() == [13, 17, 2, ref.NONE] and t[3, 1] == ref.NONE and t[5].tolist() == [16, ref.NONE] + [ref.NONE] * 2
    assert nf.tolist() == [1, 1] and fr[0] == 1
    assert pos[:3].tolist() == [14, 15, 16] and slot[2] == 11 * 16 and pos[22] == 5 and pos[23] == ref.NONE
