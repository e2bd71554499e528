"""Attention over the 4-bit cache where a row sees a part of its sequence
(chk_attn_window_q4) or shares what it sees (chk_attn_prefix_q4), without a GPU:
refusals, and the cut of the work as its host views have it - every token that a
row sees is in one part of one walk, and what a call launches and keeps room for
holds all of them."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from tests.test_kv4 import batch_of, cache_struct, last_error, seqs_struct

TILE = 64
NONE = 0xFFFFFFFF


def shared_struct(groups=1, first=4096, tokens=4096):
    return abi.ChkKvShared(first, tokens, groups)


def window_call(c, s, q=8192, nh=4, gated=0, dtype=0, q_stride=512, window=5, sinks=0, out=1 << 20, out_stride=512, ws=4096,
                ws_bytes=1 << 40):
    return abi.lib().chk_attn_window_q4(c and C.byref(c), s and C.byref(s), q, nh, gated, dtype, q_stride, window, sinks, out,
                                        out_stride, ws, ws_bytes, None)


def prefix_call(c, s, q=8192, nh=4, gated=0, dtype=0, q_stride=512, shared=shared_struct(), out=1 << 20, out_stride=512, ws=4096,
                ws_bytes=1 << 40):
    return abi.lib().chk_attn_prefix_q4(c and C.byref(c), s and C.byref(s), q, nh, gated, dtype, q_stride,
                                        shared and C.byref(shared), out, out_stride, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [window_call, prefix_call])
def test_bad_calls_are_refused(call):
    c, s = cache_struct(), seqs_struct()
    for kw, msg in [(dict(q=None), "null q"), (dict(out=None), "null out"), (dict(q=8200), "q rows"), (dict(out=8200), "out rows"),
                    (dict(q_stride=511), "q rows"), (dict(q_stride=508), "shorter"), (dict(out_stride=508), "shorter"),
                    (dict(gated=1), "shorter"), (dict(nh=3), "multiple"), (dict(nh=5000), "4096"), (dict(dtype=7), "dtype"),
                    (dict(ws=None), "workspace"), (dict(ws=4104), "workspace"), (dict(ws_bytes=8), "workspace")]:
        assert call(c, s, **kw) == -1
        assert msg in last_error(), (kw, last_error())
    assert call(None, s) == -1 and "no cache" in last_error()
    assert call(c, None) == -1 and "no sequences" in last_error()
    assert call(cache_struct(hd=64), s) == -1 and "head_dim" in last_error()
    assert call(c, seqs_struct(n=1025)) == -1 and "1024 sequences" in last_error()
    # no rows: nothing to do, and nothing needed
    none = abi.ChkKvSeqs(None, None, None, 0, 0, 0)
    assert call(c, none, q=None, out=None, ws=None, ws_bytes=0) == 0


def test_bad_views_are_refused():
    c, s = cache_struct(), seqs_struct()
    assert window_call(c, s, window=0) == -1 and "at least one token" in last_error()
    for kw, msg in [(dict(groups=1025), "1024 groups"), (dict(first=None), "null or misaligned first"),
                    (dict(tokens=None), "null or misaligned"), (dict(first=4098), "misaligned"), (dict(tokens=4097), "misaligned")]:
        assert prefix_call(c, s, shared=shared_struct(**kw)) == -1
        assert msg in last_error(), (kw, last_error())
    assert prefix_call(c, s, shared=None) == -1 and "no shared" in last_error()
    n = C.c_uint64()
    for args, msg in [((4, 3, 128, 1, 1, 1), "multiple"), ((4, 2, 64, 1, 1, 1), "head_dim"), ((4, 2, 128, 1025, 1, 1), "sequences"),
                      ((4, 2, 128, 1, 1, 1025), "groups")]:
        assert abi.lib().chk_attn_prefix_q4_workspace(*args, C.byref(n)) == -1
        assert msg in last_error()
    assert abi.lib().chk_attn_prefix_q4_workspace(4, 2, 128, 1, 1, 1, None) == -1


def test_memory_that_is_not_the_devices_is_refused():
    buf = np.zeros(1 << 16, np.uint8)
    at = (buf.ctypes.data + 255) & ~255
    c, s = cache_struct(ptr=at), seqs_struct(ptr=at)
    assert window_call(c, s, q=at, out=at, ws=at) == -1 and "device" in last_error()
    assert prefix_call(c, s, q=at, out=at, ws=at, shared=shared_struct(1, at, at)) == -1 and "device" in last_error()


# ---- the cut through a window


def window_cut(nh, nkv, hd, dtype, groups, lens, start, rows, tokens, window, sinks):
    n = len(lens)
    cut, launch = np.zeros((max(n, 1), 4), np.uint32), np.zeros(4, np.uint64)
    lens, start = np.asarray(lens, np.uint32), np.asarray(start, np.uint32)
    assert abi.lib().chk_attn_window_q4_cut(nh, nkv, hd, dtype, groups, n, rows, tokens, lens.ctypes.data, start.ctypes.data, window,
                                            sinks, cut.ctypes.data, launch.ctypes.data) == 0, last_error()
    return cut[:n].astype(np.int64), launch.astype(np.int64)


SHAPES = [(16, 2, 256, 0), (32, 8, 128, 2), (1, 1, 128, 1), (40, 1, 256, 2), (130, 1, 128, 2)]


@pytest.mark.parametrize("groups", [1, 16, 512])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_windows_cut_covers_its_tiles_and_fits_its_launches(groups, shape):
    nh, nkv, hd, dtype = shape
    group = nh // nkv
    for seed in range(60):
        rng = np.random.default_rng(seed)
        lens, rows = batch_of(rng)
        start = np.concatenate([[0], np.cumsum(rows)])
        total = int(start[-1])
        if total == 0 or total * nh > 2**28:
            continue
        window = int(rng.choice([1, 5, 63, 64, 65, 1000, 2**31]))
        sinks = int(rng.choice([0, 1, 64, 65, 500, 2**31]))
        cut, (cap, few, many, joins) = window_cut(nh, nkv, hd, dtype, groups, lens, start, total, int(max(lens.max(), 1)), window,
                                                  sinks)
        used, items, joined = 0, [0, 0], 0
        for length, n, (block, blocks, piece, parts) in zip(lens, rows, cut):
            flat, length, n = int(n) * group, int(length), int(n)
            assert blocks * block >= flat > (blocks - 1) * block or flat == blocks == 0
            if flat == 0:
                continue
            for blk in {0, blocks // 2, blocks - 1}:
                m0, m1 = int(blk * block), int(min((blk + 1) * block, flat)) - 1
                p0, p1 = length - n + m0 // group, length - n + m1 // group
                # tiles that hold a token which one of the block's rows sees
                seen = -(-(p1 + 1) // TILE) if p1 >= 0 else 0
                low = max(p0 - window + 1, 0) // TILE
                tiles = min(-(-sinks // TILE), low, seen) + max(seen - low, 0)
                own = max(-(-tiles // piece), 1)
                assert own <= parts and own * -(-tiles // own) >= tiles
            items[int(flat > 64)] += int(blocks) * nkv * int(parts)
            if parts > 1:
                used += flat * nkv * int(parts)
                joined += flat * nkv
        assert used <= cap and joined <= joins, (seed, used, cap)
        assert items[0] <= few and items[1] <= many, (seed, items, few, many)


def test_a_wide_window_is_cut_as_none():
    """Few pairs: the same parts; and the host views' own refusals."""
    lens, start = np.array([5000, 900, 3], np.uint32), np.array([0, 1, 4, 5], np.uint32)
    cut, launch = np.zeros((3, 4), np.uint32), np.zeros(4, np.uint64)
    args = (8, 2, 128, 0, 512, 3, 5, 8192, lens.ctypes.data, start.ctypes.data)
    assert abi.lib().chk_attn_q4_cut(*args, cut.ctypes.data, launch.ctypes.data) == 0
    got, at = window_cut(8, 2, 128, 0, 512, lens, start, 5, 8192, 8192, 0)
    assert np.array_equal(got, cut) and np.array_equal(at, launch)
    assert abi.lib().chk_attn_window_q4_cut(*args, 0, 3, cut.ctypes.data, launch.ctypes.data) == -1
    assert "at least one token" in last_error()
    assert abi.lib().chk_attn_window_q4_cut(*args, 1, 3, None, launch.ctypes.data) == -1


# ---- and with shared prefixes


def prefix_cut(nh, nkv, hd, dtype, groups, lens, start, rows, tokens, first, shared):
    n = len(lens)
    walks, launch = np.zeros((max(len(shared) + n, 1), 8), np.uint32), np.zeros(4, np.uint64)
    lens, start, first, shared = (np.asarray(a, np.uint32) for a in (lens, start, first, shared))
    s = abi.ChkKvShared(first.ctypes.data, shared.ctypes.data, len(shared))
    assert abi.lib().chk_attn_prefix_q4_cut(nh, nkv, hd, dtype, groups, n, rows, tokens, lens.ctypes.data, start.ctypes.data,
                                            C.byref(s), walks.ctypes.data, launch.ctypes.data) == 0, last_error()
    return walks[:len(shared) + n].astype(np.int64), launch.astype(np.int64)


def prefix_batch(rng):
    """Groups of a batch, with others between and behind them, in any state."""
    lens, rows = batch_of(rng)
    n = len(lens)
    g = int(rng.integers(1, min(n, 5) + 1))
    first = np.sort(rng.integers(0, n + 1, g + 1))
    shared = rng.integers(0, 3 * max(int(lens.max()), 64), g)
    if rng.random() < 0.7:  # lengths that hold their prefix
        for i in range(g):
            shared[i] = rng.integers(64, 5000)
            b = slice(first[i], first[i + 1])
            lens[b] += shared[i]
            rows[b] = np.minimum(rows[b], lens[b])
    if rng.random() < 0.2:
        first[-1] = n + 7
    return lens, rows, first, shared


@pytest.mark.parametrize("groups", [1, 16, 512])
@pytest.mark.parametrize("shape", SHAPES)
def test_walks_cover_every_tile_once_and_fit_their_launches(groups, shape):
    nh, nkv, hd, dtype = shape
    group = nh // nkv
    together = 0
    for seed in range(80):
        rng = np.random.default_rng(seed)
        lens, rows, first, shared = prefix_batch(rng)
        n = len(lens)
        tokens = int(max(lens.max(), 1)) - (int(rng.integers(0, 2)) if seed % 9 == 0 else 0)
        tokens = max(tokens, 1)
        held = lens <= tokens
        start = np.concatenate([[0], np.cumsum(rows)])
        total = int(start[-1])
        if total == 0 or total * nh > 2**28:
            continue
        walks, (cap, few, many, joins) = prefix_cut(nh, nkv, hd, dtype, groups, lens, start, total, tokens, first, shared)
        used, items, joined = 0, [0, 0], 0
        for v, (s0, k, length, lo, of, block, piece, parts) in enumerate(walks):
            whole = v < len(shared)
            b = v - len(shared)
            if whole:
                if k == 0:
                    continue
                together += 1
                assert length % TILE == 0 and 0 < length <= shared[v] and lo == 0 and of == NONE
                mine = [b for b in range(min(first[v], n), min(first[v + 1], n)) if walks[len(shared) + b][4] == v]
                assert len(mine) >= 2
                assert s0 == min(start[b] for b in mine) and s0 + k == max(start[b + 1] for b in mine)
                assert all(length <= lens[b] - rows[b] + 1 and held[b] for b in mine)  # every row sees all of it
            else:
                assert (s0, k, length) == (start[b], rows[b], lens[b] if held[b] else 0)
                if of != NONE:
                    assert first[of] <= b < first[of + 1] and lo == walks[of][2] // TILE and walks[of][1] > 0 and k > 0
                else:
                    assert lo == 0
            flat = int(k) * group
            if flat == 0:
                continue
            blocks = -(-flat // int(block))
            for m1 in (min(block, flat) - 1, flat - 1):
                seen = int(length) if whole else int(length) - int(k) + int(m1) // group + 1
                tiles = max(-(-max(seen, 0) // TILE) - int(lo), 0) if whole or held[b] else 0
                own = max(-(-tiles // int(piece)), 1)
                assert own <= parts and own * -(-tiles // own) >= tiles
            assert own == parts
            items[int(block > 16)] += blocks * nkv * int(parts)
            if whole or of != NONE or parts > 1:
                used += flat * nkv * int(parts)
                joined += 0 if whole else flat * nkv
        assert used <= cap and joined <= joins, (seed, used, cap, joined, joins)
        assert items[0] <= few and items[1] <= many, (seed, items, few, many)
    assert together > 5


def test_without_a_prefix_the_cut_is_plain():
    lens, start = [5000, 900, 3, 300], [0, 1, 4, 5, 105]
    cut, launch = np.zeros((4, 4), np.uint32), np.zeros(4, np.uint64)
    le, st = np.asarray(lens, np.uint32), np.asarray(start, np.uint32)
    assert abi.lib().chk_attn_q4_cut(8, 2, 128, 0, 512, 4, 105, 8192, le.ctypes.data, st.ctypes.data, cut.ctypes.data,
                                     launch.ctypes.data) == 0
    for first, shared in [([0], []), ([0, 4], [0]), ([0, 4], [63]), ([0, 1, 2, 3, 4], [640, 640, 640, 640])]:
        walks, _ = prefix_cut(8, 2, 128, 0, 512, lens, start, 105, 8192, first, shared)
        assert np.array_equal(walks[len(shared):][:, 5:], cut[:, [0, 2, 3]])
        assert np.all(walks[len(shared):][:, 4] == NONE)


def test_prefix_cut_refusals():
    z = np.zeros(64, np.uint64)
    p = z.ctypes.data
    s = abi.ChkKvShared(p, p, 1)
    ok = [4, 2, 128, 0, 512, 1, 1, 64, p, p, C.byref(s), p, p]
    assert abi.lib().chk_attn_prefix_q4_cut(*ok) == 0
    for i, v, msg in [(10, None, "groups"), (10, C.byref(abi.ChkKvShared(None, p, 1)), "null first"), (11, None, "null"),
                      (10, C.byref(abi.ChkKvShared(p, p, 1025)), "1024 groups"), (2, 64, "head_dim")]:
        assert abi.lib().chk_attn_prefix_q4_cut(*(ok[:i] + [v] + ok[i + 1:])) == -1
        assert msg in last_error()
