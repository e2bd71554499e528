"""The tiles that attention's blocks walk through a window and over shared prefixes, without a GPU: the
rules of csrc/kvq4.h compiled for the host, the parts as the kernels take them.  Every tile that holds
a token which a row of the block sees is in one part, once, and no part is empty."""

from __future__ import annotations

import ctypes as C
import subprocess

import numpy as np
import pytest

from cherenkov_amd.build import CSRC, ROOT
from tests.test_attn_views import NONE, SHAPES, TILE, prefix_batch, prefix_cut, window_cut
from tests.test_kv4 import batch_of

HOST = """
#include "kvq4.h"
using namespace chk;
// The tiles of a block's parts in turn, as the kernels go through them; their number, part ends in `ends`.
static uint32_t parts_of(Kv4Walk k, uint32_t piece, uint32_t* tiles, uint32_t* ends, uint32_t* parts) {
    *parts = kv4_parts(k.tiles, piece);
    const uint32_t per = (k.tiles + *parts - 1) / *parts, walked = k.seen > 0 ? (uint32_t)k.seen - k.gap * KV4_TILE : 0u;
    uint32_t n = 0;
    for (uint32_t z = 0; z < *parts; ++z) {
        uint32_t end = (k.tiles < (z + 1) * per ? k.tiles : (z + 1) * per) * KV4_TILE;
        if (end > walked) end = walked;
        for (uint32_t t = z * per * KV4_TILE; t < end; t += KV4_TILE)
            tiles[n++] = (t < k.head * KV4_TILE ? t : t + k.gap * KV4_TILE) / KV4_TILE;
        ends[z] = n;
    }
    return n;
}
extern "C" uint32_t through_window(uint32_t len, uint32_t n, uint32_t group, uint32_t m0, uint32_t m1, uint32_t window, uint32_t sinks,
                                   uint32_t piece, uint32_t* tiles, uint32_t* ends, uint32_t* parts) {
    return parts_of(kv4_window_walk(len, n, group, m0, m1, kv4_window(window, sinks)), piece, tiles, ends, parts);
}
extern "C" uint32_t of_walk(uint32_t len, uint32_t n, uint32_t whole, uint32_t lo, uint32_t row, uint32_t piece, uint32_t* tiles,
                            uint32_t* ends, uint32_t* parts) {
    Kv4Work w = kv4_no_work();
    w.len = len;
    w.n = n;
    w.whole = whole;
    w.lo = lo;
    Kv4Walk k;
    k.seen = whole ? (int32_t)len : (int32_t)len - (int32_t)n + (int32_t)row + 1;
    k.head = 0;
    k.gap = lo;
    k.tiles = kv4_work_tiles(w, row);
    if (k.tiles == 0) k.seen = 0;
    return parts_of(k, piece, tiles, ends, parts);
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    at = tmp_path_factory.mktemp("walks")
    (at / "walks.cpp").write_text(HOST)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT / 'include'}", f"-I{CSRC}", str(at / "walks.cpp"),
                    "-o", str(at / "walks.so")], check=True)
    return C.CDLL(str(at / "walks.so"))


def walked(fn, *args):
    tiles, ends, parts = np.zeros(1 << 16, np.uint32), np.zeros(1 << 16, np.uint32), C.c_uint32()
    n = fn(*(C.c_uint32(int(a) & 0xFFFFFFFF) for a in args), tiles.ctypes.data_as(C.c_void_p), ends.ctypes.data_as(C.c_void_p),
           C.byref(parts))
    return tiles[:n].astype(int).tolist(), ends[:parts.value].astype(int)


def visible(p0, p1, window, sinks):
    """Tiles that hold a token which a row at p0 .. p1 sees."""
    rows = range(max(p0, 0), p1 + 1)
    if not rows:
        return []
    mine = set(range(max(rows[0] - window + 1, 0) // TILE, p1 // TILE + 1))  # the rows' windows are one run
    return sorted(mine | set(range(-(-min(sinks, p1 + 1) // TILE))))


def test_visible_by_every_token():
    """The set above against each row's tokens one by one."""
    rng = np.random.default_rng(1)
    for _ in range(400):
        p0 = int(rng.integers(-5, 500))
        p1, window, sinks = p0 + int(rng.integers(0, 200)), int(rng.choice([1, 2, 63, 64, 65, 300])), int(rng.choice([0, 1, 64, 70, 900]))
        see = {t // TILE for p in range(max(p0, 0), p1 + 1) for t in range(p + 1) if t < sinks or t > p - window}
        assert visible(p0, p1, window, sinks) == sorted(see)


@pytest.mark.parametrize("groups", [16, 512, 8192])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_windows_parts_hold_every_tile_once(host, groups, shape):
    nh, nkv, hd, dtype = shape
    group = nh // nkv
    several = 0
    for seed in range(30):
        rng = np.random.default_rng(1000 + seed)
        lens, rows = batch_of(rng)
        start = np.concatenate([[0], np.cumsum(rows)])
        total = int(start[-1])
        if total == 0 or total * nh > 2**28:
            continue
        window, sinks = int(rng.choice([1, 5, 63, 64, 65, 1000, 2**31])), int(rng.choice([0, 1, 64, 65, 500, 2**31]))
        cut, _ = window_cut(nh, nkv, hd, dtype, groups, lens, start, total, int(max(lens.max(), 1)), window, sinks)
        for length, n, (block, blocks, piece, most) in zip(lens, rows, cut):
            flat = int(n) * group
            for blk in sorted({0, 1, int(blocks) // 2, int(blocks) - 1}) if flat else []:
                if not 0 <= blk < blocks:
                    continue
                m0, m1 = int(blk * block), int(min((blk + 1) * block, flat)) - 1
                tiles, ends = walked(host.through_window, length, n, group, m0, m1, window, sinks, piece)
                p = int(length) - int(n)
                assert tiles == visible(p + m0 // group, p + m1 // group, window, sinks)
                assert len(ends) <= most and (not tiles or np.all(np.diff(ends, prepend=0) > 0))
                several += len(ends) > 1
    assert several > 0 or groups < 8192


@pytest.mark.parametrize("groups", [16, 512, 8192])
@pytest.mark.parametrize("shape", SHAPES)
def test_the_walks_of_a_row_hold_every_tile_once(host, groups, shape):
    """A member's rows: the group's walk and its own together."""
    nh, nkv, hd, dtype = shape
    group = nh // nkv
    together = several = 0
    for seed in range(30):
        rng = np.random.default_rng(2000 + seed)
        lens, rows, first, shared = prefix_batch(rng)
        start = np.concatenate([[0], np.cumsum(rows)])
        total, tokens = int(start[-1]), int(max(lens.max(), 1))
        if total == 0 or total * nh > 2**28:
            continue
        walks, _ = prefix_cut(nh, nkv, hd, dtype, groups, lens, start, total, tokens, first, shared)
        for b, (s0, n, length, lo, of, block, piece, most) in enumerate(walks[len(shared):]):
            flat = int(n) * group
            blocks = -(-flat // int(block))
            before = []
            if of != NONE:
                _, k, common, _, _, _, gpiece, gmost = walks[of]
                before, ends = walked(host.of_walk, common, k, 1, 0, k - 1, gpiece)
                assert before == list(range(int(common) // TILE)) and len(ends) == gmost
                together += 1
            for blk in sorted({0, blocks // 2, blocks - 1}) if flat else []:
                m1 = int(min((blk + 1) * block, flat)) - 1
                tiles, ends = walked(host.of_walk, length, n, 0, lo, m1 // group, piece)
                p1 = int(length) - int(n) + m1 // group
                assert before + tiles == list(range(p1 // TILE + 1 if p1 >= 0 else 0)), (seed, b)
                assert len(ends) <= most and (not tiles or np.all(np.diff(ends, prepend=0) > 0))
                several += len(ends) > 1
    assert together > 5 and (several > 0 or groups < 8192)
