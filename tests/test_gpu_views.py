"""Attention over the 4-bit cache through a window and over shared prefixes on
the GPU (chk_attn_window_q4, chk_attn_prefix_q4) against plain numpy in 64 bits
(tests/view_ref.py): ragged batches of every kind of row, windows and prefixes
that end anywhere, what no row sees holding anything, states that are not sound,
graphs, streams, and a serving run of a step's calls together."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from cherenkov_amd.abi import EngineError, check, lib
from tests import kv4_ref as ref
from tests import view_ref as view
from tests.test_gpu_kv4 import KINDS, Dev, dev, random_cache, rounded, tables, torch_type

pytestmark = pytest.mark.gpu


class Views(Dev):
    def window(self, q, out, nh, gated, kind, window, sinks, ws=None, stream=None):
        self.ws = self.workspace(nh) if ws is None else ws
        check(lib().chk_attn_window_q4(C.byref(self.cache), C.byref(self.seqs), q.data_ptr(), nh, int(gated), KINDS[kind],
                                       q.stride(0), window, sinks, out.data_ptr(), out.stride(0), self.ws.data_ptr(),
                                       self.ws.numel(), stream))

    def prefix_workspace(self, nh, groups):
        import torch

        n = C.c_uint64()
        check(lib().chk_attn_prefix_q4_workspace(nh, self.host.nkv, self.host.hd, self.seqs.n, self.seqs.rows, groups, C.byref(n)))
        return torch.full((n.value,), 0xFF, dtype=torch.uint8, device="cuda")

    def share(self, first, tokens):
        self.first, self.tokens = (dev(np.asarray(a, np.uint32)) for a in (first, tokens))
        self.shared = abi.ChkKvShared(self.first.data_ptr(), self.tokens.data_ptr(), len(tokens))

    def prefix(self, q, out, nh, gated, kind, ws=None, stream=None):
        self.ws = self.prefix_workspace(nh, self.shared.groups) if ws is None else ws
        check(lib().chk_attn_prefix_q4(C.byref(self.cache), C.byref(self.seqs), q.data_ptr(), nh, int(gated), KINDS[kind],
                                       q.stride(0), C.byref(self.shared), out.data_ptr(), out.stride(0), self.ws.data_ptr(),
                                       self.ws.numel(), stream))


def close(got, want, vmax, smax, kind, hd):
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    tol = ref.tolerance(kind, hd, want, vmax, smax)
    off = np.where(nan, 0, np.abs(got - want) - np.where(nan, 0, tol))
    assert np.all(off <= 0), f"worst {off.max():.3g} over, of {np.abs(np.where(nan, 0, got - want)).max():.3g}"


def call(seed, heads, page, lens, rows, kind, gated, cache=None, window=None, share=None, tweak=None):
    """One call against the reference: window = (window, sinks) or share = (first, tokens)."""
    import torch

    nh, nkv, hd = heads
    rng = np.random.default_rng(seed)
    if cache is None:
        table, pages = tables(rng, lens, page)
        cache = random_cache(rng, pages, page, nkv, hd), table
    c, table = cache
    if tweak:
        tweak(c, table)
    start = int(rng.integers(0, 2)) + np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)
    total, wide = int(start[-1]) + 2, 2 * hd if gated else hd
    x, t = rounded(rng.normal(0, 1, (total, nh * wide + 8)), kind)
    q = t[:, :nh * wide]
    d = Views(c, table, lens, start, total)
    out = torch.full((total, nh * hd + 16), 7.0, dtype=torch_type(kind), device="cuda")
    if window:
        d.window(q, out, nh, gated, kind, *window)
    else:
        d.share(*share)
        d.prefix(q, out, nh, gated, kind)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    assert np.all(got[:, nh * hd:] == 7.0), "past the row"
    got = got[:, :nh * hd].reshape(total, nh, hd)
    want, vmax, smax = view.attend(c, table, lens, start, x[:, :nh * wide].reshape(total, nh, wide), nh, gated,
                                   *(window or (None, 0)), out=np.full((total, nh, hd), 7.0))
    close(got, want, vmax, smax, kind, hd)
    return got, want


HEADS = [(16, 2, 256), (4, 1, 128), (12, 2, 128), (8, 8, 128), (24, 2, 256), (3, 3, 256), (40, 1, 128)]
ROWS = [
    ([1], [1]),
    ([65], [1]),
    ([130], [3]),
    ([200], [70]),
    ([97], [97]),
    ([5, 0, 129, 33, 1, 260], [1, 0, 3, 0, 1, 2]),
    ([300, 70, 3, 190], [40, 9, 1, 190]),
    ([700], [1]),
]
WINDOWS = [(1, 0), (1, 1), (64, 0), (65, 4), (37, 64), (128, 65), (200, 0), (5, 150), (1000, 3)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", range(len(HEADS)))
@pytest.mark.parametrize("batch", range(len(ROWS)))
def test_window(have_gpu, kind, heads, batch):
    lens, rows = ROWS[batch]
    page = [16, 64, 32, 128][(heads + batch) % 4]
    for i in range(3):
        call(heads * 31 + batch, HEADS[heads], page, lens, rows, kind, (heads + batch) % 2 == 0,
             window=WINDOWS[(heads + 3 * batch + 2 * i) % len(WINDOWS)])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("heads,batch", [((16, 2, 256), 5), ((4, 1, 128), 7), ((8, 2, 128), 6), ((8, 1, 256), 4)])
def test_every_window(have_gpu, kind, window, heads, batch):
    call(batch, heads, 16, *ROWS[batch], kind, False, window=window)


LONG = [
    ((16, 2, 256), [9000], [1], (4000, 4)),
    ((32, 8, 128), [4000, 100, 2500, 1], [1, 1, 2, 1], (1111, 70)),
    ((6, 2, 128), [3001], [5], (2048, 2500)),
    ((8, 2, 256), [1500], [700], (300, 5)),
    ((16, 1, 128), [1200, 900], [600, 900], (129, 0)),
    ((1, 1, 128), [60000], [2], (40000, 10000)),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_windows_in_many_parts(have_gpu, kind, case):
    heads, lens, rows, window = LONG[case]
    call(case, heads, [128, 16, 64][case % 3], lens, rows, kind, case % 2 == 0, window=window)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 256)])
def test_what_no_row_sees_may_be_anything(have_gpu, kind, rows, heads):
    """Pages between the first tokens and the window are gone, and hidden tokens
    beside visible ones in their page are NaN and infinite."""
    n, window, sinks, page = 900, 200, 70, 16

    def tweak(c, table):
        seen = np.zeros(n, bool)
        for p in range(n - rows, n):
            seen[max(0, p - window + 1):p + 1] = True
        seen[:sinks] = True
        for i, t in enumerate(np.flatnonzero(~seen)):
            at = c.place(table[0], int(t))
            for w in "kv":
                c.pairs[w][at[0], :, at[1]] = [0x7FC07FC0, 0x3F807F80, 0xFF803F80][i % 3]
        for e in range(len(table[0])):  # also pages beside a visible one's in a tile
            if not seen[e * page:(e + 1) * page].any():
                table[0, e] = 0xFFFFFFFF
        assert (table == 0xFFFFFFFF).sum() > 20

    got, _ = call(3, heads, page, [n], [rows], kind, False, window=(window, sinks), tweak=tweak)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 60])
def test_a_token_that_is_not_finite_is_seen_through_its_window_alone(have_gpu, kind, rows):
    """Token 400 of 460 is NaN: NaN for the rows whose window holds it."""
    def tweak(c, table):
        at = c.place(table[0], 400)
        c.pairs["v"][at[0], :, at[1]] = 0x7FC07FC0
        c.pairs["k"][at[0], :, at[1]] = 0x7FC07FC0

    for window in (30, 59, 60, 61, 100):
        got, want = call(4, (8, 2, 128), 32, [460], [rows], kind, False, window=(window, 3), tweak=tweak)
        assert np.isnan(want).any() == (459 - 400 < window or rows > 1)


def test_windows_of_bad_tables_and_lengths(have_gpu):
    """A missing page is NaN for the rows whose window holds a token of it, a length past the table
    for all of its sequence's rows; rows before position 0 see nothing."""
    def tweak(c, table):
        table[0, 2] = 4000  # tokens 32 .. 47

    for kind in ("f32", "bf16"):
        for nh in (8, 64):
            rng = np.random.default_rng(4)
            lens, rows = [90, 40 + 100 * 16, 20, 3], [70, 3, 20, 6]
            table, pages = tables(rng, [90, 40, 20, 30], 16)
            got, want = call(4, (nh, 2, 128), 16, lens, rows, kind, False, window=(20, 2), tweak=tweak,
                             cache=(random_cache(rng, pages, 16, 2, 128), table))
            assert np.isnan(want).any() and (want == 0).any()


def test_a_window_of_everything_is_plain(have_gpu):
    """The same cut and the same sums: bit for bit where no sequence has many pairs."""
    import torch

    rng = np.random.default_rng(9)
    lens, rows = [700, 65, 1, 300], [1, 3, 1, 2]
    table, pages = tables(rng, lens, 32)
    c = random_cache(rng, pages, 32, 2, 128)
    _, q = rounded(rng.normal(0, 1, (7, 8 * 128)), "f32")
    d = Views(c, table, lens, [0, 1, 4, 5, 7], 7)
    a, b, e = (torch.zeros(7, 8 * 128, device="cuda") for _ in range(3))
    d.attend(q, a, 8, False, "f32")
    d.window(q, b, 8, False, "f32", 700, 0)
    d.window(q, e, 8, False, "f32", 0xFFFFFFFF, 0xFFFFFFFF)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, e)


@pytest.mark.parametrize("n", [65, 300, 1024])
def test_windows_of_many_sequences(have_gpu, n):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 160, n)
    rows = np.minimum(rng.integers(0, 3, n), lens + 1)
    lens[n // 2], rows[n // 2] = 350, 90
    lens[n - 1], rows[n - 1] = 270, 1
    table = rng.integers(0, 50, (n, 22)).astype(np.uint32)
    call(n, (4, 1, 128), 16, lens, rows, "bf16", False, cache=(random_cache(rng, 50, 16, 1, 128), table), window=(50, 5))


# ------------------------------------------------------------------ shared prefixes


def grouped(rng, page, nkv, hd, groups, alone, spare=3):
    """(cache, table), lens, first, tokens of groups = [(tokens, [own lengths])]: the prefix's whole pages
    are shared, the page it ends in is each sequence's own (alike); then sequences of their own."""
    lens, first = [], [0]
    for tokens, own in groups:
        lens += [tokens + n for n in own]
        first.append(len(lens))
    lens += alone
    width = max(-(-n // page) for n in lens + [1])
    pages = sum(-(-n // page) for n in lens) + spare
    c = random_cache(rng, pages, page, nkv, hd)
    ids, at = rng.permutation(pages), 0
    table = np.full((len(lens), width), pages + 5, np.uint32)
    for b, n in enumerate(lens):
        g = next((g for g in range(len(groups)) if first[g] <= b < first[g + 1]), None)
        common = 0
        if g is not None and b > first[g]:
            common = groups[g][0] // page
            table[b, :common] = table[first[g], :common]
        held = -(-n // page)
        table[b, common:held] = ids[at:at + held - common]
        at += held - common
        if g is not None and b > first[g] and groups[g][0] % page:
            rest, a, z = groups[g][0] % page, table[first[g], common], table[b, common]
            for w in "kv":
                c.codes[w][z, :, :rest], c.pairs[w][z, :, :rest] = c.codes[w][a, :, :rest], c.pairs[w][a, :, :rest]
    return (c, table), lens, first, [t for t, _ in groups]


# (groups, alone, rows)
SHARED = [
    ([(64, [1, 1])], [], [1, 1]),
    ([(640, [1, 17, 64])], [], [1, 1, 1]),
    ([(300, [3, 40, 9, 100])], [77], [3, 2, 1, 4, 2]),
    ([(128, [5, 5, 5, 5, 5, 5, 5, 5]), (190, [8, 70])], [0, 130], [1, 1, 2, 0, 1, 3, 1, 1, 2, 70, 0, 5]),
    ([(1000, [90, 80, 33])], [], [90, 70, 5]),
    ([(70, [0, 0, 1])], [], [1, 1, 1]),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", range(len(HEADS)))
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_prefix(have_gpu, kind, heads, case):
    groups, alone, rows = SHARED[case]
    page = [16, 64, 32, 128][(heads + case) % 4]
    nh, nkv, hd = HEADS[heads]
    cache, lens, first, tokens = grouped(np.random.default_rng(case), page, nkv, hd, groups, alone)
    call(heads * 31 + case, HEADS[heads], page, lens, rows, kind, (heads + case) % 2 == 0, cache=cache, share=(first, tokens))


BIG = [
    ((16, 2, 256), [(3000, [40, 1, 200, 7])], [500], [1, 1, 1, 1, 1]),
    ((32, 8, 128), [(2500, [1 + i % 50 for i in range(40)])], [], [1] * 40),
    ((24, 2, 256), [(1700, [30, 100, 7]), (1100, [5] * 9)], [900, 20], [3, 3, 3] + [3] * 9 + [3, 3]),
    ((4, 1, 128), [(1300, [200, 150, 100])], [], [200, 90, 1]),
    ((1, 1, 128), [(9000, [i + 1 for i in range(70)])], [], [1] * 70),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(BIG)))
def test_prefixes_in_many_parts(have_gpu, kind, case):
    heads, groups, alone, rows = BIG[case]
    page = [128, 16, 64][case % 3]
    cache, lens, first, tokens = grouped(np.random.default_rng(case), page, heads[1], heads[2], groups, alone)
    call(case, heads, page, lens, rows, kind, case % 2 == 0, cache=cache, share=(first, tokens))


def test_many_groups(have_gpu):
    """As many groups as sequences, of none to a few."""
    rng = np.random.default_rng(77)
    groups = [(64 * int(rng.integers(1, 4)), [int(x) for x in rng.integers(1, 30, rng.integers(0, 5))]) for _ in range(400)]
    cache, lens, first, tokens = grouped(rng, 16, 1, 128, groups, [40] * 30)
    assert len(lens) <= 1024
    rows = np.minimum(rng.integers(0, 3, len(lens)), lens)
    call(1, (4, 1, 128), 16, lens, rows, "bf16", False, cache=cache, share=(first, tokens))


def test_prefixes_that_are_not_sound(have_gpu):
    """A prefix longer than what is held, groups of nobody, past the last sequence or of none,
    members without rows, with rows before position 0 or lengths past the table: plain attention's results."""
    for kind in ("f32", "bf16"):
        for first, tokens in [([0, 5], [10**9]), ([0, 5], [0]), ([0, 0, 5, 5], [64, 640, 64]), ([0, 900], [640]), ([900, 900], [640]),
                              ([3, 5], [640]), ([0, 0xFFFFFFFF], [0xFFFFFFFF]), ([0], [])]:
            rng = np.random.default_rng(5)
            cache, lens, _, _ = grouped(rng, 16, 2, 128, [(640, [7, 30, 1, 64, 9])], [50, 3])
            lens[6], rows = 3, [1, 2, 0, 1, 3, 1, 9]
            call(2, (8, 2, 128), 16, lens, rows, kind, False, cache=cache, share=(first, tokens))
            bad = list(lens)
            bad[1] = 16 * cache[1].shape[1] + 1
            call(2, (8, 2, 128), 16, bad, rows, kind, False, cache=cache, share=(first, tokens))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_shared_token_that_is_not_finite(have_gpu, kind):
    """A page of the prefix is missing or holds NaN: NaN for all of the group's rows, others stay as they are."""
    def missing(c, table):
        table[:4, 3] = c.pages

    def poison(c, table):
        at = c.place(table[0], 100)
        c.pairs["v"][at[0], 0, at[1], 1] = 0x7FC07FC0
        c.pairs["k"][at[0], 0, at[1], 1] = 0x7FC07FC0

    for tweak in (missing, poison):
        cache, lens, first, tokens = grouped(np.random.default_rng(6), 16, 2, 128, [(320, [7, 30, 1, 64])], [200])
        got, want = call(2, (8, 2, 128), 16, lens, [1, 2, 1, 1, 2], kind, False, cache=cache, share=(first, tokens), tweak=tweak)
        assert np.isnan(want).any() and np.isfinite(want[-3:]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_prefixes_of_very_different_size(have_gpu, kind):
    """Scores far apart and values of very different size on either side of a prefix's end."""
    import torch

    for loud in (0, 1):
        rng = np.random.default_rng(8)
        nh, nkv, hd, page = 8, 1, 128, 16
        (c, table), lens, first, tokens = grouped(rng, page, nkv, hd, [(256, [20, 70, 5])], [])
        for b in range(3):
            span = range(0, 256, 5) if loud == 0 else range(256, lens[b], 3)
            for t in span:
                c.write(table[b], t, "v", (1e4 * rng.normal(0, 1, (nkv, hd))).astype(np.float32))
                c.write(table[b], t, "k", (30 * rng.normal(0, 1, (nkv, hd))).astype(np.float32))
        x, q = rounded(rng.normal(0, 1, (4, nh * hd)), kind)
        d = Views(c, table, lens, [0, 1, 3, 4], 4)
        d.share(first, tokens)
        out = torch.zeros(4, nh * hd, dtype=torch_type(kind), device="cuda")
        d.prefix(q, out, nh, False, kind)
        want, vmax, smax = view.attend(c, table, lens, [0, 1, 3, 4], x.reshape(4, nh, hd), nh, False)
        got = out.double().cpu().numpy().reshape(4, nh, hd)
        tol = ref.tolerance(kind, hd, want, vmax, smax)
        past = (kind == "f16") & (np.abs(want) + tol >= 65520) & np.isinf(got)  # (f16 ends there)
        assert np.all((np.abs(got - want) <= tol) | past), loud


# ------------------------------------------------------------------ workspaces, graphs, streams


@pytest.mark.parametrize("case", range(len(LONG)))
def test_windows_write_nothing_past_the_workspace(have_gpu, case):
    import torch

    (nh, nkv, hd), lens, rows, window = LONG[case]
    rng = np.random.default_rng(case)
    table, pages = tables(rng, lens, 64)
    start = np.concatenate([[0], np.cumsum(rows)])
    d = Views(random_cache(rng, pages, 64, nkv, hd), table, lens, start, int(start[-1]))
    need = d.workspace(nh).numel()
    ws = torch.full((need + 65536,), 0x5A, dtype=torch.uint8, device="cuda")
    q = torch.randn(int(start[-1]), nh * hd, device="cuda")
    out = torch.zeros_like(q)
    d.window(q, out, nh, False, "f32", *window, ws=ws[:need])
    torch.cuda.synchronize()
    assert torch.all(ws[need:] == 0x5A) and torch.isfinite(out).all()
    with pytest.raises(EngineError, match="workspace smaller"):
        d.window(q, out, nh, False, "f32", *window, ws=ws[:need - 1])


@pytest.mark.parametrize("case", range(len(BIG)))
def test_prefixes_write_nothing_past_the_workspace(have_gpu, case):
    import torch

    (nh, nkv, hd), groups, alone, rows = BIG[case]
    (c, table), lens, first, tokens = grouped(np.random.default_rng(case), 64, nkv, hd, groups, alone)
    start = np.concatenate([[0], np.cumsum(rows)])
    d = Views(c, table, lens, start, int(start[-1]))
    d.share(first, tokens)
    need = d.prefix_workspace(nh, len(tokens)).numel()
    ws = torch.full((need + 65536,), 0x5A, dtype=torch.uint8, device="cuda")
    q = torch.randn(int(start[-1]), nh * hd, device="cuda")
    out = torch.zeros_like(q)
    d.prefix(q, out, nh, False, "f32", ws=ws[:need])
    torch.cuda.synchronize()
    assert torch.all(ws[need:] == 0x5A) and torch.isfinite(out).all()
    with pytest.raises(EngineError, match="workspace smaller than chk_attn_prefix"):
        d.prefix(q, out, nh, False, "f32", ws=ws[:need - 1])


@pytest.mark.parametrize("which", ["window", "prefix"])
def test_views_in_a_graph(have_gpu, which):
    """Captured once, replayed as sequences grow and the shared part changes, with
    eager calls between the replays; each replay equals the eager call."""
    import torch

    rng = np.random.default_rng(33)
    nh, nkv, hd, page = 8, 2, 128, 16
    (c, table), lens, first, tokens = grouped(rng, page, nkv, hd, [(320, [90, 60, 200])], [150])
    g, e = (Views(c, table, lens, [0, 2, 4, 6, 8], 8) for _ in range(2))
    for d in (g, e):
        d.share(first, tokens)
    q = torch.zeros(8, nh * hd, device="cuda", dtype=torch.bfloat16)
    og, oe = torch.zeros_like(q), torch.zeros_like(q)

    def run(d, o, ws=None, stream=None):
        if which == "window":
            d.window(q, o, nh, False, "bf16", 100, 5, ws=ws, stream=stream)
        else:
            d.prefix(q, o, nh, False, "bf16", ws=ws, stream=stream)

    ws = g.workspace(nh) if which == "window" else g.prefix_workspace(nh, 1)
    run(g, og, ws)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        run(g, og, ws, torch.cuda.current_stream().cuda_stream)
    for step in range(30):
        q.copy_(torch.from_numpy(rng.normal(0, 1, (8, nh * hd)).astype(np.float32)))
        now = np.array([320 + 3 * step, 330 + step, 322 + 6 * step, 5 + 4 * step], np.int32)
        for d in (g, e):
            d.lens.copy_(torch.from_numpy(now))
            d.tokens.fill_([320, 64, 0, 150][step % 4])
        graph.replay()
        torch.cuda.synchronize()
        run(e, oe)
        torch.cuda.synchronize()
        assert torch.equal(og, oe) and torch.isfinite(og.float()).all(), step


@pytest.mark.parametrize("which", ["window", "prefix"])
def test_views_on_two_streams_at_once(have_gpu, which):
    import torch

    rng = np.random.default_rng(40)
    (c, table), lens, first, tokens = grouped(rng, 32, 2, 128, [(500, [90, 60, 200])], [77])
    _, q = rounded(rng.normal(0, 1, (8, 8 * 128)), "f32")
    ds = [Views(c, table, lens, [0, 2, 4, 6, 8], 8) for _ in range(2)]
    for d in ds:
        d.share(first, tokens)

    def run(d, o, ws=None, stream=None):
        if which == "window":
            d.window(q, o, 8, False, "f32", 300, 5, ws=ws, stream=stream)
        else:
            d.prefix(q, o, 8, False, "f32", ws=ws, stream=stream)

    want = torch.zeros(8, 8 * 128, device="cuda")
    run(ds[0], want)
    outs, streams = [torch.zeros_like(want) for _ in ds], [torch.cuda.Stream() for _ in ds]
    ws = [d.workspace(8) if which == "window" else d.prefix_workspace(8, 1) for d in ds]
    torch.cuda.synchronize()
    for _ in range(20):
        for d, o, s, w in zip(ds, outs, streams, ws):
            run(d, o, w, s.cuda_stream)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_host_memory_is_refused(have_gpu):
    import torch

    rng = np.random.default_rng(2)
    table, pages = tables(rng, [20], 16)
    d = Views(random_cache(rng, pages, 16, 1, 128), table, [20], [0, 1], 1)
    d.share([0, 1], [16])
    host, x = torch.zeros(1, 128), torch.zeros(1, 128, device="cuda")
    with pytest.raises(EngineError, match="not device memory"):
        d.window(x, host, 1, False, "f32", 5, 0)
    with pytest.raises(EngineError, match="not device memory"):
        d.prefix(host.pin_memory(), x, 1, False, "f32")
    first = torch.zeros(2, dtype=torch.int32)
    d.shared = abi.ChkKvShared(first.data_ptr(), d.tokens.data_ptr(), 1)
    with pytest.raises(EngineError, match="not device memory"):
        d.prefix(x, x, 1, False, "f32")


# ------------------------------------------------------------------ a step's calls together


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("which", ["window", "prefix"])
def test_a_serving_run(have_gpu, which, kind):
    """One request's prompt, forked into continuations that share its pages, drafts of which some are
    rejected, one that ends: plan, norm and rotation, append and attention for each step as one
    program's buffers, against the same rules on the host."""
    import torch

    from tests import step_ref

    rng = np.random.default_rng(70)
    n, nh, nkv, hd, page, width, pages, most = 5, 8, 2, 128, 16, 40, 90, 130
    dt = torch_type(kind)
    turn = np.zeros(32, np.uint64)
    check(lib().chk_rope_turns(1e4, 64, turn.ctypes.data))
    turns = torch.from_numpy(turn.view(np.int64)).cuda()
    norms = (1 + 0.2 * rng.normal(0, 1, (2, hd))).astype(np.float32)
    weights = torch.from_numpy(norms).bfloat16().cuda()
    norms = weights.double().cpu().numpy()
    state = dict(table=np.full((n, width), 0xFFFFFFFF, np.uint32), len=np.zeros(n, np.uint32), free=np.arange(pages, dtype=np.uint32),
                 nfree=np.array([pages, 0], np.uint32))
    on = {k: dev(v) for k, v in state.items()}
    pool = abi.ChkKvPool(*(on[k].data_ptr() for k in ("table", "len", "free", "nfree")), n, width, page, pages)
    host = ref.Cache(pages, page, nkv, hd)
    d = Views(host, state["table"], state["len"], np.zeros(n + 1), most)
    d.table, d.lens = on["table"], on["len"]
    d.seqs = abi.ChkKvSeqs(on["table"].data_ptr(), on["len"].data_ptr(), d.start.data_ptr(), n, width, most)
    d.share([0, n], [0])
    own = np.zeros(n, np.uint32)
    norm = abi.ChkQkNorm(weights[0].data_ptr(), weights[1].data_ptr(), turns.data_ptr(), 64, nh, nkv, hd, 0, 1e-6)
    pos, slot = torch.zeros(most, dtype=torch.int32, device="cuda"), torch.zeros(most, dtype=torch.int64, device="cuda")
    q, k = torch.zeros(most, nh * hd, dtype=dt, device="cuda"), torch.zeros(most, nkv * hd, dtype=dt, device="cuda")
    out = torch.zeros(most, nh * hd, dtype=dt, device="cuda")
    ws = d.workspace(nh) if which == "window" else d.prefix_workspace(nh, 1)

    steps = [([0] * n, [120, 0, 0, 0, 0])]  # the prompt
    steps.append(([115, 112, 112, 112, 112], [1, 30, 2, 5, 1]))  # cut back, and forked on its seven whole pages
    for i in range(6):
        steps.append((None, [3, 1, 2, 1, 4]))
    steps.append((0, [1, 1, 1, 0, 1]))
    steps.append((None, [1, 1, 1, 0, 1]))
    for i, (keep, want) in enumerate(steps):
        if i == 1:  # the continuations' tables begin with the prompt's pages
            t = on["table"].cpu().numpy().view(np.uint32)
            t[1:, :7] = t[0, :7]
            state["table"] = t.copy()
            state["len"] = np.array([120, 112, 112, 112, 112], np.uint32)
            own[1:] = 7
            for name in ("table", "len"):
                on[name].copy_(dev(state[name]))
            d.tokens.fill_(112)
        if keep is None:
            keep = np.maximum(state["len"].astype(int) - rng.integers(0, 3, n), 113)
            keep = np.where(state["len"] == 0, 0, keep)
        elif np.isscalar(keep):
            keep = state["len"].copy()
            keep[3] = 0  # has ended
        kp, ow, wa = (dev(np.asarray(x, np.uint32)) for x in (keep, own, want))
        check(lib().chk_kv_plan_q4(C.byref(pool), kp.data_ptr(), ow.data_ptr(), wa.data_ptr(), most, d.start.data_ptr(),
                                   pos.data_ptr(), slot.data_ptr(), None))
        x, t = rounded(rng.normal(0, 1, (most, (nh + 2 * nkv) * hd)), kind)
        check(lib().chk_qk_norm_rope(C.byref(norm), pos.data_ptr(), most, t.data_ptr(), t.stride(0), q.data_ptr(), q.stride(0),
                                     t[:, nh * hd:].data_ptr(), t.stride(0), k.data_ptr(), k.stride(0), KINDS[kind], None))
        d.append(k, t[:, (nh + nkv) * hd:], kind)
        if which == "window":
            d.window(q, out, nh, False, kind, 60, 4, ws=ws)
        else:
            d.prefix(q, out, nh, False, kind, ws=ws)
        torch.cuda.synchronize()
        names = ("table", "len", "free", "nfree", "start", "pos", "slot")
        plan = dict(zip(names, step_ref.plan(state["table"], state["len"], state["free"], state["nfree"][0], keep, own, want, most,
                                             page, pages)))
        state = {name: plan[name] for name in names[:4]}
        for name, a in (("table", on["table"]), ("len", on["len"]), ("nfree", on["nfree"]), ("start", d.start), ("pos", pos)):
            np.testing.assert_array_equal(a.cpu().numpy().view(np.uint32), plan[name], err_msg=f"{name} {i}")
        start, live = plan["start"], int(plan["start"][-1])
        gq, gk = (a[:live].double().cpu().numpy().reshape(live, -1, hd) for a in (q, k))
        for got, at, heads, w in ((gq, 0, nh, norms[0]), (gk, nh * hd, nkv, norms[1])):
            raw = x[:live, at:at + heads * hd].reshape(live, heads, hd)
            want_x, size = step_ref.norm_rope(raw, w, 1e-6, plan["pos"][:live], 1e4, 64)
            assert np.all(np.abs(got - want_x) <= step_ref.norm_rope_tolerance(kind, want_x, size))
        for b in range(n):
            for r in range(int(start[b]), int(start[b + 1])):
                host.write(state["table"][b], int(plan["pos"][r]), "k", gk[r].astype(np.float32))
                host.write(state["table"][b], int(plan["pos"][r]), "v", x[r, (nh + nkv) * hd:].reshape(nkv, hd))
        back = d.back()
        for b in range(n):
            for e in range(-(-int(state["len"][b]) // page)):
                z, m = state["table"][b, e], min(page, int(state["len"][b]) - e * page)
                for w in "kv":
                    np.testing.assert_array_equal(back.codes[w][z][:, :m], host.codes[w][z][:, :m])
        want_o, vmax, smax = view.attend(host, state["table"], state["len"], start, gq, nh, False,
                                         *((60, 4) if which == "window" else (None, 0)), out=np.zeros((live, nh, hd)))
        close(out[:live].double().cpu().numpy().reshape(live, nh, hd), want_o, vmax, smax, kind, hd)


# ------------------------------------------------------------------ more blocks than the device takes at once


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [(8, 8, 128), (32, 8, 128), (8, 8, 256), (24, 24, 256)])
@pytest.mark.parametrize("which", ["window", "prefix"])
def test_crowded_batches(have_gpu, kind, heads, which):
    """100 sequences of up to 24 kv heads: short walks are a wave's each, beside longer ones
    and rows of many pairs; and a workgroup's waves that have none."""
    rng = np.random.default_rng(12)
    nh, nkv, hd = heads
    lens = rng.integers(0, 200, 100)
    rows = np.minimum(rng.integers(0, 3, 100), lens + 1)
    lens[7], rows[7] = 1500, 1
    lens[50], rows[50] = 300, 80
    lens[99], rows[99] = 130, 1
    if which == "window":
        table = rng.integers(0, 60, (100, 94)).astype(np.uint32)
        call(12, heads, 16, lens, rows, kind, False, cache=(random_cache(rng, 60, 16, nkv, hd), table), window=(90, 5))
    else:
        table = rng.integers(0, 60, (100, 110)).astype(np.uint32)
        table[10:90, :16] = table[10, :16]
        lens[10:90] += 256
        call(12, heads, 16, lens, rows, kind, True, cache=(random_cache(rng, 60, 16, nkv, hd), table), share=([10, 90], [256]))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("which", ["window", "prefix"])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [5, 2, 40, 1]])
def test_queries_that_are_not_finite_stay_in_their_row(have_gpu, kind, which, rows):
    """Also among the rows of a group that take its prefix together; and the same call twice."""
    import torch

    rng = np.random.default_rng(80)
    nh, nkv, hd = 8, 2, 128
    (c, table), lens, first, tokens = grouped(rng, 16, nkv, hd, [(192, [50, 9, 70])], [90])
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    x = rng.normal(0, 1, (total, nh, hd)).astype(np.float32)
    bad = [(0, 0, np.nan), (1, 5, np.inf), (total - 2, 7, -np.inf), (total - 1, 3, np.nan)]
    for r, h, v in bad:
        x[r, h, 17 * h % hd] = v
    x, q = rounded(x.reshape(total, -1), kind)
    d = Views(c, table, lens, start, total)
    d.share(first, tokens)
    outs = [torch.zeros_like(q) for _ in range(2)]
    for out in outs:
        if which == "window":
            d.window(q, out, nh, False, kind, 60, 3)
        else:
            d.prefix(q, out, nh, False, kind)
    torch.cuda.synchronize()
    assert torch.equal(*(o.view({"f32": torch.int32}.get(kind, torch.int16)) for o in outs))
    got = outs[0].double().cpu().numpy().reshape(total, nh, hd)
    with np.errstate(all="ignore"):
        want, vmax, smax = view.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False,
                                       *((60, 3) if which == "window" else (None, 0)))
        tol = ref.tolerance(kind, hd, want, vmax, smax)
    fine = np.ones((total, nh), bool)
    for r, h, _ in bad:
        fine[r, h] = False
        assert np.isnan(got[r, h]).all()
    assert np.all(np.abs(got - want)[fine] <= tol[fine])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1024, 8704])
def test_groups_of_33_to_64_pairs(have_gpu, kind, tokens):
    """Eight sequences of 48 and 64 query heads over 8: blocks of few pairs behind a
    short prefix, of many behind one that fills the device."""
    for nh in (48, 64):
        cache, lens, first, shared = grouped(np.random.default_rng(3), 64, 8, 128, [(tokens, [1, 30, 2, 9, 70, 5, 66, 3])], [])
        call(3, (nh, 8, 128), 64, lens, [1] * 8, kind, False, cache=cache, share=(first, shared))
