"""The 4-bit key/value cache on the GPU (chk_kv_append_q4, chk_kv_read_q4,
chk_attn_q4) against plain numpy in 64 bits (tests/kv4_ref.py): rows written
bit for bit, read back to the type's rounding, attention over ragged batches
of shared pages within a tolerance from its roundings; what no call may touch;
bad tables and lengths; masks that leave a row nothing; graphs, streams and a
decode run of the calls together."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from cherenkov_amd.abi import EngineError, check, lib
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu

KINDS = {"f32": abi.CHK_F32, "f16": abi.CHK_F16, "bf16": abi.CHK_BF16}


def torch_type(kind):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def dev(a: np.ndarray):
    import torch

    a = np.ascontiguousarray(a)
    view = {np.dtype(np.uint32): np.int32}.get(a.dtype)
    return torch.from_numpy(a.view(view) if view else a.copy()).cuda()


def rounded(x: np.ndarray, kind: str):
    """f32 values of `kind`'s grid, and the device tensor that holds them."""
    import torch

    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch_type(kind)).cuda()
    return t.float().cpu().numpy(), t


class Dev:
    """A host cache's planes on the device and the batch's description."""

    def __init__(self, host: ref.Cache, table, lens, start, rows):
        self.host = host
        self.planes = [dev(host.codes["k"]), dev(host.codes["v"]), dev(host.pairs["k"]), dev(host.pairs["v"])]
        self.table, self.lens, self.start = (dev(np.asarray(a, np.uint32)) for a in (table, lens, start))
        self.cache = abi.ChkKvQ4(*(p.data_ptr() for p in self.planes), host.pages, host.page, host.nkv, host.hd)
        self.seqs = abi.ChkKvSeqs(self.table.data_ptr(), self.lens.data_ptr(), self.start.data_ptr(), len(lens),
                                  self.table.shape[1], rows)

    def back(self) -> ref.Cache:
        import torch

        torch.cuda.synchronize()
        c = self.host.copy()
        c.codes = {w: p.cpu().numpy() for w, p in zip("kv", self.planes[:2])}
        c.pairs = {w: p.cpu().numpy().view(np.uint32) for w, p in zip("kv", self.planes[2:])}
        return c

    def append(self, k, v, kind, stream=None):
        check(lib().chk_kv_append_q4(C.byref(self.cache), C.byref(self.seqs), k.data_ptr(), v.data_ptr(), KINDS[kind],
                                     k.stride(0), v.stride(0), stream))

    def read(self, k, v, kind, stream=None):
        check(lib().chk_kv_read_q4(C.byref(self.cache), C.byref(self.seqs), k.data_ptr(), v.data_ptr(), KINDS[kind],
                                   k.stride(0), v.stride(0), stream))

    def workspace(self, nh):
        import torch

        n = C.c_uint64()
        check(lib().chk_attn_q4_workspace(nh, self.host.nkv, self.host.hd, self.seqs.n, self.seqs.rows, C.byref(n)))
        # what the workspace holds before a call means nothing
        return torch.full((n.value,), 0xFF, dtype=torch.uint8, device="cuda")

    def attend(self, q, out, nh, gated, kind, mask=None, ws=None, stream=None):
        ws = self.workspace(nh) if ws is None else ws
        m = None
        if mask is not None:
            self.bits = dev(mask[0])
            m = C.byref(abi.ChkKvMask(self.bits.data_ptr(), mask[0].shape[1], mask[1], mask[2]))
        check(lib().chk_attn_q4(C.byref(self.cache), C.byref(self.seqs), q.data_ptr(), nh, int(gated), KINDS[kind],
                                q.stride(0), m, out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), stream))
        self.ws = ws


def tables(rng, lens, page, spare=3):
    """Pages of every sequence anywhere in the pool; unused entries name pages
    the cache does not have."""
    need = [-(-max(int(n), 0) // page) for n in lens]
    pages = sum(need) + spare
    ids = rng.permutation(pages)
    width = max(need + [1])
    table = np.full((len(lens), width), pages + 5, np.uint32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, pages


def filled(rng, lens, page, nkv, hd, loud=True):
    """A host cache whose sequences hold rows like normed keys and values."""
    table, pages = tables(rng, lens, page)
    c = ref.Cache(pages, page, nkv, hd)
    for b, n in enumerate(lens):
        for which in "kv":
            x = rng.normal(0, 1, (int(n), nkv, hd)).astype(np.float32)
            if loud:
                x[:, :, ::37] *= 5
            for t in range(int(n)):
                c.write(table[b], t, which, x[t])
    return c, table


# ------------------------------------------------------------------ rows written and read back

# lens: tokens after the call; rows: this call's
BATCHES = [
    ([1], [1]),
    ([17], [1]),
    ([40], [40]),
    ([33, 5, 64, 0, 18], [2, 5, 0, 0, 18]),
    ([16, 15, 31], [16, 15, 1]),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nkv,hd,page", [(2, 256, 16), (1, 128, 32), (3, 128, 16), (8, 128, 64)])
@pytest.mark.parametrize("batch", range(len(BATCHES)))
def test_append_and_read(have_gpu, kind, nkv, hd, page, batch):
    import torch

    lens, rows = BATCHES[batch]
    rng = np.random.default_rng(batch * 100 + hd + nkv)
    table, pages = tables(rng, lens, page)
    host = ref.Cache(pages, page, nkv, hd)
    first = 1 if batch % 2 else 0  # rows before the first sequence
    start = first + np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1]) + 3  # and behind the last
    # keys and values as parts of one wider row
    x, t = rounded(rng.normal(0, 1.5, (total, 2 * nkv * hd + 16)) * np.exp(rng.normal(0, 2, (total, 1))), kind)
    k, v = t[:, :nkv * hd], t[:, nkv * hd:2 * nkv * hd]
    d = Dev(host, table, lens, start, total)
    d.append(k, v, kind)
    got = d.back()
    for b in range(len(lens)):
        for i in range(rows[b]):
            r, p = start[b] + i, lens[b] - rows[b] + i
            host.write(table[b], p, "k", x[r, :nkv * hd].reshape(nkv, hd))
            host.write(table[b], p, "v", x[r, nkv * hd:2 * nkv * hd].reshape(nkv, hd))
    for w in "kv":  # every byte: the rows' own, and nothing else
        np.testing.assert_array_equal(got.pairs[w], host.pairs[w], err_msg=w)
        np.testing.assert_array_equal(got.codes[w], host.codes[w], err_msg=w)
    out = torch.full((2, total, nkv * hd + 8), 7.0, dtype=torch_type(kind), device="cuda")
    d.read(out[0], out[1], kind)
    torch.cuda.synchronize()
    back = out.float().cpu().numpy()
    assert np.all(back[:, :, nkv * hd:] == 7.0)
    mine = np.zeros(total, bool)
    half = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}[kind]
    for b in range(len(lens)):
        for i in range(rows[b]):
            r, p = start[b] + i, lens[b] - rows[b] + i
            mine[r] = True
            for j, w in enumerate("kv"):
                want = host.read(table[b], p, w).reshape(-1)
                # s c + b in f32, then the type: two roundings
                tol = (half + 2.0**-24) * np.abs(want) + 2.0**-25
                assert np.all(np.abs(back[j, r, :nkv * hd] - want) <= tol), (b, i, w)
    assert np.all(back[:, ~mine] == 7.0)


def test_append_edge_groups(have_gpu):
    """Groups that are constant, tiny, huge, far from zero, or hold NaN and
    infinities; ties between codes; each in f32, bit for bit."""
    import torch

    rng = np.random.default_rng(5)
    g = [np.zeros(64), np.full(64, -0.0), np.full(64, 0.3), np.full(64, -1.5), rng.normal(0, 1e-39, 64),
         np.where(np.arange(64) == 5, 1e-45, 0.0), rng.normal(0, 1e37, 64), rng.normal(1000, 0.01, 64),
         np.arange(64) / 2.0 % 15.5, np.arange(64) * 0.5 - 15, rng.integers(-8, 8, 64) / 2.0 * 1.0078125]
    for bad in (np.nan, np.inf, -np.inf):
        x = rng.normal(0, 1, 64)
        x[int(rng.integers(64))] = bad
        g.append(x)
    wide = np.zeros(64)
    wide[0], wide[1] = -3e38, 3e38
    g.append(wide)
    # a quotient that rounds onto a border in f32: one ulp to each side of it
    s = np.float32(1.0078125)
    for ulp in (-1, 0, 1):
        x = (np.arange(64) % 15 + 0.5).astype(np.float32) * s
        x = (x.view(np.int32) + ulp).view(np.float32)
        x[0], x[1] = 0.0, 15 * s
        g.append(x)
    while len(g) % 2:
        g.append(rng.normal(0, 1, 64))
    rows = np.stack(g).astype(np.float32).reshape(-1, 128)
    n = len(rows)
    table, pages = tables(rng, [n], 16)
    host = ref.Cache(pages, 16, 1, 128)
    d = Dev(host, table, [n], [0, n], n)
    t = torch.from_numpy(rows).cuda()
    d.append(t, t, "f32")
    got = d.back()
    for p in range(n):
        for w in "kv":
            host.write(table[0], p, w, rows[p][None])
            a, b = got.read(table[0], p, w), host.read(table[0], p, w)
            np.testing.assert_array_equal(a, b, err_msg=f"row {p} {w}")


def test_append_and_read_of_bad_places(have_gpu):
    """A page the cache has not, a length past the table, more rows than
    tokens: nothing written, NaN read; every other row as usual."""
    import torch

    rng = np.random.default_rng(9)
    nkv, hd, page = 2, 128, 16
    table = np.array([[0, 9, 2], [3, 0xFFFFFFFF, 4], [5, 6, 7]], np.uint32)
    lens, start = [48, 40, 50], [0, 30, 45, 65]
    host = ref.Cache(8, page, nkv, hd)
    total = 70
    x, t = rounded(rng.normal(0, 1, (total, nkv * hd)), "f32")
    d = Dev(host, table, lens, start, total)
    d.append(t, t, "f32")
    got = d.back()
    out = torch.full((2, total, nkv * hd), 7.0, device="cuda")
    d.read(out[0], out[1], "f32")
    back = out.cpu().numpy()
    for b in range(3):
        for r in range(start[b], start[b + 1]):
            p = lens[b] - (start[b + 1] - r)
            for j, w in enumerate("kv"):
                host.write(table[b], p, w, x[r].reshape(nkv, hd))
                np.testing.assert_allclose(back[j, r], host.read(table[b], p, w).reshape(-1), rtol=2.0**-23, atol=1e-30)
    for w in "kv":
        np.testing.assert_array_equal(got.pairs[w], host.pairs[w])
        np.testing.assert_array_equal(got.codes[w], host.codes[w])
    # three tokens, five rows: the first two lie before position 0
    host2 = ref.Cache(1, page, nkv, hd)
    d2 = Dev(host2, [[0]], [3], [0, 5], 5)
    d2.append(t, t, "f32")
    got2 = d2.back()
    for i in range(5):
        host2.write(np.array([0]), i - 2, "k", x[i].reshape(nkv, hd))
    np.testing.assert_array_equal(got2.codes["k"], host2.codes["k"])
    d2.read(out[0], out[1], "f32")
    back = out.cpu().numpy()
    assert np.isnan(back[:, :2]).all() and np.isfinite(back[:, 2:5]).all()


def test_starts_out_of_order_stay_inside(have_gpu):
    """Row starts past the call's rows or falling: rows that no sequence has
    stay as they were, and nothing is read or written outside."""
    import torch

    rng = np.random.default_rng(11)
    c, table = filled(rng, [20, 20, 20], 16, 1, 128)
    d = Dev(c, table, [20, 20, 20], [2, 5, 4, 400], 6)
    out = torch.full((2, 8, 128), 7.0, device="cuda")
    d.read(out[0], out[1], "f32")
    o2 = torch.full((8, 2, 128), 7.0, device="cuda")
    d.attend(torch.ones(8, 2, 128, device="cuda"), o2, 2, False, "f32")
    for a in (out[0], out[1], o2):
        a = a.cpu().numpy().reshape(8, -1)
        assert np.all(a[[0, 1, 6, 7]] == 7.0)


# ------------------------------------------------------------------ attention

HEADS = [(1, 1, 128), (4, 2, 128), (8, 1, 128), (24, 2, 256), (16, 2, 256), (4, 4, 256), (6, 2, 128), (20, 1, 256)]

ROWS = [
    ([1], [1]),
    ([2], [2]),
    ([64], [1]),
    ([65], [1]),
    ([130], [3]),
    ([200], [70]),
    ([97], [97]),
    ([5, 0, 129, 33, 1, 260], [1, 0, 3, 0, 1, 2]),
    ([40, 70, 3], [40, 9, 1]),
    ([700], [1]),
]


def attention_case(seed, nh, nkv, hd, page, lens, rows, kind, gated, mask=None, cache=None, tweak=None):
    import torch

    rng = np.random.default_rng(seed)
    c, table = filled(rng, lens, page, nkv, hd) if cache is None else cache
    if tweak:
        tweak(c, table)
    first = int(rng.integers(0, 2))
    start = first + np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)
    total = int(start[-1]) + 2
    wide = 2 * hd if gated else hd
    x, t = rounded(rng.normal(0, 1, (total, nh * wide + 8)), kind)
    q = t[:, :nh * wide]
    d = Dev(c, table, lens, start, total)
    out = torch.full((total, nh * hd + 16), 7.0, dtype=torch_type(kind), device="cuda")
    bits = None
    if mask is not None:
        bits = (mask(rng, total, max(lens)), *mask.shape)
    d.attend(q, out, nh, gated, kind, bits)
    torch.cuda.synchronize()
    got = out.float().cpu().numpy()
    assert np.all(got[:, nh * hd:] == 7.0), "past the row"
    got = got[:, :nh * hd].reshape(total, nh, hd)
    want, vmax, smax = ref.attend(c, table, lens, start, x[:, :nh * wide].reshape(total, nh, wide), nh, gated, bits,
                                  np.full((total, nh, hd), 7.0))
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    tol = ref.tolerance(kind, hd, want, vmax, smax)
    off = np.where(nan, 0, np.abs(got - want) - np.where(nan, 0, tol))
    assert np.all(off <= 0), f"worst {off.max():.3g} over, of {np.abs(np.where(nan, 0, got - want)).max():.3g}"
    return got, want


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", range(len(HEADS)))
@pytest.mark.parametrize("batch", range(len(ROWS)))
def test_attention(have_gpu, kind, heads, batch):
    nh, nkv, hd = HEADS[heads]
    lens, rows = ROWS[batch]
    page = [16, 64, 32, 128][(heads + batch) % 4]
    attention_case(heads * 31 + batch, nh, nkv, hd, page, lens, rows, kind, (heads + batch) % 2 == 0)


class Bits:
    """Random block bits: `keep` of them set."""

    def __init__(self, ratio, kblk, keep, words=None):
        self.shape, self.keep, self.words = (ratio, kblk), keep, words

    def __call__(self, rng, rows, longest):
        words = self.words or (longest // self.shape[0]) // 32 + 1
        bit = rng.random((rows, words, 32)) < self.keep
        return (bit.astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [Bits(4, 0, 0.3), Bits(4, 10, 0.1), Bits(1, 0, 0.5), Bits(1, 0, 0.0), Bits(7, 2, 0.0),
                                  Bits(4, 0, 0.5, words=1), Bits(300, 0, 0.5)],
                         ids=["4", "4_budget", "1", "empty_rows", "7_tail", "short_words", "300"])
@pytest.mark.parametrize("heads,batch", [((16, 2, 256), 5), ((4, 2, 128), 7), ((2, 2, 128), 6), ((8, 1, 128), 9)])
def test_attention_of_chosen_blocks(have_gpu, kind, bits, heads, batch):
    lens, rows = ROWS[batch]
    got, want = attention_case(batch, *heads, 16, lens, rows, kind, batch % 2 == 0, bits)
    if bits.keep == 0.0 and bits.shape == (1, 0):  # every token is a block, none chosen
        assert np.all((got == 0) | (got == 7.0))


def test_attention_past_what_a_mask_or_a_row_hides(have_gpu):
    """NaN, infinities and the largest values in tokens a row does not see:
    behind its own position, in blocks not chosen, behind the length."""
    nkv, hd, page = 2, 128, 16
    rng = np.random.default_rng(3)
    lens, rows = [150, 75], [70, 1]
    for pair in (0x7FC07FC0, 0x7F807F80, 0xFF80FF80, 0x7F7F7F7F, 0xFF7F7F7F):
        cache = filled(rng, lens, page, nkv, hd)
        c, table = cache
        for b, n in enumerate(lens):  # behind the length
            for t in range(n, len(table[b]) * page):
                at = c.place(table[b], t)
                if at:
                    for w in "kv":
                        c.pairs[w][at[0], :, at[1]] = pair
        for t in (85, 100, 149):  # a later row's own token
            at = c.place(table[0], t)
            for w in "kv":
                c.pairs[w][at[0], :, at[1]] = pair
        # blocks of 16 tokens: the fourth never chosen
        at = c.place(table[0], 16 * 3 + 2)
        for w in "kv":
            c.pairs[w][at[0], :, at[1]] = pair

        class NotThree(Bits):
            def __call__(self, rng, rows, longest):
                return np.full((rows, 1), 0xFFFFFFF7, np.uint32)

        import torch

        q_rows, nh = 71, 4
        x, q = rounded(rng.normal(0, 1, (q_rows, nh * hd)), "f32")
        start = [0, 70, 71]
        for kind in ("f32", "f16", "bf16"):
            x, q = rounded(x, kind)
            d = Dev(c, table, lens, start, q_rows)
            out = torch.zeros(q_rows, nh * hd, dtype=torch_type(kind), device="cuda")
            bits = (np.full((q_rows, 1), 0xFFFFFFF7, np.uint32), 16, 0)
            d.attend(q, out, nh, False, kind, bits)
            got = out.float().cpu().numpy().reshape(q_rows, nh, hd)
            with np.errstate(all="ignore"):
                want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(q_rows, nh, hd), nh, False, bits)
            clean = np.isfinite(want).all(axis=(1, 2)) & (vmax.max(1) < 1e6)
            assert clean[:5].all() and clean[70]  # rows 0..4 sit at 80..84
            tol = ref.tolerance(kind, hd, want[clean], vmax[clean], smax[clean])
            assert np.all(np.abs(got[clean] - want[clean]) <= tol), hex(pair)


def test_attention_of_bad_tables_and_lengths(have_gpu):
    """A missing page is NaN for the rows that see it, a length past the table
    for all of its sequence's rows; rows before position 0 see nothing."""
    import torch

    rng = np.random.default_rng(4)
    nkv, hd, page, nh = 2, 128, 16, 8
    c, table = filled(rng, [60, 40, 20, 30], page, nkv, hd)
    table[0, 2] = 4000  # tokens 32..47
    lens, rows = [60, 40 + 10 * page, 20, 3], [40, 3, 20, 6]
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    for kind in ("f32", "bf16"):
        x, q = rounded(rng.normal(0, 1, (total, nh * hd)), kind)
        d = Dev(c, table, lens, start, total)
        out = torch.zeros(total, nh * hd, dtype=torch_type(kind), device="cuda")
        d.attend(q, out, nh, False, kind)
        got = out.float().cpu().numpy().reshape(total, nh, hd)
        want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        assert np.isnan(want[12:43]).all() and np.isfinite(want[:12]).all() and np.all(want[63:66] == 0)
        ok = ~np.isnan(want).any(axis=(1, 2))
        assert np.all(np.abs(got[ok] - want[ok]) <= ref.tolerance(kind, hd, want[ok], vmax[ok], smax[ok]))


def test_attention_of_scores_far_apart(have_gpu):
    """Large queries: softmaxes of one token, exponents that underflow; and
    queries of zero: the mean of the values."""
    import torch

    rng = np.random.default_rng(6)
    nkv, hd, nh, n = 1, 128, 4, 300
    c, table = filled(rng, [n], 64, nkv, hd)
    for kind in ("f32", "f16", "bf16"):
        for scale in (0.0, 30.0, 2000.0):
            x, q = rounded(scale * rng.normal(0, 1, (5, nh * hd)), kind)
            d = Dev(c, table, [n], [0, 5], 5)
            out = torch.zeros(5, nh * hd, dtype=torch_type(kind), device="cuda")
            d.attend(q, out, nh, False, kind)
            got = out.float().cpu().numpy().reshape(5, nh, hd)
            want, vmax, smax = ref.attend(c, table, [n], [0, 5], x.reshape(5, nh, hd), nh, False)
            assert np.all(np.abs(got - want) <= ref.tolerance(kind, hd, want, vmax, smax)), (kind, scale)


def test_values_of_very_different_size(have_gpu):
    """Steps from 2^-126 to 2^60 in one sequence, the loud ones first, last and
    in between: no overflow, and the small ones are not lost where the loud
    ones are hidden."""
    import torch

    rng = np.random.default_rng(8)
    nkv, hd, nh, n = 1, 128, 2, 200
    table, pages = tables(rng, [n], 16)
    for where in (0, 100, 199):
        for size in (1e-30, 1e18):
            c = ref.Cache(pages, 16, nkv, hd)
            v = rng.normal(0, 1, (n, nkv, hd)).astype(np.float32)
            v[where] *= size
            v[(where + 7) % n] *= 1e-3
            k = rng.normal(0, 1, (n, nkv, hd)).astype(np.float32)
            for t in range(n):
                c.write(table[0], t, "k", k[t])
                c.write(table[0], t, "v", v[t])
            for kind in ("f32", "bf16"):
                x, q = rounded(rng.normal(0, 1, (n, nh * hd)), kind)
                d = Dev(c, table, [n], [0, n], n)
                out = torch.zeros(n, nh * hd, dtype=torch_type(kind), device="cuda")
                d.attend(q, out, nh, False, kind)
                got = out.float().cpu().numpy().reshape(n, nh, hd)
                want, vmax, smax = ref.attend(c, table, [n], [0, n], x.reshape(n, nh, hd), nh, False)
                assert np.all(np.abs(got - want) <= ref.tolerance(kind, hd, want, vmax, smax)), (where, size, kind)


# ------------------------------------------------------------------ the calls together


def test_decode_run_equals_prompt(have_gpu):
    """Tokens appended and attended one at a time, two sequences at once, give
    what one call over all of them gives (rows of a prompt)."""
    import torch

    rng = np.random.default_rng(21)
    nkv, hd, nh, page, n = 2, 256, 16, 16, 37
    table, pages = tables(rng, [n, n], page)
    x, kv = rounded(rng.normal(0, 1, (2, n, 2, nkv * hd)), "f32")
    qx, q = rounded(rng.normal(0, 1, (2, n, nh * 2 * hd)), "f32")
    host = ref.Cache(pages, page, nkv, hd)
    d = Dev(host, table, [n, n], [0, n, 2 * n], 2 * n)
    kk, vv = kv[:, :, 0].reshape(2 * n, -1).contiguous(), kv[:, :, 1].reshape(2 * n, -1).contiguous()
    d.append(kk, vv, "f32")
    whole = torch.zeros(2 * n, nh * hd, device="cuda")
    d.attend(q.reshape(2 * n, -1), whole, nh, True, "f32")
    full = d.back()

    e = Dev(host, table, [0, 0], [0, 1, 2], 2)
    step = torch.zeros(2, n, nh * hd, device="cuda")
    for t in range(n):
        e.lens.fill_(t + 1)
        k2, v2, q2 = (a.contiguous() for a in (kv[:, t, 0], kv[:, t, 1], q[:, t]))
        e.append(k2, v2, "f32")
        o = torch.zeros(2, nh * hd, device="cuda")
        e.attend(q2, o, nh, True, "f32")
        step[:, t] = o
    same = e.back()
    for w in "kv":
        np.testing.assert_array_equal(same.codes[w], full.codes[w])
        np.testing.assert_array_equal(same.pairs[w], full.pairs[w])
    a, b = whole.cpu().numpy().reshape(2, n, nh, hd), step.cpu().numpy().reshape(2, n, nh, hd)
    want, vmax, smax = ref.attend(full, table, [n, n], [0, n, 2 * n], qx.reshape(2 * n, nh, 2 * hd), nh, True)
    tol = ref.tolerance("f32", hd, want, vmax, smax).reshape(2, n, nh, hd)
    want = want.reshape(2, n, nh, hd)
    assert np.all(np.abs(a - want) <= tol) and np.all(np.abs(b - want) <= tol)


def test_calls_in_a_graph(have_gpu):
    """Append and attention captured once, replayed as the sequences grow, with
    eager work between the replays; each replay equals the eager calls."""
    import torch

    rng = np.random.default_rng(33)
    nkv, hd, nh, page, most = 2, 128, 8, 16, 90
    table, pages = tables(rng, [most, most, most], page)
    host = ref.Cache(pages, page, nkv, hd)
    g, e = (Dev(host, table, [1, 1, 1], [0, 1, 2, 3], 3) for _ in range(2))
    kv = torch.zeros(3, 2, nkv * hd, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(3, nh * hd, device="cuda", dtype=torch.bfloat16)
    og, oe = torch.zeros_like(q), torch.zeros_like(q)
    ws = g.workspace(nh)
    k, v = kv[:, 0], kv[:, 1]
    g.append(k, v, "bf16")
    g.attend(q, og, nh, False, "bf16", ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        st = torch.cuda.current_stream().cuda_stream
        g.append(k, v, "bf16", st)
        g.attend(q, og, nh, False, "bf16", ws=ws, stream=st)
    lens = np.array([1, 1, 1])
    for step in range(40):
        kv.copy_(torch.from_numpy(rng.normal(0, 1, (3, 2, nkv * hd)).astype(np.float32)))
        q.copy_(torch.from_numpy(rng.normal(0, 1, (3, nh * hd)).astype(np.float32)))
        for d in (g, e):
            d.lens.copy_(torch.from_numpy(lens.astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        e.append(k, v, "bf16")
        e.attend(q, oe, nh, False, "bf16")
        torch.cuda.synchronize()
        assert torch.equal(og, oe), step
        lens += [1, 2, 0]
    a, b = g.back(), e.back()
    for w in "kv":
        np.testing.assert_array_equal(a.codes[w], b.codes[w])


def test_calls_on_a_side_stream_and_two_at_once(have_gpu):
    """Two calls in flight on two streams, each with its own workspace."""
    import torch

    rng = np.random.default_rng(40)
    c, table = filled(rng, [500, 77], 32, 2, 128)
    x, q = rounded(rng.normal(0, 1, (3, 8 * 128)), "f32")
    d1, d2 = (Dev(c, table, [500, 77], [0, 2, 3], 3) for _ in range(2))
    ref_out = torch.zeros(3, 8 * 128, device="cuda")
    d1.attend(q, ref_out, 8, False, "f32")
    torch.cuda.synchronize()
    outs = [torch.zeros(3, 8 * 128, device="cuda") for _ in range(2)]
    ws = [d.workspace(8) for d in (d1, d2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for d, o, s, w in zip((d1, d2), outs, streams, ws):
            d.attend(q, o, 8, False, "f32", ws=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, ref_out)


def test_host_memory_is_refused(have_gpu):
    import torch

    rng = np.random.default_rng(2)
    c, table = filled(rng, [20], 16, 1, 128)
    d = Dev(c, table, [20], [0, 1], 1)
    host = torch.zeros(1, 128)
    x = torch.zeros(1, 128, device="cuda")
    with pytest.raises(EngineError, match="not device memory"):
        d.append(host, x, "f32")
    with pytest.raises(EngineError, match="not device memory"):
        d.attend(x, host, 1, False, "f32")
    with pytest.raises(EngineError, match="not device memory"):
        d.attend(host.pin_memory(), x, 1, False, "f32")


# ------------------------------------------------------------------ wide batches, long contexts, far pages


def random_cache(rng, pages, page, nkv, hd):
    """Planes of any codes, steps and least values as normed rows have them."""
    c = ref.Cache(pages, page, nkv, hd)
    for w in "kv":
        c.codes[w] = rng.integers(0, 256, c.codes[w].shape).astype(np.uint8)
        s, b = (rng.uniform(*r, c.pairs[w].shape).astype(np.float32).view(np.uint32) for r in ((0.05, 0.3), (-2, -1)))
        c.pairs[w] = (s >> np.uint32(16)) | (b & np.uint32(0xFFFF0000))
    return c


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [65, 300, 1024])
def test_attention_of_many_sequences(have_gpu, kind, n):
    """More sequences than lanes, rows of none to many among them, pages shared."""
    rng = np.random.default_rng(n)
    page, nkv, hd = 16, 1, 128
    lens = rng.integers(0, 41, n)
    rows = np.minimum(rng.integers(0, 3, n), lens + 1)
    lens[n // 2], rows[n // 2] = 150, 90
    lens[n - 1], rows[n - 1] = 70, 1
    table = rng.integers(0, 50, (n, 10)).astype(np.uint32)
    attention_case(n, 4, nkv, hd, page, lens, rows, kind, False, cache=(random_cache(rng, 50, page, nkv, hd), table))


@pytest.mark.parametrize("n", [65, 1024])
def test_append_to_many_sequences(have_gpu, n):
    rng = np.random.default_rng(n)
    page, nkv, hd = 16, 2, 128
    lens = rng.integers(0, 35, n)
    rows = np.minimum(rng.integers(0, 3, n), lens)
    table, pages = tables(rng, lens, page)
    host = ref.Cache(pages, page, nkv, hd)
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    x, t = rounded(rng.normal(0, 1, (2, total, nkv * hd)), "bf16")
    d = Dev(host, table, lens, start, total)
    d.append(t[0], t[1], "bf16")
    got = d.back()
    for b in range(n):
        for r in range(start[b], start[b + 1]):
            for j, w in enumerate("kv"):
                host.write(table[b], int(lens[b] - (start[b + 1] - r)), w, x[j, r].reshape(nkv, hd))
    for w in "kv":
        np.testing.assert_array_equal(got.codes[w], host.codes[w])
        np.testing.assert_array_equal(got.pairs[w], host.pairs[w])


LONG = [
    ((16, 2, 256), [9000], [1]),
    ((32, 8, 128), [4000, 100, 2500], [1, 1, 2]),
    ((6, 2, 128), [3001], [5]),
    ((8, 2, 256), [1500], [130]),
    ((16, 1, 128), [1200], [600]),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_attention_in_many_parts(have_gpu, kind, case):
    heads, lens, rows = LONG[case]
    rng = np.random.default_rng(case)
    page = [128, 16, 64][case % 3]
    table, pages = tables(rng, lens, page)
    attention_case(case, *heads, page, lens, rows, kind, case % 2 == 0,
                   cache=(random_cache(rng, pages, page, heads[1], heads[2]), table))


@pytest.mark.parametrize("case", range(len(LONG)))
def test_nothing_is_written_past_the_workspace(have_gpu, case):
    import torch

    (nh, nkv, hd), lens, rows = LONG[case]
    rng = np.random.default_rng(case)
    table, pages = tables(rng, lens, 64)
    start = np.concatenate([[0], np.cumsum(rows)])
    d = Dev(random_cache(rng, pages, 64, nkv, hd), table, lens, start, int(start[-1]))
    need = d.workspace(nh).numel()
    ws = torch.full((need + 65536,), 0x5A, dtype=torch.uint8, device="cuda")
    q = torch.randn(int(start[-1]), nh * hd, device="cuda")
    out = torch.zeros_like(q)
    d.attend(q, out, nh, False, "f32", ws=ws[:need])
    torch.cuda.synchronize()
    assert torch.all(ws[need:] == 0x5A) and torch.isfinite(out).all()
    with pytest.raises(EngineError, match="workspace smaller"):
        d.attend(q, out, nh, False, "f32", ws=ws[:need - 1])


def test_two_graphs_at_once(have_gpu):
    """Two captured calls with workspaces of their own, replayed together."""
    import torch

    rng = np.random.default_rng(50)
    c, table = filled(rng, [600, 130], 32, 2, 128)
    _, q = rounded(rng.normal(0, 1, (2, 40, 8 * 128)), "f32")
    d = [Dev(c, table, [600, 130], s, 40) for s in ([0, 1, 40], [0, 39, 40])]
    want = [torch.zeros(40, 8 * 128, device="cuda") for _ in d]
    out = [torch.zeros(40, 8 * 128, device="cuda") for _ in d]
    for a, x, w in zip(d, q, want):
        a.attend(x, w, 8, False, "f32")
    ws = [a.workspace(8) for a in d]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in d]
    for a, x, o, w, s in zip(d, q, out, ws, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            a.attend(x, o, 8, False, "f32", ws=w, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for _ in range(10):
        for o in out:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert torch.equal(o, w)


def test_pages_past_32_bits_of_bytes(have_gpu):
    """A cache whose planes of codes pass 4 GiB: its last pages written, read
    back and attended."""
    import torch

    rng = np.random.default_rng(60)
    nkv, hd, page, pages, n, rows = 2, 256, 4096, 4200, 5000, 3
    far = np.array([[pages - 1, pages - 2]], np.uint32)
    host = random_cache(rng, 2, page, nkv, hd)
    d = Dev(host, far, [n], [0, rows], rows)
    big = [torch.empty((pages, *p.shape[1:]), dtype=p.dtype, device="cuda") for p in d.planes]
    for b, p in zip(big, d.planes):
        b[pages - 1], b[pages - 2] = p[0], p[1]
    d.cache = abi.ChkKvQ4(*(b.data_ptr() for b in big), pages, page, nkv, hd)
    x, t = rounded(rng.normal(0, 1, (2, rows, nkv * hd)), "f32")
    d.append(t[0], t[1], "f32")
    near = np.array([[0, 1]], np.uint32)
    for r in range(rows):
        for j, w in enumerate("kv"):
            host.write(near[0], n - rows + r, w, x[j, r].reshape(nkv, hd))
    torch.cuda.synchronize()
    for w, code, pair in zip("kv", big[:2], big[2:]):
        for i in range(2):
            np.testing.assert_array_equal(code[pages - 1 - i].cpu().numpy(), host.codes[w][i])
            np.testing.assert_array_equal(pair[pages - 1 - i].cpu().numpy().view(np.uint32), host.pairs[w][i])
    back = torch.zeros(2, rows, nkv * hd, device="cuda")
    d.read(back[0], back[1], "f32")
    nh = 8
    xq, q = rounded(rng.normal(0, 1, (rows, nh * hd)), "f32")
    out = torch.zeros_like(q)
    d.attend(q, out, nh, False, "f32")
    torch.cuda.synchronize()
    for r in range(rows):
        for j, w in enumerate("kv"):
            np.testing.assert_allclose(back[j, r].cpu().numpy(), host.read(near[0], n - rows + r, w).reshape(-1),
                                       rtol=2.0**-23, atol=1e-30)
    want, vmax, smax = ref.attend(host, near, [n], [0, rows], xq.reshape(rows, nh, hd), nh, False)
    assert np.all(np.abs(out.cpu().numpy().reshape(rows, nh, hd) - want) <= ref.tolerance("f32", hd, want, vmax, smax))


def test_codes_at_the_borders_between_two(have_gpu):
    """Values on (k + 1/2) s, where the even code wins, and one f32 to either
    side, for steps from the least to the largest."""
    nkv, hd, page, n = 2, 128, 16, 512
    rng = np.random.default_rng(70)
    steps = np.concatenate([np.arange(-126, 121), rng.integers(-126, -95, 100), rng.integers(-126, 121, 165)])
    mant = np.concatenate([rng.integers(128, 256, 412), np.full(100, 255)])
    mant[:20] = 128 + np.arange(20)
    s = np.ldexp(mant / 128.0, steps).astype(np.float32)
    x = np.zeros((n, nkv * hd // 64, 64), np.float32)
    k = np.arange(15) + 0.5
    tie = (s[:, None] * k).astype(np.float32)  # 13 bits: exact
    groups = x.reshape(n, -1, 64)
    groups[:, :, 0:15] = tie[:, None]
    groups[:, :, 15:30] = np.nextafter(tie, np.float32(np.inf))[:, None]
    groups[:, :, 30:45] = np.nextafter(tie, np.float32(0))[:, None]
    groups[:, :, 45] = (s * 15)[:, None]
    groups[:, :, 47:] = (s[:, None, None] * rng.uniform(0, 15, (n, 4, 17))).astype(np.float32)
    table = np.arange(n // page, dtype=np.uint32)[None]
    host = ref.Cache(n // page, page, nkv, hd)
    t = dev(x.reshape(n, -1))
    d = Dev(host, table, [n], [0, n], n)
    d.append(t, t, "f32")
    got = d.back()
    for r in range(n):
        for w in "kv":
            host.write(table[0], r, w, x[r].reshape(nkv, hd))
    for w in "kv":
        np.testing.assert_array_equal(got.pairs[w], host.pairs[w])
        np.testing.assert_array_equal(got.codes[w], host.codes[w])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,rows", [([150, 33], [5, 1]), ([150, 33], [40, 30])])
def test_queries_that_are_not_finite_stay_in_their_row(have_gpu, kind, lens, rows):
    import torch

    rng = np.random.default_rng(80)
    nkv, hd, page, nh = 2, 128, 16, 8
    c, table = filled(rng, lens, page, nkv, hd)
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    x = rng.normal(0, 1, (total, nh, hd)).astype(np.float32)
    bad = [(0, 0, np.nan), (2, 5, np.inf), (4, 7, -np.inf), (total - 1, 3, np.nan)]
    for r, h, v in bad:
        x[r, h, 17 * h % hd] = v
    x, q = rounded(x.reshape(total, -1), kind)
    d = Dev(c, table, lens, start, total)
    out = torch.zeros_like(q)
    d.attend(q, out, nh, False, kind)
    got = out.float().cpu().numpy().reshape(total, nh, hd)
    with np.errstate(all="ignore"):
        want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False)
    fine = np.ones((total, nh), bool)
    for r, h, _ in bad:
        fine[r, h] = False
        assert np.isnan(got[r, h]).all()
    tol = ref.tolerance(kind, hd, want, vmax, smax)
    assert np.all(np.abs(got - want)[fine] <= tol[fine])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [(130, 1, 128), (65, 1, 256), (128, 2, 128)])
def test_one_token_of_many_heads(have_gpu, kind, heads):
    """More heads a kv head than a block of few pairs holds."""
    rng = np.random.default_rng(81)
    nh, nkv, hd = heads
    table, pages = tables(rng, [300, 1], 32)
    attention_case(81, nh, nkv, hd, 32, [300, 1], [1, 1], kind, False,
                   cache=(random_cache(rng, pages, 32, nkv, hd), table))


def test_attention_of_the_indexers_choice(have_gpu):
    """chk_qsa_select's words, row by row, as the mask of a batch's rows."""
    import torch

    rng = np.random.default_rng(82)
    nkv, hd, page, nh, ratio, kblk = 2, 256, 64, 16, 4, 40
    lens, rows = [700, 150], [3, 1]  # the second has 37 complete blocks: all visible
    table, pages = tables(rng, lens, page)
    c = random_cache(rng, pages, page, nkv, hd)
    start = np.concatenate([[0], np.cumsum(rows)])
    total, words = int(start[-1]), (max(lens) // ratio + 1 + 31) // 32
    bits = torch.zeros(total, words, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        for r in range(start[b], start[b + 1]):
            t_len = int(n - (start[b + 1] - r) + 1)
            score = torch.rand(t_len // ratio + 1, device="cuda")
            check(lib().chk_qsa_select(score.data_ptr(), t_len, kblk, ratio, bits[r].data_ptr(), None))
    torch.cuda.synchronize()
    host = bits.cpu().numpy().view(np.uint32)
    chosen = [sum(bin(int(w)).count("1") for w in row) for row in host]
    assert chosen[:3] == [kblk] * 3 and chosen[3] == 0
    x, q = rounded(rng.normal(0, 1, (total, nh * 2 * hd)), "f32")
    d = Dev(c, table, lens, start, total)
    out = torch.zeros(total, nh * hd, device="cuda")
    d.attend(q, out, nh, True, "f32", (host, ratio, kblk))
    want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(total, nh, 2 * hd), nh, True, (host, ratio, kblk))
    got = out.cpu().numpy().reshape(total, nh, hd)
    assert np.all(np.abs(got - want) <= ref.tolerance("f32", hd, want, vmax, smax))


# heads whose single tokens fold over a block's columns, fill them and pass them
@pytest.mark.parametrize("heads", [(1, 1, 128), (2, 1, 128), (4, 1, 128), (3, 1, 128), (8, 2, 128), (5, 1, 128), (16, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_single_tokens_of_extreme_caches(have_gpu, kind, heads):
    """Single tokens over values of very different size, over scores far apart,
    over pairs that are not finite and pages that are missing."""
    import torch

    nh, nkv, hd = heads
    rng = np.random.default_rng(90)
    page, lens, rows = 16, [200, 77, 130, 16], [1, 1, 1, 1]
    c, table = filled(rng, lens, page, nkv, hd)
    for t, size in ((3, 1e-30), (70, 1e10), (120, 1e3), (199, 1e-6)):
        c.write(table[0], t, "v", (size * rng.normal(0, 1, (nkv, hd))).astype(np.float32))
    for t in range(0, 77, 9):  # scores far apart
        c.write(table[1], t, "k", (300 * rng.normal(0, 1, (nkv, hd))).astype(np.float32))
    at = c.place(table[2], 100)
    for w in "kv":
        c.pairs[w][at[0], nkv - 1, at[1], 0] = 0x7FC07FC0
    table[3, 0] = 60000
    start = [0, 1, 2, 3, 4]
    for scale in (1.0, 40.0):
        x, q = rounded(scale * rng.normal(0, 1, (4, nh * hd)), kind)
        d = Dev(c, table, lens, start, 4)
        out = torch.zeros(4, nh * hd, dtype=torch_type(kind), device="cuda")
        d.attend(q, out, nh, False, kind)
        got = out.float().cpu().numpy().reshape(4, nh, hd)
        with np.errstate(all="ignore"):
            want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(4, nh, hd), nh, False)
        g = nh // nkv
        assert np.isnan(got[3]).all() and np.isnan(got[2, nh - g:]).all()
        assert np.isfinite(got[2, :nh - g]).all()
        ok = np.isfinite(want).all(axis=2)
        assert ok[:2].all()
        tol = ref.tolerance(kind, hd, want, vmax, smax)
        # f16 ends at 2^15 (2 - 2^-10) = 65504, its step there 2^5: what is 65520 or
        # more before its one rounding is infinite in f16, and so may be a result
        # whose tolerance reaches that (the values of 1e10)
        past = (kind == "f16") & (np.abs(want) + tol >= 65520) & np.isinf(got)
        assert np.all(past[ok[:, :, None] & np.isinf(got)])
        near = ok[:, :, None] & ~past
        assert np.all(np.abs(got - want)[near] <= tol[near]), scale


# ------------------------------------------------------------------ errors beyond the type's rounding


def errors(seed, heads, lens, rows, kind, q_of=None, k_of=None):
    """(got, want, smax) of a call over normal queries, keys and values, or
    those of q_of(rng, shape) and k_of(rng, shape)."""
    import torch

    rng = np.random.default_rng(seed)
    nh, nkv, hd = heads
    normal = lambda rng, shape: rng.normal(0, 1, shape)  # noqa: E731
    table, pages = tables(rng, lens, 32)
    c = ref.Cache(pages, 32, nkv, hd)
    for b, n in enumerate(lens):
        k, v = (of(rng, (n, nkv, hd)).astype(np.float32) for of in (k_of or normal, normal))
        for t in range(n):
            c.write(table[b], t, "k", k[t])
            c.write(table[b], t, "v", v[t])
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    x, q = rounded((q_of or normal)(rng, (total, nh * hd)), kind)
    d = Dev(c, table, lens, start, total)
    out = torch.zeros(total, nh * hd, dtype=torch_type(kind), device="cuda")
    d.attend(q, out, nh, False, kind)
    got = out.double().cpu().numpy().reshape(total, nh, hd)
    want, _, smax = ref.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False)
    return got, want, smax


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads,lens,rows", [((4, 1, 128), [400, 90], [1, 1]), ((16, 2, 128), [400], [2]), ((8, 1, 256), [300], [3]),
                                             ((8, 1, 128), [300], [40]), ((4, 2, 256), [260], [70])])
def test_scores_that_are_small_differences(have_gpu, kind, heads, lens, rows):
    """Queries whose elements are all near 200 over keys that order the same
    values differently: scores differ by some units, and the sums of a group's
    codes that they come from are a hundred times that where codes count from
    0, and thousands where they count from further below."""
    def orders(rng, shape):
        values = rng.normal(0, 1, 64)
        return rng.permuted(np.broadcast_to(values, (*shape[:-1], shape[-1] // 64, 64)), axis=-1).reshape(shape)

    got, want, smax = errors(91, heads, lens, rows, kind, lambda rng, s: 200 + rng.normal(0, 1, s), orders)
    off, limit = ref.beyond_rounding(kind, got, want), ref.beyond_limit(kind, smax)
    assert off <= limit, (off, limit)


# heads, lens, rows, and whether a sequence has more than 64 (row, head) pairs a kv head
ERRORS = [
    ((4, 1, 128), [500, 130, 77], [1, 1, 1], False),  # folded over a tile's columns
    ((32, 2, 128), [700, 33], [1, 3], False),
    ((24, 2, 256), [400, 64], [1, 2], False),
    ((12, 1, 256), [900], [5], False),
    ((8, 2, 128), [300], [60], True),
    ((4, 1, 128), [450, 200], [90, 33], True),
    ((8, 1, 256), [333], [77], True),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ERRORS)))
def test_errors_beyond_the_types_rounding(have_gpu, kind, case):
    """Every operand at the bits it is said to have: two f16 parts, one for the
    numerators of bf16 rows where a sequence has many pairs."""
    heads, lens, rows, many = ERRORS[case]
    got, want, smax = errors(100 + case, heads, lens, rows, kind)
    off = ref.beyond_rounding(kind, got, want)
    limit = ref.beyond_limit(kind, smax, 1 if kind == "bf16" and many else 2)
    assert off <= limit, (off, limit)


# ------------------------------------------------------------------ value groups of one number


def constant_case(name, rng, n, nkv, hd):
    """Values [n][nkv][hd] whose groups hold one number of bf16 each."""
    v = np.ones((n, nkv, hd), np.float32)
    if name == "2^30":
        v *= 2.0**30
    elif name == "-3e38":
        v *= -np.float32(2.0**127 * 1.75)
    elif name == "1e30 and 1e-30":  # a group of each
        v[:, :, :64] *= 2.0**100
        v[:, :, 64:] *= 2.0**-100
    elif name == "t":
        v *= np.arange(n)[:, None, None]
    elif name == "beside normal":
        v[::3] *= 2.0**40
        v[1::3] *= 3.0
        v[2::3] = rng.normal(0, 1, v[2::3].shape)
    else:  # one group of a row constant
        v = rng.normal(0, 1, v.shape).astype(np.float32)
        v[:, :, :64] = 2.0**27
    return ref.bf16_round(v.astype(np.float32), False)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["2^30", "-3e38", "1e30 and 1e-30", "t", "beside normal", "one group"])
@pytest.mark.parametrize("heads,lens,rows", [((4, 1, 128), [1, 256, 250], [1, 1, 1]), ((16, 2, 128), [250, 1], [1, 1]),
                                             ((4, 1, 256), [250, 1], [3, 1])])
def test_value_groups_of_one_number(have_gpu, kind, name, heads, lens, rows):
    """Rows of a constant, of any size: their steps are the least there is."""
    import torch

    rng = np.random.default_rng(110)
    nh, nkv, hd = heads
    table, pages = tables(rng, lens, 32)
    c = ref.Cache(pages, 32, nkv, hd)
    for b, n in enumerate(lens):
        v = constant_case(name, rng, n, nkv, hd)
        for t in range(n):
            # scores that rise along the sequence, by some 8 powers of two in all
            c.write(table[b], t, "k", np.full((nkv, hd), 6 * t / max(n, 2), np.float32))
            c.write(table[b], t, "v", v[t])
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    x, q = rounded(np.full((total, nh * hd), hd**-0.5), kind)
    d = Dev(c, table, lens, start, total)
    out = torch.zeros(total, nh * hd, dtype=torch_type(kind), device="cuda")
    d.attend(q, out, nh, False, kind)
    got = out.double().cpu().numpy().reshape(total, nh, hd)
    want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False)
    # (a group's tolerance is its own values')
    off = np.zeros(want.shape)
    for g in range(hd // 64):
        dims = slice(64 * g, 64 * g + 64)
        most = np.zeros((total, nh))
        for b, n in enumerate(lens):
            v = np.abs(np.stack([c.read(table[b], t, "v")[:, dims] for t in range(n)]))
            for r in range(start[b], start[b + 1]):
                seen = v[:n - (start[b + 1] - r) + 1].max((0, 2))
                most[r] = seen.repeat(nh // nkv)
        off[..., dims] = np.abs(got - want)[..., dims] - ref.tolerance(kind, hd, want[..., dims], most, smax)
    if kind == "f16":  # past its range both are infinite
        past = np.abs(want) >= 65520
        assert np.array_equal(np.isinf(got[past]), np.ones(past.sum(), bool))
        off[past] = 0
    assert np.all(off <= 0), np.nanmax(off)


@pytest.mark.parametrize("heads,n,rows", [((1, 1, 128), 1024, 1), ((1, 1, 256), 1024, 1), ((1, 1, 128), 256, 70)])
def test_small_values_over_many_tokens(have_gpu, heads, n, rows):
    """2^18 tokens of one small number, the first ones' scores 7.9 powers of two
    below the others': the sum of the numerators, which count that high where
    values are small, stays in f32.  (As many sequences over the same pages as
    leave each block one part.)"""
    import torch

    nh, nkv, hd = heads
    page, tokens = 1024, 2**18
    c = ref.Cache(tokens // page, page, nkv, hd, fill=0)
    for w, s, b in (("k", 1.0, 0.0), ("v", 2.0**-126, 2.0**-100)):
        s, b = (np.float32(a).view(np.uint32) for a in (s, b))
        c.pairs[w][:] = (s >> np.uint32(16)) | b
    low = np.float32(-7.9 / np.log2(np.e)).view(np.uint32) & np.uint32(0xFFFF0000)
    c.pairs["k"][0, :, :256] = (np.float32(1.0).view(np.uint32) >> np.uint32(16)) | low
    table = np.broadcast_to(np.arange(tokens // page, dtype=np.uint32), (n, tokens // page))
    start = rows * np.arange(n + 1)
    d = Dev(c, table, [tokens] * n, start, rows * n)
    q = torch.full((rows * n, nh * hd), hd**-0.5, device="cuda")
    out = torch.zeros(rows * n, nh * hd, device="cuda")
    d.attend(q, out, nh, False, "f32")
    # every value is 2^-100.  Equal terms may round the same way each time: a lane
    # adds at most a quarter of the 2^18 numerators one by one, half a step (2^-24)
    # of a sum that grows evenly each, 2^16 2^-24 / 2 = 2^-9 of the last; the
    # products' sums take 32 tokens at a time, 2^13 2^-24 / 2 = 2^-12
    assert torch.all((out.double() - 2.0**-100).abs() <= 2.0**-100 * (2.0**-9 + 2.0**-12))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,lens,rows", [((4, 1, 128), [90, 1], [1, 1]), ((16, 1, 128), [90], [1]), ((6, 2, 256), [200], [1]),
                                             ((8, 1, 128), [100], [30]), ((4, 1, 256), [300], [30])])
def test_values_of_zero(have_gpu, kind, heads, lens, rows):
    """Rows of zeros give zeros, and so does a group of zeros beside others."""
    import torch

    rng = np.random.default_rng(120)
    nh, nkv, hd = heads
    table, pages = tables(rng, lens, 16)
    for others in (0.0, 1.0):
        total = sum(lens)
        x, t = rounded(rng.normal(0, 1, (2, total, nkv, hd)), kind)
        t[1, :, :, :64] = 0
        t[1, :, :, 64:] *= others
        d = Dev(ref.Cache(pages, 16, nkv, hd), table, lens, np.concatenate([[0], np.cumsum(lens)]), total)
        t = t.reshape(2, total, -1)
        d.append(t[0], t[1], kind)
        start = np.concatenate([[0], np.cumsum(rows)])
        _, q = rounded(rng.normal(0, 1, (int(start[-1]), nh * hd)), kind)
        out = torch.ones_like(q)
        e = Dev(d.back(), table, lens, start, len(q))
        e.attend(q, out, nh, False, kind)
        out = out.float().cpu().numpy().reshape(-1, nh, hd)
        assert np.all(out[..., :64] == 0) and np.all((out[..., 64:] != 0) == (others != 0))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ratio", [6, 12, 18, 24])
@pytest.mark.parametrize("heads,lens,rows", [((4, 1, 128), [150, 40], [1, 1]), ((24, 2, 256), [150], [1]), ((8, 1, 128), [150, 70], [40, 20]),
                                             ((6, 1, 256), [120], [60])])
def test_value_groups_of_unlike_size(have_gpu, kind, ratio, heads, lens, rows):
    """The second group of 64 dims louder than the others by 2^ratio: each
    group's error against its own values, and what the documentation grants."""
    import torch

    rng = np.random.default_rng(130)
    nh, nkv, hd = heads
    table, pages = tables(rng, lens, 32)
    c = ref.Cache(pages, 32, nkv, hd)
    for b, n in enumerate(lens):
        k, v = rng.normal(0, 1, (2, n, nkv, hd)).astype(np.float32)
        v[:, :, 64:128] *= 2.0**ratio
        v *= 2.0**-14  # (f16 holds them)
        for t in range(n):
            c.write(table[b], t, "k", k[t])
            c.write(table[b], t, "v", v[t])
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    x, q = rounded(rng.normal(0, 1, (total, nh * hd)), kind)
    d = Dev(c, table, lens, start, total)
    out = torch.zeros(total, nh * hd, dtype=torch_type(kind), device="cuda")
    d.attend(q, out, nh, False, kind)
    got = out.double().cpu().numpy().reshape(total, nh, hd)
    want, vmax, smax = ref.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False)
    many = max(rows) * nh // nkv > 64
    for g in range(hd // 64):
        dims = slice(64 * g, 64 * g + 64)
        most = np.zeros((total, nh))
        for b, n in enumerate(lens):
            v = np.abs(np.stack([c.read(table[b], t, "v")[:, dims] for t in range(n)]))
            for r in range(start[b], start[b + 1]):
                most[r] = v[:n - (start[b + 1] - r) + 1].max((0, 2)).repeat(nh // nkv)
        tol = ref.tolerance(kind, hd, want[..., dims], most, smax)
        # many pairs: the operands of a group 2^18 below the loudest are exact
        if not many or ratio > 18:
            tol = tol + 2.0**-29 * vmax[..., None]
        off = np.abs(got - want)[..., dims]
        assert np.all(off <= tol), (g, float((off - tol).max()), float(off.max()))


@pytest.mark.parametrize("kind,bits", [("f32", 0xFFFFFFFF), ("f32", 0xFFFF0001), ("f32", 0x7FFFFFFF), ("f16", 0xFFFF), ("f16", 0x7FFF),
                                       ("f16", 0xFE00), ("bf16", 0xFFFF), ("bf16", 0x7FFF), ("bf16", 0xFFC0)])
def test_append_of_any_nan(have_gpu, kind, bits):
    """A NaN of any bits makes its group NaN, and no other."""
    import torch

    rng = np.random.default_rng(140)
    n, hd = 16, 128
    x, t = rounded(rng.normal(0, 1, (n, hd)), kind)
    raw = t.view(torch.int32 if kind == "f32" else torch.int16)
    width = 32 if kind == "f32" else 16
    bad = bits - (1 << width) if bits >> (width - 1) else bits
    for r in range(0, n, 2):
        raw[r, (5 * r) % hd] = bad
    raw[1, :64] = bad
    x = t.float().cpu().numpy()
    host = ref.Cache(1, 16, 1, hd)
    d = Dev(host, [[0]], [n], [0, n], n)
    d.append(t, t, kind)
    got = d.back()
    for r in range(n):
        for w in "kv":
            host.write(np.array([0]), r, w, x[r][None])
    for w in "kv":
        np.testing.assert_array_equal(got.pairs[w], host.pairs[w])
        np.testing.assert_array_equal(got.codes[w], host.codes[w])
    assert (got.pairs["k"] == 0x7FC07FC0).sum() == n // 2 + 1


@pytest.mark.parametrize("up,down", [(80, -78), (-78, 80), (-100, 95), (90, -120)])
@pytest.mark.parametrize("rows", [1, 40])
def test_scores_of_large_times_small(have_gpu, rows, up, down):
    """Queries and keys of very different size, f32: their scores are ordinary."""
    got, want, smax = errors(150, (4, 2, 128), [200], [rows], "f32", lambda rng, s: np.ldexp(rng.normal(0, 1, s), up),
                             lambda rng, s: np.ldexp(rng.normal(0, 1, s), down))
    assert ref.beyond_rounding("f32", got, want) <= ref.beyond_limit("f32", smax)


@pytest.mark.parametrize("heads,batch", [((16, 2, 256), 5), ((4, 1, 128), 3), ((4, 2, 128), 7), ((8, 1, 128), 9)])
@pytest.mark.parametrize("bits", [Bits(4, 0, 0.3), Bits(4, 10, 0.1), Bits(64, 1, 0.5)], ids=["4", "4_budget", "64"])
def test_attention_of_chosen_blocks_in_f16(have_gpu, bits, heads, batch):
    lens, rows = ROWS[batch]
    attention_case(160 + batch, *heads, 32, lens, rows, "f16", batch % 2 == 1, bits)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("loud", ["keys", "queries"])
@pytest.mark.parametrize("heads,lens,rows", [((4, 1, 128), [150, 40], [1, 1]), ((24, 2, 256), [150], [1]), ((8, 1, 128), [150, 70], [40, 20]),
                                             ((6, 1, 256), [120], [60])])
def test_scores_of_groups_of_unlike_size(have_gpu, kind, loud, heads, lens, rows):
    """A group of 64 dims 2^12 louder than the others, in the keys or in the
    queries, against zeros in the other: the scores are the other groups'."""
    def scaled(factor):
        def of(rng, shape):
            x = rng.normal(0, 1, shape).reshape(*shape[:-1], -1, heads[2])
            x[..., 64:128] *= factor
            return x.reshape(shape)
        return of

    of_q, of_k = (0.0, 2.0**12) if loud == "keys" else (2.0**12, 0.0)
    got, want, smax = errors(170, heads, lens, rows, kind, scaled(of_q), scaled(of_k))
    parts = 1 if kind == "bf16" and max(rows) * heads[0] // heads[1] > 64 else 2
    # the quiet queries' second part ends 2^-31 of the loudest: 2^-19 of a score's
    # parts, as 2^-21 of four times smax
    assert ref.beyond_rounding(kind, got, want) <= ref.beyond_limit(kind, 4 * smax, parts)
