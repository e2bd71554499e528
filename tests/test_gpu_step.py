"""A serving step's calls around the 4-bit cache on the GPU (chk_kv_plan_q4,
chk_qk_norm_rope): every array of a plan against plain Python, steps in a row,
taken back, in graphs and on states that are not sound; heads normed and turned
against 64 bits at far positions, odd turns, in place and strided."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from cherenkov_amd.abi import EngineError, check, lib
from tests import step_ref as ref
from tests.test_gpu_kv4 import KINDS, dev, rounded

pytestmark = pytest.mark.gpu

CANARY = 0x5A5A5A5A


class Guarded:
    """A device array of u32 (or u64) words between words that no call may touch."""

    def __init__(self, a, dtype=np.uint32):
        import torch

        self.a = np.ascontiguousarray(a, dtype)
        words = self.a.view(np.uint32).ravel()
        self.n = len(words)
        pad = np.full(64, CANARY, np.uint32)
        self.t = torch.from_numpy(np.concatenate([pad, words, pad]).view(np.int32)).cuda()
        self.ptr = self.t.data_ptr() + 256

    def back(self, sound=True):
        got = self.t.cpu().numpy().view(np.uint32)
        assert np.all(got[:64] == CANARY) and np.all(got[64 + self.n:] == CANARY), "written outside"
        return got[64:64 + self.n].view(self.a.dtype).reshape(self.a.shape)


class Pool:
    def __init__(self, table, length, free, nfree, page, pages, rows):
        n, width = table.shape
        self.table, self.len, self.free = Guarded(table), Guarded(length), Guarded(free)
        self.nfree = Guarded(np.array([nfree, 77]))
        self.start, self.pos = Guarded(np.full(n + 1, 9)), Guarded(np.full(max(rows, 1), 9))
        self.slot = Guarded(np.full(max(rows, 1), 9), np.uint64)
        self.rows, self.page, self.pages = rows, page, pages
        self.c = abi.ChkKvPool(self.table.ptr, self.len.ptr, self.free.ptr, self.nfree.ptr, n, width, page, pages)

    def plan(self, want, keep=None, own=None, stream=None, pos=True, slot=True):
        self.args = [None if a is None else Guarded(a) for a in (keep, own, want)]
        self.call(stream, pos, slot)

    def call(self, stream=None, pos=True, slot=True):
        k, o, w = (a and a.ptr for a in self.args)
        check(lib().chk_kv_plan_q4(C.byref(self.c), k, o, w, self.rows, self.start.ptr, self.pos.ptr if pos else None,
                                   self.slot.ptr if slot else None, stream))

    def state(self):
        import torch

        torch.cuda.synchronize()
        return [x.back() for x in (self.table, self.len, self.free, self.nfree, self.start)] + [
            self.pos.back()[:self.rows], self.slot.back()[:self.rows]]


NAMES = ("table", "len", "free", "nfree", "start", "pos", "slot")


def same(got, want, names=NAMES):
    for g, w, name in zip(got, want, names):
        np.testing.assert_array_equal(g, w, err_msg=name)


def state_of(rng, n, page, most, spare, width=None):
    """Sequences of up to `most` tokens, their pages anywhere, `spare` free ones."""
    length = rng.integers(0, most + 1, n)
    held = -(-length // page)
    width = width or int(held.max()) + 3
    pages = int(held.sum()) + spare + 4
    ids = rng.permutation(pages)
    table = np.full((n, width), ref.NONE, np.uint32)
    at = 0
    for b in range(n):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = np.full(pages, ref.NONE, np.uint32)
    free[:spare] = ids[at:at + spare]
    return table, length.astype(np.uint32), free, spare, pages


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 300, 1024])
@pytest.mark.parametrize("spare", [0, 3, 400])
def test_plan(have_gpu, n, page, spare):
    """Three steps in a row, each array whole, of cut-back, ended and growing
    sequences, some on pages of another's, wants that do not all find room."""
    rng = np.random.default_rng(n * 7 + page + spare)
    table, length, free, nfree, pages = state_of(rng, n, page, 5 * page, spare)
    rows = int(rng.integers(1, 40 * n + 50))
    p = Pool(table, length, free, nfree, page, pages, rows)
    for step in range(3):
        held = -(-length.astype(np.int64) // page)
        own = np.where(rng.random(n) < 0.2, np.minimum(held, 1), 0)
        keep = np.maximum(length.astype(np.int64) - rng.integers(0, 2 * page, n) * (rng.random(n) < 0.5), 0)
        keep[rng.random(n) < 0.1] = 0
        keep[rng.random(n) < 0.1] = ref.NONE
        want = np.where(rng.random(n) < 0.6, 1, rng.integers(0, 70, n))
        if step == 1:
            want[n // 2] = 0xFFFFFFFF if n % 2 else 2 * rows + 1
        args = [keep if step else None, own if step != 1 else None]
        p.plan(want, *args)
        want_state = ref.plan(table, length, free, nfree, *args, want, rows, page, pages)
        same(p.state(), want_state)
        table, length, free, (nfree, _) = want_state[:4]


@pytest.mark.parametrize("rows", [4096, 4097, 70000])
def test_plan_of_many_rows(have_gpu, rows):
    """Prompts: both ways of writing the rows, null arrays among them."""
    rng = np.random.default_rng(rows)
    table, length, free, nfree, pages = state_of(rng, 40, 16, 300, 6000, width=1000)
    want = rng.integers(0, rows // 30, 40)
    for pos, slot in [(True, True), (True, False), (False, True), (False, False)]:
        p = Pool(table, length, free, nfree, 16, pages, rows)
        p.plan(want, pos=pos, slot=slot)
        w = list(ref.plan(table, length, free, nfree, None, None, want, rows, 16, pages))
        w[5:] = [w[5] if pos else np.full(rows, 9), w[6] if slot else np.full(rows, 9)]
        same(p.state(), w)


def test_plan_to_the_brim(have_gpu):
    """Rows that fill the row arrays, tables and the pool exactly, and one more."""
    for extra in (0, 1):
        # two sequences of one page each, tables of two; 32 rows fit
        table = np.array([[0, ref.NONE], [1, ref.NONE]], np.uint32)
        p = Pool(table, [16, 16], [2, 3, 9, 9], 2, 16, 4, 32 + extra)
        args = (table, [16, 16], np.array([2, 3, 9, 9], np.uint32), 2, None, None, [16, 16 + extra], 32 + extra, 16, 4)
        p.plan([16, 16 + extra])
        same(p.state(), ref.plan(*args))
        assert p.start.back().tolist() == ([0, 16, 32] if not extra else [0, 16, 16])
        p = Pool(table, [16, 16], [2, 3, 9, 9], 2, 16, 4, 32 - extra)
        p.plan([16, 16])
        assert p.state()[4].tolist() == ([0, 16, 32] if not extra else [0, 16, 16])
    # no rows at all: pages still go back
    p = Pool(table, [16, 16], [2, 3, 9, 9], 2, 16, 4, 0)
    p.plan([0, 1], keep=[0, 16])
    st = p.state()
    assert st[1].tolist() == [0, 16] and st[2].tolist() == [2, 3, 0, 9] and st[3].tolist() == [3, 0]
    assert st[0].tolist() == [[ref.NONE, ref.NONE], [1, ref.NONE]] and st[4].tolist() == [0, 0, 0]


def test_a_step_taken_back_leaves_the_list(have_gpu):
    rng = np.random.default_rng(8)
    table, length, free, nfree, pages = state_of(rng, 200, 16, 200, 900)
    p = Pool(table, length, free, nfree, 16, pages, 9000)
    p.plan(rng.integers(0, 40, 200))
    p.plan(np.zeros(200), keep=length)
    st = p.state()
    np.testing.assert_array_equal(st[2][:nfree], free[:nfree])
    assert st[3].tolist() == [nfree, 0]
    np.testing.assert_array_equal(st[1], length)
    np.testing.assert_array_equal(st[0], table)


def test_plans_of_states_that_are_not_sound(have_gpu):
    """Lengths past the table, more free pages than the pool has, entries that name
    no page, own pages past the table: nothing outside the arrays is touched, and
    sound sequences beside them are served."""
    NONE = ref.NONE
    table = np.array([[5, 6, 7], [8, NONE, 3], [NONE] * 3, [1, 2, NONE], [0xFFFFFFF0, 4, 9]], np.uint32)
    length = np.array([0xFFFFFFFF, 200, 0, 20, 48], np.uint32)
    p = Pool(table, length, np.arange(12), 0xFFFFFFFF, 16, 12, 64)
    p.plan([1, 0xFFFFFFFF, 5, 3, 1], own=[0, 0xFFFFFFFF, 0, 9, 0])
    st = p.state()
    assert st[1][2:4].tolist() == [5, 23] and st[4].tolist() == [0, 0, 0, 5, 8, 8]
    assert st[1][[0, 1, 4]].tolist() == [0xFFFFFFFF, 200, 48]
    # all of it given back: the list ends at the pool's pages
    p.plan([0] * 5, keep=[0] * 5)
    st = p.state()
    assert st[1].tolist() == [0] * 5 and st[3][0] <= 12


def test_plan_in_a_graph(have_gpu):
    """Captured once and replayed on new wants, with eager work between; every
    replay equals the rules."""
    import torch

    rng = np.random.default_rng(12)
    table, length, free, nfree, pages = state_of(rng, 30, 16, 100, 600, width=64)
    for rows in (500, 6000):
        p = Pool(table, length, free, nfree, 16, pages, rows)
        t, ln, fr, nf = table, length, free, nfree
        p.plan(np.zeros(30), keep=np.full(30, ref.NONE))
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            p.call(torch.cuda.current_stream().cuda_stream)
        for _ in range(6):
            want = rng.integers(0, 20, 30)
            keep = np.where(rng.random(30) < 0.2, 0, ln)
            for g, a in zip((p.args[0], p.args[2]), (keep, want)):
                g.t[64:94].copy_(torch.from_numpy(a.astype(np.uint32).view(np.int32)))
            graph.replay()
            w = ref.plan(t, ln, fr, nf, keep, None, want, rows, 16, pages)
            same(p.state(), w)
            t, ln, fr, (nf, _) = w[:4]


# ------------------------------------------------------------------ heads normed and turned


def turns(theta, rot):
    t = (C.c_uint64 * max(rot // 2, 1))()
    check(lib().chk_rope_turns(theta, rot, t))
    return dev(np.frombuffer(t, np.int64))


def norm_case(seed, kind, rows, nh, nkv, hd, gated, rot, theta=1e4, far=5000, inplace=False, normed=(True, True), x_of=None,
              blank=0.2, stream=None):
    import torch

    rng = np.random.default_rng(seed)
    per = hd * (2 if gated else 1)
    wide, pad = nh * per + 2 * nkv * hd, 16
    xv = rng.normal(0, 1.5, (rows, wide + pad)) * np.exp(rng.normal(0, 2, (rows, 1)))
    if x_of:
        xv = x_of(xv)
    x, t = rounded(xv, kind)
    w, wt = rounded(rng.normal(1, 0.4, (2, hd)), "bf16")
    pos = rng.integers(0, far, rows).astype(np.uint32)
    pos[rng.random(rows) < blank] = ref.NONE
    pos_t, eps = dev(pos), 1e-5
    q, k = t[:, :nh * per], t[:, nh * per:nh * per + nkv * hd]
    if inplace:
        qo, ko = q, k
    else:
        qo = torch.full((rows, nh * per + 8), 7.0, dtype=t.dtype, device="cuda")
        ko = torch.full((rows, nkv * hd + 24), 7.0, dtype=t.dtype, device="cuda")
    tt = turns(theta, rot)
    norm = abi.ChkQkNorm(wt[0].data_ptr() if normed[0] else None, wt[1].data_ptr() if normed[1] else None,
                         tt.data_ptr() if rot else None, rot, nh, nkv, hd, int(gated), eps)
    before = t.clone()
    p = lambda a, n: a.data_ptr() if n else None  # noqa: E731
    check(lib().chk_qk_norm_rope(C.byref(norm), pos_t.data_ptr(), rows, p(q, nh), q.stride(0), p(qo, nh), qo.stride(0),
                                 p(k, nkv), k.stride(0), p(ko, nkv), ko.stride(0), KINDS[kind], stream))
    torch.cuda.synchronize()
    live = pos != ref.NONE
    eps32 = float(np.float32(eps))
    got_q, got_k = qo.float().cpu().numpy().astype(np.float64), ko.float().cpu().numpy().astype(np.float64)
    src_q = x[:, :nh * per].reshape(rows, nh, per)
    src_k = x[:, nh * per:nh * per + nkv * hd].reshape(rows, nkv, hd)
    for name, got, src, weight, heads, width in [("q", got_q, src_q, w[0] if normed[0] else None, nh, per),
                                                 ("k", got_k, src_k, w[1] if normed[1] else None, nkv, hd)]:
        if heads == 0:
            continue
        here = got[:, :heads * width].reshape(rows, heads, width)
        want, size = ref.norm_rope(src[..., :hd], weight, eps32, pos.astype(np.float64), theta, rot)
        tol = ref.norm_rope_tolerance(kind, want, size)
        off = np.abs(here[..., :hd] - want)[live]
        assert np.all(off <= tol[live]), f"{name}: {(off / tol[live]).max():.3g} of the tolerance"
        if width > hd:
            np.testing.assert_array_equal(here[live][..., hd:], src[live][..., hd:], err_msg="gates")
        # rows of none, and what lies past a row
        if inplace:
            np.testing.assert_array_equal(here[~live], src[~live])
        else:
            assert np.all(here[~live] == 7.0) and np.all(got[:, heads * width:] == 7.0)
    if inplace:  # the values beside them
        assert torch.equal(t[:, nh * per + nkv * hd:], before[:, nh * per + nkv * hd:])
    else:
        assert torch.equal(t, before)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads", [(16, 2, True), (5, 1, False), (1, 3, False), (0, 4, False), (7, 0, True)])
@pytest.mark.parametrize("rows", [1, 9, 700])
def test_norm_and_rotation(have_gpu, kind, hd, heads, rows):
    nh, nkv, gated = heads
    norm_case(rows + hd, kind, rows, nh, nkv, hd, gated, [hd // 4, hd // 2, hd][(rows + nh) % 3], theta=1e7 if nh > 4 else 1e4,
              inplace=rows == 9, blank=0.0 if rows == 1 else 0.2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [877, 900, 1300, 3500, 9000])
def test_every_row_once(have_gpu, kind, rows):
    """In place, a row taken twice would be normed twice: rows that no share of the
    device's waves divides."""
    norm_case(rows, kind, rows, 16, 2, 256, True, 64, theta=1e7, inplace=True, blank=0.01)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rot", [0, 2, 6, 10, 20, 34, 62, 126, 128])
def test_turns_of_any_width(have_gpu, kind, rot):
    for rows in (3, 2000):
        norm_case(rot, kind, rows, 6, 2, 128, rot % 4 == 2, rot, inplace=rows == 3)


@pytest.mark.parametrize("far", [2**20, 2**31, 2**32 - 1])
def test_far_positions(have_gpu, far):
    """Angles stay exact: a position's fastest pair turns 2^29 times and more."""
    norm_case(far % 97, "f32", 40, 4, 1, 128, False, 128, theta=1e4, far=far, blank=0.0)
    norm_case(far % 89, "f32", 40, 4, 1, 256, False, 64, theta=1e7, far=far, blank=0.0)


@pytest.mark.parametrize("normed", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_heads_that_are_only_turned(have_gpu, kind, normed):
    for rows in (2, 1500):
        norm_case(5, kind, rows, 4, 2, 128, False, 64, normed=normed)


def test_sizes_of_rows(have_gpu):
    """Rows of zeros give zero; sizes from 2^-60 to 2^50 keep their bits."""
    def sizes(x):
        x[::3] *= 2.0**50
        x[1::3] *= 2.0**-60
        x[5] = 0
        return x

    norm_case(3, "f32", 30, 4, 2, 128, False, 64, x_of=sizes, blank=0.0)
    norm_case(4, "bf16", 30, 4, 2, 256, False, 64, x_of=sizes, blank=0.0)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_head_that_is_not_finite_stays_alone(have_gpu, bad):
    import torch

    x = torch.randn(3, 6, 128, device="cuda")
    x[1, 2, 7] = bad
    ok = x.clone()
    ok[1, 2, 7] = 0.0
    w, tt, pos = torch.ones(128, dtype=torch.bfloat16, device="cuda"), turns(1e4, 64), dev(np.arange(3, dtype=np.uint32))
    norm = abi.ChkQkNorm(w.data_ptr(), w.data_ptr(), tt.data_ptr(), 64, 6, 0, 128, 0, 1e-6)
    outs = []
    for a in (x, ok):
        o = torch.zeros_like(a)
        check(lib().chk_qk_norm_rope(C.byref(norm), pos.data_ptr(), 3, a.data_ptr(), 768, o.data_ptr(), 768, None, 0, None, 0, 0,
                                     None))
        outs.append(o)
    torch.cuda.synchronize()
    a, b = outs
    assert torch.isnan(a[1, 2, 7])
    other = torch.ones(3, 6, dtype=torch.bool)
    other[1, 2] = False
    assert torch.equal(a[other.cuda()], b[other.cuda()])


def test_norm_in_a_graph_and_on_a_side_stream(have_gpu):
    import torch

    x = torch.randn(50, 10 * 128, device="cuda").bfloat16()
    w, tt, pos = torch.ones(128, dtype=torch.bfloat16, device="cuda"), turns(1e4, 128), dev(np.zeros(50, np.uint32))
    norm = abi.ChkQkNorm(w.data_ptr(), w.data_ptr(), tt.data_ptr(), 128, 8, 2, 128, 0, 1e-6)
    q, k = x[:, :1024], x[:, 1024:]
    outs = [[torch.zeros(50, 1024, dtype=x.dtype, device="cuda"), torch.zeros(50, 256, dtype=x.dtype, device="cuda")] for _ in "ge"]

    def call(o, stream=None):
        check(lib().chk_qk_norm_rope(C.byref(norm), pos.data_ptr(), 50, q.data_ptr(), 1280, o[0].data_ptr(), 1024, k.data_ptr(),
                                     1280, o[1].data_ptr(), 256, KINDS["bf16"], stream))

    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        call(outs[0], torch.cuda.current_stream().cuda_stream)
    for i in range(5):
        x.copy_(torch.randn(50, 1280, device="cuda"))
        pos.copy_(torch.randint(0, 9999, (50,), device="cuda", dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        call(outs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs)), i


def test_host_memory_is_refused(have_gpu):
    import torch

    p = Pool(np.zeros((1, 1), np.uint32), [1], [0], 0, 16, 1, 1)
    host = torch.zeros(64, dtype=torch.int32)
    with pytest.raises(EngineError, match="not device memory"):
        check(lib().chk_kv_plan_q4(C.byref(p.c), None, None, host.data_ptr(), 1, p.start.ptr, None, None, None))
