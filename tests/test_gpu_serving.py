"""A serving batch over the 4-bit cache, step after step as one program's buffers: plan, norm and
rotation, append and attention, each array against the same rules on the host.  Who holds which page:
a prompt forked into continuations that outlive it, and windows whose pages go back while they run."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from cherenkov_amd.abi import check, lib
from tests import kv4_ref as ref
from tests import step_ref
from tests import view_ref as view
from tests.test_gpu_kv4 import KINDS, dev, rounded, torch_type
from tests.test_gpu_pool import NONE, once, release
from tests.test_gpu_views import Views, close

pytestmark = pytest.mark.gpu


class Server:
    NAMES = ("table", "len", "free", "nfree")

    def __init__(self, seed, kind, n, pages, width, most, heads=(8, 2, 128), page=16):
        import torch

        self.rng, self.kind, self.n, self.page, self.pages, self.most, self.heads = (
            np.random.default_rng(seed), kind, n, page, pages, most, heads)
        nh, nkv, hd = heads
        turn = np.zeros(32, np.uint64)
        check(lib().chk_rope_turns(1e4, 64, turn.ctypes.data))
        self.turns = torch.from_numpy(turn.view(np.int64)).cuda()
        w = (1 + 0.2 * self.rng.normal(0, 1, (2, hd))).astype(np.float32)
        self.weights = torch.from_numpy(w).bfloat16().cuda()
        self.norms = self.weights.double().cpu().numpy()
        self.norm = abi.ChkQkNorm(self.weights[0].data_ptr(), self.weights[1].data_ptr(), self.turns.data_ptr(), 64, nh, nkv, hd,
                                  0, 1e-6)
        self.state = dict(table=np.full((n, width), NONE, np.uint32), len=np.zeros(n, np.uint32),
                          free=np.arange(pages, dtype=np.uint32), nfree=np.array([pages, 0], np.uint32))
        self.on = {k: dev(v) for k, v in self.state.items()}
        self.pool = abi.ChkKvPool(*(self.on[k].data_ptr() for k in self.NAMES), n, width, page, pages)
        self.host = ref.Cache(pages, page, nkv, hd)
        self.d = Views(self.host, self.state["table"], self.state["len"], np.zeros(n + 1), most)
        self.d.seqs = abi.ChkKvSeqs(self.on["table"].data_ptr(), self.on["len"].data_ptr(), self.d.start.data_ptr(), n, width, most)
        self.d.share([0, n], [0])
        self.own = np.zeros(n, np.uint32)
        dt = torch_type(kind)
        self.pos = torch.zeros(most, dtype=torch.int32, device="cuda")
        self.q, self.out = (torch.zeros(most, nh * hd, dtype=dt, device="cuda") for _ in range(2))
        self.k = torch.zeros(most, nkv * hd, dtype=dt, device="cuda")
        self.ws = self.d.prefix_workspace(nh, 1)

    def push(self):
        """The host's copy of the state onto the device, as a program changes it between two steps."""
        for k in self.NAMES:
            self.on[k].copy_(dev(self.state[k]))

    def step(self, keep, want, window=None):
        """One step; the rows of each sequence."""
        import torch

        nh, nkv, hd = self.heads
        keep = self.state["len"] if keep is None else keep
        kp, ow, wa = (dev(np.asarray(x, np.uint32)) for x in (keep, self.own, want))
        check(lib().chk_kv_plan_q4(C.byref(self.pool), kp.data_ptr(), ow.data_ptr(), wa.data_ptr(), self.most,
                                   self.d.start.data_ptr(), self.pos.data_ptr(), None, None))
        x, t = rounded(self.rng.normal(0, 1, (self.most, (nh + 2 * nkv) * hd)), self.kind)
        check(lib().chk_qk_norm_rope(C.byref(self.norm), self.pos.data_ptr(), self.most, t.data_ptr(), t.stride(0),
                                     self.q.data_ptr(), self.q.stride(0), t[:, nh * hd:].data_ptr(), t.stride(0),
                                     self.k.data_ptr(), self.k.stride(0), KINDS[self.kind], None))
        self.d.append(self.k, t[:, (nh + nkv) * hd:], self.kind)
        if window:
            self.d.window(self.q, self.out, nh, False, self.kind, *window, ws=self.ws)
        else:
            self.d.prefix(self.q, self.out, nh, False, self.kind, ws=self.ws)
        torch.cuda.synchronize()
        s = self.state
        plan = step_ref.plan(s["table"], s["len"], s["free"], s["nfree"][0], keep, self.own, want, self.most, self.page, self.pages)
        self.state = dict(zip(self.NAMES, plan[:4]))
        start, pos = plan[4], plan[5]
        for name, a, w in [(k, self.on[k], self.state[k]) for k in self.NAMES] + [("start", self.d.start, start), ("pos", self.pos, pos)]:
            np.testing.assert_array_equal(a.cpu().numpy().view(np.uint32), w, err_msg=name)
        live = int(start[-1])
        gq, gk = (a[:live].double().cpu().numpy().reshape(live, h, hd) for a, h in ((self.q, nh), (self.k, nkv)))
        for got, at, heads, w in ((gq, 0, nh, self.norms[0]), (gk, nh * hd, nkv, self.norms[1])):
            want_x, size = step_ref.norm_rope(x[:live, at:at + heads * hd].reshape(live, heads, hd), w, 1e-6, pos[:live], 1e4, 64)
            assert np.all(np.abs(got - want_x) <= step_ref.norm_rope_tolerance(self.kind, want_x, size))
        for b in range(self.n):
            for r in range(int(start[b]), int(start[b + 1])):
                self.host.write(self.state["table"][b], int(pos[r]), "k", gk[r].astype(np.float32))
                self.host.write(self.state["table"][b], int(pos[r]), "v", x[r, (nh + nkv) * hd:].reshape(nkv, hd))
        back = self.d.back()
        for w in "kv":  # the whole cache: nothing of another sequence's is written over
            np.testing.assert_array_equal(back.codes[w], self.host.codes[w])
            np.testing.assert_array_equal(back.pairs[w], self.host.pairs[w])
        want_o, vmax, smax = view.attend(self.host, self.state["table"], self.state["len"], start, gq, nh, False,
                                         *(window or (None, 0)), out=np.zeros((live, nh, hd)))
        assert np.isfinite(want_o).all()
        close(self.out[:live].double().cpu().numpy().reshape(live, nh, hd), want_o, vmax, smax, self.kind, hd)
        return np.diff(start.astype(np.int64))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_prompts_owner_ends_before_its_readers(have_gpu, kind):
    """A prompt's seven whole pages, read by four continuations: own counts them for every one of the
    five.  The prompt ends first and another request takes its place; the last reader ends with an own of
    0, and they go back with it."""
    s = Server(5, kind, 5, 60, 20, 140)
    s.step([0] * 5, [120, 0, 0, 0, 0])
    table = s.state["table"]
    prompt = [int(x) for x in table[0, :7]]
    table[1:, :7] = table[0, :7]
    s.state["len"][1:] = 112
    s.own[:] = 7
    s.push()
    s.d.tokens.fill_(112)
    assert s.step([120, 112, 112, 112, 112], [1, 30, 2, 5, 1]).tolist() == [1, 30, 2, 5, 1]
    state = lambda: (s.state["table"], s.state["len"], s.page, s.state["free"], int(s.state["nfree"][0]), s.pages)  # noqa: E731
    once(*state(), shared=prompt)
    # the prompt's sequence ends; its seven pages stay
    s.step([0, NONE, NONE, NONE, NONE], [0, 1, 1, 1, 1])
    once(*state(), shared=prompt)
    assert not np.isin(prompt, s.state["free"][:s.state["nfree"][0]]).any()
    # another request in that place, on pages that are free: none of the prompt's is among them
    s.own[0] = 0
    s.d.first.copy_(dev(np.array([1, 5], np.uint32)))
    s.step([0, NONE, NONE, NONE, NONE], [130, 1, 1, 1, 1])
    assert not np.isin(prompt, s.state["table"][0]).any()
    s.step(None, [2, 1, 3, 1, 1])
    # rejected drafts, never below the shared pages; one cut into them has no row and harms no one
    keep = np.maximum(s.state["len"].astype(int) - 2, 112)
    keep[3] = 100
    assert s.step(keep, [1, 1, 1, 4, 1]).tolist() == [1, 1, 1, 0, 1]
    # readers end one after the other, the last with all that is left
    for last in (3, 1, 4):
        keep = s.state["len"].copy()
        keep[last] = 0
        s.step(keep, np.where(keep > 0, 1, 0))
        once(*state(), shared=prompt)
    s.own[2] = 0
    keep = s.state["len"].copy()
    keep[2] = 0
    s.step(keep, [1, 0, 0, 0, 0])
    once(*state())
    s.step([0] * 5, [0] * 5)
    assert s.state["nfree"].tolist() == [60, 0]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(40, 20), (16, 0)])
def test_a_windowed_batch_gives_pages_back(have_gpu, kind, window, sinks):
    """Requests through a window with first tokens that stay: what it has left goes back while they
    run and is others' pages a step later; their first pages come back with their end."""
    s = Server(6, kind, 4, 34, 30, 120)
    wants = [[90, 5, 0, 33], [1, 40, 20, 3], [20, 1, 60, 1], [1, 3, 1, 2], [30, 30, 1, 1], [2, 1, 30, 30], [1, 1, 1, 1]]
    freed = 0
    for i, want in enumerate(wants):
        keep = np.maximum(s.state["len"].astype(int) - [0, 2, 1, 3], 0)
        if i == 4:
            keep[0] = 0  # ends, and another begins in its place
        got = s.step(keep, want, window=(window, sinks))
        assert got.sum() > 0
        t, free, nf = s.state["table"], s.state["free"], int(s.state["nfree"][0])
        once(t, s.state["len"], s.page, free, nf, s.pages)
        for b in range(4):  # (three tokens further back may be cut off again)
            was = nf
            nf = release(t, np.maximum(s.state["len"].astype(int) - 3, 0), free, nf, b, s.page, window, sinks)
            freed += nf - was
        s.state["nfree"] = np.array([nf, 0], np.uint32)
        s.push()
        once(t, s.state["len"], s.page, free, nf, s.pages)
    assert freed >= 4
    s.step([0] * 4, [0] * 4, window=(window, sinks))
    assert s.state["nfree"].tolist() == [34, 0] and np.all(s.state["table"] == NONE)
