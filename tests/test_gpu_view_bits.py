"""How many bits the softmax's numerators keep where rows see a part of their
sequence or share a prefix (chk_attn_window_q4, chk_attn_prefix_q4): two tokens of
opposite values and nearly equal scores, whose difference is all that is left, in
blocks of few and of many (row, head) pairs, against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from tests import kv4_ref as ref
from tests import view_ref as view
from tests.test_gpu_kv4 import rounded, torch_type
from tests.test_gpu_views import Views

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def opposites(tokens: int, page: int, hd: int, seen) -> tuple[ref.Cache, np.ndarray]:
    """One sequence's pages.  Keys are 0 but for dim 0, -1 at odd tokens, and dim 64, -8 at
    tokens that `seen` does not name; values are 1 at even tokens and -1 at odd ones."""
    pages = -(-tokens // page)
    c = ref.Cache(pages, page, 1, hd, fill=0)
    table = np.arange(pages, dtype=np.uint32)[None]
    code = {w: np.full((pages * page, hd), 8, np.uint8) for w in "kv"}
    t = np.arange(tokens)
    code["k"][t[t % 2 == 1], 0] = 7
    code["k"][t[~np.isin(t, seen)], 64] = 0
    code["v"][t[t % 2 == 1]] = 7
    bf16 = lambda x: np.float32(x).view(np.uint32) >> np.uint32(16)  # noqa: E731
    for w, s, b in (("k", 1, -8), ("v", 2, -15)):
        x = code[w][:, ref.order(hd, ref.UNIT[w])]
        c.codes[w][:] = (x[:, 0::2] | (x[:, 1::2] << 4)).reshape(c.codes[w].shape)
        c.pairs[w][:] = bf16(s) | (bf16(b) << np.uint32(16))
    return c, table


# (seqs, rows each, query heads): few pairs, and more than any block of few takes
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("which,seqs,rows,nh", [("window", 1, 3, 4), ("window", 1, 90, 2), ("prefix", 3, 1, 4), ("prefix", 12, 1, 8),
                                                ("prefix", 9, 3, 8)])
def test_differences_of_numerators(have_gpu, kind, hd, which, seqs, rows, nh):
    """Each row sees one even and one odd token whose scores are d apart, 2^-9 < d < 2^-6: its output is
    (1 - e^-d) / (1 + e^-d), a difference of numerators near 1.  How far that may be off, u = 2^-24:

      scores      d itself to a few u of it; counted with the value step's log2, below 16 in
                  magnitude, and rounded there: 2^-21 of a numerator
      exponential 2 u of it
      numerators  in two f16 parts, 2^-23 and less; in one they would be off by up to 2^-12
      products    at most eight sums that are not exact, none above three numerators: 24 u
      sum, quotient  4 u

    all of it below 2^-18 beside outputs of 2^-10 to 2^-7, and half a step of the type.
    """
    import torch

    rng = np.random.default_rng(rows * hd + nh)
    shared, page = 128, 64
    seen = np.arange(2) if which == "prefix" else np.arange(400)
    n = shared + rows if which == "prefix" else 300
    c, row = opposites(n, page, hd, seen)
    table = np.repeat(row, seqs, 0)
    lens, start = [n] * seqs, rows * np.arange(seqs + 1)
    total = int(start[-1])
    x = np.zeros((total, nh, hd), np.float32)
    x[..., 0] = hd**0.5 * 2.0 ** rng.uniform(-8.9, -6.1, (total, nh))
    x[..., 64] = 40 * hd**0.5  # what is not seen scores 320 less
    x, q = rounded(x.reshape(total, -1), kind)
    d = Views(c, table, lens, start, total)
    out = torch.zeros(total, nh * hd, dtype=torch_type(kind), device="cuda")
    if which == "window":
        d.window(q, out, nh, False, kind, 2, 0)
    else:
        d.share([0, seqs], [shared])
        d.prefix(q, out, nh, False, kind)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy().reshape(total, nh, hd)
    want, _, _ = view.attend(c, table, lens, start, x.reshape(total, nh, hd), nh, False, *((2, 0) if which == "window" else (None, 0)))
    assert np.all((2.0**-10.1 < np.abs(want)) & (np.abs(want) < 2.0**-7))
    off = np.abs(got - want) - (2.0**-18 + HALF[kind] * np.abs(want))
    assert np.all(off <= 0), f"{(off > 0).mean():.3f} of the outputs off by up to {np.abs(got - want).max():.3g}"
