"""The 4-bit key/value cache in plain numpy, 64 bits: what its planes hold for
given rows, what they stand for, and attention over it.  Test support."""

from __future__ import annotations

import numpy as np


def bf16_round(x: np.ndarray, up: bool) -> np.ndarray:
    """f32 values moved to bf16 towards +inf or -inf (as f32)."""
    x = np.asarray(x, np.float32)
    bits = x.view(np.uint32)
    cut = bits & np.uint32(0xFFFF0000)
    away = (bits >> np.uint32(31) == 0) == up  # towards larger magnitude
    moved = np.where((cut != bits) & away, cut + np.uint32(0x10000), cut).astype(np.uint32)
    return np.where(np.isnan(x), np.float32(np.nan), moved.view(np.float32))


def quantise(x: np.ndarray):
    """codes (uint8) [..., hd], s and b (f32 values of bf16) [..., hd / 64]."""
    with np.errstate(all="ignore"):
        g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 64)
        lo, hi = g.min(-1), g.max(-1)
        b = bf16_round(lo, False)
        s = bf16_round((hi - b) / np.float32(15.0), True)
        s = np.maximum(s, np.float32(2.0**-126))
        bad = ~(np.isfinite(g).all(-1) & np.isfinite(s) & np.isfinite(b))
        u = (g - b[..., None]).astype(np.float64)
        c = np.rint(u / s[..., None].astype(np.float64))
        c = np.where(np.isfinite(c), c, 0).clip(0, 15).astype(np.uint8)
        nan = np.float32(np.nan)
        return c.reshape(x.shape), np.where(bad, nan, s), np.where(bad, nan, b)


def stands_for(c: np.ndarray, s: np.ndarray, b: np.ndarray) -> np.ndarray:
    g = c.reshape(*c.shape[:-1], -1, 64).astype(np.float64)
    return (g * s[..., None].astype(np.float64) + b[..., None].astype(np.float64)).reshape(c.shape)


def order(hd: int, unit: int) -> np.ndarray:
    """order[i] = the dim whose code is nibble i of a stored row."""
    out = []
    ng = hd // 64
    for u in range(hd // unit):
        out += [64 * (u % ng) + unit * (u // ng) + j for j in range(unit)]
    return np.array(out)


UNIT = {"k": 16, "v": 4}


class Cache:
    """Host copy of the planes: codes [pages][nkv][page][hd / 2] bytes, pairs
    [pages][nkv][page][hd / 64] words."""

    def __init__(self, pages: int, page: int, nkv: int, hd: int, fill: int = 0xA5):
        self.pages, self.page, self.nkv, self.hd = pages, page, nkv, hd
        self.codes = {w: np.full((pages, nkv, page, hd // 2), fill, np.uint8) for w in "kv"}
        self.pairs = {w: np.full((pages, nkv, page, hd // 64), fill * 0x01010101, np.uint32) for w in "kv"}

    def copy(self) -> "Cache":
        c = Cache.__new__(Cache)
        c.pages, c.page, c.nkv, c.hd = self.pages, self.page, self.nkv, self.hd
        c.codes = {w: self.codes[w].copy() for w in "kv"}
        c.pairs = {w: self.pairs[w].copy() for w in "kv"}
        return c

    def place(self, table: np.ndarray, p: int):
        """(page id, offset) of position p, None where the table has none."""
        if p < 0 or p // self.page >= len(table) or table[p // self.page] >= self.pages:
            return None
        return int(table[p // self.page]), p % self.page

    def write(self, table: np.ndarray, p: int, which: str, row: np.ndarray) -> None:
        """One token's row [nkv][hd] (f32 values)."""
        at = self.place(table, p)
        if at is None:
            return
        c, s, b = quantise(row)
        c = c[:, order(self.hd, UNIT[which])]
        self.codes[which][at[0], :, at[1]] = c[:, 0::2] | (c[:, 1::2] << 4)
        pair = (s.astype(np.float32).view(np.uint32) >> 16) | (b.astype(np.float32).view(np.uint32) & np.uint32(0xFFFF0000))
        nan = np.isnan(s)
        self.pairs[which][at[0], :, at[1]] = np.where(nan, np.uint32(0x7FC07FC0), pair)

    def read(self, table: np.ndarray, p: int, which: str) -> np.ndarray:
        """[nkv][hd] in 64 bits, NaN where no page holds it."""
        at = self.place(table, p)
        if at is None:
            return np.full((self.nkv, self.hd), np.nan)
        byte = self.codes[which][at[0], :, at[1]]
        nib = np.stack([byte & 15, byte >> 4], -1).reshape(self.nkv, self.hd)
        c = np.empty_like(nib)
        c[:, order(self.hd, UNIT[which])] = nib
        pair = self.pairs[which][at[0], :, at[1]]
        s = (pair << np.uint32(16)).view(np.float32)
        b = (pair & np.uint32(0xFFFF0000)).view(np.float32)
        return stands_for(c, s, b)


def rows_of(start, b, rows):
    s0 = min(int(start[b]), rows)
    return s0, min(max(int(start[b + 1]), s0), rows)


def visible(p: int, t: np.ndarray, bits, ratio: int, kblk: int) -> np.ndarray:
    vis = t <= p
    if bits is not None:
        nblk, blk = (p + 1) // ratio, t // ratio
        if nblk > kblk:
            word = np.minimum(blk // 32, len(bits) - 1)
            on = (blk // 32 < len(bits)) & ((bits[word] >> (blk % 32).astype(np.uint32)) & 1 == 1)
            vis &= (blk >= nblk) | on
    return vis


def attend(cache: Cache, table, lens, start, q: np.ndarray, nh: int, gated: bool, mask=None, out=None):
    """out [rows][nh][hd] in 64 bits (rows of no sequence as in `out`), and for
    each row and head what its tolerance scales with: the largest magnitude of
    a value's parts among the visible tokens, and that of a score's parts."""
    rows, hd, g = q.shape[0], cache.hd, nh // cache.nkv
    out = np.zeros((rows, nh, hd)) if out is None else out.astype(np.float64)
    vmax, smax = np.zeros((rows, nh)), np.zeros((rows, nh))
    for b in range(len(lens)):
        s0, s1 = rows_of(start, b, rows)
        n = int(lens[b])
        if s1 == s0:
            continue
        if n > len(table[b]) * cache.page:
            out[s0:s1] = np.nan
            continue
        k = np.stack([cache.read(table[b], t, "k") for t in range(n)]) if n else np.zeros((0, cache.nkv, hd))
        v = np.stack([cache.read(table[b], t, "v") for t in range(n)]) if n else np.zeros((0, cache.nkv, hd))
        t = np.arange(n)
        for r in range(s0, s1):
            p = n - (s1 - r)
            vis = visible(p, t, None if mask is None else mask[0][r], *(mask[1:] if mask else (1, 0))) if p >= 0 else t < 0
            for h in range(nh):
                if not vis.any():
                    out[r, h] = 0.0
                    continue
                kk, vv = k[vis, h // g], v[vis, h // g]
                qq = q[r, h, :hd].astype(np.float64)
                s = kk @ qq * hd**-0.5
                w = np.exp(s - s.max())
                o = (w @ vv) / w.sum()
                if gated:
                    o = o / (1 + np.exp(-q[r, h, hd:].astype(np.float64)))
                out[r, h] = o
                vmax[r, h] = np.abs(vv).max()
                smax[r, h] = (np.abs(kk) @ np.abs(qq)).max() * hd**-0.5
    return out, vmax, smax


def tolerance(kind: str, hd: int, want: np.ndarray, vmax: np.ndarray, smax: np.ndarray) -> np.ndarray:
    """How far a kernel's out may be from `want`, per element.

    The stored parts s c and b of a group are at most three times its largest
    magnitude m (b >= -m, s c <= hi - lo + a step <= 2.2 m), so sums over them
    carry at most 3.2 times what sums over the values would; call that K.
      scores   f32 sums of hd products: a rounding of 2^-24 of the running sum
               for each, taken as independent: 2 sqrt(hd) 2^-24 K smax.  16-bit
               types are granted 1039 / 15 times more, what codes that stay on
               the 1024 of their f16 form would carry.  q in two f16 parts (f32
               only): 2^-22 K smax.
      softmax  twice the score's error (numerator and denominator), and 2^-22
               for the exponential.
      values   numerators in two f16 parts 2^-22, or one for bf16: 2^-11, each
               of K vmax; f32 sums 2^-20 of it.
      out      half a step of the type, of want (and the gate's 2^-21).
    """
    big = 3.2
    amp = 1.0 if kind == "f32" else 1039 / 15
    score = big * smax * (2 * hd**0.5 * 2.0**-24 * amp + 2.0**-22)
    parts = {"f32": 2.0**-22, "f16": 2.0**-22, "bf16": 2.0**-11}[kind] + 2.0**-20
    half = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}[kind]
    tol = vmax * (2 * score + 2.0**-22 + big * parts)
    tiny = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-134}[kind]
    return tol[..., None] + (half + 2.0**-21) * np.abs(want) + tiny


HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # half a step, relative


def rounded_to(x: np.ndarray, kind: str) -> np.ndarray:
    """64 bits rounded once to `kind`, ties to even."""
    if kind != "bf16":
        with np.errstate(over="ignore"):
            return x.astype({"f32": np.float32, "f16": np.float16}[kind]).astype(np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 256) / 256, e)


def beyond_rounding(kind: str, got: np.ndarray, want: np.ndarray) -> float:
    """How far `got` is from `want` rounded once, as a root mean square relative
    to want's: what is left of an error once the type's own rounding is off."""
    return float(np.sqrt(((got - rounded_to(want, kind)) ** 2).mean() / (want**2).mean()))


def beyond_limit(kind: str, smax: np.ndarray, parts: int = 2) -> float:
    """What `beyond_rounding` may be where values are independent and of mean 0,
    numerators in f16 parts.

    Then a relative error e of the numerators, independent from token to token,
    is one of e of the outputs' root mean square.  e: a score is some ten f32
    roundings, 2^-24 each of a sum of its parts, which stays below half of
    3.2 smax (see `tolerance`) where it wanders; sqrt(10) 1.6 < 8, so 2^-21 smax;
    the exponential and two parts 2^-21; one part 2^-11 / sqrt(3).
    An output of 16 bits shows e as steps of 2 HALF at most, relative, taken
    with a chance of e over that step: a mean square of 2 HALF e.  Twice that
    square for the chance in their number.
    """
    e = 2.0**-21 * (1 + float(np.sqrt((smax**2).mean()))) + (2.0**-11 / 3**0.5 if parts == 1 else 0.0)
    return (2 * (2 * HALF[kind] * e + e * e)) ** 0.5
