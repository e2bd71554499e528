"""Attention over the 4-bit cache where rows see a window of their sequence, in
plain numpy and 64 bits.  Test support."""

from __future__ import annotations

import numpy as np

from tests import kv4_ref as ref


def values(cache: ref.Cache, table_row: np.ndarray, n: int, which: str) -> np.ndarray:
    """[n][nkv][hd]: what tokens 0 .. n of a sequence stand for, NaN where no page holds them."""
    if n == 0:
        return np.zeros((0, cache.nkv, cache.hd))
    t = np.arange(n)
    e = t // cache.page
    ids = np.asarray(table_row, np.int64)[np.minimum(e, len(table_row) - 1)]
    lost = (e >= len(table_row)) | (ids >= cache.pages)
    ids = np.where(lost, 0, ids)
    byte = cache.codes[which][ids, :, t % cache.page]
    nib = np.stack([byte & 15, byte >> 4], -1).reshape(n, cache.nkv, cache.hd)
    c = np.empty_like(nib)
    c[..., ref.order(cache.hd, ref.UNIT[which])] = nib
    pair = cache.pairs[which][ids, :, t % cache.page]
    s, b = (pair << np.uint32(16)).view(np.float32), (pair & np.uint32(0xFFFF0000)).view(np.float32)
    with np.errstate(invalid="ignore"):
        x = ref.stands_for(c, s, b)
    x[lost] = np.nan
    return x


def attend(cache, table, lens, start, q, nh, gated, window=None, sinks=0, out=None):
    """As kv4_ref.attend, rows at p seeing t <= p with t < sinks or t > p - window
    (None: all)."""
    rows, hd, g = q.shape[0], cache.hd, nh // cache.nkv
    out = np.zeros((rows, nh, hd)) if out is None else out.astype(np.float64)
    vmax, smax = np.zeros((rows, nh)), np.zeros((rows, nh))
    for b in range(len(lens)):
        s0, s1 = ref.rows_of(start, b, rows)
        n = int(lens[b])
        if s1 == s0:
            continue
        if n > len(table[b]) * cache.page:
            out[s0:s1] = np.nan
            continue
        k, v = values(cache, table[b], n, "k"), values(cache, table[b], n, "v")
        t = np.arange(n)[None]
        p = n - (s1 - np.arange(s0, s1))[:, None]
        see = t <= p
        if window is not None:
            see &= (t < sinks) | (t > p - window)
        some = see.any(1)
        for h in range(nh):
            # (what no row sees may be anything)
            kk, vv = (np.where(see.any(0)[:, None], x[:, h // g], 0.0) for x in (k, v))
            qq = q[s0:s1, h, :hd].astype(np.float64)
            with np.errstate(invalid="ignore"):
                s = np.where(see, qq @ kk.T * hd**-0.5, -np.inf)
                top = np.where(some, s.max(1, initial=-np.inf), 0.0)[:, None]
                w = np.exp(s - top)
                l = w.sum(1, keepdims=True)
                o = np.where(some[:, None], np.where(see, w, 0.0) @ np.nan_to_num(vv) / np.where(l == 0, 1, l), 0.0)
                lost = (see & np.isnan(kk).any(1) | see & np.isnan(vv).any(1)).any(1)
                o[lost] = np.nan
                if gated:
                    o = o / (1 + np.exp(-q[s0:s1, h, hd:].astype(np.float64)))
                out[s0:s1, h] = o
                vmax[s0:s1, h] = np.where(see, np.abs(np.nan_to_num(vv)).max(1)[None], 0).max(1, initial=0)
                smax[s0:s1, h] = np.where(see, np.abs(qq) @ np.abs(np.nan_to_num(kk)).T, 0).max(1, initial=0) * hd**-0.5
    return out, vmax, smax
