"""A serving step's plan and the norm and rotation of its heads in plain Python
and numpy, 64 bits.  Test support."""

from __future__ import annotations

import numpy as np

NONE = 0xFFFFFFFF


def plan(table, length, free, nfree, keep, own, want, rows, page, pages):
    """The rules of chk_kv_plan_q4 one sequence and one page at a time, on copies:
    (table, len, free, [free pages, lacked], start, pos, slot)."""
    table, length, free = table.copy(), [int(x) for x in length], free.copy()
    n, width = table.shape
    top = min(int(nfree), pages)
    full = lambda t: min(-(-t // page), width)  # noqa: E731
    left = []
    for b in reversed(range(n)):
        cut = length[b] if keep is None else min(int(keep[b]), length[b])
        first = max(full(cut), 0 if own is None else int(own[b]))
        for e in reversed(range(first, full(length[b]))):
            if table[b, e] < pages:  # (a window's page that is gone already gives none back)
                if top < pages:
                    free[top] = table[b, e]
                top += 1
            table[b, e] = NONE
        left.insert(0, cut)
    top = min(top, pages)
    avail, asked, needs = top, 0, 0
    start, pos, slot, out = [0], [], [], []
    for b in range(n):
        w = int(want[b])
        if own is not None and left[b] % page and left[b] // page < int(own[b]) <= width:
            w = 0
        if left[b] + w > width * page:
            w = 0
        asked += w
        if asked > rows:
            w = 0
        need = full(left[b] + w) - full(left[b])
        needs += need
        if need and needs > avail:
            w = need = 0
        for i in range(need):
            top -= 1
            table[b, full(left[b]) + i] = free[top]
        for p in range(left[b], left[b] + w):
            pos.append(p)
            at = int(table[b, p // page])
            slot.append(at * page + p % page if at < pages else 2**64 - 1)
        out.append(left[b] + w)
        start.append(start[-1] + w)
    pos += [NONE] * (rows - len(pos))
    slot += [2**64 - 1] * (rows - len(slot))
    return (table, np.array(out, np.uint32), free, np.array([top, max(0, needs - avail)], np.uint32),
            np.array(start, np.uint32), np.array(pos, np.uint32), np.array(slot, np.uint64))


def norm_rope(x, w, eps, pos, theta, rot):
    """[rows][heads][hd] in 64 bits, and what a result's error scales with: |a| + |b|
    of its pair (|y| where it is not turned)."""
    x = np.asarray(x, np.float64)
    y = x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    if rot == 0:
        return y, np.abs(y)
    half = rot // 2
    # (80-bit floats: a position of 2^32 takes 32 of a 64-bit float's 53)
    wide = np.longdouble
    angle = np.asarray(pos, wide)[:, None] * wide(theta) ** (wide(-2) * np.arange(half) / wide(rot))
    angle = np.fmod(angle, 8 * np.arctan(wide(1)))
    c, s = (f(angle).astype(np.float64)[:, None] for f in (np.cos, np.sin))
    a, b = y[..., :half], y[..., half:rot]
    size = np.abs(a) + np.abs(b)
    return (np.concatenate([a * c - b * s, b * c + a * s, y[..., rot:]], -1),
            np.concatenate([size, size, np.abs(y[..., rot:])], -1))


def norm_rope_tolerance(kind, want, size):
    """How far a result may be from `want`, per element, in units of u = 2^-24.

      norm      the squares' sum: at most 16 roundings on terms of one sign, 16 u
                of it and 8 u of its root; the reciprocal root 2 u; the product
                with it 1 u: 11 u of |y|
      angle     what is left of an eighth of a turn, at most pi / 4, and its factor
                and product rounded, 3 u each of it: 2.4 u; cut at 2^-32 of a turn
                and Taylor's remainder 0.1 u; the sums' own roundings 2 u: 5 u
                absolute in sine and cosine
      turned    the products with the weight and the dim and their sum: 3 u
    so 19 u (|a| + |b|); and half a step of the type, of want.
    """
    u = 2.0**-24
    half = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}[kind]
    tiny = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-134}[kind]
    return 19 * u * size * (1 + half) + half * np.abs(want) + tiny
