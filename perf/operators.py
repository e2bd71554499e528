"""The cache of keys and values in 4 bits, as timed cases: rows quantised into
it and read back, and attention over it, from single tokens of many sequences
to prompts.

A cache is pages of `page` tokens per kv head.  64 consecutive dims of one
token and head are a group: 4-bit codes c, a bf16 step s and a bf16 least
value b, and the group stands for s c + b.  A row of hd dims is hd / 2 bytes,
two codes a byte, the lower nibble first, its dims in units of 16 (keys) or 4
(values) that take the groups in turn (`_order`).

Where `own` is false every pass runs in elementary torch operations over the
batch padded to its longest sequence; where it is true it goes through
chk_kv_append_q4, chk_kv_read_q4 and chk_attn_q4.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
# bytes of a stored value: half a byte of code, 4 bytes of (s, b) per 64
STORED = 0.5 + 4 / 64

# ------------------------------------------------------------------ cases
#
# seqs     sequences of the call
# rows     rows of the longest sequence in this call (its last positions)
# ctx      tokens the longest sequence holds before them
# ragged   sequences of all lengths up to those, one of them without rows
# nh, nkv, hd, gated   heads; gated: q rows hold [q | gate] per head
# page     tokens a page
# budget   tokens of chosen blocks a row keeps of its context (0: all)

MODEL = dict(nh=16, nkv=2, hd=256, gated=True, type="f32")


def listed() -> list[dict]:
    return [
        # a decode step of one request: its token's keys and values written,
        # then attended over, 2184 tokens in (the benchmark's mid-decode context)
        dict(name="step_1", kind="step", seqs=1, rows=1, ctx=2183, ragged=False, page=64, budget=0, **MODEL),
        # the same far into a long conversation
        dict(name="step_1_32k", kind="step", seqs=1, rows=1, ctx=31999, ragged=False, page=64, budget=0, **MODEL),
        # a serving batch: 64 requests of all lengths, a token each, short pages
        dict(name="step_64_ragged", kind="step", seqs=64, rows=1, ctx=8191, ragged=True, page=16, budget=0, nh=32, nkv=8,
             hd=128, gated=False, type="bf16"),
        # a few very long requests, twelve query heads a kv head
        dict(name="step_8_long", kind="step", seqs=8, rows=1, ctx=131071, ragged=False, page=256, budget=0, nh=24, nkv=2,
             hd=256, gated=False, type="f16"),
        # a verify step: three rows behind 700 tokens
        dict(name="verify_3", kind="step", seqs=1, rows=3, ctx=700, ragged=False, page=64, budget=0, **MODEL),
        # the next turn of a conversation, an odd number of rows
        dict(name="turn_333", kind="attend", seqs=1, rows=333, ctx=1500, ragged=False, page=64, budget=0, **MODEL),
        # a prompt from an empty context
        dict(name="prompt_2048", kind="attend", seqs=1, rows=2048, ctx=0, ragged=False, page=64, budget=0, **MODEL),
        # several prompts at once, the largest call
        dict(name="prompt_4_ragged", kind="attend", seqs=4, rows=4096, ctx=0, ragged=True, page=128, budget=0, nh=32,
             nkv=8, hd=128, gated=False, type="bf16"),
        # rows of a document past the indexer's budget, the chosen blocks alone
        dict(name="document_chosen", kind="attend", seqs=1, rows=250, ctx=11000, ragged=False, page=64, budget=2048,
             nh=8, nkv=2, hd=256, gated=True, type="f32"),
        # one token's keys and values written and read back: the smallest call
        dict(name="write_1", kind="write", seqs=1, rows=1, ctx=999, ragged=False, page=64, nkv=2, hd=256, type="f32"),
        # prompts' keys and values written, and read back as the next layer's check does
        dict(name="write_16k_ragged", kind="write", seqs=6, rows=4099, ctx=700, ragged=True, page=16, nkv=8, hd=128,
             type="bf16"),
        # a whole long context read back (a cache handed to a 16-bit consumer)
        dict(name="read_32k", kind="read", seqs=2, rows=32000, ctx=0, ragged=False, page=64, nkv=2, hd=256, type="f16"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["step", "step", "step", "attend", "attend", "attend", "write", "read"])
    nkv, hd = rng.choice([1, 2, 4, 8]), rng.choice([128, 256])
    c = dict(kind=kind, ragged=rng.random() < 0.6, page=rng.choice([16, 32, 64, 128, 256, 1024]), nkv=nkv, hd=hd,
             type=rng.choice(["f32", "f16", "bf16"]))
    if kind in ("write", "read"):
        # tokens of the whole call: up to write_16k_ragged's, and read_32k's
        c["seqs"] = _log(rng, 1, 64)
        most = (24000 if kind == "write" else 60000) * 1024 // (c["seqs"] * 2 * nkv * hd)
        c["rows"] = _log(rng, 1, max(2, most))
        c["ctx"] = rng.choice([0, _log(rng, 1, 4096)])
        return c
    g = rng.choice([1, 2, 4, 8, 12])
    c.update(nh=nkv * g, gated=rng.random() < 0.5, budget=0)
    if kind == "step":
        c["seqs"], c["rows"] = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 3, 4])
        c["ctx"] = _log(rng, 1, min(131071, 8 * 131072 * 512 // (c["seqs"] * nkv * hd)))
    else:
        c["seqs"], c["rows"] = rng.choice([1, 1, 2, 3, 5]), _log(rng, 5, 4096)
        c["ctx"] = rng.choice([0, _log(rng, 1, 30000)])
        # no dearer than prompt_4_ragged: rows (ctx + rows / 2) pairs a sequence
        pairs = 6.5e10 / (c["seqs"] * nkv * g * hd)
        c["rows"] = max(1, min(c["rows"], int(math.sqrt(c["ctx"] ** 2 + 2 * pairs) - c["ctx"])))
        if rng.random() < 0.3:
            c["budget"] = rng.choice([256, 1024, 2048])
    return c


RATIO = 4  # tokens a block of the indexer


def _shares(case: dict) -> list[float]:
    if not case["ragged"]:
        return [1.0] * case["seqs"]
    return [1.0] + [(0.37 + 0.6180339887 * b) % 1.0 for b in range(1, case["seqs"])]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Tokens of each sequence, this call's rows included, and those rows."""
    share = _shares(case)
    ctx = [int(case["ctx"] * f) for f in share]
    step = case["kind"] == "step"
    rows = [case["rows"] if step else max(1, int(case["rows"] * f)) for f in share]
    if case["ragged"] and case["seqs"] > 2:
        rows[case["seqs"] // 2] = 0
    return [c + n for c, n in zip(ctx, rows)], rows


# ------------------------------------------------------------------ inputs


def _order(hd: int, unit: int) -> torch.Tensor:
    """The dim that each code of a stored row belongs to: units of `unit` dims,
    unit u the (u / groups)-th of group u % groups."""
    i, groups = torch.arange(hd), hd // 64
    u = i // unit
    return 64 * (u % groups) + unit * (u // groups) + i % unit


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 31)


def _plane(g: torch.Generator, case: dict, pages: int) -> tuple[torch.Tensor, torch.Tensor]:
    """A plane as quantised rows of a norm leave it: bytes and (s, b) pairs.
    A few channels are far larger than the others, as in trained keys."""
    nkv, page, hd = case["nkv"], case["page"], case["hd"]
    shape = (pages, nkv, page)
    c = torch.randn(*shape, hd, generator=g, device=DEV).mul_(2.9).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
    codes = c[..., 0::2] | (c[..., 1::2] << 4)
    s = 0.3 * torch.exp(0.25 * torch.randn(*shape, hd // 64, generator=g, device=DEV))
    loud = 1 + 2 * (torch.rand(nkv, 1, hd // 64, generator=g, device=DEV) < 0.25)
    s = (s * loud).bfloat16()
    b = (-7.5 * s.float() + 0.2 * torch.randn(*shape, hd // 64, generator=g, device=DEV)).bfloat16()
    return codes.contiguous(), torch.stack([s, b], -1).contiguous()


def _inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    lens, rows = _lengths(case)
    page, nkv, hd, kind = case["page"], case["nkv"], case["hd"], case["kind"]
    dt = TYPES[case["type"]]
    width = max(1, -(-max(lens) // page))
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    # every sequence's pages lie anywhere in the pool
    place = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    first = np.concatenate([[0], np.cumsum(need)[:-1]])
    at = torch.tensor(first, device=DEV)[:, None] + torch.arange(width, device=DEV)[None]
    live = torch.arange(width, device=DEV)[None] < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(live, place[at.clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device=DEV))
    k, ks = _plane(g, case, pages)
    v, vs = _plane(g, case, pages)
    start = np.concatenate([[0], np.cumsum(rows)])
    T = int(start[-1])
    st = dict(k=k, v=v, ks=ks, vs=vs, table=table.contiguous(), lens_host=lens, rows_host=rows, T=T,
              lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
              start=torch.tensor(start, dtype=torch.int32, device=DEV))
    if kind in ("step", "write"):
        # keys and values as halves of one projection's rows
        kv = torch.randn(max(T, 1), 2, nkv, hd, generator=g, device=DEV)
        kv[:, 0, :, ::29] *= 6
        st["kv"] = kv.to(dt)
    if kind in ("step", "attend"):
        st["q"] = torch.randn(max(T, 1), case["nh"], hd * (2 if case["gated"] else 1), generator=g, device=DEV).to(dt)
        if case["budget"]:
            nblk_max = max(lens) // RATIO
            keep = case["budget"] // RATIO
            pos = _positions(st)
            score = torch.rand(T, max(nblk_max, 1), generator=g, device=DEV)
            score = torch.where(torch.arange(max(nblk_max, 1), device=DEV)[None] < ((pos + 1) // RATIO)[:, None], score, -1.0)
            chosen = torch.zeros(T, (nblk_max + 32) // 32 * 32, dtype=torch.int64, device=DEV)
            top = score.topk(min(keep, score.shape[1]), dim=1).indices
            chosen.scatter_(1, top, 1)
            words = (chosen.view(T, -1, 32) << torch.arange(32, device=DEV)).sum(-1)
            st["mask"] = torch.where(words >= 2**31, words - 2**32, words).to(torch.int32).contiguous()
    return st


def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    st["case"] = case
    dt, nkv, hd = TYPES[case["type"]], case["nkv"], case["hd"]
    if case["kind"] in ("write", "read"):
        st["out"] = torch.zeros(2, max(st["T"], 1), nkv, hd, dtype=dt, device=DEV)
    else:
        st["out"] = torch.zeros(max(st["T"], 1), case["nh"], hd, dtype=dt, device=DEV)
    st["orders"] = [_order(hd, u).to(DEV) for u in (16, 4)]
    st["seq"] = torch.repeat_interleave(torch.arange(case["seqs"], device=DEV),
                                        torch.tensor(st["rows_host"], device=DEV))
    st["pos"] = _positions(st)
    return st


def _positions(st: dict) -> torch.Tensor:
    rows = torch.tensor(st["rows_host"], device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(st["rows_host"]), device=DEV), rows)
    first = st["lens"].long() - rows - st["start"][:-1].long()
    return torch.arange(st["T"], device=DEV) + first[seq]


# ------------------------------------------------------------------ plain form


def _floor_bf16(x: torch.Tensor) -> torch.Tensor:
    bits = x.view(torch.int32)
    cut = bits & -65536
    down = torch.where((bits < 0) & (bits != cut), cut + 65536, cut)
    return down.view(torch.float32)


def _quantise(x: torch.Tensor):
    """Codes (int64), s and b of rows [..., hd] in 32 bits; the quotient that
    is rounded to a code in 64, since a code's border decides it."""
    g = x.float().reshape(*x.shape[:-1], -1, 64)
    lo, hi = g.amin(-1), g.amax(-1)
    b = _floor_bf16(lo)
    # divided by a tensor: by a number it would be a product with 1/15, rounded
    s = (-_floor_bf16(-((hi - b) / torch.full_like(b, 15.0)))).clamp(min=2.0**-126)
    u = (g - b[..., None]).double() / s[..., None].double()
    return u.round().clamp(0, 15).reshape(x.shape), s, b


def _write_plain(st: dict) -> None:
    case = st["case"]
    seq, pos, page = st["seq"], st["pos"], case["page"]
    at, slot = st["table"][seq, pos // page].long(), pos % page
    for half, codes, pairs, order in zip((0, 1), (st["k"], st["v"]), (st["ks"], st["vs"]), st["orders"]):
        c, s, b = _quantise(st["kv"][: st["T"], half])
        c = c.to(torch.uint8)[..., order]
        codes[at, :, slot] = c[..., 0::2] | (c[..., 1::2] << 4)
        pairs[at, :, slot] = torch.stack([s, b], -1).bfloat16()


def _values_plain(st: dict, codes, pairs, order, seq, pos) -> torch.Tensor:
    """[..., nkv, hd] in 32 bits: the values at positions `pos` of sequences `seq`."""
    page = st["case"]["page"]
    at, slot = st["table"][seq, pos // page].long(), pos % page
    byte = codes[at, :, slot]
    c = torch.empty(*byte.shape[:-1], byte.shape[-1] * 2, device=DEV)
    nib = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).float()
    c[..., order] = nib
    p = pairs[at, :, slot].float()
    g = c.reshape(*c.shape[:-1], -1, 64)
    return (g * p[..., :1] + p[..., 1:]).reshape(c.shape)


def _read_plain(st: dict):
    seq, pos, dt = st["seq"], st["pos"], TYPES[st["case"]["type"]]
    k = _values_plain(st, st["k"], st["ks"], st["orders"][0], seq, pos)
    v = _values_plain(st, st["v"], st["vs"], st["orders"][1], seq, pos)
    return {"k": k.to(dt), "v": v.to(dt)}


def _attend_plain(st: dict) -> torch.Tensor:
    case = st["case"]
    nh, nkv, hd, n, dt = case["nh"], case["nkv"], case["hd"], case["seqs"], TYPES[case["type"]]
    G, L, R = nh // nkv, max(st["lens_host"]), max(st["rows_host"])
    T, seq, pos = st["T"], st["seq"], st["pos"]
    t = torch.arange(L, device=DEV)
    inside = t[None] < st["lens"][:, None]
    tt = torch.where(inside, t[None], 0)
    of = torch.arange(n, device=DEV)[:, None].expand(n, L)
    k = _values_plain(st, st["k"], st["ks"], st["orders"][0], of, tt)
    v = _values_plain(st, st["v"], st["vs"], st["orders"][1], of, tt)
    # rows padded to the longest sequence's
    i = torch.arange(T, device=DEV) - st["start"][seq].long()
    q = torch.zeros(n, R, nh, hd, device=DEV)
    q[seq, i] = st["q"][:T, :, :hd].float()
    see = torch.zeros(n, R, L, dtype=torch.bool, device=DEV)
    vis = (t[None] <= pos[:, None])
    if case["budget"]:
        nblk, blk = ((pos + 1) // RATIO)[:, None], (t // RATIO)[None]
        bit = (st["mask"][:, (t // RATIO) // 32] >> ((t // RATIO) % 32)) & 1
        vis = vis & ((blk >= nblk) | (nblk <= case["budget"] // RATIO) | (bit == 1))
    see[seq, i] = vis
    # [n, nkv, G R, hd] x [n, nkv, hd, L]
    q = q.view(n, R, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, G * R, hd)
    s = torch.matmul(q * hd**-0.5, k.permute(0, 2, 3, 1).contiguous()).view(n, nkv, G, R, L)
    s = s.masked_fill(~see[:, None, None], float("-inf"))
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    den = s.sum(-1)
    o = torch.matmul(s.view(n, nkv, G * R, L), v.permute(0, 2, 1, 3).contiguous()).view(n, nkv, G, R, hd)
    o = o / torch.where(den > 0, den, 1.0)[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(n, R, nh, hd)[seq, i]
    if case["gated"]:
        o = o * torch.sigmoid(st["q"][:T, :, hd:].float())
    return o.to(dt)


# ------------------------------------------------------------------ the framework's calls


def _handle(st: dict):
    """What a program keeps beside its buffers: the cache's and the batch's
    descriptions, the workspace and the library."""
    import ctypes as C

    from cherenkov_amd import abi

    case, L = st["case"], abi.lib()
    nkv, hd, T = case["nkv"], case["hd"], st["T"]
    cache = abi.ChkKvQ4(st["k"].data_ptr(), st["v"].data_ptr(), st["ks"].data_ptr(), st["vs"].data_ptr(),
                        st["k"].shape[0], case["page"], nkv, hd)
    seqs = abi.ChkKvSeqs(st["table"].data_ptr(), st["lens"].data_ptr(), st["start"].data_ptr(), case["seqs"],
                         st["table"].shape[1], T)
    dt = {"f32": abi.CHK_F32, "f16": abi.CHK_F16, "bf16": abi.CHK_BF16}[case["type"]]
    c, s = C.byref(cache), C.byref(seqs)
    calls, keep = [], [cache, seqs]
    if case["kind"] in ("step", "write"):
        kv = st["kv"]
        calls.append((L.chk_kv_append_q4, (c, s, kv[:, 0].data_ptr(), kv[:, 1].data_ptr(), dt, kv.stride(0),
                                           kv.stride(0))))
    if case["kind"] in ("write", "read"):
        o = st["out"]
        calls.append((L.chk_kv_read_q4, (c, s, o[0].data_ptr(), o[1].data_ptr(), dt, o.stride(1), o.stride(1))))
    else:
        mask = None
        if case["budget"]:
            m = abi.ChkKvMask(st["mask"].data_ptr(), st["mask"].shape[1], RATIO, case["budget"] // RATIO)
            keep.append(m)
            mask = C.byref(m)
        need = C.c_uint64()
        abi.check(L.chk_attn_q4_workspace(case["nh"], nkv, hd, case["seqs"], T, C.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=DEV)
        keep.append(ws)
        q, o = st["q"], st["out"]
        calls.append((L.chk_attn_q4, (c, s, q.data_ptr(), case["nh"], int(case["gated"]), dt, q.stride(0), mask,
                                      o.data_ptr(), o.stride(0), ws.data_ptr(), need.value)))
    st["handle"] = (calls, keep, abi.check)
    return st["handle"]


def run(st: dict):
    kind, T = st["case"]["kind"], st["T"]
    if own:
        calls, _, check = st.get("handle") or _handle(st)
        stream = torch.cuda.current_stream().cuda_stream
        for fn, args in calls:
            check(fn(*args, stream))
        out = st["out"]
        return {"k": out[0, :T], "v": out[1, :T]} if kind in ("write", "read") else {"out": out[:T]}
    if kind in ("step", "write"):
        _write_plain(st)
    return _read_plain(st) if kind in ("write", "read") else {"out": _attend_plain(st)}


def work(case: dict) -> dict:
    lens, rows = _lengths(case)
    nkv, hd, size = case["nkv"], case["hd"], SIZES[case["type"]]
    T, row = sum(rows), 2 * nkv * hd
    if case["kind"] == "write":
        # the values in, the codes out and in again, the values out
        return {"bytes": T * row * 2 * (size + STORED), "flops": 8 * T * row}
    if case["kind"] == "read":
        return {"bytes": T * row * (size + STORED), "flops": 2 * T * row}
    pairs = cache = 0
    for n, r in zip(lens, rows):
        if not r:
            continue
        seen = [min(p + 1, case["budget"] + (p + 1) % RATIO) if case["budget"] else p + 1 for p in (n - r, n - 1)]
        if case["budget"]:
            pairs += sum(min(p + 1, case["budget"] + (p + 1) % RATIO) for p in range(n - r, n))
        else:
            pairs += r * (2 * n - r + 1) // 2
        cache += min(n, r * seen[1])
    nh = case["nh"]
    return {"bytes": cache * row * STORED + T * nh * hd * size * (3 if case["gated"] else 2)
            + (T * row * size if case["kind"] == "step" else 0), "flops": 4 * nh * hd * pairs}


# ------------------------------------------------------------------ 64 bits


def _round8(x: torch.Tensor, up: bool) -> torch.Tensor:
    """x (64 bits) rounded to 8 significant bits, upwards or downwards."""
    m, e = torch.frexp(x)
    m = m * 256
    return torch.ldexp((m.ceil() if up else m.floor()) / 256, e)


def _stands_for(x: torch.Tensor) -> torch.Tensor:
    """What rows [..., hd] stand for once stored."""
    g = x.float().unflatten(-1, (-1, 64))
    least = _round8(g.min(-1, keepdim=True).values.double(), False)
    # the step is defined through 32-bit roundings of the spread and its 15th
    spread = (g.max(-1, keepdim=True).values - least.float()) / torch.tensor(15.0, device=DEV)
    step = _round8(spread.double(), True).clamp(min=2.0**-126)
    off = (g - least.float()).double()
    return (torch.round(off / step).clamp(0, 15) * step + least).reshape(x.shape)


def _stored64(case: dict, st: dict, b: int, which: str) -> torch.Tensor:
    """[len, nkv, hd] of sequence b as the cache holds it before the call."""
    n, page, hd = st["lens_host"][b], case["page"], case["hd"]
    order = _order(hd, 16 if which == "k" else 4).tolist()
    ids = st["table"][b, : -(-n // page)].long()
    byte = st[which][ids].transpose(1, 2).reshape(-1, case["nkv"], hd // 2)[:n]
    pair = st[which + "s"][ids].transpose(1, 2).reshape(-1, case["nkv"], hd // 64, 2)[:n].double()
    x = torch.empty(n, case["nkv"], hd, dtype=torch.float64, device=DEV)
    x[..., order[0::2]] = (byte % 16).double()
    x[..., order[1::2]] = (byte // 16).double()
    return x * pair[..., 0].repeat_interleave(64, -1) + pair[..., 1].repeat_interleave(64, -1)


def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    lens, rows, hd = st["lens_host"], st["rows_host"], case["hd"]
    if case["kind"] == "write":
        kv = _stands_for(st["kv"][: st["T"]])
        return {"k": kv[:, 0], "v": kv[:, 1]}
    if case["kind"] == "read":
        return {w: torch.cat([_stored64(case, st, b, w)[lens[b] - rows[b]:] for b in range(case["seqs"])]) for w in "kv"}
    nh, nkv = case["nh"], case["nkv"]
    outs, at = [], 0
    for b in range(case["seqs"]):
        n, r = lens[b], rows[b]
        if not r:
            continue
        k, v = _stored64(case, st, b, "k"), _stored64(case, st, b, "v")
        if case["kind"] == "step":
            new = _stands_for(st["kv"][at:at + r])
            k[n - r:], v[n - r:] = new[:, 0], new[:, 1]
        q = st["q"][at:at + r].double()
        t = torch.arange(n, device=DEV)
        for i0 in range(0, r, 256):
            i1 = min(r, i0 + 256)
            p = torch.arange(n - r + i0, n - r + i1, device=DEV)[:, None]
            hide = t > p
            if case["budget"]:
                whole = (p + 1) // RATIO
                bits = st["mask"][at + i0:at + i1].long() & 0xFFFFFFFF
                picked = (bits[:, (t // RATIO) // 32] // 2 ** ((t // RATIO) % 32)) % 2 == 1
                hide = hide | ((whole > case["budget"] // RATIO) & (t // RATIO < whole) & ~picked)
            heads = []
            for h in range(nh):
                s = q[i0:i1, h, :hd] @ k[:, h * nkv // nh].T / math.sqrt(hd)
                o = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v[:, h * nkv // nh]
                heads.append(o / (1 + torch.exp(-q[i0:i1, h, hd:])) if case["gated"] else o)
            outs.append(torch.stack(heads, 1))
        at += r
    return {"out": torch.cat(outs)}
