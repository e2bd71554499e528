"""A step of a serving batch over the 4-bit key/value cache, as timed cases:
the batch's tables and slots planned on the device, queries and keys normed and
rotated, attention through a sliding window with first tokens that stay
visible, and attention of sequences that share a long prefix.

The cache is pages of `page` tokens per kv head.  64 consecutive dims of one
token and head are a group: 4-bit codes c, a bf16 step s and a bf16 least value
b, and the group stands for s c + b.  A row of hd dims is hd / 2 bytes, two
codes a byte, the lower nibble first, its dims in units of 16 (keys) or 4
(values) that take the groups in turn (`_dim_of`).

Where `own` is false every pass runs in elementary torch operations; where it
is true it goes through chk_kv_plan_q4, chk_qk_norm_rope, chk_attn_window_q4 and
chk_attn_prefix_q4.
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
NONE = -1  # 0xffffffff: no page, no position

# ------------------------------------------------------------------ cases
#
# plan    seqs requests of up to ctx tokens; each drops the last `drop` of them
#         (rejected drafts), a share `ended` of them all; each then wants `rows`
#         (ragged: up to that many), in row arrays `pad` longer; `free` spare pages
#         beside what they want, negative: too few
# rotate  rows of one fused projection (queries, gates, keys, values)
# window  rows at the end of each sequence see `sinks` first tokens and their
#         last `window`
# prefix  `groups` of `per` sequences with `shared` common tokens, `alone` others;
#         each goes on by up to ctx tokens of its own and its rows

MODEL = dict(nh=16, nkv=2, hd=256, gated=True, type="f32")
WIDE = dict(nh=32, nkv=8, hd=128, gated=False, type="bf16")


def listed() -> list[dict]:
    return [
        # the next token of one request: a length, at times a page
        dict(name="plan_1", kind="plan", seqs=1, ctx=2183, rows=1, ragged=False, drop=0, ended=0.0, pad=0, free=8, page=64),
        # a verify step of 64 requests: three drafts each, of which some were rejected; a few requests have ended
        dict(name="plan_64_verify", kind="plan", seqs=64, ctx=8191, rows=3, ragged=False, drop=3, ended=0.1, pad=7, free=50,
             page=16),
        # a full batch with prompts of all lengths among the single tokens, and a pool that runs out
        dict(name="plan_900_prompts", kind="plan", seqs=900, ctx=2000, rows=300, ragged=True, drop=4, ended=0.0, pad=1000,
             free=-900, page=16),
        # one token's heads, a quarter of each rotated
        dict(name="rotate_1", kind="rotate", rows=1, far=2184, rot=64, theta=1e7, blank=0, **MODEL),
        # a turn's rows behind a long conversation, a padded batch
        dict(name="rotate_333", kind="rotate", rows=333, far=131000, rot=64, theta=1e7, blank=11, nh=24, nkv=2, hd=256,
             gated=False, type="f16"),
        # prompts, heads rotated whole
        dict(name="rotate_16k", kind="rotate", rows=16389, far=32000, rot=128, theta=1e4, blank=0, **WIDE),
        # a token far into a conversation that keeps its last 2048 tokens and the first four
        dict(name="window_1", kind="window", seqs=1, rows=1, ctx=31999, ragged=False, window=2048, sinks=4, page=64, **MODEL),
        # a serving batch of all lengths, short pages, odd window
        dict(name="window_64_ragged", kind="window", seqs=64, rows=1, ctx=8191, ragged=True, window=1000, sinks=5, page=16,
             **WIDE),
        # prompts far longer than the window
        dict(name="window_prompts", kind="window", seqs=2, rows=8191, ctx=0, ragged=True, window=1024, sinks=64, page=128,
             **WIDE),
        # four continuations of one prompt
        dict(name="prefix_4", kind="prefix", groups=1, per=4, alone=0, shared=2048, ctx=37, rows=1, ragged=False, page=64,
             **MODEL),
        # a batch of requests behind one long instruction, lengths of their own
        dict(name="prefix_64_ragged", kind="prefix", groups=1, per=64, alone=0, shared=8192, ctx=700, rows=1, ragged=True,
             page=16, **WIDE),
        # verify rows of two groups over long documents, and requests of neither
        dict(name="prefix_2_verify", kind="prefix", groups=2, per=12, alone=3, shared=30000, ctx=900, rows=3, ragged=True,
             page=256, nh=24, nkv=2, hd=256, gated=False, type="f16"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["plan", "rotate", "window", "window", "prefix", "prefix"])
    if kind == "plan":
        seqs = _log(rng, 1, 1024)
        rows = rng.choice([1, 1, 2, 4, _log(rng, 1, max(2, 200000 // seqs))])
        return dict(kind=kind, seqs=seqs, ctx=_log(rng, 1, min(131071, 4000000 // seqs)), rows=rows,
                    ragged=rng.random() < 0.6, drop=rng.choice([0, 0, 1, 4, 40]), ended=rng.choice([0.0, 0.0, 0.1, 0.5]),
                    pad=rng.choice([0, 1, 333]), free=rng.choice([0, 5, 1000, -1, -20, -500]),
                    page=rng.choice([16, 32, 64, 256, 1024]))
    nkv, hd = rng.choice([1, 2, 4, 8]), rng.choice([128, 256])
    g = rng.choice([1, 2, 4, 8, 12])
    heads = dict(nh=nkv * g, nkv=nkv, hd=hd, gated=rng.random() < 0.5, type=rng.choice(["f32", "f16", "bf16"]))
    if kind == "rotate":
        heads["hd"] = hd = rng.choice([64, 128, 256])
        most = 80_000_000 // ((heads["nh"] * (2 if heads["gated"] else 1) + nkv) * hd)
        return dict(kind=kind, rows=_log(rng, 1, min(most, 16384)), far=_log(rng, 10, 1_000_000),
                    rot=rng.choice([hd // 4, hd // 2, hd, 20]), theta=rng.choice([1e4, 1e7]),
                    blank=rng.choice([0, 0, 1, 9]), **heads)
    page = rng.choice([16, 32, 64, 128, 256, 1024])
    if kind == "window":
        c = dict(kind=kind, ragged=rng.random() < 0.6, window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 17, 64, 200]),
                 page=page, **heads)
        if rng.random() < 0.6:
            c["seqs"], c["rows"] = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 3, 4])
            c["ctx"] = _log(rng, 1, min(131071, 8 * 131072 * 512 // (c["seqs"] * nkv * hd)))
        else:
            # no dearer than window_prompts: rows x (window + sinks) pairs a sequence
            c["seqs"] = rng.choice([1, 1, 2, 3, 5])
            c["rows"] = _log(rng, 5, 8192)
            c["ctx"] = rng.choice([0, _log(rng, 1, 30000)])
            pairs = 5e10 / (c["seqs"] * nkv * g * hd)
            c["rows"] = max(1, min(c["rows"], int(pairs / (c["window"] + c["sinks"]))))
        return c
    c = dict(kind=kind, groups=rng.choice([1, 1, 2, 3]), per=_log(rng, 1, 64), alone=rng.choice([0, 0, 1, 5]),
             ctx=_log(rng, 1, 2000), rows=rng.choice([1, 1, 1, 2, 4, _log(rng, 1, 100)]), ragged=rng.random() < 0.6, page=page,
             **heads)
    n = c["groups"] * c["per"] + c["alone"]
    pairs = 5e10 / (n * c["rows"] * nkv * g * hd)
    c["shared"] = _log(rng, 16, int(max(17, min(60000, pairs))))
    return c


def _share(b: int, ragged: bool) -> float:
    return (0.37 + 0.6180339887 * b) % 1.0 if ragged and b else 1.0


def _batch(case: dict) -> tuple[list[int], list[int], list[int]]:
    """Tokens of each sequence (this call's rows included), those rows, and the
    tokens that it shares with its group."""
    if case["kind"] == "window":
        n, shared = case["seqs"], [0] * case["seqs"]
    else:
        n = case["groups"] * case["per"] + case["alone"]
        # whole pages are shared, a little fewer in each further group
        of = [max(1, int(case["shared"] * 0.8**g)) // case["page"] * case["page"] for g in range(case["groups"])]
        shared = [of[b // case["per"]] if b < case["groups"] * case["per"] else 0 for b in range(n)]
    step = case["rows"] <= 4
    rows = [case["rows"] if step else max(1, int(case["rows"] * _share(b, case["ragged"]))) for b in range(n)]
    if case["ragged"] and n > 2:
        rows[n // 2] = 0
    return [s + int(case["ctx"] * _share(b, case["ragged"])) + r for b, (s, r) in enumerate(zip(shared, rows))], rows, shared


# ------------------------------------------------------------------ inputs


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 6271 + 17)


def _dim_of(hd: int, unit: int) -> torch.Tensor:
    """The dim of each code of a stored row: units of `unit` dims, unit u the
    (u / groups)-th of group u % groups."""
    i, groups = torch.arange(hd), hd // 64
    u = i // unit
    return 64 * (u % groups) + unit * (u // groups) + i % unit


def _plane(g: torch.Generator, case: dict, pages: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Bytes and (s, b) pairs as normed rows leave them, a few groups louder."""
    nkv, page, hd = case["nkv"], case["page"], case["hd"]
    c = torch.randn(pages, nkv, page, hd, generator=g, device=DEV).mul_(2.9).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
    codes = c[..., 0::2] | (c[..., 1::2] << 4)
    s = 0.3 * torch.exp(0.25 * torch.randn(pages, nkv, page, hd // 64, generator=g, device=DEV))
    s = (s * (1 + 2 * (torch.rand(nkv, 1, hd // 64, generator=g, device=DEV) < 0.25))).bfloat16()
    b = (-7.5 * s.float() + 0.2 * torch.randn(pages, nkv, page, hd // 64, generator=g, device=DEV)).bfloat16()
    return codes.contiguous(), torch.stack([s, b], -1).contiguous()


def _i32(x) -> torch.Tensor:
    return torch.tensor(np.asarray(x, np.int64), device=DEV).to(torch.int32)


def _inputs_plan(case: dict, seed: int) -> dict:
    rng = np.random.default_rng(seed * 101 + 7)
    n, page = case["seqs"], case["page"]
    lens = np.array([1 + int((case["ctx"] - 1) * _share(b, case["ragged"])) for b in range(n)])
    gone = rng.random(n) < case["ended"]
    keep = np.where(gone, 0, np.maximum(lens - rng.integers(0, case["drop"] + 1, n), 0))
    # most requests of a ragged batch want a token, some a prompt
    want = np.full(n, case["rows"])
    if case["ragged"]:
        want = np.array([1 if b % 10 < 7 else 1 + int((case["rows"] - 1) * _share(b, True)) for b in range(n)])
    rows = int(want.sum()) + case["pad"]
    want = np.where(gone, 0, rng.permutation(want))
    # some begin with pages of another's
    held = -(-lens // page)
    first = np.where(rng.random(n) < 0.2, np.minimum(held, 2), 0)
    # (a length never falls below what a request does not own itself, unless it ends)
    keep = np.where(gone, keep, np.maximum(keep, np.minimum(first * page, lens)))
    width = int((-(-(lens + case["rows"]) // page)).max()) + 1
    need = np.maximum(-(-(keep + want) // page) - -(-keep // page), 0).sum()
    back = np.maximum(held - np.maximum(-(-keep // page), first), 0).sum()
    spare = max(0, int(need - back) + case["free"])
    # (a pool that holds more than these requests have and may take)
    pages = int(held.sum()) + rows // page + n + max(0, case["free"])
    ids = rng.permutation(pages)
    table = np.full((n, width), NONE)
    at = 0
    for b in range(n):
        table[b, : held[b]] = ids[at : at + held[b]]
        at += held[b]
    free = np.full(pages, NONE)
    free[:spare] = ids[at : at + spare]
    return dict(table=_i32(table), len=_i32(lens), free=_i32(free), nfree=_i32([spare, 0]), keep=_i32(keep), first=_i32(first),
                want=_i32(want), pages=pages, width=width, rows=rows,
                host=dict(table=table, len=lens, free=free, nfree=spare, keep=keep, first=first, want=want))


def _inputs_rotate(case: dict, seed: int) -> dict:
    g = _gen(seed)
    rows, nh, nkv, hd = case["rows"], case["nh"], case["nkv"], case["hd"]
    wide = nh * hd * (2 if case["gated"] else 1)
    x = torch.randn(rows, wide + 2 * nkv * hd, generator=g, device=DEV)
    x[:, ::29] *= 6
    w = (1 + 0.3 * torch.randn(2, hd, generator=g, device=DEV)).bfloat16()
    pos = torch.randint(0, case["far"], (rows,), generator=g, device=DEV, dtype=torch.int32)
    if case["blank"]:  # rows of a padded batch
        pos[max(1, rows - case["blank"]) :] = NONE
    return dict(x=x.to(TYPES[case["type"]]), w=w, pos=pos, wide=wide)


def _inputs_attend(case: dict, seed: int) -> dict:
    g = _gen(seed)
    lens, rows, shared = _batch(case)
    page, n = case["page"], len(lens)
    width = max(1, -(-max(lens) // page))
    per = case.get("per", 1)
    held, owned = [-(-t // page) for t in lens], []
    # a group's common pages are the first sequence's
    lead = [b // per * per if shared[b] else b for b in range(n)]
    owned = [h - (shared[b] // page if lead[b] != b else 0) for b, h in enumerate(held)]
    pages = sum(owned) + 3
    ids = np.asarray(torch.randperm(pages, generator=g, device=DEV).cpu())
    table = np.zeros((n, width), np.int64)
    at = 0
    for b in range(n):
        common = shared[b] // page if lead[b] != b else 0
        table[b, :common] = table[lead[b], :common]
        table[b, common : held[b]] = ids[at : at + owned[b]]
        at += owned[b]
    k, ks = _plane(g, case, pages)
    v, vs = _plane(g, case, pages)
    start = np.concatenate([[0], np.cumsum(rows)])
    T = int(start[-1])
    st = dict(k=k, v=v, ks=ks, vs=vs, table=_i32(table), len=_i32(lens), start=_i32(start), lens=lens, rows=rows, shared=shared,
              T=T, width=width)
    st["q"] = torch.randn(max(T, 1), case["nh"], case["hd"] * (2 if case["gated"] else 1), generator=g,
                          device=DEV).to(TYPES[case["type"]])
    if case["kind"] == "prefix":
        st["first"] = _i32([per * i for i in range(case["groups"] + 1)])
        st["tokens"] = _i32([shared[per * i] for i in range(case["groups"])])
    return st


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    if kind == "plan":
        st = _inputs_plan(case, seed)
        st["start"] = torch.zeros(case["seqs"] + 1, dtype=torch.int32, device=DEV)
        st["pos"] = torch.zeros(st["rows"], dtype=torch.int32, device=DEV)
        st["slot"] = torch.zeros(st["rows"], dtype=torch.int64, device=DEV)
    elif kind == "rotate":
        st = _inputs_rotate(case, seed)
        dt, rows = TYPES[case["type"]], case["rows"]
        st["q_out"] = torch.zeros(rows, st["wide"], dtype=dt, device=DEV)
        st["k_out"] = torch.zeros(rows, case["nkv"] * case["hd"], dtype=dt, device=DEV)
        j = torch.arange(case["rot"] // 2, dtype=torch.float64)
        st["freq"] = (case["theta"] ** (-2 * j / case["rot"])).to(DEV)
    else:
        st = _inputs_attend(case, seed)
        st["out"] = torch.zeros(max(st["T"], 1), case["nh"], case["hd"], dtype=TYPES[case["type"]], device=DEV)
        st["dims"] = [_dim_of(case["hd"], u).to(DEV) for u in (16, 4)]
    st["case"] = case
    return st


# ------------------------------------------------------------------ plain forms


def _pages(t: torch.Tensor, page: int) -> torch.Tensor:
    return (t + page - 1) // page


def _plan_plain(st: dict) -> dict:
    """Rows of a table at once, whole-table masks; one state to the next in place."""
    case = st["case"]
    page, width, rows, pages, n = case["page"], st["width"], st["rows"], st["pages"], case["seqs"]
    table, free = st["table"].long(), st["free"].long()
    held0 = _pages(st["len"].long(), page)
    have = torch.minimum(st["keep"].long(), st["len"].long())
    held1 = _pages(have, page)
    e = torch.arange(width, device=DEV)[None]
    # pages given back go on top of the list, the last sequence's last page first
    low = torch.maximum(held1, st["first"].long())
    back = (held0 - low).clamp(min=0)
    behind = back.flip(0).cumsum(0).flip(0) - back
    gives = (e >= low[:, None]) & (e < held0[:, None])
    at = st["nfree"][0].long() + behind[:, None] + held0[:, None] - 1 - e
    room = torch.cat([free, free.new_zeros(1)])
    room.scatter_(0, torch.where(gives, at, pages).flatten(), table.flatten())
    room = room[:pages]
    avail = st["nfree"][0].long() + back.sum()
    # who is served: rows and table have room, and the pages last
    want = st["want"].long()
    want = torch.where(have + want > width * page, 0, want)
    want = torch.where(want.cumsum(0) > rows, 0, want)
    need = _pages(have + want, page) - held1
    upto = need.cumsum(0)
    served = (need == 0) | (upto <= avail)
    want = torch.where(served, want, 0)
    got = torch.where(served, need, 0)
    takes = (e >= held1[:, None]) & (e < (held1 + got)[:, None])
    src = avail - 1 - (upto - need)[:, None] - (e - held1[:, None])
    gone = (e >= (held1 + got)[:, None]) & (e >= low[:, None]) & (e < held0[:, None])
    table = torch.where(takes, room[src.clamp(0, pages - 1)], torch.where(gone, NONE, table))
    now = have + want
    start = torch.cat([want.new_zeros(1), want.cumsum(0)])
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(start[1:], r, right=True).clamp(max=n - 1)
    pos = now[b] - (start[b + 1] - r)
    slot = table[b, (pos // page).clamp(0, width - 1)] * page + pos % page
    live = r < start[-1]
    st["table"].copy_(table)
    st["free"].copy_(room)
    st["len"].copy_(now)
    st["nfree"].copy_(torch.stack([avail - got.sum(), (upto[-1] - avail).clamp(min=0)]))
    st["start"].copy_(start)
    st["pos"].copy_(torch.where(live, pos, NONE))
    st["slot"].copy_(torch.where(live, slot, NONE))
    return _plan_out(st)


def _plan_out(st: dict) -> dict:
    return {k: st[k] for k in ("table", "len", "free", "nfree", "start", "pos", "slot")}


EPS = 1e-6


def _rotate_plain(st: dict) -> dict:
    case = st["case"]
    rows, nh, nkv, hd, rot = case["rows"], case["nh"], case["nkv"], case["hd"], case["rot"]
    per = hd * (2 if case["gated"] else 1)
    live = (st["pos"] >= 0)[:, None]
    # far positions' angles in 64 bits
    turn = st["pos"].double()[:, None] * st["freq"][None]
    cos, sin = torch.cos(turn).float()[:, None], torch.sin(turn).float()[:, None]

    def one(x, w):
        x = x.float()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y[..., : rot // 2], y[..., rot // 2 : rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], -1)

    q = st["x"][:, : nh * per].view(rows, nh, per)
    k = st["x"][:, nh * per : nh * per + nkv * hd].view(rows, nkv, hd)
    yq = one(q[..., :hd], st["w"][0])
    if case["gated"]:
        yq = torch.cat([yq, q[..., hd:].float()], -1)
    dt = TYPES[case["type"]]
    st["q_out"].copy_(torch.where(live, yq.reshape(rows, -1).to(dt), st["q_out"]))
    st["k_out"].copy_(torch.where(live, one(k, st["w"][1]).reshape(rows, -1).to(dt), st["k_out"]))
    return {"q": st["q_out"], "k": st["k_out"]}


def _values(st: dict, which: str, seq: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
    """[..., nkv, hd] in 32 bits: tokens t of sequences seq."""
    page = st["case"]["page"]
    at, slot = st["table"][seq, t // page].long(), t % page
    byte, pair = st[which][at, :, slot], st[which + "s"][at, :, slot].float()
    c = torch.empty(*byte.shape[:-1], byte.shape[-1] * 2, device=DEV)
    c[..., st["dims"][0 if which == "k" else 1]] = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).float()
    g = c.unflatten(-1, (-1, 64))
    return (g * pair[..., :1] + pair[..., 1:]).flatten(-2)


def _queries(st: dict, r0: int, r1: int) -> torch.Tensor:
    """[nkv, group, rows, hd] in 32 bits, scaled."""
    case = st["case"]
    q = st["q"][r0:r1, :, : case["hd"]].float() * case["hd"] ** -0.5
    return q.unflatten(1, (case["nkv"], -1)).permute(1, 2, 0, 3)


def _out(st: dict, r0: int, r1: int, num: torch.Tensor, den: torch.Tensor) -> None:
    """Rows r0.. from [nkv, group, rows, hd] numerators and their sums."""
    case = st["case"]
    o = (num / den).permute(2, 0, 1, 3).flatten(1, 2)
    if case["gated"]:
        o = o * torch.sigmoid(st["q"][r0:r1, :, case["hd"] :].float())
    st["out"][r0:r1] = o.to(st["out"].dtype)


def _softmax_of(parts: list, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Numerators and sums over parts (scores [nkv, G, rows, t], values [nkv, t, hd])."""
    top = torch.stack([s.amax(-1) for s, _ in parts if s.shape[-1]]).amax(0)[..., None]
    num, den = 0.0, 0.0
    for s, v in parts:
        e = torch.exp(s - top)
        num = num + torch.matmul(e.flatten(1, 2), v).view(*e.shape[:3], -1)
        den = den + e.sum(-1, keepdim=True)
    return num, den


def _scores(q: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """[nkv, G, rows, t] of q [nkv, G, rows, hd] and k [t, nkv, hd]."""
    return torch.matmul(q.flatten(1, 2), k.permute(1, 2, 0).contiguous()).view(*q.shape[:3], -1)


def _window_plain(st: dict) -> torch.Tensor:
    """Sequence by sequence, up to 1024 rows at a time over the tokens that any of them sees."""
    case = st["case"]
    win, sinks, r0 = case["window"], case["sinks"], 0
    for b, (n, rows) in enumerate(zip(st["lens"], st["rows"])):
        for i in range(0, rows, 1024):
            m = min(1024, rows - i)
            p0, p1 = n - rows + i, n - rows + i + m - 1
            low = max(0, p0 - win + 1)
            cut = min(sinks, low)
            t = torch.cat([torch.arange(cut, device=DEV), torch.arange(low, p1 + 1, device=DEV)])
            p = torch.arange(p0, p1 + 1, device=DEV)[:, None]
            see = (t[None] <= p) & ((t[None] > p - win) | (t[None] < sinks))
            seq = torch.full_like(t, b)
            q = _queries(st, r0 + i, r0 + i + m)
            s = _scores(q, _values(st, "k", seq, t)).masked_fill(~see, float("-inf"))
            v = _values(st, "v", seq, t).permute(1, 0, 2).contiguous()
            _out(st, r0 + i, r0 + i + m, *_softmax_of([(s, v)], m))
        r0 += rows
    return st["out"][: st["T"]]


def _prefix_plain(st: dict) -> torch.Tensor:
    """A group's common tokens against all of its rows at once, then each sequence's own."""
    case = st["case"]
    per, n = case["per"], len(st["lens"])
    starts = np.concatenate([[0], np.cumsum(st["rows"])])
    spans = [(g * per, (g + 1) * per) for g in range(case["groups"])]
    spans += [(b, b + 1) for b in range(case["groups"] * per, n)]
    for b0, b1 in spans:
        P, r0, r1 = st["shared"][b0], int(starts[b0]), int(starts[b1])
        if r0 == r1:
            continue
        q = _queries(st, r0, r1)
        t = torch.arange(P, device=DEV)
        first = torch.full_like(t, b0)
        common = _scores(q, _values(st, "k", first, t))
        vc = _values(st, "v", first, t).permute(1, 0, 2).contiguous()
        for b in range(b0, b1):
            rows = st["rows"][b]
            if rows == 0:
                continue
            i0, i1 = int(starts[b]) - r0, int(starts[b]) - r0 + rows
            t = torch.arange(P, st["lens"][b], device=DEV)
            p = torch.arange(st["lens"][b] - rows, st["lens"][b], device=DEV)[:, None]
            seq = torch.full_like(t, b)
            s = _scores(q[:, :, i0:i1], _values(st, "k", seq, t)).masked_fill(t[None] > p, float("-inf"))
            v = _values(st, "v", seq, t).permute(1, 0, 2).contiguous()
            _out(st, r0 + i0, r0 + i1, *_softmax_of([(common[:, :, i0:i1], vc), (s, v)], rows))
    return st["out"][: st["T"]]


# ------------------------------------------------------------------ the framework's calls


def _handle(st: dict):
    """What a program keeps beside its buffers: descriptions, the rotation's
    table, the workspace and the library."""
    import ctypes as C

    from cherenkov_amd import abi

    case, L, kind = st["case"], abi.lib(), st["case"]["kind"]
    if kind == "plan":
        # (a request that holds less than its first pages, and goes on, goes on in a page of its own)
        last = st["keep"] // case["page"]
        st["own"] = torch.where((st["keep"] % case["page"] > 0) & (last < st["first"]), last, st["first"])
        pool = abi.ChkKvPool(st["table"].data_ptr(), st["len"].data_ptr(), st["free"].data_ptr(), st["nfree"].data_ptr(),
                             case["seqs"], st["width"], case["page"], st["pages"])
        keep = [pool]
        call = (L.chk_kv_plan_q4, (C.byref(pool), st["keep"].data_ptr(), st["own"].data_ptr(), st["want"].data_ptr(),
                                   st["rows"], st["start"].data_ptr(), st["pos"].data_ptr(), st["slot"].data_ptr()))
    elif kind == "rotate":
        turn = (C.c_uint64 * (case["rot"] // 2))()
        abi.check(L.chk_rope_turns(case["theta"], case["rot"], turn))
        turns = torch.tensor(np.frombuffer(turn, np.int64).copy(), device=DEV)
        norm = abi.ChkQkNorm(st["w"][0].data_ptr(), st["w"][1].data_ptr(), turns.data_ptr(), case["rot"], case["nh"],
                             case["nkv"], case["hd"], int(case["gated"]), EPS)
        dt = {"f32": abi.CHK_F32, "f16": abi.CHK_F16, "bf16": abi.CHK_BF16}[case["type"]]
        x, q, k = st["x"], st["q_out"], st["k_out"]
        keep = [turns, norm]
        call = (L.chk_qk_norm_rope, (C.byref(norm), st["pos"].data_ptr(), case["rows"], x.data_ptr(), x.stride(0),
                                     q.data_ptr(), q.stride(0), x[:, st["wide"]:].data_ptr(), x.stride(0), k.data_ptr(),
                                     k.stride(0), dt))
    else:
        cache = abi.ChkKvQ4(st["k"].data_ptr(), st["v"].data_ptr(), st["ks"].data_ptr(), st["vs"].data_ptr(),
                            st["k"].shape[0], case["page"], case["nkv"], case["hd"])
        n, T = len(st["lens"]), st["T"]
        seqs = abi.ChkKvSeqs(st["table"].data_ptr(), st["len"].data_ptr(), st["start"].data_ptr(), n, st["width"], T)
        dt = {"f32": abi.CHK_F32, "f16": abi.CHK_F16, "bf16": abi.CHK_BF16}[case["type"]]
        need, q, o = C.c_uint64(), st["q"], st["out"]
        keep = [cache, seqs]
        if kind == "window":
            abi.check(L.chk_attn_q4_workspace(case["nh"], case["nkv"], case["hd"], n, T, C.byref(need)))
            how = (case["window"], case["sinks"])
            fn = L.chk_attn_window_q4
        else:
            abi.check(L.chk_attn_prefix_q4_workspace(case["nh"], case["nkv"], case["hd"], n, T, case["groups"], C.byref(need)))
            shared = abi.ChkKvShared(st["first"].data_ptr(), st["tokens"].data_ptr(), case["groups"])
            keep.append(shared)
            how = (C.byref(shared),)
            fn = L.chk_attn_prefix_q4
        ws = torch.empty(need.value, dtype=torch.uint8, device=DEV)
        keep.append(ws)
        call = (fn, (C.byref(cache), C.byref(seqs), q.data_ptr(), case["nh"], int(case["gated"]), dt, q.stride(0), *how,
                     o.data_ptr(), o.stride(0), ws.data_ptr(), need.value))
    st["handle"] = (*call, keep, abi.check)
    return st["handle"]


def run(st: dict):
    kind = st["case"]["kind"]
    if own:
        fn, args, _, check = st.get("handle") or _handle(st)
        check(fn(*args, torch.cuda.current_stream().cuda_stream))
        if kind == "plan":
            return _plan_out(st)
        return {"q": st["q_out"], "k": st["k_out"]} if kind == "rotate" else {"out": st["out"][: st["T"]]}
    if kind == "plan":
        return _plan_plain(st)
    if kind == "rotate":
        return _rotate_plain(st)
    return {"out": _window_plain(st) if kind == "window" else _prefix_plain(st)}


# ------------------------------------------------------------------ what cannot be done without


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "plan":
        n, page = case["seqs"], case["page"]
        rows = n * case["rows"] if not case["ragged"] else int(n * (0.85 + 0.15 * case["rows"]))
        # lengths, wants, keeps and starts; a table entry and a slot a row; pages in and out
        return {"bytes": n * 4 * 6 + rows * (4 + 8) + (rows // page + n) * 8, "flops": 4 * rows + 16 * n}
    size, nkv, hd, nh = SIZES[case["type"]], case["nkv"], case["hd"], case["nh"]
    if kind == "rotate":
        rows = max(1, case["rows"] - case["blank"])
        q = nh * hd * (2 if case["gated"] else 1)
        return {"bytes": rows * ((q + nkv * hd) * size * 2 + 4) + 4 * hd + 4 * case["rot"],
                "flops": rows * (nh + nkv) * (4 * hd + 3 * case["rot"])}
    lens, rows, shared = _batch(case)
    pairs = cache = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        if r == 0:
            continue
        if kind == "window":
            most = case["window"] + case["sinks"]
            pairs += sum(min(p + 1, most) for p in range(n - r, n))
            cache += min(n, most + r - 1)
        else:
            pairs += r * (2 * n - r + 1) // 2
            cache += n - shared[b] + (shared[b] if b % case["per"] == 0 else 0)
    return {"bytes": cache * 2 * nkv * hd * STORED + sum(rows) * nh * hd * size * (3 if case["gated"] else 2),
            "flops": 4 * nh * hd * pairs}


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _exact_plan(case: dict, seed: int) -> dict:
    """The rules one sequence and one page at a time, on a stack of free pages."""
    st = _inputs_plan(case, seed)
    h, page, width, rows = st["host"], case["page"], st["width"], st["rows"]
    table, n = h["table"].copy(), case["seqs"]
    stack, nf = h["free"].copy(), h["nfree"]
    lens = []
    for b in reversed(range(n)):
        left = min(int(h["keep"][b]), int(h["len"][b]))
        for e in reversed(range(max(-(-left // page), int(h["first"][b])), -(-int(h["len"][b]) // page))):
            stack[nf] = table[b, e]
            nf += 1
            table[b, e] = NONE
        lens.append(left)
    lens.reverse()
    wanted = total = 0
    avail, start, pos, slot = nf, [0], [], []
    for b in range(n):
        w = int(h["want"][b])
        if lens[b] + w > width * page:
            w = 0
        wanted += w
        if wanted > rows:
            w = 0
        need = -(-(lens[b] + w) // page) - -(-lens[b] // page)
        total += need
        if need and total > avail:
            w = need = 0
        for i in range(need):
            nf -= 1
            table[b, -(-lens[b] // page) + i] = stack[nf]
        for p in range(lens[b], lens[b] + w):
            pos.append(p)
            slot.append(int(table[b, p // page]) * page + p % page)
        lens[b] += w
        start.append(start[-1] + w)
    blank = [NONE] * (rows - len(pos))
    return {"table": _i32(table), "len": _i32(lens), "free": _i32(stack), "nfree": _i32([nf, max(0, total - avail)]),
            "start": _i32(start), "pos": _i32(pos + blank), "slot": torch.tensor(slot + blank, dtype=torch.int64, device=DEV)}


def _exact_rotate(case: dict, seed: int) -> dict:
    st = _inputs_rotate(case, seed)
    rows, nh, nkv, hd, rot = case["rows"], case["nh"], case["nkv"], case["hd"], case["rot"]
    x, w = st["x"].double(), st["w"].double()
    pos = st["pos"].double()
    half = rot // 2
    j = torch.arange(half, dtype=torch.float64, device=DEV)
    z = torch.polar(torch.ones(rows, half, dtype=torch.float64, device=DEV),
                    pos[:, None] * torch.exp(-2 * j / rot * math.log(case["theta"])))
    q_out = torch.zeros(rows, st["wide"], dtype=torch.float64, device=DEV)
    k_out = torch.zeros(rows, nkv * hd, dtype=torch.float64, device=DEV)
    live = st["pos"] >= 0
    per = hd * (2 if case["gated"] else 1)
    for h in range(nh + nkv):
        at = h * per if h < nh else st["wide"] + (h - nh) * hd
        v = x[:, at : at + hd]
        v = v * torch.rsqrt(v.square().sum(-1, keepdim=True) / hd + EPS) * w[0 if h < nh else 1]
        c = torch.complex(v[:, :half], v[:, half:rot]) * z
        v = torch.cat([c.real, c.imag, v[:, rot:]], 1)
        to, o = (q_out, h * per) if h < nh else (k_out, (h - nh) * hd)
        to[live, o : o + hd] = v[live]
        if h < nh and case["gated"]:
            to[live, o + hd : o + per] = x[live, at + hd : at + per]
    return {"q": q_out, "k": k_out}


def _stored64(case: dict, st: dict, b: int, which: str, t0: int, t1: int) -> torch.Tensor:
    """[t1 - t0, nkv, hd]: what tokens t0.. of sequence b stand for."""
    page, hd = case["page"], case["hd"]
    dims = _dim_of(hd, 16 if which == "k" else 4).tolist()
    t = torch.arange(t0, t1, device=DEV)
    ids = st["table"][b].long()[t // page]
    byte, pair = st[which][ids, :, t % page], st[which + "s"][ids, :, t % page].double()
    x = torch.empty(t1 - t0, case["nkv"], hd, dtype=torch.float64, device=DEV)
    x[..., dims[0::2]] = (byte % 16).double()
    x[..., dims[1::2]] = (byte // 16).double()
    return x * pair[..., 0].repeat_interleave(64, -1) + pair[..., 1].repeat_interleave(64, -1)


def _exact_attend(case: dict, seed: int) -> dict:
    st = _inputs_attend(case, seed)
    hd, nh, nkv = case["hd"], case["nh"], case["nkv"]
    win = case.get("window", 1 << 40)
    sinks = case.get("sinks", 0)
    outs, at = [], 0
    for b, (n, rows) in enumerate(zip(st["lens"], st["rows"])):
        for i in range(0, rows, 512):
            m = min(512, rows - i)
            p = torch.arange(n - rows + i, n - rows + i + m, device=DEV)[:, None]
            low, high = max(0, n - rows + i - win + 1), n - rows + i + m
            head = min(sinks, low)
            t = torch.cat([torch.arange(head, device=DEV), torch.arange(low, high, device=DEV)])
            k = torch.cat([_stored64(case, st, b, "k", 0, head), _stored64(case, st, b, "k", low, high)])
            v = torch.cat([_stored64(case, st, b, "v", 0, head), _stored64(case, st, b, "v", low, high)])
            hide = (t > p) | ((t <= p - win) & (t >= sinks))
            q = st["q"][at + i : at + i + m].double()
            heads = []
            for h in range(nh):
                s = q[:, h, :hd] @ k[:, h * nkv // nh].T / math.sqrt(hd)
                o = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v[:, h * nkv // nh]
                heads.append(o / (1 + torch.exp(-q[:, h, hd:])) if case["gated"] else o)
            outs.append(torch.stack(heads, 1))
        at += rows
    return {"out": torch.cat(outs) if outs else torch.zeros(0, nh, hd, dtype=torch.float64, device=DEV)}


def exact(case: dict, seed: int):
    if case["kind"] == "plan":
        return _exact_plan(case, seed)
    return _exact_rotate(case, seed) if case["kind"] == "rotate" else _exact_attend(case, seed)
