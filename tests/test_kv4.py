"""The 4-bit key/value cache without a GPU: the pair rule and the slot rule
that the kernels share with host code, the plain oracle against its own
definition, and every refusal of the entry points (all made before any device
call)."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from tests import kv4_ref as ref

if not abi.LIB_PATH.exists():
    pytest.skip("libcherenkov.so not built (run __graft_entry__.build())", allow_module_level=True)


def last_error() -> str:
    return abi.lib().chk_last_error().decode()


def pair(group: np.ndarray):
    g = np.ascontiguousarray(group, np.float32)
    s, b = C.c_uint16(), C.c_uint16()
    assert abi.lib().chk_kv_pair_q4(g.ctypes.data, C.byref(s), C.byref(b)) == 0
    return (np.array([s.value << 16, b.value << 16], np.uint32)).view(np.float32)


GROUPS = {
    "normal": lambda r: r.normal(0, 1, 64),
    "offset": lambda r: r.normal(100, 0.1, 64),
    "negative": lambda r: -np.abs(r.normal(3, 1, 64)) - 1,
    "constant": lambda r: np.full(64, 0.3),
    "bf16_constant": lambda r: np.full(64, -1.5),
    "zero": lambda r: np.zeros(64),
    "negative_zero": lambda r: np.full(64, -0.0),
    "tiny": lambda r: r.normal(0, 1e-39, 64),
    "least": lambda r: np.where(np.arange(64) == 5, 1e-45, 0.0),
    "huge": lambda r: r.normal(0, 1e37, 64),
    "one_loud": lambda r: np.where(np.arange(64) == 63, 300.0, r.normal(0, 1, 64)),
}


@pytest.mark.parametrize("name", sorted(GROUPS))
def test_pair_is_the_rule_and_covers_every_value(name):
    for seed in range(20):
        x = GROUPS[name](np.random.default_rng(seed)).astype(np.float32)
        s, b = pair(x)
        c, rs, rb = ref.quantise(x[None])
        assert (s, b) == (rs[0, 0], rb[0, 0])
        assert b <= x.min() and s >= 2.0**-126
        back = ref.stands_for(c, rs, rb)[0]
        # half a step, and what f32(x - b) loses
        assert np.all(np.abs(back - x) <= s / 2 + 2.0**-24 * np.abs(x.astype(np.float64) - b) + 2.0**-149)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_pair_of_a_group_with_no_finite_range_is_nan(bad):
    x = np.linspace(-1, 1, 64).astype(np.float32)
    x[17] = bad
    assert np.isnan(pair(x)).all()
    wide = np.zeros(64, np.float32)
    wide[0], wide[1] = -3.0e38, 3.0e38
    assert np.isnan(pair(wide)).all()


def test_oracle_order_is_a_permutation_and_units_take_groups_in_turn():
    for hd in (128, 256):
        for unit in (16, 4):
            o = ref.order(hd, unit)
            assert sorted(o) == list(range(hd))
            first = o[::unit]
            assert [d // 64 for d in first[: hd // 64]] == list(range(hd // 64))
            assert all(np.array_equal(o[i:i + unit], np.arange(f, f + unit)) for i, f in zip(range(0, hd, unit), first))


def test_oracle_rounds_codes_to_nearest_even():
    x = np.zeros(64, np.float32)
    x[0], x[1], x[2], x[3] = 15.0, 0.5, 1.5, 2.5  # s = 1, b = 0
    c, s, b = ref.quantise(x[None])
    assert s[0, 0] == 1.0 and b[0, 0] == 0.0
    assert c[0, :4].tolist() == [15, 0, 2, 2]


def cache_struct(pages=4, page=16, nkv=2, hd=128, ptr=4096):
    return abi.ChkKvQ4(ptr, ptr, ptr, ptr, pages, page, nkv, hd)


def test_slot_of_a_token():
    L = abi.lib()
    c = cache_struct(pages=7, page=32)
    table = np.array([3, 0, 6, 7, 0xFFFFFFFF], np.uint32)
    slot = C.c_uint64()
    for t in range(96):
        assert L.chk_kv_slot_q4(C.byref(c), table.ctypes.data, 5, t, C.byref(slot)) == 0
        assert slot.value == int(table[t // 32]) * 32 + t % 32
    # page 7 and page 2^32 - 1 are not the cache's; entry 5 is past the table
    for t in (96, 127, 128, 159, 160, 2**32 - 1):
        assert L.chk_kv_slot_q4(C.byref(c), table.ctypes.data, 5, t, C.byref(slot)) == -1
        assert "no page of the cache holds this token" in last_error()
    big = cache_struct(pages=2**31, page=2**20)
    far = np.array([2**31 - 1], np.uint32)
    assert L.chk_kv_slot_q4(C.byref(big), far.ctypes.data, 1, 2**20 - 1, C.byref(slot)) == 0
    assert slot.value == 2**51 - 1


def seqs_struct(n=2, width=3, rows=5, ptr=4096):
    return abi.ChkKvSeqs(ptr, ptr, ptr, n, width, rows)


CACHE_BAD = [
    (dict(hd=64), "head_dim must be 128 or 256"),
    (dict(hd=192), "head_dim must be 128 or 256"),
    (dict(nkv=0), "kv heads"),
    (dict(nkv=1025), "kv heads"),
    (dict(page=8), "page must be a power of two"),
    (dict(page=48), "page must be a power of two"),
    (dict(page=0), "page must be a power of two"),
    (dict(page=1 << 21), "page must be a power of two"),
    (dict(pages=0), "at least one page"),
    (dict(ptr=0), "null cache plane"),
    (dict(ptr=4104), "16-byte aligned"),
]
SEQS_BAD = [
    (dict(n=1025), "at most 1024 sequences"),
    (dict(n=0), "rows without a sequence"),
    (dict(width=0), "at least one page"),
    (dict(width=(1 << 26) + 1), "2^30 tokens"),
    (dict(ptr=0), "null table, len or start"),
    (dict(ptr=4098), "4-byte aligned"),
]


def rows_call(which, c, s, p=8192, dtype=0, stride=256):
    fn = getattr(abi.lib(), which)
    return fn(c and C.byref(c), s and C.byref(s), p, p, dtype, stride, stride, None)


def attn_call(c, s, q=8192, nh=4, gated=0, dtype=0, q_stride=512, mask=None, out=1 << 20, out_stride=512, ws=4096,
              ws_bytes=1 << 40):
    return abi.lib().chk_attn_q4(c and C.byref(c), s and C.byref(s), q, nh, gated, dtype, q_stride, mask, out, out_stride,
                                 ws, ws_bytes, None)


@pytest.mark.parametrize("which", ["chk_kv_append_q4", "chk_kv_read_q4", "chk_attn_q4"])
def test_bad_caches_and_sequences_are_refused(which):
    call = attn_call if which == "chk_attn_q4" else lambda c, s: rows_call(which, c, s)
    for kw, msg in CACHE_BAD:
        assert call(cache_struct(**kw), seqs_struct()) == -1
        assert msg in last_error(), (kw, last_error())
    for kw, msg in SEQS_BAD:
        assert call(cache_struct(), seqs_struct(**kw)) == -1
        assert msg in last_error(), (kw, last_error())
    assert call(None, seqs_struct()) == -1 and "no cache" in last_error()
    assert call(cache_struct(), None) == -1 and "no sequences" in last_error()


@pytest.mark.parametrize("which", ["chk_kv_append_q4", "chk_kv_read_q4"])
def test_bad_rows_are_refused(which):
    c, s = cache_struct(), seqs_struct()
    for kw, msg in [(dict(dtype=3), "dtype"), (dict(p=None), "null k"), (dict(p=8200), "k rows must be 16-byte aligned"),
                    (dict(stride=255), "16-byte aligned"), (dict(stride=252), "stride shorter"),
                    (dict(dtype=1, stride=260), "16-byte aligned"), (dict(stride=1 << 41), "stride")]:
        assert rows_call(which, c, s, **kw) == -1
        assert msg in last_error(), (kw, last_error())
    assert rows_call(which, c, seqs_struct(rows=2**27)) == -1 and "2^27" in last_error()


def test_bad_attention_arguments_are_refused():
    c, s = cache_struct(), seqs_struct()
    mask = lambda **kw: C.byref(abi.ChkKvMask(**dict(dict(bits=4096, words=4, ratio=4, kblk=1), **kw)))  # noqa: E731
    for kw, msg in [(dict(dtype=9), "dtype"), (dict(nh=3), "multiple of nkv"), (dict(nh=0), "multiple of nkv"),
                    (dict(nh=4098), "at most 4096"), (dict(q=None), "null q"), (dict(q=8196), "q rows"),
                    (dict(q_stride=508), "stride shorter"), (dict(gated=1), "q row stride shorter"),
                    (dict(out=None), "null out"), (dict(out_stride=508), "out row stride"), (dict(out=8194), "out rows"),
                    (dict(ws=None), "workspace"), (dict(ws=4100), "workspace"), (dict(ws_bytes=0), "workspace smaller"),
                    (dict(mask=mask(bits=None)), "mask"), (dict(mask=mask(bits=4098)), "mask"),
                    (dict(mask=mask(ratio=0)), "ratio"), (dict(mask=mask(words=0)), "words")]:
        assert attn_call(c, s, **kw) == -1
        assert msg in last_error(), (kw, last_error())
    n = C.c_uint64()
    for args, msg in [((4, 2, 64, 1, 1), "head_dim"), ((5, 2, 128, 1, 1), "multiple"), ((4, 0, 128, 1, 1), "multiple"),
                      ((4, 2, 128, 1025, 1), "1024 sequences")]:
        assert abi.lib().chk_attn_q4_workspace(*args, C.byref(n)) == -1
        assert msg in last_error()
    assert abi.lib().chk_attn_q4_workspace(4, 2, 128, 1, 1, None) == -1


def test_calls_without_rows_do_nothing():
    c, s = cache_struct(), seqs_struct(n=0, width=0, rows=0, ptr=0)
    for which in ("chk_kv_append_q4", "chk_kv_read_q4"):
        assert rows_call(which, c, s) == 0
    assert attn_call(c, s) == 0


def test_memory_that_is_not_the_devices_is_refused():
    """Host memory (or any address, without a device) never reaches a kernel."""
    buf = np.zeros(1 << 16, np.uint8)
    at = (buf.ctypes.data + 255) & ~255
    assert rows_call("chk_kv_append_q4", cache_struct(ptr=at), seqs_struct(ptr=at), p=at) == -1
    assert "device" in last_error()
    assert attn_call(cache_struct(ptr=at), seqs_struct(ptr=at), q=at, out=at, ws=at) == -1
    assert "device" in last_error()


def test_oracle_attention_of_one_token_and_of_none():
    rng = np.random.default_rng(0)
    c = ref.Cache(2, 16, 1, 128)
    table = np.array([[1]], np.uint32)
    k, v = rng.normal(size=(2, 1, 1, 128)).astype(np.float32)
    c.write(table[0], 0, "k", k[0])
    c.write(table[0], 0, "v", v[0])
    q = rng.normal(size=(2, 2, 128)).astype(np.float32)
    # two rows, one token: the first row sits before position 0
    out, _, _ = ref.attend(c, table, [1], [0, 2], q, 2, False)
    assert np.all(out[0] == 0)
    assert np.allclose(out[1], c.read(table[0], 0, "v")[0], atol=0)


# ---- the cut of attention's work: the rule that every workgroup follows

TILE = 64


def cut_of(nh, nkv, hd, dtype, groups, lens, start, rows, tokens):
    n = len(lens)
    cut = np.zeros((max(n, 1), 4), np.uint32)
    launch = np.zeros(4, np.uint64)
    lens, start = np.asarray(lens, np.uint32), np.asarray(start, np.uint32)
    assert abi.lib().chk_attn_q4_cut(nh, nkv, hd, dtype, groups, n, rows, tokens, lens.ctypes.data, start.ctypes.data,
                                     cut.ctypes.data, launch.ctypes.data) == 0, last_error()
    return cut[:n].astype(np.int64), launch.astype(np.int64)


def batch_of(rng):
    """Lengths and rows as they come: single tokens, a few, prompts, mixed."""
    n = int(rng.choice([1, 2, 7, 64, 65, 300, 1024]))
    most = int(rng.choice([1, 70, 1000, 40000]))
    kind = rng.integers(4)
    lens = rng.integers(0, most + 1, n)
    rows = {0: np.ones(n, int), 1: rng.integers(0, 5, n), 2: lens.copy(), 3: rng.integers(0, 400, n)}[int(kind)]
    return lens, np.minimum(rows, lens + rng.integers(0, 2, n))


@pytest.mark.parametrize("groups", [1, 16, 512])
@pytest.mark.parametrize("shape", [(16, 2, 256, 0), (32, 8, 128, 2), (1, 1, 128, 1), (40, 1, 256, 2), (130, 1, 128, 2)])
def test_the_cut_covers_every_tile_and_fits_its_launches(groups, shape):
    """A block's parts cover its tiles, no more of them are made than workgroups
    launched, and no more partial rows than the workspace holds."""
    nh, nkv, hd, dtype = shape
    group = nh // nkv
    for seed in range(40):
        rng = np.random.default_rng(seed)
        lens, rows = batch_of(rng)
        start = np.concatenate([[0], np.cumsum(rows)])
        total = int(start[-1])
        if total == 0 or total * nh > 2**28:
            continue
        cut, (cap, few, many, joins) = cut_of(nh, nkv, hd, dtype, groups, lens, start, total, int(max(lens.max(), 1)))
        used, items, joined = 0, [0, 0], 0
        for length, n, (block, blocks, piece, parts) in zip(lens, rows, cut):
            flat = int(n) * group
            assert blocks * block >= flat > (blocks - 1) * block or flat == blocks == 0
            if flat == 0:
                continue
            for m1 in (min(block, flat) - 1, max((blocks - 1) * block, 1) - 1, flat - 1):  # last pairs of some blocks
                seen = int(length) - int(n) + m1 // group + 1
                tiles = -(-max(seen, 0) // TILE)
                own = max(-(-tiles // piece), 1)
                per = -(-tiles // own)
                assert own <= parts and own * per >= tiles
            assert own == parts  # of the last block
            items[int(flat > 64)] += blocks * nkv * int(parts)
            if parts > 1:
                used += flat * nkv * int(parts)
                joined += flat * nkv
        assert used <= cap and joined <= joins
        assert items[0] <= few and items[1] <= many, (seed, items, few, many)


def test_a_cut_without_sequences_and_its_refusals():
    cut, launch = cut_of(4, 2, 128, 0, 512, [], [0], 0, 64)
    assert len(cut) == 0 and launch[1] == 0 and launch[2] == 0
    z = np.zeros(8, np.uint64)
    p = z.ctypes.data
    for args, msg in [((4, 3, 128, 0, 512, 1, 1, 1, p, p, p, p), "multiple"), ((4, 2, 96, 0, 512, 1, 1, 1, p, p, p, p), "head_dim"),
                      ((4, 2, 128, 5, 512, 1, 1, 1, p, p, p, p), "dtype"), ((4, 2, 128, 0, 0, 1, 1, 1, p, p, p, p), "workgroups"),
                      ((4, 2, 128, 0, 512, 1, 1, 1, None, p, p, p), "null"), ((4, 2, 128, 0, 512, 1, 1, 1, p, p, p, None), "null")]:
        assert abi.lib().chk_attn_q4_cut(*args) == -1
        assert msg in last_error()
    for args, msg in [((4, 2, 128, 0, 512, 1, 2**27, 1, p, p, p, p), "2^28"), ((4, 2, 128, 0, 512, 1, 1, 2**31, p, p, p, p), "2^30")]:
        assert abi.lib().chk_attn_q4_cut(*args) == -1
        assert msg in last_error()


def test_a_length_past_the_table_is_cut_as_none():
    a, _ = cut_of(4, 2, 128, 0, 512, [5000, 900], [0, 1, 2], 2, 1024)
    b, _ = cut_of(4, 2, 128, 0, 512, [0, 900], [0, 1, 2], 2, 1024)
    assert np.array_equal(a, b)


# ---- what the GPU tests' error limit lets pass


def plain_attention(rng, kind, fault, rows=16, n=400, hd=128):
    """(got, want, smax): attention of one head, `got` as a kernel with `fault`
    gives it and rounded to `kind`, `want` in 64 bits."""
    k, v, q = (rng.normal(0, 1, s) for s in ((n, hd), (n, hd), (rows, hd)))
    q = ref.rounded_to(q, kind)
    kd = ref.stands_for(*ref.quantise(k))
    vd = ref.stands_for(*ref.quantise(v))
    half = lambda x: x.astype(np.float16).astype(np.float64)  # noqa: E731

    def attend(q, parts):
        sc = q @ kd.T * hd**-0.5
        p = np.exp(sc - sc.max(1, keepdims=True)) * 2.0**10
        hi = half(p)
        return (hi + (half(p - hi) if parts == 2 else 0)) @ vd / p.sum(1, keepdims=True)

    want = attend(q, 2)
    got = attend(half(q) if fault == "query" else q, 1 if fault == "numerators" else 2)
    if fault == "zeros":
        got = np.zeros_like(got)
    smax = (np.abs(q) @ np.abs(kd).T).max(1) * hd**-0.5
    return ref.rounded_to(got, kind), want, smax


@pytest.mark.parametrize("kind,fault,passes", [
    *((kind, None, True) for kind in ("f32", "f16", "bf16")), *((kind, "zeros", False) for kind in ("f32", "f16", "bf16")),
    *((kind, "numerators", False) for kind in ("f32", "f16", "bf16")), ("f32", "query", False)])
def test_the_error_limit_tells_lost_bits(kind, fault, passes):
    for seed in range(5):
        got, want, smax = plain_attention(np.random.default_rng(seed), kind, fault)
        off = ref.beyond_rounding(kind, got, want)
        assert (off <= ref.beyond_limit(kind, smax)) == passes, (seed, off, ref.beyond_limit(kind, smax))
    if fault == "numerators":  # what it is for
        assert off <= ref.beyond_limit(kind, smax, 1)


@pytest.mark.parametrize("bits", [0x7FC00000, 0xFFC00000, 0x7FFFFFFF, 0xFFFFFFFF, 0xFFFFE000, 0xFFFF0001, 0x7F800001, 0xFF800001])
@pytest.mark.parametrize("where", [0, 31, 63])
def test_pair_of_a_group_with_any_nan_is_nan(bits, where):
    """Whatever bits a NaN has: rounding them as a number's would carry into the
    sign of some."""
    x = np.linspace(-1, 1, 64).astype(np.float32)
    x.view(np.uint32)[where] = bits
    assert np.isnan(pair(x)).all()
    assert np.isnan(pair(x.view(np.uint32)[where:where + 1].repeat(64).view(np.float32))).all()


def test_calls_without_rows_take_null_rows():
    """An empty tensor has no address: a batch without rows passes none."""
    c, s = cache_struct(), seqs_struct(rows=0)
    for which in ("chk_kv_append_q4", "chk_kv_read_q4"):
        assert rows_call(which, c, s, p=None) == 0, last_error()
        assert rows_call(which, c, s, p=None, dtype=3) == -1 and "dtype" in last_error()
    assert attn_call(c, s, q=None, out=None, ws=None, ws_bytes=0) == 0, last_error()
    assert attn_call(c, s, q=None, out=None, ws=None, ws_bytes=0, nh=3) == -1 and "multiple of nkv" in last_error()


def test_more_rows_than_a_launch_holds_are_refused():
    """A launch is under 2^32 threads: 64 of them a row of 256 f32 dims."""
    c = cache_struct(nkv=1)
    for which in ("chk_kv_append_q4", "chk_kv_read_q4"):
        assert rows_call(which, c, seqs_struct(rows=2**25 + 1)) == -1
        assert "2^25" in last_error()
        assert rows_call(which, c, seqs_struct(rows=2**25)) == -1  # host memory
        assert "device" in last_error()
