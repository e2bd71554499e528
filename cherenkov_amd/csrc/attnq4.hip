// Causal attention over the 4-bit key/value cache (kvq4.h) for the rows of a
// batch of sequences, one to many rows each (what a block does: attnq4_few.h,
// attnq4_many.h; parts joined: attnq4_join.h).
//
// Mathematics.  With a group's value s c + b held as s (c - 8) + (b + 8 s), Q_g
// the sum of the query over group g and P the softmax's numerators,
//   score_t = sum_g s_tg (sum_{d in g} q_d (c - 8)_td) + (b + 8 s)_tg Q_g
//   out_d   = sum_t (P_t s_tg) (c - 8)_td + sum_t P_t (b + 8 s)_tg   (g that of d)
// so both products run on the codes themselves, which f16 holds exactly, and
// the cache's values are never formed; counted from 8, neither product is a
// difference of large sums.  q and P s are the other operands: in two f16
// parts (22 bits), but for q of 16-bit rows, which one holds, and for bf16 rows
// of many pairs (attnq4.h, Q4Form).  P s of a row's largest token and group is
// 2^7 to 2^15 in f16, whose least is 2^-24: what is 2^-32 of it and less is lost,
// and a group 2^10 quieter than the loudest begins to lose bits.  The softmax runs
// in one pass with a running reference, its maximum and sum in f32, as every
// sum.
//
// k_attn_q4 takes sequences with up to 64 (row, head) pairs a kv head: single
// tokens, drafts to verify.  A workgroup takes 16 flattened pairs and a part of
// the tokens, its four waves every fourth step of 64 tokens (of 128 dims) or 32
// (of 256).  v_mfma_f32_16x16x32_f16 takes keys as its A operand (a lane: one
// token's 8 codes of one word) and queries as B, so a lane ends with the scores
// of ONE row for 4 tokens a subtile, and those are, in place, its part of the A
// operand of the second product: nothing crosses lanes between the two.  The
// token order inside a subtile (token 4 (m % 4) + m / 4 in row m) makes the
// values' loads whole: four tokens, 256 or 512 bytes, an instruction.  A step's
// loads are in flight through the step before it.
//
// What bounds it, as measured.  Long contexts of several sequences: memory (8
// f16 rows of 24 x 256 over 600 MB of cache: 134 us, 4.5 TB/s).  64 ragged bf16
// sequences of 32 x 128, four pairs each: 79 us, 3.9 TB/s, memory and the vector
// unit alike (the call 93 us, 109 with the columns' 16 rows of scores, not
// folded).  One token over a short context: latency (12 us: launch and cut 3,
// first loads 2.5, a step 2.9, the waves' join 2).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <type_traits>
#include <vector>

#include "attnq4_few.h"
#include "attnq4_join.h"
#include "kvq4_host.h"

namespace chk {

template <int HD, class T>
__global__ void __launch_bounds__(256, 2) k_attn_q4(AttnQ4Args a) {
    __shared__ FewLds<HD, Q4_ALL> sm;
    const Planner<Q4_ALL> plan(a, threadIdx.x & 63);
    Item it;
    uint32_t none;
    if (plan.find<Q4_FEW>(blockIdx.x, it, none)) few_block<HD, T, Q4_ALL>(a, it, false, sm);
}

// Workgroups that the work is cut for: two a compute unit.
static uint32_t cut_groups() { return 2 * kv4_cus(); }

static void check_heads(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t n) {
    kv4_ensure(hd == 128 || hd == 256, "head_dim must be 128 or 256");
    kv4_ensure(nkv >= 1 && nkv <= 1024 && nh >= nkv && nh % nkv == 0 && nh <= 4096,
               "nh must be a multiple of nkv, at most 4096");
    kv4_ensure(n <= KV4_MAX_SEQS, "at most 1024 sequences a call");
}

// A call's shape, as its launches and its workspace depend on it.
struct AttnQ4Shape {
    uint32_t group, nkv, hd, n, rows, groups;  // groups: workgroups that the work is cut for
    uint32_t shared;                           // groups of shared prefixes
    bool prefix;
};

// Partial rows of a call: numerators, then (maximum, sum) pairs.  The widest
// blocks of any type, so that one workspace serves all.  With shared prefixes the
// plan's walks and sums follow.
static uint64_t partial_rows(const AttnQ4Shape& s) {
    const uint32_t block = attn_q4_block(s.hd, CHK_BF16);
    return s.prefix ? kv4_prefix_partial_rows(s.rows, s.group, s.nkv, s.n, s.groups, block)
                    : kv4_partial_rows(s.rows, s.group, s.groups, block);
}
static uint64_t walks_at(const AttnQ4Shape& s) { return (partial_rows(s) * (s.hd * 4 + 8) + 15) / 16 * 16; }
static uint64_t workspace_bytes(const AttnQ4Shape& s) {
    if (!s.prefix) return partial_rows(s) * (s.hd * 4 + 8);
    return walks_at(s) + ((uint64_t)s.shared + s.n) * (sizeof(Kv4Work) + Q4_KINDS * 4);
}

// What a call launches: all of it from what the host knows, the lengths and row
// starts being the device's.
// tokens: the most that a row's walk may be over; block: pairs of a many-pairs block; least:
// least tiles of a few-pairs part; cap: partial rows of the workspace; whole: no walk is cut.
static AttnQ4Launch attn_launch(const AttnQ4Shape& s, uint64_t tokens, uint32_t block, uint32_t least, uint64_t cap, bool whole) {
    AttnQ4Launch l{};
    const uint64_t flat = (uint64_t)s.rows * s.group, tiles = (tokens + KV4_TILE - 1) / KV4_TILE;
    // A workgroup for every part, as many as there can be: parts < tiles / piece
    // + 1, so one for each block and `groups` more of the sequences with few
    // pairs, 2 groups of those with many (whose cost may be half of their tiles);
    // nor are there more parts than pieces of a full table.  The rest find
    // nothing and end.
    uint64_t few = std::min(flat / KV4_ROWS + s.n, (uint64_t)s.n * (KV4_FEW / KV4_ROWS));
    uint64_t many = flat > KV4_FEW ? flat / block + std::min((uint64_t)s.n, flat / (KV4_FEW + 1)) : 0;
    if (s.shared) {  // and the groups' rows once more
        few += std::min(flat / KV4_ROWS + s.shared, (uint64_t)s.shared * (KV4_FEW / KV4_ROWS));
        if (flat > KV4_SHARED_FEW) many += flat / block + std::min((uint64_t)s.shared, flat / (KV4_SHARED_FEW + 1));
    }
    few *= s.nkv;
    many *= s.nkv;
    l.few = (uint32_t)std::min(few + s.groups, few * std::max<uint64_t>((tiles + least - 1) / least, 1));
    if (many) l.many = (uint32_t)std::min(many + 2 * s.groups, many * std::max<uint64_t>((tiles + 1) / 2, 1));
    // a row with parts has two at least
    l.joins = whole ? 0u : (uint32_t)std::min<uint64_t>(flat * s.nkv, cap / 2 + 1);
    // rows that give the device fewer waves than it has are read by a team of
    // lanes a part; else a wave takes one row, or as many as leave the device 8
    // waves a SIMD (16384 rows of two parts: 23.7 us with one, 19.9 with two)
    l.split = l.joins <= 2 * s.groups;
    l.run = l.split ? 1u : (l.joins + 16 * s.groups - 1) / (16 * s.groups);
    return l;
}

// What the host knows of the walks through a window: the most tokens of one, in whole
// tiles, and the least tiles of a part.  Where no walk is over more than two steps of four
// waves (of many pairs: the tiles of one), none is cut and there is nothing to join: a launch
// less for a step more (one f32 row of 16 x 256 through 2 tokens and 4 first ones 10.9 us for
// 14.6, 64 bf16 rows of 32 x 128 through 15 and 4 11.0 for 13.6).
struct WindowBounds {
    uint64_t tokens;
    uint32_t least;
    bool whole;
};
static WindowBounds window_bounds(uint64_t tokens, uint64_t rows, uint32_t group, Kv4Window v, const Kv4Blocks& shapes, uint32_t least) {
    // (a sequence of one row; one with enough of them for blocks of many pairs)
    const uint32_t one = kv4_window_span((uint32_t)tokens, 1, group, v, shapes).tiles;
    const uint32_t lots = kv4_window_span((uint32_t)tokens, KV4_FEW / group + 1, group, v, shapes).tiles;
    const bool many = rows * group > KV4_FEW, whole = many ? lots <= least && one <= 2 * least : one <= 2 * least;
    return WindowBounds{(uint64_t)std::max(one, many ? lots : 0u) * KV4_TILE, whole ? 2 * least : least, whole};
}

// A call's q, out and workspace.
struct AttnQ4Rows {
    const void* q;
    uint32_t nh, gated, dtype;
    uint64_t q_stride;
    void* out;
    uint64_t out_stride;
    void* ws;
    uint64_t ws_bytes;
};

template <int V>
static void attn_call(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const AttnQ4Rows& r, const ChkKvMask* mask, uint32_t window,
                      uint32_t sinks, const ChkKvShared* shared, void* stream) {
    const char* small = V == Q4_PREFIX ? "workspace smaller than chk_attn_prefix_q4_workspace says"
                                       : "workspace smaller than chk_attn_q4_workspace says";
    AttnQ4Args a{};
    a.c = kv4_cache(cache);
    a.s = kv4_seqs(cache, seqs);
    kv4_dtype(r.dtype);
    check_heads(r.nh, cache->nkv, cache->hd, a.s.n);
    if (V == Q4_WINDOW) kv4_ensure(window >= 1, "a window has at least one token");
    if (V == Q4_PREFIX) {
        kv4_ensure(shared, "no shared prefixes given");
        kv4_ensure(shared->groups <= KV4_MAX_SEQS, "at most 1024 groups a call");
    }
    if (a.s.rows == 0) return;
    kv4_rows_arg(r.q, r.q_stride, (uint64_t)r.nh * cache->hd * (r.gated ? 2 : 1), r.dtype, "q");
    kv4_rows_arg(r.out, r.out_stride, (uint64_t)r.nh * cache->hd, r.dtype, "out");
    kv4_ensure(r.ws && kv4_aligned(r.ws, 16), "null or misaligned workspace");
    kv4_ensure((uint64_t)a.s.rows * r.nh <= 1u << 28, "at most 2^28 rows x heads a call");
    if (mask) {
        kv4_ensure(mask->bits && kv4_aligned(mask->bits, 4), "null or misaligned mask");
        kv4_ensure(mask->ratio >= 1 && mask->words >= 1, "ratio and words must be positive");
        a.mask = mask->bits;
        a.words = mask->words;
        a.ratio = mask->ratio;
        a.kblk = mask->kblk;
    }
    if (V == Q4_PREFIX && shared->groups)
        kv4_ensure(shared->first && shared->tokens && kv4_aligned(shared->first, 4) && kv4_aligned(shared->tokens, 4),
                   "null or misaligned first or tokens");
    kv4_ensure(r.ws_bytes >= 16, small);
    const hipStream_t st = (hipStream_t)stream;
    const bool groups = V == Q4_PREFIX && shared->groups;
    kv4_on_device({cache->k, cache->v, cache->ks, cache->vs, seqs->table, seqs->len, seqs->start, r.q, r.out, r.ws,
                   mask ? mask->bits : r.q, groups ? shared->first : r.q, groups ? shared->tokens : r.q}, st);
    a.groups = cut_groups();
    a.block = attn_q4_block(cache->hd, r.dtype);
    a.least = KV4_WAVES * q4_step(cache->hd) / KV4_TILE;
    a.group = r.nh / cache->nkv;
    const AttnQ4Shape s{a.group, a.c.nkv, cache->hd, a.s.n, a.s.rows, a.groups, groups ? shared->groups : 0u, V == Q4_PREFIX};
    const uint64_t cap = partial_rows(s);
    kv4_ensure(r.ws_bytes >= workspace_bytes(s), small);
    a.q = r.q;
    a.out = r.out;
    a.q_stride = r.q_stride;
    a.out_stride = r.out_stride;
    a.gated = r.gated ? 1u : 0u;
    a.scale = 1.4426950408889634f / sqrtf((float)cache->hd);
    a.cap = (uint32_t)cap;
    a.po = (float*)r.ws;
    a.pml = (float2*)((uint8_t*)r.ws + cap * cache->hd * 4);
    if (V == Q4_PREFIX) {
        a.shared = s.shared;
        a.of_group = groups ? shared->first : nullptr;
        a.of_tokens = groups ? shared->tokens : nullptr;
        a.work = (Kv4Work*)((uint8_t*)r.ws + walks_at(s));
        a.upto = (uint32_t*)(a.work + s.shared + s.n);
    }
    uint64_t tokens = (uint64_t)seqs->table_width * cache->page;
    a.shapes = kv4_block_shapes(a.group, a.block);
    bool whole = false;
    if (V == Q4_WINDOW) {
        a.view = kv4_window(window, sinks);
        const WindowBounds w = window_bounds(tokens, a.s.rows, a.group, a.view, a.shapes, a.least);
        tokens = w.tokens;
        a.least = w.least;
        whole = w.whole;
    }
    const AttnQ4Launch l = attn_launch(s, tokens, a.block, a.least, cap, whole);
    a.run = l.run;
    if (V != Q4_ALL) {
        a.any_many = l.many ? 1u : 0u;
        launch_attn_q4_view(a, V, cache->hd, r.dtype, l, st);
        return;
    }
    if (l.many) launch_attn_q4_many(a, cache->hd, r.dtype, l.many, st);
    kv4_switch(cache->hd, r.dtype, [&](auto hd, auto t) {
        constexpr int H = decltype(hd)::value;
        using E = typename decltype(t)::type;
        kv4_launch(k_attn_q4<H, E>, dim3(l.few), CHK_WG, st, a);
        launch_join<H, E, Q4_ALL>(a, l, st);
    });
}

// ---- host views of a call's cut

static void cut_args(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t dtype, uint32_t groups, uint32_t n, uint32_t rows,
                     uint64_t tokens, const uint32_t* len, const uint32_t* start, const uint32_t* cut, const uint64_t* launch) {
    check_heads(nh, nkv, hd, n);
    kv4_dtype(dtype);
    kv4_ensure(groups >= 1 && groups <= 1u << 16, "1..=65536 workgroups");
    kv4_ensure(launch && (n == 0 || (len && start && cut)), "null pointer");
    kv4_ensure((uint64_t)rows * nh <= 1u << 28, "at most 2^28 rows x heads a call");
    kv4_ensure(tokens <= 1u << 30, "a sequence's table may hold 2^30 tokens");
}
static void launch_sizes(const AttnQ4Shape& s, uint64_t tokens, uint32_t block, uint32_t least, bool whole, uint64_t* launch) {
    const uint64_t cap = partial_rows(s);
    const AttnQ4Launch l = attn_launch(s, tokens, block, least, cap, whole);
    launch[0] = cap;
    launch[1] = l.few;
    launch[2] = l.many;
    launch[3] = l.joins;
}

static void add(Kv4Trial& t, Kv4Trial u) {
    t.few += u.few;
    t.many += u.many;
    t.load += u.load;
    t.cut |= u.cut;
}
// The share of a call with a view: the first of `tries` that fits, else the first.
template <class F>
static Kv4Share best_share(uint64_t cost, uint32_t groups, uint32_t least, uint32_t tries, F&& trial) {
    const uint32_t s = kv4_share_few(cost, groups, least);
    for (uint32_t i = 0; i < tries; ++i) {
        const Kv4Share now = kv4_view_share(s, least, i);
        if (kv4_fits(trial(now), groups, now)) return now;
    }
    return kv4_view_share(s, least, 0);
}

// view: null where rows see everything before them
static void cut_call(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t dtype, uint32_t groups, uint32_t n, uint32_t rows,
                     uint64_t tokens, const uint32_t* len, const uint32_t* start, const Kv4Window* view, uint32_t* cut,
                     uint64_t* launch) {
    cut_args(nh, nkv, hd, dtype, groups, n, rows, tokens, len, start, cut, launch);
    const auto held = [&](uint32_t b) { return len[b] <= tokens ? len[b] : 0u; };  // as the kernels take it
    const uint32_t group = nh / nkv, block = attn_q4_block(hd, dtype);
    const Kv4Blocks shapes = kv4_block_shapes(group, block);
    WindowBounds w{tokens, KV4_WAVES * q4_step(hd) / KV4_TILE, false};
    if (view) w = window_bounds(tokens, rows, group, *view, shapes, w.least);
    const uint32_t least = w.least;
    Kv4Share share;
    uint64_t sum[2] = {0, 0};
    for (uint32_t b = 0; b < n; ++b) {
        uint32_t s0, s1;
        kv4_rows(start, b, rows, s0, s1);
        sum[(s1 - s0) * group > KV4_FEW] +=
            view ? kv4_window_cost(kv4_window_span(held(b), s1 - s0, group, *view, shapes), held(b), s1 - s0, group, shapes)
                 : kv4_cost(held(b), s1 - s0, group, block);
    }
    share.few = kv4_share_few(sum[0] * nkv, groups, least);
    share.many = kv4_share(sum[1] * nkv, groups, 2);
    if (view)
        share = best_share((sum[0] + KV4_MANY_COST * sum[1]) * nkv, groups, least, n <= 64 ? KV4_TRIES : 1, [&](Kv4Share now) {
            Kv4Trial t{0, 0, 0, 0};
            for (uint32_t b = 0; b < n; ++b) {
                uint32_t s0, s1;
                kv4_rows(start, b, rows, s0, s1);
                const Kv4Span w = kv4_window_span(held(b), s1 - s0, group, *view, shapes);
                add(t, kv4_trial(w.many, w.blocks, w.tiles, nkv, now));
            }
            return t;
        });
    for (uint32_t b = 0; b < n; ++b) {
        uint32_t s0, s1;
        kv4_rows(start, b, rows, s0, s1);
        Kv4Cut c = kv4_cut(held(b), s1 - s0, group, block, share);
        if (view && c.flat) c.parts = kv4_parts(kv4_window_span(held(b), s1 - s0, group, *view, shapes).tiles, c.piece);
        cut[4 * b] = c.block;
        cut[4 * b + 1] = c.blocks;
        cut[4 * b + 2] = c.piece;
        cut[4 * b + 3] = c.parts;
    }
    launch_sizes({group, nkv, hd, n, rows, groups, 0, false}, w.tokens, block, least, w.whole, launch);
}

}  // namespace chk

using namespace chk;

extern "C" {

int chk_attn_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated, uint32_t dtype,
                uint64_t q_stride, const ChkKvMask* mask, void* out, uint64_t out_stride, void* ws, uint64_t ws_bytes,
                void* stream) {
    return kv4_try([&] {
        attn_call<Q4_ALL>(cache, seqs, {q, nh, gated, dtype, q_stride, out, out_stride, ws, ws_bytes}, mask, 0, 0, nullptr, stream);
    });
}

int chk_attn_q4_workspace(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t n, uint32_t rows, uint64_t* bytes) {
    return kv4_try([&] {
        kv4_ensure(bytes, "null pointer");
        check_heads(nh, nkv, hd, n);
        *bytes = workspace_bytes({nh / nkv, nkv, hd, n, rows, cut_groups(), 0, false});
    });
}

int chk_attn_window_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated, uint32_t dtype,
                       uint64_t q_stride, uint32_t window, uint32_t sinks, void* out, uint64_t out_stride, void* ws,
                       uint64_t ws_bytes, void* stream) {
    return kv4_try([&] {
        attn_call<Q4_WINDOW>(cache, seqs, {q, nh, gated, dtype, q_stride, out, out_stride, ws, ws_bytes}, nullptr,
                             window, sinks, nullptr, stream);
    });
}

int chk_attn_prefix_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated, uint32_t dtype,
                       uint64_t q_stride, const ChkKvShared* shared, void* out, uint64_t out_stride, void* ws,
                       uint64_t ws_bytes, void* stream) {
    return kv4_try([&] {
        attn_call<Q4_PREFIX>(cache, seqs, {q, nh, gated, dtype, q_stride, out, out_stride, ws, ws_bytes}, nullptr, 0, 0, shared,
                             stream);
    });
}

int chk_attn_prefix_q4_workspace(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t n, uint32_t rows, uint32_t groups,
                                 uint64_t* bytes) {
    return kv4_try([&] {
        kv4_ensure(bytes, "null pointer");
        check_heads(nh, nkv, hd, n);
        kv4_ensure(groups <= KV4_MAX_SEQS, "at most 1024 groups a call");
        *bytes = workspace_bytes({nh / nkv, nkv, hd, n, rows, cut_groups(), groups, true});
    });
}

int chk_attn_q4_cut(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t dtype, uint32_t groups, uint32_t n, uint32_t rows,
                    uint64_t tokens, const uint32_t* len, const uint32_t* start, uint32_t* cut, uint64_t* launch) {
    return kv4_try([&] { cut_call(nh, nkv, hd, dtype, groups, n, rows, tokens, len, start, nullptr, cut, launch); });
}

int chk_attn_window_q4_cut(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t dtype, uint32_t groups, uint32_t n, uint32_t rows,
                           uint64_t tokens, const uint32_t* len, const uint32_t* start, uint32_t window, uint32_t sinks,
                           uint32_t* cut, uint64_t* launch) {
    return kv4_try([&] {
        kv4_ensure(window >= 1, "a window has at least one token");
        cut_args(nh, nkv, hd, dtype, groups, n, rows, tokens, len, start, cut, launch);
        const Kv4Window v = kv4_window(window, sinks);
        cut_call(nh, nkv, hd, dtype, groups, n, rows, tokens, len, start, &v, cut, launch);
    });
}

int chk_attn_prefix_q4_cut(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t dtype, uint32_t groups, uint32_t n, uint32_t rows,
                           uint64_t tokens, const uint32_t* len, const uint32_t* start, const ChkKvShared* shared,
                           uint32_t* walks, uint64_t* launch) {
    return kv4_try([&] {
        cut_args(nh, nkv, hd, dtype, groups, n, rows, tokens, len, start, walks, launch);
        kv4_ensure(shared && shared->groups <= KV4_MAX_SEQS, "at most 1024 groups a call");
        kv4_ensure(shared->groups == 0 || (shared->first && shared->tokens), "null first or tokens");
        const uint32_t group = nh / nkv, block = attn_q4_block(hd, dtype), least = KV4_WAVES * q4_step(hd) / KV4_TILE;
        const Kv4Blocks shapes = kv4_block_shapes(group, block);
        std::vector<Kv4Work> work;
        std::vector<uint32_t> of(n, KV4_NO_GROUP);
        struct Seq {
            uint32_t s0, n, len;
            bool held;
        };
        std::vector<Seq> seqs(n);
        for (uint32_t b = 0; b < n; ++b) {
            uint32_t s0, s1;
            kv4_rows(start, b, rows, s0, s1);
            const bool held = len[b] <= tokens;
            seqs[b] = {s0, s1 - s0, held ? len[b] : 0u, held};
        }
        for (uint32_t g = 0; g < shared->groups; ++g) {
            const uint32_t f0 = std::min(shared->first[g], n), f1 = std::min(std::max(shared->first[g + 1], f0), n);
            Kv4Group r{0u, 0u, 0xffffffffu, 0u, 0xffffffffu, 0u, 0u};
            for (uint32_t b = f0; b < f1; ++b) {
                const Seq& q = seqs[b];
                if (!kv4_member(q.n, q.len, q.held)) continue;
                of[b] = g;
                if (!r.members++) r.lead = b;
                r.s0 = std::min(r.s0, q.s0);
                r.s1 = std::max(r.s1, q.s0 + q.n);
                r.least = std::min(r.least, q.len - q.n + 1);
                r.most = std::max(r.most, q.len);
                r.cost += kv4_blocks_cost(q.n * group, q.n * group > KV4_FEW, shapes);
            }
            work.push_back(kv4_group_work(r, shared->tokens[g], group, shapes, KV4_SHARED_SMALL * groups / nkv));
        }
        for (uint32_t b = 0; b < n; ++b) {
            const Seq& q = seqs[b];
            const uint32_t g = of[b], t = g != KV4_NO_GROUP && work[g].n ? work[g].len : 0u;
            work.push_back(kv4_seq_work(b, q.s0, q.n, q.len, q.held, group, t ? g : KV4_NO_GROUP, t));
        }
        uint64_t cost[2] = {0, 0};
        for (const Kv4Work& k : work) cost[k.many] += kv4_work_cost(k, group, shapes);
        const Kv4Share share = best_share((cost[0] + KV4_MANY_COST * cost[1]) * nkv, groups, least, KV4_TRIES, [&](Kv4Share now) {
            Kv4Trial t{0, 0, 0, 0};
            for (const Kv4Work& k : work)
                add(t, kv4_trial(k.many, kv4_blocks(k.n * group, k.many, shapes), kv4_work_most(k), nkv, now));
            return t;
        });
        uint32_t* to = walks;
        for (Kv4Work& k : work) {
            kv4_work_cut(k, share, false, least);
            const uint32_t w[8] = {k.s0, k.n, k.len, k.lo, k.group, k.many ? block : KV4_ROWS, k.piece, k.parts};
            to = std::copy(w, w + 8, to);
        }
        launch_sizes({group, nkv, hd, n, rows, groups, shared->groups, true}, tokens, block, least, false, launch);
    });
}

}  // extern "C"
