// The 4-bit key/value cache: where a token's row sits and what it holds.
// Shared by the kernels and by host code (the checks of the entry points and
// the host-side views of the same rules).
//
// A group is 64 consecutive dims of one (token, kv head).  With lo and hi its
// least and largest value, it is held as
//   b = lo rounded down to bf16,
//   s = fl(fl(hi - b) / 15) rounded up to bf16, at least 2^-126,
//   c = the integer nearest to fl(x - b) / s (ties to even), in 0..15,
// and stands for s c + b.  Rounding b down and s up puts every value inside
// [b, b + 15 s], so nothing is cut off and |x - (s c + b)| <= s / 2 up to the
// rounding of x - b.  bf16 for s and b as in the 4-bit weights: 4.5 bits a
// value, and no magnitude of f32 is out of reach.  A group with a NaN or an
// infinity, or whose spread or ends pass the largest bf16, gets s = b = NaN.
//
// A row of hd dims is hd / 2 bytes of codes, the lower nibble first, in units
// that take the row's hd / 64 groups in turn, so that a lane of the attention
// kernel finds its part of every group in one piece:
//   keys    units of 16 dims (8 bytes): unit u holds dims 64 (u % ng) + 16 (u / ng) + 0..15
//   values  units of 4 dims (2 bytes):  unit u holds dims 64 (u % ng) + 4 (u / ng) + 0..3
// and hd / 64 words s | b << 16.  Planes: codes [pages][nkv][page][hd / 2]
// bytes, words [pages][nkv][page][hd / 64]; a head's tokens lie together
// within a page, so a tile of tokens is one piece of memory and no line of it
// is shared with another head.
#pragma once

#include <stdint.h>

#include "cherenkov/kernels.h"
#include "cherenkov/synth.h"

namespace chk {

constexpr uint32_t KV4_MAX_SEQS = 1024;
constexpr uint32_t KV4_NO_PAGE = 0xffffffffu;
constexpr uint32_t KV4_NAN_PAIR = 0x7fc07fc0u;  // s = b = NaN

struct Kv4Cache {
    uint8_t *k, *v;
    uint32_t *ks, *vs;
    uint32_t pages, page_log2, nkv;
};

struct Kv4Seqs {
    const uint32_t *table, *len, *start;
    uint32_t n, width, rows;
};

// The page that holds token t of a sequence, KV4_NO_PAGE where the table ends
// before it or names a page that the cache has not.
static inline CHK_HD uint32_t kv4_page(const uint32_t* table_row, uint32_t width, uint32_t page_log2, uint32_t pages, uint32_t t) {
    const uint32_t e = t >> page_log2;
    if (e >= width) return KV4_NO_PAGE;
    const uint32_t id = table_row[e];
    return id < pages ? id : KV4_NO_PAGE;
}

// Row index of (page id, head, token) in units of one row of a plane.
static inline CHK_HD uint64_t kv4_row(uint32_t id, uint32_t nkv, uint32_t page_log2, uint32_t head, uint32_t t) {
    const uint32_t page = 1u << page_log2;
    return (((uint64_t)id * nkv + head) << page_log2) + (t & (page - 1));
}

// The rows [s0, s1) of the call that belong to sequence b: start[b] to
// start[b + 1], kept inside the call's rows.
static inline CHK_HD void kv4_rows(const uint32_t* start, uint32_t b, uint32_t rows, uint32_t& s0, uint32_t& s1) {
    const uint32_t x = start[b], y = start[b + 1];
    s0 = x < rows ? x : rows;
    s1 = y < s0 ? s0 : y < rows ? y : rows;
}

// The sequence of row r: the last b with start[b] <= r, if r < start[b + 1];
// n where the row belongs to none.
static inline CHK_HD uint32_t kv4_seq_of(const uint32_t* start, uint32_t n, uint32_t r) {
    uint32_t lo = 0, hi = n;  // start[lo - 1] <= r < start[hi] (virtually)
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (start[mid] <= r) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0) return n;
    const uint32_t b = lo - 1;
    return r < start[b + 1] ? b : n;
}

// A group's (s, b) from its least and largest value, as f32 bit patterns with
// 16 significant bits; NaN twice where the group holds no such pair.
static inline CHK_HD uint32_t kv4_bits(float x) {
    union {
        float f;
        uint32_t u;
    } c;
    c.f = x;
    return c.u;
}
static inline CHK_HD float kv4_float(uint32_t u) {
    union {
        uint32_t u;
        float f;
    } c;
    c.u = u;
    return c.f;
}
static inline CHK_HD void kv4_pair(float lo, float hi, float& s, float& b) {
    const uint32_t l = kv4_bits(lo);
    uint32_t bb = l & 0xffff0000u;
    if ((l >> 31) && bb != l) bb += 0x10000u;  // down: away from zero below it
    b = kv4_float(bb);
    const uint32_t q = kv4_bits((hi - b) / 15.0f);
    uint32_t sb = q & 0xffff0000u;
    if (sb != q) sb += 0x10000u;  // up (hi >= b)
    if (sb < 0x00800000u) sb = 0x00800000u;
    s = kv4_float(sb);
    // exponent field of ones: infinity or NaN (q before its rounding, which
    // carries a NaN of many ones into the sign)
    const uint32_t inf = 0x7f800000u;
    if ((bb & inf) == inf || (q & inf) == inf || (sb & inf) == inf) s = b = kv4_float(0x7fc00000u);
}

// ---- how attention's work is cut (the same on the host and in every
// workgroup, from the lengths and row starts alone)
//
// A sequence's n rows are n G flattened (row, query head) pairs of each kv
// head, G = nh / nkv, and its tokens come in tiles of 64.
//   few pairs (up to 64): blocks of 16, a workgroup each, whose four waves share
//       out the tiles;
//   many: blocks of `block` (64 or 128), a workgroup each, whose waves take the
//       rows and share the tiles.
// A block's tiles are cut into parts until the batch's blocks fill the device
// with equal shares, no more; a block that sees less than the last one of its
// sequence has fewer parts.
constexpr uint32_t KV4_TILE = 64;
constexpr uint32_t KV4_ROWS = 16;   // of a few-pairs block
constexpr uint32_t KV4_WAVES = 4;   // of a workgroup
constexpr uint32_t KV4_FEW = 64;    // most pairs of a few-pairs sequence

// Tiles of a workgroup's part, for sequences with few pairs and with many.
struct Kv4Share {
    uint32_t few, many;
};

struct Kv4Cut {
    uint32_t flat;    // (row, head) pairs of one kv head
    uint32_t many;
    uint32_t block;   // pairs of a block
    uint32_t blocks;
    uint32_t piece;   // most tiles of a part
    uint32_t parts;   // of the last block, which has most
};

static inline CHK_HD uint32_t kv4_block(uint32_t flat, uint32_t block) { return flat <= KV4_FEW ? KV4_ROWS : block; }

// Tokens that the pairs up to m see: n rows of `group` pairs each, len tokens.
static inline CHK_HD int32_t kv4_seen(uint32_t len, uint32_t n, uint32_t group, uint32_t m) {
    return (int32_t)len - (int32_t)n + (int32_t)(m / group) + 1;
}
static inline CHK_HD uint32_t kv4_tiles(int32_t seen) { return seen > 0 ? ((uint32_t)seen + KV4_TILE - 1) / KV4_TILE : 0u; }
static inline CHK_HD uint32_t kv4_parts(uint32_t tiles, uint32_t piece) { return tiles <= piece ? 1u : (tiles + piece - 1) / piece; }

// The tiles of a sequence's blocks, of one kv head: their number times the mean
// of the first and the last one's (rounded up: at least half the last one's).
static inline CHK_HD uint64_t kv4_cost(uint32_t len, uint32_t n, uint32_t group, uint32_t block) {
    const uint32_t flat = n * group, r = kv4_block(flat, block);
    if (flat == 0) return 0;
    const uint32_t first = kv4_tiles(kv4_seen(len, n, group, (flat < r ? flat : r) - 1)), last = kv4_tiles((int32_t)len);
    return (uint64_t)((flat + r - 1) / r) * ((first + last + 1) / 2);
}

// Tiles of a part.  `tiles`: that sum over the sequences of a kind and the kv
// heads; `groups`: workgroups at once, two a compute unit; `least`: tiles that
// give every wave of a workgroup work.
static inline CHK_HD uint32_t kv4_share(uint64_t tiles, uint32_t groups, uint32_t least) {
    const uint64_t t = tiles + groups - 1, s = t >> 32 ? t / groups : (uint32_t)t / groups;
    return s < least ? least : s > 0x3fffffffu ? 0x3fffffffu : (uint32_t)s;
}
// Few pairs: up to two steps a wave (2 least tiles), one workgroup a compute
// unit takes as long as two with half the work, and leaves half the parts to
// join (32000 tokens of 2 heads: 28 us with 500 parts, 25 with 250).
static inline CHK_HD uint32_t kv4_share_few(uint64_t tiles, uint32_t groups, uint32_t least) {
    const uint32_t one = kv4_share(2 * tiles, groups, least);
    return one <= 2 * least ? one : kv4_share(tiles, groups, 2 * least);
}

static inline CHK_HD Kv4Cut kv4_cut(uint32_t len, uint32_t n, uint32_t group, uint32_t block, Kv4Share share) {
    Kv4Cut c;
    c.flat = n * group;
    c.many = c.flat > KV4_FEW;
    c.block = kv4_block(c.flat, block);
    c.blocks = (c.flat + c.block - 1) / c.block;
    c.piece = c.many ? share.many : share.few;
    c.parts = c.flat ? kv4_parts(kv4_tiles((int32_t)len), c.piece) : 1u;
    return c;
}

// ---- views: rows that see a part of what is before them
//
// A block's walk is over two runs of tiles, [0, head) and [head + gap, end): the
// first tokens and the window's of any of its rows, or a sequence's tokens
// behind a shared prefix (head 0).  The walk is counted as if the gap were not
// there; the block's parts are shares of it.

// With views, blocks of few and of many pairs are one launch, so one share of the
// device gives the parts of both: in tiles of a few-pairs block, of which a tile of many
// pairs takes two (64 f16 pairs of 256 dims 2.2 us a compute unit, 16 of them 1.05).
// A share that leaves a few workgroups more than the device takes at once costs
// them a round of their own, so somewhat larger ones are tried (64 bf16 rows of 32 x 128
// behind 8192 tokens 51 us for 56; 64 through windows of 1000 level).
constexpr uint32_t KV4_TRIES = 4;
constexpr uint32_t KV4_START = 4;  // what a workgroup takes beside its tiles, in tiles: some 5 us
constexpr uint32_t KV4_MANY_COST = 2;

static inline CHK_HD Kv4Share kv4_view_share(uint32_t share, uint32_t least, uint32_t tried) {
    const uint32_t s = share + share * tried / 12;
    Kv4Share r;
    r.few = (s + least - 1) & ~(least - 1);  // (steps that all four waves have; least is a power of two)
    r.many = (s + 1) / 2 < 2 ? 2 : (s + 1) / 2;
    return r;
}
// What a walk is of a trial: workgroups, the tiles and starts of those of few pairs,
// and whether it is cut; bounded so that sums stay in 32 bits.
struct Kv4Trial {
    uint32_t few, many, load, cut;
};
static inline CHK_HD uint32_t kv4_bounded(uint64_t v) { return v < 1u << 20 ? (uint32_t)v : 1u << 20; }
static inline CHK_HD Kv4Trial kv4_trial(uint32_t many, uint32_t blocks, uint32_t tiles, uint32_t nkv, Kv4Share share) {
    const uint32_t parts = kv4_parts(tiles, many ? share.many : share.few);
    const uint64_t n = (uint64_t)blocks * nkv;
    Kv4Trial t{0, 0, 0, parts > 1 && n > 0};
    (many ? t.many : t.few) = kv4_bounded(n * parts);
    if (!many) t.load = kv4_bounded(n * (tiles + KV4_START * parts));
    return t;
}
// Nothing cut; all at once; or those of few pairs one after the other where those of
// many leave room.
static inline CHK_HD bool kv4_fits(Kv4Trial t, uint32_t groups, Kv4Share share) {
    if (!t.cut) return true;
    if (t.many > groups) return false;
    const uint32_t left = groups - t.many;
    return t.few <= left || t.load <= (uint64_t)left * (share.few + KV4_START);
}

// Shared prefixes: where there are more workgroups than the device takes at once, a few-pairs
// block whose walk is at most a step of four waves (`least` tiles) is a wave's alone, four
// to a workgroup: most of what such a workgroup takes is its start and its waves' join
// (129 bf16 rows of 8 x 256 over as many kv heads, up to 60 tokens behind three prefixes of
// 1024: 40 us for 52; with walks of up to three steps those are level, and 64 rows of 32 x 128
// behind 8192 tokens take 57 for 53, a wave's tiles coming one after the other).
static inline CHK_HD bool kv4_crowded(Kv4Trial t, uint32_t groups) { return t.few + t.many > groups; }
static inline CHK_HD bool kv4_solo(bool crowded, uint32_t many, uint32_t parts, uint32_t tiles, uint32_t least) {
    return crowded && !many && parts == 1 && tiles <= least;
}

// Blocks of few [0] and of many [1] pairs: their pairs (log2), the rows before that of
// their last pair, the most rows behind that of the first.
struct Kv4Blocks {
    uint16_t pairs[2], first[2], behind[2];
};
static inline CHK_HD Kv4Blocks kv4_block_shapes(uint32_t group, uint32_t block) {
    Kv4Blocks s{};
    for (int i = 0; i < 2; ++i) {
        const uint32_t r = i ? block : KV4_ROWS;
        s.pairs[i] = r == 16 ? 4 : r == 64 ? 6 : 7;
        s.first[i] = (uint16_t)((r - 1) / group);
        s.behind[i] = (uint16_t)((r + group - 2) / group);
    }
    return s;
}
static inline CHK_HD uint32_t kv4_blocks(uint32_t flat, uint32_t many, const Kv4Blocks& s) {
    const uint32_t lg = many ? s.pairs[1] : s.pairs[0];
    return (flat + (1u << lg) - 1) >> lg;
}

struct Kv4Window {
    uint32_t window, sinks;  // window >= 1; neither past 2^30
};
static inline CHK_HD Kv4Window kv4_window(uint32_t window, uint32_t sinks) {
    const uint32_t most = 1u << 30;  // (past a table's 2^30 tokens every window is the same)
    return Kv4Window{window < most ? window : most, sinks < most ? sinks : most};
}

struct Kv4Walk {
    int32_t seen;         // tokens before the last row's end, the gap's included
    uint32_t tiles;       // of the walk
    uint32_t head, gap;   // tiles
};

// Walk of the pairs m0..m1 through a window.
static inline CHK_HD Kv4Walk kv4_window_walk(uint32_t len, uint32_t n, uint32_t group, uint32_t m0, uint32_t m1, Kv4Window v) {
    Kv4Walk k;
    k.seen = kv4_seen(len, n, group, m1);
    const int32_t low = kv4_seen(len, n, group, m0) - (int32_t)v.window;  // the first row's first token of its window
    const uint32_t from = low > 0 ? (uint32_t)low / KV4_TILE : 0u, first = (v.sinks + KV4_TILE - 1) / KV4_TILE;
    k.head = first < from ? first : from;
    k.gap = from - k.head;
    k.tiles = kv4_tiles(k.seen);
    k.tiles = k.tiles > k.gap ? k.tiles - k.gap : 0u;
    return k;
}

// What a sequence is to the cut through a window: its blocks, and a bound of the tiles
// of any of them (a block's rows and their windows are a run of window + rows - 1 tokens).
struct Kv4Span {
    uint32_t flat, many, blocks, tiles;
};
static inline CHK_HD Kv4Span kv4_window_span(uint32_t len, uint32_t n, uint32_t group, Kv4Window v, const Kv4Blocks& shapes) {
    Kv4Span s;
    s.flat = n * group;
    s.many = s.flat > KV4_FEW;
    s.blocks = kv4_blocks(s.flat, s.many, shapes);
    const uint32_t run = v.window + (s.many ? shapes.behind[1] : shapes.behind[0]);
    const uint32_t most = (v.sinks + KV4_TILE - 1) / KV4_TILE + (run + 2 * KV4_TILE - 2) / KV4_TILE, all = kv4_tiles((int32_t)len);
    s.tiles = all < most ? all : most;
    return s;
}
// kv4_cost through a window: blocks rise by the rows' tokens until their walk is
// full.  At least half the most a block (few pairs: all of it), as there.
static inline CHK_HD uint64_t kv4_window_cost(const Kv4Span& s, uint32_t len, uint32_t n, uint32_t group, const Kv4Blocks& shapes) {
    uint64_t cost = (uint64_t)s.blocks * s.tiles;
    if (s.many) {
        const uint32_t first = kv4_tiles((int32_t)len - (int32_t)n + (int32_t)shapes.first[1] + 1);
        if (first < s.tiles) {
            uint64_t rising = ((uint64_t)(s.tiles - first) * KV4_TILE * group) >> shapes.pairs[1];
            if (rising > s.blocks) rising = s.blocks;
            cost -= rising * (s.tiles - first) / 2;
        }
    }
    return cost;
}

// A shared prefix.  Sequences first[g] .. first[g + 1] begin with the same tokens[g]
// tokens; all of the group's rows take those in one walk, as rows of one sequence that
// see all of it, and then each sequence's rows take the rest of their own.  Whole
// tiles are shared, and no more than every row of the group sees: so the result is
// that of plain causal attention.  Members are the group's sequences that have
// rows, a table that holds their length and no rows before position 0.
//
// A walk of the call: the groups' come first, then the sequences'.
struct Kv4Work {
    uint32_t seq;          // whose table
    uint32_t s0, n, len;   // rows; tokens (of a group: the shared ones)
    uint32_t lo;           // tile that the walk begins at
    uint32_t held, whole;  // whole: every row sees all of it
    uint32_t part;         // its rows' results are always joined
    uint32_t group;        // of a sequence whose rows a group's walk has begun: its index
    uint32_t most;         // tokens that a row may see in all (bounds the sums)
    uint32_t many;         // blocks of many pairs
    uint32_t solo;         // a wave a block
    uint32_t base;         // first partial row
    uint32_t parts, piece;
    uint32_t pad;
};
constexpr uint32_t KV4_NO_GROUP = 0xffffffffu;
// A group of up to SHARED_FEW pairs takes few-pairs blocks, and one of up to KV4_FEW
// where those have no more than SHARED_SMALL tiles for each workgroup of the device (kv
// heads together): twice the vector work then costs less than the other blocks' longer
// start (48 bf16 pairs of 128 dims in two groups behind 46080 and 36864 tokens 31 us for 41;
// 64 f16 pairs of two kv heads of 256 behind 16320 level; of 8 kv heads behind 29952, 30
// tiles each, 80 for 65 the other way).
constexpr uint32_t KV4_SHARED_FEW = 32;
constexpr uint32_t KV4_SHARED_SMALL = 8;

// What a group's members come to.
struct Kv4Group {
    uint32_t lead, members;
    uint32_t s0, s1;   // their rows
    uint32_t least;    // tokens that each of their rows sees
    uint32_t most;     // tokens of the longest
    uint32_t cost;     // of a tile of theirs, one by one (kv4_blocks_cost)
};

static inline CHK_HD bool kv4_member(uint32_t n, uint32_t len, bool held) { return n > 0 && held && len >= n; }
static inline CHK_HD uint32_t kv4_blocks_cost(uint32_t flat, uint32_t many, const Kv4Blocks& shapes) {
    return kv4_blocks(flat, many, shapes) * (many ? KV4_MANY_COST : 1u);
}
static inline CHK_HD Kv4Work kv4_no_work() {
    return Kv4Work{0, 0, 0, 0, 0, 1, 0, 0, KV4_NO_GROUP, 0, 0, 0, 0, 1, 1, 0};
}
// The group's walk; none (n = 0) where it would not save a quarter of what its members'
// blocks cost: rows that fill blocks of their own share nothing but reads, which the
// caches have, and then pay for the join.
// small: tiles of few-pairs blocks of one kv head (KV4_SHARED_SMALL).
static inline CHK_HD Kv4Work kv4_group_work(const Kv4Group& g, uint32_t tokens, uint32_t group, const Kv4Blocks& shapes,
                                            uint32_t small) {
    Kv4Work k = kv4_no_work();
    k.whole = k.part = 1;
    if (g.members < 2) return k;
    k.len = (tokens < g.least ? tokens : g.least) / KV4_TILE * KV4_TILE;
    const uint32_t n = g.s1 - g.s0, flat = n * group, tiles = k.len / KV4_TILE;
    const uint32_t many = flat > KV4_FEW || (flat > KV4_SHARED_FEW && kv4_blocks(flat, 0, shapes) * tiles > small);
    if (k.len == 0 || 4ull * kv4_blocks_cost(flat, many, shapes) > 3ull * g.cost) return k;
    k.seq = g.lead;
    k.s0 = g.s0;
    k.n = n;
    k.most = g.most;
    k.many = many;
    return k;
}
// A sequence's walk; group, shared: those of its group's walk, KV4_NO_GROUP where
// there is none or it is no member.
static inline CHK_HD Kv4Work kv4_seq_work(uint32_t b, uint32_t s0, uint32_t n, uint32_t len, bool held, uint32_t heads,
                                          uint32_t group, uint32_t shared) {
    Kv4Work k = kv4_no_work();
    k.seq = b;
    k.s0 = s0;
    k.n = n;
    k.len = k.most = len;
    k.held = held ? 1 : 0;
    k.many = n * heads > KV4_FEW;
    if (group != KV4_NO_GROUP) {
        k.lo = shared / KV4_TILE;
        k.part = 1;
        k.group = group;
    }
    return k;
}

// Tiles of the block whose last pair is of the walk's row `row`.
static inline CHK_HD uint32_t kv4_work_tiles(const Kv4Work& k, uint32_t row) {
    const int32_t seen = !k.held ? 0 : k.whole ? (int32_t)k.len : (int32_t)k.len - (int32_t)k.n + (int32_t)row + 1;
    const uint32_t t = kv4_tiles(seen);
    return t > k.lo ? t - k.lo : 0u;
}
static inline CHK_HD uint32_t kv4_work_most(const Kv4Work& k) { return k.n ? kv4_work_tiles(k, k.n - 1) : 0u; }
// kv4_cost and kv4_cut of a walk.
static inline CHK_HD uint64_t kv4_work_cost(const Kv4Work& k, uint32_t group, const Kv4Blocks& shapes) {
    if (k.n == 0) return 0;
    const uint32_t at = k.many ? shapes.first[1] : shapes.first[0];
    const uint32_t first = kv4_work_tiles(k, at < k.n ? at : k.n - 1), last = kv4_work_most(k);
    return (uint64_t)kv4_blocks(k.n * group, k.many, shapes) * ((first + last + 1) / 2);
}
static inline CHK_HD void kv4_work_cut(Kv4Work& k, Kv4Share share, bool crowded, uint32_t least) {
    k.piece = k.many ? share.many : share.few;
    const uint32_t tiles = kv4_work_most(k);
    k.parts = kv4_parts(tiles, k.piece);
    k.solo = kv4_solo(crowded, k.many, k.parts, tiles, least);
}
// What a walk adds to a call: workgroups, partial rows, and rows to join (a group's
// are joined with its sequences').
static inline CHK_HD uint32_t kv4_work_items(const Kv4Work& k, uint32_t group, const Kv4Blocks& shapes, uint32_t nkv) {
    return kv4_blocks(k.n * group, k.many, shapes) * nkv * k.parts;
}
static inline CHK_HD uint32_t kv4_work_partials(const Kv4Work& k, uint32_t group, uint32_t nkv) {
    return k.part || k.parts > 1 ? k.n * group * nkv * k.parts : 0u;
}
static inline CHK_HD uint32_t kv4_work_joins(const Kv4Work& k, uint32_t group, uint32_t nkv) {
    return !k.whole && (k.part || k.parts > 1) ? k.n * group * nkv : 0u;
}

// Rows of partial results that a call may leave in its workspace.  A sequence
// whose last block has parts > 1 has parts < 2 tiles / piece, tiles that
// block's, and leaves at most flat nkv parts rows, flat at most the pairs of
// its blocks.  The sum of blocks nkv cost / piece over a kind's sequences is at
// most `groups`, and the cost at least half of `tiles` a block: 4 groups pairs
// a block in all.  (Few pairs are at most 64 rows, so their first block sees a
// tile less than the last at most, and the mean, rounded up, is the last one's:
// 2 groups.)
static inline CHK_HD uint64_t kv4_partial_rows(uint64_t rows, uint32_t group, uint32_t groups, uint32_t block) {
    const uint64_t f = rows * group;
    uint64_t r = 2ull * groups * (f < KV4_ROWS ? f : KV4_ROWS);
    if (f > KV4_FEW) r += 4ull * groups * block;
    return r + KV4_ROWS;
}
// And with shared prefixes, in walks that have one part too: a pair of a member's
// rows leaves one of its prefix and one of its own.  With F pairs in its rows, m
// members and blocks of B, a group's walk is taken where 2 F / B <= 3/4 (2 F / B + 4 m)
// at most (a member of few pairs has 4 blocks, of f many f / B + 1), so F <= 6 m B.
static inline CHK_HD uint64_t kv4_prefix_partial_rows(uint64_t rows, uint32_t group, uint32_t nkv, uint32_t n, uint32_t groups,
                                                      uint32_t block) {
    const uint64_t f = rows * group, most = 6ull * n * block;
    uint64_t r = 2ull * groups * (f < KV4_ROWS ? f : KV4_ROWS);
    if (f > KV4_SHARED_FEW) r += 4ull * groups * block;
    return r + KV4_ROWS + 2ull * (f < most ? f : most) * nkv;
}

}  // namespace chk
