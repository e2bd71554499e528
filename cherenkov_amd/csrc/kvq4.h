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
    const uint64_t s = (tiles + groups - 1) / groups;
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

}  // namespace chk
