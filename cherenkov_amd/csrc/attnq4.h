// Causal attention over the 4-bit key/value cache: what its kernels share (the
// arguments, the cut of the work, operands in f16 parts, the end of a row).
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "kernels_internal.h"
#include "kvq4.h"

namespace chk {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

struct AttnQ4Args {
    Kv4Cache c;
    Kv4Seqs s;
    const void* q;
    void* out;
    uint64_t q_stride, out_stride;  // elements
    uint32_t group, gated;          // group: query heads a kv head
    float scale;                    // log2(e) / sqrt(hd): scores count in powers of two
    const uint32_t* mask;           // null: none
    uint32_t words, ratio, kblk;
    uint32_t groups;      // workgroups that the work is cut for
    uint32_t block;       // rows of a workgroup where a sequence has many
    uint32_t least;       // least tiles of a workgroup's part where it has few
    uint32_t run;         // rows of a wave of the join
    uint32_t cap;         // partial rows of the workspace
    float* po;            // [cap][hd] numerators
    float2* pml;          // [cap] (maximum, sum)
};

// Tokens of a step of k_attn_q4, of which its four waves take every fourth: 256
// dims take the registers of 64 tokens of 128.
constexpr CHK_HD uint32_t q4_step(uint32_t hd) { return hd == 128 ? 64u : 32u; }

// ---- the cut, by each wave for itself: lane = sequence

// Inclusive sum over the lanes.
CHK_DEV uint32_t wave_scan(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
    return v;
}
CHK_DEV uint32_t lane_value(uint32_t v, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane); }

// One lane's sequence.
struct SeqLane {
    uint32_t s0, n, len;  // len 0 where the table cannot hold it
    bool held;  // its table can hold its length
};

CHK_DEV SeqLane seq_lane(const AttnQ4Args& a, uint32_t b) {
    SeqLane q{0, 0, 0, true};
    if (b < a.s.n) {
        uint32_t s1;
        kv4_rows(a.s.start, b, a.s.rows, q.s0, s1);
        q.n = s1 - q.s0;
        q.len = a.s.len[b];
        q.held = q.len <= (uint64_t)a.s.width << a.c.page_log2;
        if (!q.held) q.len = 0;
    }
    return q;
}

// Where an item of the launch lies: a sequence (uniform over the wave).
struct Item {
    uint32_t b, s0, n, len, held;
    Kv4Cut cut;
    uint32_t local;  // item within the sequence
    uint32_t base;   // its first partial row
};

enum Q4Items { Q4_FEW, Q4_MANY, Q4_JOIN };

struct Planner {
    const AttnQ4Args& a;
    uint32_t lane;
    Kv4Share share;
    SeqLane first;  // of the first 64 sequences

    // A sum over the lanes, exact: 16 bits at a time in f32.
    CHK_DEV static uint64_t exact_sum(uint64_t v) {
        return (uint64_t)wave_sum((float)(uint32_t)(v & 0xffff)) + ((uint64_t)wave_sum((float)(uint32_t)((v >> 16) & 0xffff)) << 16) +
               ((uint64_t)wave_sum((float)(uint32_t)((v >> 32) & 0xffff)) << 32);
    }

    CHK_DEV Planner(const AttnQ4Args& a_, uint32_t lane_) : a(a_), lane(lane_) {
        first = seq_lane(a, lane);
        uint64_t few = 0, many = 0;
        for (uint32_t c0 = 0; c0 < a.s.n; c0 += 64) {
            const SeqLane q = c0 ? seq_lane(a, c0 + lane) : first;
            const bool lots = q.n * a.group > KV4_FEW;
            const uint64_t w = kv4_cost(q.len, q.n, a.group, a.block);
            few += exact_sum(lots ? 0 : w);
            if (__any(lots)) many += exact_sum(lots ? w : 0);
        }
        // a wave of a few-pairs block takes a step at least, of the others two tiles
        share.few = (uint32_t)__builtin_amdgcn_readfirstlane((int)kv4_share_few(few * a.c.nkv, a.groups, a.least));
        share.many = (uint32_t)__builtin_amdgcn_readfirstlane((int)kv4_share(many * a.c.nkv, a.groups, 2));
    }

    // The sequence of item x; false past the last.  Items: the pieces of blocks
    // of the sequences with few or with many pairs, or the flattened rows of
    // sequences cut in parts (what is joined).
    template <Q4Items KIND>
    CHK_DEV bool find(uint32_t x, Item& it) const {
        uint32_t items = 0, rows = 0;
        for (uint32_t c0 = 0; c0 < a.s.n; c0 += 64) {
            const SeqLane q = c0 ? seq_lane(a, c0 + lane) : first;
            const Kv4Cut cut = kv4_cut(q.len, q.n, a.group, a.block, share);
            const uint32_t nrow = cut.parts > 1 ? cut.flat * a.c.nkv : 0u;
            const uint32_t nitem = KIND == Q4_JOIN ? nrow : (KIND == Q4_MANY) == (cut.many != 0) ? cut.blocks * a.c.nkv * cut.parts : 0u;
            const uint32_t iin = wave_scan(nitem) + items, rin = wave_scan(nrow * cut.parts) + rows;
            const uint64_t past = __ballot(iin > x);
            if (past) {
                const uint32_t l = (uint32_t)__builtin_ctzll(past);
                it.b = c0 + l;
                it.s0 = lane_value(q.s0, l);
                it.n = lane_value(q.n, l);
                it.len = lane_value(q.len, l);
                it.held = lane_value(q.held ? 1u : 0u, l);
                it.cut = kv4_cut(it.len, it.n, a.group, a.block, share);
                it.local = x - (lane_value(iin, l) - lane_value(nitem, l));
                it.base = lane_value(rin, l) - lane_value(nrow * cut.parts, l);
                return true;
            }
            items = lane_value(iin, 63);
            rows = lane_value(rin, 63);
        }
        return false;
    }
};

// ---- pieces of the wave's work

// f16 parts of the operands beside the codes.  q: 16-bit rows' fit one, f32 rows'
// take two (22 bits).  P s, the numerators: two.  Of bf16 rows of a sequence
// with many pairs (PM) one, rounded to 11 bits beside the 8 that out keeps:
// two cost a prompt a quarter of its time (4 x 4096 rows of 32 x 128, 570 us
// against 456), and their error, averaged over the tokens, is a tenth of out's.
// Single tokens, bound by memory, have two (64 rows, 95 us against 92).
template <class T>
struct Q4Form {
    static constexpr int PQ = sizeof(T) == 4 ? 2 : 1, PP = 2, PM = std::is_same<T, __bf16>::value ? 1 : 2;
};

CHK_DEV void load16(const float* p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 f = reinterpret_cast<const float4*>(p)[i];
        v[4 * i] = f.x;
        v[4 * i + 1] = f.y;
        v[4 * i + 2] = f.z;
        v[4 * i + 3] = f.w;
    }
}
CHK_DEV void load16(const _Float16* p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const h8v f = reinterpret_cast<const h8v*>(p)[i];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] = (float)f[j];
    }
}
CHK_DEV void load16(const __bf16* p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 f = reinterpret_cast<const uint4*>(p)[i];
        const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
            v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
}

CHK_DEV uint32_t pack_h2(float a, float b) { return __builtin_bit_cast(uint32_t, h2v{(_Float16)a, (_Float16)b}); }

// Codes count from their middle, c - 8 (and b + 8 s for b): of either sign, so
// neither product is a difference of large sums.  A masked nibble on the bits
// of 1024 is 1024 + c in f16, or 1024 + 16 c where the mask keeps it in place.
// (Key codes left on their 1024, its part of the product taken off in f32, are
// four additions a word less, 3 to 5 % of single tokens over long contexts, but
// scores that are small differences came out 1 % off.)
constexpr float KV4_EVEN = 1032.0f, KV4_ODD = 1152.0f;
CHK_DEV uint32_t centred(uint32_t u, bool odd) {
    const _Float16 f = (_Float16)(odd ? KV4_ODD : KV4_EVEN);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, u) - h2{f, f});
}

// The eight codes of a word, in the order nibble 0, 4, 1, 5, 2, 6, 3, 7 and
// those of odd nibbles 16-fold.
CHK_DEV h8v codes_h8(uint32_t w, const Q4Consts& k) {
    const uint32_t w8 = w >> 8;
    return __builtin_bit_cast(h8v, make_uint4(centred((w & k.m1) | k.magic, false), centred((w & k.m2) | k.magic, true),
                                              centred((w8 & k.m1) | k.magic, false), centred((w8 & k.m2) | k.magic, true)));
}

// A lane's value joined with those of the lanes 16, 32 and 48 further (the four
// token quarters of a row), on lane-half swaps: every lane ends with the result.
template <class F>
CHK_DEV float over_quarters(float v, F&& join) {
    typedef unsigned u2v __attribute__((ext_vector_type(2)));
    u2v r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = join(__uint_as_float(r.x), __uint_as_float(r.y));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return join(__uint_as_float(r.x), __uint_as_float(r.y));
}
CHK_DEV float quarters_max(float v) {
    return over_quarters(v, [](float a, float b) __attribute__((always_inline)) { return fmaxf(a, b); });
}
CHK_DEV float quarters_sum(float v) {
    return over_quarters(v, [](float a, float b) __attribute__((always_inline)) { return a + b; });
}
// f16 parts of a pair: hi to nearest, lo what it leaves.  The values are made
// opaque first: a product's conversion may otherwise be fused (one rounding) in
// one place and not in another, and lo then belongs to another hi.
template <int PARTS>
CHK_DEV void split_h2(float a, float b, uint32_t& hi, uint32_t& lo) {
    asm("" : "+v"(a), "+v"(b));
    const h2v h = h2v{(_Float16)a, (_Float16)b};
    hi = __builtin_bit_cast(uint32_t, h);
    if (PARTS > 1) lo = pack_h2(a - (float)h.x, b - (float)h.y);
}
// The value of the row 4 kq + i (held by lane 4 kq + i) where the products'
// results want it; the lane number opaque, so that no address waits in a register.
CHK_DEV float of_row(float v, uint32_t kq, int i) {
    uint32_t l = 4 * kq + i;
    asm volatile("" : "+v"(l));
    return __shfl(v, (int)l, 64);
}

// The tokens of a step that a row's mask hides: bit j for token t0 + 4 j + kq,
// j < n.  nblk: the complete blocks that the mask holds for.  Blocks of four
// tokens, the indexer's of every preset, are one bit of the step's word each
// (t0 is a multiple of 32 tokens, n at most 16); others are looked up.
CHK_DEV uint32_t hidden(const AttnQ4Args& a, uint32_t row, uint32_t nblk, uint32_t t0, uint32_t kq, uint32_t n) {
    if (a.ratio == 4) {
        const uint32_t b0 = t0 >> 2, wi = b0 >> 5;
        const uint32_t word = nblk && wi < a.words ? a.mask[(size_t)row * a.words + wi] : 0u;
        const uint32_t held = nblk > b0 ? nblk - b0 : 0u;
        return ~(word >> (b0 & 31)) & (held < 16u ? (1u << held) - 1u : 0xffffu);
    }
    uint32_t hide = 0u;
#pragma unroll 1
    for (uint32_t j = 0; j < n; ++j) {
        const uint32_t bk = (t0 + 4 * j + kq) / a.ratio;
        const bool see = bk >= nblk || ((bk >> 5) < a.words && ((a.mask[(size_t)row * a.words + (bk >> 5)] >> (bk & 31)) & 1u));
        hide |= (see ? 0u : 1u) << j;
    }
    return hide;
}

// Orders LDS accesses of one wave: its own memory, no other wave's.
CHK_DEV void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// log2: the numerators run that far above the row's reference before it is
// moved, so most steps move nothing; 15 - that below f16's top at the start.
constexpr float KV4_P_TOP = 8.0f;
// log2: the spread of value steps that one bound serves.  The reference counts
// the value step in (P s is what f16 holds), so a token 2^12 below the bound
// still has its leading bits above f16's least; beyond it each token's own is
// taken, 16 more additions a step.
constexpr float KV4_SPAN = 12.0f;
// The reference counts |b + 8 s| in too, that factor down: P (b + 8 s) is an f32
// sum, below 2^(15 + 64) a token, and only groups of one number, whose step is
// the least, have so large a quotient (else s is 2^-28 of the values or more).
constexpr float KV4_BIAS = 0x1p-64f;
// A step of values as attention takes it: the least, 2^-126, which groups of one
// number (zeros) have, as none.  P s of it has no bits in f16, and what s (c - 8)
// then lacks of b + 8 s would be left over, 2^-123 for a group of zeros.
CHK_DEV float value_step(uint32_t pair) {
    const float s = __uint_as_float(pair << 16);
    return fabsf(s) <= 0x1p-126f ? 0.0f : s;
}
// log2 of the least size that a token of a sequence of `len` is counted with: P
// rises to 2^15 over it, and a sum of len such stays below 2^127.
CHK_DEV float least_size(uint32_t len) { return -96.0f + (len > 0x10000u ? 16.0f - (float)__builtin_clz(len - 1) : 0.0f); }

// out = numerators / sum [* sigmoid(gate)]; a row that saw nothing is 0.
template <int HD, class T>
CHK_DEV void finish(const AttnQ4Args& a, uint64_t row, uint32_t h, uint32_t d, float4 o, float L) {
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    if (a.gated) {
        const T* gp = (const T*)a.q + row * a.q_stride + (uint64_t)h * HD * 2 + HD + d;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= sigmoidf_((float)gp[j]);
    }
    T* op = (T*)a.out + row * a.out_stride + (uint64_t)h * HD + d;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(op) = make_float4(v[0], v[1], v[2], v[3]);
    else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4*>(op) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    }
}

// The kernel for sequences with many pairs (attnq4_rows.hip): the rows of its
// workgroups, and its launch.
uint32_t attn_q4_block(uint32_t hd, uint32_t dtype);
void launch_attn_q4_many(const AttnQ4Args& a, uint32_t hd, uint32_t dtype, uint32_t grid, hipStream_t st);

}  // namespace chk
