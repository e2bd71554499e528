// Attention of blocks of many (row, head) pairs of a kv head (attnq4_rows.hip); with a view,
// of few too (attnq4_view.hip).
#pragma once

#include "attnq4_few.h"

namespace chk {

CHK_DEV uint32_t pk_mul(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, a) * __builtin_bit_cast(h2v, b));
}
CHK_DEV uint32_t h_bits(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v); }
CHK_DEV uint32_t both(uint32_t h) { return h | (h << 16); }

template <int HD>
struct ManyLds {
    static constexpr int NG = HD / 64, TS = q4_step(HD), NS = TS / 16, HS = TS / 32;
    // arrays by token: token 4 i + a of a subtile sits at 4 a + i, where row
    // 4 a + i of the first product's result is
    struct Pairs {
        alignas(16) float ce[TS], fv[TS], gv[TS];  // 2^e of the keys; f and 2^-f of the values
        alignas(16) uint32_t sk[NG][TS];           // keys' s 2^-e, twice
        alignas(16) _Float16 sv[NG][TS];           // values' s 2^-f
        alignas(16) _Float16 bk[NS][2][16][8];     // keys' (b + 8 s) 2^-e: parts hi, hi | lo of the groups, then 0
        alignas(16) _Float16 bv[2 * NG][TS];       // values': parts hi, lo of the groups
        uint32_t odd[TS];                          // groups of the values that are not finite
        uint32_t any[2];
    };
    uint4 k[2][NS * NG * 2][64];
    uint4 v[2][HS * NG * 4][64];
    Pairs pr[3];
};

// One item of the many-pairs kind: 64 RB pairs.  With a view, one of the few-pairs kind
// behind the last of those: one launch for both.  (The body is the kernel's own: as a
// function that it calls, 128 dims of bf16 spill 20 registers.)
template <int HD, class T, int RB, int V>
__global__ void __launch_bounds__(256, 2) k_attn_q4_rows(AttnQ4Args a) {
    using Form = Q4Form<T>;
    using Pairs = typename ManyLds<HD>::Pairs;
    constexpr int NG = HD / 64, PQ = Form::PQ, PP = V == Q4_ALL ? Form::PM : Form::PP;
    constexpr int TS = HD == 128 ? 64 : 32, NS = TS / 16, HS = TS / 32;  // tokens, subtiles and depth steps of P V
    constexpr int AHEAD = RB > 1 ? 4 : 6;
    constexpr float TOP = KV4_P_TOP, LIFT = 15.0f - TOP;
    __shared__ union {
        ManyLds<HD> many;
        FewLds<HD, V> few;
    } lds;
    ManyLds<HD>& sm = lds.many;
    const uint32_t lane = threadIdx.x & 63, w = wave_id(), col = lane & 15, kq = lane >> 4;
    const Q4Consts kc;
    Item it;
    {
        const Planner<V> plan(a, lane);
        uint32_t many = 0, none;
        const bool found = (V == Q4_ALL || a.any_many) && plan.template find<Q4_MANY>(blockIdx.x, it, many);
        if (V == Q4_ALL && !found) return;
        if (V != Q4_ALL && !found) {
            uint32_t few;
            bool solo = false;
            if (!plan.template find<Q4_FEW>(blockIdx.x - many, it, few)) {
                if (V != Q4_PREFIX) return;
                solo = true;
                if (!plan.template find<Q4_SOLO>((blockIdx.x - many - few) * KV4_WAVES + w, it, none)) return;
            }
            few_block<HD, T, V>(a, it, V == Q4_PREFIX && solo, lds.few);
            return;
        }
    }
    const uint32_t hk = it.local % a.c.nkv, y = it.local / a.c.nkv;
    // blocks later in the sequence see more tokens: longest first
    const uint32_t z = y / it.cut.blocks, blk = it.cut.blocks - 1 - y % it.cut.blocks;
    const uint32_t m_wg = blk * (64 * RB), m0 = m_wg + w * (16 * RB), flat = it.cut.flat;
    const int32_t before = (int32_t)it.len - (int32_t)it.n;
    // tokens that the workgroup's last row sees, and this wave's first
    int32_t wg_see;
    const Kv4Walk view = walk_of<V>(a, it, m_wg, min(m_wg + 64 * RB, flat) - 1, wg_see);
    const int32_t seen = view.seen;
    const int32_t all_see = V == Q4_PREFIX && it.whole ? wg_see : kv4_seen(it.len, it.n, a.group, min(m0, flat - 1));
    const uint32_t tiles = view.tiles, parts = kv4_parts(tiles, it.cut.piece);
    // the walk's token t in the sequence
    const uint32_t head = view.head * KV4_TILE, gap = view.gap * KV4_TILE;
    auto real = [&](uint32_t t) __attribute__((always_inline)) { return V == Q4_ALL || t < head ? t : t + gap; };
    if (z >= parts) return;
    const uint32_t per = (tiles + parts - 1) / parts;
    const uint32_t tbeg = z * per * KV4_TILE;
    const uint32_t tend = seen > 0 ? min(min(tiles, (z + 1) * per) * KV4_TILE, (uint32_t)seen - (V == Q4_ALL ? 0u : gap)) : 0u;
    const uint32_t steps = tbeg < tend ? (tend - tbeg + TS - 1) / TS : 0u;

    // ---- loads: of codes (a wave: groups 2 cp and 2 cp + 1 of subtile cs) and of
    // pairs, each through its own entry of the table
    const uint32_t* table = a.s.table + (size_t)it.b * a.s.width;
    const uint32_t lg = a.c.page_log2;
    const uint32_t last16 = seen > 0 ? ((uint32_t)seen - 1) & ~15u : 0u;
    const uint32_t cp = HD == 256 ? w >> 1 : 0u, cs = HD == 256 ? w & 1 : w;
    auto sub_of = [&](uint32_t s) __attribute__((always_inline)) { return min(real(tbeg + s * TS) + 16 * cs, last16); };
    auto entry = [&](uint32_t s) __attribute__((always_inline)) { return table[sub_of(s) >> lg]; };
    // (a thread: the pair of one token and group, of the keys in waves 0 and 1 and
    // of the values in 2 and 3)
    const uint32_t ptok = (threadIdx.x & 127) / NG, pg = threadIdx.x % NG;
    const uint32_t least = (uint32_t)(least_size(V == Q4_PREFIX ? it.most : it.len) + 141.0f);
    uint32_t pr;
    auto pair_sub = [&](uint32_t s) __attribute__((always_inline)) { return min(real(tbeg + s * TS) + (ptok & ~15u), last16); };
    auto pair_entry = [&](uint32_t s) __attribute__((always_inline)) { return table[pair_sub(s) >> lg]; };
    auto load_pair = [&](uint32_t s, uint32_t id) __attribute__((always_inline)) {
        const uint64_t r = (((uint64_t)(id < a.c.pages ? id : 0u) * a.c.nkv + hk) << lg) + (pair_sub(s) & ((1u << lg) - 1));
        pr = (w < 2 ? a.c.ks : a.c.vs)[(r + (ptok & 15)) * NG + pg];
        if (id >= a.c.pages) pr = KV4_NAN_PAIR;
    };
    uint4 kcode;
    uint32_t vcode[4];
    const uint32_t koff = (4 * (col & 3) + (col >> 2)) * (HD / 2) + (kq * NG + 2 * cp) * 8;
    const uint32_t voff = kq * (HD / 2) + (col * NG + 2 * cp) * 2;
    auto load_codes = [&](uint32_t s, uint32_t id) __attribute__((always_inline)) {
        id = (uint32_t)__builtin_amdgcn_readfirstlane((int)id);
        const uint64_t sub = (((uint64_t)(id < a.c.pages ? id : 0u) * a.c.nkv + hk) << lg) + (sub_of(s) & ((1u << lg) - 1));
        kcode = *reinterpret_cast<const uint4*>(a.c.k + sub * (HD / 2) + koff);
#pragma unroll
        for (int i = 0; i < 4; ++i) vcode[i] = *reinterpret_cast<const uint32_t*>(a.c.v + sub * (HD / 2) + voff + i * 4 * (HD / 2));
    };

    // ---- pairs of step s into the ring
    auto stage_pair = [&](uint32_t s, uint32_t slot) __attribute__((always_inline)) {
        Pairs& P = sm.pr[slot];
        const uint32_t c = (int32_t)(real(tbeg + s * TS) + ptok) >= seen ? 0u : pr;
        const uint32_t st = ptok >> 4, x = ptok & 15, in = 4 * (x & 3) + (x >> 2), pos = 16 * st + in;
        float sz = value_step(c), ba = fmaf(sz, 8.0f, __uint_as_float(c & 0xffff0000u));
        uint32_t odd = 0u;
        if (!(fabsf(sz) < 0x1p125f && fabsf(ba) < INFINITY)) {
            odd = 1u << pg;
            sz = ba = 0.0f;
        }
        // over the token's groups: most < 2^(e8 - 126)
        float most = fmaxf(8.0f * fabsf(sz), fabsf(ba));
        most = fmaxf(most, CHK_DPPF(most, 0xb1, 0xf, most));
        odd |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)odd, 0xb1, 0xf, 0xf, false);
        if (NG > 2) {
            most = fmaxf(most, CHK_DPPF(most, 0x4e, 0xf, most));
            odd |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)odd, 0x4e, 0xf, 0xf, false);
        }
        // keys' largest to [2^11, 2^12); values' to [2^14, 2^15), their exponent f
        // not below least_size (numerators rise as it falls)
        const uint32_t e8 = max(__float_as_uint(most) >> 23, w < 2 ? 12u : least);
        const float scale = __uint_as_float(((w < 2 ? 265u : 268u) - e8) << 23);
        const _Float16 sh = (_Float16)(sz * scale);
        const float v = ba * scale;
        const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
        if (w < 2) {
            P.sk[pg][pos] = both((uint32_t)__builtin_bit_cast(uint16_t, sh));
            P.bk[st][0][in][pg] = hi;
            P.bk[st][0][in][NG + pg] = hi;
            P.bk[st][1][in][pg] = lo;
            if (pg == 0) P.ce[pos] = odd ? NAN : __uint_as_float((e8 - 11u) << 23);
        } else {
            P.sv[pg][pos] = sh;
            P.bv[pg][pos] = hi;
            P.bv[NG + pg][pos] = lo;
            if (pg == 0) {
                P.fv[pos] = (float)(int32_t)e8 - 141.0f;
                P.gv[pos] = __uint_as_float((268u - e8) << 23);
                P.odd[pos] = odd;
            }
            const uint32_t any = __any(odd != 0u) ? 1u : 0u;
            if (lane == 0) P.any[w & 1] = any;
        }
    };

    // ---- operands of step s from the codes
    auto convert = [&](uint32_t s, uint32_t slot) __attribute__((always_inline)) {
        const Pairs& P = sm.pr[slot];
        const uint32_t sixteenth = both(0x2c00u);
        const uint32_t wd[4] = {kcode.x, kcode.y, kcode.z, kcode.w};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t g = 2 * cp + i, se = P.sk[g][16 * cs + col], so = pk_mul(se, sixteenth);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const uint4 u = __builtin_bit_cast(uint4, codes_h8(wd[2 * i + ks], kc));
                sm.k[s & 1][(cs * NG + g) * 2 + ks][lane] =
                    make_uint4(pk_mul(u.x, se), pk_mul(u.y, so), pk_mul(u.z, se), pk_mul(u.w, so));
            }
        }
        // values: this subtile's half of an operand's eight tokens
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t g = 2 * cp + i;
            const uint2 se = *reinterpret_cast<const uint2*>(&P.sv[g][16 * cs + 4 * kq]);
            const uint2 so = make_uint2(pk_mul(se.x, sixteenth), pk_mul(se.y, sixteenth));
            const uint32_t sel = i ? 0x07060302u : 0x05040100u;
            const uint32_t h0 = __builtin_amdgcn_perm(vcode[1], vcode[0], sel), h1 = __builtin_amdgcn_perm(vcode[3], vcode[2], sel);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t m = e & 1 ? kc.m2 : kc.m1;
                const uint32_t u0 = centred(((e & 2 ? h0 >> 8 : h0) & m) | kc.magic, e & 1);
                const uint32_t u1 = centred(((e & 2 ? h1 >> 8 : h1) & m) | kc.magic, e & 1);
                reinterpret_cast<uint2*>(&sm.v[s & 1][((cs >> 1) * NG + g) * 4 + e][lane])[cs & 1] =
                    make_uint2(pk_mul(u0, e & 1 ? so.x : se.x), pk_mul(u1, e & 1 ? so.y : se.y));
            }
        }
    };

    // ---- this lane's rows (the scores' columns) and their queries
    int32_t p[RB];
    uint32_t nblk[RB], row[RB];
    h8v qf[RB][PQ][NG][2], qb[RB];
    float rf[RB];  // scores: result x 2^e x rf
    bool any_mask = false;
    uint32_t id = entry(0), pid = pair_entry(0);
    // slots of the keys' least values past the groups' are 0 for good
    for (uint32_t i = threadIdx.x; i < 3 * NS * 2 * 16; i += CHK_WG) {
        const uint32_t in = i & 31;
        *reinterpret_cast<uint4*>(sm.pr[i / (NS * 32)].bk[(i / 32) % NS][in >> 4][in & 15]) = make_uint4(0u, 0u, 0u, 0u);
    }
    load_pair(0, pid);
    load_codes(0, id);
    id = entry(1);
    pid = pair_entry(1);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const uint32_t m = min(m0 + 16 * rb + col, flat - 1), mi = m / a.group, mg = m - mi * a.group;
        p[rb] = before + (int32_t)mi;
        row[rb] = it.s0 + mi;
        nblk[rb] = a.mask && p[rb] >= 0 ? (uint32_t)(p[rb] + 1) / a.ratio : 0u;
        nblk[rb] = nblk[rb] > a.kblk ? nblk[rb] : 0u;
        any_mask = any_mask || __any(nblk[rb] != 0u);
        const T* src = (const T*)a.q + (uint64_t)row[rb] * a.q_stride + (uint64_t)(hk * a.group + mg) * HD * (a.gated ? 2 : 1);
        float v[NG][16], mx = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) load16(src + 64 * g + 16 * kq, v[g]);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(v[g][i]));
        mx = quarters_max(mx);
        // largest to [2^8, 2^9): a group's sum stays in f16
        const uint32_t e8 = min(max(__float_as_uint(mx) >> 23, 9u), 254u);
        const float up = __uint_as_float((262u - e8) << 23);
        rf[rb] = __uint_as_float((e8 - 8u) << 23) * a.scale;
        uint32_t qs[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float sum = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x0 = v[g][8 * ks + j] * up, x1 = v[g][8 * ks + j + 4] * up;
                    sum += x0 + x1;
                    split_h2<PQ>(x0, x1, hi[j], lo[j]);
                }
                qf[rb][0][g][ks] = __builtin_bit_cast(h8v, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                if (PQ > 1) qf[rb][PQ - 1][g][ks] = __builtin_bit_cast(h8v, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            sum = quarters_sum(sum);
            const uint32_t h = h_bits(sum), r = h_bits(sum - (float)__builtin_bit_cast(_Float16, (uint16_t)h));
            qs[g / 2] |= h << (16 * (g % 2));
            if (kq == 0) qs[(NG + g) / 2] |= r << (16 * (g % 2));
        }
        if (kq > 1) qs[0] = qs[1] = 0u;
        qb[rb] = __builtin_bit_cast(h8v, make_uint4(qs[0], qs[1], qs[2], qs[3]));
    }

    f4v o[RB][NG * 4], obt[RB];
    float l[RB], mref[RB];
    uint32_t poison[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        l[rb] = 0.0f;
        mref[rb] = -INFINITY;
        poison[rb] = 0u;
        obt[rb] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) o[rb][i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    __syncthreads();
    stage_pair(0, 0);
    load_pair(1, pid);
    pid = pair_entry(2);
    __syncthreads();
    convert(0, 0);
    load_codes(1, id);
    id = entry(2);
    stage_pair(1, 1);
    load_pair(2, pid);
    pid = pair_entry(3);
    __syncthreads();

    uint32_t r0 = 0, r1 = 1, r2 = 2;  // ring slots of steps s, s + 1, s + 2
#pragma unroll 1
    for (uint32_t s = 0; s < steps; ++s) {
        // the next step's operands, the one after's codes, the third's pairs
        convert(s + 1, r1);
        load_codes(s + 2, id);
        id = entry(s + 3);
        stage_pair(s + 2, r2);
        load_pair(s + 3, pid);
        pid = pair_entry(s + 4);
        const uint32_t t0 = real(tbeg + s * TS);
        {
            const Pairs& P = sm.pr[r0];
            const uint4(*kf)[64] = sm.k[s & 1];
            const uint4(*vf)[64] = sm.v[s & 1];
            // ---- scores: a chain of products for every subtile, row block and
            // part of the query, side by side (a product waits for the one before
            // it in its chain)
            float xs[RB][NS][4];
            // (a wave in its products leaves the vector unit to the other workgroup's: 1 to 3 %)
            __builtin_amdgcn_s_setprio(0);
            {
                constexpr int CH = RB * NS * PQ > 4 ? NS / 2 : NS;  // subtiles at a time
#pragma unroll
                for (int s0 = 0; s0 < NS; s0 += CH) {
                    f4v d[CH][RB][PQ];
#pragma unroll
                    for (int st = 0; st < CH; ++st) {
                        const h8v bk = *reinterpret_cast<const h8v*>(P.bk[s0 + st][kq & 1][col]);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            d[st][rb][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bk, qb[rb], f4v{0, 0, 0, 0}, 0, 0, 0);
                            if (PQ > 1) d[st][rb][PQ - 1] = f4v{0, 0, 0, 0};
                        }
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                            for (int st = 0; st < CH; ++st) {
                                const h8v f = __builtin_bit_cast(h8v, kf[((s0 + st) * NG + g) * 2 + ks][lane]);
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                                    for (int q = 0; q < PQ; ++q)
                                        d[st][rb][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, qf[rb][q][g][ks], d[st][rb][q], 0, 0, 0);
                            }
#pragma unroll
                    for (int st = 0; st < CH; ++st) {
                        const float4 ce = *reinterpret_cast<const float4*>(&P.ce[16 * (s0 + st) + 4 * kq]);
                        const float4 fv = *reinterpret_cast<const float4*>(&P.fv[16 * (s0 + st) + 4 * kq]);
                        const float cc[4] = {ce.x, ce.y, ce.z, ce.w}, ff[4] = {fv.x, fv.y, fv.z, fv.w};
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float v = d[st][rb][0][i];
                                if (PQ > 1) v += d[st][rb][PQ - 1][i];
                                xs[rb][s0 + st][i] = fmaf(v * rf[rb], cc[i], ff[i]);
                            }
                    }
                    // operands are read AHEAD reads in front of their products
                    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
                    for (int i = 0; i < CH * (NG * 2 + 1); ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, RB * PQ, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    }
                    if (RB > 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_setprio(1);
            // ---- what a row does not see
            if ((int32_t)(t0 + TS) > all_see) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int st = 0; st < NS; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((int32_t)(t0 + 16 * st + 4 * i) > p[rb] - (int32_t)kq) xs[rb][st][i] = -INFINITY;
            }
            if (V == Q4_WINDOW && (int32_t)t0 < seen - (int32_t)a.view.window && t0 + TS > a.view.sinks) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int st = 0; st < NS; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t t = t0 + 16 * st + 4 * i + kq;
                            if ((int32_t)t <= p[rb] - (int32_t)a.view.window && t >= a.view.sinks) xs[rb][st][i] = -INFINITY;
                        }
            }
            if (V == Q4_ALL && any_mask) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const uint32_t hide = hidden(a, row[rb], nblk[rb], t0, kq, 4 * NS);
#pragma unroll
                    for (int st = 0; st < NS; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((hide >> (4 * st + i)) & 1u) xs[rb][st][i] = -INFINITY;
                }
            }
            // ---- values that are not finite: NaN for the rows that see them
            if (P.any[0] | P.any[1]) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int st = 0; st < NS; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (xs[rb][st][i] != -INFINITY) poison[rb] |= P.odd[16 * st + 4 * kq + i];
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                // ---- the running reference, moved where a numerator would pass 2^15
                float mx = -INFINITY;
#pragma unroll
                for (int st = 0; st < NS; ++st)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, xs[rb][st][i]);
                mx = quarters_max(mx) - LIFT;
                if (__any(mx > mref[rb] + TOP)) {
                    const float mn = fmaxf(mx, mref[rb]);
                    const float al = mref[rb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mref[rb] - mn);
                    mref[rb] = mn;
                    l[rb] *= al;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float ar = of_row(al, kq, i);
                        obt[rb][i] *= ar;
#pragma unroll
                        for (int j = 0; j < NG * 4; ++j) o[rb][j][i] *= ar;
                    }
                }
                const float msafe = mref[rb] == -INFINITY ? 0.0f : mref[rb];
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    const float4 gv = *reinterpret_cast<const float4*>(&P.gv[16 * st + 4 * kq]);
                    const float gg[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        xs[rb][st][i] = __builtin_amdgcn_exp2f(xs[rb][st][i] - msafe);
                        l[rb] = fmaf(xs[rb][st][i], gg[i], l[rb]);
                    }
                }
            }
            // ---- P . V
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int h = 0; h < HS; ++h) {
                h8v pf[RB][PP];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        split_h2<PP>(xs[rb][2 * h + j / 2][2 * (j % 2)], xs[rb][2 * h + j / 2][2 * (j % 2) + 1], hi[j], lo[j]);
                    pf[rb][0] = __builtin_bit_cast(h8v, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                    if (PP > 1) pf[rb][PP - 1] = __builtin_bit_cast(h8v, make_uint4(lo[0], lo[1], lo[2], lo[3]));
                }
                uint2 b0 = make_uint2(0u, 0u), b1 = b0;
                if (col < 2 * NG) {
                    b0 = *reinterpret_cast<const uint2*>(&P.bv[col][32 * h + 4 * kq]);
                    b1 = *reinterpret_cast<const uint2*>(&P.bv[col][32 * h + 16 + 4 * kq]);
                }
                const h8v bf = __builtin_bit_cast(h8v, make_uint4(b0.x, b0.y, b1.x, b1.y));
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int q = 0; q < PP; ++q) obt[rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf[rb][q], bf, obt[rb], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NG * 4; ++j) {
                    const h8v f = __builtin_bit_cast(h8v, vf[h * NG * 4 + j][lane]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                        for (int q = 0; q < PP; ++q)
                            o[rb][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf[rb][q], f, o[rb][j], 0, 0, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 1);
#pragma unroll
                for (int i = 0; i < NG * 4 + 1; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, RB * PP, 1);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
                }
                if (RB > 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(1);
        __syncthreads();
        const uint32_t r = r0;
        r0 = r1;
        r1 = r2;
        r2 = r;
    }

    // ---- out, or this part's numerators
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        l[rb] = quarters_sum(l[rb]);
        uint32_t po = poison[rb];
        po |= (uint32_t)__shfl_xor((int)po, 16, 64);
        po |= (uint32_t)__shfl_xor((int)po, 32, 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = m0 + 16 * rb + 4 * kq + i;
            const float L = of_row(l[rb], kq, i), M = of_row(mref[rb], kq, i);
            const uint32_t bad = (uint32_t)__float_as_uint(of_row(__uint_as_float(po), kq, i));
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t src = 16 * kq + g;
                asm volatile("" : "+v"(src));
                float bias = __shfl(obt[rb][i], (int)src, 64) + __shfl(obt[rb][i], (int)src + NG, 64);
                if ((bad >> g) & 1u) bias = NAN;
                const float4 v = make_float4(o[rb][4 * g][i] + bias, o[rb][4 * g + 1][i] + bias, o[rb][4 * g + 2][i] + bias,
                                             o[rb][4 * g + 3][i] + bias);
                if (m >= flat) continue;
                const uint32_t d = 64 * g + 4 * col;
                if (parts > 1 || (V == Q4_PREFIX && it.part)) {
                    const uint32_t at = it.base + (z * a.c.nkv + hk) * flat + m;
                    if (at < a.cap) {
                        *reinterpret_cast<float4*>(a.po + (size_t)at * HD + d) = v;
                        if (d == 0) a.pml[at] = make_float2(M, L);
                    }
                } else {
                    const uint32_t mi = m / a.group;
                    finish<HD, T>(a, (uint64_t)it.s0 + mi, hk * a.group + m - mi * a.group, d, v, it.held ? L : NAN);
                }
            }
        }
    }
}

}  // namespace chk
