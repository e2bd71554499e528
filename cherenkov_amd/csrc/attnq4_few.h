// k_attn_q4's work on one item: 16 (row, head) pairs of a kv head and a part of the
// tokens that they see (attnq4.hip).
#pragma once

#include "attnq4.h"

namespace chk {

template <int HD>
struct FewPairs {
    static constexpr uint32_t STEP = q4_step(HD);
    alignas(16) float2 k[STEP][HD / 64];
    alignas(16) float2 v[STEP][HD / 64];
    float size[STEP];
};
template <int HD, int V>
struct FewLds {
    union {
        FewPairs<HD> pair[KV4_WAVES];
        float o[KV4_WAVES][KV4_ROWS][HD + 4];
    };
    float2 ml[KV4_WAVES][KV4_ROWS];
};
// With shared prefixes a wave may have an item of its own, and its numerators lie apart
// from the other waves' pairs.
template <int HD>
struct FewLds<HD, Q4_PREFIX> {
    FewPairs<HD> pair[KV4_WAVES];
    float o[KV4_WAVES][KV4_ROWS][HD + 4];
    float2 ml[KV4_WAVES][KV4_ROWS];
};

// One item of the few-pairs kind: the workgroup's four waves', or each wave's own (solo).
template <int HD, class T, int V>
CHK_DEV void few_block(const AttnQ4Args& a, const Item& it, bool solo, FewLds<HD, V>& sm) {
    using Form = Q4Form<T>;
    constexpr int NG = HD / 64, PQ = Form::PQ, PP = Form::PP;
    // P s stays below 2^15 in f16 (and the least of a token 2^SPAN below the
    // largest keeps the bits that the parts have)
    constexpr float TOP = KV4_P_TOP;
    constexpr float LIFT = 15.0f - TOP;  // log2, taken off the reference
    constexpr uint32_t STEP = q4_step(HD);
    constexpr int NS = STEP / 16;
    const uint32_t lane = threadIdx.x & 63, w = wave_id(), col = lane & 15, kq = lane >> 4;
    const Q4Consts kc;
    const T* qp = (const T*)a.q;

    const Kv4Cut& cut = it.cut;
    const uint32_t hk = it.local % a.c.nkv, y = it.local / a.c.nkv;
    const uint32_t z = y / cut.blocks, blk = cut.blocks - 1 - y % cut.blocks;  // longest blocks first
    const uint32_t m0 = blk * KV4_ROWS;
    // positions: row i of the sequence at before + i
    const int32_t before = (int32_t)it.len - (int32_t)it.n;
    // tokens that the block's last row sees, and its first
    int32_t all_see;
    const Kv4Walk view = walk_of<V>(a, it, m0, min(m0 + KV4_ROWS, cut.flat) - 1, all_see);
    const int32_t seen = view.seen;
    const uint32_t tiles = view.tiles, parts = kv4_parts(tiles, cut.piece);
    // the walk's token t in the sequence
    const uint32_t head = view.head * KV4_TILE, gap = view.gap * KV4_TILE;
    auto real = [&](uint32_t t) __attribute__((always_inline)) { return V == Q4_ALL || t < head ? t : t + gap; };
    if (z >= parts) return;
    const uint32_t per = (tiles + parts - 1) / parts;

    // Folded: where the block's pairs fill a quarter of the columns, all four
    // quarters hold them, and quarter `cls` takes subtile cls of every step: rows
    // of their own, joined at the end, whose scores are a quarter of the vector
    // work.  (256 dims have two subtiles a step, and no registers for both forms.)
    constexpr uint32_t FOLD = KV4_ROWS / NS;  // pairs
    const bool fold = HD == 128 && cut.flat - m0 <= FOLD;
    const uint32_t cls = col / FOLD;
    // this lane's row (the scores' column)
    const uint32_t m = min(m0 + (fold ? col % FOLD : col), cut.flat - 1), mi = m / a.group, mg = m - mi * a.group;
    const int32_t p = before + (int32_t)mi;
    const uint32_t row = it.s0 + mi;
    // complete blocks of a row that its mask holds for, else 0: all visible
    uint32_t nblk = a.mask && p >= 0 ? (uint32_t)(p + 1) / a.ratio : 0u;
    nblk = nblk > a.kblk ? nblk : 0u;
    const bool any_mask = __any(nblk != 0u);

    // ---- the wave's steps and their loads.  A step's table entries are read
    // two steps ahead, its pairs and keys once the keys before them are used,
    // its values after the values before them: loads are in flight throughout
    // in the registers of one step.
    const uint32_t* table = a.s.table + (size_t)it.b * a.s.width;
    const uint32_t lg = a.c.page_log2;
    const uint32_t last16 = seen > 0 ? ((uint32_t)seen - 1) & ~15u : 0u;
    const uint32_t tend = seen > 0 ? min(min(tiles, (z + 1) * per) * KV4_TILE, (uint32_t)seen - (V == Q4_ALL ? 0u : gap)) : 0u;
    const uint32_t tl = lane % STEP;
    uint32_t t0 = z * per * KV4_TILE + (solo ? 0u : w * STEP);
    const uint32_t NEXT = solo ? STEP : KV4_WAVES * STEP;
    // the page of this lane's subtile; one behind the last visible token
    // repeats its subtile
    auto entry = [&](uint32_t t) __attribute__((always_inline)) {
        return table[min(t + (tl & ~15u), last16) >> lg];
    };
    uint64_t sub_l, sub[NS];
    bool bad_l;
    auto place = [&](uint32_t t, uint32_t id) __attribute__((always_inline)) {
        bad_l = id >= a.c.pages;
        sub_l = (((uint64_t)(bad_l ? 0u : id) * a.c.nkv + hk) << lg) + (min(t + (tl & ~15u), last16) & ((1u << lg) - 1));
#pragma unroll
        for (int st = 0; st < NS; ++st)
            sub[st] = (uint64_t)lane_value((uint32_t)sub_l, 16 * st) | ((uint64_t)lane_value((uint32_t)(sub_l >> 32), 16 * st) << 32);
    };
    uint32_t pk[NG], pv[NG];
    uint4 kw[NS][NG / 2];
    uint32_t vw[NS][4][NG / 2];
    auto load_keys = [&]() __attribute__((always_inline)) {
        const uint32_t* kp = a.c.ks + (sub_l + col) * NG;
        const uint32_t* vp = a.c.vs + (sub_l + col) * NG;
        if constexpr (NG == 2) {
            const uint2 x0 = *reinterpret_cast<const uint2*>(kp), x1 = *reinterpret_cast<const uint2*>(vp);
            pk[0] = x0.x, pk[1] = x0.y, pv[0] = x1.x, pv[1] = x1.y;
        } else {
            const uint4 x0 = *reinterpret_cast<const uint4*>(kp), x1 = *reinterpret_cast<const uint4*>(vp);
            pk[0] = x0.x, pk[1] = x0.y, pk[2] = x0.z, pk[3] = x0.w;
            pv[0] = x1.x, pv[1] = x1.y, pv[2] = x1.z, pv[3] = x1.w;
        }
        asm volatile("" ::: "memory");  // compiler only: the codes' loads stay behind the pairs'
        // lane = token 4 (col % 4) + col / 4, its part kq of every group
        const uint32_t ktok = 4 * (col & 3) + (col >> 2);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const uint4* cp = reinterpret_cast<const uint4*>(a.c.k + sub[st] * (HD / 2)) + (ktok * (HD / 32) + kq * (NG / 2));
#pragma unroll
            for (int i = 0; i < NG / 2; ++i) kw[st][i] = cp[i];
        }
    };
    auto load_values = [&]() __attribute__((always_inline)) {
        // lane = dims 4 col .. of every group, tokens 4 i + kq
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* cp = a.c.v + sub[st] * (HD / 2) + ((4 * i + kq) * (HD / 2) + col * NG * 2);
                if constexpr (NG == 2) vw[st][i][0] = *reinterpret_cast<const uint32_t*>(cp);
                else {
                    const uint2 u = *reinterpret_cast<const uint2*>(cp);
                    vw[st][i][0] = u.x;
                    vw[st][i][1] = u.y;
                }
            }
    };
    // (a wave without a step loads too, token 0's: a branch would make what
    // follows wait for every load)
    uint32_t id_next = entry(real(t0));

    // ---- the query: f16 parts scaled to a largest element in [2^10, 2^11)
    h8v qf[PQ][NG][2];
    float qsum[NG], cf;
    {
        float v[NG][16];
        const T* src = qp + (uint64_t)row * a.q_stride + (uint64_t)(hk * a.group + mg) * HD * (a.gated ? 2 : 1);
#pragma unroll
        for (int g = 0; g < NG; ++g) load16(src + 64 * g + 16 * kq, v[g]);
        asm volatile("" ::: "memory");  // compiler only: the step's loads stay behind the query's
        place(real(t0), id_next);
        load_keys();
        id_next = entry(real(t0 + NEXT));
        load_values();
        asm volatile("" ::: "memory");
        float mx = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(v[g][i]));
        mx = quarters_max(mx);
        const uint32_t e8 = min(max(__float_as_uint(mx) >> 23, 11u), 254u);
        const float up = __uint_as_float((264u - e8) << 23);
        cf = __uint_as_float((e8 - 10u) << 23) * a.scale;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float s = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x0 = v[g][8 * ks + j] * up, x1 = v[g][8 * ks + j + 4] * up;
                    s += x0 + x1;
                    if (j & 1) {
                        x0 *= 0.0625f;
                        x1 *= 0.0625f;
                    }
                    split_h2<PQ>(x0, x1, hi[j], lo[j]);
                }
                qf[0][g][ks] = __builtin_bit_cast(h8v, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                if (PQ > 1) qf[PQ - 1][g][ks] = __builtin_bit_cast(h8v, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            qsum[g] = quarters_sum(s);
        }
    }

    f4v o[NG][4];
    float ob[NG], l = 0.0f, mref = -INFINITY;
    const float least = least_size(V == Q4_PREFIX ? it.most : it.len);
    float bound = least;  // log2 of a bound of the value steps, uniform over the wave
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        ob[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][e] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto walk = [&](auto folded) __attribute__((always_inline)) {
        constexpr bool F = decltype(folded)::value;
        constexpr int XS = F ? 1 : NS;  // subtiles of a lane's scores
        auto sub = [&](int x) __attribute__((always_inline)) { return F ? cls : (uint32_t)x; };
#pragma unroll 1
        while (t0 < tend) {
            const uint32_t tr = real(t0);
            // ---- (s, b) through LDS: lane = token; what no row of the wave sees
            // is 0, and a pair that is not finite is kept out of the products.
            const bool out_of = (int32_t)(tr + tl) >= seen;
            float vmax = 0.0f, bmax = 0.0f;
            uint32_t odd = 0u;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t ck = out_of ? 0u : bad_l ? KV4_NAN_PAIR : pk[g], cv = out_of ? 0u : bad_l ? KV4_NAN_PAIR : pv[g];
                const float ksz = __uint_as_float(ck << 16);
                sm.pair[w].k[tl][g] = make_float2(ksz, fmaf(ksz, 8.0f, __uint_as_float(ck & 0xffff0000u)));
                float2 sb = make_float2(value_step(cv), 0.0f);
                sb.y = fmaf(sb.x, 8.0f, __uint_as_float(cv & 0xffff0000u));
                if (!(fabsf(sb.x) < INFINITY && fabsf(sb.y) < INFINITY)) {
                    odd |= 1u << g;
                    sb = make_float2(0.0f, 0.0f);
                }
                vmax = fmaxf(vmax, fabsf(sb.x));
                bmax = fmaxf(bmax, fabsf(sb.y));
                sm.pair[w].v[tl][g] = sb;
            }
            // log2 of a bound of the token's value steps (numerators rise as it
            // falls); the least steps need no bits
            const float size = fmaxf((float)(int32_t)(__float_as_uint(fmaxf(vmax, bmax * KV4_BIAS)) >> 23) - 126.0f, least);
            const bool some = vmax > 0x1p-120f;
            sm.pair[w].size[tl] = size;
            // one bound for the step where it serves every token
            bool spread = false;
            if (!__all(size <= bound && (!some || size >= bound - KV4_SPAN))) {
                const float hi = wave_max(size), lo = -wave_max(some ? -size : -1000.0f);
                bound = __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(hi)));
                spread = __any(lo < hi - KV4_SPAN);
            }
            wave_lds();

            // ---- scores, in powers of two
            float xs[XS][4];
            f4v own[NG];
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                f4v d[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint4 kk = kw[st][g / 2];
                    uint32_t w0 = g & 1 ? kk.z : kk.x, w1 = g & 1 ? kk.w : kk.y;
                    asm volatile("" : "+v"(w0), "+v"(w1));  // (else they are converted where they load)
                    const h8v f0 = codes_h8(w0, kc), f1 = codes_h8(w1, kc);
                    d[g] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = 0; q < PQ; ++q) {
                        d[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f0, qf[q][g][0], d[g], 0, 0, 0);
                        d[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f1, qf[q][g][1], d[g], 0, 0, 0);
                    }
                    if (NG > 2) __builtin_amdgcn_sched_barrier(0);
                }
                if (F) {  // its own subtile's of all
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i) own[g][i] = st == 0 || cls == (uint32_t)st ? d[g][i] : own[g][i];
                }
                if (!F || st == NS - 1) {
                    const int x = F ? 0 : st;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2* pr = sm.pair[w].k[16 * sub(x) + 4 * i + kq];
                        float s = 0.0f;
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            const float2 sb = pr[g];
                            s = fmaf(sb.x, F ? own[g][i] : d[g][i], s);
                            s = fmaf(sb.y, qsum[g], s);
                        }
                        xs[x][i] = s * cf;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            const uint32_t tn = t0 + NEXT;
            place(real(tn), id_next);
            load_keys();
            id_next = entry(real(tn + NEXT));
            asm volatile("" ::: "memory");
            // ---- what a row does not see
            if ((int32_t)(tr + STEP) > all_see) {
#pragma unroll
                for (int x = 0; x < XS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((int32_t)(tr + 16 * sub(x) + 4 * i) > p - (int32_t)kq) xs[x][i] = -INFINITY;
            }
            if (V == Q4_WINDOW && (int32_t)tr < seen - (int32_t)a.view.window && tr + STEP > a.view.sinks) {
#pragma unroll
                for (int x = 0; x < XS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t t = tr + 16 * sub(x) + 4 * i + kq;
                        if ((int32_t)t <= p - (int32_t)a.view.window && t >= a.view.sinks) xs[x][i] = -INFINITY;
                    }
            }
            if (V == Q4_ALL && any_mask) {
                const uint32_t hide = hidden(a, row, nblk, tr, kq, 4 * NS);
#pragma unroll
                for (int x = 0; x < XS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((hide >> (4 * sub(x) + i)) & 1u) xs[x][i] = -INFINITY;
            }
            // ---- pairs that are not finite: NaN for the rows that see them,
            // nothing for the others
            if (__any(odd != 0u)) {
                wave_lds();  // (the keys' pairs have been read)
                sm.pair[w].k[tl][0].x = __uint_as_float(odd);
                wave_lds();
#pragma unroll
                for (int x = 0; x < XS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t f = __float_as_uint(sm.pair[w].k[16 * sub(x) + 4 * i + kq][0].x);
#pragma unroll
                        for (int g = 0; g < NG; ++g)
                            if (((f >> g) & 1u) && xs[x][i] != -INFINITY) ob[g] = NAN;
                    }
            }
            // ---- the running reference: of score + log2 of the value step, so
            // that P s, what f16 has to hold, is at most 2^15 whatever the steps
            // are; moved where it would pass that
            float mx = -INFINITY;
            if (!spread) {
#pragma unroll
                for (int x = 0; x < XS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, xs[x][i]);
                mx += bound - LIFT;
            } else {  // (a row takes no account of a step that it does not see)
#pragma unroll
                for (int x = 0; x < XS; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, xs[x][i] + (sm.pair[w].size[16 * sub(x) + 4 * i + kq] - LIFT));
            }
            mx = quarters_max(mx);
            if (__any(mx > mref + TOP)) {
                const float mn = fmaxf(mx, mref);
                const float al = mref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mref - mn);
                mref = mn;
                l *= al;
                float ar[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) ar[i] = of_row(al, kq, i);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    ob[g] *= al;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[g][e][i] *= ar[i];
                }
            }
            const float msafe = mref == -INFINITY ? 0.0f : mref;
#pragma unroll
            for (int x = 0; x < XS; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    xs[x][i] = __builtin_amdgcn_exp2f(xs[x][i] - msafe);
                    l += xs[x][i];
                }

            // ---- P . V
            {
                uint32_t own2[PP][NG][2];  // folded: P s of the lane's subtile, two tokens a word
#pragma unroll
                for (int h = 0; h < NS / 2; ++h) {
#pragma unroll
                    for (int gp = 0; gp < NG; gp += 2) {  // two groups at a time
                        uint32_t pf[PP][2][4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {  // slot pairs: subtile 2h + j / 2, tokens 2 (j % 2), + 1
                            const int st = 2 * h + j / 2, i = 2 * (j % 2);
                            if (!F || (h == 0 && j < 2)) {
                                const int x = F ? 0 : st;
                                const float2* r0 = sm.pair[w].v[16 * sub(x) + 4 * i + kq] + gp;
                                const float2* r1 = sm.pair[w].v[16 * sub(x) + 4 * (i + 1) + kq] + gp;
                                const float p0 = xs[x][i], p1 = xs[x][i + 1];
#pragma unroll
                                for (int g = 0; g < 2; ++g) {
                                    const float2 s0 = r0[g], s1 = r1[g];
                                    const float u0 = p0 * s0.x, u1 = p1 * s1.x;
                                    ob[gp + g] = fmaf(p0, s0.y, ob[gp + g]);
                                    ob[gp + g] = fmaf(p1, s1.y, ob[gp + g]);
                                    uint32_t hi, lo = 0u;
                                    split_h2<PP>(u0, u1, hi, lo);
                                    if (F) {
                                        own2[0][gp + g][j] = hi;
                                        if (PP > 1) own2[PP - 1][gp + g][j] = lo;
                                    } else {
                                        pf[0][g][j] = hi;
                                        if (PP > 1) pf[PP - 1][g][j] = lo;
                                    }
                                }
                            }
                            if (F) {  // nothing for the other subtiles
#pragma unroll
                                for (int g = 0; g < 2; ++g)
#pragma unroll
                                    for (int q = 0; q < PP; ++q) pf[q][g][j] = cls == (uint32_t)st ? own2[q][gp + g][j % 2] : 0u;
                            }
                        }
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            uint32_t vh[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int st = 2 * h + j / 2, i = 2 * (j % 2);
                                vh[j] = __builtin_amdgcn_perm(vw[st][i + 1][gp / 2], vw[st][i][gp / 2], g ? 0x07060302u : 0x05040100u);
                                asm volatile("" : "+v"(vh[j]));  // (else every conversion moves up front)
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                uint32_t vf[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const uint32_t u = ((e & 2 ? vh[j] >> 8 : vh[j]) & (e & 1 ? kc.m2 : kc.m1)) | kc.magic;
                                    vf[j] = centred(u, e & 1);
                                }
                                const h8v vb = __builtin_bit_cast(h8v, make_uint4(vf[0], vf[1], vf[2], vf[3]));
#pragma unroll
                                for (int q = 0; q < PP; ++q)
                                    o[gp + g][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                        __builtin_bit_cast(h8v, make_uint4(pf[q][g][0], pf[q][g][1], pf[q][g][2], pf[q][g][3])),
                                        vb, o[gp + g][e], 0, 0, 0);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
            }
            wave_lds();
            load_values();
            t0 = tn;
        }
    };
    if constexpr (HD == 128) {
        if (fold) walk(std::true_type{});
        else walk(std::false_type{});
    } else walk(std::false_type{});

    // ---- the wave's numerators into LDS, its waves of the same rows joined
    l = quarters_sum(l);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        ob[g] = quarters_sum(ob[g]);
    }
    if (!solo) __syncthreads();
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float bias = of_row(ob[g], kq, i);
            *reinterpret_cast<float4*>(&sm.o[w][4 * kq + i][64 * g + 4 * col]) =
                make_float4(o[g][0][i] + bias, fmaf(o[g][1][i], 0.0625f, bias), o[g][2][i] + bias, fmaf(o[g][3][i], 0.0625f, bias));
        }
    if (kq == 0) sm.ml[w][col] = make_float2(mref, l);
    if (solo) wave_lds();
    else __syncthreads();
    const uint32_t rows = min(KV4_ROWS, cut.flat - m0);
    auto join = [&](auto alone, auto folded) __attribute__((always_inline)) {
        constexpr bool ALONE = decltype(alone)::value;
        constexpr uint32_t WAVES = ALONE ? 1u : KV4_WAVES;
        constexpr uint32_t COPIES = decltype(folded)::value ? NS : 1;  // rows ri, ri + FOLD, ..
        const uint32_t f0 = ALONE ? w : 0u;
        for (uint32_t i = ALONE ? lane : threadIdx.x; i < rows * (HD / 4); i += ALONE ? 64u : CHK_WG) {
            const uint32_t ri = i / (HD / 4), d = 4 * (i % (HD / 4));
            float2 ml[COPIES][WAVES];
            float M = -INFINITY;
#pragma unroll
            for (uint32_t c = 0; c < COPIES; ++c)
#pragma unroll
                for (uint32_t f = 0; f < WAVES; ++f) {
                    ml[c][f] = sm.ml[f0 + f][ri + c * FOLD];
                    M = fmaxf(M, ml[c][f].x);
                }
            float L = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t c = 0; c < COPIES; ++c)
#pragma unroll
                for (uint32_t f = 0; f < WAVES; ++f) {
                    const float wt = ml[c][f].x == M ? 1.0f : __builtin_amdgcn_exp2f(ml[c][f].x - M);
                    const float4 v = *reinterpret_cast<const float4*>(&sm.o[f0 + f][ri + c * FOLD][d]);
                    L = fmaf(ml[c][f].y, wt, L);
                    acc.x = fmaf(v.x, wt, acc.x);
                    acc.y = fmaf(v.y, wt, acc.y);
                    acc.z = fmaf(v.z, wt, acc.z);
                    acc.w = fmaf(v.w, wt, acc.w);
                }
            const uint32_t fm = m0 + ri;
            if (parts > 1 || (V == Q4_PREFIX && it.part)) {
                const uint32_t at = it.base + (z * a.c.nkv + hk) * cut.flat + fm;
                if (at < a.cap) {
                    *reinterpret_cast<float4*>(a.po + (size_t)at * HD + d) = acc;
                    if (d == 0) a.pml[at] = make_float2(M, L);
                }
            } else {
                const uint32_t ri2 = fm / a.group, h = hk * a.group + fm % a.group;
                finish<HD, T>(a, (uint64_t)it.s0 + ri2, h, d, acc, it.held ? L : NAN);
            }
        }
    };
    auto join_of = [&](auto folded) __attribute__((always_inline)) {
        if (V == Q4_PREFIX && solo) join(std::true_type{}, folded);
        else join(std::false_type{}, folded);
    };
    if constexpr (HD == 128) {
        if (fold) join_of(std::true_type{});
        else join_of(std::false_type{});
    } else join_of(std::false_type{});
}

}  // namespace chk
