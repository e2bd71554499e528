// Causal attention over the 4-bit key/value cache (kvq4.h) for the rows of a
// batch of sequences, one to many rows each.
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

#include "attnq4.h"
#include "kvq4_host.h"

namespace chk {

template <int HD, class T, int V>
__global__ void __launch_bounds__(256, 2) k_attn_q4(AttnQ4Args a) {
    using Form = Q4Form<T>;
    constexpr int NG = HD / 64, PQ = Form::PQ, PP = Form::PP;
    // P s stays below 2^15 in f16 (and the least of a token 2^SPAN below the
    // largest keeps the bits that the parts have)
    constexpr float TOP = KV4_P_TOP;
    constexpr float LIFT = 15.0f - TOP;  // log2, taken off the reference
    constexpr int OROW = HD + 4;
    constexpr uint32_t STEP = q4_step(HD);
    constexpr int NS = STEP / 16;
    __shared__ union {
        struct {
            alignas(16) float2 k[STEP][NG];
            alignas(16) float2 v[STEP][NG];
            float size[STEP];
        } pair[KV4_WAVES];
        float o[KV4_WAVES][KV4_ROWS][OROW];
    } sm;
    __shared__ float2 sml[KV4_WAVES][KV4_ROWS];
    const uint32_t lane = threadIdx.x & 63, w = wave_id(), col = lane & 15, kq = lane >> 4;
    const Q4Consts kc;
    const Planner<V> plan(a, lane);
    const T* qp = (const T*)a.q;

    {
        Item it;
        if (!plan.template find<Q4_FEW>(blockIdx.x, it)) return;
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
        uint32_t t0 = z * per * KV4_TILE + w * STEP;
        constexpr uint32_t NEXT = KV4_WAVES * STEP;
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
        __syncthreads();
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float bias = of_row(ob[g], kq, i);
                *reinterpret_cast<float4*>(&sm.o[w][4 * kq + i][64 * g + 4 * col]) =
                    make_float4(o[g][0][i] + bias, fmaf(o[g][1][i], 0.0625f, bias), o[g][2][i] + bias, fmaf(o[g][3][i], 0.0625f, bias));
            }
        if (kq == 0) sml[w][col] = make_float2(mref, l);
        __syncthreads();
        const uint32_t rows = min(KV4_ROWS, cut.flat - m0);
        for (uint32_t i = threadIdx.x; i < rows * (HD / 4); i += CHK_WG) {
            const uint32_t ri = i / (HD / 4), d = 4 * (i % (HD / 4));
            const uint32_t ends = fold ? KV4_ROWS : ri + 1;  // folded: rows ri, ri + FOLD, ..
            float M = -INFINITY;
            for (uint32_t c = ri; c < ends; c += FOLD)
#pragma unroll
                for (uint32_t f = 0; f < KV4_WAVES; ++f) M = fmaxf(M, sml[f][c].x);
            float L = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t c = ri; c < ends; c += FOLD)
#pragma unroll
                for (uint32_t f = 0; f < KV4_WAVES; ++f) {
                    const float2 ml = sml[f][c];
                    const float wt = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
                    const float4 v = *reinterpret_cast<const float4*>(&sm.o[f][c][d]);
                    L = fmaf(ml.y, wt, L);
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
    }
}

// A running (maximum, sum, numerators) of parts of a row.
template <int E>
struct Joined {
    typedef float vec __attribute__((ext_vector_type(E)));
    float M, L;
    vec acc;
    CHK_DEV void add(float m, float l, vec v) {
        const float mn = fmaxf(M, m);
        const float w0 = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - mn), w1 = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        M = mn;
        L = fmaf(l, w1, L * w0);
        acc = acc * w0 + v * w1;
    }
};

// Joins the parts of a row; a row of partial numerators is hd floats.
//   SPLIT: few rows of many parts: a workgroup takes 64 dims of a row, each of
//       its sixteen teams of sixteen lanes every sixteenth part (a compute unit
//       reads some 130 GB/s: 125 parts of a row by one took 11 us of 15);
//   else a wave takes a row, HD / 64 dims a lane.
template <int HD, class T, bool SPLIT, int V>
__global__ void __launch_bounds__(256) k_attn_q4_join(AttnQ4Args a) {
    constexpr int E = SPLIT ? 4 : HD / 64, U = 8;
    constexpr uint32_t TEAM = SPLIT ? 16 : 64, TEAMS = SPLIT ? CHK_WG / TEAM : 1, PIECES = SPLIT ? HD / 64 : 1;
    typedef typename Joined<E>::vec Vec;
    __shared__ Joined<E> sm[KV4_WAVES][TEAM];
    const uint32_t lane = threadIdx.x & 63, w = wave_id();
    const Planner<V> plan(a, lane);
    const uint32_t team = threadIdx.x / TEAM, d = (SPLIT ? blockIdx.x % PIECES * 64 : 0u) + E * (lane % TEAM);
    // items of a wave (of the workgroup, SPLIT): a.run consecutive rows, one
    // sequence's looked up once
    const uint32_t x0 = (SPLIT ? blockIdx.x / PIECES : blockIdx.x * KV4_WAVES + w) * a.run;
    Item it, pre;       // pre: the prefix that the sequence's group has taken
    uint32_t left = 0;  // rows of the sequence behind this one
    for (uint32_t x = x0; x < x0 + a.run; ++x) {
        if (left) {
            --left;
            ++it.local;
        } else {
            // (waves with rows of their own leave one by one: nothing waits)
            if (!plan.template find<Q4_JOIN>(x, it)) break;
            if constexpr (V == Q4_PREFIX)
                if (it.group != KV4_NO_GROUP) plan.load(it.group, pre);
            left = it.cut.flat * a.c.nkv - 1 - it.local;
        }
        const uint32_t flat = it.cut.flat, stride = a.c.nkv * flat, hk = it.local / flat, m = it.local % flat;
        const uint32_t m1 = min((m / it.cut.block + 1) * it.cut.block, flat) - 1;  // of the row's block, the last
        int32_t see;
        const uint32_t own = kv4_parts(V == Q4_ALL ? kv4_tiles(kv4_seen(it.len, it.n, a.group, m1))
                                                   : walk_of<V>(a, it, m / it.cut.block * it.cut.block, m1, see).tiles, it.cut.piece);
        if (own == 1 && !(V == Q4_PREFIX && it.part)) continue;  // written whole
        const uint32_t first = it.base + it.local;  // local = hk flat + m
        // parts: the sequence's own, then its prefix's
        uint32_t parts = own, first2 = 0u, stride2 = 0u;
        if (V == Q4_PREFIX && it.group != KV4_NO_GROUP) {
            parts += kv4_parts(kv4_tiles((int32_t)pre.len), pre.cut.piece);
            stride2 = a.c.nkv * pre.cut.flat;
            first2 = pre.base + hk * pre.cut.flat + (it.s0 - pre.s0) * a.group + m;
        }
        const uint64_t row = (uint64_t)it.s0 + m / a.group;
        const uint32_t h = hk * a.group + m % a.group;
        T gate[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            gate[j] = a.gated ? ((const T*)a.q)[row * a.q_stride + (uint64_t)h * HD * 2 + HD + d + j] : (T)0.0f;
        Joined<E> r;
        r.M = -INFINITY;
        r.L = 0.0f;
        r.acc = 0.0f;
        for (uint32_t z = SPLIT ? team : 0u; z < parts; z += TEAMS * U) {
            Vec v[U];
            float2 ml[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t y = min(z + u * TEAMS, parts - 1);
                const uint32_t at = min(V == Q4_PREFIX && y >= own ? first2 + (y - own) * stride2 : first + y * stride, a.cap - 1);
                v[u] = *reinterpret_cast<const Vec*>(a.po + (size_t)at * HD + d);
                ml[u] = a.pml[at];
            }
            float mb = r.M;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (z + u * TEAMS < parts) mb = fmaxf(mb, ml[u].x);
            const float w0 = r.M == mb ? 1.0f : __builtin_amdgcn_exp2f(r.M - mb);
            r.M = mb;
            r.L *= w0;
            r.acc *= w0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (z + u * TEAMS >= parts) break;
                const float wt = ml[u].x == mb ? 1.0f : __builtin_amdgcn_exp2f(ml[u].x - mb);
                r.L = fmaf(ml[u].y, wt, r.L);
                r.acc += v[u] * wt;
            }
        }
        if (SPLIT) {
            // the wave's four teams, then the four waves
#pragma unroll
            for (int o = 16; o < 64; o *= 2) {
                Vec v;
#pragma unroll
                for (int j = 0; j < E; ++j) v[j] = __shfl_xor(r.acc[j], o, 64);
                const float m2 = __shfl_xor(r.M, o, 64), l2 = __shfl_xor(r.L, o, 64);
                r.add(m2, l2, v);
            }
            if (lane < TEAM) sm[w][lane] = r;
            __syncthreads();
            if (threadIdx.x < TEAM) {
#pragma unroll
                for (uint32_t i = 1; i < KV4_WAVES; ++i) r.add(sm[i][lane].M, sm[i][lane].L, sm[i][lane].acc);
            }
            __syncthreads();
        }
        if (!SPLIT || threadIdx.x < TEAM) {
            const float inv = r.L == 0.0f ? 0.0f : 1.0f / r.L;
            T* op = (T*)a.out + row * a.out_stride + (uint64_t)h * HD + d;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                float v = r.acc[j] * inv;
                if (a.gated) v *= sigmoidf_((float)gate[j]);
                op[j] = (T)v;
            }
        }
    }
}

// A call's walks with shared prefixes (Kv4Work) and the sums in which the launches
// behind this one find their items: one workgroup, two walks a thread.
constexpr uint32_t Q4_PLAN_WG = 1024;

__global__ void __launch_bounds__(Q4_PLAN_WG) k_attn_q4_plan(AttnQ4Args a) {
    constexpr uint32_t WAVES = Q4_PLAN_WG / 64, MEMBER = 1u << 31, HELD = 1u << 30;
    static_assert(Q4_PLAN_WG >= KV4_MAX_SEQS, "a sequence a thread");
    __shared__ struct {
        uint32_t s0[KV4_MAX_SEQS], n[KV4_MAX_SEQS], len[KV4_MAX_SEQS];  // n: with MEMBER and HELD
        uint32_t group[KV4_MAX_SEQS];
        Kv4Group g[KV4_MAX_SEQS];
        uint32_t shared[KV4_MAX_SEQS];  // tokens of a group's walk
        unsigned long long cost[2];     // of few and of many pairs
        uint32_t sum[Q4_KINDS + 1][WAVES];
    } sm;
    const uint32_t x = threadIdx.x, lane = x & 63, w = wave_id();
    const SeqLane own = seq_lane(a, x);
    if (x < 2) sm.cost[x] = 0ull;
    if (x < a.s.n) {
        sm.s0[x] = own.s0;
        sm.len[x] = own.len;
        sm.n[x] = own.n | (own.held ? HELD : 0u) | (kv4_member(own.n, own.len, own.held) ? MEMBER : 0u);
        sm.group[x] = KV4_NO_GROUP;
    }
    __syncthreads();
    // ---- a wave a group: what its members come to
    for (uint32_t g = w; g < a.shared; g += WAVES) {
        const uint32_t f0 = min(a.of_group[g], a.s.n), f1 = min(max(a.of_group[g + 1], f0), a.s.n);
        Kv4Group r{0u, 0u, 0xffffffffu, 0u, 0xffffffffu, 0u, 0u};
        for (uint32_t c0 = f0; c0 < f1; c0 += 64) {
            const uint32_t b = min(c0 + lane, f1 - 1), nb = sm.n[b], n = nb & ~(MEMBER | HELD), len = sm.len[b];
            const bool in = c0 + lane < f1 && (nb & MEMBER);
            if (in) sm.group[b] = g;
            const uint64_t any = __ballot(in);
            if (!any) continue;
            if (!r.members) r.lead = c0 + (uint32_t)__builtin_ctzll(any);
            r.members += (uint32_t)__builtin_popcountll(any);
            r.s0 = min(r.s0, ~wave_top(in ? ~sm.s0[b] : 0u));
            r.s1 = max(r.s1, wave_top(in ? sm.s0[b] + n : 0u));
            r.least = min(r.least, ~wave_top(in ? ~(len - n + 1) : 0u));
            r.most = max(r.most, wave_top(in ? len : 0u));
            r.blocks += lane_value(wave_scan(in ? kv4_blocks(n * a.group, n * a.group > KV4_FEW, a.block) : 0u), 63);
        }
        if (lane == 0) {
            sm.g[g] = r;
            const Kv4Work k = kv4_group_work(r, a.of_tokens[g], a.group, a.block);
            sm.shared[g] = k.n ? k.len : 0u;
        }
    }
    __syncthreads();
    // ---- the walks, two a thread; what they cost, and so the parts
    const uint32_t nv = a.shared + a.s.n;
    Kv4Work k[2];
    unsigned long long cost[2] = {0ull, 0ull};
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t v = 2 * x + i;
        if (v >= nv) k[i] = kv4_no_work();
        else if (v < a.shared) k[i] = kv4_group_work(sm.g[v], a.of_tokens[v], a.group, a.block);
        else {
            const uint32_t b = v - a.shared, nb = sm.n[b];
            uint32_t g = sm.group[b];
            const uint32_t tokens = g != KV4_NO_GROUP ? sm.shared[g] : 0u;
            if (!tokens) g = KV4_NO_GROUP;
            k[i] = kv4_seq_work(b, sm.s0[b], nb & ~(MEMBER | HELD), sm.len[b], (nb & HELD) != 0u, a.group, g, tokens);
        }
        (k[i].many ? cost[1] : cost[0]) += kv4_work_cost(k[i], a.group, a.block);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (cost[i]) atomicAdd(&sm.cost[i], cost[i]);
    __syncthreads();
    const Kv4Share share{kv4_share_few(sm.cost[0] * a.c.nkv, a.groups, a.least), kv4_share(sm.cost[1] * a.c.nkv, a.groups, 2)};
    // ---- sums over the walks: items of each kind, rows to join, partial rows
    uint32_t add[2][Q4_KINDS + 1], upto[Q4_KINDS + 1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        kv4_work_cut(k[i], a.group, share);
        const uint32_t items = kv4_work_items(k[i], a.group, a.block, a.c.nkv);
        add[i][Q4_FEW] = k[i].many ? 0u : items;
        add[i][Q4_MANY] = k[i].many ? items : 0u;
        add[i][Q4_JOIN] = kv4_work_joins(k[i], a.group, a.c.nkv);
        add[i][Q4_KINDS] = kv4_work_partials(k[i], a.group, a.c.nkv);
    }
#pragma unroll
    for (int j = 0; j <= Q4_KINDS; ++j) {
        upto[j] = wave_scan(add[0][j] + add[1][j]);
        if (lane == 63) sm.sum[j][w] = upto[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j <= Q4_KINDS; ++j) {
        const uint32_t t = wave_scan(lane < WAVES ? sm.sum[j][lane] : 0u);
        upto[j] += (w ? lane_value(t, w - 1) : 0u) - add[1][j];  // of the first of the two
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t v = 2 * x + i;
        if (v >= nv) break;
#pragma unroll
        for (int j = 0; j < Q4_KINDS; ++j) a.upto[j * nv + v] = upto[j] + (i ? add[1][j] : 0u);
        k[i].base = upto[Q4_KINDS] - (i ? 0u : add[0][Q4_KINDS]);
        a.work[v] = k[i];
    }
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
struct AttnQ4Launch {
    uint32_t few, many;    // workgroups (many: 0 where no sequence can have many pairs)
    uint32_t joins, run;   // rows that may have parts, and how many of them a wave takes
    bool split;
};
// tokens: the most that a row's walk may be over; block: pairs of a many-pairs block; least:
// least tiles of a few-pairs part; cap: partial rows of the workspace.
static AttnQ4Launch attn_launch(const AttnQ4Shape& s, uint64_t tokens, uint32_t block, uint32_t least, uint64_t cap) {
    AttnQ4Launch l{};
    const uint64_t flat = (uint64_t)s.rows * s.group, tiles = (tokens + KV4_TILE - 1) / KV4_TILE;
    // A workgroup for every part, as many as there can be: parts < tiles / piece
    // + 1, so one for each block and `groups` more of the sequences with few
    // pairs, 2 groups of those with many (whose cost may be half of their tiles);
    // nor are there more parts than pieces of a full table.  The rest find
    // nothing and end.
    uint64_t few = std::min(flat / KV4_ROWS + s.n, (uint64_t)s.n * (KV4_FEW / KV4_ROWS));
    uint64_t many = flat > KV4_FEW ? flat / block + std::min((uint64_t)s.n, flat / (KV4_FEW + 1)) : 0;
    if (s.shared) {  // a block for a group with few, and the groups' rows once more
        few += s.shared;
        if (flat > KV4_SHARED_FEW) many += flat / block + std::min((uint64_t)s.shared, flat / (KV4_SHARED_FEW + 1));
    }
    few *= s.nkv;
    many *= s.nkv;
    l.few = (uint32_t)std::min(few + s.groups, few * std::max<uint64_t>((tiles + least - 1) / least, 1));
    if (many) l.many = (uint32_t)std::min(many + 2 * s.groups, many * std::max<uint64_t>((tiles + 1) / 2, 1));
    // a row with parts has two at least
    l.joins = (uint32_t)std::min<uint64_t>(flat * s.nkv, cap / 2 + 1);
    // rows that give the device fewer waves than it has are read by a team of
    // lanes a part; else a wave takes one row, or as many as leave the device 8
    // waves a SIMD (16384 rows of two parts: 23.7 us with one, 19.9 with two)
    l.split = l.joins <= 2 * s.groups;
    l.run = l.split ? 1u : (l.joins + 16 * s.groups - 1) / (16 * s.groups);
    return l;
}

static Kv4Window window_arg(uint32_t window, uint32_t sinks) {
    kv4_ensure(window >= 1, "a window has at least one token");
    // (past a table's 2^30 tokens every window is the same)
    return Kv4Window{std::min(window, 1u << 30), std::min(sinks, 1u << 30)};
}
// The most tokens that a block's walk through a window is over, in whole tiles.
static uint64_t window_tokens(uint64_t tokens, uint32_t group, uint32_t block, Kv4Window v) {
    return (uint64_t)kv4_window_most((uint32_t)tokens, group, block, v) * KV4_TILE;
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
static void attn_call(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const AttnQ4Rows& r, const ChkKvMask* mask, Kv4Window window,
                      const ChkKvShared* shared, void* stream) {
    const char* small = V == Q4_PREFIX ? "workspace smaller than chk_attn_prefix_q4_workspace says"
                                       : "workspace smaller than chk_attn_q4_workspace says";
    AttnQ4Args a{};
    a.c = kv4_cache(cache);
    a.s = kv4_seqs(cache, seqs);
    kv4_dtype(r.dtype);
    check_heads(r.nh, cache->nkv, cache->hd, a.s.n);
    if (V == Q4_WINDOW) a.view = window_arg(window.window, window.sinks);
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
    if (V == Q4_WINDOW) tokens = window_tokens(tokens, a.group, a.block, a.view);
    const AttnQ4Launch l = attn_launch(s, tokens, a.block, a.least, cap);
    a.run = l.run;
    if (V == Q4_PREFIX) kv4_launch(k_attn_q4_plan, dim3(1), Q4_PLAN_WG, st, a);
    if (l.many) launch_attn_q4_many(a, V, cache->hd, r.dtype, l.many, st);
    kv4_switch(cache->hd, r.dtype, [&](auto hd, auto t) {
        constexpr int H = decltype(hd)::value;
        using E = typename decltype(t)::type;
        kv4_launch(k_attn_q4<H, E, V>, dim3(l.few), CHK_WG, st, a);
        // split: HD / 64 workgroups a row; else a wave a run of rows
        const uint32_t runs = (l.joins + l.run - 1) / l.run;
        if (l.split) kv4_launch(k_attn_q4_join<H, E, true, V>, dim3(l.joins * (H / 64)), CHK_WG, st, a);
        else kv4_launch(k_attn_q4_join<H, E, false, V>, dim3((runs + KV4_WAVES - 1) / KV4_WAVES), CHK_WG, st, a);
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
static void launch_sizes(const AttnQ4Shape& s, uint64_t tokens, uint32_t block, uint32_t least, uint64_t* launch) {
    const uint64_t cap = partial_rows(s);
    const AttnQ4Launch l = attn_launch(s, tokens, block, least, cap);
    launch[0] = cap;
    launch[1] = l.few;
    launch[2] = l.many;
    launch[3] = l.joins;
}

// view: null where rows see everything before them
static void cut_call(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t dtype, uint32_t groups, uint32_t n, uint32_t rows,
                     uint64_t tokens, const uint32_t* len, const uint32_t* start, const Kv4Window* view, uint32_t* cut,
                     uint64_t* launch) {
    cut_args(nh, nkv, hd, dtype, groups, n, rows, tokens, len, start, cut, launch);
    const auto held = [&](uint32_t b) { return len[b] <= tokens ? len[b] : 0u; };  // as the kernels take it
    const uint32_t group = nh / nkv, block = attn_q4_block(hd, dtype), least = KV4_WAVES * q4_step(hd) / KV4_TILE;
    Kv4Share share;
    uint64_t sum[2] = {0, 0};
    for (uint32_t b = 0; b < n; ++b) {
        uint32_t s0, s1;
        kv4_rows(start, b, rows, s0, s1);
        sum[(s1 - s0) * group > KV4_FEW] += view ? kv4_window_cost(held(b), s1 - s0, group, block, *view)
                                                 : kv4_cost(held(b), s1 - s0, group, block);
    }
    share.few = kv4_share_few(sum[0] * nkv, groups, least);
    share.many = kv4_share(sum[1] * nkv, groups, 2);
    for (uint32_t b = 0; b < n; ++b) {
        uint32_t s0, s1;
        kv4_rows(start, b, rows, s0, s1);
        const Kv4Cut c = view ? kv4_window_cut(held(b), s1 - s0, group, block, share, *view)
                              : kv4_cut(held(b), s1 - s0, group, block, share);
        cut[4 * b] = c.block;
        cut[4 * b + 1] = c.blocks;
        cut[4 * b + 2] = c.piece;
        cut[4 * b + 3] = c.parts;
    }
    launch_sizes({group, nkv, hd, n, rows, groups, 0, false}, view ? window_tokens(tokens, group, block, *view) : tokens, block,
                 least, launch);
}

}  // namespace chk

using namespace chk;

extern "C" {

int chk_attn_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated, uint32_t dtype,
                uint64_t q_stride, const ChkKvMask* mask, void* out, uint64_t out_stride, void* ws, uint64_t ws_bytes,
                void* stream) {
    return kv4_try([&] {
        attn_call<Q4_ALL>(cache, seqs, {q, nh, gated, dtype, q_stride, out, out_stride, ws, ws_bytes}, mask, {}, nullptr, stream);
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
                             {window, sinks}, nullptr, stream);
    });
}

int chk_attn_prefix_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated, uint32_t dtype,
                       uint64_t q_stride, const ChkKvShared* shared, void* out, uint64_t out_stride, void* ws,
                       uint64_t ws_bytes, void* stream) {
    return kv4_try([&] {
        attn_call<Q4_PREFIX>(cache, seqs, {q, nh, gated, dtype, q_stride, out, out_stride, ws, ws_bytes}, nullptr, {}, shared,
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
        const Kv4Window v = window_arg(window, sinks);
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
                r.blocks += kv4_blocks(q.n * group, q.n * group > KV4_FEW, block);
            }
            work.push_back(kv4_group_work(r, shared->tokens[g], group, block));
        }
        for (uint32_t b = 0; b < n; ++b) {
            const Seq& q = seqs[b];
            const uint32_t g = of[b], t = g != KV4_NO_GROUP && work[g].n ? work[g].len : 0u;
            work.push_back(kv4_seq_work(b, q.s0, q.n, q.len, q.held, group, t ? g : KV4_NO_GROUP, t));
        }
        uint64_t cost[2] = {0, 0};
        for (const Kv4Work& k : work) cost[k.many] += kv4_work_cost(k, group, block);
        const Kv4Share share{kv4_share_few(cost[0] * nkv, groups, least), kv4_share(cost[1] * nkv, groups, 2)};
        uint32_t* to = walks;
        for (Kv4Work& k : work) {
            kv4_work_cut(k, group, share);
            const uint32_t w[8] = {k.s0, k.n, k.len, k.lo, k.group, k.many ? block : KV4_ROWS, k.piece, k.parts};
            to = std::copy(w, w + 8, to);
        }
        launch_sizes({group, nkv, hd, n, rows, groups, shared->groups, true}, tokens, block, least, launch);
    });
}

}  // extern "C"
