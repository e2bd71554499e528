// Attention over the 4-bit cache where rows see a window of their sequence, or
// sequences share a prefix (kvq4.h): the blocks of attnq4.hip and attnq4_rows.hip over
// walks with a gap, of both kinds in one launch.
//
// Mathematics: as there; a softmax over a set of tokens is its parts' (maximum, sum,
// numerators) joined, whatever the parts are.  So a group's prefix is a part of each of
// its rows, taken for all of them at once, and a walk that leaves tiles out is the same
// sum without them.
//
// What bounds it, as measured.  Few rows: launches and first loads (one f32 row of 16 x 256
// through 2048 tokens: attention 11.7 us, its parts' join 4.5; four behind a prefix of 2048 plan 4.6,
// attention 12.9, join 4.3).  64 bf16 rows of 32 x 128: through windows of 1000 25 us, 2.8
// TB/s, half of it steps; behind 8192 common tokens 36.  Many rows: the vector unit, as there
// (two prompts of 8191 and 8092 rows through 1024 tokens 582 us, 0.46 PFLOP/s of the mathematics'
// operations; 78 f16 rows of 24 x 256 in two groups behind 30000 tokens 126, 0.37).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attnq4_join.h"
#include "attnq4_many.h"
#include "kvq4_host.h"

namespace chk {

// A call's walks with shared prefixes (Kv4Work) and the sums in which the launches
// behind this one find their items: one workgroup, of as many threads as the call has
// groups or sequences, up to two walks a thread.
//
// Latency bounds it: three loads deep and five barriers, and what lies between is a few
// hundred instructions of one wave (no division for a walk but the parts'; for the call, the
// share's and KV4_SHARED_SMALL's).
constexpr uint32_t Q4_PLAN_WG = 1024;

__global__ void __launch_bounds__(Q4_PLAN_WG) k_attn_q4_plan(AttnQ4Args a, uint32_t waves) {
    constexpr uint32_t WAVES = Q4_PLAN_WG / 64, MEMBER = 1u << 31, HELD = 1u << 30, MANY = 1u << 31;
    static_assert(Q4_PLAN_WG >= KV4_MAX_SEQS, "a sequence a thread");
    __shared__ struct {
        uint32_t s0[KV4_MAX_SEQS], n[KV4_MAX_SEQS], len[KV4_MAX_SEQS];  // n: with MEMBER and HELD
        uint32_t group[KV4_MAX_SEQS];
        uint32_t first[KV4_MAX_SEQS + 1], tokens[KV4_MAX_SEQS];
        Kv4Group g[KV4_MAX_SEQS];
        uint32_t shared[KV4_MAX_SEQS];  // tokens of a group's walk
        uint32_t blocks[2 * KV4_MAX_SEQS], tiles[2 * KV4_MAX_SEQS];  // of a walk; blocks with MANY
        unsigned long long cost[WAVES];
        uint32_t fits[KV4_TRIES], crowded[KV4_TRIES];
        uint32_t sum[Q4_KINDS + 1][WAVES];
    } sm;
    const uint32_t x = threadIdx.x, lane = x & 63, w = wave_id();
    const SeqLane own = seq_lane(a, x);
    const uint32_t small = KV4_SHARED_SMALL * a.groups / a.c.nkv;
    if (x < a.shared) {
        sm.first[x] = a.of_group[x];
        sm.tokens[x] = a.of_tokens[x];
    }
    if (x == 0 && a.shared) sm.first[a.shared] = a.of_group[a.shared];
    if (x < a.s.n) {
        sm.s0[x] = own.s0;
        sm.len[x] = own.len;
        sm.n[x] = own.n | (own.held ? HELD : 0u) | (kv4_member(own.n, own.len, own.held) ? MEMBER : 0u);
        sm.group[x] = KV4_NO_GROUP;
    }
    __syncthreads();
    // ---- a wave a group: what its members come to
    for (uint32_t g = w; g < a.shared; g += waves) {
        const uint32_t f0 = min(sm.first[g], a.s.n), f1 = min(max(sm.first[g + 1], f0), a.s.n);
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
            r.cost += lanes_sum32(in ? kv4_blocks_cost(n * a.group, n * a.group > KV4_FEW, a.shapes) : 0u);
        }
        if (lane == 0) {
            sm.g[g] = r;
            const Kv4Work k = kv4_group_work(r, sm.tokens[g], a.group, a.shapes, small);
            sm.shared[g] = k.n ? k.len : 0u;
        }
    }
    __syncthreads();
    // ---- the walks; what they cost, and so the parts
    const uint32_t nv = a.shared + a.s.n, per = nv > 64 * waves ? 2u : 1u;
    Kv4Work k[2];
    unsigned long long cost = 0ull;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t v = per * x + i;
        k[i] = kv4_no_work();
        if (i >= per || v >= nv) continue;
        if (v < a.shared) k[i] = kv4_group_work(sm.g[v], sm.tokens[v], a.group, a.shapes, small);
        else {
            const uint32_t b = v - a.shared, nb = sm.n[b];
            uint32_t g = sm.group[b];
            const uint32_t tokens = g != KV4_NO_GROUP ? sm.shared[g] : 0u;
            if (!tokens) g = KV4_NO_GROUP;
            k[i] = kv4_seq_work(b, sm.s0[b], nb & ~(MEMBER | HELD), sm.len[b], (nb & HELD) != 0u, a.group, g, tokens);
        }
        sm.blocks[v] = kv4_blocks(k[i].n * a.group, k[i].many, a.shapes) | (k[i].many ? MANY : 0u);
        sm.tiles[v] = kv4_work_most(k[i]);
        cost += kv4_work_cost(k[i], a.group, a.shapes) * (k[i].many ? KV4_MANY_COST : 1u);
    }
    cost = __any(cost >> 25) ? lanes_sum(cost) : lanes_sum32((uint32_t)cost);
    if (lane == 0) sm.cost[w] = cost;
    __syncthreads();
    cost = 0ull;
    for (uint32_t i = 0; i < waves; ++i) cost += sm.cost[i];
    const uint32_t share = (uint32_t)__builtin_amdgcn_readfirstlane((int)kv4_share_few(cost * a.c.nkv, a.groups, a.least));
    for (uint32_t i = w; i < KV4_TRIES; i += waves) {  // a wave a trial, up to one that fits
        const Kv4Share now = kv4_view_share(share, a.least, i);
        Kv4Trial t{0, 0, 0, 0};
        for (uint32_t v = lane; v < nv; v += 64) {
            const uint32_t blocks = sm.blocks[v];
            const Kv4Trial u = kv4_trial(blocks & MANY, blocks & ~MANY, sm.tiles[v], a.c.nkv, now);
            t.few += u.few;
            t.many += u.many;
            t.load += u.load;
            t.cut |= u.cut;
        }
        t.cut = __any(t.cut);
        t.few = lanes_sum32(t.few);
        t.many = lanes_sum32(t.many);
        t.load = lanes_sum32(t.load);
        const bool fits = kv4_fits(t, a.groups, now);
        if (lane == 0) {
            sm.fits[i] = fits ? 1u : 0u;
            sm.crowded[i] = kv4_crowded(t, a.groups) ? 1u : 0u;
        }
        if (fits) break;
    }
    __syncthreads();
    uint32_t tried = 0;
    while (tried < KV4_TRIES && !sm.fits[tried]) ++tried;
    if (tried == KV4_TRIES) tried = 0;
    const Kv4Share parts = kv4_view_share(share, a.least, tried);
    const bool crowded = sm.crowded[tried];
    // ---- sums over the walks: items of each kind, rows to join, partial rows
    uint32_t add[2][Q4_KINDS + 1], upto[Q4_KINDS + 1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        kv4_work_cut(k[i], parts, crowded, a.least);
        const uint32_t items = kv4_work_items(k[i], a.group, a.shapes, a.c.nkv);
        add[i][Q4_FEW] = k[i].many || k[i].solo ? 0u : items;
        add[i][Q4_SOLO] = k[i].solo ? items : 0u;
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
        if (w) {  // (the first wave's stand)
            const uint32_t t = wave_scan(lane < waves ? sm.sum[j][lane] : 0u);
            upto[j] += lane_value(t, w - 1);
        }
        upto[j] -= add[1][j];  // of the first of the two
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t v = per * x + i;
        if (i >= per || v >= nv) break;
#pragma unroll
        for (int j = 0; j < Q4_KINDS; ++j) a.upto[j * nv + v] = upto[j] + (i ? add[1][j] : 0u);
        k[i].base = upto[Q4_KINDS] - (i ? 0u : add[0][Q4_KINDS]);
        a.work[v] = k[i];
    }
}

template <int V>
static void launch_view(const AttnQ4Args& a, uint32_t hd, uint32_t dtype, const AttnQ4Launch& l, hipStream_t st) {
    if (V == Q4_PREFIX) {
        // a thread a group, a sequence and a walk (two where they are more than 1024)
        const uint32_t threads = std::min(a.shared + a.s.n, Q4_PLAN_WG);
        const uint32_t waves = (threads + 63) / 64;
        kv4_launch(k_attn_q4_plan, dim3(1), 64 * waves, st, a, waves);
    }
    kv4_switch(hd, dtype, [&](auto h, auto t) {
        constexpr int H = decltype(h)::value;
        using E = typename decltype(t)::type;
        constexpr int RB = H == 128 && std::is_same<E, __bf16>::value ? 2 : 1;
        kv4_launch(k_attn_q4_rows<H, E, RB, V>, dim3(l.few + l.many), CHK_WG, st, a);
        launch_join<H, E, V>(a, l, st);
    });
}
void launch_attn_q4_view(const AttnQ4Args& a, int view, uint32_t hd, uint32_t dtype, const AttnQ4Launch& l, hipStream_t st) {
    if (view == Q4_WINDOW) launch_view<Q4_WINDOW>(a, hd, dtype, l, st);
    else launch_view<Q4_PREFIX>(a, hd, dtype, l, st);
}

}  // namespace chk
