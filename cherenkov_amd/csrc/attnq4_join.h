// Parts of a row's attention joined.
#pragma once

#include "attnq4.h"
#include "kvq4_host.h"

namespace chk {

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
    uint32_t none;
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
            if (!plan.template find<Q4_JOIN>(x, it, none)) break;
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

template <int HD, class T, int V>
void launch_join(const AttnQ4Args& a, const AttnQ4Launch& l, hipStream_t st) {
    if (l.joins == 0) return;
    // split: HD / 64 workgroups a row; else a wave a run of rows
    const uint32_t runs = (l.joins + l.run - 1) / l.run;
    if (l.split) kv4_launch(k_attn_q4_join<HD, T, true, V>, dim3(l.joins * (HD / 64)), CHK_WG, st, a);
    else kv4_launch(k_attn_q4_join<HD, T, false, V>, dim3((runs + KV4_WAVES - 1) / KV4_WAVES), CHK_WG, st, a);
}

}  // namespace chk
