// The norm of each query and key head and its rotation, rows of a batch.
//
//   y = x / sqrt(mean(x^2) + eps) * w,   (y_j, y_{j + r/2}) turned by pos * turn_j
// for the first r dims of a head (norm_rope of attn.hip, for 16-bit rows too,
// rows of any batch, and angles that stay exact at far positions).
//
// The angle.  turn_j is in 2^-64 of a turn, so pos turn_j modulo 2^64 is the
// angle, and its upper word is enough: one 32-bit product and one upper half.
// The quarter of the circle nearest to it is taken off in integers; what is left, an
// integer of at most 2^29, is rounded to f32, to 2^-24 of itself, as are its factor and
// their product, an angle of at most pi / 4; Taylor's sums of degree 9 and 10 end 2e-9
// and 1e-10 from sine and cosine.
//
// One pass over memory, bound by it.  A lane takes 16 bytes of a head, 8 or 4
// dims, so a head is 8 to 64 lanes, its sum of squares a few row operations, and
// a wave takes a row's heads, 64 / (lanes a head) at a time: a piece.  A row's angles are
// computed once, one a lane, and read back from LDS in the lane's order; a dim's
// partner comes by lane permutes, or through LDS where half the turned dims do
// not fill whole lanes.
//
// What it took to be bound by memory (16389 bf16 rows of 32 + 8 x 128, 336 MB; a
// large copy needs 65 us): the vector unit's work and a wave's start.  Angles for
// every lane's own dims, weights selected head by head and the norm ahead of
// the turn took 78 us; waves of one row each, weights read again for every row,
// 80; waves that go from row to row with weights in registers and the next
// piece's load in flight, factors as above, 63, 5.3 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "kernels_internal.h"
#include "kvq4_host.h"

namespace chk {

struct QkArgs {
    const void *q, *k;
    void *q_out, *k_out;
    uint64_t q_stride, q_out_stride, k_stride, k_out_stride;  // elements
    const uint16_t *q_norm, *k_norm;
    const uint64_t* turn;
    const uint32_t* pos;
    uint32_t rows, nh, nkv, gated, gates;  // gates: heads whose gate is copied
    uint32_t half;                         // turned pairs of a head
    uint32_t waves, row_step;              // of a row; rows at once
    float eps;
};

// cos and sin of `turns` in 2^-32 of a turn.
CHK_DEV float2 turned(uint32_t turns) {
    const uint32_t quarter = (turns + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(turns - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
    const float x2 = x * x;
    const float s = x * fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float c = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
    return make_float2((quarter + 1) & 2 ? -u : u, quarter & 2 ? -v : v);
}

// A piece: 16 bytes a lane of 64 / LANES heads.
template <int HD, class T>
struct QkPiece {
    static constexpr int N = 16 / sizeof(T), LANES = HD / N, HEADS = 64 / LANES;
    typedef T vec __attribute__((ext_vector_type(N)));
};

// A wave takes every a.waves-th piece of every a.row_step-th row, the next one's
// load in flight, across its rows.  With weight and angle of a dim folded into one
// factor for the dim and one for its partner, a piece is, past its sum of squares,
// (x inv) cw + (x' inv) sw (normed first: x cw may be past f32 where that is not); the factors of a row's queries and keys wait in LDS, the
// partner x' comes as it was loaded, four permutes a lane.
template <int HD, class T, bool NT>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkArgs a) {
    typedef QkPiece<HD, T> P;
    typedef typename P::vec Vec;
    typedef uint32_t u4v __attribute__((ext_vector_type(4)));
    constexpr int N = P::N, PAIRS = (HD / 2 + 63) / 64;  // turned pairs of a lane
    __shared__ struct {
        alignas(16) float2 f[2][HD];  // (cw, sw) of queries and keys
        float line[64 * N];
    } sm[CHK_WG / 64];
    const uint32_t lane = threadIdx.x & 63, w = wave_id();
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * (CHK_WG / 64) + w));
    const uint32_t share = wave % a.waves, half = a.half;
    uint32_t row = wave / a.waves;
    const uint32_t pq = (a.nh + P::HEADS - 1) / P::HEADS, pk = (a.nkv + P::HEADS - 1) / P::HEADS;
    const uint32_t pieces = pq + pk + (a.gates + P::HEADS - 1) / P::HEADS;
    // (the last workgroup's waves past the rows at once)
    if (row >= min(a.rows, a.row_step)) return;
    const uint32_t d0 = lane % P::LANES * N, sub = lane / P::LANES;
    const uint32_t wide = a.gated ? 2 * HD : HD;
    auto& L = sm[w];

    // piece p of row r: its first element for this lane; the heads of its kind that
    // are left there (a lane past them repeats the last)
    auto place = [&](uint32_t r, uint32_t p, const void* q, const void* k, uint64_t qs, uint64_t ks, uint32_t& left) __attribute__((always_inline)) {
        const bool is_k = p >= pq && p < pq + pk, is_gate = p >= pq + pk;
        const uint32_t h = (p - (is_k ? pq : is_gate ? pq + pk : 0u)) * P::HEADS;
        left = (is_k ? a.nkv : a.nh) - h;
        const uint32_t apart = is_k ? HD : wide;
        const T* base = (is_k ? (const T*)k + r * ks : (const T*)q + r * qs) + (size_t)h * apart + (is_gate ? HD : 0);
        return base + (min(sub, left - 1) * apart + d0);
    };
    auto load = [&](uint32_t r, uint32_t p) __attribute__((always_inline)) {
        uint32_t left;
        return *reinterpret_cast<const Vec*>(place(min(r, a.rows - 1), p, a.q, a.k, a.q_stride, a.k_stride, left));
    };
    // the next item to load
    uint32_t lr = row, lp = share;
    auto next = [&](uint32_t& r, uint32_t& p) __attribute__((always_inline)) {
        p += a.waves;
        if (p >= pieces) {
            p = share;
            r += a.row_step;
        }
    };
    uint32_t pos = a.pos[row];
    Vec x = load(lr, lp);
    next(lr, lp);
    // ---- weights and turns of this lane's pairs; factors of the dims that are not turned
    float wt[2][PAIRS][2];
    uint64_t turn[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const uint32_t j = lane + 64 * i;
        turn[i] = j < half ? a.turn[j] : 0u;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint16_t* g = k ? a.k_norm : a.q_norm;
            wt[k][i][0] = g && j < half ? bf16f(g[j]) : 1.0f;
            wt[k][i][1] = g && j < half ? bf16f(g[j + half]) : 1.0f;
        }
    }
    for (uint32_t d = 2 * half + lane; d < HD; d += 64) {
        L.f[0][d] = make_float2(a.q_norm ? bf16f(a.q_norm[d]) : 1.0f, 0.0f);
        L.f[1][d] = make_float2(a.k_norm ? bf16f(a.k_norm[d]) : 1.0f, 0.0f);
    }
    // half in whole lanes: a partner is a lane's same element
    const bool whole = half % N == 0, turns = d0 < 2 * half;
    const int mate = whole && turns ? (int)lane + (d0 < half ? (int)(half / N) : -(int)(half / N)) : (int)lane;

    uint32_t p = share;
    bool fresh = true;
    while (row < a.rows) {
        if (fresh) {  // the row's angles, one a lane
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const uint32_t j = lane + 64 * i;
                if (j < half) {
                    const float2 c = turned(__umulhi(pos, (uint32_t)turn[i]) + pos * (uint32_t)(turn[i] >> 32));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        L.f[k][j] = make_float2(c.x * wt[k][i][0], -c.y * wt[k][i][1]);
                        L.f[k][j + half] = make_float2(c.x * wt[k][i][1], c.y * wt[k][i][0]);
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            fresh = false;
        }
        const uint32_t kind = p < pq ? 0u : p < pq + pk ? 1u : 2u;
        Vec r = x;
        x = load(lr, lp);
        next(lr, lp);
        if (kind != 2u) {
            float y[N], ss = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                y[i] = (float)r[i];
                ss = fmaf(y[i], y[i], ss);
            }
            float inv = 1.0f;
            if (kind ? a.k_norm : a.q_norm) inv = __builtin_amdgcn_rsqf(fmaf(group_sum<P::LANES>(ss), 1.0f / HD, a.eps));
            float o[N];
            if (whole) {
                const u4v raw = __builtin_bit_cast(u4v, r);
                u4v other;
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // (what is not turned takes nothing from a dim that may be infinite)
                    const uint32_t v = (uint32_t)__shfl((int)raw[i], mate, 64);
                    other[i] = turns ? v : 0u;
                }
                const Vec xo = __builtin_bit_cast(Vec, other);
#pragma unroll
                for (int i = 0; i < N; ++i) o[i] = (float)xo[i];
            } else {
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < N; ++i) L.line[lane * N + i] = y[i];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                const uint32_t head = lane * N - d0;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t d = d0 + i;
                    o[i] = d < 2 * half ? L.line[head + (d < half ? d + half : d - half)] : 0.0f;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float4 f = *reinterpret_cast<const float4*>(&L.f[kind][d0 + i]);
                r[i] = (T)fmaf(o[i] * inv, f.y, y[i] * inv * f.x);
                r[i + 1] = (T)fmaf(o[i + 1] * inv, f.w, y[i + 1] * inv * f.z);
            }
        }
        uint32_t left;
        Vec* to = reinterpret_cast<Vec*>(const_cast<T*>(place(row, p, a.q_out, a.k_out, a.q_out_stride, a.k_out_stride, left)));
        if (sub < left && pos != 0xffffffffu) {
            if (NT) __builtin_nontemporal_store(r, to);
            else *to = r;
        }
        const uint32_t was = row;
        next(row, p);
        if (row != was) {
            fresh = true;
            pos = row < a.rows ? a.pos[row] : 0u;
        }
    }
}

template <int HD, class T>
static void launch_qk(QkArgs& a, hipStream_t st) {
    typedef QkPiece<HD, T> P;
    const uint32_t pieces = (a.nh + P::HEADS - 1) / P::HEADS + (a.nkv + P::HEADS - 1) / P::HEADS + (a.gates + P::HEADS - 1) / P::HEADS;
    // Six waves a SIMD: rows that give fewer with two waves each take more, up to
    // a wave a piece (333 f16 rows of 24 + 2 x 256: 11.8 us with one, 6.0 with
    // three, 5.4 with all thirteen; 16389 bf16 rows of 32 + 8 x 128 64.6 with one
    // or all ten, 63.1 with two).
    const uint32_t waves = 6 * 4 * kv4_cus();
    a.waves = std::min(std::max((waves + a.rows - 1) / a.rows, 2u), pieces);
    a.row_step = std::max(1u, std::min(a.rows, waves / a.waves));
    const dim3 groups((uint32_t)(((uint64_t)a.row_step * a.waves + CHK_WG / 64 - 1) / (CHK_WG / 64)));
    // rows that the caches would not hold until they are read go out past them
    // (16389 bf16 rows: 63 us against 69; f32 2048: 25.5 against 27)
    const uint64_t bytes = (uint64_t)a.rows * ((uint64_t)a.nh + a.gates + a.nkv) * HD * sizeof(T);
    if (bytes > 32u << 20) kv4_launch(k_qk_norm_rope<HD, T, true>, groups, CHK_WG, st, a);
    else kv4_launch(k_qk_norm_rope<HD, T, false>, groups, CHK_WG, st, a);
}

static void qk_call(const ChkQkNorm* n, const uint32_t* pos, uint32_t rows, const void* q, uint64_t q_stride, void* q_out,
                    uint64_t q_out_stride, const void* k, uint64_t k_stride, void* k_out, uint64_t k_out_stride,
                    uint32_t dtype, void* stream) {
    kv4_ensure(n, "no norm given");
    kv4_ensure(n->hd == 64 || n->hd == 128 || n->hd == 256, "head_dim must be 64, 128 or 256");
    kv4_ensure(n->nh + (uint64_t)n->nkv >= 1 && n->nh <= 4096 && n->nkv <= 4096, "1..=4096 query or key heads");
    kv4_ensure(n->rot % 2 == 0 && n->rot <= n->hd, "rot must be even, at most head_dim");
    kv4_ensure(n->eps >= 0x1p-100f && n->eps < INFINITY, "eps must be finite, at least 2^-100");
    kv4_dtype(dtype);
    kv4_ensure(rows <= 1u << 25, "at most 2^25 rows a call");
    kv4_ensure((uint64_t)rows * (n->nh + n->nkv) <= 1u << 28, "at most 2^28 rows x heads a call");
    if (rows == 0) return;
    kv4_ensure(pos && kv4_aligned(pos, 4), "null or misaligned pos");
    kv4_ensure(kv4_aligned(n->q_norm, 2) && kv4_aligned(n->k_norm, 2), "misaligned norm weights");
    kv4_ensure(n->rot == 0 || (n->turn && kv4_aligned(n->turn, 8)), "null or misaligned turn");
    const uint64_t qw = (uint64_t)n->nh * n->hd * (n->gated ? 2 : 1), kw = (uint64_t)n->nkv * n->hd;
    if (n->nh) {
        kv4_rows_arg(q, q_stride, qw, dtype, "q");
        kv4_rows_arg(q_out, q_out_stride, qw, dtype, "q_out");
        kv4_ensure(q != q_out || q_stride == q_out_stride, "q in place must keep its stride");
    }
    if (n->nkv) {
        kv4_rows_arg(k, k_stride, kw, dtype, "k");
        kv4_rows_arg(k_out, k_out_stride, kw, dtype, "k_out");
        kv4_ensure(k != k_out || k_stride == k_out_stride, "k in place must keep its stride");
    }
    const hipStream_t st = (hipStream_t)stream;
    kv4_on_device({pos, n->q_norm ? (const void*)n->q_norm : pos, n->k_norm ? (const void*)n->k_norm : pos,
                   n->rot ? (const void*)n->turn : pos, n->nh ? q : pos, n->nh ? q_out : pos, n->nkv ? k : pos,
                   n->nkv ? k_out : pos}, st);
    QkArgs a{q, k, q_out, k_out, q_stride, q_out_stride, k_stride, k_out_stride, n->q_norm, n->k_norm, n->turn, pos,
             rows, n->nh, n->nkv, n->gated ? 1u : 0u, n->gated && q != q_out ? n->nh : 0u, n->rot / 2, 0, 0, n->eps};
    auto on = [&](auto hd) {
        constexpr int H = decltype(hd)::value;
        if (dtype == CHK_F32) launch_qk<H, float>(a, st);
        else if (dtype == CHK_F16) launch_qk<H, _Float16>(a, st);
        else launch_qk<H, __bf16>(a, st);
    };
    if (n->hd == 64) on(std::integral_constant<int, 64>{});
    else if (n->hd == 128) on(std::integral_constant<int, 128>{});
    else on(std::integral_constant<int, 256>{});
}

}  // namespace chk

using namespace chk;

extern "C" {

int chk_qk_norm_rope(const ChkQkNorm* norm, const uint32_t* pos, uint32_t rows, const void* q, uint64_t q_stride,
                     void* q_out, uint64_t q_out_stride, const void* k, uint64_t k_stride, void* k_out,
                     uint64_t k_out_stride, uint32_t dtype, void* stream) {
    return kv4_try([&] {
        qk_call(norm, pos, rows, q, q_stride, q_out, q_out_stride, k, k_stride, k_out, k_out_stride, dtype, stream);
    });
}

int chk_rope_turns(double theta, uint32_t rot, uint64_t* turn) {
    return kv4_try([&] {
        kv4_ensure(turn || rot == 0, "null pointer");
        kv4_ensure(rot % 2 == 0 && rot <= 256, "rot must be even, at most 256");
        kv4_ensure(theta > 1.0 && theta < INFINITY, "theta must be finite, above 1");
        // 64 bits of mantissa; at most 2^64 / 2 pi, so nothing wraps
        const long double two_pi = 6.283185307179586476925286766559L;
        for (uint32_t j = 0; j < rot / 2; ++j)
            turn[j] = (uint64_t)std::rint(powl((long double)theta, -2.0L * j / rot) / two_pi * 0x1p64L);
    });
}

}  // extern "C"
