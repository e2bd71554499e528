// The norm of each query and key head and its rotation, rows of a batch.
//
//   y = x / sqrt(mean(x^2) + eps) * w,   (y_j, y_{j + r/2}) turned by pos * turn_j
// for the first r dims of a head (norm_rope of attn.hip, for 16-bit rows too,
// rows of any batch, and angles that stay exact at far positions).
//
// The angle.  turn_j is in 2^-64 of a turn, so pos turn_j modulo 2^64 is the
// angle, and its upper word is enough: one 32-bit product and one upper half.
// The eighth of the circle nearest to it is taken off in integers; what is left,
// at most pi / 4, is exact to 2^-25 of itself in f32, and Taylor's sums of
// degree 9 and 10 end 2e-9 and 1e-10 from sine and cosine.
//
// One pass over memory, bound by it.  A lane takes 16 bytes of a head, 8 or 4
// dims, so a head is 8 to 64 lanes, its sum of squares a few row operations, and
// a wave takes one row's heads, 64 / (lanes a head) at a time, four such pieces'
// loads in flight.  A row's angles are computed once, one a lane, and read
// back from LDS in the lane's order; a dim's partner comes by lane permutes,
// or through LDS where half the turned dims do not fill whole lanes.  Few rows:
// a wave a piece.
#include <hip/hip_runtime.h>

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
    uint32_t waves;                        // of a row
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

// U pieces' loads in flight a wave.
template <int HD, class T, int U>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkArgs a) {
    typedef QkPiece<HD, T> P;
    typedef typename P::vec Vec;
    constexpr int N = P::N;
    __shared__ float2 angle[CHK_WG / 64][HD / 2];
    __shared__ float line[CHK_WG / 64][64 * N];
    const uint32_t lane = threadIdx.x & 63, w = wave_id();
    const uint64_t wave = (uint64_t)blockIdx.x * (CHK_WG / 64) + w;
    const uint32_t row = (uint32_t)(wave / a.waves), share = (uint32_t)(wave % a.waves);
    if (row >= a.rows) return;
    const uint32_t pos = a.pos[row];
    if (pos == 0xffffffffu) return;
    const uint32_t d0 = lane % P::LANES * N, sub = lane / P::LANES, half = a.half;
    // heads: queries, keys, then the gates that are only copied
    const uint32_t heads = a.nh + a.nkv + a.gates;
    const uint32_t wide = a.gated ? 2 * HD : HD;
    const T *qr = (const T*)a.q + row * a.q_stride, *kr = (const T*)a.k + row * a.k_stride;
    T *qo = (T*)a.q_out + row * a.q_out_stride, *ko = (T*)a.k_out + row * a.k_out_stride;
    auto src = [&](uint32_t h) __attribute__((always_inline)) {
        return h < a.nh ? qr + h * wide + d0 : h < a.nh + a.nkv ? kr + (h - a.nh) * HD + d0 : qr + (h - a.nh - a.nkv) * wide + HD + d0;
    };
    auto dst = [&](uint32_t h) __attribute__((always_inline)) {
        return h < a.nh ? qo + h * wide + d0 : h < a.nh + a.nkv ? ko + (h - a.nh) * HD + d0 : qo + (h - a.nh - a.nkv) * wide + HD + d0;
    };
    const uint32_t step = a.waves * P::HEADS;
    uint32_t h0 = share * P::HEADS + sub;
    Vec x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const Vec*>(src(min(h0 + u * step, heads - 1)));
    // ---- weights and angles
    float wq[N], wk[N], cs[N], sn[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        wq[i] = a.q_norm ? bf16f(a.q_norm[d0 + i]) : 1.0f;
        wk[i] = a.k_norm ? bf16f(a.k_norm[d0 + i]) : 1.0f;
        cs[i] = 1.0f;
        sn[i] = 0.0f;
    }
    for (uint32_t j = lane; j < half; j += 64) {
        const uint64_t t = a.turn[j];
        angle[w][j] = turned(__umulhi(pos, (uint32_t)t) + pos * (uint32_t)(t >> 32));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t d = d0 + i;
        if (d < 2 * half) {
            const float2 c = angle[w][d < half ? d : d - half];
            cs[i] = c.x;
            sn[i] = d < half ? -c.y : c.y;
        }
    }
    // half in whole lanes: a partner is a lane's same element
    const bool whole = half % N == 0;
    const int mate = whole && d0 < 2 * half ? (int)lane + (d0 < half ? (int)(half / N) : -(int)(half / N)) : (int)lane;

    for (; __any(h0 < heads); h0 += U * step) {
        if (U > 1 && h0 >= U * step) {
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const Vec*>(src(min(h0 + u * step, heads - 1)));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t h = h0 + u * step;
            const bool is_q = h < a.nh, is_gate = h >= a.nh + a.nkv;
            float y[N], ss = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                y[i] = (float)x[u][i];
                ss = fmaf(y[i], y[i], ss);
            }
            ss = group_sum<P::LANES>(ss);
            float inv = __builtin_amdgcn_rsqf(fmaf(ss, 1.0f / HD, a.eps));
            if (!(is_q ? a.q_norm : a.k_norm)) inv = 1.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = y[i] * inv * (is_q ? wq[i] : wk[i]);
            if (half) {
                float o[N];
                if (whole) {
#pragma unroll
                    for (int i = 0; i < N; ++i) o[i] = __shfl(y[i], mate, 64);
                } else {
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int i = 0; i < N; ++i) line[w][lane * N + i] = y[i];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const uint32_t d = d0 + i;
                        o[i] = line[w][sub * HD + (d < half ? d + half : d < 2 * half ? d - half : d)];
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = fmaf(y[i], cs[i], o[i] * sn[i]);
            }
            Vec r;
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = (T)y[i];
            if (is_gate) r = x[u];
            if (h < heads) *reinterpret_cast<Vec*>(dst(h)) = r;
        }
    }
}

template <int HD, class T>
static void launch_qk(QkArgs& a, hipStream_t st) {
    typedef QkPiece<HD, T> P;
    const uint32_t pieces = (a.nh + a.nkv + a.gates + P::HEADS - 1) / P::HEADS;
    constexpr uint32_t MANY = 4096;
    // waves of the device with a wave a piece
    const bool few = (uint64_t)a.rows * pieces <= MANY;
    a.waves = few ? pieces : 1u;
    const uint64_t groups = ((uint64_t)a.rows * a.waves + CHK_WG / 64 - 1) / (CHK_WG / 64);
    if (few) kv4_launch(k_qk_norm_rope<HD, T, 1>, dim3((uint32_t)groups), CHK_WG, st, a);
    else kv4_launch(k_qk_norm_rope<HD, T, 4>, dim3((uint32_t)groups), CHK_WG, st, a);
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
             rows, n->nh, n->nkv, n->gated ? 1u : 0u, n->gated && q != q_out ? n->nh : 0u, n->rot / 2, 0, n->eps};
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
