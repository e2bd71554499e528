// The 4-bit key/value cache (kvq4.h): rows quantised as they are written and
// rows read back.
//
// Both are one pass over memory.  Written, a row of hd values is 2 (f32) or 1
// (16-bit) KB and more read for hd / 2 + hd / 16 bytes stored, so the loads
// bound it; sixteen lanes take a row of values, four or eight dims of every
// group each (a lane's codes are then one stored piece), and the group's ends
// meet over lanes.
#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

#include "kernels_internal.h"
#include "kvq4.h"
#include "kvq4_host.h"

namespace chk {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));

CHK_DEV float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
CHK_DEV float4 load4(const _Float16* p) {
    const h4 v = *reinterpret_cast<const h4*>(p);
    return make_float4((float)v.x, (float)v.y, (float)v.z, (float)v.w);
}
CHK_DEV float4 load4(const __bf16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                       __uint_as_float(v.y & 0xffff0000u));
}
CHK_DEV void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
CHK_DEV void store4(_Float16* p, float a, float b, float c, float d) {
    *reinterpret_cast<h4*>(p) = h4{(_Float16)a, (_Float16)b, (_Float16)c, (_Float16)d};
}
CHK_DEV void store4(__bf16* p, float a, float b, float c, float d) {
    *reinterpret_cast<b4*>(p) = b4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
}

// The call's row starts into LDS (one read of them for the workgroup); a
// lookup of a row's sequence is then a search in LDS.
CHK_DEV void stage_starts(const Kv4Seqs& s, uint32_t* ss) {
    for (uint32_t i = threadIdx.x; i <= s.n; i += CHK_WG) ss[i] = s.start[i];
    __syncthreads();
}

// Position of row r of the call and its sequence; false where the row belongs
// to no sequence.  The position is negative where a sequence has more rows
// than tokens.
CHK_DEV bool row_place(const Kv4Seqs& s, const uint32_t* ss, uint32_t r, uint32_t& b, int64_t& p) {
    if (r >= s.rows) return false;
    b = kv4_seq_of(ss, s.n, r);
    if (b >= s.n) return false;
    uint32_t s0, s1;
    kv4_rows(ss, b, s.rows, s0, s1);
    p = (int64_t)s.len[b] - (int64_t)(s1 - r);
    return true;
}

// Where position p of sequence b is stored, as a row index of a plane without
// its head; false where the table does not hold it.
CHK_DEV bool place(const Kv4Cache& c, const Kv4Seqs& s, uint32_t b, int64_t p, uint32_t head, uint64_t& row) {
    if (p < 0 || p >= (int64_t)s.width << c.page_log2) return false;
    const uint32_t id = kv4_page(s.table + (size_t)b * s.width, s.width, c.page_log2, c.pages, (uint32_t)p);
    if (id == KV4_NO_PAGE) return false;
    row = kv4_row(id, c.nkv, c.page_log2, head, (uint32_t)p);
    return true;
}

// The code of u = x - b >= 0 at step s: the integer nearest to u / s.  The
// product with 1 / s (v_rcp, 1 ulp) may land across a border; the remainder
// e = u - q s is exact in f32 (q s has 12 bits, |e| < s), so comparing it with
// s / 2 decides, an odd q giving way where they are equal.
CHK_DEV uint32_t code_of(float u, float inv, float s, uint32_t half) {
    const float q = rintf(u * inv);
    const float e = fmaf(-q, s, u);
    uint32_t i = (uint32_t)q;
    const float h = __uint_as_float(half - (i & 1u));
    i += e > h ? 1u : 0u;
    i -= e < -h ? 1u : 0u;
    return i & 15u;
}

// One item = one (row, head) of the keys (V = 0) or the values (V = 1).
//   keys    4 ng lanes an item, lane g + ng kq... : 16 dims of one group
//   values  16 lanes an item, 4 dims of each of the ng groups
template <int HD, class T, int V>
CHK_DEV void append_item(const Kv4Cache& c, const Kv4Seqs& s, const uint32_t* ss, const T* x, uint64_t stride) {
    constexpr int NG = HD / 64, LANES = V ? 16 : 4 * NG, GL = V ? 16 : 4, PG = V ? NG : 1, N4 = V ? 1 : 4;
    const uint64_t t = (uint64_t)blockIdx.x * CHK_WG + threadIdx.x;
    const uint32_t l = (uint32_t)(t % LANES);
    const uint64_t item = t / LANES;
    const uint32_t r = (uint32_t)(item / c.nkv), head = (uint32_t)(item % c.nkv);
    uint32_t b = 0;
    int64_t p = 0;
    uint64_t row = 0;
    const bool live = row_place(s, ss, r, b, p) && place(c, s, b, p, head, row);
    // every lane of the wave takes part in the reductions
    const T* src = x + (live ? r : 0) * stride + (uint64_t)head * HD;
    const uint32_t g0 = V ? 0 : l / 4, kq = l % 4;
#pragma unroll
    for (int gi = 0; gi < PG; ++gi) {
        const uint32_t g = V ? (uint32_t)gi : g0;
        const uint32_t d0 = 64 * g + (V ? 4 * l : 16 * kq);
        float v[4 * N4];
        float lo = INFINITY, hi = -INFINITY, nan = 0.0f;
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            const float4 f = live ? load4(src + d0 + 4 * i) : make_float4(0, 0, 0, 0);
            v[4 * i] = f.x;
            v[4 * i + 1] = f.y;
            v[4 * i + 2] = f.z;
            v[4 * i + 3] = f.w;
        }
#pragma unroll
        for (int i = 0; i < 4 * N4; ++i) {
            lo = fminf(lo, v[i]);
            hi = fmaxf(hi, v[i]);
            nan = fmaf(v[i], 0.0f, nan);  // NaN from a NaN or an infinity
        }
#pragma unroll
        for (int m = GL / 2; m >= 1; m >>= 1) {
            lo = fminf(lo, __shfl_xor(lo, m, 64));
            hi = fmaxf(hi, __shfl_xor(hi, m, 64));
            nan += __shfl_xor(nan, m, 64);
        }
        float st, bs;
        kv4_pair(lo, nan == nan ? hi : nan, st, bs);
        const float inv = __builtin_amdgcn_rcpf(st);
        const uint32_t half = __float_as_uint(0.5f * st);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 4 * N4; ++i) w[i / 8] |= code_of(v[i] - bs, inv, st, half) << (4 * (i % 8));
        if (!live) continue;
        const uint32_t pair = (__float_as_uint(st) >> 16) | (__float_as_uint(bs) & 0xffff0000u);
        if (V) {
            reinterpret_cast<uint16_t*>(c.v + row * (HD / 2))[l * NG + g] = (uint16_t)w[0];
            if (l == 0) c.vs[row * NG + g] = pair;
        } else {
            reinterpret_cast<uint2*>(c.k + row * (HD / 2))[kq * NG + g] = make_uint2(w[0], w[1]);
            if (kq == 0) c.ks[row * NG + g] = pair;
        }
    }
}

template <int HD, class T>
__global__ void __launch_bounds__(256) k_kv4_append(Kv4Cache c, Kv4Seqs s, const T* k, const T* v, uint64_t ks,
                                                    uint64_t vs) {
    __shared__ uint32_t ss[KV4_MAX_SEQS + 1];
    stage_starts(s, ss);
    if (blockIdx.y == 0) append_item<HD, T, 0>(c, s, ss, k, ks);
    else append_item<HD, T, 1>(c, s, ss, v, vs);
}

// A token that the table does not hold reads as NaN.
template <int HD, class T, int V>
CHK_DEV void read_item(const Kv4Cache& c, const Kv4Seqs& s, const uint32_t* ss, T* x, uint64_t stride) {
    constexpr int NG = HD / 64, LANES = V ? 16 : 4 * NG, PG = V ? NG : 1, N4 = V ? 1 : 4;
    const uint64_t t = (uint64_t)blockIdx.x * CHK_WG + threadIdx.x;
    const uint32_t l = (uint32_t)(t % LANES);
    const uint64_t item = t / LANES;
    const uint32_t r = (uint32_t)(item / c.nkv), head = (uint32_t)(item % c.nkv);
    uint32_t b;
    int64_t p;
    if (!row_place(s, ss, r, b, p)) return;
    uint64_t row = 0;
    const bool held = place(c, s, b, p, head, row);
    T* dst = x + r * stride + (uint64_t)head * HD;
    const uint32_t g0 = V ? 0 : l / 4, kq = l % 4;
#pragma unroll
    for (int gi = 0; gi < PG; ++gi) {
        const uint32_t g = V ? (uint32_t)gi : g0;
        const uint32_t d0 = 64 * g + (V ? 4 * l : 16 * kq);
        uint32_t w[2] = {0u, 0u}, pair = KV4_NAN_PAIR;
        if (held) {
            if (V) {
                w[0] = reinterpret_cast<const uint16_t*>(c.v + row * (HD / 2))[l * NG + g];
                pair = c.vs[row * NG + g];
            } else {
                const uint2 u = reinterpret_cast<const uint2*>(c.k + row * (HD / 2))[kq * NG + g];
                w[0] = u.x;
                w[1] = u.y;
                pair = c.ks[row * NG + g];
            }
        }
        const float st = __uint_as_float(pair << 16), bs = __uint_as_float(pair & 0xffff0000u);
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = fmaf((float)((w[i / 2] >> (16 * (i % 2) + 4 * j)) & 15u), st, bs);
            store4(dst + d0 + 4 * i, f[0], f[1], f[2], f[3]);
        }
    }
}

template <int HD, class T>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4Cache c, Kv4Seqs s, T* k, T* v, uint64_t ks, uint64_t vs) {
    __shared__ uint32_t ss[KV4_MAX_SEQS + 1];
    stage_starts(s, ss);
    if (blockIdx.y == 0) read_item<HD, T, 0>(c, s, ss, k, ks);
    else read_item<HD, T, 1>(c, s, ss, v, vs);
}

template <int HD, class T>
static void launch_rows(bool append, const Kv4Cache& c, const Kv4Seqs& s, void* k, void* v, uint64_t ks, uint64_t vs,
                        hipStream_t st) {
    // 16 lanes an item (keys of 128 dims need 8)
    const uint64_t items = (uint64_t)s.rows * c.nkv;
    const dim3 grid((uint32_t)((items * 16 + CHK_WG - 1) / CHK_WG), 2);
    if (append) kv4_launch(k_kv4_append<HD, T>, grid, CHK_WG, st, c, s, (const T*)k, (const T*)v, ks, vs);
    else kv4_launch(k_kv4_read<HD, T>, grid, CHK_WG, st, c, s, (T*)k, (T*)v, ks, vs);
}

static void rows_call(bool append, const ChkKvQ4* cache, const ChkKvSeqs* seqs, void* k, void* v, uint32_t dtype,
                      uint64_t ks, uint64_t vs, void* stream) {
    const Kv4Cache c = kv4_cache(cache);
    const Kv4Seqs s = kv4_seqs(cache, seqs);
    kv4_dtype(dtype);
    const uint64_t row = (uint64_t)cache->nkv * cache->hd;
    kv4_rows_arg(k, ks, row, dtype, "k");
    kv4_rows_arg(v, vs, row, dtype, "v");
    kv4_ensure((uint64_t)s.rows * cache->nkv <= 1u << 27, "at most 2^27 rows x kv heads a call");
    if (s.rows == 0) return;
    kv4_on_device({cache->k, cache->v, cache->ks, cache->vs, seqs->table, seqs->len, seqs->start, k, v});
    const hipStream_t st = (hipStream_t)stream;
    kv4_switch(cache->hd, dtype, [&](auto hd, auto t) {
        launch_rows<decltype(hd)::value, typename decltype(t)::type>(append, c, s, k, v, ks, vs, st);
    });
}

}  // namespace chk

using namespace chk;

extern "C" {

int chk_kv_append_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* k, const void* v, uint32_t dtype,
                     uint64_t k_stride, uint64_t v_stride, void* stream) {
    return kv4_try([&] {
        rows_call(true, cache, seqs, const_cast<void*>(k), const_cast<void*>(v), dtype, k_stride, v_stride, stream);
    });
}

int chk_kv_read_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, void* k, void* v, uint32_t dtype, uint64_t k_stride,
                   uint64_t v_stride, void* stream) {
    return kv4_try([&] { rows_call(false, cache, seqs, k, v, dtype, k_stride, v_stride, stream); });
}

int chk_kv_slot_q4(const ChkKvQ4* cache, const uint32_t* table_row, uint32_t width, uint32_t t, uint64_t* slot) {
    return kv4_try([&] {
        kv4_ensure(cache && slot && (table_row || width == 0), "null pointer");
        kv4_ensure(cache->page >= KV4_MIN_PAGE && (cache->page & (cache->page - 1)) == 0,
                   "page must be a power of two of at least 16 tokens");
        const uint32_t lg = kv4_log2(cache->page);
        const uint32_t id = kv4_page(table_row, width, lg, cache->pages, t);
        kv4_ensure(id != KV4_NO_PAGE, "no page of the cache holds this token");
        *slot = kv4_row(id, 1, lg, 0, t);
    });
}

int chk_kv_pair_q4(const float* group, uint16_t* s, uint16_t* b) {
    return kv4_try([&] {
        kv4_ensure(group && s && b, "null pointer");
        float lo = group[0], hi = group[0], nan = 0.0f;
        for (int i = 0; i < 64; ++i) {
            lo = group[i] < lo ? group[i] : lo;
            hi = group[i] > hi ? group[i] : hi;
            nan += group[i] * 0.0f;
        }
        float st, bs;
        kv4_pair(lo, nan == nan ? hi : nan, st, bs);
        *s = (uint16_t)(kv4_bits(st) >> 16);
        *b = (uint16_t)(kv4_bits(bs) >> 16);
    });
}

}  // extern "C"
