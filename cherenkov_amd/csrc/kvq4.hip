// The 4-bit key/value cache (kvq4.h): rows quantised as they are written and
// rows read back.
//
// Both are one pass over memory, bound by it: written, a row of hd values is
// 4 hd or 2 hd bytes read for hd / 2 + hd / 16 stored.  A lane takes 16 bytes
// of a row (4 or 8 dims), so a wave's rows are whole pieces of memory, and a
// group's ends meet over the 16 or 8 lanes that hold it.  A workgroup takes
// consecutive rows of one head: their codes and pairs are consecutive bytes of
// a page, written by one workgroup, where rows with all their heads would have
// left lines half written by workgroups of two XCDs.  One row a lane: the waves
// of a full device hold enough loads by themselves (two or four rows a lane
// measured 4 to 10 % behind for appending, level for reading back).
//
// Measured: 16000 bf16 rows of 8 x 128 written and read back in 35 us, 168 MB
// and two launches; 64000 f16 rows of 2 x 256 read back in 27 us, 6.2 TB/s
// over the 168 MB moved (a large copy: 4.9).
#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

#include "kernels_internal.h"
#include "kvq4.h"
#include "kvq4_host.h"

namespace chk {

// What a lane takes: 16 bytes of a row, 4 or 8 values.
template <class T>
struct Piece {
    static constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(N)));
};

// The row starts and lengths in LDS, one read of them for the workgroup; a lookup of a
// row's sequence is then a search in LDS.
struct SeqsLds {
    uint32_t start[KV4_MAX_SEQS + 1], len[KV4_MAX_SEQS];
};
CHK_DEV void stage_seqs(const Kv4Seqs& s, SeqsLds& q) {
    for (uint32_t i = threadIdx.x; i <= s.n; i += CHK_WG) {
        q.start[i] = s.start[i];
        if (i < s.n) q.len[i] = s.len[i];
    }
}

// Position of row r of the call and its sequence; false where the row belongs
// to no sequence.  The position is negative where a sequence has more rows
// than tokens.
CHK_DEV bool row_place(const Kv4Seqs& s, const SeqsLds& q, uint32_t r, uint32_t& b, int64_t& p) {
    if (r >= s.rows) return false;
    b = kv4_seq_of(q.start, s.n, r);
    if (b >= s.n) return false;
    uint32_t s0, s1;
    kv4_rows(q.start, b, s.rows, s0, s1);
    p = (int64_t)q.len[b] - (int64_t)(s1 - r);
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

// max/min over the 8 or 16 lanes of a group (a NaN stays), by row operations.
template <int LANES, bool MAX>
CHK_DEV float group_end(float v) {
    auto step = [&](float o) { return MAX ? __builtin_elementwise_maximum(v, o) : __builtin_elementwise_minimum(v, o); };
    v = step(CHK_DPP(v, 0xb1, 0xf, v));   // lane ^ 1
    v = step(CHK_DPP(v, 0x4e, 0xf, v));   // lane ^ 2
    v = step(CHK_DPP(v, 0x141, 0xf, v));  // the other four of eight
    if (LANES == 16) v = step(CHK_DPP(v, 0x140, 0xf, v));  // the other eight of sixteen
    return v;
}

// One lane's part of one row: 4 or 8 consecutive values of one group into
// codes, and the group's pair.
//
// The code of u = x - b >= 0 at step s is the integer nearest to u / s, ties
// to even.  With t = fl(u fl(1 / s)) (v_rcp, 1 ulp) and the remainder
// e = u - t s, t + e fl(1 / s) is u / s to 2^-45 of itself.  s has 8
// significant bits, so (k + 1/2) s is a float, and u is it or at least one of
// u's ulps away, 0.502 ulp or more of the quotient: the rounded quotient lies
// on u / s's side of k + 1/2, on it where u / s does, and rounding it to an
// integer gives the same as rounding u / s.  e is exact while u is far from
// the subnormals; a group with a smaller step is multiplied by 2^64 first.
// Adding 3 2^22 rounds to the integer, in the sum's low bits.
template <int N>
CHK_DEV uint32_t quantise(const float* v, uint32_t& pair) {
    constexpr int LANES = 64 / N;
    float lo = v[0], hi = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) {
        lo = __builtin_elementwise_minimum(lo, v[i]);
        hi = __builtin_elementwise_maximum(hi, v[i]);
    }
    float s, b;
    kv4_pair(group_end<LANES, false>(lo), group_end<LANES, true>(hi), s, b);
    pair = (__float_as_uint(s) >> 16) | (__float_as_uint(b) & 0xffff0000u);
    float u[N], st = s;
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = v[i] - b;
    if (s < 0x1p-96f) {
        st *= 0x1p64f;
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] *= 0x1p64f;
    }
    const float inv = __builtin_amdgcn_rcpf(st);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = u[i] * inv;
        w += __float_as_uint(fmaf(fmaf(-t, st, u[i]), inv, t) + 0x3p22f) << (4 * i);
    }
    // less the sums' own bits, 0x4b400000 << 4 i
    w -= 0x4b400000u + 0xb4000000u + 0x40000000u;
    return s == s ? w : 0u;
}

// Which piece of the call is this lane's: a workgroup takes ROWS consecutive
// rows of head blockIdx.y.
template <int HD, class T>
struct Lane {
    static constexpr int N = Piece<T>::N, ROW = HD / N, ROWS = CHK_WG / ROW, NG = HD / 64;
    uint32_t row, dim, g, within;  // the row, this lane's first dim, its group and its place there
    CHK_DEV Lane() {
        row = blockIdx.x * ROWS + threadIdx.x / ROW;
        dim = threadIdx.x % ROW * N;
        g = dim / 64;
        within = dim % 64;
    }
    // the codes of 4 dims, as a 2-byte index into a row
    CHK_DEV uint32_t key() const { return (within / 16 * NG + g) * 4 + within % 16 / 4; }
    CHK_DEV uint32_t val(int i) const { return (within / 4 + i) * NG + g; }
};

template <int HD, class T>
__global__ void __launch_bounds__(256) k_kv4_append(Kv4Cache c, Kv4Seqs s, const T* k, const T* v, uint64_t ks,
                                                    uint64_t vs) {
    typedef Lane<HD, T> L;
    typedef typename Piece<T>::vec Vec;
    constexpr int N = L::N, NG = L::NG;
    __shared__ SeqsLds q;
    const L l;
    // in flight while the row's place is looked up; past the last row the last
    // row again, unused
    const uint64_t r = min(l.row, s.rows - 1);
    const Vec x[2] = {*reinterpret_cast<const Vec*>(k + r * ks + blockIdx.y * HD + l.dim),
                      *reinterpret_cast<const Vec*>(v + r * vs + blockIdx.y * HD + l.dim)};
    stage_seqs(s, q);
    __syncthreads();
    uint32_t b;
    int64_t p;
    uint64_t row;
    const bool live = row_place(s, q, l.row, b, p) && place(c, s, b, p, blockIdx.y, row);
    uint32_t w[2], pair[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = (float)x[h][j];
        w[h] = quantise<N>(f, pair[h]);  // every lane takes part
    }
    if (!live) return;
    uint16_t* kr = reinterpret_cast<uint16_t*>(c.k + row * (HD / 2)) + l.key();
    uint16_t* vr = reinterpret_cast<uint16_t*>(c.v + row * (HD / 2));
    if (N == 8) *reinterpret_cast<uint32_t*>(kr) = w[0];
    else *kr = (uint16_t)w[0];
#pragma unroll
    for (int j = 0; j < N / 4; ++j) vr[l.val(j)] = (uint16_t)(w[1] >> (16 * j));
    if (l.within == 0) {
        c.ks[row * NG + l.g] = pair[0];
        c.vs[row * NG + l.g] = pair[1];
    }
}

// A token that the table does not hold reads as NaN.  The rows go out past the
// caches (they are many times what is read, and a call's are rarely all read
// before they would have been evicted): 64000 f16 rows of 2 x 256 in 27 us
// against 50 with ordinary stores.
template <int HD, class T>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4Cache c, Kv4Seqs s, T* k, T* v, uint64_t ks, uint64_t vs) {
    typedef Lane<HD, T> L;
    typedef typename Piece<T>::vec Vec;
    constexpr int N = L::N, NG = L::NG;
    __shared__ SeqsLds q;
    stage_seqs(s, q);
    __syncthreads();
    const L l;
    uint32_t b;
    int64_t p;
    uint64_t row;
    if (!row_place(s, q, l.row, b, p)) return;
    uint32_t w[2] = {0u, 0u}, pair[2] = {KV4_NAN_PAIR, KV4_NAN_PAIR};
    if (place(c, s, b, p, blockIdx.y, row)) {
        const uint16_t* kr = reinterpret_cast<const uint16_t*>(c.k + row * (HD / 2)) + l.key();
        const uint16_t* vr = reinterpret_cast<const uint16_t*>(c.v + row * (HD / 2));
        w[0] = N == 8 ? *reinterpret_cast<const uint32_t*>(kr) : *kr;
#pragma unroll
        for (int j = 0; j < N / 4; ++j) w[1] |= (uint32_t)vr[l.val(j)] << (16 * j);
        pair[0] = c.ks[row * NG + l.g];
        pair[1] = c.vs[row * NG + l.g];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float st = __uint_as_float(pair[h] << 16), bs = __uint_as_float(pair[h] & 0xffff0000u);
        Vec x;
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = (T)fmaf((float)((w[h] >> (4 * j)) & 15u), st, bs);
        T* dst = (h ? v + (uint64_t)l.row * vs : k + (uint64_t)l.row * ks) + blockIdx.y * HD + l.dim;
        __builtin_nontemporal_store(x, reinterpret_cast<Vec*>(dst));
    }
}

template <int HD, class T>
static void launch_rows(bool append, const Kv4Cache& c, const Kv4Seqs& s, void* k, void* v, uint64_t ks, uint64_t vs,
                        hipStream_t st) {
    constexpr uint32_t rows = Lane<HD, T>::ROWS;
    const dim3 grid((s.rows + rows - 1) / rows, c.nkv);
    if (append) kv4_launch(k_kv4_append<HD, T>, grid, CHK_WG, st, c, s, (const T*)k, (const T*)v, ks, vs);
    else kv4_launch(k_kv4_read<HD, T>, grid, CHK_WG, st, c, s, (T*)k, (T*)v, ks, vs);
}

static void rows_call(bool append, const ChkKvQ4* cache, const ChkKvSeqs* seqs, void* k, void* v, uint32_t dtype,
                      uint64_t ks, uint64_t vs, void* stream) {
    const Kv4Cache c = kv4_cache(cache);
    const Kv4Seqs s = kv4_seqs(cache, seqs);
    kv4_dtype(dtype);
    if (s.rows == 0) return;
    const uint64_t row = (uint64_t)cache->nkv * cache->hd;
    kv4_rows_arg(k, ks, row, dtype, "k");
    kv4_rows_arg(v, vs, row, dtype, "v");
    kv4_ensure((uint64_t)s.rows * cache->nkv <= 1u << 27, "at most 2^27 rows x kv heads a call");
    kv4_ensure(s.rows <= 1u << 25, "at most 2^25 rows a call");  // 64 threads a row at most: a launch has under 2^32
    const hipStream_t st = (hipStream_t)stream;
    kv4_on_device({cache->k, cache->v, cache->ks, cache->vs, seqs->table, seqs->len, seqs->start, k, v}, st);
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
