// Causal attention over the 4-bit key/value cache (kvq4.h) for the rows of a
// batch of sequences.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "kernels_internal.h"
#include "kvq4.h"
#include "kvq4_host.h"

namespace chk {

struct AttnQ4Args {
    Kv4Cache c;
    Kv4Seqs s;
    const void* q;
    void* out;
    uint64_t q_stride, out_stride;  // elements
    uint32_t nh, group, gated;      // group: query heads a kv head
    float scale;
    const uint32_t* mask;  // null: none
    uint32_t words, ratio, kblk;
};

// Is token t visible to a row at position p?
CHK_DEV bool visible(const AttnQ4Args& a, uint32_t row, int64_t p, uint32_t t) {
    if ((int64_t)t > p) return false;
    if (!a.mask) return true;
    const uint32_t nblk = (uint32_t)((p + 1) / a.ratio), blk = t / a.ratio;
    if (nblk <= a.kblk || blk >= nblk) return true;
    return (blk >> 5) < a.words && ((a.mask[(size_t)row * a.words + (blk >> 5)] >> (blk & 31)) & 1u);
}

// One workgroup per (row, head), 64 tokens at a time: four threads a token
// score a quarter of the head each, wave 0 keeps the running maximum and sum,
// thread d sums dim d of the values.
template <int HD, class T>
__global__ void __launch_bounds__(256) k_attn_q4(AttnQ4Args a) {
    constexpr int NG = HD / 64;
    __shared__ uint32_t ss[KV4_MAX_SEQS + 1];
    __shared__ float sq[HD], sp[64];
    __shared__ uint64_t srow[64];
    __shared__ float sal;
    const uint32_t t = threadIdx.x, r = blockIdx.x, h = blockIdx.y, hk = h / a.group;
    for (uint32_t i = t; i <= a.s.n; i += CHK_WG) ss[i] = a.s.start[i];
    __syncthreads();
    const uint32_t b = kv4_seq_of(ss, a.s.n, r);
    if (b >= a.s.n) return;
    uint32_t s0, s1;
    kv4_rows(ss, b, a.s.rows, s0, s1);
    const uint32_t len = a.s.len[b];
    const bool held = len <= (uint64_t)a.s.width << a.c.page_log2;
    const int64_t p = held ? (int64_t)len - (int64_t)(s1 - r) : -1;
    const T* q = (const T*)a.q + r * a.q_stride + (uint64_t)h * HD * (a.gated ? 2 : 1);
    if (t < HD) sq[t] = (float)q[t];
    const uint32_t* table = a.s.table + (size_t)b * a.s.width;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int64_t t0 = 0; t0 <= p; t0 += 64) {
        __syncthreads();
        const uint32_t tok = (uint32_t)t0 + (t >> 2), quarter = t & 3;
        float acc = 0.0f;
        const bool vis = tok <= p && visible(a, r, p, tok);
        if (vis) {
            const uint32_t id = kv4_page(table, a.s.width, a.c.page_log2, a.c.pages, tok);
            const uint64_t row = id == KV4_NO_PAGE ? ~0ull : kv4_row(id, a.c.nkv, a.c.page_log2, hk, tok);
            if (quarter == 0) srow[t >> 2] = row;
            if (row == ~0ull) acc = NAN;
            else
                for (int g = 0; g < NG; ++g) {
                    const uint32_t pair = a.c.ks[row * NG + g];
                    const float s = __uint_as_float(pair << 16), bs = __uint_as_float(pair & 0xffff0000u);
                    const uint2 w = reinterpret_cast<const uint2*>(a.c.k + row * (HD / 2))[quarter * NG + g];
                    for (int j = 0; j < 16; ++j)
                        acc += sq[64 * g + 16 * quarter + j] * fmaf((float)(((j < 8 ? w.x : w.y) >> (4 * (j & 7))) & 15u), s, bs);
                }
        }
        acc += __shfl_xor(acc, 1, 64);
        acc += __shfl_xor(acc, 2, 64);
        if (quarter == 0) sp[t >> 2] = vis ? acc * a.scale : -INFINITY;
        __syncthreads();
        if (t < 64) {
            const float s = sp[t];
            float mx = wave_max(s);
            const float mn = fmaxf(m, mx);
            const float pv = s == -INFINITY ? 0.0f : expf(s - mn);
            const float al = m == -INFINITY ? 0.0f : expf(m - mn);
            l = l * al + wave_sum(pv);
            m = mn;
            sp[t] = pv;
            if (t == 0) sal = al;
        }
        __syncthreads();
        if (t < HD) {
            o *= sal;
            const uint32_t g = t / 64, n = (t % 64) / 4;
            for (int64_t j = 0; j < 64 && t0 + j <= p; ++j) {
                if (sp[j] == 0.0f) continue;
                const uint64_t row = srow[j];
                if (row == ~0ull) {
                    o = NAN;
                    continue;
                }
                const uint32_t pair = a.c.vs[row * NG + g];
                const uint32_t w = reinterpret_cast<const uint16_t*>(a.c.v + row * (HD / 2))[n * NG + g];
                o += sp[j] * fmaf((float)((w >> (4 * (t & 3))) & 15u), __uint_as_float(pair << 16),
                                  __uint_as_float(pair & 0xffff0000u));
            }
        }
    }
    if (t == 0) sal = l;
    __syncthreads();
    if (t < HD) {
        float v = p < 0 ? 0.0f : sal > 0.0f ? o / sal : sal == 0.0f ? 0.0f : NAN;
        if (!held) v = NAN;
        else if (a.gated) v *= sigmoidf_((float)q[HD + t]);
        ((T*)a.out)[r * a.out_stride + (uint64_t)h * HD + t] = (T)v;
    }
}

static uint64_t workspace_bytes(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t n, uint32_t rows) {
    kv4_ensure(hd == 128 || hd == 256, "head_dim must be 128 or 256");
    kv4_ensure(nkv >= 1 && nh >= nkv && nh % nkv == 0 && nh <= 4096, "nh must be a multiple of nkv, at most 4096");
    kv4_ensure(n <= KV4_MAX_SEQS, "at most 1024 sequences a call");
    return 256;
}

static void attn_call(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated,
                      uint32_t dtype, uint64_t q_stride, const ChkKvMask* mask, void* out, uint64_t out_stride, void* ws,
                      uint64_t ws_bytes, void* stream) {
    AttnQ4Args a{};
    a.c = kv4_cache(cache);
    a.s = kv4_seqs(cache, seqs);
    kv4_dtype(dtype);
    const uint64_t need = workspace_bytes(nh, cache->nkv, cache->hd, a.s.n, a.s.rows);
    kv4_rows_arg(q, q_stride, (uint64_t)nh * cache->hd * (gated ? 2 : 1), dtype, "q");
    kv4_rows_arg(out, out_stride, (uint64_t)nh * cache->hd, dtype, "out");
    kv4_ensure(ws && kv4_aligned(ws, 16), "null or misaligned workspace");
    kv4_ensure(ws_bytes >= need, "workspace smaller than chk_attn_q4_workspace says");
    if (mask) {
        kv4_ensure(mask->bits && kv4_aligned(mask->bits, 4), "null or misaligned mask");
        kv4_ensure(mask->ratio >= 1 && mask->words >= 1, "ratio and words must be positive");
        a.mask = mask->bits;
        a.words = mask->words;
        a.ratio = mask->ratio;
        a.kblk = mask->kblk;
    }
    if (a.s.rows == 0) return;
    kv4_on_device({cache->k, cache->v, cache->ks, cache->vs, seqs->table, seqs->len, seqs->start, q, out, ws});
    if (mask) kv4_on_device({mask->bits});
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.nh = nh;
    a.group = nh / cache->nkv;
    a.gated = gated ? 1u : 0u;
    a.scale = 1.0f / sqrtf((float)cache->hd);
    kv4_switch(cache->hd, dtype, [&](auto hd, auto t) {
        kv4_launch(k_attn_q4<decltype(hd)::value, typename decltype(t)::type>, dim3(a.s.rows, nh), CHK_WG,
                   (hipStream_t)stream, a);
    });
}

}  // namespace chk

using namespace chk;

extern "C" {

int chk_attn_q4(const ChkKvQ4* cache, const ChkKvSeqs* seqs, const void* q, uint32_t nh, uint32_t gated, uint32_t dtype,
                uint64_t q_stride, const ChkKvMask* mask, void* out, uint64_t out_stride, void* ws, uint64_t ws_bytes,
                void* stream) {
    return kv4_try([&] {
        attn_call(cache, seqs, q, nh, gated, dtype, q_stride, mask, out, out_stride, ws, ws_bytes, stream);
    });
}

int chk_attn_q4_workspace(uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t n, uint32_t rows, uint64_t* bytes) {
    return kv4_try([&] {
        kv4_ensure(bytes, "null pointer");
        *bytes = workspace_bytes(nh, nkv, hd, n, rows);
    });
}

}  // extern "C"
