// A step's plan over a pool of pages of the 4-bit cache: sequences cut back,
// pages given back and taken, row starts, positions and slots.
//
// With h(t) = ceil(t / page), a sequence of len tokens cut back to l gives back
// its entries from max(h(l), own) to h(len), those of them that name a page, and needs
// h(l + want) - h(l) for its rows.  Everything else is sums over the sequences in
// turn: of pages given back (from the last one on: the list is a stack, and a step
// taken back leaves it as it was), of wants (who still finds room in the row arrays),
// of needs (who still finds pages), of the wants that are served (the row starts).
//
// One workgroup, a sequence a thread, carries the state on; sums are wave scans
// on row operations met over LDS.  Pages then go one a thread, its sequence found
// by a search over the sums in LDS: first all that are given back, then, behind
// a barrier, those taken.  So the work of a step is spread over the threads
// whatever a single sequence has of it.  Entries given back are looked at before the
// needs are served, so that none that names no page is counted; where there is one,
// those that do are packed by sums over 1024 entries at a time.
//
// What bounds it is latency: a handful of dependent reads.  One request 3.0 us, 64 of
// three drafts 5.7; 900 with prompts 8.7, and the 41000 rows' positions and slots, a launch
// of their own over the device, 3.9.  (Pages four a thread in flight: level.)
#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

#include "kernels_internal.h"
#include "kvq4.h"
#include "kvq4_host.h"

namespace chk {

constexpr uint32_t PLAN_WG = 1024;
constexpr uint32_t PLAN_ROWS = 1u << 21;  // rows of a call stay below: sums of 1024 wants in 32 bits

struct PlanArgs {
    uint32_t *table, *len, *free, *nfree;
    const uint32_t *keep, *own, *want;
    uint32_t *start, *pos;
    uint64_t* slot;
    uint32_t n, width, page_log2, pages, rows;
    uint32_t here;  // rows' positions by this launch too
};

// Pages of t tokens, in a table of `width`.
CHK_DEV uint32_t plan_pages(uint32_t t, uint32_t page_log2, uint32_t width) {
    const uint32_t h = (t >> page_log2) + ((t & ((1u << page_log2) - 1)) ? 1u : 0u);
    return h < width ? h : width;
}

// Position and slot of row r, in sequence b whose rows end at `end`, tokens `now`.
CHK_DEV void plan_row(const PlanArgs& a, uint32_t r, uint32_t b, uint32_t end, uint32_t now) {
    const uint32_t p = now - (end - r);
    if (a.pos) a.pos[r] = p;
    if (a.slot) {
        const uint32_t id = kv4_page(a.table + (size_t)b * a.width, a.width, a.page_log2, a.pages, p);
        a.slot[r] = id == KV4_NO_PAGE ? ~0ull : ((uint64_t)id << a.page_log2) + (p & ((1u << a.page_log2) - 1));
    }
}
CHK_DEV void plan_no_row(const PlanArgs& a, uint32_t r) {
    if (a.pos) a.pos[r] = 0xffffffffu;
    if (a.slot) a.slot[r] = ~0ull;
}

// The first of sums[0..n) (rising) above x.
CHK_DEV uint32_t plan_find(const uint32_t* sums, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (sums[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_WG) k_kv4_plan(PlanArgs a) {
    constexpr uint32_t WAVES = PLAN_WG / 64;
    __shared__ uint32_t part[4][WAVES];
    __shared__ uint32_t back_to[KV4_MAX_SEQS], need_to[KV4_MAX_SEQS], rows_to[KV4_MAX_SEQS];  // inclusive sums
    __shared__ uint32_t back_lo[KV4_MAX_SEQS], held[KV4_MAX_SEQS], now[KV4_MAX_SEQS];
    __shared__ uint32_t taken, gone;
    const uint32_t b = threadIdx.x, lane = b & 63, w = wave_id();
    const bool live = b < a.n;
    // inclusive sum over the workgroup; slot: LDS of its own a call
    auto scan = [&](uint32_t v, uint32_t slot, uint32_t& total) {
        v = wave_scan(v);
        if (lane == 63) part[slot][w] = v;
        __syncthreads();
        const uint32_t t = wave_scan(lane < WAVES ? part[slot][lane] : 0u);
        total = (uint32_t)__builtin_amdgcn_readlane((int)t, WAVES - 1);
        return v + (w ? (uint32_t)__builtin_amdgcn_readlane((int)t, (int)w - 1) : 0u);
    };
    const uint32_t len = live ? a.len[b] : 0u, keep = live && a.keep ? a.keep[b] : 0xffffffffu;
    const uint32_t own = live && a.own ? a.own[b] : 0u;
    uint32_t want = live ? a.want[b] : 0u;
    const uint32_t nfree = min(a.nfree[0], a.pages);
    if (threadIdx.x == 0) taken = gone = 0u;

    // ---- cut back
    const uint32_t l = min(len, keep), h0 = plan_pages(len, a.page_log2, a.width), h1 = plan_pages(l, a.page_log2, a.width);
    const uint32_t lo = max(h1, own), back = h0 > lo ? h0 - lo : 0u;
    // ---- rows go on in the page where what is left ends: not in another's
    if ((l & ((1u << a.page_log2) - 1)) && own <= a.width && l >> a.page_log2 < own) want = 0u;
    // ---- wants that table and row arrays hold (any above `rows` counts as that much: the sum stays in 32 bits)
    if ((uint64_t)l + want > (uint64_t)a.width << a.page_log2) want = 0u;
    uint32_t backs, wants;
    const uint32_t bsum = scan(back, 0, backs);
    if (live) {
        back_to[b] = bsum;
        back_lo[b] = lo;
    }
    if (scan(min(want, a.rows + 1), 1, wants) > a.rows) want = 0u;
    // ---- number i of the entries given back is entry back_lo + i - (those of the sequences before)
    auto entry = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t s = plan_find(back_to, a.n, i);
        const uint32_t e = s < a.n ? back_lo[s] + i - (s ? back_to[s - 1] : 0u) : a.width;
        return e < a.width ? a.table + (size_t)s * a.width + e : nullptr;
    };
    // those that name no page (a thread's first entry is kept: one dependent load less further down)
    uint32_t *first = nullptr, id = 0u;
    for (uint32_t i0 = 64 * w; i0 < backs; i0 += PLAN_WG) {
        uint32_t* p = i0 + lane < backs ? entry(i0 + lane) : nullptr;
        const uint32_t x = p ? *p : KV4_NO_PAGE;
        const uint64_t none = __ballot(i0 + lane < backs && x >= a.pages);
        if (none && lane == 0) atomicAdd(&gone, (uint32_t)__builtin_popcountll(none));
        if (i0 == 64 * w) first = p, id = x;
    }
    if (backs) __syncthreads();
    const uint32_t lost = gone;
    // ---- and the pages
    const uint32_t avail = min(nfree + (backs - lost), a.pages);
    uint32_t need = plan_pages(l + want, a.page_log2, a.width) - h1, needs, rows;
    const uint32_t nsum = scan(need, 2, needs);
    if (need && nsum > avail) want = need = 0u;
    const uint32_t rsum = scan(want, 3, rows);
    if (live) {
        need_to[b] = nsum;
        rows_to[b] = rsum;
        held[b] = h1;
        now[b] = l + want;
        a.len[b] = l + want;
        a.start[b] = rsum - want;
        if (need) atomicMax(&taken, nsum);
    }
    if (b + 1 == a.n) a.start[a.n] = rsum;
    __syncthreads();

    // ---- pages given back: the list takes them in the opposite order
    auto give = [&](uint32_t* p, uint32_t x, uint32_t at) __attribute__((always_inline)) {
        if (at < a.pages) a.free[at] = x;
        *p = KV4_NO_PAGE;
    };
    if (!lost) {
        if (first) give(first, id, nfree + (backs - 1 - b));
        for (uint32_t i = b + PLAN_WG; i < backs; i += PLAN_WG) {
            uint32_t* p = entry(i);
            give(p, *p, nfree + (backs - 1 - i));
        }
    } else {  // a place is the number of those that name a page before it
        uint32_t at = nfree, slot = 0u, named;
        for (uint32_t j0 = 0; j0 < backs; j0 += PLAN_WG, at += named, slot ^= 1u) {
            uint32_t* p = j0 + b < backs ? entry(backs - 1 - (j0 + b)) : nullptr;
            const uint32_t x = p ? *p : KV4_NO_PAGE, is = x < a.pages ? 1u : 0u, upto = scan(is, slot, named);
            if (is) give(p, x, at + upto - 1);
            else if (p) *p = KV4_NO_PAGE;
        }
    }
    __syncthreads();
    // ---- pages taken, from the list's end
    const uint32_t take = taken;
    for (uint32_t i = threadIdx.x; i < take; i += PLAN_WG) {
        const uint32_t s = plan_find(need_to, a.n, i);
        if (s >= a.n) break;
        const uint32_t e = held[s] + i - (s ? need_to[s - 1] : 0u);
        if (e < a.width) a.table[(size_t)s * a.width + e] = a.free[avail - 1 - i];
    }
    if (threadIdx.x == 0) {
        a.nfree[0] = avail - take;
        a.nfree[1] = needs > avail ? needs - avail : 0u;
    }
    if (!a.here) return;
    __syncthreads();
    for (uint32_t r = threadIdx.x; r < a.rows; r += PLAN_WG) {
        if (r >= rows) plan_no_row(a, r);
        else {
            const uint32_t s = plan_find(rows_to, a.n, r);
            plan_row(a, r, s, rows_to[s], now[s]);
        }
    }
}

// The rows of a plan that has many: start, len and table as the state's launch left them.
__global__ void __launch_bounds__(256) k_kv4_plan_rows(PlanArgs a) {
    __shared__ uint32_t to[KV4_MAX_SEQS], now[KV4_MAX_SEQS];
    for (uint32_t i = threadIdx.x; i < a.n; i += CHK_WG) {
        to[i] = a.start[i + 1];
        now[i] = a.len[i];
    }
    __syncthreads();
    const uint32_t r = blockIdx.x * CHK_WG + threadIdx.x;
    if (r >= a.rows) return;
    const uint32_t s = plan_find(to, a.n, r);
    if (s >= a.n) plan_no_row(a, r);
    else plan_row(a, r, s, to[s], now[s]);
}

static void plan_call(const ChkKvPool* pool, const uint32_t* keep, const uint32_t* own, const uint32_t* want, uint32_t rows,
                      uint32_t* start, uint32_t* pos, uint64_t* slot, void* stream) {
    kv4_ensure(pool, "no pool given");
    kv4_ensure(pool->n <= KV4_MAX_SEQS, "at most 1024 sequences a call");
    kv4_page_size(pool->page);
    kv4_ensure(pool->pages >= 1 && pool->pages < 0xffffffffu, "a pool has at least one page");
    kv4_ensure((uint64_t)pool->table_width * pool->page <= 1u << 30, "a sequence's table may hold 2^30 tokens");
    // (sums of entries given back, and the loops over them, in 32 bits)
    kv4_ensure((uint64_t)pool->n * pool->table_width <= 1u << 31, "a pool's tables may hold 2^31 entries");
    kv4_ensure(rows < PLAN_ROWS, "at most 2^21 - 1 rows a plan");
    kv4_ensure(pool->n > 0 || rows == 0, "rows without a sequence");
    if (pool->n == 0) return;
    kv4_ensure(pool->table_width >= 1, "a sequence's table must name at least one page");
    kv4_ensure(pool->table && pool->len && pool->free && pool->nfree, "null table, len, free or nfree");
    kv4_ensure(want && start, "null want or start");
    kv4_ensure(kv4_aligned(pool->table, 4) && kv4_aligned(pool->len, 4) && kv4_aligned(pool->free, 4) &&
                   kv4_aligned(pool->nfree, 4) && kv4_aligned(keep, 4) && kv4_aligned(own, 4) && kv4_aligned(want, 4) &&
                   kv4_aligned(start, 4) && kv4_aligned(pos, 4),
               "a pool's and a plan's arrays must be 4-byte aligned");
    kv4_ensure(kv4_aligned(slot, 8), "slot must be 8-byte aligned");
    const hipStream_t st = (hipStream_t)stream;
    kv4_on_device({pool->table, pool->len, pool->free, pool->nfree, want, start, keep ? keep : want, own ? own : want,
                   pos ? pos : start, slot ? (const void*)slot : start}, st);
    PlanArgs a{pool->table, pool->len, pool->free, pool->nfree, keep, own, want, start, pos, slot,
               pool->n, pool->table_width, kv4_log2(pool->page), pool->pages, rows, 0};
    const bool any = rows && (pos || slot);
    // 4096 rows are four a thread of the state's workgroup
    a.here = any && rows <= 4 * PLAN_WG;
    kv4_launch(k_kv4_plan, dim3(1), PLAN_WG, st, a);
    if (any && !a.here) kv4_launch(k_kv4_plan_rows, dim3((rows + CHK_WG - 1) / CHK_WG), CHK_WG, st, a);
}

}  // namespace chk

using namespace chk;

extern "C" int chk_kv_plan_q4(const ChkKvPool* pool, const uint32_t* keep, const uint32_t* own, const uint32_t* want,
                              uint32_t rows, uint32_t* start, uint32_t* pos, uint64_t* slot, void* stream) {
    return kv4_try([&] { plan_call(pool, keep, own, want, rows, start, pos, slot, stream); });
}
