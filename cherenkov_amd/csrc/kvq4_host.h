// Host side of the 4-bit cache's entry points: argument checks, the dispatch
// on head dim and type, and errors as the C ABI reports them.
#pragma once

#include <hip/hip_runtime.h>

#include <exception>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "internal.h"
#include "kvq4.h"

namespace chk {

constexpr uint32_t KV4_MIN_PAGE = 16;

inline void kv4_ensure(bool ok, const char* msg) {
    if (!ok) throw std::runtime_error(msg);
}

// Runs an entry point's body; no exception leaves it.
template <class F>
int kv4_try(F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        g_err = e.what();
    } catch (...) {
        g_err = "unknown error";
    }
    return -1;
}

inline uint32_t kv4_log2(uint32_t v) {
    uint32_t l = 0;
    while ((1u << l) < v && l < 31) ++l;
    return l;
}

inline bool kv4_aligned(const void* p, uint64_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

inline Kv4Cache kv4_cache(const ChkKvQ4* c) {
    kv4_ensure(c, "no cache given");
    kv4_ensure(c->hd == 128 || c->hd == 256, "head_dim must be 128 or 256");
    kv4_ensure(c->nkv >= 1 && c->nkv <= 1024, "1..=1024 kv heads");
    kv4_ensure(c->page >= KV4_MIN_PAGE && c->page <= 1u << 20 && (c->page & (c->page - 1)) == 0,
               "page must be a power of two of 16..=1048576 tokens");
    kv4_ensure(c->pages >= 1 && c->pages < 0xffffffffu, "a cache has at least one page");
    kv4_ensure(c->k && c->v && c->ks && c->vs, "null cache plane");
    kv4_ensure(kv4_aligned(c->k, 16) && kv4_aligned(c->v, 16) && kv4_aligned(c->ks, 16) && kv4_aligned(c->vs, 16),
               "cache planes must be 16-byte aligned");
    return Kv4Cache{(uint8_t*)c->k, (uint8_t*)c->v, (uint32_t*)c->ks, (uint32_t*)c->vs, c->pages, kv4_log2(c->page), c->nkv};
}

inline Kv4Seqs kv4_seqs(const ChkKvQ4* c, const ChkKvSeqs* s) {
    kv4_ensure(s, "no sequences given");
    kv4_ensure(s->n <= KV4_MAX_SEQS, "at most 1024 sequences a call");
    kv4_ensure(s->n > 0 || s->rows == 0, "rows without a sequence");
    kv4_ensure((uint64_t)s->table_width * c->page <= 1u << 30, "a sequence's table may hold 2^30 tokens");
    if (s->rows) {
        kv4_ensure(s->table_width >= 1, "a sequence's table must name at least one page");
        kv4_ensure(s->table && s->len && s->start, "null table, len or start");
        kv4_ensure(kv4_aligned(s->table, 4) && kv4_aligned(s->len, 4) && kv4_aligned(s->start, 4),
                   "table, len and start must be 4-byte aligned");
    }
    return Kv4Seqs{s->table, s->len, s->start, s->n, s->table_width, s->rows};
}

inline uint32_t kv4_dtype(uint32_t dtype) {
    kv4_ensure(dtype == CHK_F32 || dtype == CHK_F16 || dtype == CHK_BF16, "dtype must be CHK_F32, CHK_F16 or CHK_BF16");
    return dtype == CHK_F32 ? 4 : 2;
}

// A rows argument: 16-byte accesses within a row of `row` elements.
inline void kv4_rows_arg(const void* p, uint64_t stride, uint64_t row, uint32_t dtype, const char* name) {
    const uint64_t size = kv4_dtype(dtype);
    const std::string n(name);
    if (!p) throw std::runtime_error("null " + n);
    if (!kv4_aligned(p, 16) || (stride * size) % 16) throw std::runtime_error(n + " rows must be 16-byte aligned");
    if (stride < row || stride > (1ull << 40)) throw std::runtime_error(n + " row stride shorter than a row");
}

// Every pointer of a call is memory of the current device, and the stream is
// the device's: memory of another device or of the host would fault in the
// kernel.
inline void kv4_on_device(std::initializer_list<const void*> ptrs, hipStream_t st) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) throw std::runtime_error("no device");
    for (const void* p : ptrs) {
        hipPointerAttribute_t a{};
        const hipError_t e = hipPointerGetAttributes(&a, p);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            throw std::runtime_error("an argument is not device memory");
        }
        if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged)
            throw std::runtime_error("an argument is not device memory");
        if (a.device != dev) throw std::runtime_error("an argument lies on another device than the current one");
    }
    hipDevice_t of = dev;
    if (st && hipStreamGetDevice(st, &of) != hipSuccess) {
        (void)hipGetLastError();
        throw std::runtime_error("not a stream");
    }
    if (of != dev) throw std::runtime_error("the stream is another device's than the current one");
}

// Launches a kernel and reports its own status (an error that an earlier call
// of the program left behind is not this call's).
template <class... A>
void kv4_launch(void (*fn)(A...), dim3 grid, uint32_t threads, hipStream_t st, A... a) {
    void* args[] = {&a...};
    const hipError_t e = hipLaunchKernel((const void*)fn, grid, dim3(threads), args, 0, st);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        throw std::runtime_error(std::string("HIP launch error ") + hipGetErrorString(e));
    }
}

template <class T>
struct Kv4Type {
    using type = T;
};

template <class F>
void kv4_switch(uint32_t hd, uint32_t dtype, F&& f) {
    auto on = [&](auto h) {
        if (dtype == CHK_F32) f(h, Kv4Type<float>{});
        else if (dtype == CHK_F16) f(h, Kv4Type<_Float16>{});
        else f(h, Kv4Type<__bf16>{});
    };
    if (hd == 128) on(std::integral_constant<int, 128>{});
    else on(std::integral_constant<int, 256>{});
}

}  // namespace chk
