// Device-side view of a paged cache (cera_hip_paged_kv), shared by its kernels.
#pragma once
#include "common.hip.h"
#include "host_common.h"
#include "paged_plan.h"

struct PagedView {
    const int32_t* table;
    const uint32_t* lens;
    uint64_t page_stride, head_stride;   // elements
    uint32_t n_kv, n_pages, max_pages, page_log2, max_len;
};
static inline PagedView paged_view(const cera_hip_paged_kv& c, uint32_t max_len) {
    PagedView v{};
    v.table = c.table;
    v.lens = c.lens;
    v.page_stride = paged_stride(c);
    v.head_stride = static_cast<uint64_t>(c.page_size) * c.head_dim;
    v.n_kv = c.n_kv_heads;
    v.n_pages = c.n_pages;
    v.max_pages = c.max_pages;
    v.page_log2 = static_cast<uint32_t>(__builtin_ctz(c.page_size));
    v.max_len = paged_max_len(c, max_len);
    return v;
}

// What no kernel of the call writes, by scalar loads where the index is the same in all lanes: a vector load's wait is one for all
// loads in flight before it.
template <typename T> using PagedConst = const __attribute__((address_space(4))) T*;
template <typename T> __device__ __forceinline__ PagedConst<T> paged_const(const T* p) { return (PagedConst<T>)p; }

__device__ __forceinline__ PagedRows paged_rows(const uint32_t* q_first, const uint32_t* lens, uint32_t s, uint32_t n_rows, uint32_t max_queries, uint32_t max_len) {
    const uint32_t len = paged_const(lens)[s];
    return q_first ? paged_chunk_rows(paged_const(q_first)[s], paged_const(q_first)[s + 1], len, n_rows, max_queries, max_len) : paged_one_row(s, len, max_len);
}

// The page of position t (t < max_len, so the table has its column); *ok turns false where the table names none of the pool's, and the
// page is then 0, whose memory is there.
__device__ __forceinline__ uint32_t paged_page(const PagedView& v, uint32_t seq, uint32_t t, bool& ok) {
    const uint32_t p = static_cast<uint32_t>(v.table[static_cast<uint64_t>(seq) * v.max_pages + (t >> v.page_log2)]);
    if (p >= v.n_pages) ok = false;
    return p < v.n_pages ? p : 0u;
}
// element of position t's row of kv head g
template <int HD>
__device__ __forceinline__ uint64_t paged_row(const PagedView& v, uint32_t page, uint32_t g, uint32_t t) {
    return page * v.page_stride + g * v.head_stride + static_cast<uint64_t>(t & ((1u << v.page_log2) - 1)) * HD;
}

// Rows that nothing reads again before the caches have seen much else.
template <typename T> using PagedRaw = uint32_t __attribute__((ext_vector_type(sizeof(T) / 4)));
template <typename T> __device__ __forceinline__ T paged_stream(const void* p) { return __builtin_bit_cast(T, __builtin_nontemporal_load(static_cast<const PagedRaw<T>*>(p))); }
template <typename T> __device__ __forceinline__ void paged_stream(void* p, T x) { __builtin_nontemporal_store(__builtin_bit_cast(PagedRaw<T>, x), static_cast<PagedRaw<T>*>(p)); }

// Infinities and NaN have the largest exponent: the magnitudes' running maximum, as integers, tells whether any is among many.
typedef unsigned short paged_u2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t paged_most(uint32_t top, uint32_t pair) {   // of halves, both of a pair at once
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(paged_u2, top), __builtin_bit_cast(paged_u2, pair & 0x7FFF7FFFu)));
}
__device__ __forceinline__ uint32_t paged_most(uint32_t top, float x) { return max(top, __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu); }
__device__ __forceinline__ bool paged_odd_pair(uint32_t x) { return (x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u; }
__device__ __forceinline__ bool paged_odd(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7F800000u) == 0x7F800000u; }
// the value, 0 in the place of such a one
__device__ __forceinline__ uint32_t paged_even(uint32_t x) { return x & ~(((x & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((x & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u)); }
__device__ __forceinline__ float paged_even(float x) { return paged_odd(x) ? 0.0f : x; }

// The context's device while a call lasts: a caller may have made another one current.
struct PagedDevice {
    int before = -1;
    hipError_t err = hipSuccess;
    explicit PagedDevice(int device) {
        if ((err = hipGetDevice(&before)) != hipSuccess) { before = -1; return; }
        if (before == device) before = -1;
        else err = hipSetDevice(device);
    }
    ~PagedDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
