// What the calls on a paged cache check on the host, and which positions a row sees.  Plain arithmetic, without the device's headers.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "cera_hip.h"

#if defined(__HIPCC__)
#define PAGED_HD __host__ __device__ inline
#else
#define PAGED_HD inline
#endif

struct PagedCheck {
    cera_hip_status st;
    const char* msg;   // null: in order
};
inline PagedCheck paged_no(cera_hip_status st, const char* msg) { return {st, msg}; }
inline bool paged_aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

inline uint64_t paged_capacity(const cera_hip_paged_kv& c) { return static_cast<uint64_t>(c.max_pages) * c.page_size; }
inline uint64_t paged_stride(const cera_hip_paged_kv& c) {
    return c.page_stride ? c.page_stride : static_cast<uint64_t>(c.n_kv_heads) * c.page_size * c.head_dim;
}
// the longest sequence that a call may meet
inline uint32_t paged_max_len(const cera_hip_paged_kv& c, uint32_t max_len) {
    const uint64_t cap = paged_capacity(c);
    return static_cast<uint32_t>(max_len ? std::min<uint64_t>(max_len, cap) : cap);
}

inline PagedCheck paged_check_kv(const cera_hip_paged_kv* c) {
    if (!c) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged cache: null");
    if (c->kv_type != CERA_HIP_KV_F32 && c->kv_type != CERA_HIP_KV_F16) return paged_no(CERA_HIP_ERR_UNSUPPORTED_DTYPE, "paged cache: kv_type is CERA_HIP_KV_F32 or CERA_HIP_KV_F16");
    if (!c->k || !c->v || !c->table || !c->lens) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged cache: k, v, table or lens is null");
    if (c->head_dim != 64 && c->head_dim != 128) return paged_no(CERA_HIP_ERR_SHAPE, "paged cache: head_dim 64 or 128");
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return paged_no(CERA_HIP_ERR_SHAPE, "paged cache: page_size 16, 32, 64, 128 or 256");
    if (c->n_kv_heads == 0 || c->n_kv_heads > 1024) return paged_no(CERA_HIP_ERR_SHAPE, "paged cache: 1 to 1024 kv heads");
    if (c->n_pages == 0 || c->n_pages > 0x7FFFFFFFu || c->max_pages == 0 || paged_capacity(*c) > (1ull << 30)) return paged_no(CERA_HIP_ERR_SHAPE, "paged cache: pages of the pool, pages of a sequence (at most 2^30 positions)");
    if (c->n_seqs > 65535) return paged_no(CERA_HIP_ERR_SHAPE, "paged cache: at most 65535 sequences");
    if (c->page_stride && (c->page_stride % 8 || c->page_stride < static_cast<uint64_t>(c->n_kv_heads) * c->page_size * c->head_dim || c->page_stride > (1ull << 40)))
        return paged_no(CERA_HIP_ERR_SHAPE, "paged cache: page_stride is below a page, or no multiple of 8");
    if (!paged_aligned(c->k, 16) || !paged_aligned(c->v, 16) || !paged_aligned(c->table, 4) || !paged_aligned(c->lens, 4)) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged cache: k and v are 16-byte aligned, table and lens 4-byte");
    return {CERA_HIP_OK, nullptr};
}

inline bool paged_row_stride_ok(uint64_t stride, uint64_t row) { return stride == 0 || (stride >= row && stride % 4 == 0 && stride <= (1ull << 40)); }

inline PagedCheck paged_check_attn(const cera_hip_paged_kv* c, const cera_hip_paged_attn* a) {
    const PagedCheck kv = paged_check_kv(c);
    if (kv.msg) return kv;
    if (!a || !a->q || !a->out) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged attention: q or out is null");
    if (!a->k_new != !a->v_new) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged attention: k_new and v_new come together");
    if (a->n_heads == 0 || a->n_heads % c->n_kv_heads || a->n_heads > 65536) return paged_no(CERA_HIP_ERR_SHAPE, "paged attention: n_heads must be a multiple of n_kv_heads");
    if (a->n_heads / c->n_kv_heads > 1024) return paged_no(CERA_HIP_ERR_SHAPE, "paged attention: at most 1024 query heads a kv head");
    if (!(std::fabs(a->scale) <= 1e30f)) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged attention: scale must be finite, at most 10^30");
    if (!a->q_first && a->n_rows != c->n_seqs) return paged_no(CERA_HIP_ERR_SHAPE, "paged attention: without q_first there is one row a sequence");
    if (a->n_rows > (1u << 30)) return paged_no(CERA_HIP_ERR_SHAPE, "paged attention: at most 2^30 rows");
    const uint64_t q_row = static_cast<uint64_t>(a->n_heads) * c->head_dim, kv_row = static_cast<uint64_t>(c->n_kv_heads) * c->head_dim;
    if (!paged_row_stride_ok(a->q_stride, q_row) || !paged_row_stride_ok(a->out_stride, q_row) || !paged_row_stride_ok(a->kv_stride, kv_row))
        return paged_no(CERA_HIP_ERR_SHAPE, "paged attention: a stride is below a row, or no multiple of 4");
    if (!paged_aligned(a->q, 16) || !paged_aligned(a->out, 16) || !paged_aligned(a->k_new, 16) || !paged_aligned(a->v_new, 16) || !paged_aligned(a->q_first, 4) || !paged_aligned(a->mass, 4))
        return paged_no(CERA_HIP_ERR_ARGUMENT, "paged attention: q, k_new, v_new and out are 16-byte aligned, q_first and mass 4-byte");
    if (a->mass && a->q_first && !(a->mass_fresh && a->k_new)) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged attention: mass with q_first only sets the new positions' to 0 (mass_fresh, k_new)");
    if (a->mass && (a->mass_stride < paged_max_len(*c, a->max_len) || a->mass_stride > (1ull << 40))) return paged_no(CERA_HIP_ERR_SHAPE, "paged attention: mass_stride is below the longest sequence");
    return {CERA_HIP_OK, nullptr};
}

inline PagedCheck paged_check_evict(const cera_hip_paged_kv* c, const cera_hip_paged_evict* e) {
    const PagedCheck kv = paged_check_kv(c);
    if (kv.msg) return kv;
    if (!e || !e->mass || !e->new_lens) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged eviction: mass or new_lens is null");
    if (e->new_lens == c->lens) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged eviction: new_lens is not lens");
    if (!paged_aligned(e->mass, 4) || !paged_aligned(e->new_lens, 4) || !paged_aligned(e->kept, 4)) return paged_no(CERA_HIP_ERR_ARGUMENT, "paged eviction: mass, new_lens and kept are 4-byte aligned");
    if (e->budget == 0 || e->budget > (1u << 30) || static_cast<uint64_t>(e->n_first) + e->n_recent > e->budget) return paged_no(CERA_HIP_ERR_SHAPE, "paged eviction: n_first + n_recent <= budget, budget from 1");
    if (e->mass_stride < paged_max_len(*c, e->max_len) || e->mass_stride > (1ull << 40)) return paged_no(CERA_HIP_ERR_SHAPE, "paged eviction: mass_stride is below the longest sequence");
    return {CERA_HIP_OK, nullptr};
}

inline PagedCheck verify_check(const cera_hip_verify_draft* d) {
    if (!d || !d->target || !d->tokens || (!d->uniform && d->temperature != 0) || !d->accepted || !d->out_tokens) return paged_no(CERA_HIP_ERR_ARGUMENT, "verify_draft: a pointer is null");
    if (d->vocab == 0 || d->vocab > (1u << 24)) return paged_no(CERA_HIP_ERR_SHAPE, "verify_draft: a vocabulary of 1 to 2^24 tokens");
    if (d->max_draft == 0 || d->max_draft > 64) return paged_no(CERA_HIP_ERR_SHAPE, "verify_draft: 1 to 64 drafted tokens");
    if (d->n_seqs > 65535) return paged_no(CERA_HIP_ERR_SHAPE, "verify_draft: at most 65535 sequences");
    if (!(d->temperature >= 0 && d->temperature <= 1e6f)) return paged_no(CERA_HIP_ERR_ARGUMENT, "verify_draft: a temperature of 0 to 10^6");
    if (d->row_stride && (d->row_stride < d->vocab || d->row_stride > (1ull << 40))) return paged_no(CERA_HIP_ERR_SHAPE, "verify_draft: row_stride is below the vocabulary");
    for (const void* p : {static_cast<const void*>(d->target), static_cast<const void*>(d->draft), static_cast<const void*>(d->tokens), static_cast<const void*>(d->n_draft),
                          static_cast<const void*>(d->uniform), static_cast<const void*>(d->accepted), static_cast<const void*>(d->out_tokens)})
        if (!paged_aligned(p, 4)) return paged_no(CERA_HIP_ERR_ARGUMENT, "verify_draft: pointers are 4-byte aligned");
    return {CERA_HIP_OK, nullptr};
}

// The rows of one sequence in a call.
struct PagedRows {
    uint32_t first, n;   // rows of q and out; n = 0: none
    uint32_t len;        // positions of the sequence; row first + i is at position len - n + i
    bool bad;            // lengths or rows out of order: [first, first + n) get NaN, nothing else is touched
};
// one row a sequence, and rows [a, b)
PAGED_HD PagedRows paged_one_row(uint32_t s, uint32_t len, uint32_t max_len) {
    PagedRows r;
    r.len = len;
    r.first = s;
    r.n = 1;
    r.bad = len > max_len;
    return r;
}
PAGED_HD PagedRows paged_chunk_rows(uint32_t a, uint32_t b, uint32_t len, uint32_t n_rows, uint32_t max_queries, uint32_t max_len) {
    PagedRows r;
    r.len = len;
    r.bad = a > b || b > n_rows || b - a > max_queries || b - a > len || len > max_len;
    r.first = a < n_rows ? a : n_rows;
    const uint32_t end = b < n_rows ? b : n_rows;
    r.n = end > r.first ? end - r.first : 0;
    return r;
}

// Positions that the row at position P sees: [0, sink_end) and [start, P], sink_end <= start.
struct PagedSeen {
    uint32_t sink_end, start;
};
PAGED_HD PagedSeen paged_seen(uint32_t P, uint32_t window, uint32_t n_sink) {
    PagedSeen v;
    v.start = window && P + 1 > window ? P + 1 - window : 0;
    v.sink_end = n_sink < v.start ? n_sink : v.start;
    return v;
}

// How the tiles of a kv head and group of columns are cut among workgroups.  wide: kv heads times groups; chunk: the groups are those of
// a chunk's many columns.
struct PagedCut {
    uint32_t spans;   // workgroups, of equal numbers of tiles; 0: one for each sequence
    uint32_t least;   // tiles of a workgroup at least
};
inline PagedCut paged_cut(uint32_t max_len, uint32_t max_queries, uint32_t window, uint32_t n_sink, uint32_t tile, uint32_t wide, uint32_t n_seqs, bool chunk, bool half, uint32_t n_cu) {
    // tiles that a sequence of max_len may have: those of the window and of the first positions each touch one more at their ends
    uint64_t most = (static_cast<uint64_t>(max_len) + tile - 1) / tile;
    if (window) most = std::min(most, (static_cast<uint64_t>(window) + max_queries + tile - 1) / tile + 1 + (static_cast<uint64_t>(n_sink) + tile - 1) / tile);
    PagedCut c;
    // Parts of about equal size, two workgroups a CU: 84 us for 32 sequences of up to 8000 positions, 90 with one a CU, 92 with three; 31, 32
    // and 41 behind a window of 1024.  Groups of columns that fill the chip by themselves are not cut, nor are short sequences: parts
    // cost a launch more, and their results, 64 KB each of a chunk's 128 columns, are written and read again.
    // Single tokens, half cache, cut and uncut, by the number of workgroups without parts: 8 of them, 500 positions 13.5 and 11.7 us, 900
    // 14.5 and 19.7; 32, 640 18.3 and 16.3, 900 19.5 and 21.3; 192, 1056 behind a window 32.8 and 26.4, 1400 35.0 and 30.9, of up to 1400 26.2 and 27.7, of up
    // to 2000 29.8 and 36.1; 256, 2000 52 and 45, of up to 3000 46 and 52.  F32 cache, a tile of which takes twice as long: 32, of up to 500 23.3
    // and 22.4, 640 21.9 and 26.7; 128, 640 32.7 and 28.6, 900 36.1 and 40.1; 256, 900 52 and 44; 512, of up to 1400 75 and 89.
    // Chunks: up to one workgroup a CU without parts, 300 tokens at 1000 positions 38 and 51 us, 400 tokens 30 and 28, f32 52 and 110, 44 and 50;
    // up to two, two sequences of 600 tokens 52 and 44, 30 tokens at up to 3000 for 48 of them 114 and 135, f32 two of up to 600 57 and 74; two
    // and more, 100 tokens at 2000 149 and 127, at up to 2000 95 and 96, 300 at up to 3000 150 and 145, 100 at up to 4000 149 and 169, f32 six of 700
    // 224 and 183, 100 at up to 2000 158 and 216.
    // Workgroups without parts are counted as if every sequence had max_queries rows, above and here: chunks of few rows beside the longest count for more.
    const uint64_t uncut = static_cast<uint64_t>(wide) * n_seqs;
    uint32_t longest;   // that stays whole
    if (chunk && uncut >= 2 * n_cu) longest = half ? 3200 : 1024;
    else if (chunk && uncut > n_cu) longest = half ? 1024 : 512;
    else if (chunk) longest = half ? 512 : 256;
    else if (uncut >= n_cu) longest = half ? 2048 : 1024;
    else if (8 * uncut >= 3 * n_cu) longest = half ? 1280 : 640;
    else longest = half ? 640 : 384;
    c.least = 256 / tile;
    c.spans = most * tile <= longest || n_cu < wide || most * n_seqs > 0x7FFFFFFFu ? 0 : 2 * n_cu / wide;
    return c;
}
