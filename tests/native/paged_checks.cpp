// What the calls on a paged cache refuse, the rows of a sequence and what a row sees (csrc/paged_plan.h), checked without a GPU.
#include <cstdio>
#include <cstring>
#include <functional>
#include <vector>

#include "paged_plan.h"

static int failures = 0;
static void expect(bool ok, const char* what) {
    if (!ok) {
        std::printf("%s\n", what);
        ++failures;
    }
}

int main() {
    alignas(16) static float mem[64];
    static int32_t table[4];
    static uint32_t lens[2], other[2];
    cera_hip_paged_kv c{};
    c.kv_type = CERA_HIP_KV_F16; c.n_kv_heads = 2; c.head_dim = 64; c.page_size = 16; c.n_pages = 5; c.n_seqs = 2; c.max_pages = 2; c.k = mem; c.v = mem; c.table = table; c.lens = lens;
    cera_hip_paged_attn a{};
    a.q = mem; a.out = mem; a.n_rows = 2; a.n_heads = 4; a.scale = 1.0f;
    cera_hip_paged_evict e{};
    e.mass = mem; e.mass_stride = 32; e.new_lens = other; e.budget = 8; e.n_first = 4; e.n_recent = 4;
    cera_hip_verify_draft d{};
    d.n_seqs = 1; d.max_draft = 2; d.vocab = 10; d.temperature = 1.0f; d.target = mem; d.tokens = table; d.uniform = mem; d.accepted = lens; d.out_tokens = table;
    expect(!paged_check_attn(&c, &a).msg && !paged_check_evict(&c, &e).msg && !verify_check(&d).msg, "valid calls");

    auto kv = [&](cera_hip_status st, const char* what, const std::function<void(cera_hip_paged_kv&)>& f) {
        cera_hip_paged_kv x = c;
        f(x);
        for (const PagedCheck& r : {paged_check_kv(&x), paged_check_attn(&x, &a), paged_check_evict(&x, &e)}) expect(r.msg && r.st == st, what);
    };
    kv(CERA_HIP_ERR_UNSUPPORTED_DTYPE, "type", [](auto& x) { x.kv_type = 2; });
    kv(CERA_HIP_ERR_ARGUMENT, "null k", [](auto& x) { x.k = nullptr; });
    kv(CERA_HIP_ERR_ARGUMENT, "null table", [](auto& x) { x.table = nullptr; });
    kv(CERA_HIP_ERR_ARGUMENT, "k alignment", [](auto& x) { x.k = reinterpret_cast<char*>(mem) + 8; });
    kv(CERA_HIP_ERR_SHAPE, "head size", [](auto& x) { x.head_dim = 96; });
    for (uint32_t p : {0u, 8u, 24u, 512u}) kv(CERA_HIP_ERR_SHAPE, "page size", [=](auto& x) { x.page_size = p; });
    kv(CERA_HIP_ERR_SHAPE, "no kv heads", [](auto& x) { x.n_kv_heads = 0; });
    kv(CERA_HIP_ERR_SHAPE, "no pages", [](auto& x) { x.n_pages = 0; });
    kv(CERA_HIP_ERR_SHAPE, "too many pages", [](auto& x) { x.n_pages = 0x80000000u; });
    kv(CERA_HIP_ERR_SHAPE, "too many positions", [](auto& x) { x.max_pages = (1u << 26) + 1; });
    kv(CERA_HIP_ERR_SHAPE, "too many sequences", [](auto& x) { x.n_seqs = 65536; });
    for (uint64_t s : {2047ull, 2044ull, 2052ull, ~0ull & ~7ull}) kv(CERA_HIP_ERR_SHAPE, "page stride", [=](auto& x) { x.page_stride = s; });

    auto attn = [&](cera_hip_status st, const char* what, const std::function<void(cera_hip_paged_attn&)>& f) {
        cera_hip_paged_attn x = a;
        f(x);
        const PagedCheck r = paged_check_attn(&c, &x);
        expect(r.msg && r.st == st, what);
    };
    attn(CERA_HIP_ERR_ARGUMENT, "null q", [](auto& x) { x.q = nullptr; });
    attn(CERA_HIP_ERR_ARGUMENT, "k_new alone", [](auto& x) { x.k_new = mem; });
    attn(CERA_HIP_ERR_SHAPE, "heads", [](auto& x) { x.n_heads = 3; });
    attn(CERA_HIP_ERR_SHAPE, "no heads", [](auto& x) { x.n_heads = 0; });
    attn(CERA_HIP_ERR_ARGUMENT, "scale", [](auto& x) { x.scale = INFINITY; });
    attn(CERA_HIP_ERR_ARGUMENT, "scale too large", [](auto& x) { x.scale = -2e30f; });
    attn(CERA_HIP_ERR_SHAPE, "heads of a kv head", [](auto& x) { x.n_heads = 2050; });
    attn(CERA_HIP_ERR_SHAPE, "rows", [](auto& x) { x.n_rows = 3; });
    attn(CERA_HIP_ERR_SHAPE, "q stride", [](auto& x) { x.q_stride = 255; });
    attn(CERA_HIP_ERR_SHAPE, "q stride of odd size", [](auto& x) { x.q_stride = 257; });
    attn(CERA_HIP_ERR_SHAPE, "kv stride", [](auto& x) { x.kv_stride = 64; });
    attn(CERA_HIP_ERR_ARGUMENT, "out alignment", [](auto& x) { x.out = mem + 1; });
    attn(CERA_HIP_ERR_ARGUMENT, "mass with chunks", [&](auto& x) { x.mass = mem; x.mass_stride = 32; x.q_first = lens; });
    attn(CERA_HIP_ERR_SHAPE, "mass stride", [](auto& x) { x.mass = mem; x.mass_stride = 31; });
    {
        cera_hip_paged_attn x = a;
        x.mass = mem; x.mass_stride = 20; x.max_len = 20;
        expect(!paged_check_attn(&c, &x).msg, "mass stride of max_len");
    }
    auto ev = [&](cera_hip_status st, const char* what, const std::function<void(cera_hip_paged_evict&)>& f) {
        cera_hip_paged_evict x = e;
        f(x);
        const PagedCheck r = paged_check_evict(&c, &x);
        expect(r.msg && r.st == st, what);
    };
    ev(CERA_HIP_ERR_ARGUMENT, "null mass", [](auto& x) { x.mass = nullptr; });
    ev(CERA_HIP_ERR_ARGUMENT, "new_lens in place", [&](auto& x) { x.new_lens = lens; });
    ev(CERA_HIP_ERR_SHAPE, "no budget", [](auto& x) { x.budget = 0; x.n_first = x.n_recent = 0; });
    ev(CERA_HIP_ERR_SHAPE, "ends over the budget", [](auto& x) { x.n_recent = 5; });
    ev(CERA_HIP_ERR_SHAPE, "ends that wrap", [](auto& x) { x.n_first = 0xFFFFFFFFu; x.n_recent = 9; });
    ev(CERA_HIP_ERR_SHAPE, "mass stride", [](auto& x) { x.mass_stride = 31; });
    auto vd = [&](cera_hip_status st, const char* what, const std::function<void(cera_hip_verify_draft&)>& f) {
        cera_hip_verify_draft x = d;
        f(x);
        const PagedCheck r = verify_check(&x);
        expect(r.msg && r.st == st, what);
    };
    vd(CERA_HIP_ERR_ARGUMENT, "null target", [](auto& x) { x.target = nullptr; });
    vd(CERA_HIP_ERR_ARGUMENT, "temperature", [](auto& x) { x.temperature = -1.0f; });
    vd(CERA_HIP_ERR_ARGUMENT, "temperature NaN", [](auto& x) { x.temperature = NAN; });
    vd(CERA_HIP_ERR_ARGUMENT, "temperature too high", [](auto& x) { x.temperature = 2e6f; });
    vd(CERA_HIP_ERR_SHAPE, "vocabulary", [](auto& x) { x.vocab = 0; });
    vd(CERA_HIP_ERR_SHAPE, "drafts", [](auto& x) { x.max_draft = 65; });
    vd(CERA_HIP_ERR_SHAPE, "no drafts", [](auto& x) { x.max_draft = 0; });
    vd(CERA_HIP_ERR_SHAPE, "row stride", [](auto& x) { x.row_stride = 9; });

    // rows of a sequence
    const uint32_t n[5] = {40, 20, 30, 8, 0}, f[6] = {3, 1, 8, 11, 21, 20};
    struct Want { uint32_t first, n; bool bad; };
    const Want want[5] = {{3, 0, true}, {1, 7, true}, {8, 3, false}, {11, 9, true}, {20, 0, true}};
    for (uint32_t s = 0; s < 5; ++s) {
        const PagedRows r = paged_chunk_rows(f[s], f[s + 1], n[s], 20, 6, 64);
        expect(r.first == want[s].first && r.n == want[s].n && r.bad == want[s].bad, "rows of a sequence");
        expect(static_cast<uint64_t>(r.first) + r.n <= 20, "rows stay in bounds");
    }
    expect(paged_one_row(0, n[0], 39).bad && !paged_one_row(4, n[4], 39).bad, "lengths of the decode form");
    // what a row sees, against the definition
    for (uint32_t P = 0; P < 40; ++P)
        for (uint32_t w : {0u, 1u, 7u, 16u, 39u, 40u, 100u, 0xFFFFFFFFu})
            for (uint32_t k : {0u, 1u, 4u, 20u, 100u, 0xFFFFFFFFu}) {
                const PagedSeen v = paged_seen(P, w, k);
                expect(v.sink_end <= v.start, "sinks end before the window");
                for (uint64_t t = 0; t <= P; ++t) {
                    const bool in = t < k || w == 0 || t + w > P, got = t < v.sink_end || t >= v.start;
                    expect(in == got, "what a row sees");
                }
            }
    // parts: a kv head's workgroups fit the chip twice, and the count of all tiles fits 32 bits
    for (uint32_t len : {1u, 300u, 5000u, 1u << 30})
        for (uint32_t seqs : {1u, 64u, 65535u})
            for (uint32_t wide : {1u, 8u, 100u, 300u, 5000u})
                for (uint32_t window : {0u, 1000u, 0xFFFFFFFFu})
                    for (bool chunk : {false, true})
                      for (bool half : {false, true}) {
                        const PagedCut cut = paged_cut(len, 7, window, 4, 32, wide, seqs, chunk, half, 256);
                        expect(cut.least >= 1 && static_cast<uint64_t>(cut.spans) * wide <= 1024, "parts of a sequence");
                        expect(cut.spans == 0 || (window && window < len) || (static_cast<uint64_t>(len) + 31) / 32 * seqs < 0x80000000ull, "tiles fit 32 bits");
                    }
    return failures != 0;
}
