// Calls that the contract of the paged cache's operators allows, and what they need (csrc/paged_plan.h), checked without a GPU.
#include <cstdio>

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
    static uint32_t lens[2], first[3];
    cera_hip_paged_kv c{};
    c.kv_type = CERA_HIP_KV_F16; c.n_kv_heads = 2; c.head_dim = 64; c.page_size = 16; c.n_pages = 5; c.n_seqs = 2; c.max_pages = 2; c.k = mem; c.v = mem; c.table = table; c.lens = lens;
    // a chunk's new positions' weights set to 0
    cera_hip_paged_attn a{};
    a.q = mem; a.out = mem; a.n_rows = 9; a.n_heads = 4; a.scale = 1.0f; a.q_first = first; a.mass = mem; a.mass_stride = 32; a.mass_fresh = 1; a.k_new = mem; a.v_new = mem;
    expect(!paged_check_attn(&c, &a).msg, "mass of a chunk");
    auto no = [&](cera_hip_status st, const char* what, auto f) {
        cera_hip_paged_attn x = a;
        f(x);
        const PagedCheck r = paged_check_attn(&c, &x);
        expect(r.msg && r.st == st, what);
    };
    no(CERA_HIP_ERR_ARGUMENT, "mass of a chunk that is not to be set", [](auto& x) { x.mass_fresh = 0; });
    no(CERA_HIP_ERR_ARGUMENT, "mass of a chunk without new rows", [](auto& x) { x.k_new = x.v_new = nullptr; });
    no(CERA_HIP_ERR_SHAPE, "mass stride of a chunk", [](auto& x) { x.mass_stride = 31; });
    // at temperature 0 no random number and no draft's distribution is read
    cera_hip_verify_draft d{};
    d.n_seqs = 1; d.max_draft = 2; d.vocab = 10; d.target = mem; d.tokens = table; d.accepted = lens; d.out_tokens = table;
    expect(!verify_check(&d).msg, "no random numbers at temperature 0");
    d.temperature = 1e-30f;
    expect(verify_check(&d).msg && verify_check(&d).st == CERA_HIP_ERR_ARGUMENT, "no random numbers at a temperature");
    return failures != 0;
}
