// Attention of new tokens over a paged cache (cera_hip_paged_attn_dev; contract in include/cera_hip.h).
#include <type_traits>

#include "paged.hip.h"
#include "paged_attn.hip.h"

// ---- the new rows into their pages ---------------------------------------------------------------------------------
// grid = (blocks, sequences); a thread moves four floats of a row's keys and values
template <typename KV, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedView c, KV* __restrict__ kp, KV* __restrict__ vp, const float* __restrict__ k_new,
                                                           const float* __restrict__ v_new, uint64_t kv_stride, const uint32_t* __restrict__ q_first,
                                                           uint32_t n_rows, uint32_t max_queries, float* __restrict__ mass, uint64_t mass_stride) {
    const uint32_t s = blockIdx.y;
    const PagedRows r = paged_rows(q_first, c.lens, s, n_rows, max_queries, c.max_len);
    if (r.bad || r.len == 0) return;
    const uint32_t per_row = c.n_kv * (HD / 4);
    const uint64_t items = static_cast<uint64_t>(r.n) * per_row;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < items; i += gridDim.x * 256ull) {
        const uint32_t row = static_cast<uint32_t>(i / per_row), at = static_cast<uint32_t>(i % per_row), g = at / (HD / 4), c4 = at % (HD / 4);
        const uint32_t t = r.len - r.n + row;
        bool ok = true;
        const uint32_t page = paged_page(c, s, t, ok);
        if (!ok) continue;
        const uint64_t dst = paged_row<HD>(c, page, g, t), src = (r.first + static_cast<uint64_t>(row)) * kv_stride + g * HD;
        KvOps<KV>::st4(kp + dst, c4, *reinterpret_cast<const float4*>(k_new + src + 4 * c4));
        KvOps<KV>::st4(vp + dst, c4, *reinterpret_cast<const float4*>(v_new + src + 4 * c4));
        if (mass && c4 == 0) mass[(static_cast<uint64_t>(s) * c.n_kv + g) * mass_stride + t] = 0.0f;
    }
}

// ---- the parts of a sequence joined --------------------------------------------------------------------------------
// grid = (kv heads * column groups, columns of a group, sequences), HD / 4 threads: four values each
template <int HD>
__global__ __launch_bounds__(64) void paged_merge_kernel(PagedView c, PagedOp a) {
    const uint32_t g = blockIdx.x / a.n_cg, cg = blockIdx.x % a.n_cg, s = blockIdx.z, d = threadIdx.x * 4;
    const PagedRows r = paged_rows(a.q_first, c.lens, s, a.n_rows, a.max_queries, c.max_len);
    if (r.bad || r.len == 0) return;   // written by the attention's launch
    const uint32_t n_cols = r.n * a.G, col = cg * a.n_cols + blockIdx.y;
    if (col >= n_cols) return;
    const PagedTiles t = paged_tiles(r, cg * a.n_cols, min(cg * a.n_cols + a.n_cols, n_cols) - 1, a);
    const uint32_t parts = (t.n + a.part_tiles - 1) / a.part_tiles;
    if (parts <= 1 || threadIdx.x >= HD / 4) return;
    const uint64_t first = ((static_cast<uint64_t>(s) * gridDim.x + blockIdx.x) * a.max_parts) * a.n_cols + blockIdx.y;
    float M = PAGED_LOWEST;
    for (uint32_t p = 0; p < parts; ++p) M = fmaxf(M, a.ml[(first + static_cast<uint64_t>(p) * a.n_cols) * 2]);
    float L = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t p = 0; p < parts; ++p) {
        const uint64_t at = first + static_cast<uint64_t>(p) * a.n_cols;
        const float f = __builtin_amdgcn_exp2f(a.ml[at * 2] - M);
        const float4 x = *reinterpret_cast<const float4*>(a.acc + at * HD + d);
        L = fmaf(f, a.ml[at * 2 + 1], L);
        o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    *reinterpret_cast<float4*>(a.out + (r.first + static_cast<uint64_t>(col / a.G)) * a.out_stride + (g * a.G + col % a.G) * HD + d) = o;
}

// ---- weights added up by position ----------------------------------------------------------------------------------
// grid = (blocks of positions, kv heads, sequences).  The scores lie as the attention left them, in the base-2 domain.
__global__ __launch_bounds__(256) void paged_mass_kernel(PagedView c, PagedOp a) {
    extern __shared__ float sh[];   // [G] maximum, [G] 1 / sum
    const uint32_t g = blockIdx.y, s = blockIdx.z;
    const PagedRows r = paged_rows(nullptr, c.lens, s, a.n_rows, 1, c.max_len);
    if (r.bad || r.len == 0) return;
    const uint32_t P = r.len - 1;
    const PagedSeen v = paged_seen(P, a.window, a.n_sink);
    const uint32_t n_seen = v.sink_end + (P + 1 - v.start);
    if (blockIdx.x * 1024u >= n_seen) return;
    for (uint32_t h = threadIdx.x; h < a.G; h += 256) {
        const uint32_t cg = h / a.n_cols, last = min(cg * a.n_cols + a.n_cols, a.G) - 1;
        const PagedTiles t = paged_tiles(r, cg * a.n_cols, last, a);
        const uint32_t parts = (t.n + a.part_tiles - 1) / a.part_tiles;
        const uint64_t first = ((static_cast<uint64_t>(s) * c.n_kv * a.n_cg + g * a.n_cg + cg) * a.max_parts) * a.n_cols + h % a.n_cols;
        float M = PAGED_LOWEST, L = 0.0f;
        for (uint32_t p = 0; p < parts; ++p) M = fmaxf(M, a.ml[(first + static_cast<uint64_t>(p) * a.n_cols) * 2]);
        for (uint32_t p = 0; p < parts; ++p) {
            const uint64_t at = first + static_cast<uint64_t>(p) * a.n_cols;
            L = fmaf(__builtin_amdgcn_exp2f(a.ml[at * 2] - M), a.ml[at * 2 + 1], L);
        }
        sh[h] = M - PAGED_P_LOG2;
        sh[a.G + h] = L == 0.0f ? 0.0f : 1.0f / L;   // NaN where a page was bad
    }
    __syncthreads();
    float* const m = a.mass + (static_cast<uint64_t>(s) * c.n_kv + g) * a.mass_stride;
    for (uint32_t i = blockIdx.x * 1024u + threadIdx.x; i < min(n_seen, blockIdx.x * 1024u + 1024u); i += 256) {
        const uint32_t t = i < v.sink_end ? i : v.start + (i - v.sink_end);
        float sum = 0.0f;
        for (uint32_t h = 0; h < a.G; ++h)
            sum = fmaf(__builtin_amdgcn_exp2f(a.scores[(static_cast<uint64_t>(s) * c.n_kv * a.G + g * a.G + h) * a.score_stride + t] - sh[h]), sh[a.G + h], sum);
        if (sum == sum) m[t] += sum;
    }
}

template <typename KV, int HD>
static cera_hip_status paged_attn_launch(cera_hip_ctx* ctx, const cera_hip_paged_kv& c, const cera_hip_paged_attn& in) {
    constexpr bool HALF = sizeof(KV) == 2;
    const PagedView v = paged_view(c, in.max_len);
    PagedOp a{};
    a.q = in.q; a.out = in.out; a.mass = in.mass; a.q_first = in.q_first;
    a.q_stride = in.q_stride ? in.q_stride : static_cast<uint64_t>(in.n_heads) * HD;
    a.out_stride = in.out_stride ? in.out_stride : static_cast<uint64_t>(in.n_heads) * HD;
    a.mass_stride = in.mass_stride;
    a.n_rows = in.n_rows;
    a.max_queries = in.q_first ? (in.max_queries ? std::min(in.max_queries, in.n_rows) : in.n_rows) : 1;
    a.G = in.n_heads / c.n_kv_heads;
    a.scale2 = in.scale * 1.44269504088896340736f;
    a.window = in.window; a.n_sink = in.n_sink;
    const uint64_t cols = static_cast<uint64_t>(a.max_queries) * a.G;
    const uint32_t cb = HALF && cols > 8 ? 2 : 1;
    a.n_cols = (HALF ? 8 : 16) * cb;
    a.n_cg = static_cast<uint32_t>((cols + a.n_cols - 1) / a.n_cols);
    if (static_cast<uint64_t>(c.n_kv_heads) * a.n_cg > (1u << 23)) return cera_fail(ctx, CERA_HIP_ERR_SHAPE, "paged attention: too many rows of a sequence for one call");
    a.tile = HALF ? 32 : 16;
    const PagedCut cut = paged_cut(v.max_len, a.max_queries, a.window, a.n_sink, a.tile, static_cast<uint64_t>(c.n_seqs) * c.n_kv_heads * a.n_cg, ctx->n_cu);
    a.part_tiles = cut.part_tiles;
    a.max_parts = cut.max_parts;
    a.score_stride = a.mass ? (static_cast<uint64_t>(v.max_len) + 31) / 32 * 32 : 0;
    auto bytes = [&](uint64_t parts) {
        const uint64_t n = parts > 1 || a.mass ? static_cast<uint64_t>(c.n_seqs) * c.n_kv_heads * a.n_cg * parts * a.n_cols : 0;
        return n * (parts > 1 ? HD + 2 : 2) * 4 + a.score_stride * c.n_seqs * in.n_heads * 4;
    };
    void* ws = nullptr;
    if (a.max_parts > 1) {
        CERA_TRY(cera_scratch_if_room(ctx, 15, bytes(a.max_parts), &ws));
        if (!ws) {   // one workgroup walks all of a sequence
            a.max_parts = 1;
            a.part_tiles = 0x7FFFFFFFu;
        }
    }
    if (!ws && bytes(a.max_parts)) CERA_TRY(cera_scratch(ctx, 15, bytes(a.max_parts), &ws));
    a.scores = static_cast<float*>(ws);
    a.ml = a.scores + a.score_stride * c.n_seqs * in.n_heads;
    a.acc = a.ml + static_cast<uint64_t>(c.n_seqs) * c.n_kv_heads * a.n_cg * a.max_parts * a.n_cols * 2;
    if (in.k_new) {
        const uint64_t items = static_cast<uint64_t>(a.max_queries) * c.n_kv_heads * (HD / 4);
        hipLaunchKernelGGL((paged_append_kernel<KV, HD>), dim3(static_cast<uint32_t>(std::min<uint64_t>((items + 255) / 256, 1024)), c.n_seqs), dim3(256), 0, ctx->stream, v,
                           static_cast<KV*>(c.k), static_cast<KV*>(c.v), in.k_new, in.v_new, in.kv_stride ? in.kv_stride : static_cast<uint64_t>(c.n_kv_heads) * HD, a.q_first, a.n_rows,
                           a.max_queries, in.mass_fresh ? a.mass : nullptr, a.mass_stride);
    }
    const dim3 grid(c.n_kv_heads * a.n_cg, a.max_parts, c.n_seqs);
    auto launch = [&](auto tag) {
        constexpr int CB = decltype(tag)::value;
        if (a.mass) hipLaunchKernelGGL((paged_attn_kernel<KV, HD, CB, true>), grid, dim3(256), 0, ctx->stream, v, static_cast<const KV*>(c.k), static_cast<const KV*>(c.v), a);
        else hipLaunchKernelGGL((paged_attn_kernel<KV, HD, CB, false>), grid, dim3(256), 0, ctx->stream, v, static_cast<const KV*>(c.k), static_cast<const KV*>(c.v), a);
    };
    if (cb == 2) {
        if constexpr (HALF) launch(std::integral_constant<int, 2>{});
    } else {
        launch(std::integral_constant<int, 1>{});
    }
    if (a.max_parts > 1) hipLaunchKernelGGL((paged_merge_kernel<HD>), dim3(c.n_kv_heads * a.n_cg, a.n_cols, c.n_seqs), dim3(64), 0, ctx->stream, v, a);
    if (a.mass) {
        const uint64_t most = a.window ? std::min<uint64_t>(v.max_len, static_cast<uint64_t>(a.window) + a.n_sink) : v.max_len;
        hipLaunchKernelGGL(paged_mass_kernel, dim3(static_cast<uint32_t>((most + 1023) / 1024), c.n_kv_heads, c.n_seqs), dim3(256), a.G * 8, ctx->stream, v, a);
    }
    HIP_TRY(ctx, hipGetLastError());
    return CERA_HIP_OK;
}

extern "C" cera_hip_status cera_hip_paged_attn_dev(cera_hip_ctx* ctx, const cera_hip_paged_kv* c, const cera_hip_paged_attn* a) {
    if (!ctx) return CERA_HIP_ERR_ARGUMENT;
    std::lock_guard<std::recursive_mutex> op_lk(ctx->op_mu);
    const PagedCheck no = paged_check_attn(c, a);
    if (no.msg) return cera_fail(ctx, no.st, no.msg);
    if (c->n_seqs == 0 || a->n_rows == 0) return CERA_HIP_OK;
    const PagedDevice dev(ctx->device);
    HIP_TRY(ctx, dev.err);
    if (c->kv_type == CERA_HIP_KV_F16) return c->head_dim == 128 ? paged_attn_launch<kv_half, 128>(ctx, *c, *a) : paged_attn_launch<kv_half, 64>(ctx, *c, *a);
    return c->head_dim == 128 ? paged_attn_launch<float, 128>(ctx, *c, *a) : paged_attn_launch<float, 64>(ctx, *c, *a);
}
