// Attention of new tokens over a paged cache (cera_hip_paged_attn_dev; contract in include/cera_hip.h).
#include "paged.hip.h"

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

// ---- attention, a wavefront per row and query head -----------------------------------------------------------------
// grid = (query heads, rows of a sequence, sequences)
template <typename KV, int HD>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedView c, const KV* __restrict__ kp, const KV* __restrict__ vp, const float* __restrict__ q, uint64_t q_stride,
                                                        float* __restrict__ out, uint64_t out_stride, const uint32_t* __restrict__ q_first, uint32_t n_rows,
                                                        uint32_t max_queries, uint32_t G, float scale, uint32_t window, uint32_t n_sink, float* __restrict__ mass, uint64_t mass_stride) {
    constexpr int E = HD / 64;
    const uint32_t s = blockIdx.z, h = blockIdx.x, g = h / G, lane = threadIdx.x;
    const PagedRows r = paged_rows(q_first, c.lens, s, n_rows, max_queries, c.max_len);
    for (uint32_t i = blockIdx.y; i < r.n; i += gridDim.y) {
        float* o = out + (r.first + static_cast<uint64_t>(i)) * out_stride + h * HD + lane * E;
        float acc[E] = {}, m = -3.402823466e38f, l = 0.0f;   // finite, so that a score of -inf has weight 0
        bool ok = !r.bad;
        if (ok && r.len) {
            float x[E];
            for (int e = 0; e < E; ++e) x[e] = q[(r.first + static_cast<uint64_t>(i)) * q_stride + h * HD + lane * E + e];
            const uint32_t P = r.len - r.n + i;
            const PagedSeen v = paged_seen(P, window, n_sink);
            auto score = [&](uint32_t t, uint32_t page) {
                float d = 0.0f;
                for (int e = 0; e < E; ++e) d = fmaf(x[e], static_cast<float>(kp[paged_row<HD>(c, page, g, t) + lane * E + e]), d);
                return wave_sum(d) * scale;
            };
            for (uint32_t t = v.sink_end ? 0 : v.start; t <= P; t = t + 1 == v.sink_end ? v.start : t + 1) {
                const uint32_t page = paged_page(c, s, t, ok);
                const float sc = score(t, page), mn = fmaxf(m, sc), corr = expf(m - mn), p = expf(sc - mn);
                m = mn;
                l = l * corr + p;
                for (int e = 0; e < E; ++e) acc[e] = fmaf(p, static_cast<float>(vp[paged_row<HD>(c, page, g, t) + lane * E + e]), acc[e] * corr);
            }
            if (mass && ok)
                for (uint32_t t = v.sink_end ? 0 : v.start; t <= P; t = t + 1 == v.sink_end ? v.start : t + 1) {
                    const float p = expf(score(t, paged_page(c, s, t, ok)) - m) / l;
                    if (lane == 0) atomicAdd(mass + (static_cast<uint64_t>(s) * c.n_kv + g) * mass_stride + t, p);
                }
            for (int e = 0; e < E; ++e) acc[e] = l == 0.0f ? 0.0f : acc[e] / l;
        }
        for (int e = 0; e < E; ++e) o[e] = ok ? acc[e] : __builtin_nanf("");
    }
}

template <typename KV, int HD>
static void paged_attn_launch(cera_hip_ctx* ctx, const cera_hip_paged_kv& c, const cera_hip_paged_attn& a) {
    const PagedView v = paged_view(c, a.max_len);
    const uint64_t q_stride = a.q_stride ? a.q_stride : a.n_heads * HD, out_stride = a.out_stride ? a.out_stride : a.n_heads * HD;
    const uint32_t mq = a.q_first ? (a.max_queries ? std::min(a.max_queries, a.n_rows) : a.n_rows) : 1;
    if (a.k_new)
        hipLaunchKernelGGL((paged_append_kernel<KV, HD>), dim3(std::min<uint64_t>((static_cast<uint64_t>(mq) * c.n_kv_heads * (HD / 4) + 255) / 256, 1024), c.n_seqs), dim3(256), 0, ctx->stream, v,
                           static_cast<KV*>(c.k), static_cast<KV*>(c.v), a.k_new, a.v_new, a.kv_stride ? a.kv_stride : c.n_kv_heads * HD, a.q_first, a.n_rows, mq, a.mass, a.mass_stride);
    hipLaunchKernelGGL((paged_attn_kernel<KV, HD>), dim3(a.n_heads, std::min(mq, 65535u), c.n_seqs), dim3(64), 0, ctx->stream, v, static_cast<const KV*>(c.k), static_cast<const KV*>(c.v), a.q,
                       q_stride, a.out, out_stride, a.q_first, a.n_rows, mq, a.n_heads / c.n_kv_heads, a.scale, a.window, a.n_sink, a.mass, a.mass_stride);
}

extern "C" cera_hip_status cera_hip_paged_attn_dev(cera_hip_ctx* ctx, const cera_hip_paged_kv* c, const cera_hip_paged_attn* a) {
    if (!ctx) return CERA_HIP_ERR_ARGUMENT;
    std::lock_guard<std::recursive_mutex> op_lk(ctx->op_mu);
    const PagedCheck no = paged_check_attn(c, a);
    if (no.msg) return cera_fail(ctx, no.st, no.msg);
    if (c->n_seqs == 0 || a->n_rows == 0) return CERA_HIP_OK;
    const PagedDevice dev(ctx->device);
    HIP_TRY(ctx, dev.err);
    if (c->kv_type == CERA_HIP_KV_F16) {
        if (c->head_dim == 128) paged_attn_launch<kv_half, 128>(ctx, *c, *a);
        else paged_attn_launch<kv_half, 64>(ctx, *c, *a);
    } else {
        if (c->head_dim == 128) paged_attn_launch<float, 128>(ctx, *c, *a);
        else paged_attn_launch<float, 64>(ctx, *c, *a);
    }
    HIP_TRY(ctx, hipGetLastError());
    return CERA_HIP_OK;
}
