// Eviction from a paged cache by accumulated attention weight (cera_hip_paged_evict_dev; contract in include/cera_hip.h).
//
// Two launches.  The first chooses: a workgroup per (kv head, sequence) finds the weight of the last position that stays by radix
// selection on the weights' bits, in three passes of 11, 11 and 10 bits, and writes the positions that stay in their order.  The
// second moves: position i takes the row of position kept[i] >= i, so that a walk upwards in place never reads what it has
// written, as long as all rows of a step are read before the step writes.
//
// 16 sequences of up to 8192 positions of 8 kv heads of 128, half cache, brought to 4096: the choice takes 14 us, bound by the latency of
// its passes (a histogram in LDS and a scan each), the move 108 us, bound by memory: 0.54 GB in and out, 5.0 TB/s, where a large copy
// reaches 4.8.  A workgroup of 1024 threads moves 128 bytes of every row of one kv head's keys or values, two of them a CU (one a CU: a fifth
// more), the next step's rows on their way while this one's are written; non-temporal, 8 us less.
#include "paged.hip.h"

static constexpr uint32_t EV_THREADS = 1024, EV_BINS = 2048;

// a weight as an integer of the same order: -0 as 0, every NaN above all numbers
__device__ __forceinline__ uint32_t evict_key(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t b = __builtin_bit_cast(uint32_t, w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// grid = (kv heads, sequences).  kept: [n_seqs][n_kv][budget]; cut[s]: positions of a sequence that is cut, else 0
__global__ __launch_bounds__(EV_THREADS) void paged_evict_select_kernel(PagedView c, float* __restrict__ mass, uint64_t mass_stride, uint32_t budget, uint32_t n_first,
                                                                        uint32_t n_recent, uint32_t* __restrict__ kept_ws, int32_t* __restrict__ kept_out,
                                                                        uint32_t* __restrict__ new_lens, uint32_t* __restrict__ cut) {
    __shared__ uint32_t hist[EV_BINS], wave_tot[EV_THREADS / 64], sh[4];
    const uint32_t g = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t len = c.lens[s];
    const uint64_t sg = static_cast<uint64_t>(s) * c.n_kv + g;
    bool ok = len <= c.max_len;
    float* const mw = mass + sg * mass_stride;
    // the middle [lo, hi) of a sequence that is cut has more than `need` positions; its first keys stay in registers between the passes
    const uint32_t lo = n_first, hi = len - n_recent, need = budget - n_first - n_recent;
    constexpr uint32_t HELD = 8;
    uint32_t held[HELD];
#pragma unroll
    for (uint32_t u = 0; u < HELD; ++u) {
        const uint32_t t = lo + tid + u * EV_THREADS;
        held[u] = ok && len > budget && t < hi ? evict_key(mw[t]) : 0;
    }
    if (ok)
        for (uint32_t p = tid; p << c.page_log2 < len; p += EV_THREADS) (void)paged_page(c, s, p << c.page_log2, ok);
    ok = __syncthreads_and(ok);
    int32_t* const out = kept_out ? kept_out + sg * budget : nullptr;
    if (!ok || len <= budget) {
        if (out)
            for (uint32_t i = tid; i < budget; i += EV_THREADS) out[i] = ok && i < len ? static_cast<int32_t>(i) : -1;
        if (g == 0 && tid == 0) { new_lens[s] = len; cut[s] = 0; }
        return;
    }
    // radix selection: `prefix` holds the bits found so far, `left` how many of those that share them still stay
    uint32_t prefix = 0, left = need;
    if (need) {
        for (int pass = 0; pass < 3; ++pass) {
            const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, above = shift + bits;
            for (uint32_t b = tid; b < EV_BINS; b += EV_THREADS) hist[b] = 0;
            __syncthreads();
            auto count = [&](uint32_t k) {
                if (pass == 0 || k >> above == prefix >> above) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
            };
#pragma unroll
            for (uint32_t u = 0; u < HELD; ++u)
                if (lo + tid + u * EV_THREADS < hi) count(held[u]);
            for (uint32_t t = lo + tid + HELD * EV_THREADS; t < hi; t += EV_THREADS) count(evict_key(mw[t]));
            __syncthreads();
            // from the top bin down to the one in which the count reaches `left`: two bins a thread, thread 0 has the highest
            const uint32_t top = (1u << bits) - 1, n_thr = (1u << bits) / 2;
            uint32_t a = 0, b = 0;
            if (tid < n_thr) { a = hist[top - 2 * tid]; b = hist[top - 2 * tid - 1]; }
            uint32_t sum = a + b, inc = sum;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = __shfl_up(inc, d);
                if (lane >= static_cast<uint32_t>(d)) inc += o;
            }
            if (lane == 63) wave_tot[w] = inc;
            __syncthreads();
            uint32_t before = inc - sum;
#pragma unroll
            for (uint32_t i = 0; i < EV_THREADS / 64; ++i) {   // all loads in flight
                const uint32_t x = wave_tot[i];
                before += i < w ? x : 0;
            }
            if (before < left && before + sum >= left) {
                const bool second = before + a < left;
                sh[0] = prefix | (top - 2 * tid - (second ? 1 : 0)) << shift;
                sh[1] = left - before - (second ? a : 0);
            }
            __syncthreads();
            prefix = sh[0];
            left = sh[1];
        }
    }
    // in order: larger ones and the ends stay, of the equal ones the first `left`; HELD rows of a position a thread at a time
    uint32_t base_gt = 0, base_eq = 0;
    uint32_t* const ws = kept_ws + sg * budget;
    for (uint32_t t0 = 0; t0 < len; t0 += HELD * EV_THREADS) {
        float x[HELD];
        uint64_t bg[HELD], be[HELD];
#pragma unroll
        for (uint32_t u = 0; u < HELD; ++u) x[u] = mw[min(t0 + u * EV_THREADS + tid, len - 1)];
#pragma unroll
        for (uint32_t u = 0; u < HELD; ++u) {
            const uint32_t t = t0 + u * EV_THREADS + tid, k = evict_key(x[u]);
            const bool in = t < len, mid = t >= lo && t < hi;
            bg[u] = __ballot(in && (!mid || (need && k > prefix)));
            be[u] = __ballot(in && mid && need && k == prefix);
            if (lane == 0) hist[u * (EV_THREADS / 64) + w] = __popcll(bg[u]) | __popcll(be[u]) << 16;   // both at most 64 * 128 when added up
        }
        __syncthreads();
        // running sums over the step's 128 wavefronts and rows
        const uint32_t c0 = hist[2 * lane], c1 = hist[2 * lane + 1];
        uint32_t inc = c0 + c1;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(inc, d);
            if (lane >= static_cast<uint32_t>(d)) inc += o;
        }
        const uint32_t first = inc - c0 - c1, below = first + c0;   // in front of entries 2 lane, 2 lane + 1
#pragma unroll
        for (uint32_t u = 0; u < HELD; ++u) {
            const uint32_t at = u * (EV_THREADS / 64) + w, v = w & 1 ? __shfl(below, at >> 1) : __shfl(first, at >> 1);
            const uint64_t under = (1ull << lane) - 1;
            const uint32_t n_gt = base_gt + (v & 0xFFFF) + __popcll(bg[u] & under), n_eq = base_eq + (v >> 16) + __popcll(be[u] & under);
            const bool gt = bg[u] >> lane & 1, eq = be[u] >> lane & 1;
            if (gt || (eq && n_eq < left)) {
                const uint32_t t = t0 + u * EV_THREADS + tid, dst = n_gt + min(n_eq, left);
                ws[dst] = t;
                if (out) out[dst] = static_cast<int32_t>(t);
                mw[dst] = x[u];   // dst <= t, and all of this step's weights are read
            }
        }
        const uint32_t all = __shfl(inc, 63);
        base_gt += all & 0xFFFF;
        base_eq += all >> 16;
        __syncthreads();
    }
    if (g == 0 && tid == 0) { new_lens[s] = budget; cut[s] = len; }
}

// grid = (128-byte columns of a row, 2 * kv heads, sequences): keys, then values.  Eight lanes of 16 bytes a row.
// A step's rows are on their way while the ones before are written: sources lie behind all of what is written until then.
static constexpr uint32_t EV_ROWS = EV_THREADS / 8, EV_UNROLL = 2, EV_STEP = EV_ROWS * EV_UNROLL;   // rows of a pass, passes and rows of a step
template <typename KV, int HD>
__global__ __launch_bounds__(EV_THREADS, 8) void paged_evict_move_kernel(PagedView c, KV* __restrict__ kp, KV* __restrict__ vp, uint32_t budget, const uint32_t* __restrict__ kept,
                                                                      const uint32_t* __restrict__ cut) {
    const uint32_t s = blockIdx.z, g = blockIdx.y >> 1, j = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    if (cut[s] == 0) return;
    uint8_t* const pool = reinterpret_cast<uint8_t*>(blockIdx.y & 1 ? vp : kp) + blockIdx.x * 128 + j * 16;
    const uint32_t* const idx = kept + (static_cast<uint64_t>(s) * c.n_kv + g) * budget;
    bool ok = true;   // the pages were looked over when the positions were chosen
    auto at = [&](uint32_t t) { return pool + paged_row<HD>(c, paged_page(c, s, t, ok), g, t) * sizeof(KV); };
    struct Step {
        uint4 row[EV_UNROLL];
        uint32_t from[EV_UNROLL];
    };
    auto positions = [&](Step& x, uint32_t i0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < EV_UNROLL; ++u) {
            const uint32_t i = i0 + u * EV_ROWS + r0;
            x.from[u] = i < budget ? idx[i] : i;   // a row that stays where it is needs nothing
        }
    };
    auto read = [&](Step& x, uint32_t i0) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < EV_UNROLL; ++u)
            if (x.from[u] != i0 + u * EV_ROWS + r0) x.row[u] = paged_stream<uint4>(at(x.from[u]));
    };
    auto write = [&](Step& x, uint32_t i0) __attribute__((always_inline)) {
        // every wavefront has this step's rows in its registers
#pragma unroll
        for (uint32_t u = 0; u < EV_UNROLL; ++u) asm volatile("" : "+v"(x.row[u].x), "+v"(x.row[u].y), "+v"(x.row[u].z), "+v"(x.row[u].w));
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (uint32_t u = 0; u < EV_UNROLL; ++u) {
            const uint32_t i = i0 + u * EV_ROWS + r0;
            if (x.from[u] != i) paged_stream(at(i), x.row[u]);
        }
    };
    Step a, b;
#pragma unroll
    for (uint32_t u = 0; u < EV_UNROLL; ++u) a.row[u] = b.row[u] = make_uint4(0, 0, 0, 0);
    positions(a, 0);
    read(a, 0);
    positions(b, EV_STEP);
    for (uint32_t i0 = 0; i0 < budget; i0 += 2 * EV_STEP) {
        read(b, i0 + EV_STEP);
        write(a, i0);
        positions(a, i0 + 2 * EV_STEP);
        read(a, i0 + 2 * EV_STEP);
        write(b, i0 + EV_STEP);
        positions(b, i0 + 3 * EV_STEP);
    }
}

template <typename KV, int HD>
static void paged_evict_launch(cera_hip_ctx* ctx, const cera_hip_paged_kv& c, const cera_hip_paged_evict& e, uint32_t* kept, uint32_t* cut) {
    const PagedView v = paged_view(c, e.max_len);
    hipLaunchKernelGGL(paged_evict_select_kernel, dim3(c.n_kv_heads, c.n_seqs), dim3(EV_THREADS), 0, ctx->stream, v, e.mass, e.mass_stride, e.budget, e.n_first, e.n_recent, kept, e.kept,
                       e.new_lens, cut);
    hipLaunchKernelGGL((paged_evict_move_kernel<KV, HD>), dim3(HD * sizeof(KV) / 128, 2 * c.n_kv_heads, c.n_seqs), dim3(EV_THREADS), 0, ctx->stream, v, static_cast<KV*>(c.k), static_cast<KV*>(c.v),
                       e.budget, kept, cut);
}

extern "C" cera_hip_status cera_hip_paged_evict_dev(cera_hip_ctx* ctx, const cera_hip_paged_kv* c, const cera_hip_paged_evict* e) {
    if (!ctx) return CERA_HIP_ERR_ARGUMENT;
    std::lock_guard<std::recursive_mutex> op_lk(ctx->op_mu);
    const PagedCheck no = paged_check_evict(c, e);
    if (no.msg) return cera_fail(ctx, no.st, no.msg);
    if (c->n_seqs == 0) return CERA_HIP_OK;
    const PagedDevice dev(ctx->device);
    HIP_TRY(ctx, dev.err);
    // a budget behind the longest sequence cuts none; the list then needs no room
    const uint64_t list = e->budget < paged_max_len(*c, e->max_len) ? static_cast<uint64_t>(c->n_seqs) * c->n_kv_heads * e->budget : 0;
    void* ws;
    CERA_TRY(cera_scratch(ctx, 15, (list + c->n_seqs) * 4, &ws));
    uint32_t* const cut = static_cast<uint32_t*>(ws);
    uint32_t* const kept = cut + c->n_seqs;
    if (c->kv_type == CERA_HIP_KV_F16) {
        if (c->head_dim == 128) paged_evict_launch<kv_half, 128>(ctx, *c, *e, kept, cut);
        else paged_evict_launch<kv_half, 64>(ctx, *c, *e, kept, cut);
    } else {
        if (c->head_dim == 128) paged_evict_launch<float, 128>(ctx, *c, *e, kept, cut);
        else paged_evict_launch<float, 64>(ctx, *c, *e, kept, cut);
    }
    HIP_TRY(ctx, hipGetLastError());
    return CERA_HIP_OK;
}
