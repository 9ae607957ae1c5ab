// Attention of new tokens over a paged cache (cera_hip_paged_attn_dev; contract in include/cera_hip.h).
#include "paged.hip.h"
#include "paged_attn.hip.h"
#include "paged_chunk.hip.h"

// ---- chunks: the new rows into their pages -----------------------------------------------------------------------------
// grid = (blocks, sequences); a thread moves four floats of a row's keys and values.  Bound by memory: 6 to 7 us for 2048 rows of 8 kv heads
// of 128, 25 MB.  Few columns need it not: their workgroups take the new rows from the call's (51.5 us with this launch, 50.2 without,
// for 16 sequences of 5 drafts).
template <typename KV, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedView c, KV* __restrict__ kp, KV* __restrict__ vp, const float* __restrict__ k_new,
                                                           const float* __restrict__ v_new, uint64_t kv_stride, const uint32_t* __restrict__ q_first,
                                                           uint32_t n_rows, uint32_t max_queries) {
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
    }
}
// their weights to 0, in a launch of its own: as arguments of the other it cost each call 0.4 us
__global__ __launch_bounds__(256) void paged_fresh_kernel(PagedView c, float* __restrict__ mass, uint64_t mass_stride, const uint32_t* __restrict__ q_first, uint32_t n_rows, uint32_t max_queries) {
    const uint32_t s = blockIdx.y;
    const PagedRows r = paged_rows(q_first, c.lens, s, n_rows, max_queries, c.max_len);
    if (r.bad) return;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < static_cast<uint64_t>(r.n) * c.n_kv; i += gridDim.x * 256ull)
        mass[(static_cast<uint64_t>(s) * c.n_kv + i / r.n) * mass_stride + (r.len - r.n + i % r.n)] = 0.0f;
}

// ---- attention ------------------------------------------------------------------------------------------------------
template <typename KV_, int HD, int CB, bool TWIN, bool MASS> struct PagedFew {
    using KV = KV_;
    static constexpr int NC = (TWIN ? 8 : 16) * CB, DIM = HD;
    using Shared = PagedShared<NC, HD>;
    template <class... A> __device__ static __forceinline__ void part(Shared& sh, A&&... x) { paged_attn_part<KV, HD, CB, TWIN, MASS>(sh, x...); }
};
template <typename KV_, int HD> struct PagedMany {
    using KV = KV_;
    static constexpr int NC = 128, DIM = HD;
    using Shared = PagedChunkShared<KV, HD>;
    template <class... A> __device__ static __forceinline__ void part(Shared& sh, A&&... x) { paged_chunk_part<KV, HD>(sh, x...); }
};

// Groups of columns that are not cut, of all sequences: the longest first, and every second round of the chip the other way round, so
// that a CU's add up to about the same.  A group's length is its last position's, or the window: item k is found from the number of
// groups that are at least 32 L long, for which a lane each looks at its sequence.  128 to 101 us for 24 sequences with 100
// tokens each at up to 2000 positions, 60 to 50 for 12 of up to 700 tokens, 273 to 203 for 8 with 300 each at 3000; below 8 sequences the search costs
// what it saves: 6 of up to 700 tokens 46.7 without it and 49.7 with it, of 700 91.0 and 88.4.  Above 64, more than a wavefront's lanes, the table's order.
struct PagedItem { uint32_t seq, cg; bool none; };
__device__ __forceinline__ PagedItem paged_item(const PagedView& c, const PagedOp& a, uint32_t n_seqs, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63, rows = max(1u, a.n_cols / a.G);   // rows of a group
    uint32_t len = 0, groups = 0;
    if (lane < n_seqs) {
        const PagedRows r = paged_rows(a.q_first, c.lens, lane, a.n_rows, a.max_queries, c.max_len);
        if (r.n) groups = r.bad || r.len == 0 ? 1 : (r.n * a.G + a.n_cols - 1) / a.n_cols;
        len = r.bad ? 0 : r.len;
    }
    auto sum = [](uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(wave_sum(static_cast<float>(x))))); };   // below 2^24
    const uint32_t none = (a.window ? min(c.max_len, a.window) : c.max_len) / 32 + 1;   // the lowest level that no group reaches
    auto at_least = [&](uint32_t level) { return level == 0 ? groups : level >= none || len < 32 * level ? 0 : min(groups, (len - 32 * level) / rows + 1); };
    const uint32_t all = sum(groups), in_round = k % a.round, round0 = k - in_round;
    if (k >= all) return {0, 0, true};
    if (round0 / a.round & 1) k = round0 + min(a.round, all - round0) - 1 - in_round;
    // the largest level that more than k groups reach
    uint32_t lo = 0, hi = none;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (sum(at_least(mid)) > k) lo = mid; else hi = mid;
    }
    const uint32_t above = at_least(lo + 1), n = at_least(lo) - above;
    uint32_t inc = n;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(inc, d);
        if (lane >= static_cast<uint32_t>(d)) inc += o;
    }
    k -= sum(above);
    const int x = __builtin_ctzll(__ballot(inc > k));
    const uint32_t i = __builtin_amdgcn_readlane(above, x) + k - __builtin_amdgcn_readlane(inc - n, x);   // from the sequence's last group
    return {static_cast<uint32_t>(x), static_cast<uint32_t>(__builtin_amdgcn_readlane(groups, x)) - 1 - i, false};
}

// A kv head and group of columns has one list of tiles, sequence after sequence.  Either a workgroup takes a sequence of it, grid =
// (kv heads * groups, sequences), or each takes a span of equal length, grid = (kv heads * groups, spans): ragged sequences then cost
// what their sum costs.  Only the first and the last sequence of a span can be cut: slots 2 span and 2 span + 1.
// Work: PagedFew or PagedMany below.
template <class Work>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedView c, typename Work::KV* __restrict__ kp, typename Work::KV* __restrict__ vp, PagedOp a, uint32_t n_seqs) {
    constexpr int NC = Work::NC;
    __shared__ typename Work::Shared sh;
    // kv heads side by side, so that a head's workgroups share an XCD's L2 where there are eight
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = blockIdx.x % c.n_kv;
    uint32_t cg = a.n_cg - 1 - blockIdx.x / c.n_kv;   // the columns with the most positions first
    uint32_t s = blockIdx.y, j = 0, left = 0xFFFFFFFFu, span = 0;   // the sequence, the first of its tiles, tiles left of the span
    if constexpr (NC == 128) {
        if (a.ordered) {
            const PagedItem it = paged_item(c, a, n_seqs, (blockIdx.y * gridDim.x + blockIdx.x) / c.n_kv);
            if (it.none) return;
            s = it.seq;
            cg = it.cg;
        }
    }
    const uint32_t c0 = cg * NC;
    uint32_t s_end = s + 1;
    if (a.spans) {
        span = blockIdx.y;
        s_end = n_seqs;
        // all tiles, and the sequence that has tile `at`; up to 64 sequences by one look at their lengths
        uint32_t total = 0, at = 0, share = 0;
        for (int pass = 0; pass < 2; ++pass) {
            uint32_t before = 0;
            bool found = false;
            for (uint32_t b = 0; b < n_seqs && !found; b += 64) {
                const uint32_t n = b + lane < n_seqs ? paged_count(c, a, b + lane, c0) : 0;
                uint32_t inc = n;
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t o = __shfl_up(inc, d);
                    if (lane >= static_cast<uint32_t>(d)) inc += o;
                }
                const uint32_t sum = __builtin_amdgcn_readlane(inc, 63);
                if (pass == 0) total += sum;
                if (pass == 0 && n_seqs <= 64) {
                    share = max(a.least, (total + a.spans - 1) / a.spans);
                    at = span * share;
                    pass = 1;
                }
                if (pass == 1) {
                    const uint64_t over = __ballot(before + inc > at);
                    if (over) {
                        const int x = __builtin_ctzll(over);
                        s = b + x;
                        j = at - before - __builtin_amdgcn_readlane(inc - n, x);
                        found = true;
                    }
                }
                before += sum;
            }
            if (pass == 0) {
                share = max(a.least, (total + a.spans - 1) / a.spans);
                at = span * share;
            }
        }
        if (at >= total) return;
        left = min(share, total - at);
        s = __builtin_amdgcn_readfirstlane(s);
        j = __builtin_amdgcn_readfirstlane(j);
    }
    for (; s < s_end && left; ++s, j = 0) {
        const PagedRows r = paged_rows(a.q_first, c.lens, s, a.n_rows, a.max_queries, c.max_len);
        if (r.bad || r.len == 0) {
            // nothing is known of these rows but where they are
            if (cg == 0) {
                for (uint32_t row = 0; row < r.n; ++row)
                    for (uint32_t i = tid; i < a.G * Work::DIM; i += 256)
                        a.out[(r.first + static_cast<uint64_t>(row)) * a.out_stride + g * a.G * Work::DIM + i] = r.bad ? __builtin_nanf("") : 0.0f;
                --left;
            }
            continue;
        }
        const uint32_t n_cols = r.n * a.G;
        if (c0 >= n_cols) continue;
        const uint32_t c_last = min(c0 + NC, n_cols) - 1;
        const PagedTiles tiles = paged_tiles(r, c0, c_last, a);
        const uint32_t j_end = left < tiles.n - j ? j + left : tiles.n;
        Work::part(sh, c, kp, vp, a, g, cg, s, r, tiles, c0, c_last, j, j_end, 2 * span + (j == 0));
        if (a.spans) {
            if (tid == 0) {
                // the first part says who has the first, the last who has the last
                uint32_t* const cut = reinterpret_cast<uint32_t*>(a.cut + static_cast<uint64_t>(g * a.n_cg + cg) * n_seqs + s);
                if (j == 0) cut[0] = span;
                if (j_end == tiles.n) cut[1] = span;
            }
            left -= j_end - j;
            __syncthreads();   // the shared memory again
        }
    }
}

// ---- the parts of a sequence joined, and weights added up by position ------------------------------------------------
// grid = (workgroups, sequences): those of the columns first, then (a.mass) those of 1024 positions of a kv head each.
// Columns: HD / 4 threads of four values for each of SPLIT shares of a column's parts.  Positions: the scores lie as the attention
// left them, in the base-2 domain.
// What bounds it are its launch and two loads in a row: 4.8 us for 16 sequences' 5 rows of 32 heads in about 4 parts each, 4.9 us for two
// in 64, 10 us with the weights of 32 sequences of up to 8000 positions.
static constexpr uint32_t PAGED_MASS_POS = 1024;
// part p of a sequence lies this many slots behind slot 2 (its first workgroup)
__device__ __forceinline__ uint64_t paged_slot(uint32_t p) { return p == 0 ? 1 : 2 * static_cast<uint64_t>(p); }
template <int HD, int SPLIT>
__global__ __launch_bounds__(256, 8) void paged_finish_kernel(PagedView c, PagedOp a, uint32_t merge_blocks, uint32_t mass_blocks, float p_log2) {
    constexpr uint32_t COLS = 256 / (HD / 4 * SPLIT);
    __shared__ __attribute__((aligned(16))) float4 s_o[SPLIT > 1 ? 256 : 1];
    __shared__ float s_m[SPLIT > 1 ? 256 : 1], s_l[SPLIT > 1 ? 256 : 1];
    extern __shared__ float s_h[];   // [G] maximum, [G] 1 / sum
    const uint32_t s = blockIdx.y, tid = threadIdx.x;
    const PagedRows r = paged_rows(a.q_first, c.lens, s, a.n_rows, a.max_queries, c.max_len);
    const bool merge = blockIdx.x < merge_blocks;
    const uint32_t blocks = (a.n_cols + COLS - 1) / COLS, gx = merge ? blockIdx.x / blocks : 0;
    const uint2 cut = merge ? a.cut[static_cast<uint64_t>(gx) * gridDim.y + s] : make_uint2(0, 0);   // on its way beside the lengths
    if (r.bad || r.len == 0) return;   // written by the attention's launch
    const uint32_t n_cols = r.n * a.G;
    if (merge) {
        const uint32_t g = gx / a.n_cg, cg = gx % a.n_cg;
        const uint32_t x = tid % (HD / 4), share = tid / (HD / 4) % SPLIT, lcol = blockIdx.x % blocks * COLS + tid / (HD / 4 * SPLIT), col = cg * a.n_cols + lcol;
        if (cg * a.n_cols + blockIdx.x % blocks * COLS >= n_cols) return;
        const uint32_t parts = cut.y - cut.x + 1;
        if (parts == 1) return;
        const bool mine = lcol < a.n_cols && col < n_cols;
        const uint64_t first = (static_cast<uint64_t>(gx) * 2 * a.spans + 2 * cut.x) * a.n_cols + (mine ? lcol : 0);
        float M = PAGED_LOWEST, L = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (uint32_t p = share; p < parts; p += SPLIT) {
            const uint64_t at = first + paged_slot(p) * a.n_cols;
            const float2 y_ml = *reinterpret_cast<const float2*>(a.ml + at * 2);
            const float4 y = *reinterpret_cast<const float4*>(a.acc + at * HD + 4 * x);
            const float m = fmaxf(M, y_ml.x), f0 = __builtin_amdgcn_exp2f(M - m), f = __builtin_amdgcn_exp2f(y_ml.x - m);
            M = m;
            L = fmaf(f, y_ml.y, L * f0);
            o.x = fmaf(f, y.x, o.x * f0); o.y = fmaf(f, y.y, o.y * f0); o.z = fmaf(f, y.z, o.z * f0); o.w = fmaf(f, y.w, o.w * f0);
        }
        if constexpr (SPLIT > 1) {
            s_o[tid] = o;
            s_m[tid] = M;
            s_l[tid] = L;
            __syncthreads();
            if (share) return;
            for (uint32_t i = 1; i < SPLIT; ++i) M = fmaxf(M, s_m[tid + i * (HD / 4)]);
            L = 0.0f;
            o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t i = 0; i < SPLIT; ++i) {
                const uint32_t u = tid + i * (HD / 4);
                const float f = __builtin_amdgcn_exp2f(s_m[u] - M);
                const float4 y = s_o[u];
                L = fmaf(f, s_l[u], L);
                o.x = fmaf(f, y.x, o.x); o.y = fmaf(f, y.y, o.y); o.z = fmaf(f, y.z, o.z); o.w = fmaf(f, y.w, o.w);
            }
        }
        if (!mine) return;
        const float inv = 1.0f / L;
        o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
        *reinterpret_cast<float4*>(a.out + (r.first + static_cast<uint64_t>(col / a.G)) * a.out_stride + (g * a.G + col % a.G) * HD + 4 * x) = o;
        return;
    }
    const uint32_t g = (blockIdx.x - merge_blocks) / mass_blocks, i0 = (blockIdx.x - merge_blocks) % mass_blocks * PAGED_MASS_POS, P = r.len - 1;
    const PagedSeen v = paged_seen(P, a.window, a.n_sink);
    const uint32_t n_seen = v.sink_end + (P + 1 - v.start);
    if (i0 >= n_seen) return;
    float* const mass = a.mass + (static_cast<uint64_t>(s) * c.n_kv + g) * a.mass_stride;
    const float* const sc = a.scores + (static_cast<uint64_t>(s) * c.n_kv + g) * a.G * a.score_stride;
    // four positions a thread: their loads are in flight together, and beside those of the sums
    constexpr uint32_t N = PAGED_MASS_POS / 256;
    uint32_t t[N];
    float before[N], sum[N];
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
        const uint32_t i = min(i0 + u * 256 + tid, n_seen - 1);
        t[u] = i < v.sink_end ? i : v.start + (i - v.sink_end);
        before[u] = mass[t[u]];
        sum[u] = 0.0f;
    }
    for (uint32_t h = tid >> 6; h < a.G; h += 4) {   // a wavefront per head, its lanes over the parts
        const uint32_t cg = h / a.n_cols;
        const uint64_t gh = g * a.n_cg + cg;
        const uint2 cut_h = a.spans ? a.cut[gh * gridDim.y + s] : make_uint2(0, 0);
        float M = PAGED_LOWEST, L = 0.0f;
        if (cut_h.x == cut_h.y) {
            const float* const ml = a.ml_seq + ((gh * gridDim.y + s) * a.n_cols + h % a.n_cols) * 2;
            M = ml[0];
            L = ml[1];
        } else {
            const uint64_t first = (gh * 2 * a.spans + 2 * cut_h.x) * a.n_cols + h % a.n_cols;
            for (uint32_t p = tid & 63; p <= cut_h.y - cut_h.x; p += 64) {
                const float2 y = *reinterpret_cast<const float2*>(a.ml + (first + paged_slot(p) * a.n_cols) * 2);
                const float m = fmaxf(M, y.x);
                L = fmaf(__builtin_amdgcn_exp2f(y.x - m), y.y, L * __builtin_amdgcn_exp2f(M - m));
                M = m;
            }
            const float m = wave_max(M);
            L = wave_sum(L * __builtin_amdgcn_exp2f(M - m));
            M = m;
        }
        if ((tid & 63) == 0) {
            s_h[h] = M - p_log2;
            s_h[a.G + h] = L > 0.0f ? 1.0f / L : 0.0f;   // a head that is no number, or has met a bad page, adds nothing
        }
    }
    __syncthreads();
#pragma unroll 2
    for (uint32_t h = 0; h < a.G; ++h) {
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)   // an exponent is p_log2 at most, but for NaN: 0 times any number is 0
            sum[u] = fmaf(__builtin_amdgcn_exp2f(fminf(sc[h * a.score_stride + t[u]] - s_h[h], 100.0f)), s_h[a.G + h], sum[u]);
    }
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
        const bool fresh = a.mass_fresh && t[u] == P;
        if (i0 + u * 256 + tid < n_seen && (fresh || sum[u] != 0.0f)) mass[t[u]] = (fresh ? 0.0f : before[u]) + sum[u];
    }
}

template <typename KV, int HD>
static cera_hip_status paged_attn_launch(cera_hip_ctx* ctx, const cera_hip_paged_kv& c, const cera_hip_paged_attn& in) {
    constexpr bool HALF = sizeof(KV) == 2;
    const PagedView v = paged_view(c, in.max_len);
    PagedOp a{};
    a.q = in.q; a.out = in.out; a.q_first = in.q_first;
    a.q_stride = in.q_stride ? in.q_stride : static_cast<uint64_t>(in.n_heads) * HD;
    a.out_stride = in.out_stride ? in.out_stride : static_cast<uint64_t>(in.n_heads) * HD;
    a.kv_stride = in.kv_stride ? in.kv_stride : static_cast<uint64_t>(c.n_kv_heads) * HD;
    a.mass = in.mass;
    const bool weights = in.mass && !in.q_first;
    a.mass_stride = in.mass_stride;
    a.mass_fresh = in.k_new && in.mass_fresh;
    a.n_rows = in.n_rows;
    a.max_queries = in.q_first ? (in.max_queries ? std::min(in.max_queries, in.n_rows) : in.n_rows) : 1;
    a.G = in.n_heads / c.n_kv_heads;
    a.scale2 = in.scale * 1.44269504088896340736f;
    a.window = in.window; a.n_sink = in.n_sink;
    const uint64_t cols = static_cast<uint64_t>(a.max_queries) * a.G;
    // 16 sequences of 4000 positions, few columns' kernel and many columns': half cache, 32 columns 67 and 81 us, 40 columns 103 and 85;
    // f32, 16 columns 96 and 142, 20 columns 149 and 142.  Few columns of a half cache: 20 columns in one group of 32 take 64 us, in two of 16
    // 85, 32 columns 67 and 96.
    const bool many = in.q_first && cols > (HALF ? 32 : 16);
    const bool twin = HALF && cols <= 8, two = HALF && cols > 16;
    a.n_cols = many ? 128 : twin ? 8 : two ? 32 : 16;
    a.n_cg = static_cast<uint32_t>((cols + a.n_cols - 1) / a.n_cols);
    if (static_cast<uint64_t>(c.n_kv_heads) * a.n_cg > (1u << 23)) return cera_fail(ctx, CERA_HIP_ERR_SHAPE, "paged attention: too many rows of a sequence for one call");
    a.tile = HALF || many ? 32 : 16;
    a.round = std::max(1u, ctx->n_cu / c.n_kv_heads);
    const uint32_t wide = c.n_kv_heads * a.n_cg;
    const PagedCut cut = paged_cut(v.max_len, a.max_queries, a.window, a.n_sink, a.tile, wide, c.n_seqs, many, HALF, ctx->n_cu);
    a.spans = cut.spans;
    a.ordered = many && !a.spans && c.n_seqs >= 8 && c.n_seqs <= 64 && static_cast<uint64_t>(wide) * c.n_seqs > ctx->n_cu && static_cast<uint64_t>(a.n_cg) * c.n_seqs < (1u << 24);
    a.least = cut.least;
    a.score_stride = weights ? (static_cast<uint64_t>(v.max_len) + 31) / 32 * 32 : 0;
    // scores | results of parts | maxima and sums of parts | of whole sequences | who has a sequence's parts
    const uint64_t scores = a.score_stride * c.n_seqs * in.n_heads, seqs = static_cast<uint64_t>(wide) * c.n_seqs, ml_seq = weights ? seqs * a.n_cols * 2 : 0;
    auto parts = [&] { return static_cast<uint64_t>(wide) * 2 * a.spans * a.n_cols; };
    auto bytes = [&] { return 4 * (scores + parts() * (HD + 2) + ml_seq + (a.spans ? 2 * seqs : 0)); };
    void* ws = nullptr;
    // A workspace that has to grow takes half as much again, if there is room: it waits for all that is queued, and the scores of a longest
    // sequence that rises from call to call would need it anew every 32 positions.
    if (ctx->scratch[15] && bytes() > ctx->scratch_bytes[15]) CERA_TRY(cera_scratch_if_room(ctx, 15, bytes() + bytes() / 2, &ws));
    if (a.spans && !ws) {
        CERA_TRY(cera_scratch_if_room(ctx, 15, bytes(), &ws));
        if (!ws) a.spans = 0;
    }
    if (!ws && bytes()) CERA_TRY(cera_scratch(ctx, 15, bytes(), &ws));
    a.scores = static_cast<float*>(ws);
    a.acc = a.scores + scores;
    a.ml = a.acc + parts() * HD;
    a.ml_seq = a.ml + parts() * 2;
    a.cut = reinterpret_cast<uint2*>(a.ml_seq + ml_seq);
    if (in.k_new && many) {
        auto blocks = [&](uint64_t items) { return dim3(static_cast<uint32_t>(std::min<uint64_t>((items + 255) / 256, 1024)), c.n_seqs); };
        const uint64_t rows = static_cast<uint64_t>(a.max_queries) * c.n_kv_heads;
        hipLaunchKernelGGL((paged_append_kernel<KV, HD>), blocks(rows * (HD / 4)), dim3(256), 0, ctx->stream, v, static_cast<KV*>(c.k), static_cast<KV*>(c.v), in.k_new, in.v_new, a.kv_stride,
                           a.q_first, a.n_rows, a.max_queries);
        if (in.mass) hipLaunchKernelGGL(paged_fresh_kernel, blocks(rows), dim3(256), 0, ctx->stream, v, in.mass, in.mass_stride, a.q_first, a.n_rows, a.max_queries);
    } else {
        a.k_new = in.k_new;
        a.v_new = in.v_new;
    }
    const dim3 grid(wide, a.spans ? a.spans : c.n_seqs);
    auto launch = [&](auto tag) {
        using Work = decltype(tag);
        hipLaunchKernelGGL(paged_attn_kernel<Work>, grid, dim3(256), 0, ctx->stream, v, static_cast<KV*>(c.k), static_cast<KV*>(c.v), a, c.n_seqs);
    };
    if (many) {
        launch(PagedMany<KV, HD>{});
    } else if constexpr (HALF) {
        if (twin) { if (weights) launch(PagedFew<KV, HD, 1, true, true>{}); else launch(PagedFew<KV, HD, 1, true, false>{}); }
        else if (two) { if (weights) launch(PagedFew<KV, HD, 2, false, true>{}); else launch(PagedFew<KV, HD, 2, false, false>{}); }
        else { if (weights) launch(PagedFew<KV, HD, 1, false, true>{}); else launch(PagedFew<KV, HD, 1, false, false>{}); }
    } else {
        if (weights) launch(PagedFew<KV, HD, 1, false, true>{}); else launch(PagedFew<KV, HD, 1, false, false>{});
    }
    if (a.spans || weights) {
        // A column's parts shared out among eight: 15.8 us for one sequence of 8000 positions in 64 parts, 17.6 in one thread's turn; 1000 rows
        // in 6 parts 236 and 218.  Of more columns than make two thousand workgroups few have so many parts: 81 and 72 us for 48 sequences
        // of 5 rows, 74 and 64 for 16 of 20.
        const bool shared = a.spans > 8 && static_cast<uint64_t>(wide) * a.n_cols * c.n_seqs <= 2048;
        const uint32_t cols_wg = 256 / (HD / 4 * (shared ? 8 : 1)), merge = a.spans ? wide * ((a.n_cols + cols_wg - 1) / cols_wg) : 0;
        const uint64_t most = a.window ? std::min<uint64_t>(v.max_len, static_cast<uint64_t>(a.window) + a.n_sink) : v.max_len;
        const uint32_t mass = weights ? static_cast<uint32_t>((most + PAGED_MASS_POS - 1) / PAGED_MASS_POS) : 0;
        const dim3 blocks(merge + mass * c.n_kv_heads, c.n_seqs);
        if (shared) hipLaunchKernelGGL((paged_finish_kernel<HD, 8>), blocks, dim3(256), a.G * 8, ctx->stream, v, a, merge, mass, paged_p_log2<KV>);
        else hipLaunchKernelGGL((paged_finish_kernel<HD, 1>), blocks, dim3(256), a.G * 8, ctx->stream, v, a, merge, mass, paged_p_log2<KV>);
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
