// Attention of few (row, query head) columns of a kv head over a paged cache, split over the cache's length.
//
// For every column c: s[t] = scale q_c . K[t], out_c = sum_t softmax(s)[t] V[t], with running maximum and sum (base 2).  Both products
// run on the matrix cores, K and V straight from memory into registers:
//   S^T = K Q^T    A = 16 positions x 32 (f32: 4) dims: a lane loads 16 bytes of its position's row; B = the columns' q.
//   O^T = V^T P^T  B = the weights in the registers where the scores are: the lane of column c holds positions 4g + r of each 16;
//                  A = V^T: a lane loads whole pieces of its positions' rows and transposes them in registers (f32: takes them as they are).
// Half cache: K and V are exact in half precision, q and the weights are pairs hi + lo of halves that take columns c and c + 8 of the
// 16: f32's accuracy for the price of eight columns a product.  q is brought to a largest magnitude of 2^8 by a power of two, the
// weights to 2^14, so that low halves stay normal.  F32 cache: the f32 matrix instruction, 16 columns.
// What bounds it is the stream of K and V.
#pragma once
#include "paged.hip.h"

#define PAGED_LOWEST (-3.402823466e38f)   // a running maximum before any score: finite, so that -inf has weight 0
#define PAGED_P_LOG2 14.0f                // weights are held times 2^14

typedef float paged_f4 __attribute__((ext_vector_type(4)));
typedef _Float16 paged_h8 __attribute__((ext_vector_type(8)));

struct PagedOp {
    const float* q;
    float *out, *mass;
    const uint32_t* q_first;
    uint64_t q_stride, out_stride, mass_stride;
    uint32_t n_rows, max_queries, G;
    float scale2;   // times log2 e
    uint32_t window, n_sink;
    uint32_t n_cols, n_cg;                   // columns of a workgroup, groups of them a kv head
    uint32_t tile, part_tiles, max_parts;    // positions of a tile, tiles of a part
    float *acc, *ml;                         // [seq][kv head][group][part][column] x [HD], x (maximum, sum)
    float* scores;                           // [seq][head][score_stride]
    uint64_t score_stride;
};

// The tiles that columns c0 .. c1 see: [0, sinks) and [main, ...), n in all.
struct PagedTiles {
    uint32_t n, sinks, main;
    uint32_t P_lo, P_hi, start_lo, start_hi, sink_lo, sink_hi;   // of the first and the last of their rows
};
__device__ __forceinline__ PagedTiles paged_tiles(const PagedRows& r, uint32_t c0, uint32_t c1, const PagedOp& a) {
    PagedTiles t;
    t.P_lo = r.len - r.n + c0 / a.G;
    t.P_hi = r.len - r.n + c1 / a.G;
    const PagedSeen lo = paged_seen(t.P_lo, a.window, a.n_sink), hi = paged_seen(t.P_hi, a.window, a.n_sink);
    t.start_lo = lo.start; t.start_hi = hi.start;
    t.sink_lo = lo.sink_end; t.sink_hi = hi.sink_end;
    t.main = lo.start / a.tile;
    t.sinks = min((hi.sink_end + a.tile - 1) / a.tile, t.main);
    t.n = t.sinks + t.P_hi / a.tile - t.main + 1;
    return t;
}

__device__ __forceinline__ float paged_xor_max(float v) {   // over the four lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float paged_xor_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// What a wavefront holds of a tile.
template <typename KV, int HD> struct PagedTile;
template <int HD> struct PagedTile<kv_half, HD> {
    static constexpr int POS = 32, SUB = 2, KS = HD / 32, VW = HD / 32;   // VW: dwords of a lane's piece of a V row
    uint4 k[SUB][KS];
    uint32_t v[8][VW];
};
template <int HD> struct PagedTile<float, HD> {
    static constexpr int POS = 16, SUB = 1, KS = HD / 16, VW = HD / 64;   // VW: float4 of a lane's pieces of a V row
    float4 k[SUB][KS];
    float4 v[4][VW];
};

template <typename KV, int HD, int CB, bool MASS>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedView c, const KV* __restrict__ kp, const KV* __restrict__ vp, PagedOp a) {
    constexpr bool HALF = sizeof(KV) == 2;
    using Tile = PagedTile<KV, HD>;
    constexpr int POS = Tile::POS, SUB = Tile::SUB, KS = Tile::KS, NS = 4 * SUB;   // NS: scores of a lane and column block
    constexpr int CW = HALF ? 8 : 16, NC = CW * CB;
    constexpr int NO = HD / 16;                                                    // 16-row tiles of O^T
    constexpr int OLD = HD + 4;
    __shared__ __attribute__((aligned(16))) float s_o[4][NC][OLD];
    __shared__ float s_m[4][NC], s_l[4][NC];

    const uint32_t tid = threadIdx.x, lane = tid & 63, w = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid >> 6)));
    const uint32_t g = blockIdx.x / a.n_cg, cg = blockIdx.x % a.n_cg, part = blockIdx.y, s = blockIdx.z;
    const PagedRows r = paged_rows(a.q_first, c.lens, s, a.n_rows, a.max_queries, c.max_len);
    const uint32_t c0 = cg * NC;
    if (r.bad || r.len == 0) {
        // nothing is known of these rows but where they are
        if (part == 0 && cg == 0)
            for (uint32_t i = tid; i < a.G * HD; i += 256)
                for (uint32_t row = 0; row < r.n; ++row)
                    a.out[(r.first + static_cast<uint64_t>(row)) * a.out_stride + g * a.G * HD + i] = r.bad ? __builtin_nanf("") : 0.0f;
        return;
    }
    const uint32_t n_cols = r.n * a.G;
    if (c0 >= n_cols) return;
    const uint32_t c_last = min(c0 + NC, n_cols) - 1;
    const PagedTiles tiles = paged_tiles(r, c0, c_last, a);
    const uint32_t j_end = min((part + 1) * a.part_tiles, tiles.n);   // a part that is all has part_tiles up to 2^31 - 1
    if (part * a.part_tiles >= tiles.n) return;
    const bool alone = tiles.n <= a.part_tiles;

    // ---- the lane's columns
    const uint32_t lc = lane & 15, lg = lane >> 4;
    const bool low = HALF && (lc & 8);
    uint32_t P[CB], start[CB], sink[CB], col[CB];
    float mul[CB];
    uint4 qh[HALF ? CB : 1][HALF ? KS : 1];
    float4 qf[HALF ? 1 : CB][HALF ? 1 : KS];
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        col[b] = c0 + b * CW + (HALF ? lc & 7 : lc);
        const uint32_t cc = min(col[b], c_last), i = cc / a.G, h = g * a.G + cc % a.G;
        P[b] = r.len - r.n + i;
        const PagedSeen v = paged_seen(P[b], a.window, a.n_sink);
        start[b] = v.start;
        sink[b] = v.sink_end;
        const float* const qp = a.q + (r.first + static_cast<uint64_t>(i)) * a.q_stride + h * HD;
        mul[b] = a.scale2;
        if constexpr (HALF) {
            float x[KS][8];
            float top = 0.0f;
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                const float4 u = *reinterpret_cast<const float4*>(qp + 32 * st + 8 * lg), y = *reinterpret_cast<const float4*>(qp + 32 * st + 8 * lg + 4);
                x[st][0] = u.x; x[st][1] = u.y; x[st][2] = u.z; x[st][3] = u.w; x[st][4] = y.x; x[st][5] = y.y; x[st][6] = y.z; x[st][7] = y.w;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[st][e]));
            }
            top = paged_xor_max(top);
            int up = top > 0.0f && top < __builtin_inff() ? 9 - __builtin_amdgcn_frexp_expf(top) : 0;   // |q| 2^up < 2^9
            up = min(up, 100);
            mul[b] = ldexpf(a.scale2, -up);
            const uint32_t mask = low ? 0xFFFFE000u : 0u;
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                uint32_t d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y0 = ldexpf(x[st][2 * e], up), y1 = ldexpf(x[st][2 * e + 1], up);
                    const float z0 = y0 - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y0) & mask), z1 = y1 - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y1) & mask);
                    d[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(z0, z1));
                }
                qh[b][st] = make_uint4(d[0], d[1], d[2], d[3]);
            }
        } else {
#pragma unroll
            for (int st = 0; st < KS; ++st) qf[b][st] = *reinterpret_cast<const float4*>(qp + 16 * st + 4 * lg);
        }
    }

    // ---- tiles
    bool ok = true;
    const int32_t* const table = c.table + static_cast<uint64_t>(s) * c.max_pages;
    const uint32_t in_page = (1u << c.page_log2) - 1;
    auto tile_of = [&](uint32_t j) { return (j < tiles.sinks ? j : tiles.main + (j - tiles.sinks)) * POS; };
    // a row that some column sees
    auto live = [&](uint32_t t) { return t <= tiles.P_hi && (t >= tiles.start_lo || t < tiles.sink_hi); };
    auto whole = [&](uint32_t t0) { return (t0 >= tiles.start_hi && t0 + (POS - 1) <= tiles.P_lo) || t0 + (POS - 1) < tiles.sink_lo; };
    auto load = [&](Tile& f, uint32_t j) __attribute__((always_inline)) {
        const uint32_t t0 = tile_of(j);
        uint64_t at[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const uint32_t lo = t0 + 16 * u;
            uint32_t page = 0;
            if (lo <= tiles.P_hi && (lo + 15 >= tiles.start_lo || lo < tiles.sink_hi)) {
                page = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(table[lo >> c.page_log2]));
                if (page >= c.n_pages) {
                    ok = false;
                    page = 0;
                }
            }
            at[u] = page * c.page_stride + g * c.head_stride + static_cast<uint64_t>(lo & in_page) * HD;
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int st = 0; st < KS; ++st) f.k[u][st] = *reinterpret_cast<const std::remove_reference_t<decltype(f.k[u][st])>*>(kp + at[u] + lc * HD + (lg + 4 * st) * (16 / sizeof(KV)));
        if constexpr (HALF) {
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                const KV* const row = vp + at[p >> 2] + (4 * lg + (p & 3)) * HD + lc * (HD / 16);
                if constexpr (HD == 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(row);
                    f.v[p][0] = x.x; f.v[p][1] = x.y; f.v[p][2] = x.z; f.v[p][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(row);
                    f.v[p][0] = x.x; f.v[p][1] = x.y;
                }
            }
        } else {
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int h = 0; h < Tile::VW; ++h) f.v[p][h] = *reinterpret_cast<const float4*>(vp + at[0] + (4 * lg + p) * HD + 64 * h + 4 * lc);
        }
    };

    float m[CB], l[CB];
    paged_f4 o[CB][NO];
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        m[b] = PAGED_LOWEST;
        l[b] = 0.0f;
#pragma unroll
        for (int i = 0; i < NO; ++i) o[b][i] = paged_f4{0.f, 0.f, 0.f, 0.f};
    }

    auto compute = [&](Tile& f, uint32_t j) __attribute__((always_inline)) {
        const uint32_t t0 = tile_of(j);
        const bool edge = !whole(t0);
        if (edge) {   // what no column sees may hold anything, and 0 times that is not 0
#pragma unroll
            for (int p = 0; p < NS; ++p)
                if (!live(t0 + 16 * (p >> 2) + 4 * lg + (p & 3))) {
                    if constexpr (HALF) {
#pragma unroll
                        for (int e = 0; e < Tile::VW; ++e) f.v[p][e] = 0;
                    } else {
#pragma unroll
                        for (int e = 0; e < Tile::VW; ++e) f.v[p][e] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
        }
        uint4 ph[HALF ? CB : 1];
        float pf[HALF ? 1 : CB][4];
#pragma unroll
        for (int b = 0; b < CB; ++b) {
            float x[NS];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                paged_f4 d = {0.f, 0.f, 0.f, 0.f};
                if constexpr (HALF) {
#pragma unroll
                    for (int st = 0; st < KS; ++st)
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(paged_h8, f.k[u][st]), __builtin_bit_cast(paged_h8, qh[b][st]), d, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[e] += dpp_f<0x128>(d[e]);   // columns c and c + 8: row_ror 8
                } else {
#pragma unroll
                    for (int st = 0; st < KS; ++st) {
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32(f.k[u][st].x, qf[b][st].x, d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32(f.k[u][st].y, qf[b][st].y, d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32(f.k[u][st].z, qf[b][st].z, d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32(f.k[u][st].w, qf[b][st].w, d, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * u + e] = d[e] * mul[b];
            }
            if (edge) {
#pragma unroll
                for (int p = 0; p < NS; ++p) {
                    const uint32_t t = t0 + 16 * (p >> 2) + 4 * lg + (p & 3);
                    if (!(t < sink[b] || (t >= start[b] && t <= P[b]))) x[p] = -__builtin_inff();
                }
            }
            if (MASS) {
                if (!low && col[b] <= c_last) {
                    float* const to = a.scores + (static_cast<uint64_t>(s) * c.n_kv * a.G + g * a.G + col[b]) * a.score_stride + t0 + 4 * lg;
#pragma unroll
                    for (int u = 0; u < SUB; ++u) *reinterpret_cast<float4*>(to + 16 * u) = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
                }
            }
            float top = x[0];
#pragma unroll
            for (int p = 1; p < NS; ++p) top = fmaxf(top, x[p]);
            if (__any(top > m[b])) {
                const float mn = fmaxf(m[b], paged_xor_max(top)), f0 = __builtin_amdgcn_exp2f(m[b] - mn);
                m[b] = mn;
                l[b] *= f0;
#pragma unroll
                for (int i = 0; i < NO; ++i) o[b][i] *= f0;
            }
            const float base = m[b] - PAGED_P_LOG2;
#pragma unroll
            for (int p = 0; p < NS; ++p) {
                x[p] = __builtin_amdgcn_exp2f(x[p] - base);
                l[b] += x[p];
            }
            if constexpr (HALF) {
                const uint32_t mask = low ? 0xFFFFE000u : 0u;
                uint32_t d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z0 = x[2 * e] - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x[2 * e]) & mask),
                                z1 = x[2 * e + 1] - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x[2 * e + 1]) & mask);
                    d[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(z0, z1));
                }
                ph[b] = make_uint4(d[0], d[1], d[2], d[3]);
            } else {
#pragma unroll
                for (int p = 0; p < 4; ++p) pf[b][p] = x[p];
            }
        }
        // ---- O^T += V^T P^T
        if constexpr (HALF) {
#pragma unroll
            for (int i = 0; i < NO; ++i) {   // row n of tile i is dim n (HD / 16) + i
                uint32_t d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = __builtin_amdgcn_perm(f.v[2 * e + 1][i >> 1], f.v[2 * e][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
                const paged_h8 va = __builtin_bit_cast(paged_h8, make_uint4(d[0], d[1], d[2], d[3]));
#pragma unroll
                for (int b = 0; b < CB; ++b) o[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, __builtin_bit_cast(paged_h8, ph[b]), o[b][i], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int h = 0; h < Tile::VW; ++h) {   // row n of tile 4h + e is dim 64 h + 4 n + e
                    const float4 x = f.v[p][h];
#pragma unroll
                    for (int b = 0; b < CB; ++b) {
                        o[b][4 * h + 0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, pf[b][p], o[b][4 * h + 0], 0, 0, 0);
                        o[b][4 * h + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, pf[b][p], o[b][4 * h + 1], 0, 0, 0);
                        o[b][4 * h + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, pf[b][p], o[b][4 * h + 2], 0, 0, 0);
                        o[b][4 * h + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, pf[b][p], o[b][4 * h + 3], 0, 0, 0);
                    }
                }
        }
    };

    // the next tile's loads are on their way while one is multiplied, where the registers hold two
    uint32_t j = part * a.part_tiles + w;
    Tile fa;
    if constexpr (CB == 2 && HD == 128) {
        for (; j < j_end; j += 4) {
            load(fa, j);
            compute(fa, j);
        }
    } else {
        Tile fb;
        if (j < j_end) load(fa, j);
        while (j < j_end) {
            if (j + 4 < j_end) load(fb, j + 4);
            compute(fa, j);
            j += 4;
            if (j >= j_end) break;
            if (j + 4 < j_end) load(fa, j + 4);
            compute(fb, j);
            j += 4;
        }
    }

    // ---- the four wavefronts joined
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        l[b] = paged_xor_sum(l[b]);
        if (!ok) l[b] = __builtin_nanf("");
        const uint32_t lcol = b * CW + (HALF ? lc & 7 : lc);
        if (lg == 0 && !low) {
            s_m[w][lcol] = m[b];
            s_l[w][lcol] = l[b];
        }
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        const uint32_t lcol = b * CW + (HALF ? lc & 7 : lc);
        const float M = fmaxf(fmaxf(s_m[0][lcol], s_m[1][lcol]), fmaxf(s_m[2][lcol], s_m[3][lcol])), f0 = __builtin_amdgcn_exp2f(m[b] - M);
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = o[b][i][e];
                if constexpr (HALF) x += dpp_f<0x128>(x);
                const uint32_t d = HALF ? (4 * lg + e) * (HD / 16) + i : 64 * (i >> 2) + 4 * (4 * lg + e) + (i & 3);
                if (!low) s_o[w][lcol][d] = x * f0;
            }
    }
    __syncthreads();
    const uint64_t item = (static_cast<uint64_t>(s) * gridDim.x + blockIdx.x) * a.max_parts + part;
    for (uint32_t i = tid; i < NC * (HD / 4); i += 256) {
        const uint32_t lcol = i / (HD / 4), d = i % (HD / 4) * 4, cc = c0 + lcol;
        if (cc > c_last) continue;
        const float M = fmaxf(fmaxf(s_m[0][lcol], s_m[1][lcol]), fmaxf(s_m[2][lcol], s_m[3][lcol]));
        float L = 0.0f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            L = fmaf(__builtin_amdgcn_exp2f(s_m[u][lcol] - M), s_l[u][lcol], L);
            const float4 y = *reinterpret_cast<const float4*>(&s_o[u][lcol][d]);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        if (alone) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            *reinterpret_cast<float4*>(a.out + (r.first + static_cast<uint64_t>(cc / a.G)) * a.out_stride + (g * a.G + cc % a.G) * HD + d) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        } else {
            *reinterpret_cast<float4*>(a.acc + (item * NC + lcol) * HD + d) = x;
        }
        if ((MASS || !alone) && d == 0) {
            a.ml[(item * NC + lcol) * 2] = M;
            a.ml[(item * NC + lcol) * 2 + 1] = L;
        }
    }
}
