// Attention of few (row, query head) columns of a kv head over a paged cache, split over the cache's length.
//
// For every column c: s[t] = scale q_c . K[t], out_c = sum_t softmax(s)[t] V[t], with running maximum and sum (base 2).  Both products
// run on the matrix cores, K and V straight from memory into registers:
//   S^T = K Q^T    A = 16 positions x 32 (f32: 4) dims: a lane loads 16 bytes of its position's row; B = the columns' q.
//   O^T = V^T P^T  B = the weights in the registers where the scores are: the lane of column c holds positions 4g + r of each 16;
//                  A = V^T: a lane loads whole pieces of its positions' rows and transposes them in registers (f32: takes them as they are).
// Half cache: K and V are exact in half precision, q and the weights are pairs hi + lo of halves, for f32's accuracy: with up to eight
// columns (TWIN) the pair takes columns c and c + 8 of the 16 in one product, else hi and lo have a product each.  q is brought to a
// largest magnitude of 2^8 by a power of two, the weights to 2^14, so that low halves stay normal.  F32 cache: the f32 matrix
// instruction, 16 columns.
// What bounds it is the stream of K and V: 32 sequences of 8000 positions, 8 kv heads of 128, half cache, 162 us for 1.05 GB, 6.5 TB/s,
// where a large copy reaches 4.8; an f32 cache the same.  Hence: non-temporal loads (187 us without; a cache that the last-level
// cache still holds costs 5 to 10 % more so, but between two steps of a model come its weights), no LDS between memory and the matrix cores (a tile
// is read by one wavefront, once), the next tile's keys in flight from behind the scores on and its values from behind the weights on,
// page numbers by scalar loads, whose wait is not one for the tiles.
// Eight columns and their low halves in one product: 167 us for those sequences, with two products 174.
#pragma once
#include "paged.hip.h"

#define PAGED_LOWEST (-3.402823466e38f)   // a running maximum before any score: finite, so that -inf has weight 0
// Weights are held times 2^14 for a half cache, whose values are below 2^16; for an f32 cache times 2^-4, so that 2^30 of them on values of
// 10^30 stay in f32's range.
template <typename KV> constexpr float paged_p_log2 = sizeof(KV) == 2 ? 14.0f : -4.0f;

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
    const float *k_new, *v_new;              // few columns: the rows' own keys and values, or null
    uint64_t kv_stride;
    uint32_t mass_fresh;
    uint32_t n_cols, n_cg;                   // columns of a workgroup, groups of them a kv head
    uint32_t tile;                           // positions of a tile
    uint32_t round;                          // groups of a kv head that the chip's CUs have one each of
    bool ordered;                            // workgroups take uncut groups of all sequences, the longest first
    uint32_t spans, least;                   // workgroups of a kv head and group, and their least number of tiles; spans 0: one for each sequence
    float *acc, *ml;                         // [kv head, group][2 spans][column] x [HD], x (maximum, sum)
    uint2* cut;                              // [kv head, group][seq]: first and last workgroup of a sequence that is cut
    float* ml_seq;                           // with mass: [kv head, group][seq][column] x (maximum, sum) of a sequence that is not
    float* scores;                           // with mass: [seq][head][score_stride]
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

// Tiles of sequence s for the columns from c0 on: none where it has no such columns; where nothing can be read, one for the first
// columns' workgroup, which writes the rows.
__device__ __forceinline__ uint32_t paged_count(const PagedView& c, const PagedOp& a, uint32_t s, uint32_t c0) {
    const PagedRows r = paged_rows(a.q_first, c.lens, s, a.n_rows, a.max_queries, c.max_len);
    if (r.bad || r.len == 0) return c0 == 0;
    const uint32_t n_cols = r.n * a.G;
    return c0 < n_cols ? paged_tiles(r, c0, min(c0 + a.n_cols, n_cols) - 1, a).n : 0;
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

// Two floats as halves.  TWIN: a lane's share of the pair, the high halves (mask 0) or the low ones (mask PAGED_HIGH); else both.
#define PAGED_HIGH 0xFFFFE000u   // a float's bits that a half holds, rounded towards 0
template <bool TWIN> __device__ __forceinline__ void paged_pair(float x, float y, uint32_t mask, uint32_t& hi, uint32_t& lo) {
    const uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
    if constexpr (TWIN) {
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x - __builtin_bit_cast(float, a & mask), y - __builtin_bit_cast(float, b & mask)));
    } else {
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x - __builtin_bit_cast(float, a & PAGED_HIGH), y - __builtin_bit_cast(float, b & PAGED_HIGH)));
    }
}

// A query's values as halves, high ones rounded away from 0: low ones then have the other sign, or are 0, and a key that is infinite
// gives inf - inf or inf * 0, which is NaN, whatever the signs.  A NaN stays one in the low half.
typedef _Float16 paged_h2 __attribute__((ext_vector_type(2)));
typedef float paged_f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t paged_near(float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(paged_f2{x, y}, paged_h2)); }   // to the nearest even
__device__ __forceinline__ void paged_query(float x, float y, uint32_t& hi, uint32_t& lo) {
    const float a = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) + ~PAGED_HIGH) & PAGED_HIGH), b = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, y) + ~PAGED_HIGH) & PAGED_HIGH);
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    lo = paged_near(x - a, y - b);
}

template <int NC, int HD> struct PagedShared {
    __attribute__((aligned(16))) float o[4][NC][HD + 4];
    float m[4][NC], l[4][NC];
};

// Tiles [j_begin, j_end) of sequence s for one group of columns, by a workgroup of four wavefronts; slot: of a part's results.
template <typename KV, int HD, int CB, bool TWIN, bool MASS>
__device__ __forceinline__ void paged_attn_part(PagedShared<(TWIN ? 8 : 16) * CB, HD>& sh, const PagedView& c, KV* __restrict__ kp, KV* __restrict__ vp, const PagedOp& a, uint32_t g,
                                                uint32_t cg, uint32_t s, const PagedRows& r, const PagedTiles& tiles, uint32_t c0, uint32_t c_last, uint32_t j_begin, uint32_t j_end, uint32_t slot) {
    constexpr bool HALF = sizeof(KV) == 2;
    using Tile = PagedTile<KV, HD>;
    constexpr int POS = Tile::POS, SUB = Tile::SUB, KS = Tile::KS, NS = 4 * SUB;   // NS: scores of a lane and column block
    static_assert(!TWIN || (HALF && CB == 1), "eight columns and their low halves");
    constexpr int CW = TWIN ? 8 : 16, NC = CW * CB;
    constexpr int NO = HD / 16;                                                    // 16-row tiles of O^T
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid >> 6)));
    const bool alone = j_begin == 0 && j_end == tiles.n;
    const uint32_t lc = lane & 15, lg = lane >> 4;
    // ---- tiles
    bool ok = true;
    const PagedConst<int32_t> table = paged_const(c.table + static_cast<uint64_t>(s) * c.max_pages);
    const uint32_t in_page = (1u << c.page_log2) - 1;
    auto tile_of = [&](uint32_t j) { return (j < tiles.sinks ? j : tiles.main + (j - tiles.sinks)) * POS; };
    // a lane's first bytes of a 16-position block of keys, of values
    const uint32_t k_lane = (lc * HD + lg * (16 / sizeof(KV))) * sizeof(KV), v_lane = (4 * lg * HD + lc * (HALF ? HD / 16 : 4)) * sizeof(KV);
    // a row that some column sees
    auto live = [&](uint32_t t) { return t <= tiles.P_hi && (t >= tiles.start_lo || t < tiles.sink_hi); };
    auto whole = [&](uint32_t t0) { return (t0 >= tiles.start_hi && t0 + (POS - 1) <= tiles.P_lo) || t0 + (POS - 1) < tiles.sink_lo; };
    Tile f;
    uint64_t at[SUB];   // elements of the tile's blocks of 16 positions
    auto find = [&](uint32_t j) __attribute__((always_inline)) {
        const uint32_t t0 = tile_of(j);
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const uint32_t lo = t0 + 16 * u;
            uint32_t page = 0;
            if (lo <= tiles.P_hi && (lo + 15 >= tiles.start_lo || lo < tiles.sink_hi)) {
                page = static_cast<uint32_t>(table[lo >> c.page_log2]);
                if (page >= c.n_pages) {
                    ok = false;
                    page = 0;
                }
            }
            at[u] = page * c.page_stride + g * c.head_stride + static_cast<uint64_t>(lo & in_page) * HD;
        }
    };
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const uint8_t* const base = reinterpret_cast<const uint8_t*>(kp + at[u]) + k_lane;
#pragma unroll
            for (int st = 0; st < KS; ++st) f.k[u][st] = paged_stream<std::remove_reference_t<decltype(f.k[u][st])>>(base + 64 * st);
        }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const uint8_t* const base = reinterpret_cast<const uint8_t*>(vp + at[u]) + v_lane;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if constexpr (!HALF) {
#pragma unroll
                    for (int h = 0; h < Tile::VW; ++h) f.v[p][h] = paged_stream<float4>(base + p * HD * 4 + 256 * h);
                } else if constexpr (HD == 128) {
                    const uint4 x = paged_stream<uint4>(base + p * HD * 2);
                    f.v[4 * u + p][0] = x.x; f.v[4 * u + p][1] = x.y; f.v[4 * u + p][2] = x.z; f.v[4 * u + p][3] = x.w;
                } else {
                    const uint2 x = paged_stream<uint2>(base + p * HD * 2);
                    f.v[4 * u + p][0] = x.x; f.v[4 * u + p][1] = x.y;
                }
            }
        }
    };
    // The call's own rows, positions new0 on, are not in their pages yet: lanes that hold a piece of one take it from the new rows,
    // narrowed as the cache's.
    const uint32_t new0 = r.len - r.n;
    auto own_row = [&](const float* rows, uint32_t t) { return rows + (r.first + static_cast<uint64_t>(t - new0)) * a.kv_stride + g * HD; };
    auto own_key = [&](uint32_t t0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const uint32_t t = t0 + 16 * u + lc;
            if (t >= new0 && t <= tiles.P_hi) {
                const float* const kn = own_row(a.k_new, t) + lg * (16 / sizeof(KV));
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    if constexpr (HALF) {
                        const float4 y = *reinterpret_cast<const float4*>(kn + 32 * st), z = *reinterpret_cast<const float4*>(kn + 32 * st + 4);
                        f.k[u][st] = make_uint4(f2h(y.x) | f2h(y.y) << 16, f2h(y.z) | f2h(y.w) << 16, f2h(z.x) | f2h(z.y) << 16, f2h(z.z) | f2h(z.w) << 16);
                    } else {
                        f.k[u][st] = *reinterpret_cast<const float4*>(kn + 16 * st);
                    }
                }
            }
        }
    };
    auto own_value = [&](uint32_t t0) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NS; ++p) {
            const uint32_t t = t0 + 16 * (p >> 2) + 4 * lg + (p & 3);
            if (t >= new0 && t <= tiles.P_hi) {
                const float* const vn = own_row(a.v_new, t) + lc * (HALF ? HD / 16 : 4);
#pragma unroll
                for (int e = 0; e < Tile::VW; ++e) {
                    if constexpr (HALF) {
                        const float2 y = *reinterpret_cast<const float2*>(vn + 2 * e);
                        f.v[p][e] = f2h(y.x) | f2h(y.y) << 16;
                    } else {
                        f.v[p][e] = *reinterpret_cast<const float4*>(vn + 64 * e);
                    }
                }
            }
        }
    };

    // the first tile is on its way while the columns are made ready
    uint32_t j = j_begin + w;
    if (j < j_end) {
        find(j);
        load_k();
        load_v();
    }

    // ---- the lane's columns
    const bool low = TWIN && (lc & 8);
    uint32_t P[CB], start[CB], sink[CB], col[CB];
    float mul[CB];
    // two blocks of pairs are more than the registers hold beside the rest: those lie in LDS, where the results meet later
    constexpr bool AWAY = HALF && CB == 2;
    uint4 qh[HALF && !AWAY ? CB : 1][HALF && !AWAY ? KS : 1], ql[HALF && !TWIN && !AWAY ? CB : 1][HALF && !TWIN && !AWAY ? KS : 1];
    uint4* const q_away = reinterpret_cast<uint4*>(&sh.o[0][0][0]) + lane;   // [block][step][high, low][lane]
    float4 qf[HALF ? 1 : CB][HALF ? 1 : KS];
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        col[b] = c0 + b * CW + (TWIN ? lc & 7 : lc);
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
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                uint32_t d[4], n[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    paged_query(ldexpf(x[st][2 * e], up), ldexpf(x[st][2 * e + 1], up), d[e], n[e]);
                    if (low) d[e] = n[e];
                }
                if constexpr (AWAY) {
                    if (w == static_cast<uint32_t>(b)) {
                        q_away[(2 * (b * KS + st)) * 64] = make_uint4(d[0], d[1], d[2], d[3]);
                        q_away[(2 * (b * KS + st) + 1) * 64] = make_uint4(n[0], n[1], n[2], n[3]);
                    }
                } else {
                    qh[b][st] = make_uint4(d[0], d[1], d[2], d[3]);
                    if constexpr (!TWIN) ql[b][st] = make_uint4(n[0], n[1], n[2], n[3]);
                }
            }
        } else {
#pragma unroll
            for (int st = 0; st < KS; ++st) qf[b][st] = *reinterpret_cast<const float4*>(qp + 16 * st + 4 * lg);
        }
    }

    if constexpr (AWAY) lds_barrier();
    // An infinity or NaN in a query or in a key that it sees makes their score not finite.  +inf and NaN reach the sum by themselves;
    // -inf, whose weight would be 0, cannot come from a half cache (paged_query); over an f32 cache it shows in the smallest score that a
    // lane has seen: 129 us for 128 of two sequences of up to 60000.
    float m[CB], l[CB], least[HALF ? 1 : CB];
    paged_f4 o[CB][NO];
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        m[b] = PAGED_LOWEST;
        l[b] = 0.0f;
        if constexpr (!HALF) least[b] = 0.0f;
#pragma unroll
        for (int i = 0; i < NO; ++i) o[b][i] = paged_f4{0.f, 0.f, 0.f, 0.f};
    }

    for (; j < j_end; j += 4) {
        const uint32_t t0 = tile_of(j);
        const bool edge = !whole(t0);
        const bool newest = a.k_new && t0 + POS > new0, more = j + 4 < j_end;
        if (newest) own_key(t0);
        if (more) find(j + 4);
        uint4 ph[HALF ? CB : 1], pl[HALF && !TWIN ? CB : 1];
        float pf[HALF ? 1 : CB][4];
        float x[CB][NS];
#pragma unroll
        for (int b = 0; b < CB; ++b) {
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                paged_f4 d = {0.f, 0.f, 0.f, 0.f};
                if constexpr (HALF) {
#pragma unroll
                    for (int st = 0; st < KS; ++st) {
                        uint4 hi, lo;
                        if constexpr (AWAY) {
                            hi = q_away[(2 * (b * KS + st)) * 64];
                            lo = q_away[(2 * (b * KS + st) + 1) * 64];
                        } else {
                            hi = qh[b][st];
                            if constexpr (!TWIN) lo = ql[b][st];
                        }
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(paged_h8, f.k[u][st]), __builtin_bit_cast(paged_h8, hi), d, 0, 0, 0);
                        if constexpr (!TWIN) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(paged_h8, f.k[u][st]), __builtin_bit_cast(paged_h8, lo), d, 0, 0, 0);
                    }
                    if constexpr (TWIN) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[e] += dpp_f<0x128>(d[e]);   // columns c and c + 8: row_ror 8
                    }
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
                for (int e = 0; e < 4; ++e) x[b][4 * u + e] = d[e] * mul[b];
            }
        }
        // the next tile's keys are on their way while this one's weights are made, its values while the next one's scores are
        if (more) load_k();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < CB; ++b) {
            if (edge) {
#pragma unroll
                for (int p = 0; p < NS; ++p) {
                    const uint32_t t = t0 + 16 * (p >> 2) + 4 * lg + (p & 3);
                    const bool sees = t < sink[b] || (t >= start[b] && t <= P[b]);
                    if constexpr (!HALF) least[b] = fminf(least[b], sees ? x[b][p] : 0.0f);
                    if (!sees) x[b][p] = -__builtin_inff();
                }
            } else if constexpr (!HALF) {
#pragma unroll
                for (int p = 0; p < NS; ++p) least[b] = fminf(least[b], x[b][p]);
            }
            if (MASS) {
                if (!low && col[b] <= c_last) {
                    float* const to = a.scores + (static_cast<uint64_t>(s) * c.n_kv * a.G + g * a.G + col[b]) * a.score_stride + t0 + 4 * lg;
#pragma unroll
                    for (int u = 0; u < SUB; ++u) *reinterpret_cast<float4*>(to + 16 * u) = make_float4(x[b][4 * u], x[b][4 * u + 1], x[b][4 * u + 2], x[b][4 * u + 3]);
                }
            }
            float top = x[b][0];
#pragma unroll
            for (int p = 1; p < NS; ++p) top = fmaxf(top, x[b][p]);
            if (__any(top > m[b])) {
                const float mn = fmaxf(m[b], paged_xor_max(top)), f0 = __builtin_amdgcn_exp2f(m[b] - mn);
                m[b] = mn;
                l[b] *= f0;
#pragma unroll
                for (int i = 0; i < NO; ++i) o[b][i] *= f0;
            }
            const float base = m[b] - paged_p_log2<KV>;
#pragma unroll
            for (int p = 0; p < NS; ++p) {
                x[b][p] = __builtin_amdgcn_exp2f(x[b][p] - base);
                l[b] += x[b][p];
            }
            if constexpr (HALF) {
                const uint32_t mask = low ? PAGED_HIGH : 0u;
                uint32_t d[4], n[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) paged_pair<TWIN>(x[b][2 * e], x[b][2 * e + 1], mask, d[e], n[e]);
                ph[b] = make_uint4(d[0], d[1], d[2], d[3]);
                if constexpr (!TWIN) pl[b] = make_uint4(n[0], n[1], n[2], n[3]);
            } else {
#pragma unroll
                for (int p = 0; p < 4; ++p) pf[b][p] = x[b][p];
            }
        }
        if (newest) own_value(t0);
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
        // Nor is 0 times an infinity or NaN that only some columns see: those leave the product and are added to theirs here.
        if (edge && tiles.P_lo != tiles.P_hi) {
            uint32_t most = 0;
#pragma unroll
            for (int p = 0; p < NS; ++p)
#pragma unroll
                for (int e = 0; e < Tile::VW; ++e) {
                    if constexpr (HALF) most = paged_most(most, f.v[p][e]);
                    else most = paged_most(paged_most(paged_most(paged_most(most, f.v[p][e].x), f.v[p][e].y), f.v[p][e].z), f.v[p][e].w);
                }
            if (__any(HALF ? paged_odd_pair(most) : paged_odd(__builtin_bit_cast(float, most)))) {
#pragma unroll
                for (int p = 0; p < NS; ++p)
#pragma unroll
                    for (int e = 0; e < Tile::VW; ++e) {
                        if constexpr (HALF) f.v[p][e] = paged_even(f.v[p][e]);
                        else f.v[p][e] = make_float4(paged_even(f.v[p][e].x), paged_even(f.v[p][e].y), paged_even(f.v[p][e].z), paged_even(f.v[p][e].w));
                    }
                for (uint32_t t = t0; t < t0 + POS; ++t) {
                    if (!live(t)) continue;
                    const uint32_t page = static_cast<uint32_t>(table[t >> c.page_log2]);
                    const KV* const row = vp + paged_row<HD>(c, page < c.n_pages ? page : 0, g, t);
                    const float* const vn = a.k_new && t >= new0 ? own_row(a.v_new, t) : nullptr;
#pragma unroll
                    for (int b = 0; b < CB; ++b)
                        if (!low && (t < sink[b] || (t >= start[b] && t <= P[b]))) {
#pragma unroll
                            for (int i = 0; i < NO; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t dim = HALF ? (4 * lg + e) * (HD / 16) + i : 64 * (i >> 2) + 4 * (4 * lg + e) + (i & 3);
                                    const float y = vn ? static_cast<float>(static_cast<KV>(vn[dim])) : static_cast<float>(row[dim]);
                                    if (paged_odd(y)) o[b][i][e] += y;
                                    if (e == 3) asm volatile("" ::: "memory");   // few registers: this hardly ever runs
                                }
                        }
                }
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
                for (int b = 0; b < CB; ++b) {
                    o[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, __builtin_bit_cast(paged_h8, ph[b]), o[b][i], 0, 0, 0);
                    if constexpr (!TWIN) o[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, __builtin_bit_cast(paged_h8, pl[b]), o[b][i], 0, 0, 0);
                }
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
        if (more) load_v();
        __builtin_amdgcn_sched_barrier(0);
    }

    // ---- the new rows into their pages, by the workgroup that has the last one's tile
    if (a.k_new && cg == (r.n * a.G - 1) / NC && j_end == tiles.n) {
        if (!MASS && a.q_first && a.mass)   // a chunk's new positions start at no weight
            for (uint32_t i = tid; i < r.n; i += 256) a.mass[(static_cast<uint64_t>(s) * c.n_kv + g) * a.mass_stride + new0 + i] = 0.0f;
        for (uint32_t i = tid; i < r.n * (HD / 2); i += 256) {
            const uint32_t t = new0 + i / (HD / 2), part = i % (HD / 2), c4 = part % (HD / 4);
            bool in = true;
            const uint32_t page = paged_page(c, s, t, in);
            if (in) KvOps<KV>::st4((part < HD / 4 ? kp : vp) + paged_row<HD>(c, page, g, t), c4, *reinterpret_cast<const float4*>(own_row(part < HD / 4 ? a.k_new : a.v_new, t) + 4 * c4));
        }
    }
    // ---- the four wavefronts joined
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        if constexpr (!HALF) l[b] = least[b] == -__builtin_inff() ? __builtin_nanf("") : l[b];
        if (!ok) l[b] = __builtin_nanf("");
        l[b] = paged_xor_sum(l[b]);
        const uint32_t lcol = b * CW + (TWIN ? lc & 7 : lc);
        if (lg == 0 && !low) {
            sh.m[w][lcol] = m[b];
            sh.l[w][lcol] = l[b];
        }
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < CB; ++b) {
        const uint32_t lcol = b * CW + (TWIN ? lc & 7 : lc);
        const float M = fmaxf(fmaxf(sh.m[0][lcol], sh.m[1][lcol]), fmaxf(sh.m[2][lcol], sh.m[3][lcol])), f0 = __builtin_amdgcn_exp2f(m[b] - M);
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = o[b][i][e];
                if constexpr (TWIN) x += dpp_f<0x128>(x);
                const uint32_t d = HALF ? (4 * lg + e) * (HD / 16) + i : 64 * (i >> 2) + 4 * (4 * lg + e) + (i & 3);
                if (!low) sh.o[w][lcol][d] = x * f0;
            }
    }
    __syncthreads();
    const uint32_t gx = g * a.n_cg + cg;
    const uint64_t item = static_cast<uint64_t>(gx) * 2 * a.spans + slot;
    for (uint32_t i = tid; i < NC * (HD / 4); i += 256) {
        const uint32_t lcol = i / (HD / 4), d = i % (HD / 4) * 4, cc = c0 + lcol;
        if (cc > c_last) continue;
        const float M = fmaxf(fmaxf(sh.m[0][lcol], sh.m[1][lcol]), fmaxf(sh.m[2][lcol], sh.m[3][lcol]));
        float L = 0.0f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            L = fmaf(__builtin_amdgcn_exp2f(sh.m[u][lcol] - M), sh.l[u][lcol], L);
            const float4 y = *reinterpret_cast<const float4*>(&sh.o[u][lcol][d]);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        if (alone) {
            const float inv = 1.0f / L;   // a row sees itself
            *reinterpret_cast<float4*>(a.out + (r.first + static_cast<uint64_t>(cc / a.G)) * a.out_stride + (g * a.G + cc % a.G) * HD + d) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            if (MASS && d == 0) *reinterpret_cast<float2*>(a.ml_seq + ((static_cast<uint64_t>(gx) * a.n_rows + s) * NC + lcol) * 2) = make_float2(M, L);
        } else {
            *reinterpret_cast<float4*>(a.acc + (item * NC + lcol) * HD + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(a.ml + (item * NC + lcol) * 2) = make_float2(M, L);
        }
    }
}
