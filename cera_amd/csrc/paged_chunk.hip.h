// Attention of many (row, query head) columns of a kv head over a paged cache: chunks of new tokens.
//
// The products are those of paged_attn.hip.h in 32 x 32 x 16 form, S^T = K Q^T and O^T = V^T P^T, a wavefront for 32 columns, four of
// them on the same tiles of 32 positions in LDS.  A row's 16-byte pieces lie at places exchanged by its number, so that neither the
// keys' reads (a lane per row) nor the values' (transposing reads of 4 rows x 16 dims) meet in a bank.
// q and the weights are pairs hi + lo of halves here too, two products each: f32's accuracy at twice the operations.
// Half cache: loads go straight into LDS, the next tile's while this one is multiplied, one barrier a tile; the exchange is made on the
// way in, by what a lane loads.
// F32 cache: keys become pairs of halves on their way into LDS, brought to a largest magnitude below 2^15 by a power of two of each row,
// which goes into its scores: three products.  A query and a key are then off by 2^-23 at most, and the product of their low halves, which
// is left out, is below 2^-22.  Values and weights, whose sum has no room for a power of two a row, become three bfloat16 each, which
// have f32's range: six products.  All of it takes a quarter of the f32 instruction's clocks.
// What bounds it are the matrix cores and the power that they take.  2048 rows at 6000 positions, 32 heads of 128, half cache: 320 to
// 350 us from card to card, 0.52 to 0.47 PFLOP/s of the operator, twice that of the instruction, where a large library product reaches 1.14;
// 243 us where all data are zeros and the clock stays up.  The instruction is busy for 57 % of the cycles, the softmax between the
// products in the shadow of the other wavefronts; a workgroup alone takes 1.1 us a tile, two on a CU 2.2 together.  Keys are in no
// bank twice.  What did not help: the next scores beside the softmax (spills, twice the time), three buffers, two accumulators of scores.
// F32 cache: 2.1 us a tile of 64 dims for a lone workgroup, half of it the splitting of values into parts; two buffers of parts, put
// beside the products, cost the third workgroup a CU its registers: 50 us for 44.
#pragma once
#include <type_traits>

#include "lds_dma.hip.h"
#include "paged_attn.hip.h"

typedef float paged_f16v __attribute__((ext_vector_type(16)));
typedef __bf16 paged_b8 __attribute__((ext_vector_type(8)));
typedef short paged_s4 __attribute__((ext_vector_type(4)));
typedef short paged_s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) paged_s4* paged_lds4;

template <typename KV, int HD> struct PagedChunkShared;
template <int HD> struct PagedChunkShared<kv_half, HD> {
    __attribute__((aligned(1024))) uint8_t tile[2][2][32 * HD * 2];   // [buffer][keys, values]
    uint32_t bad, odd[4];   // a bad page; whether a block of this tile, of the next had infinities or NaN among values that only some columns see
};
template <int HD> struct PagedChunkShared<float, HD> {
    __attribute__((aligned(1024))) uint8_t tile[1][2][32 * HD * 2];   // keys' and values' first parts
    __attribute__((aligned(1024))) uint8_t more[3][32 * HD * 2];      // the keys' second part, the values' second and third
    __attribute__((aligned(16))) int up[32];                          // the power of two of a row of keys
    uint32_t bad, odd[4];   // a bad page; whether a wavefront's rows of the tile had infinities or NaN among values that only some columns see
};

// two floats as three bfloat16 each: 24 bits in all
__device__ __forceinline__ void paged_thirds(float x, float y, uint32_t (&d)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
        d[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        x -= __builtin_bit_cast(float, a & 0xFFFF0000u);
        y -= __builtin_bit_cast(float, b & 0xFFFF0000u);
    }
}

// place of 16-byte piece `piece` in row `row` of a tile
template <int HD, bool VALUES> __device__ __forceinline__ uint32_t paged_piece(uint32_t row, uint32_t piece) {
    if constexpr (HD == 128) return piece ^ (VALUES ? (row & 3) << 2 : row & 15);
    else return piece ^ (VALUES ? (row >> 1 & 1) << 2 : row >> 1 & 7);
}

// Tiles [j_begin, j_end) of sequence s for 128 columns from c0 on; slot: of a part's results.
template <typename KV, int HD>
__device__ __forceinline__ void paged_chunk_part(PagedChunkShared<KV, HD>& sh, const PagedView& c, const KV* __restrict__ kp, const KV* __restrict__ vp, const PagedOp& a, uint32_t g,
                                                 uint32_t cg, uint32_t s, const PagedRows& r, const PagedTiles& tiles, uint32_t c0, uint32_t c_last, uint32_t j_begin, uint32_t j_end,
                                                 uint32_t slot) {
    constexpr bool PAIRS = sizeof(KV) == 4;              // keys and values too
    constexpr int KS = HD / 16, ND = HD / 32;            // steps over the dims, 32-row tiles of O^T
    constexpr uint32_t ROW = HD * 2, PIECES = HD / 8;    // bytes and 16-byte pieces of a row
    constexpr uint32_t ROWS_KB = 1024 / ROW;             // rows of one load of a wavefront
    constexpr int LOADS = 16 / ROWS_KB;                  // loads of a block of 16 positions
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid >> 6)));
    const uint32_t lc = lane & 31, half = lane >> 5;
    const bool alone = j_begin == 0 && j_end == tiles.n;
    const uint32_t in_page = (1u << c.page_log2) - 1;
    const PagedConst<int32_t> table = paged_const(c.table + static_cast<uint64_t>(s) * c.max_pages);
    auto tile_of = [&](uint32_t j) { return (j < tiles.sinks ? j : tiles.main + (j - tiles.sinks)) * 32; };

    // ---- loads of a half cache: a wavefront has one block of 16 positions of the tile's keys or of its values
    bool ok = true;
    auto page_of = [&](uint32_t lo) __attribute__((always_inline)) {   // element of a position whose block of 16 some column sees
        uint32_t page = static_cast<uint32_t>(table[lo >> c.page_log2]);
        if (page >= c.n_pages) {
            ok = false;
            page = 0;
        }
        return page * c.page_stride + g * c.head_stride + static_cast<uint64_t>(lo & in_page) * HD;
    };
    auto used = [&](uint32_t lo) { return lo <= tiles.P_hi && (lo + 15 >= tiles.start_lo || lo < tiles.sink_hi); };
    auto live = [&](uint32_t t) { return t <= tiles.P_hi && (t >= tiles.start_lo || t < tiles.sink_hi); };
    const uint32_t blk = w & 1;
    const bool values = w >= 2;
    const uint8_t* const pool = reinterpret_cast<const uint8_t*>(values ? vp : kp);
    uint32_t off[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
        const uint32_t row = k * ROWS_KB + lane / PIECES, at = lane % PIECES;   // of the block; its number in the tile differs by 16, which no exchange looks at
        off[k] = row * ROW + (values ? paged_piece<HD, true>(row, at) : paged_piece<HD, false>(row, at)) * 16;
    }
    const uint32_t dst = lds_addr(sh.tile[0][values]) + blk * 16 * ROW;
    auto load = [&](uint32_t j, uint32_t buf) __attribute__((always_inline)) {
        const uint32_t lo = tile_of(j) + 16 * blk;
        if (used(lo)) {
            const uint8_t* const src = lds_dma_base(pool + page_of(lo) * sizeof(KV));
#pragma unroll
            for (int k = 0; k < LOADS; ++k) lds_dma_1k(src, off[k], dst + buf * (2 * 32 * ROW) + k * 1024);
        }
    };
    // ---- of an f32 cache: eight threads a row, its float4 number part, part + 8, ..; wavefronts 0 and 1 have the tile's first block
    constexpr int NF = HD / 32;
    const uint32_t f_row = tid >> 3, f_part = tid & 7;
    float4 fk[PAIRS ? NF : 1], fv[PAIRS ? NF : 1];
    auto fetch = [&](uint32_t j) __attribute__((always_inline)) {
        const uint32_t t0 = tile_of(j), lo = t0 + 16 * (w >> 1);
        const bool in = used(lo);
        const uint64_t at = (in ? page_of(lo) : 0) + static_cast<uint64_t>(f_row & 15) * HD + 4 * f_part;
        const bool seen_row = in && live(t0 + f_row);
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            fk[i] = fv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (seen_row) {   // what no column sees may be anything: zeros in its place
                fk[i] = *reinterpret_cast<const float4*>(kp + at + 32 * i);
                fv[i] = *reinterpret_cast<const float4*>(vp + at + 32 * i);
            }
        }
    };
    // Tiles that some column sees not all of (a few more may count).  0 times an infinity or NaN is not 0: there, such values leave the
    // product and are added to the columns that see them apart.
    const uint32_t look_from = tiles.P_lo < 31 ? 0 : tiles.P_lo - 31, look_below = tiles.start_lo + (tiles.P_hi - tiles.P_lo);
    auto put = [&](bool look) __attribute__((always_inline)) {
        if (look) {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < NF; ++i) most = paged_most(paged_most(paged_most(paged_most(most, fv[i].x), fv[i].y), fv[i].z), fv[i].w);
            const bool odd = __any(paged_odd(__builtin_bit_cast(float, most)));
            if (lane == 0) sh.odd[w] = odd;
            if (odd) {
#pragma unroll
                for (int i = 0; i < NF; ++i) fv[i] = make_float4(paged_even(fv[i].x), paged_even(fv[i].y), paged_even(fv[i].z), paged_even(fv[i].w));
            }
        }
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < NF; ++i) top = fmaxf(fmaxf(fmaxf(top, fabsf(fk[i].x)), fmaxf(fabsf(fk[i].y), fabsf(fk[i].z))), fabsf(fk[i].w));
        top = fmaxf(top, dpp_f<0xB1>(top));
        top = fmaxf(top, dpp_f<0x4E>(top));
        top = fmaxf(top, dpp_f<0x141>(top));   // of the row's eight lanes
        const int up = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;   // |k| 2^-up < 2^15
        if constexpr (PAIRS) {
            if (f_part == 0) sh.up[f_row] = up;
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                const float y[4] = {ldexpf(fk[i].x, -up), ldexpf(fk[i].y, -up), ldexpf(fk[i].z, -up), ldexpf(fk[i].w, -up)};
                uint32_t hi[2], lo[2], v[2][3];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    hi[e] = paged_near(y[2 * e], y[2 * e + 1]);
                    lo[e] = paged_near(y[2 * e] - h2f(hi[e] & 0xFFFF), y[2 * e + 1] - h2f(hi[e] >> 16));
                }
                paged_thirds(fv[i].x, fv[i].y, v[0]);
                paged_thirds(fv[i].z, fv[i].w, v[1]);
                const uint32_t k_at = f_row * ROW + paged_piece<HD, false>(f_row, (f_part + 8 * i) >> 1) * 16 + (f_part & 1) * 8;
                const uint32_t v_at = f_row * ROW + paged_piece<HD, true>(f_row, (f_part + 8 * i) >> 1) * 16 + (f_part & 1) * 8;
                *reinterpret_cast<uint2*>(sh.tile[0][0] + k_at) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(sh.more[0] + k_at) = make_uint2(lo[0], lo[1]);
                *reinterpret_cast<uint2*>(sh.tile[0][1] + v_at) = make_uint2(v[0][0], v[1][0]);
                *reinterpret_cast<uint2*>(sh.more[1] + v_at) = make_uint2(v[0][1], v[1][1]);
                *reinterpret_cast<uint2*>(sh.more[2] + v_at) = make_uint2(v[0][2], v[1][2]);
            }
        }
    };
    if (tid == 0) sh.bad = 0;
    uint32_t j = j_begin, buf = 0;
    if constexpr (PAIRS) fetch(j);
    else load(j, 0);

    // ---- the lane's column
    const uint32_t w0 = c0 + 32 * w, col = w0 + lc, cc = min(col, c_last), qi = cc / a.G, h = g * a.G + cc % a.G;
    const uint32_t P = r.len - r.n + qi;
    const PagedSeen seen = paged_seen(P, a.window, a.n_sink);
    // of the wavefront's first and last column
    const uint32_t P_lo = r.len - r.n + min(w0, c_last) / a.G, P_hi = r.len - r.n + min(w0 + 31, c_last) / a.G;
    const PagedSeen seen_lo = paged_seen(P_lo, a.window, a.n_sink), seen_hi = paged_seen(P_hi, a.window, a.n_sink);
    const bool idle = w0 > c_last;
    uint4 qh[KS], ql[KS];
    float mul;
    int q_up;
    {
        const float* const qp = a.q + (r.first + static_cast<uint64_t>(qi)) * a.q_stride + h * HD + 8 * half;
        float4 f[2 * KS];
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) f[i] = *reinterpret_cast<const float4*>(qp + 16 * (i >> 1) + 4 * (i & 1));
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) top = fmaxf(fmaxf(fmaxf(top, fabsf(f[i].x)), fmaxf(fabsf(f[i].y), fabsf(f[i].z))), fabsf(f[i].w));
        top = fmaxf(top, __shfl_xor(top, 32));
        int up = top > 0.0f && top < __builtin_inff() ? 9 - __builtin_amdgcn_frexp_expf(top) : 0;   // |q| 2^up < 2^9
        up = min(up, 100);
        q_up = up;
        // The scale's fraction goes into the query: a score is then its product times a power of two, exactly, whatever its size, and with the
        // sign the largest product is the largest score.
        const int e = __builtin_amdgcn_frexp_expf(a.scale2);
        mul = ldexpf(1.0f, min(PAIRS ? e : e - up, 127));
        const float by = ldexpf(__builtin_amdgcn_frexp_mantf(a.scale2), up);
#pragma unroll
        for (int st = 0; st < KS; ++st) {
            const float y[8] = {f[2 * st].x * by, f[2 * st].y * by, f[2 * st].z * by, f[2 * st].w * by, f[2 * st + 1].x * by, f[2 * st + 1].y * by, f[2 * st + 1].z * by, f[2 * st + 1].w * by};
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (PAIRS) {   // a key that is infinite is NaN in its second half
                    hi[e] = paged_near(y[2 * e], y[2 * e + 1]);
                    lo[e] = paged_near(y[2 * e] - h2f(hi[e] & 0xFFFF), y[2 * e + 1] - h2f(hi[e] >> 16));
                } else {
                    paged_query(y[2 * e], y[2 * e + 1], hi[e], lo[e]);
                }
            }
            qh[st] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            ql[st] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    float m = PAGED_LOWEST, base = PAGED_LOWEST, l = 0.0f;   // largest product; its score less the weights' exponent; sum of weights
    paged_f16v o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;

    // From 2^24 on a score has no room for the weights' factor: rounded, it would give weights that a half does not hold.
    auto base_of = [&](float top) { return PAIRS || fabsf(top) < 16777216.0f ? top - paged_p_log2<KV> : top; };

    // where a lane reads: keys by row lc, pieces 2 st + half; values by rows 4 half + (lane & 15) / 4, dims 16 (lane / 16 & 1) + 4 (lane & 3)
    const uint32_t v_row = 4 * half + (lane >> 2 & 3), v_piece = 2 * (lane >> 4 & 1) + (lane >> 1 & 1), v_byte = 8 * (lane & 1);

    auto add_odd = [&](uint32_t t0) __attribute__((always_inline)) {
        for (uint32_t t = t0; t < t0 + 32; ++t) {
            if (!live(t)) continue;
            const KV* const row = vp + page_of(t) + 4 * half;
            if (t < seen.sink_end || (t >= seen.start && t <= P)) {
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float y = static_cast<float>(row[32 * i + 8 * (e >> 2) + (e & 3)]);
                        if (paged_odd(y)) o[i][e] += y;
                        if ((e & 3) == 3) asm volatile("" ::: "memory");   // few registers: this hardly ever runs
                    }
            }
        }
    };

    for (; j < j_end; ++j, buf ^= 1) {
        const uint32_t t0 = tile_of(j);
        const bool look = t0 >= look_from || t0 < look_below;
        if constexpr (PAIRS) {
            if (j != j_begin) lds_barrier();   // every wavefront is past its reads
            put(look);
            if (j + 1 < j_end) fetch(j + 1);
            lds_barrier();
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wavefront's part of the tile is in
            if (values && look) {   // what no column sees becomes 0
                uint4* const at = reinterpret_cast<uint4*>(sh.tile[buf][1] + blk * 16 * ROW) + lane;
                uint4 y[LOADS];
                uint32_t most = 0;
#pragma unroll
                for (int k = 0; k < LOADS; ++k) {
                    y[k] = at[64 * k];
                    if (!live(t0 + 16 * blk + k * ROWS_KB + lane / PIECES)) at[64 * k] = y[k] = make_uint4(0, 0, 0, 0);
                    most = paged_most(paged_most(paged_most(paged_most(most, y[k].x), y[k].y), y[k].z), y[k].w);
                }
                const bool odd = __any(paged_odd_pair(most));
                if (odd)
#pragma unroll
                    for (int k = 0; k < LOADS; ++k) at[64 * k] = make_uint4(paged_even(y[k].x), paged_even(y[k].y), paged_even(y[k].z), paged_even(y[k].w));
                if (lane == 0) sh.odd[2 * (j & 1) + blk] = odd;
            }
            __syncthreads();   // the tile is whole, and every wavefront is past its reads of the other buffer
            if (j + 1 < j_end) load(j + 1, buf ^ 1);
        }
        if (idle || t0 > P_hi || (t0 + 31 < seen_lo.start && t0 >= seen_hi.sink_end)) continue;
        const uint32_t now = PAIRS ? 0 : buf;
        const uint8_t *const kt = sh.tile[now][0], *const vt = sh.tile[now][1];
        paged_f16v x;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
        for (int st = 0; st < KS; ++st) {
            const paged_h8 k = __builtin_bit_cast(paged_h8, *reinterpret_cast<const uint4*>(kt + lc * ROW + paged_piece<HD, false>(lc, 2 * st + half) * 16));
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, __builtin_bit_cast(paged_h8, qh[st]), x, 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, __builtin_bit_cast(paged_h8, ql[st]), x, 0, 0, 0);
            if constexpr (PAIRS) {
                const paged_h8 kl = __builtin_bit_cast(paged_h8, *reinterpret_cast<const uint4*>(sh.more[0] + lc * ROW + paged_piece<HD, false>(lc, 2 * st + half) * 16));
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, __builtin_bit_cast(paged_h8, qh[st]), x, 0, 0, 0);
            }
        }
        if constexpr (PAIRS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int4 up = *reinterpret_cast<const int4*>(&sh.up[8 * i + 4 * half]);
                x[4 * i] = ldexpf(x[4 * i], up.x - q_up);
                x[4 * i + 1] = ldexpf(x[4 * i + 1], up.y - q_up);
                x[4 * i + 2] = ldexpf(x[4 * i + 2], up.z - q_up);
                x[4 * i + 3] = ldexpf(x[4 * i + 3], up.w - q_up);
            }
        }
        // the values of the first 16 positions are on their way while the weights are made
        auto read = [&](const uint8_t* tile, int kk, int i) __attribute__((always_inline)) {
            // slot e of a half is position 16 kk + 8 (e / 4) + 4 half + e % 4
            paged_s4 v[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint32_t row = 16 * kk + 8 * b + v_row;
                v[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((paged_lds4)(tile + row * ROW + paged_piece<HD, true>(row, 4 * i + v_piece) * 16 + v_byte));
            }
            return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
        };
        paged_s8 va[PAIRS ? 1 : ND];
        if constexpr (!PAIRS) {
#pragma unroll
            for (int i = 0; i < ND; ++i) va[i] = read(vt, 0, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        // product e is of position t0 + 8 (e / 4) + 4 half + e % 4
        const bool edge = !((t0 >= seen_hi.start && t0 + 31 <= P_lo) || t0 + 31 < seen_lo.sink_end);
        uint32_t out_of_sight = 0;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t t = t0 + 8 * (e >> 2) + 4 * half + (e & 3);
                if (!(t < seen.sink_end || (t >= seen.start && t <= P))) {
                    x[e] = -__builtin_inff();
                    out_of_sight |= 1u << e;
                }
            }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
        if (__any(top > m)) {
            m = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
            const float b = m == PAGED_LOWEST ? base : base_of(m * mul), f0 = __builtin_amdgcn_exp2f(base - b);   // from nothing seen: 0
            base = b;
            l *= f0;
#pragma unroll
            for (int i = 0; i < ND; ++i) o[i] *= f0;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], mul, -base));
        if (edge) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = out_of_sight >> e & 1 ? 0.0f : x[e];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) l += x[e];
        // weights as halves (three bfloat16), their products with the values
        constexpr int NP = PAIRS ? 3 : 2;
        uint4 p[2][NP];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint32_t d[4][NP];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y0 = x[8 * kk + 2 * e], y1 = x[8 * kk + 2 * e + 1];
                if constexpr (PAIRS) {
                    paged_thirds(y0, y1, d[e]);
                } else {
                    d[e][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y0, y1));
                    d[e][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y0 - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y0) & 0xFFFFE000u),
                                                                                      y1 - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y1) & 0xFFFFE000u)));
                }
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) p[kk][n] = make_uint4(d[0][n], d[1][n], d[2][n], d[3][n]);
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                if constexpr (PAIRS) {
                    auto add = [&](paged_b8 v, int n) { o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(paged_b8, p[kk][n]), o[i], 0, 0, 0); };
                    const paged_b8 v3 = __builtin_bit_cast(paged_b8, read(sh.more[2], kk, i));
                    add(v3, 0);
                    const paged_b8 v2 = __builtin_bit_cast(paged_b8, read(sh.more[1], kk, i));
                    add(v2, 1);
                    add(v2, 0);
                    const paged_b8 v1 = __builtin_bit_cast(paged_b8, read(vt, kk, i));
                    add(v1, 2);
                    add(v1, 1);
                    add(v1, 0);
                } else {
                    const paged_h8 v = __builtin_bit_cast(paged_h8, kk == 0 ? va[i] : read(vt, kk, i));
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, __builtin_bit_cast(paged_h8, p[kk][0]), o[i], 0, 0, 0);
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, __builtin_bit_cast(paged_h8, p[kk][1]), o[i], 0, 0, 0);
                }
            }
        if (look) {
            const uint32_t* const odd = &sh.odd[PAIRS ? 0 : 2 * (j & 1)];
            if (odd[0] | odd[1] | (PAIRS ? odd[2] | odd[3] : 0)) add_odd(t0);
        }
    }
    l += __shfl_xor(l, 32);
    if (!ok) sh.bad = 1;
    __syncthreads();
    if (sh.bad) l = __builtin_nanf("");
    if (col > c_last) return;
    const uint64_t item = (static_cast<uint64_t>(g * a.n_cg + cg) * 2 * a.spans + slot) * a.n_cols + 32 * w + lc;
    float* const to = alone ? a.out + (r.first + static_cast<uint64_t>(qi)) * a.out_stride + h * HD : a.acc + item * HD;
    const float inv = !alone ? 1.0f : 1.0f / l;   // a row sees itself
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *reinterpret_cast<float4*>(to + 32 * i + 8 * e + 4 * half) = make_float4(o[i][4 * e] * inv, o[i][4 * e + 1] * inv, o[i][4 * e + 2] * inv, o[i][4 * e + 3] * inv);
    if (!alone && half == 0) *reinterpret_cast<float2*>(a.ml + item * 2) = make_float2(base + paged_p_log2<KV>, l);
}
