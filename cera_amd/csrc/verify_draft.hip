// Verification of drafted tokens (cera_hip_verify_draft_dev; contract in include/cera_hip.h).
//
// A row of logits is cut into chunks.  The first launch writes each chunk's maximum and sum of exponentials.  The second forms every
// sequence's decision from them (each workgroup for itself) and the chunk sums of the weights that the next token is drawn from; the
// workgroup of a sequence that is done last finds the chunk and in it the token.  Sums are in 64 bits: the draw compares a running sum
// over the vocabulary with a random number, and an error e in it moves each of some 10^5 borders by e.  Temperature 0 needs the maxima
// only.
//
// 64 sequences of 5 drafts of 32000 tokens: 24 us for the first launch, 90 MB at 3.8 TB/s, bound by the exponentials in 64 bits (without
// them, at temperature 0, 49 MB take 9.3 us, 5.3 TB/s), and 19 us for the second, bound by the latency of what follows from each other:
// sums, decision, weights, ticket, draw.  A launch for the draw of its own took 3 us more; fences in the place of the loads and stores
// that pass the XCD's L2 by 3 us, or 45 where every wavefront has one.
#include <cmath>

#include "paged.hip.h"

// A chunk is a wavefront's, 16 tokens a lane, so that no barrier is between its loads and its result; a workgroup has four.
static constexpr uint32_t VD_CHUNK = 1024, VD_THREADS = 256, VD_PER = VD_CHUNK / 64;
static constexpr uint32_t VD_MAX = 64;   // most drafted tokens

struct VdArgs {
    const float *target, *draft, *uniform;
    const int32_t* tokens;
    const uint32_t* n_draft;
    uint32_t* accepted;
    int32_t* out_tokens;
    uint64_t row_stride;
    uint32_t n_seqs, max_draft, vocab, n_chunks;
    double c;          // log2 e / temperature; 0: the largest logit
    double* sum;       // [row][chunk] sums of exp((z - max) / t); row: target rows, then draft rows
    float* top;        // [row][chunk] maxima; NaN where the chunk holds a NaN or +inf
    uint32_t* arg;     // [row][chunk] (t = 0) the maximum's index
    double* mass;      // [seq][chunk] sums of the weights of the next token
    uint32_t* done;    // [seq] workgroups that have their sums
};

// e^((z - top) / t) for z <= top, as 2^k 2^f with k + f = (z - top) c, c = log2 e / t, |f| <= 1/2, and 2^f by its Taylor series to
// f^11: 6e-15 of the value, and the difference's rounding, 2^-53 of the exponent; the largest itself is 1 at every t.  -inf gives 0.
constexpr double vd_taylor(int n) {   // ln(2)^n / n!
    double x = 1.0;
    for (int i = 1; i <= n; ++i) x *= 0.69314718055994530942 / i;
    return x;
}
__device__ __forceinline__ double vd_exp(float z, double c, double top) {
    const double t = (static_cast<double>(fmaxf(z, -3.402823466e38f)) - top) * c, k = __builtin_rint(t), f = t - k;
    double p = vd_taylor(11);
    p = fma(p, f, vd_taylor(10));
    p = fma(p, f, vd_taylor(9));
    p = fma(p, f, vd_taylor(8));
    p = fma(p, f, vd_taylor(7));
    p = fma(p, f, vd_taylor(6));
    p = fma(p, f, vd_taylor(5));
    p = fma(p, f, vd_taylor(4));
    p = fma(p, f, vd_taylor(3));
    p = fma(p, f, vd_taylor(2));
    p = fma(p, f, vd_taylor(1));
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(fmax(k, -3000.0)));
}

__device__ __forceinline__ const float* vd_row(const VdArgs& a, uint32_t row) {
    const uint32_t nt = a.n_seqs * (a.max_draft + 1);
    return row < nt ? a.target + row * a.row_stride : a.draft + (row - nt) * a.row_stride;
}

// a lane's token number e of a chunk: four in a row, 64 lanes side by side
typedef float vd_float4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ uint32_t vd_token(uint32_t chunk, uint32_t lane, uint32_t e) { return chunk * VD_CHUNK + 256 * (e >> 2) + 4 * lane + (e & 3); }

// grid = (rows, chunks / 4)
__global__ __launch_bounds__(VD_THREADS) void verify_rows_kernel(VdArgs a) {
    const uint32_t row = blockIdx.x, nt = a.n_seqs * (a.max_draft + 1), lane = threadIdx.x & 63, chunk = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t s = row < nt ? row / (a.max_draft + 1) : (row - nt) / a.max_draft, i = row < nt ? row % (a.max_draft + 1) : (row - nt) % a.max_draft;
    const uint32_t n = a.n_draft ? a.n_draft[s] : a.max_draft;
    if (row < nt && i == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.done[s] = 0;
    if (n > a.max_draft || i > n || (row >= nt && i == n) || chunk >= a.n_chunks) return;   // a row that is not asked for
    const float* const z = vd_row(a, row);
    float x[VD_PER], top = -__builtin_inff();
    bool bad = false;
    // all loads at once, four tokens each: a row need not be aligned to them
    if (chunk * VD_CHUNK + VD_CHUNK <= a.vocab) {
#pragma unroll
        for (uint32_t e = 0; e < VD_PER; e += 4) {
            const vd_float4 y = *reinterpret_cast<const vd_float4*>(z + vd_token(chunk, lane, e));
            x[e] = y.x; x[e + 1] = y.y; x[e + 2] = y.z; x[e + 3] = y.w;
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < VD_PER; ++e) {
            const uint32_t v = vd_token(chunk, lane, e);
            x[e] = z[min(v, a.vocab - 1)];
            x[e] = v < a.vocab ? x[e] : -__builtin_inff();
        }
    }
#pragma unroll
    for (uint32_t e = 0; e < VD_PER; ++e) {
        bad |= !(x[e] < __builtin_inff());
        top = fmaxf(top, x[e]);
    }
    const float mine = top;
    top = wave_max(top);
    bad = __any(bad);
    const uint64_t o = static_cast<uint64_t>(row) * a.n_chunks + chunk;
    if (lane == 0) a.top[o] = bad ? __builtin_nanf("") : top;
    if (a.c == 0.0) {
        uint32_t at = 0xFFFFFFFFu;   // the first that has the maximum
#pragma unroll
        for (uint32_t e = VD_PER; e-- > 0;) at = x[e] == top ? vd_token(chunk, lane, e) : at;
        at = mine == top && at < a.vocab ? at : 0xFFFFFFFFu;
        for (int d = 32; d; d >>= 1) at = min(at, static_cast<uint32_t>(__shfl_xor(at, d)));
        if (lane == 0) a.arg[o] = at;
    } else {
        double sum = 0.0;
        if (!bad && top > -__builtin_inff()) {
#pragma unroll
            for (uint32_t e = 0; e < VD_PER; ++e) sum += vd_exp(x[e], a.c, top);
            sum = wave_sum_f64(sum);
        }
        if (lane == 0) a.sum[o] = sum;
    }
}

struct VdRow { double top, sum; bool ok; };   // of a whole row
// 256 chunks' maxima and sums, four a lane
struct VdPart { float t[4]; double u[4]; };
__device__ __forceinline__ VdPart vd_part(const VdArgs& a, uint32_t row, uint32_t c0) {
    const uint64_t at = static_cast<uint64_t>(row) * a.n_chunks;
    VdPart x;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) x.t[e] = a.top[at + min(c0 + 64 * e + (threadIdx.x & 63), a.n_chunks - 1)];
    if (a.c != 0.0)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) x.u[e] = a.sum[at + min(c0 + 64 * e + (threadIdx.x & 63), a.n_chunks - 1)];
    return x;
}
// by one wavefront, every lane has it; x: the row's first chunks
__device__ __forceinline__ VdRow vd_whole(const VdArgs& a, uint32_t row, VdPart x) {
    float m = -__builtin_inff();
    double sum = 0.0;
    bool bad = false;
    for (uint32_t c0 = 0; c0 < a.n_chunks; c0 += 256) {
        if (c0) x = vd_part(a, row, c0);
        float top = -__builtin_inff();
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            bad |= x.t[e] != x.t[e];
            top = fmaxf(top, x.t[e]);
        }
        top = fmaxf(m, wave_max(top));
        if (a.c == 0.0 || !(top > -__builtin_inff())) {
            m = top;
            continue;
        }
        if (sum > 0.0) sum *= vd_exp(m, a.c, top);
        m = top;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (c0 + 64 * e + (threadIdx.x & 63) < a.n_chunks && x.t[e] > -__builtin_inff()) sum += x.u[e] * vd_exp(x.t[e], a.c, top);
    }
    VdRow r{m, 0.0, !__any(bad) && m > -__builtin_inff()};
    if (r.ok && a.c != 0.0) r.sum = wave_sum_f64(sum);
    return r;
}
__device__ __forceinline__ double vd_p(const VdArgs& a, const VdRow& r, float z) { return vd_exp(z, a.c, r.top) / r.sum; }

struct VdDecision {
    VdRow p, q;         // of the row that the next token is drawn from
    uint32_t n, j;      // drafts, accepted
    bool ok, rest;      // rest: drawn from max(p - q, 0)
    uint32_t token;     // the rejected one
};
struct VdShared {
    VdRow p[VD_MAX + 1], q[VD_MAX];
    uint8_t verdict[VD_MAX];   // 0: rejected, 1: accepted, 2: a row is out of order
};
// index of the row's maximum `top`, by one wavefront: in the first chunk that has it
__device__ __forceinline__ uint32_t vd_best(const VdArgs& a, uint32_t row, double top) {
    const uint64_t at = static_cast<uint64_t>(row) * a.n_chunks;
    uint32_t best = 0xFFFFFFFFu;
    for (uint32_t c = threadIdx.x & 63; c < a.n_chunks; c += 64)
        if (a.top[at + c] == static_cast<float>(top)) { best = a.arg[at + c]; break; }
    for (int x = 32; x; x >>= 1) best = min(best, static_cast<uint32_t>(__shfl_xor(best, x)));
    return best;
}
// by a workgroup, a wavefront per row at a time
__device__ __forceinline__ VdDecision vd_decide(const VdArgs& a, uint32_t s, VdShared& sh) {
    const uint32_t w = threadIdx.x >> 6, nt = a.n_seqs * (a.max_draft + 1);
    VdDecision d{};
    d.n = a.n_draft ? a.n_draft[s] : a.max_draft;
    if (d.n > a.max_draft) { d.n = 0; return d; }
    for (uint32_t i = w; i <= d.n; i += blockDim.x / 64) {
        const uint32_t row = s * (a.max_draft + 1) + i, drow = nt + s * a.max_draft + i;
        const uint32_t tok = i < d.n ? static_cast<uint32_t>(a.tokens[static_cast<uint64_t>(s) * a.max_draft + i]) : 0;
        const bool asked = i < d.n && tok < a.vocab && a.c != 0.0;
        const float z = asked ? a.target[row * a.row_stride + tok] : 0.0f, y = asked && a.draft ? a.draft[(drow - nt) * a.row_stride + tok] : 0.0f;
        const bool both = a.draft && i < d.n;
        const VdPart p0 = vd_part(a, row, 0), q0 = vd_part(a, both ? drow : row, 0);
        const VdRow p = vd_whole(a, row, p0);
        VdRow q{0.0, 1.0, true};
        if (both) q = vd_whole(a, drow, q0);
        uint8_t v = p.ok && q.ok ? 0 : 2;
        if (a.c == 0.0) {
            if (p.ok && tok == vd_best(a, row, p.top)) v = 1;
        } else if (v == 0 && asked) {
            const double qx = a.draft ? vd_p(a, q, y) : 1.0;
            if (static_cast<double>(a.uniform[static_cast<uint64_t>(s) * (a.max_draft + 1) + i]) * qx < vd_p(a, p, z)) v = 1;
        }
        if ((threadIdx.x & 63) == 0) {
            sh.p[i] = p;
            if (i < d.n) {
                sh.q[i] = q;
                sh.verdict[i] = v;
            }
        }
    }
    __syncthreads();
    while (d.j < d.n && sh.verdict[d.j] == 1) ++d.j;
    d.p = sh.p[d.j];
    d.rest = d.j < d.n;
    d.ok = d.p.ok && (!d.rest || sh.verdict[d.j] == 0);
    if (d.rest) {
        d.token = static_cast<uint32_t>(a.tokens[static_cast<uint64_t>(s) * a.max_draft + d.j]);
        d.q = sh.q[d.j];
    }
    return d;
}
// the weights of tokens v0 + step e as the next one
template <uint32_t N> __device__ __forceinline__ void vd_weights(const VdArgs& a, const VdDecision& d, const float* z, const float* y, uint32_t v0, uint32_t step, bool rest, double (&w)[N]) {
    float x[N], u[N];
#pragma unroll
    for (uint32_t e = 0; e < N; ++e) x[e] = z[min(v0 + e * step, a.vocab - 1)];
    if (y)
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) u[e] = y[min(v0 + e * step, a.vocab - 1)];
    const double inv_p = 1.0 / d.p.sum, inv_q = y ? 1.0 / d.q.sum : 0.0;
#pragma unroll
    for (uint32_t e = 0; e < N; ++e) {
        const uint32_t v = v0 + e * step;
        w[e] = vd_exp(x[e], a.c, d.p.top) * inv_p;
        if (rest) {
            const double q = y ? vd_exp(u[e], a.c, d.q.top) * inv_q : v == d.token ? 1.0 : 0.0;
            w[e] = fmax(w[e] - q, 0.0);
        }
        if (v >= a.vocab) w[e] = 0.0;
    }
}

// inclusive running sum over a wavefront's lanes
template <int CTRL, int ROWS> __device__ __forceinline__ double vd_from(double v) {   // another lane's value, 0 where there is none
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xF, true), hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xF, true);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double vd_scan(double v) {
    v += vd_from<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
    v += vd_from<0x112, 0xF>(v);
    v += vd_from<0x114, 0xF>(v);
    v += vd_from<0x118, 0xF>(v);
    v += vd_from<0x142, 0xA>(v);   // lanes 15 and 47 to the rows behind them
    v += vd_from<0x143, 0xC>(v);   // lane 31 to the upper half
    return v;
}

// grid = (chunks / 8, sequences), temperature 0: (1, sequences).  The weights' sums of eight chunks; the sequence's workgroup that is
// done last draws the token.
__global__ __launch_bounds__(2 * VD_THREADS) void verify_pick_kernel(VdArgs a) {
    __shared__ VdShared shd;
    __shared__ double wave_sum_of[8], sh_left;
    __shared__ uint32_t sh_chunk, sh_rest, first, last, ticket;
    const uint32_t s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const VdDecision d = vd_decide(a, s, shd);
    const uint32_t row = s * (a.max_draft + 1) + d.j;
    const float* const z = a.target + row * a.row_stride;
    const float* const y = a.draft && d.rest ? a.draft + (static_cast<uint64_t>(s) * a.max_draft + d.j) * a.row_stride : nullptr;
    double* const m = a.mass + static_cast<uint64_t>(s) * a.n_chunks;
    int32_t next = -1;
    if (d.ok && a.c == 0.0) {
        next = static_cast<int32_t>(vd_best(a, row, d.p.top));
    } else if (d.ok) {
        const uint32_t mine_chunk = blockIdx.x * 8 + w;
        if (mine_chunk < a.n_chunks) {
            double x[VD_PER], sum = 0.0;
            vd_weights(a, d, z, y, mine_chunk * VD_CHUNK + lane, 64, d.rest, x);
#pragma unroll
            for (uint32_t e = 0; e < VD_PER; ++e) sum += x[e];
            sum = wave_sum_f64(sum);
            if (lane == 0) __hip_atomic_store(&m[mine_chunk], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every wavefront's sums are out before the ticket is drawn
        __syncthreads();
        if (tid == 0) ticket = __hip_atomic_fetch_add(&a.done[s], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (ticket != gridDim.x - 1) return;
        if (w == 0) {
            auto sum = [&](auto x) {
                double t = 0.0;
                for (uint32_t c = lane; c < a.n_chunks; c += 64) t += x(c);
                return wave_sum_f64(t);
            };
            // as the other workgroups wrote them, whatever this XCD's L2 holds
            auto weight = [&](uint32_t c) { return __hip_atomic_load(&m[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
            double total = sum(weight);
            // where nothing is left of p - q (p = q but for roundings), p itself
            const bool rest = d.rest && total > 0.0;
            auto chunk = [&](uint32_t c) {
                if (rest || !d.rest) return weight(c);
                const uint64_t o = static_cast<uint64_t>(row) * a.n_chunks + c;
                return a.top[o] > -__builtin_inff() ? a.sum[o] * vd_p(a, d.p, a.top[o]) : 0.0;
            };
            if (rest != d.rest) total = sum(chunk);
            const double want = static_cast<double>(a.uniform[static_cast<uint64_t>(s) * (a.max_draft + 1) + a.max_draft]) * total;
            // the first chunk whose running sum is over what is wanted; should roundings leave none, the last with any weight
            double run = 0.0, left = 0.0;
            uint32_t in = 0;
            for (uint32_t b = 0; b < a.n_chunks; b += 64) {
                const double x = b + lane < a.n_chunks ? chunk(b + lane) : 0.0, inc = run + vd_scan(x);
                const uint64_t any = __ballot(x > 0.0), over = __ballot(x > 0.0 && inc > want);
                const int at = over ? __builtin_ctzll(over) : any ? 63 - __builtin_clzll(any) : -1;
                if (at >= 0) {
                    in = b + at;
                    left = want - __shfl(inc - x, at);
                }
                if (over) break;
                run = __shfl(inc, 63);
            }
            if (lane == 0) {
                sh_chunk = in;
                sh_left = left;
                sh_rest = rest;
                first = 0xFFFFFFFFu;
                last = 0;
            }
        }
        __syncthreads();
        const bool rest = sh_rest != 0;
        const uint32_t v0 = sh_chunk * VD_CHUNK;
        // a thread has two tokens in a row
        constexpr uint32_t N = VD_CHUNK / (2 * VD_THREADS);
        const uint32_t v1 = v0 + tid * N;
        double x[N], sum = 0.0;
        vd_weights(a, d, z, y, v1, 1, rest, x);
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) {
            sum += x[e];
            if (x[e] > 0.0) mine = v1 + e + 1;
        }
        const double inc = vd_scan(sum);
        if (lane == 63) wave_sum_of[w] = inc;
        if (mine) atomicMax(&last, mine);   // the chunk's last token with any weight
        __syncthreads();
        double run = inc - sum;
        for (uint32_t i = 0; i < w; ++i) run += wave_sum_of[i];
        // the first token whose running sum is over what is wanted
        uint32_t found = 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) {
            run += x[e];
            if (x[e] > 0.0 && run > sh_left) found = min(found, v1 + e);
        }
        if (found != 0xFFFFFFFFu) atomicMin(&first, found);
        __syncthreads();
        next = static_cast<int32_t>(first != 0xFFFFFFFFu ? first : last - 1);
    } else if (blockIdx.x) {
        return;
    }
    if (tid == 0) a.accepted[s] = d.j;
    for (uint32_t i = tid; i <= a.max_draft; i += 2 * VD_THREADS)
        a.out_tokens[static_cast<uint64_t>(s) * (a.max_draft + 1) + i] = i < d.j ? a.tokens[static_cast<uint64_t>(s) * a.max_draft + i] : i == d.j ? next : -1;
}

extern "C" cera_hip_status cera_hip_verify_draft_dev(cera_hip_ctx* ctx, const cera_hip_verify_draft* d) {
    if (!ctx) return CERA_HIP_ERR_ARGUMENT;
    std::lock_guard<std::recursive_mutex> op_lk(ctx->op_mu);
    const PagedCheck no = verify_check(d);
    if (no.msg) return cera_fail(ctx, no.st, no.msg);
    if (d->n_seqs == 0) return CERA_HIP_OK;
    const PagedDevice dev(ctx->device);
    HIP_TRY(ctx, dev.err);
    VdArgs a{};
    a.target = d->target; a.draft = d->temperature > 0 ? d->draft : nullptr; a.uniform = d->uniform; a.tokens = d->tokens; a.n_draft = d->n_draft;
    a.accepted = d->accepted; a.out_tokens = d->out_tokens;
    a.row_stride = d->row_stride ? d->row_stride : d->vocab;
    a.n_seqs = d->n_seqs; a.max_draft = d->max_draft; a.vocab = d->vocab;
    a.n_chunks = (d->vocab + VD_CHUNK - 1) / VD_CHUNK;
    a.c = d->temperature > 0 ? 1.4426950408889634074 / static_cast<double>(d->temperature) : 0.0;
    const uint32_t rows = d->n_seqs * (d->max_draft + 1) + (a.draft ? d->n_seqs * d->max_draft : 0);
    const uint64_t parts = static_cast<uint64_t>(rows) * a.n_chunks;
    void* ws;
    CERA_TRY(cera_scratch(ctx, 15, parts * 16 + static_cast<uint64_t>(d->n_seqs) * (a.n_chunks * 8 + 4), &ws));
    a.sum = static_cast<double*>(ws);
    a.mass = a.sum + parts;
    a.top = reinterpret_cast<float*>(a.mass + static_cast<uint64_t>(d->n_seqs) * a.n_chunks);
    a.arg = reinterpret_cast<uint32_t*>(a.top + parts);
    a.done = a.arg + parts;
    hipLaunchKernelGGL(verify_rows_kernel, dim3(rows, (a.n_chunks + 3) / 4), dim3(VD_THREADS), 0, ctx->stream, a);
    hipLaunchKernelGGL(verify_pick_kernel, dim3(a.c != 0.0 ? (a.n_chunks + 7) / 8 : 1, d->n_seqs), dim3(2 * VD_THREADS), 0, ctx->stream, a);
    HIP_TRY(ctx, hipGetLastError());
    return CERA_HIP_OK;
}
