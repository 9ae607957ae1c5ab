// Verification of drafted tokens (cera_hip_verify_draft_dev; contract in include/cera_hip.h).
//
// A row of logits is cut into chunks.  The first launch writes each chunk's maximum and sum of exponentials; the second forms every
// sequence's decision from them (each workgroup for itself) and the chunk sums of the weights that the next token is drawn from; the
// third finds the chunk and in it the token.  Sums are in 64 bits: the draw compares a running sum over the vocabulary with a
// random number, and an error e in it moves each of some 10^5 borders by e.  Temperature 0 needs the maxima only: two launches.
#include <cmath>

#include "paged.hip.h"

// A chunk is a wavefront's, 16 tokens a lane, so that no barrier is between its loads and its result; a workgroup has four.
static constexpr uint32_t VD_CHUNK = 1024, VD_THREADS = 256, VD_PER = VD_CHUNK / 64;
static constexpr uint32_t VD_MAX = 64;   // most drafted tokens

struct VdDecision;
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
    VdDecision* decided;   // [seq]
};

// e^((z - top) / t) for z <= top, as 2^k 2^f with k + f = z c - top c, c = log2 e / t, |f| <= 1/2, and 2^f by its Taylor series to
// f^11: 6e-15 of the value, and the rounding of z c, 1e-16 of the exponent.  -inf gives 0.
constexpr double vd_taylor(int n) {   // ln(2)^n / n!
    double x = 1.0;
    for (int i = 1; i <= n; ++i) x *= 0.69314718055994530942 / i;
    return x;
}
__device__ __forceinline__ double vd_exp(float z, double c, double top_c) {
    const double t = fma(static_cast<double>(fmaxf(z, -3.402823466e38f)), c, -top_c), k = __builtin_rint(t), f = t - k;
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

// grid = (rows, chunks / 4)
__global__ __launch_bounds__(VD_THREADS) void verify_rows_kernel(VdArgs a) {
    const uint32_t row = blockIdx.x, nt = a.n_seqs * (a.max_draft + 1), lane = threadIdx.x & 63, chunk = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t s = row < nt ? row / (a.max_draft + 1) : (row - nt) / a.max_draft, i = row < nt ? row % (a.max_draft + 1) : (row - nt) % a.max_draft;
    const uint32_t n = a.n_draft ? a.n_draft[s] : a.max_draft;
    if (n > a.max_draft || i > n || (row >= nt && i == n) || chunk >= a.n_chunks) return;   // a row that is not asked for
    const float* const z = vd_row(a, row);
    const uint32_t v0 = chunk * VD_CHUNK + lane;
    float x[VD_PER], top = -__builtin_inff();
    bool bad = false;
    // all loads at once: without branches
#pragma unroll
    for (uint32_t e = 0; e < VD_PER; ++e) x[e] = z[min(v0 + e * 64, a.vocab - 1)];
#pragma unroll
    for (uint32_t e = 0; e < VD_PER; ++e) {
        x[e] = v0 + e * 64 < a.vocab ? x[e] : -__builtin_inff();
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
        for (uint32_t e = VD_PER; e-- > 0;) at = x[e] == top ? v0 + e * 64 : at;
        at = mine == top && at < a.vocab ? at : 0xFFFFFFFFu;
        for (int d = 32; d; d >>= 1) at = min(at, static_cast<uint32_t>(__shfl_xor(at, d)));
        if (lane == 0) a.arg[o] = at;
    } else {
        double sum = 0.0;
        if (!bad && top > -__builtin_inff()) {
            const double top_c = top * a.c;
#pragma unroll
            for (uint32_t e = 0; e < VD_PER; ++e) sum += vd_exp(x[e], a.c, top_c);
            sum = wave_sum_f64(sum);
        }
        if (lane == 0) a.sum[o] = sum;
    }
}

struct VdRow { double top, sum; bool ok; };   // of a whole row
// by one wavefront, every lane has it
__device__ __forceinline__ VdRow vd_whole(const VdArgs& a, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63;
    const float* const top = a.top + static_cast<uint64_t>(row) * a.n_chunks;
    float m = -__builtin_inff();
    bool bad = false;
    for (uint32_t c = lane; c < a.n_chunks; c += 64) {
        const float t = top[c];
        bad |= t != t;
        m = fmaxf(m, t);
    }
    m = wave_max(m);
    VdRow r{m, 0.0, !__any(bad) && m > -__builtin_inff()};
    if (!r.ok || a.c == 0.0) return r;
    const double* const sum = a.sum + static_cast<uint64_t>(row) * a.n_chunks;
    double v = 0.0;
    for (uint32_t c = lane; c < a.n_chunks; c += 64)
        if (top[c] > -__builtin_inff()) v += sum[c] * vd_exp(top[c], a.c, r.top * a.c);
    r.sum = wave_sum_f64(v);
    return r;
}
__device__ __forceinline__ double vd_p(const VdArgs& a, const VdRow& r, float z) { return vd_exp(z, a.c, r.top * a.c) / r.sum; }

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
        const VdRow p = vd_whole(a, row);
        VdRow q{0.0, 1.0, true};
        if (a.draft && i < d.n) q = vd_whole(a, drow);
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
        w[e] = vd_exp(x[e], a.c, d.p.top * a.c) * inv_p;
        if (rest) {
            const double q = y ? vd_exp(u[e], a.c, d.q.top * a.c) * inv_q : v == d.token ? 1.0 : 0.0;
            w[e] = fmax(w[e] - q, 0.0);
        }
        if (v >= a.vocab) w[e] = 0.0;
    }
}

// grid = (chunks / 8, sequences)
__global__ __launch_bounds__(2 * VD_THREADS) void verify_mass_kernel(VdArgs a) {
    __shared__ VdShared shd;
    const uint32_t s = blockIdx.y, chunk = blockIdx.x * 8 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const VdDecision d = vd_decide(a, s, shd);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.decided[s] = d;
    if (!d.ok || chunk >= a.n_chunks) return;
    const float* const z = a.target + (static_cast<uint64_t>(s) * (a.max_draft + 1) + d.j) * a.row_stride;
    const float* const y = a.draft && d.rest ? a.draft + (static_cast<uint64_t>(s) * a.max_draft + d.j) * a.row_stride : nullptr;
    double x[VD_PER], sum = 0.0;
    vd_weights(a, d, z, y, chunk * VD_CHUNK + lane, 64, d.rest, x);
#pragma unroll
    for (uint32_t e = 0; e < VD_PER; ++e) sum += x[e];
    sum = wave_sum_f64(sum);
    if (lane == 0) a.mass[static_cast<uint64_t>(s) * a.n_chunks + chunk] = sum;
}

// inclusive running sum over a wavefront's lanes
__device__ __forceinline__ double vd_scan(double v) {
    const uint32_t lane = threadIdx.x & 63;
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d);
        if (lane >= static_cast<uint32_t>(d)) v += o;
    }
    return v;
}

// grid = sequences
__global__ __launch_bounds__(VD_THREADS) void verify_pick_kernel(VdArgs a) {
    __shared__ double wave_sum_of[4], sh_left;
    __shared__ VdShared shd;
    __shared__ uint32_t sh_chunk, sh_rest, first, last;
    const uint32_t s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const VdDecision d = a.c == 0.0 ? vd_decide(a, s, shd) : a.decided[s];
    const uint32_t row = s * (a.max_draft + 1) + d.j;
    int32_t next = -1;
    if (d.ok && a.c == 0.0) {
        next = static_cast<int32_t>(vd_best(a, row, d.p.top));
    } else if (d.ok) {
        if (w == 0) {
            const double* const m = a.mass + static_cast<uint64_t>(s) * a.n_chunks;
            auto sum = [&](auto x) {
                double t = 0.0;
                for (uint32_t c = lane; c < a.n_chunks; c += 64) t += x(c);
                return wave_sum_f64(t);
            };
            double total = sum([&](uint32_t c) { return m[c]; });
            // where nothing is left of p - q (p = q but for roundings), p itself
            const bool rest = d.rest && total > 0.0;
            auto chunk = [&](uint32_t c) {
                if (rest || !d.rest) return m[c];
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
        const float* const z = a.target + row * a.row_stride;
        const float* const y = a.draft && d.rest ? a.draft + (static_cast<uint64_t>(s) * a.max_draft + d.j) * a.row_stride : nullptr;
        const bool rest = sh_rest != 0;
        const uint32_t v0 = sh_chunk * VD_CHUNK;
        // a thread has four tokens in a row
        constexpr uint32_t N = VD_CHUNK / VD_THREADS;
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
    }
    if (tid == 0) a.accepted[s] = d.j;
    for (uint32_t i = tid; i <= a.max_draft; i += VD_THREADS)
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
    CERA_TRY(cera_scratch(ctx, 15, parts * 16 + static_cast<uint64_t>(d->n_seqs) * (a.n_chunks * 8 + sizeof(VdDecision)), &ws));
    a.sum = static_cast<double*>(ws);
    a.mass = a.sum + parts;
    a.decided = reinterpret_cast<VdDecision*>(a.mass + static_cast<uint64_t>(d->n_seqs) * a.n_chunks);
    a.top = reinterpret_cast<float*>(a.decided + d->n_seqs);
    a.arg = reinterpret_cast<uint32_t*>(a.top + parts);
    hipLaunchKernelGGL(verify_rows_kernel, dim3(rows, (a.n_chunks + 3) / 4), dim3(VD_THREADS), 0, ctx->stream, a);
    if (a.c != 0.0) hipLaunchKernelGGL(verify_mass_kernel, dim3((a.n_chunks + 7) / 8, d->n_seqs), dim3(2 * VD_THREADS), 0, ctx->stream, a);
    hipLaunchKernelGGL(verify_pick_kernel, dim3(d->n_seqs), dim3(VD_THREADS), 0, ctx->stream, a);
    HIP_TRY(ctx, hipGetLastError());
    return CERA_HIP_OK;
}
