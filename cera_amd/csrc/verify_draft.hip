// Verification of drafted tokens (cera_hip_verify_draft_dev; contract in include/cera_hip.h).
//
// A row of logits is cut into chunks.  The first launch writes each chunk's maximum and sum of exponentials; the second forms every
// sequence's decision from them (each workgroup for itself) and the chunk sums of the weights that the next token is drawn from; the
// third finds the chunk and in it the token.  Sums are in 64 bits: the draw compares a running sum over the vocabulary with a
// random number, and an error e in it moves each of some 10^5 borders by e.  Temperature 0 needs the maxima only: two launches.
#include <cmath>

#include "paged.hip.h"

static constexpr uint32_t VD_CHUNK = 4096, VD_THREADS = 256, VD_PER = VD_CHUNK / VD_THREADS;
static constexpr uint32_t VD_MAX = 64;   // most drafted tokens

struct VdArgs {
    const float *target, *draft, *uniform;
    const int32_t* tokens;
    const uint32_t* n_draft;
    uint32_t* accepted;
    int32_t* out_tokens;
    uint64_t row_stride;
    uint32_t n_seqs, max_draft, vocab, n_chunks;
    double inv_t;      // 0: the largest logit
    double* sum;       // [row][chunk] sums of exp((z - max) / t); row: target rows, then draft rows
    float* top;        // [row][chunk] maxima; NaN where the chunk holds a NaN or +inf
    uint32_t* arg;     // [row][chunk] (t = 0) the maximum's index
    double* mass;      // [seq][chunk] sums of the weights of the next token
};

__device__ __forceinline__ const float* vd_row(const VdArgs& a, uint32_t row) {
    const uint32_t nt = a.n_seqs * (a.max_draft + 1);
    return row < nt ? a.target + row * a.row_stride : a.draft + (row - nt) * a.row_stride;
}

// sum over a workgroup of 256 in a fixed order; the total in every thread
__device__ __forceinline__ double vd_block_sum(double v, double* sh) {
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// grid = (rows, chunks)
__global__ __launch_bounds__(VD_THREADS) void verify_rows_kernel(VdArgs a) {
    __shared__ double sh[4];
    __shared__ float shf[4];
    __shared__ uint32_t shi[4];
    const uint32_t row = blockIdx.x, nt = a.n_seqs * (a.max_draft + 1), tid = threadIdx.x;
    const uint32_t s = row < nt ? row / (a.max_draft + 1) : (row - nt) / a.max_draft, i = row < nt ? row % (a.max_draft + 1) : (row - nt) % a.max_draft;
    const uint32_t n = a.n_draft ? a.n_draft[s] : a.max_draft;
    if (n > a.max_draft || i > n || (row >= nt && i == n)) return;   // a row that is not asked for
    const float* const z = vd_row(a, row);
    const uint32_t v0 = blockIdx.y * VD_CHUNK;
    float x[VD_PER], top = -__builtin_inff();
    uint32_t at = 0xFFFFFFFFu;
    bool bad = false;
#pragma unroll
    for (uint32_t e = 0; e < VD_PER; ++e) {
        const uint32_t v = v0 + e * VD_THREADS + tid;
        x[e] = v < a.vocab ? z[v] : -__builtin_inff();
        bad |= !(x[e] < __builtin_inff());
        if (x[e] > top || (at == 0xFFFFFFFFu && v < a.vocab && x[e] == top)) { top = x[e]; at = v; }
    }
    const float mine = top;
    top = wave_max(top);
    if ((tid & 63) == 0) shf[tid >> 6] = top;
    bad = __syncthreads_or(bad);
    top = fmaxf(fmaxf(shf[0], shf[1]), fmaxf(shf[2], shf[3]));
    const uint64_t o = static_cast<uint64_t>(row) * a.n_chunks + blockIdx.y;
    if (a.inv_t == 0.0) {
        uint32_t best = mine == top ? at : 0xFFFFFFFFu;
        for (int d = 32; d; d >>= 1) best = min(best, static_cast<uint32_t>(__shfl_xor(best, d)));
        if ((tid & 63) == 0) shi[tid >> 6] = best;
        __syncthreads();
        if (tid == 0) a.arg[o] = min(min(shi[0], shi[1]), min(shi[2], shi[3]));
    } else if (!bad && top > -__builtin_inff()) {
        double sum = 0.0;
#pragma unroll
        for (uint32_t e = 0; e < VD_PER; ++e) sum += exp((static_cast<double>(x[e]) - top) * a.inv_t);
        sum = vd_block_sum(sum, sh);
        if (tid == 0) a.sum[o] = sum;
    } else if (tid == 0) {
        a.sum[o] = 0.0;
    }
    if (tid == 0) a.top[o] = bad ? __builtin_nanf("") : top;
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
    if (!r.ok || a.inv_t == 0.0) return r;
    const double* const sum = a.sum + static_cast<uint64_t>(row) * a.n_chunks;
    double v = 0.0;
    for (uint32_t c = lane; c < a.n_chunks; c += 64)
        if (top[c] > -__builtin_inff()) v += sum[c] * exp((static_cast<double>(top[c]) - r.top) * a.inv_t);
    r.sum = wave_sum_f64(v);
    return r;
}
__device__ __forceinline__ double vd_p(const VdArgs& a, const VdRow& r, float z) { return exp((static_cast<double>(z) - r.top) * a.inv_t) / r.sum; }

struct VdDecision {
    VdRow p, q;         // of the row that the next token is drawn from
    uint32_t n, j;      // drafts, accepted
    bool ok, rest;      // rest: drawn from max(p - q, 0)
    uint32_t token;     // the rejected one
};
// by a workgroup of four wavefronts
__device__ __forceinline__ VdDecision vd_decide(const VdArgs& a, uint32_t s, uint8_t* verdict) {
    const uint32_t w = threadIdx.x >> 6, nt = a.n_seqs * (a.max_draft + 1);
    VdDecision d{};
    d.n = a.n_draft ? a.n_draft[s] : a.max_draft;
    if (d.n > a.max_draft) { d.n = 0; return d; }
    for (uint32_t i = w; i < d.n; i += 4) {   // 0: rejected, 1: accepted, 2: a row is out of order
        const uint32_t tok = static_cast<uint32_t>(a.tokens[static_cast<uint64_t>(s) * a.max_draft + i]), row = s * (a.max_draft + 1) + i, drow = nt + s * a.max_draft + i;
        const VdRow p = vd_whole(a, row);
        uint8_t v = p.ok ? 0 : 2;
        if (a.inv_t == 0.0) {
            uint32_t best = 0xFFFFFFFFu;   // the row's maximum is in the first chunk that has it
            for (uint32_t c = threadIdx.x & 63; c < a.n_chunks; c += 64)
                if (a.top[static_cast<uint64_t>(row) * a.n_chunks + c] == static_cast<float>(p.top)) { best = a.arg[static_cast<uint64_t>(row) * a.n_chunks + c]; break; }
            for (int x = 32; x; x >>= 1) best = min(best, static_cast<uint32_t>(__shfl_xor(best, x)));
            if (p.ok && tok == best) v = 1;
        } else {
            VdRow q{0.0, 1.0, true};
            if (a.draft) q = vd_whole(a, drow);
            if (!q.ok) v = 2;
            if (v == 0 && tok < a.vocab) {
                const double qx = a.draft ? vd_p(a, q, a.draft[(drow - nt) * a.row_stride + tok]) : 1.0;
                if (static_cast<double>(a.uniform[static_cast<uint64_t>(s) * (a.max_draft + 1) + i]) * qx < vd_p(a, p, a.target[row * a.row_stride + tok])) v = 1;
            }
        }
        if ((threadIdx.x & 63) == 0) verdict[i] = v;
    }
    __syncthreads();
    while (d.j < d.n && verdict[d.j] == 1) ++d.j;
    d.p = vd_whole(a, s * (a.max_draft + 1) + d.j);
    d.ok = d.p.ok && (d.j == d.n || verdict[d.j] == 0);
    d.rest = d.j < d.n;
    if (d.rest) {
        d.token = static_cast<uint32_t>(a.tokens[static_cast<uint64_t>(s) * a.max_draft + d.j]);
        if (a.draft && a.inv_t != 0.0) d.q = vd_whole(a, nt + s * a.max_draft + d.j);
    }
    return d;
}
// the weight of token v as the next one
__device__ __forceinline__ double vd_weight(const VdArgs& a, const VdDecision& d, const float* z, const float* y, uint32_t v, bool rest) {
    const double p = vd_p(a, d.p, z[v]);
    if (!rest) return p;
    const double q = y ? vd_p(a, d.q, y[v]) : v == d.token ? 1.0 : 0.0;
    return p > q ? p - q : 0.0;
}

// grid = (chunks, sequences)
__global__ __launch_bounds__(VD_THREADS) void verify_mass_kernel(VdArgs a) {
    __shared__ double sh[4];
    __shared__ uint8_t verdict[VD_MAX];
    const uint32_t s = blockIdx.y;
    const VdDecision d = vd_decide(a, s, verdict);
    double sum = 0.0;
    if (d.ok) {
        const float* const z = a.target + (static_cast<uint64_t>(s) * (a.max_draft + 1) + d.j) * a.row_stride;
        const float* const y = a.draft ? a.draft + (static_cast<uint64_t>(s) * a.max_draft + d.j) * a.row_stride : nullptr;
        const uint32_t v0 = blockIdx.x * VD_CHUNK + threadIdx.x * VD_PER, v1 = min(v0 + VD_PER, a.vocab);
        for (uint32_t v = v0; v < v1; ++v) sum += vd_weight(a, d, z, y, v, d.rest);
    }
    sum = vd_block_sum(sum, sh);
    if (threadIdx.x == 0) a.mass[static_cast<uint64_t>(s) * a.n_chunks + blockIdx.x] = sum;
}

// grid = sequences
__global__ __launch_bounds__(VD_THREADS) void verify_pick_kernel(VdArgs a) {
    __shared__ double part[VD_THREADS], sh_left;
    __shared__ uint8_t verdict[VD_MAX];
    __shared__ uint32_t sh_chunk, sh_rest, sh_token;
    const uint32_t s = blockIdx.x, tid = threadIdx.x;
    const VdDecision d = vd_decide(a, s, verdict);
    const uint32_t row = s * (a.max_draft + 1) + d.j;
    int32_t next = -1;
    if (d.ok && a.inv_t == 0.0) {
        if (tid == 0)
            for (uint32_t c = 0; c < a.n_chunks; ++c)
                if (a.top[static_cast<uint64_t>(row) * a.n_chunks + c] == static_cast<float>(d.p.top)) { next = static_cast<int32_t>(a.arg[static_cast<uint64_t>(row) * a.n_chunks + c]); break; }
    } else if (d.ok) {
        if (tid == 0) {
            // where nothing is left of p - q (p = q but for roundings), p itself
            const double* m = a.mass + static_cast<uint64_t>(s) * a.n_chunks;
            double total = 0.0;
            for (uint32_t c = 0; c < a.n_chunks; ++c) total += m[c];
            const bool rest = d.rest && total > 0.0;
            auto chunk = [&](uint32_t c) {
                if (rest || !d.rest) return m[c];
                const uint64_t o = static_cast<uint64_t>(row) * a.n_chunks + c;
                return a.top[o] > -__builtin_inff() ? a.sum[o] * exp((static_cast<double>(a.top[o]) - d.p.top) * a.inv_t) / d.p.sum : 0.0;
            };
            if (rest != d.rest) {
                total = 0.0;
                for (uint32_t c = 0; c < a.n_chunks; ++c) total += chunk(c);
            }
            const double want = static_cast<double>(a.uniform[static_cast<uint64_t>(s) * (a.max_draft + 1) + a.max_draft]) * total;
            double run = 0.0, left = 0.0;
            uint32_t in = 0;
            for (uint32_t c = 0; c < a.n_chunks; ++c) {
                const double x = chunk(c);
                if (x > 0.0) { in = c; left = want - run; }   // the last chunk with any weight, should roundings leave none
                run += x;
                if (x > 0.0 && run > want) break;
            }
            sh_chunk = in;
            sh_left = left;
            sh_rest = rest;
            sh_token = 0;
        }
        __syncthreads();
        const float* const z = a.target + row * a.row_stride;
        const float* const y = a.draft ? a.draft + (static_cast<uint64_t>(s) * a.max_draft + d.j) * a.row_stride : nullptr;
        const bool rest = sh_rest != 0;
        const uint32_t v0 = sh_chunk * VD_CHUNK + tid * VD_PER, v1 = min(v0 + VD_PER, a.vocab);
        double sum = 0.0;
        uint32_t last = 0;
        for (uint32_t v = v0; v < v1; ++v) {
            const double x = vd_weight(a, d, z, y, v, rest);
            sum += x;
            if (x > 0.0) last = v + 1;
        }
        part[tid] = sum;
        if (last) atomicMax(&sh_token, last);   // the chunk's last token with any weight
        __syncthreads();
        double before = 0.0;
        for (uint32_t i = 0; i < tid; ++i) before += part[i];
        const bool here = before + sum > sh_left && !(before > sh_left);
        // the first token whose running sum is over what is wanted
        uint32_t found = 0xFFFFFFFFu;
        if (here) {
            double run = before;
            for (uint32_t v = v0; v < v1 && found == 0xFFFFFFFFu; ++v) {
                const double x = vd_weight(a, d, z, y, v, rest);
                run += x;
                if (x > 0.0 && run > sh_left) found = v;
            }
        }
        __shared__ uint32_t first;
        if (tid == 0) first = 0xFFFFFFFFu;
        __syncthreads();
        if (found != 0xFFFFFFFFu) atomicMin(&first, found);
        __syncthreads();
        next = static_cast<int32_t>(first != 0xFFFFFFFFu ? first : sh_token - 1);
    }
    if (tid == 0) a.accepted[s] = d.j;
    for (uint32_t i = tid; i <= a.max_draft; i += VD_THREADS) {
        int32_t v = -1;
        if (i < d.j) v = a.tokens[static_cast<uint64_t>(s) * a.max_draft + i];
        else if (i == d.j && tid == 0) v = next;
        if (!(i == d.j && tid != 0)) a.out_tokens[static_cast<uint64_t>(s) * (a.max_draft + 1) + i] = v;
    }
    if (tid == 0 && d.j) a.out_tokens[static_cast<uint64_t>(s) * (a.max_draft + 1) + d.j] = next;
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
    a.inv_t = d->temperature > 0 ? 1.0 / static_cast<double>(d->temperature) : 0.0;
    const uint32_t rows = d->n_seqs * (d->max_draft + 1) + (a.draft ? d->n_seqs * d->max_draft : 0);
    const uint64_t parts = static_cast<uint64_t>(rows) * a.n_chunks;
    void* ws;
    CERA_TRY(cera_scratch(ctx, 15, parts * 16 + static_cast<uint64_t>(d->n_seqs) * a.n_chunks * 8, &ws));
    a.sum = static_cast<double*>(ws);
    a.mass = a.sum + parts;
    a.top = reinterpret_cast<float*>(a.mass + static_cast<uint64_t>(d->n_seqs) * a.n_chunks);
    a.arg = reinterpret_cast<uint32_t*>(a.top + parts);
    hipLaunchKernelGGL(verify_rows_kernel, dim3(rows, a.n_chunks), dim3(VD_THREADS), 0, ctx->stream, a);
    if (a.inv_t != 0.0) hipLaunchKernelGGL(verify_mass_kernel, dim3(a.n_chunks, d->n_seqs), dim3(VD_THREADS), 0, ctx->stream, a);
    hipLaunchKernelGGL(verify_pick_kernel, dim3(d->n_seqs), dim3(VD_THREADS), 0, ctx->stream, a);
    HIP_TRY(ctx, hipGetLastError());
    return CERA_HIP_OK;
}
