// Verification of drafted tokens for gfx950: which of a sequence's drafted tokens the target model's distributions
// keep, and the token that follows them, from given random numbers.
//
// p_i = softmax(softcap(logits of row i) / T), q_i the draft's distribution (one-hot at the drafted token d_i where
// none is given).  Draft i is kept while u_i q_i(d_i) < p_i(d_i); at the first that is not, the next token is drawn
// from max(p_i - q_i, 0), and from p of the row behind the last draft if all are kept: the smallest index whose
// running sum passes u * (the whole sum).  Kept tokens then follow the target's distribution exactly.  With T = 0,
// p is one-hot at the largest logit (lowest index first).
//
// Exponentials and sums are 64 bits wide: a token is decided where a running sum over up to a few hundred thousand
// terms passes a border, and with fp32 sums (1e-7 of the whole) about one draw in a hundred would fall on another
// token than the definition's; with 64 bits it is one in 1e8.
#pragma once
#include "hipdec_common.h"

#define VF_THREADS 256
#define VF_PER 16                                            // logits per thread
#define VF_CHUNK (VF_THREADS * VF_PER)

struct VfStat { double sum; float top; uint32_t arg; };      // of one chunk of one row: max z, its first index, sum exp((z - max) / T)

struct VerifyArgs {
    const void *logits;
    long long row_stride, prob_stride;                       // elements between rows
    const int *drafts, *n_drafts;
    const float *probs, *u;
    int n_seqs, max_drafts, vocab, chunks;
    double inv_t;                                            // 0: greedy
    float softcap;
    VfStat *stats;                                           // [row][chunk]
    double *sums;                                            // [seq][chunk] of max(p - q, 0)
    uint32_t *tokens;
    int *accepted;
};

__device__ __forceinline__ int vf_drafts(const VerifyArgs &a, int s) {
    return a.n_drafts ? min(max(a.n_drafts[s], 0), a.max_drafts) : a.max_drafts;
}
template <bool B16> __device__ __forceinline__ float vf_logit(const VerifyArgs &a, long long row, int i) {
    const long long at = row * a.row_stride + i;
    const float x = B16 ? bf16_to_f32(((const uint16_t *)a.logits)[at]) : ((const float *)a.logits)[at];
    return x == x ? x : -INFINITY;                           // a NaN is no possible token
}
__device__ __forceinline__ double vf_capped(const VerifyArgs &a, float x) {
    return a.softcap > 0.0f ? (double)a.softcap * tanh((double)x / (double)a.softcap) : (double)x;
}
// exp((z - max z) / T); the maximum's own weight is 1 also where it is infinite, an impossible token's is 0
__device__ __forceinline__ double vf_weight(const VerifyArgs &a, float x, float top) {
    if (x == top) return x == -INFINITY ? 0.0 : 1.0;
    return x == -INFINITY ? 0.0 : exp((vf_capped(a, x) - vf_capped(a, top)) * a.inv_t);
}
__device__ __forceinline__ double vf_wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
    return v;
}

// The statistics of every row that a sequence's drafts reach, one workgroup per chunk.
template <bool B16> __global__ __launch_bounds__(VF_THREADS) void k_verify_stats(VerifyArgs a) {
    __shared__ float st[4];
    __shared__ uint32_t si[4];
    __shared__ double ss[4];
    const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks;
    const int s = row / (a.max_drafts + 1);
    if (row - s * (a.max_drafts + 1) > vf_drafts(a, s)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float x[VF_PER];
    float top = -INFINITY; uint32_t arg = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < VF_PER; ++i) {
        const int at = chunk * VF_CHUNK + i * VF_THREADS + tid;
        x[i] = at < a.vocab ? vf_logit<B16>(a, row, at) : -INFINITY;
        if (x[i] > top) { top = x[i]; arg = (uint32_t)at; }
    }
    wave_argbest(top, arg);
    if (lane == 0) { st[wave] = top; si[wave] = arg; }
    __syncthreads();
    top = st[0]; arg = si[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) if (better(st[w], si[w], top, arg)) { top = st[w]; arg = si[w]; }
    double sum = 0.0;
    if (a.inv_t > 0.0) {
#pragma unroll
        for (int i = 0; i < VF_PER; ++i) sum += vf_weight(a, x[i], top);
        sum = vf_wave_sum(sum);
        if (lane == 0) ss[wave] = sum;
        __syncthreads();
        sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
    }
    if (tid == 0) a.stats[(size_t)row * a.chunks + chunk] = VfStat{sum, top, arg};
}

// One row's maximum, its first index, and the sum over the whole row (a wave, every lane with the result).
__device__ __forceinline__ void vf_row(const VerifyArgs &a, long long row, float &top, uint32_t &arg, double &sum) {
    const VfStat *st = a.stats + (size_t)row * a.chunks;
    top = -INFINITY; arg = 0xffffffffu;
    for (int i = threadIdx.x & 63; i < a.chunks; i += WAVE)
        if (better(st[i].top, st[i].arg, top, arg)) { top = st[i].top; arg = st[i].arg; }
    wave_argbest(top, arg);
    sum = 0.0;
    if (a.inv_t > 0.0) {
        for (int i = threadIdx.x & 63; i < a.chunks; i += WAVE) sum += st[i].sum * vf_weight(a, st[i].top, top);
        sum = vf_wave_sum(sum);
    }
}

struct VfPlace { int kept, n; long long row; float top; uint32_t arg; double inv; };

// How many drafts of sequence s are kept, and the row the next token is drawn from (every thread with the result).
template <bool B16> __device__ __forceinline__ VfPlace vf_decide(const VerifyArgs &a, int s) {
    __shared__ int first;                                    // the first draft that is not kept
    const int n = vf_drafts(a, s), wave = threadIdx.x >> 6, K = a.max_drafts;
    if (threadIdx.x == 0) first = n;
    __syncthreads();
    for (int i = wave; i < n; i += VF_THREADS / WAVE) {
        const long long row = (long long)s * (K + 1) + i;
        float top; uint32_t arg; double sum;
        vf_row(a, row, top, arg, sum);
        const int d = a.drafts[(size_t)s * K + i];
        bool keep = false;
        if ((unsigned)d < (unsigned)a.vocab) {
            if (a.inv_t > 0.0) {
                const double p = sum > 0.0 ? vf_weight(a, vf_logit<B16>(a, row, d), top) / sum : 0.0;
                const double q = a.probs ? (double)a.probs[((long long)s * K + i) * a.prob_stride + d] : 1.0;
                keep = (double)a.u[(size_t)s * (K + 1) + i] * q < p;
            } else {
                keep = (uint32_t)d == arg;
            }
        }
        if (!keep && (threadIdx.x & 63) == 0) atomicMin(&first, i);
    }
    __syncthreads();
    VfPlace at;
    at.n = n; at.kept = first;
    at.row = (long long)s * (K + 1) + at.kept;
    double sum;
    vf_row(a, at.row, at.top, at.arg, sum);
    at.inv = sum > 0.0 ? 1.0 / sum : 0.0;
    return at;
}

// The weight of token i in what the next token is drawn from; `rest`: the part of the target the draft did not cover.
template <bool B16> __device__ __forceinline__ double vf_mass(const VerifyArgs &a, const VfPlace &at, int s, int i, bool rest) {
    const double p = vf_weight(a, vf_logit<B16>(a, at.row, i), at.top) * at.inv;
    if (!rest) return p;
    const long long d = (long long)s * a.max_drafts + at.kept;
    const double q = a.probs ? (double)a.probs[d * a.prob_stride + i] : a.drafts[d] == i ? 1.0 : 0.0;
    return fmax(p - q, 0.0);                                 // (a NaN in q leaves 0)
}

// Chunk sums of max(p - q, 0) at a sequence's first draft that is not kept.
template <bool B16> __global__ __launch_bounds__(VF_THREADS) void k_verify_sums(VerifyArgs a) {
    __shared__ double ss[4];
    const int chunk = blockIdx.x % a.chunks, s = blockIdx.x / a.chunks;
    const VfPlace at = vf_decide<B16>(a, s);
    if (at.kept == at.n || !(a.inv_t > 0.0)) return;         // the statistics hold the target's own sums
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < VF_PER; ++j) {
        const int i = chunk * VF_CHUNK + j * VF_THREADS + (int)threadIdx.x;
        if (i < a.vocab) sum += vf_mass<B16>(a, at, s, i, true);
    }
    sum = vf_wave_sum(sum);
    if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.sums[(size_t)s * a.chunks + chunk] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

// running sum over the lanes of a wave, the lane's own term included
__device__ __forceinline__ double vf_wave_scan(double v) {
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const double w = __shfl_up(v, o, WAVE);
        if ((int)(threadIdx.x & 63) >= o) v += w;
    }
    return v;
}

// The draw: the chunk where the running sum passes the border, then the token inside it.
template <bool B16> __global__ __launch_bounds__(VF_THREADS) void k_verify_draw(VerifyArgs a) {
    __shared__ double part[VF_THREADS / WAVE], left;
    __shared__ int chunk, from_rest, hit, last;
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, K = a.max_drafts;
    const VfPlace at = vf_decide<B16>(a, s);
    for (int i = tid; i <= K; i += VF_THREADS)
        if (i != at.kept) a.tokens[(size_t)s * (K + 1) + i] = i < at.kept ? (uint32_t)a.drafts[(size_t)s * K + i] : 0xffffffffu;
    if (tid == 0) a.accepted[s] = at.kept;
    uint32_t *out = a.tokens + (size_t)s * (K + 1) + at.kept;
    if (!(a.inv_t > 0.0) || at.inv == 0.0) {                 // greedy; or no possible token at all (arg is 0xffffffff then)
        if (tid == 0) *out = at.arg;
        return;
    }
    if (wave == 0) {                                         // at most 64 chunks: one a lane
        bool rest = at.kept < at.n;
        double mine = rest && lane < a.chunks ? a.sums[(size_t)s * a.chunks + lane] : 0.0;
        // all drafts kept, or the draft's distribution covers the target's everywhere: the target's own
        if (!rest || !__any(mine > 0.0)) {
            rest = false;
            const VfStat *st = a.stats + (size_t)at.row * a.chunks;
            mine = lane < a.chunks ? st[lane].sum * vf_weight(a, st[lane].top, at.top) * at.inv : 0.0;
        }
        const double run = vf_wave_scan(mine), border = (double)a.u[(size_t)s * (K + 1) + K] * __shfl(run, 63, WAVE);
        const uint64_t some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && run > border);
        // (no chunk passes the border where the random number is 1 or the sums round down: the last one with any weight)
        const int c = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some);
        const double before = __shfl_up(run, 1, WAVE);
        if (lane == c) { chunk = c; from_rest = rest; left = border - (lane ? before : 0.0); hit = 0x7fffffff; last = 0; }
    }
    __syncthreads();
    const int i0 = chunk * VF_CHUNK + tid * VF_PER;          // in index order
    double w[VF_PER], mine = 0.0;
#pragma unroll
    for (int j = 0; j < VF_PER; ++j) {
        w[j] = i0 + j < a.vocab ? vf_mass<B16>(a, at, s, i0 + j, from_rest) : 0.0;
        mine += w[j];
    }
    const double run = vf_wave_scan(mine);
    if (lane == 63) part[wave] = run;
    __syncthreads();
    const double before = __shfl_up(run, 1, WAVE);
    double r = lane ? before : 0.0;
#pragma unroll
    for (int k = 0; k < VF_THREADS / WAVE; ++k) if (k < wave) r += part[k];
    int mine_hit = 0x7fffffff, mine_last = -1;
#pragma unroll
    for (int j = 0; j < VF_PER; ++j) {
        r += w[j];
        if (w[j] > 0.0) { mine_last = i0 + j; if (r > left) mine_hit = min(mine_hit, i0 + j); }
    }
    if (mine_hit != 0x7fffffff) atomicMin(&hit, mine_hit);
    if (mine_last >= 0) atomicMax(&last, mine_last);
    __syncthreads();
    if (tid == 0) *out = (uint32_t)(hit != 0x7fffffff ? hit : last);
}
