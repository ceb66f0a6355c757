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
// token than the definition's; with 64 bits it is one in 1e8 (with a soft cap, whose 1e-14 a temperature divides, at most one in 1e7).
// Measured (MI355X): one sequence of four looked-up drafts over 32768 tokens 10.4 us of kernels; 32 of up to 7 drafts with
// probabilities 17.7 us; 64 of up to 5 over 131071 bf16 logits with a soft cap 82 us, where a vector instruction issues in
// 98 % of the statistics' cycles (60 per logit, 38 of them 64 bits wide).  At temperature 0, two launches, 5.8 / 9.9 / 20.7 us.
#pragma once
#include "hipdec_wave64.h"

// A chunk is what one wave takes: 64 * PER logits.  No barrier stands between a chunk's loads and its result, so the waves of
// a CU drift apart and one's loads run under another's arithmetic (with a workgroup to a chunk and two barriers in it
// 32 requests of 7 drafts took 30.2 us, so 24.5; the draw of one token 7.4 us, so 3.0).
#define VF_STATS 256                                         // threads of the kernels: statistics,
#define VF_DECIDE 512                                        // decision and rest
#define VF_MAX_CHUNKS 256                                    // of a row: four a lane

struct VfStat { double sum; float top; uint32_t arg; };      // of one chunk of one row: max logit, the sum of weights (T > 0) or the maximum's first index (T = 0; else 0xffffffff)
struct VfPlace { double inv; float top; int kept; };         // where a sequence's next token is drawn: 1 / the row's sum (0: nothing to draw), its maximum

struct VerifyArgs {
    const void *logits;
    long long row_stride, prob_stride;                       // elements between rows
    const int *drafts, *n_drafts;
    const float *probs, *u;
    int n_seqs, max_drafts, vocab, chunks;
    double k;                                                // log2(e) / T; 0: greedy
    double cap, cap_k;                                       // soft cap (0: none) and 2 log2(e) / cap
    VfStat *stats;                                           // [row][chunk]
    double *sums;                                            // [seq][chunk] of max(p - q, 0)
    VfPlace *places;                                         // [seq]
    uint32_t *tokens;
    int *accepted;
};

__device__ __forceinline__ int vf_drafts(const VerifyArgs &a, int s) {
    return a.n_drafts ? min(max(a.n_drafts[s], 0), a.max_drafts) : a.max_drafts;
}
// stored logit as a number: a NaN is no possible token; infinite ones share the whole, and at temperature 0 are the largest
__device__ __forceinline__ float vf_most(const VerifyArgs &a) { return a.k > 0.0 ? 3.4028235e38f : INFINITY; }
template <bool B16> __device__ __forceinline__ float vf_number(uint32_t raw, float most) {
    const float x = B16 ? bf16_to_f32(raw) : __uint_as_float(raw);
    return fminf(x == x ? x : -INFINITY, most);
}
template <bool B16> __device__ __forceinline__ uint32_t vf_raw(const void *row, int i) {
    return B16 ? ((const uint16_t *)row)[i] : ((const uint32_t *)row)[i];
}
template <bool B16> __device__ __forceinline__ const void *vf_row_of(const VerifyArgs &a, long long row) {
    return B16 ? (const void *)((const uint16_t *)a.logits + row * a.row_stride) : (const void *)((const float *)a.logits + row * a.row_stride);
}
template <bool B16> __device__ __forceinline__ float vf_logit(const VerifyArgs &a, long long row, int i) {
    return vf_number<B16>(vf_raw<B16>(vf_row_of<B16>(a, row), i), vf_most(a));
}
// PER logits of a lane: those of its wave's chunk 64 apart, or neighbours; -inf behind the vocabulary.  (All of them are
// asked for before the first is looked at; the chunk is the same for the whole wave, and so is the question whether it
// ends inside the vocabulary: with the check
// around every load they went one after the other: 256 rows of 131071 took 79 us, so 50.)
template <bool B16, int PER, bool NEAR> __device__ __forceinline__ void vf_logits(const VerifyArgs &a, long long row, int chunk, float *x) {
    const int first = chunk * PER * WAVE, lane = threadIdx.x & 63, step = NEAR ? 1 : WAVE, mine = first + (NEAR ? lane * PER : lane);
    const void *p = vf_row_of<B16>(a, row);
    const float most = vf_most(a);
    uint32_t raw[PER];
    if (first + PER * WAVE <= a.vocab) {
#pragma unroll
        for (int i = 0; i < PER; ++i) raw[i] = vf_raw<B16>(p, mine + i * step);
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = vf_number<B16>(raw[i], most);
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) raw[i] = vf_raw<B16>(p, min(mine + i * step, a.vocab - 1));
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = mine + i * step < a.vocab ? vf_number<B16>(raw[i], most) : -INFINITY;
    }
}
// a probability of the draft's, or a random number, as it counts: a negative one is 0 (a token that the target cannot give, or that
// lies behind the vocabulary, would have a rest otherwise, and a draft that it cannot give would be kept); a NaN stays one
__device__ __forceinline__ float vf_from0(float x) { return x < 0.0f ? 0.0f : x; }
// the draft's probabilities of the same tokens
template <int PER, bool NEAR> __device__ __forceinline__ void vf_guess(const VerifyArgs &a, long long draft, int chunk, float *q) {
    const int lane = threadIdx.x & 63, step = NEAR ? 1 : WAVE, mine = chunk * PER * WAVE + (NEAR ? lane * PER : lane);
    if (a.probs) {
        const float *p = a.probs + draft * a.prob_stride;
#pragma unroll
        for (int i = 0; i < PER; ++i) q[i] = vf_from0(p[min(mine + i * step, a.vocab - 1)]);   // (behind the vocabulary the target has nothing)
    } else {
        const int d = a.drafts[draft];
#pragma unroll
        for (int i = 0; i < PER; ++i) q[i] = d == mine + i * step ? 1.0f : 0.0f;
    }
}
// this thread's wave, known to be one number for the whole wave
__device__ __forceinline__ int vf_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// 2^y = 2^n 2^f for -1021 <= y <= 1022 with n = y to the nearest, read off the last bits of y + 1.5 * 2^52; f = y - n.
__device__ __forceinline__ double vf_parts(double y, uint32_t &n) {
    const double whole = 6755399441055744.0, t = y + whole;
    n = (uint32_t)__double2loint(t);
    return y - (t - whole);
}
// (2^f - 1) / f for |f| <= 1/2: the polynomial of degree 9 through its values at the ten Chebyshev nodes (worked out in 60 digits),
// 1.5e-15 of it, so that 2^f near 1 and the soft cap of small logits are right relative to themselves.  (Degree 8 leaves 9e-14: with
// it the soft cap was off by 2e-13 of itself, and each of up to 262144 borders of a draw by as much of the whole.  The kernels' time
// on large calls is their instructions, most of them these.)
__device__ __forceinline__ double vf_slope(double f) {
    double p = 7.070977866508138e-09;
    p = fma(p, f, 1.0205905413765595e-07);
    p = fma(p, f, 1.3215451633221434e-06);
    p = fma(p, f, 1.5252672924850737e-05);
    p = fma(p, f, 1.5403530424776529e-04);
    p = fma(p, f, 1.3333558200794592e-03);
    p = fma(p, f, 9.618129107618665e-03);
    p = fma(p, f, 5.550410866465167e-02);
    p = fma(p, f, 2.4022650695910075e-01);
    return fma(p, f, 6.931471805599462e-01);
}
__device__ __forceinline__ double vf_exp2(double y) {
    uint32_t n;
    const double f = vf_parts(y, n), p = fma(vf_slope(f), f, 1.0);
    return __hiloint2double(__double2hiint(p) + (int)(n << 20), __double2loint(p));
}
// softcap(x) / cap = tanh(x / cap) = E / (E + 2) with E = e^(2 x / cap) - 1 = 2^n (2^f - 1) + (2^n - 1): nothing cancels, so
// it is right to 1e-14 of itself, at a cap far above the logits too.  Past 2^+-100 it is +-1.  (The plain form without cap.)
template <bool CAP> __device__ __forceinline__ double vf_capped(const VerifyArgs &a, float x) {
    // (the last product stays a number of its own: fused into the difference of two caps, as this compiler does where it may, a
    // logit's difference to itself would be that product's rounding, not 0, and a tiny temperature makes that the whole weight)
#pragma clang fp contract(off)
    if (!CAP) return (double)x;
    const float far = 34.657359f * (float)a.cap;             // 100 of 2 log2(e) / cap
    uint32_t n;
    const double f = vf_parts((double)fminf(fmaxf(x, -far), far) * a.cap_k, n);
    const double two_n = __hiloint2double((int)(0x3ff00000u + (n << 20)), 0);
    const double e = fma(vf_slope(f) * f, two_n, two_n - 1.0), d = e + 2.0;
    double r = __builtin_amdgcn_rcp(d);                      // good to 2^-24; Newton's step squares that
    r = fma(r, fma(-d, r, 1.0), r);
    return e * r;
}
// exp((z - max z) / T) with ztop = the row's maximum, as vf_capped has it; impossible tokens, and what lies 2^1021 below the maximum, are 0.
// EXACT_ZERO: whether the difference of 0 and 2^-1021 counts (it does where a token is picked, not in a row's sum).
template <bool CAP, bool EXACT_ZERO> __device__ __forceinline__ double vf_weight(const VerifyArgs &a, float x, double ztop) {
    double y = fmax((vf_capped<CAP>(a, x) - ztop) * (CAP ? a.cap * a.k : a.k), -1021.0);   // (a row of nothing else: -inf + inf, a NaN, counts as -1021)
    // (the cap's last bits can put a logit that it saturates above the maximum's, which a small temperature multiplies without limit)
    if (CAP) y = fmin(y, 0.0);
    const double w = vf_exp2(y);
    if (CAP && x == -INFINITY) return 0.0;
    return EXACT_ZERO ? y > -1021.0 ? w : 0.0 : w;
}
// max(p - q, 0), a NaN in q leaves 0.  (One fused operation wherever it is taken: a chunk whose sum is above 0 holds a
// token that is.)
__device__ __forceinline__ double vf_rest(double weight, double inv, float q) { return fmax(fma(weight, inv, -(double)q), 0.0); }
__device__ __forceinline__ double vf_wave_sum(double v) { return wave_read_f64(wave_scan_f64(v), 63); }

// The statistics of every row that a sequence's drafts reach, a wave per chunk.
template <bool B16, bool CAP, int PER> __global__ __launch_bounds__(VF_STATS) void k_verify_stats(VerifyArgs a) {
    const int per_row = (a.chunks + VF_STATS / WAVE - 1) / (VF_STATS / WAVE);
    const int row = blockIdx.x / per_row, chunk = (int)(blockIdx.x % per_row) * (VF_STATS / WAVE) + vf_wave();
    const int s = row / (a.max_drafts + 1), lane = threadIdx.x & 63;
    if (chunk >= a.chunks) return;
    float x[PER];
    const bool unused = row - s * (a.max_drafts + 1) > vf_drafts(a, s);
    if (PER > 4 && unused) return;                           // (few logits are asked for without waiting for the draft's length)
    vf_logits<B16, PER, false>(a, row, chunk, x);
    if (unused) return;
    float top = x[0];
    uint32_t arg = 0xffffffffu;
    double sum = 0.0;
    if (a.k > 0.0) {
#pragma unroll
        for (int i = 1; i < PER; ++i) top = fmaxf(top, x[i]);
        top = wave_max_dpp(top);
        const double ztop = vf_capped<CAP>(a, top);
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += vf_weight<CAP, false>(a, x[i], ztop);
        sum = top == -INFINITY ? 0.0 : vf_wave_sum(sum);
    } else {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (x[i] > top) { top = x[i]; arg = (uint32_t)((chunk * PER + i) * WAVE + lane); }
        wave_argbest(top, arg);
    }
    if (lane == 0) a.stats[(size_t)row * a.chunks + chunk] = VfStat{sum, top, arg};
}

// The decision, by every workgroup of the sequence for itself (a wave per row, all of them at once up to seven drafts), then
// each wave's chunk of max(p - q, 0) where a draft was not kept.  The sequence's first workgroup writes what is known
// by now: the kept drafts and, where T = 0 or nothing is possible, the next token.
template <bool B16, bool CAP, int PER> __global__ __launch_bounds__(VF_DECIDE) void k_verify_decide(VerifyArgs a) {
    __shared__ double s_inv[256];                            // of each row (max_drafts <= 255)
    __shared__ float s_top[256];
    __shared__ uint32_t s_arg[256];
    __shared__ int s_kept;
    const int tid = threadIdx.x, lane = tid & 63, wave = vf_wave(), K = a.max_drafts;
    const int parts = a.k > 0.0 ? (a.chunks + VF_DECIDE / WAVE - 1) / (VF_DECIDE / WAVE) : 1;
    const int s = blockIdx.x / parts, part = blockIdx.x % parts;
    const int n = vf_drafts(a, s);
    if (tid == 0) s_kept = n;
    __syncthreads();
    for (int i = wave; i <= n; i += VF_DECIDE / WAVE) {
        const long long row = (long long)s * (K + 1) + i;
        const int d = i < n ? a.drafts[(size_t)s * K + i] : -1;
        const VfStat *st = a.stats + (size_t)row * a.chunks;
        float top = -INFINITY; uint32_t arg = 0xffffffffu;
        VfStat mine[VF_MAX_CHUNKS / WAVE];
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[j] = st[min(lane + 64 * j, a.chunks - 1)];
        const bool real = (unsigned)d < (unsigned)a.vocab;
        const int at = real ? d : 0;
        const float logit = vf_logit<B16>(a, row, at), x = real ? logit : -INFINITY;
        const bool sampled = a.k > 0.0 && i < n;
        const double q = sampled && a.probs ? (double)vf_from0(a.probs[((long long)s * K + i) * a.prob_stride + at]) : 1.0;
        const double u = sampled ? (double)vf_from0(a.u[(size_t)s * (K + 1) + i]) : 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (lane + 64 * j >= a.chunks) mine[j] = VfStat{0.0, -INFINITY, 0xffffffffu};
#pragma unroll
        for (int j = 0; j < 4; ++j) if (better(mine[j].top, mine[j].arg, top, arg)) { top = mine[j].top; arg = mine[j].arg; }
        double sum = 0.0, ztop = 0.0;
        if (a.k > 0.0) {
            top = wave_max_dpp(top);
            ztop = vf_capped<CAP>(a, top);
#pragma unroll
            for (int j = 0; j < 4; ++j) if (64 * j < a.chunks) sum += mine[j].sum * vf_weight<CAP, true>(a, mine[j].top, ztop);
            sum = vf_wave_sum(sum);
        } else {
            wave_argbest(top, arg);
        }
        const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
        const bool keep = real && (a.k > 0.0 ? u * q < vf_weight<CAP, true>(a, x, ztop) * inv : (uint32_t)d == arg);
        if (lane == 0) {
            s_inv[i] = inv; s_top[i] = top; s_arg[i] = arg;
            if (i < n && !keep) atomicMin(&s_kept, i);
        }
    }
    __syncthreads();
    const int kept = s_kept;
    const double inv = s_inv[kept];
    const float top = s_top[kept];
    if (part == 0) {
        uint32_t *out = a.tokens + (size_t)s * (K + 1);
        const bool known = !(a.k > 0.0) || inv == 0.0;       // (the index of a row without a possible token is 0xffffffff)
        for (int i = tid; i <= K; i += VF_DECIDE)
            if (i != kept || known) out[i] = i < kept ? (uint32_t)a.drafts[(size_t)s * K + i] : i == kept ? s_arg[kept] : 0xffffffffu;
        if (tid == 0) { a.accepted[s] = kept; a.places[s] = VfPlace{inv, top, kept}; }
    }
    if (kept == n || !(a.k > 0.0)) return;                   // behind the last draft the statistics hold the sums
    const long long row = (long long)s * (K + 1) + kept, dr = (long long)s * K + kept;
    const double ztop = vf_capped<CAP>(a, top);
    const int chunk = part * (VF_DECIDE / WAVE) + wave;
    if (chunk >= a.chunks) return;
    float x[PER], q[PER];
    vf_logits<B16, PER, false>(a, row, chunk, x);
    vf_guess<PER, false>(a, dr, chunk, q);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += vf_rest(vf_weight<CAP, true>(a, x[j], ztop), inv, q[j]);
    sum = vf_wave_sum(sum);
    if (lane == 0) a.sums[(size_t)s * a.chunks + chunk] = sum;
}

// The draw, a wave per sequence: the chunk where the running sum passes the border (four chunks a lane), then the token
// inside it.
template <bool B16, bool CAP, int PER> __global__ __launch_bounds__(WAVE) void k_verify_draw(VerifyArgs a) {
    const int s = blockIdx.x, lane = threadIdx.x, K = a.max_drafts;
    const int n = vf_drafts(a, s);
    const VfPlace at = a.places[s];
    const float u = vf_from0(a.u[(size_t)s * (K + 1) + K]);
    double mine[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[j] = a.sums[(size_t)s * a.chunks + min(4 * lane + j, a.chunks - 1)];
#pragma unroll
    for (int j = 0; j < 4; ++j) if (4 * lane + j >= a.chunks) mine[j] = 0.0;
    if (at.inv == 0.0) return;                               // no possible token: already written
    const long long row = (long long)s * (K + 1) + at.kept, dr = (long long)s * K + at.kept;
    const double ztop = vf_capped<CAP>(a, at.top);
    // all drafts kept (no sums were written then), or the draft's distribution covers the target's everywhere: the target's own
    const bool rest = at.kept < n && __ballot(mine[0] > 0.0 || mine[1] > 0.0 || mine[2] > 0.0 || mine[3] > 0.0) != 0;
    if (!rest)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const VfStat st = a.stats[(size_t)row * a.chunks + min(4 * lane + j, a.chunks - 1)];
            mine[j] = 4 * lane + j < a.chunks ? st.sum * vf_weight<CAP, true>(a, st.top, ztop) * at.inv : 0.0;
        }
    // (a random number of 1 or more, or none: no running sum passes the border, and the last possible token it is)
    double run = wave_scan_f64((mine[0] + mine[1]) + (mine[2] + mine[3]));
    const double border = u < 1.0f ? (double)u * wave_read_f64(run, 63) : INFINITY;
    run = wave_before_f64(run);
    int in = -1, end = -1;                                   // chunk that passes the border; last chunk with any weight
    double in_left = 0.0, end_left = 0.0;                    // ... and what of the border is left where it begins
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (mine[j] > 0.0) {
            end = 4 * lane + j; end_left = border - run;
            if (in < 0 && run + mine[j] > border) { in = end; in_left = end_left; }
        }
        run += mine[j];
    }
    const uint64_t ins = __ballot(in >= 0), ends = __ballot(end >= 0);
    const int from = ins ? __ffsll((unsigned long long)ins) - 1 : 63 - __clzll((long long)ends);
    const int chunk = __builtin_amdgcn_readlane(ins ? in : end, from);
    const double left = wave_read_f64(ins ? in_left : end_left, from);

    float x[PER], q[PER] = {};
    vf_logits<B16, PER, true>(a, row, chunk, x);
    if (rest) vf_guess<PER, true>(a, dr, chunk, q);
    double w[PER], sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const double t = vf_weight<CAP, true>(a, x[j], ztop);
        w[j] = rest ? vf_rest(t, at.inv, q[j]) : t * at.inv;
        sum += w[j];
    }
    double r = wave_before_f64(wave_scan_f64(sum));
    const int i0 = chunk * PER * WAVE + lane * PER;          // in index order
    int hit = -1, last = -1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        r += w[j];
        if (w[j] > 0.0) { last = i0 + j; if (r > left && hit < 0) hit = last; }
    }
    const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
    if (hits ? lane == __ffsll((unsigned long long)hits) - 1 : lane == 63 - __clzll((long long)lasts))
        a.tokens[(size_t)s * (K + 1) + at.kept] = (uint32_t)(hits ? hit : last);
}
