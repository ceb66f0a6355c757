// More of the draft-verification kernels' own source on the CPU, one check per name on the command line, against a restatement
// in long double: numbers outside their range, temperatures near 0.  Unlike verify_drafts.cpp it runs the waves' running sums and maxima from their
// own source too (kernel_wave64.inc: the data-parallel moves are stood in for, not the functions above them), and the
// reciprocal is good to 24 bits only, as the instruction is.
#define wave_scan_f64 whole_scan_f64
#define wave_read_f64 whole_read_f64
#define wave_before_f64 whole_before_f64
#define wave_max_dpp whole_max_dpp
#include "emu_ops.h"
#undef wave_scan_f64
#undef wave_read_f64
#undef wave_before_f64
#undef wave_max_dpp
#undef __builtin_amdgcn_rcp
#define __builtin_amdgcn_rcp(x) ((double)(float)(1.0 / (x)))

namespace emu {
// v_mov_b32 with a data-parallel move: `old` where the lane's row is masked out or the move has no source for it
inline int dpp(int old, int src, int ctrl, int row_mask) {
    const uint64_t *all = share(src);
    const int l = lane(), row = l / 16;
    int from = -1;
    if (ctrl > 0x110 && ctrl < 0x120) from = l % 16 >= (ctrl & 15) ? l - (ctrl & 15) : -1;   // row_shr
    else if (ctrl == 0x138) from = l - 1;                                                    // wave_shr:1
    else if (ctrl == 0x142) from = row ? 16 * row - 1 : -1;                                  // row_bcast:15
    else if (ctrl == 0x143) from = row > 1 ? 31 : -1;                                        // row_bcast:31
    else std::abort();
    return (row_mask >> row & 1) && from >= 0 ? of_bits<int>(all[from]) : old;
}
}  // namespace emu
#define __builtin_amdgcn_update_dpp(old, src, ctrl, rows, banks, bound) emu::dpp((old), (src), (ctrl), (rows))
#undef __builtin_amdgcn_readlane
#define __builtin_amdgcn_readlane(v, l) emu::from_lane((int)(v), (l))
static inline float __int_as_float(int i) { return emu::of_bits<float>((uint32_t)i); }
#include "kernel_wave64.inc"
#include "kernel_verify.inc"
#include <cstdio>
#include <cstring>
#include <random>

static std::mt19937 rng(11);
static float normal(float s) { return std::normal_distribution<float>(0.0f, s)(rng); }
static float uniform() { return std::uniform_real_distribution<float>(0.0f, 1.0f)(rng); }

struct Drafts {
    int S, K, V;
    float T, cap;
    bool with_probs;
    std::vector<float> lg, q, u;                             // [S][K + 1][V], [S][K][V], [S][K + 1]
    std::vector<int> d, n;
    Drafts(int S, int K, int V, float T, float cap, bool with_probs) : S(S), K(K), V(V), T(T), cap(cap), with_probs(with_probs),
        lg((size_t)S * (K + 1) * V), q((size_t)S * K * V), u((size_t)S * (K + 1)), d((size_t)S * K), n(S, K) {
        for (float &x : lg) x = normal(3.0f);
        for (float &x : u) x = uniform();
        for (int s = 0; s < S; ++s)
            for (int i = 0; i < K; ++i) {
                double sum = 0.0;
                for (int j = 0; j < V; ++j) sum += prob(s, i)[j] = std::exp(0.8f * row(s, i)[j]);
                for (int j = 0; j < V; ++j) prob(s, i)[j] /= (float)sum;
                int best = (int)(rng() % V);
                for (int k = 0; k < 300; ++k) { const int c = (int)(rng() % V); if (row(s, i)[c] > row(s, i)[best]) best = c; }
                d[s * K + i] = best;
            }
    }
    float *row(int s, int i) { return &lg[((size_t)s * (K + 1) + i) * V]; }
    float *prob(int s, int i) { return &q[((size_t)s * K + i) * V]; }
};
struct Decided { std::vector<uint32_t> tokens; std::vector<int> accepted; };

// the kernels on heap blocks of their exact sizes
template <class T> static T *copy_of(const std::vector<T> &v) { T *p = (T *)std::malloc(v.size() * sizeof(T) + !v.size()); if (v.size()) std::memcpy(p, v.data(), v.size() * sizeof(T)); return p; }
template <bool CAP, int PER> static Decided run(Drafts &c) {
    const int rows = c.S * (c.K + 1), chunks = (c.V + PER * WAVE - 1) / (PER * WAVE);
    float *lg = copy_of(c.lg), *q = c.with_probs ? copy_of(c.q) : nullptr, *u = copy_of(c.u);
    int *d = copy_of(c.d), *n = copy_of(c.n);
    VfStat *st = copy_of(std::vector<VfStat>((size_t)rows * chunks));
    double *sums = copy_of(std::vector<double>((size_t)c.S * chunks, NAN));
    VfPlace *pl = copy_of(std::vector<VfPlace>(c.S));
    uint32_t *tok = copy_of(std::vector<uint32_t>((size_t)c.S * (c.K + 1), 12345u));
    int *acc = copy_of(std::vector<int>(c.S, -9));
    const double log2e = 1.4426950408889634074;
    VerifyArgs a{lg, c.V, c.V, d, n, q, u, c.S, c.K, c.V, chunks, c.T > 0 ? log2e / c.T : 0.0, c.cap, CAP ? 2 * log2e / c.cap : 0.0, st, sums, pl, tok, acc};
    emu::launch_grid([&] { k_verify_stats<false, CAP, PER>(a); }, (unsigned)(rows * ((chunks + VF_STATS / WAVE - 1) / (VF_STATS / WAVE))), VF_STATS);
    emu::launch_grid([&] { k_verify_decide<false, CAP, PER>(a); }, (unsigned)(c.T > 0 ? c.S * ((chunks + VF_DECIDE / WAVE - 1) / (VF_DECIDE / WAVE)) : c.S), VF_DECIDE);
    if (c.T > 0) emu::launch_grid([&] { k_verify_draw<false, CAP, PER>(a); }, (unsigned)c.S, WAVE);
    Decided r{std::vector<uint32_t>(tok, tok + (size_t)c.S * (c.K + 1)), std::vector<int>(acc, acc + c.S)};
    for (void *p : {(void *)lg, (void *)q, (void *)u, (void *)d, (void *)n, (void *)st, (void *)sums, (void *)pl, (void *)tok, (void *)acc}) std::free(p);
    return r;
}

// the definition; a negative probability or random number counts as 0
static Decided wanted(Drafts &c) {
    Decided r{std::vector<uint32_t>((size_t)c.S * (c.K + 1), 0xffffffffu), std::vector<int>(c.S, 0)};
    std::vector<long double> p(c.V), w(c.V);
    auto from0 = [](float x) { return x < 0.0f ? 0.0f : x; };
    for (int s = 0; s < c.S; ++s) {
        const int n = std::min(std::max(c.n[s], 0), c.K);
        uint32_t next = 0xffffffffu;
        int i = 0;
        for (;; ++i) {
            const float *x = c.row(s, i);
            auto z = [&](int j) -> long double { return !(x[j] > -INFINITY) ? -INFINITY : c.cap > 0 ? c.cap * tanhl((long double)x[j] / c.cap) : (long double)x[j]; };
            int best = -1;
            for (int j = 0; j < c.V; ++j) if (x[j] > -INFINITY && (best < 0 || x[j] > x[best])) best = j;
            long double sum = 0.0;
            for (int j = 0; j < c.V; ++j) sum += p[j] = best < 0 ? 0.0L : c.T > 0 ? expl((z(j) - z(best)) / c.T) : (long double)(j == best);
            if (best >= 0) for (long double &v : p) v /= sum;
            auto draw = [&](const std::vector<long double> &w) {
                long double whole = 0.0, run = 0.0;
                uint32_t last = 0xffffffffu;
                for (long double v : w) whole += v;
                for (int j = 0; j < c.V; ++j) if ((run += w[j], w[j] > 0)) { last = (uint32_t)j; if (run > (long double)from0(c.u[s * (c.K + 1) + c.K]) * whole) break; }
                return last;
            };
            const bool behind = i == n;
            const int d = behind ? -1 : c.d[s * c.K + i];
            auto guess = [&](int j) -> long double { return c.with_probs ? from0(c.prob(s, i)[j]) : (float)(j == d); };
            if (!behind && d >= 0 && d < c.V && (c.T > 0 ? (long double)from0(c.u[s * (c.K + 1) + i]) * guess(d) < p[d] : d == best)) { r.tokens[s * (c.K + 1) + i] = (uint32_t)d; continue; }
            if (c.T <= 0) { next = (uint32_t)best; break; }
            long double rest = 0.0;
            if (!behind) for (int j = 0; j < c.V; ++j) rest += w[j] = std::fmax(p[j] - guess(j), 0.0L);
            next = draw(rest > 0 ? w : p);
            break;
        }
        r.tokens[s * (c.K + 1) + i] = next;
        r.accepted[s] = i;
    }
    return r;
}
static int compared(const char *what, const Decided &got, const Decided &want) {
    int wrong = 0;
    for (size_t i = 0; i < want.accepted.size(); ++i)
        if (got.accepted[i] != want.accepted[i]) { ++wrong; std::printf("  %s: sequence %zu keeps %d, want %d\n", what, i, got.accepted[i], want.accepted[i]); }
    for (size_t i = 0; i < want.tokens.size(); ++i)
        if (got.tokens[i] != want.tokens[i]) { ++wrong; std::printf("  %s: place %zu has %u, want %u\n", what, i, got.tokens[i], want.tokens[i]); }
    return wrong;
}

// Negative probabilities, at the last token of a vocabulary that ends inside a chunk, at tokens the target cannot give and all
// over; negative random numbers with drafts the target cannot give.
static int negative_numbers() {
    int wrong = 0;
    for (bool with_probs : {true, false}) {
        Drafts c(6, 2, 1031, 0.9f, 0.0f, with_probs);
        for (int s = 0; s < c.S; ++s)
            for (int i = 0; i < c.K; ++i) {
                float *p = c.prob(s, i);
                if (s < 3) c.u[s * 3] = c.u[s * 3 + 1] = 0.99999f;
                if (s == 0) p[c.V - 1] = -0.7f;
                if (s == 1) for (int j = 5; j < c.V; j += 7) { c.row(s, i)[j] = -INFINITY; p[j] = -0.5f; }
                if (s == 2) for (int j = 0; j < c.V; ++j) p[j] = -p[j];
                if (s == 3) { c.row(s, i)[c.d[s * c.K + i]] = -INFINITY; c.u[s * 3 + i] = -0.25f; p[c.d[s * c.K + i]] = 0.3f; }
                if (s == 4) { c.row(s, i)[c.d[s * c.K + i]] = -INFINITY; p[c.d[s * c.K + i]] = -0.3f; }
            }
        c.u[5 * 3 + 2] = -3.0f;
        c.u[4 * 3 + 2] = -INFINITY;
        wrong += compared(with_probs ? "probabilities" : "looked up", run<false, 4>(c), wanted(c));
    }
    return wrong;
}

// A soft cap that every other logit saturates, at temperatures down to the smallest: the saturated ones lie within the last bits of
// each other, and nothing but one of them may be kept or drawn.
static int tiny_temperatures() {
    int wrong = 0;
    for (float T : {1e-12f, 1e-18f, 1e-20f, 1e-30f, 1.17549435e-38f})
        for (bool with_probs : {false, true}) {
            Drafts c(8, 3, 700, T, 2.0f, with_probs);
            for (int s = 0; s < c.S; ++s)
                for (int i = 0; i <= c.K; ++i) {
                    for (int j = 0; j < c.V; ++j) c.row(s, i)[j] = j % 2 ? 40.0f + 30.0f * uniform() : normal(2.0f);
                    for (int j = 0; i < c.K && j < c.V; ++j) c.prob(s, i)[j] = 1.0f / c.V;
                    if (i < c.K) c.d[s * c.K + i] = (int)(rng() % c.V);
                }
            const Decided got = run<true, 4>(c);
            for (int s = 0; s < c.S; ++s)
                for (int i = 0; i <= c.K; ++i) {
                    const uint32_t t = got.tokens[s * (c.K + 1) + i];
                    const bool ok = i > got.accepted[s] ? t == 0xffffffffu : t < (uint32_t)c.V && t % 2 == 1;
                    if (!ok) { ++wrong; std::printf("  temperature %g: sequence %d place %d has %u\n", T, s, i, t); }
                }
        }
    return wrong;
}

// Temperature 0: an infinite logit is above the largest finite one, and the first of equals is taken; drafts among them.
static int greedy_infinities() {
    int wrong = 0;
    for (float cap : {0.0f, 4.0f}) {
        Drafts c(5, 2, 1500, 0.0f, cap, true);
        for (int s = 0; s < c.S; ++s)
            for (int i = 0; i <= c.K; ++i) {
                float *x = c.row(s, i);
                x[3] = 3.4028235e38f;
                if (s) x[500] = x[1400] = INFINITY;
                if (s == 2) x[40] = INFINITY;
                if (s == 3) for (int j = 0; j < c.V; ++j) x[j] = j % 2 ? -INFINITY : NAN;
                if (i < c.K) c.d[s * c.K + i] = s == 0 ? 3 : s == 1 ? (i ? 1400 : 500) : s == 2 ? 40 : s == 3 ? 1 : 3;
            }
        wrong += compared(cap > 0 ? "soft cap" : "no cap", cap > 0 ? run<true, 4>(c) : run<false, 4>(c), wanted(c));
    }
    return wrong;
}

// Eight logits a lane (chunks of 512), the form of 4 to 12 million logits and of vocabularies of 65537 .. 131072: several chunks,
// the last one ending inside, and one chunk.
static int eight_logits_a_lane() {
    int wrong = 0;
    for (int V : {4700, 1537, 300})
        for (bool with_probs : {true, false}) {
            Drafts c(7, 3, V, 0.8f, 0.0f, with_probs), d(7, 2, V, 1.1f, 12.0f, with_probs), e(4, 2, V, 0.0f, 0.0f, with_probs);
            c.n = {3, 0, 1, 2, 3, 9, -1};
            wrong += compared("no cap", run<false, 8>(c), wanted(c)) + compared("soft cap", run<true, 8>(d), wanted(d)) + compared("temperature 0", run<false, 8>(e), wanted(e));
        }
    return wrong;
}

// A soft cap and a small temperature: what lies too far below the maximum for 64 bits has no probability at all, as without a cap.
// A random number of 0 finds the first token that has one, and a draft that covers those leaves no rest.
static int far_below_the_maximum() {
    int wrong = 0;
    for (float cap : {0.0f, 30.0f})
        for (bool with_probs : {true, false}) {
            Drafts c(4, 2, 600, 1e-3f, cap, with_probs);
            for (int s = 0; s < c.S; ++s)
                for (int i = 0; i <= c.K; ++i) {
                    for (int j = 0; j < c.V; ++j) c.row(s, i)[j] = j < 100 || j % 3 == 0 ? -30.0f : 25.0f + normal(1e-3f);
                    for (int j = 0; i < c.K && j < c.V; ++j) c.prob(s, i)[j] = s == 3 || j == 101 ? 0.0f : 1.0f;
                    if (i < c.K) { c.d[s * c.K + i] = s == 2 ? 7 : 400; c.u[s * 3 + i] = s == 2 ? 0.0f : 0.9f; }
                    if (s == 1) for (int j = 0; i < c.K && j < c.V; ++j) c.prob(s, i)[j] = j < 100 ? 0.0f : 1.0f;
                }
            c.u[2] = c.u[11] = 0.0f;
            wrong += compared(cap > 0 ? "soft cap" : "no cap", cap > 0 ? run<true, 4>(c) : run<false, 4>(c), wanted(c));
        }
    return wrong;
}

// The soft cap and the exponential against long double.  Allowed: the polynomial's 1.5e-15, the reciprocal's 2^-48 = 3.6e-15 behind
// one Newton step and some ten roundings of 1.1e-16: 1e-14 of the value; the exponential, without a reciprocal, 4e-15.
static int elementary_accuracy() {
    int wrong = 0;
    long double worst = 0.0, worst_e = 0.0;
    VerifyArgs a{};
    for (float cap : {1e-3f, 0.5f, 2.0f, 5.0f, 30.0f, 50.0f, 1e4f, 1e8f, 1e30f}) {
        a.cap = cap;
        a.cap_k = 2 * 1.4426950408889634074 / a.cap;
        for (int i = 0; i < 20000; ++i) {
            const float x = (i % 2 ? -1.0f : 1.0f) * cap * (float)std::pow(10.0, -12.0 + 13.6 * i / 20000);
            const long double want = tanhl((long double)x / cap), got = vf_capped<true>(a, x);
            worst = std::fmax(worst, std::fabs(got / want - 1.0L));
        }
    }
    for (int i = 0; i <= 40000; ++i) {
        const double y = i < 20000 ? -1021.0 * i / 20000 : -1.0 * (i - 20000) / 20000;
        worst_e = std::fmax(worst_e, std::fabs((long double)vf_exp2(y) / exp2l(y) - 1.0L));
    }
    std::printf("soft cap off by up to %.2Lg of itself, exponential %.2Lg\n", worst, worst_e);
    wrong += !(worst <= 1e-14L) + !(worst_e <= 4e-15L) + (vf_exp2(0.0) != 1.0) + (vf_capped<true>(a, 0.0f) != 0.0);
    return wrong;
}

int main(int argc, char **argv) {
    const struct { const char *name; int (*check)(); } checks[] = {{"negative_numbers", negative_numbers}, {"tiny_temperatures", tiny_temperatures},
                                                               {"elementary_accuracy", elementary_accuracy}, {"greedy_infinities", greedy_infinities},
                                                               {"eight_logits_a_lane", eight_logits_a_lane}, {"far_below_the_maximum", far_below_the_maximum}};
    for (const auto &c : checks)
        if (argc > 1 && !std::strcmp(argv[1], c.name)) {
            const int wrong = c.check();
            std::printf("%s: %d wrong\n", c.name, wrong);
            return wrong ? 1 : 0;
        }
    return 2;
}
