// The draft-verification kernels' own source (kernel_verify.inc) on the CPU against a sequential fp64 restatement, token for
// token: vocabularies that end inside a chunk, drafts of unequal length (below 0 and above the maximum among them), tokens
// outside the vocabulary, NaN, -inf and +inf logits, rows of nothing but -inf, a draft that covers the target everywhere,
// NaN probabilities, random numbers 0 and 1, soft cap, ties at temperature 0.  Every buffer is a heap block of its exact size.
#include "emu_ops.h"
#include "kernel_verify.inc"
#include <cstdio>
#include <random>

static std::mt19937 rng(5);
static int failures = 0;
template <class T> static T *heap(size_t n) { return (T *)std::malloc(n * sizeof(T) ? n * sizeof(T) : 1); }

// what a sequence of each number has that is out of the ordinary
enum { PLAIN, ALL_IMPOSSIBLE, NAN_LOGITS, INF_LOGIT, COVERED, OUTSIDE, U_ZERO, U_ONE, NAN_PROBS, TIES, SPECIALS };

template <bool B16, bool CAP, int PER> static void run(const char *what, int vocab, int K, float T, float cap, bool probs) {
    const int S = SPECIALS, rows = S * (K + 1), chunks = (vocab + PER * WAVE - 1) / (PER * WAVE), stride = vocab + 3;
    std::normal_distribution<float> nd(0.0f, 3.0f);
    std::uniform_real_distribution<float> ud(0.0f, 1.0f);
    void *lg = std::malloc((size_t)rows * stride * (B16 ? 2 : 4));
    auto set = [&](size_t i, float x) { if (B16) ((uint16_t *)lg)[i] = f32_to_bf16_rne(x); else ((float *)lg)[i] = x; };
    auto get = [&](size_t i) -> float { return B16 ? bf16_to_f32(((const uint16_t *)lg)[i]) : ((const float *)lg)[i]; };
    for (size_t i = 0; i < (size_t)rows * stride; ++i) set(i, i % stride < (size_t)vocab ? nd(rng) : NAN);
    int *drafts = heap<int>((size_t)S * K), *n = heap<int>(S);
    float *u = heap<float>((size_t)S * (K + 1)), *q = probs ? heap<float>((size_t)S * K * stride) : nullptr;
    for (int i = 0; i < S * (K + 1); ++i) u[i] = ud(rng);
    for (int s = 0; s < S; ++s) n[s] = s == 0 ? K + 5 : s == 5 ? K : s == 6 ? -3 : (s + 1) % (K + 1);
    for (int s = 0; s < S; ++s) {
        for (int i = 0; i <= K; ++i) {
            const size_t at = ((size_t)s * (K + 1) + i) * stride;
            for (int j = 0; j < vocab; ++j) {
                if (s == ALL_IMPOSSIBLE && i == (K > 1 ? 1 : 0)) set(at + j, -INFINITY);
                if (s == NAN_LOGITS && j % 3 == 0) set(at + j, NAN);
                if (s == INF_LOGIT && (j == 7 || j == vocab - 1)) set(at + j, INFINITY);
                if (s == TIES) set(at + j, (float)(j % 5));
                if (s == U_ZERO && j < 40) set(at + j, -INFINITY);
            }
            if (i == K) continue;
            // drafts the target likes, so that some are kept: the best of a few
            int d = (int)(rng() % vocab);
            for (int k = 0; k < 400; ++k) { const int c = (int)(rng() % vocab); if (get(at + c) > get(at + d) || get(at + d) != get(at + d)) d = c; }
            if (s == INF_LOGIT) d = 7;
            if (s == TIES) d = 4;
            if (s == OUTSIDE) d = i % 2 ? -1 : vocab;
            drafts[s * K + i] = d;
            if (!probs) continue;
            float *row = q + ((size_t)s * K + i) * stride;
            double sum = 0.0;
            for (int j = 0; j < vocab; ++j) { const float x = get(at + j); row[j] = x == x && x < 1e30f ? std::exp((x + 0.3f * nd(rng)) / (T > 0 ? T : 1.0f)) : 0.0f; sum += row[j]; }
            for (int j = 0; j < vocab; ++j) row[j] = s == COVERED ? 1.0f : s == NAN_PROBS && j % 2 ? NAN : sum > 0 ? (float)(row[j] / sum) : 0.0f;
            for (int j = vocab; j < stride; ++j) row[j] = NAN;
        }
        if (s == U_ZERO) for (int i = 0; i <= K; ++i) u[s * (K + 1) + i] = 0.0f;
        if (s == U_ONE) u[s * (K + 1) + K] = 1.0f;
    }
    VfStat *st = heap<VfStat>((size_t)rows * chunks);
    double *sums = heap<double>((size_t)S * chunks);
    VfPlace *pl = heap<VfPlace>(S);
    uint32_t *tok = heap<uint32_t>((size_t)S * (K + 1));
    int *acc = heap<int>(S);
    std::memset(st, 0x7f, (size_t)rows * chunks * sizeof(VfStat)); std::memset(sums, 0x7f, (size_t)S * chunks * 8); std::memset(pl, 0x7f, S * sizeof(VfPlace));
    const double log2e = 1.4426950408889634074;
    VerifyArgs a{lg, stride, stride, drafts, n, q, T > 0 ? u : nullptr, S, K, vocab, chunks, T > 0 ? log2e / T : 0.0, cap, cap > 0 ? 2 * log2e / cap : 0.0, st, sums, pl, tok, acc};
    emu::launch_grid([&] { k_verify_stats<B16, CAP, PER>(a); }, (unsigned)(rows * ((chunks + VF_STATS / WAVE - 1) / (VF_STATS / WAVE))), VF_STATS);
    emu::launch_grid([&] { k_verify_decide<B16, CAP, PER>(a); }, (unsigned)(T > 0 ? S * ((chunks + VF_DECIDE / WAVE - 1) / (VF_DECIDE / WAVE)) : S), VF_DECIDE);
    if (T > 0) emu::launch_grid([&] { k_verify_draw<B16, CAP, PER>(a); }, (unsigned)S, WAVE);

    int wrong = 0, kept_all = 0;
    std::vector<double> p(vocab), qq(vocab);
    for (int s = 0; s < S; ++s) {
        const int nd_ = std::min(std::max(n[s], 0), K);
        int i = 0;
        uint32_t next = 0xffffffffu;
        for (;; ++i) {
            const size_t at = ((size_t)s * (K + 1) + i) * stride;
            double top = -INFINITY, sum = 0.0;
            int best = -1;
            auto z = [&](int j) { float x = get(at + j); if (!(x == x)) x = -INFINITY; x = std::fmin(x, 3.4028235e38f); return cap > 0 && x > -INFINITY ? cap * std::tanh((double)x / cap) : (double)x; };
            for (int j = 0; j < vocab; ++j) if (z(j) > top) { top = z(j); best = j; }
            for (int j = 0; j < vocab; ++j) { p[j] = top == -INFINITY ? 0.0 : T > 0 ? std::exp((z(j) - top) / T) : j == best; sum += p[j]; }
            for (int j = 0; j < vocab; ++j) p[j] = sum > 0 ? p[j] / sum : 0.0;
            auto draw = [&](const std::vector<double> &w) {
                double whole = 0.0, r = 0.0;
                int last = -1;
                for (double x : w) whole += x;
                for (int j = 0; j < vocab; ++j) { r += w[j]; if (w[j] > 0) { last = j; if (r > (double)u[s * (K + 1) + K] * whole) return (uint32_t)j; } }
                return (uint32_t)last;
            };
            if (i == nd_) { next = best < 0 ? 0xffffffffu : T > 0 ? draw(p) : (uint32_t)best; break; }
            const int d = drafts[s * K + i];
            const bool in = d >= 0 && d < vocab;
            for (int j = 0; j < vocab; ++j) qq[j] = probs && T > 0 ? (double)q[((size_t)s * K + i) * stride + j] : j == d ? 1.0 : 0.0;
            if (in && (T > 0 ? (double)u[s * (K + 1) + i] * qq[d] < p[d] : d == best)) continue;
            if (best < 0) { next = 0xffffffffu; break; }
            if (T <= 0) { next = (uint32_t)best; break; }
            double whole = 0.0;
            for (int j = 0; j < vocab; ++j) { const double r = p[j] - qq[j]; qq[j] = r > 0 ? r : 0.0; whole += qq[j]; }
            next = draw(whole > 0 ? qq : p);
            break;
        }
        kept_all += i == nd_;
        if (acc[s] != i) { ++wrong; std::printf("  sequence %d: %d kept, want %d\n", s, acc[s], i); }
        for (int j = 0; j <= K; ++j) {
            const uint32_t want = j < i ? (uint32_t)drafts[s * K + j] : j == i ? next : 0xffffffffu, got = tok[s * (K + 1) + j];
            if (got != want) { ++wrong; std::printf("  sequence %d place %d: %u, want %u\n", s, j, got, want); }
        }
    }
    std::printf("%s: %d sequences, all drafts kept in %d, %d mismatches%s\n", what, S, kept_all, wrong, wrong ? "  FAIL" : "");
    failures += wrong != 0;
    std::free(lg); std::free(drafts); std::free(n); std::free(u); std::free(q); std::free(st); std::free(sums); std::free(pl); std::free(tok); std::free(acc);
}

int main() {
    run<false, false, 4>("k_verify_* fp32, draft probabilities", 2500, 3, 0.8f, 0.0f, true);
    run<true, true, 4>("k_verify_* bf16, soft cap, draft probabilities", 1031, 2, 1.3f, 20.0f, true);
    run<false, true, 16>("k_verify_* fp32, soft cap, looked-up drafts", 4099, 2, 0.6f, 5.0f, false);
    run<true, false, 16>("k_verify_* bf16, looked-up drafts, one chunk", 300, 5, 1.0f, 0.0f, false);
    run<false, false, 4>("k_verify_* fp32, temperature 0", 1500, 3, 0.0f, 0.0f, true);
    run<false, false, 4>("k_verify_* fp32, seven drafts", 1024, 7, 0.05f, 0.0f, true);
    std::printf("%d checks failed\n", failures);
    return failures ? 1 : 0;
}
