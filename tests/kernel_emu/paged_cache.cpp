// The paged-cache kernels' own source (kernel_paged.inc) on the CPU: k_rope_append, k_attn_paged in each of its forms and
// k_attn_paged_join against fp64 restatements, with page tables that name pages outside the pool, rows without slots,
// NaN in every slot that does not count, lengths that end inside a block and inside a split, shared sequences, fp32
// and bf16 rows and caches, more than 16 query heads per key head.  Every buffer is a heap block of its exact size.
#include "emu_ops.h"
#include "kernel_paged.inc"
#include <cstdio>
#include <random>

static std::mt19937 rng(3);
static float urand(float a) { return std::uniform_real_distribution<float>(-a, a)(rng); }
static int failures = 0;
static void report(bool ok, const char *what, double worst, double allowed) {
    std::printf("%s: worst %.3g (allowed %.3g)%s\n", what, worst, allowed, ok ? "" : "  FAIL");
    if (!ok) ++failures;
}
template <class T> static T *heap(size_t n) { return (T *)std::malloc(n * sizeof(T) ? n * sizeof(T) : 1); }

struct Pool {
    int pages, page, seqs, per, kvh, hd;
    bool b16, token_major;
    char *k, *v;
    int *table;
    size_t count() const { return (size_t)pages * page * kvh * hd; }
    size_t index(int p, int slot, int h, int d) const {
        return token_major ? (((size_t)p * page + slot) * kvh + h) * hd + d : (((size_t)p * kvh + h) * page + slot) * hd + d;
    }
    double get(const char *m, size_t i) const { return b16 ? (double)bf16_to_f32(((const uint16_t *)m)[i]) : (double)((const float *)m)[i]; }
    void set(char *m, size_t i, float x) { if (b16) ((uint16_t *)m)[i] = f32_to_bf16_rne(x); else ((float *)m)[i] = x; }
    PagedView view() const {
        const long long e = b16 ? 2 : 4;
        PagedView c{k, v, 0, 0, 0, table, pages, 0, seqs, per, kvh};
        c.stride_page = e * page * kvh * hd;
        c.stride_slot = e * (token_major ? kvh * hd : hd);
        c.stride_head = e * (token_major ? hd : page * hd);
        while ((1 << c.page_shift) < page) ++c.page_shift;
        return c;
    }
    Pool(int pages, int page, int seqs, int per, int kvh, int hd, bool b16, bool tm)
        : pages(pages), page(page), seqs(seqs), per(per), kvh(kvh), hd(hd), b16(b16), token_major(tm) {
        k = heap<char>(count() * (b16 ? 2 : 4)); v = heap<char>(count() * (b16 ? 2 : 4));
        table = heap<int>((size_t)seqs * per);
        for (size_t i = 0; i < count(); ++i) { set(k, i, NAN); set(v, i, NAN); }
        std::vector<int> order(pages);
        for (int i = 0; i < pages; ++i) order[i] = i;
        std::shuffle(order.begin(), order.end(), rng);
        for (int i = 0; i < seqs * per; ++i) table[i] = order[i % pages];
    }
    ~Pool() { std::free(k); std::free(v); std::free(table); }
    bool real(int seq, int slot, int *p) const {
        *p = table[(size_t)seq * per + slot / page];
        return *p >= 0 && *p < pages;
    }
};

template <int HD, bool QB, bool CB, bool FEW, int WAVES>
static void attention(const char *what, int g, int kvh, int page, bool tm, std::vector<int> lens, std::vector<int> seqs, int chunk, bool bad) {
    const int rows = (int)lens.size(), heads = g * kvh, n_seqs = *std::max_element(seqs.begin(), seqs.end()) + 1;
    const int max_len = *std::max_element(lens.begin(), lens.end()), per = max_len / page + 2, wide = heads * HD + 8;
    Pool pool(n_seqs * per, page, n_seqs, per, kvh, HD, CB, tm);
    // numbers where a slot counts; everything else stays NaN
    for (int r = 0; r < rows; ++r)
        for (int s = 0; s < lens[r]; ++s) {
            int p;
            if (seqs[r] < 0 || !pool.real(seqs[r], s, &p)) continue;
            for (int h = 0; h < kvh; ++h)
                for (int d = 0; d < HD; ++d) {
                    const size_t i = pool.index(p, s % page, h, d);
                    if (pool.get(pool.k, i) == pool.get(pool.k, i)) continue;
                    pool.set(pool.k, i, urand(1.5f)); pool.set(pool.v, i, urand(1.0f));
                }
        }
    if (bad)                                                 // pages that do not exist, and (where page 0 is read for them) NaN there
        for (int s = 0; s < n_seqs; ++s) { pool.table[s * per] = s % 2 ? -1 : pool.pages; if (per > 3) pool.table[s * per + 2] = 0x7fffffff; }
    void *q = std::malloc((size_t)rows * wide * (QB ? 2 : 4)), *out = std::malloc((size_t)rows * wide * (QB ? 2 : 4));
    auto get = [&](const void *m, size_t i) -> double { return QB ? (double)bf16_to_f32(((const uint16_t *)m)[i]) : (double)((const float *)m)[i]; };
    for (size_t i = 0; i < (size_t)rows * wide; ++i) {
        if (QB) { ((uint16_t *)q)[i] = f32_to_bf16_rne(urand(2.0f)); ((uint16_t *)out)[i] = 0x4240; }
        else { ((float *)q)[i] = urand(2.0f); ((float *)out)[i] = 48.0f; }
    }
    int *d_lens = heap<int>(rows), *d_seqs = heap<int>(rows);
    std::copy(lens.begin(), lens.end(), d_lens); std::copy(seqs.begin(), seqs.end(), d_seqs);
    const float scale = 1.0f / std::sqrt((float)HD);
    const int splits = (max_len + chunk - 1) / chunk ? (max_len + chunk - 1) / chunk : 1, tiles = (g + 15) / 16;
    float *po = heap<float>((size_t)rows * heads * splits * HD), *pml = heap<float>((size_t)rows * heads * splits * 2);
    PagedAttn a{pool.view(), q, out, wide, wide, d_lens, d_seqs, heads, g, tiles, max_len, chunk, splits, scale * 1.44269504f, po, pml};
    emu::launch_grid([&] { k_attn_paged<HD, QB, CB, FEW, WAVES>(a); }, (unsigned)(rows * kvh * tiles * splits), 64 * WAVES);
    if (splits > 1) emu::launch_grid([&] { k_attn_paged_join<HD, QB>(a); }, (unsigned)(rows * heads), 256);
    double worst = 0.0;
    for (int r = 0; r < rows; ++r) {
        for (int h = 0; h < heads; ++h) {
            std::vector<double> w(std::max(lens[r], 1), 0.0), o(HD, 0.0);
            double m = -1e300, l = 0.0;
            int p;
            const int n = seqs[r] < 0 ? 0 : lens[r];
            for (int s = 0; s < n; ++s) {
                if (!pool.real(seqs[r], s, &p)) continue;
                double d = 0.0;
                for (int e = 0; e < HD; ++e) d += get(q, (size_t)r * wide + h * HD + e) * pool.get(pool.k, pool.index(p, s % page, h / g, e));
                w[s] = d * scale; m = std::fmax(m, w[s]);
            }
            for (int s = 0; s < n; ++s) {
                if (!pool.real(seqs[r], s, &p)) continue;
                const double x = std::exp(w[s] - m);
                l += x;
                for (int e = 0; e < HD; ++e) o[e] += x * pool.get(pool.v, pool.index(p, s % page, h / g, e));
            }
            for (int e = 0; e < HD; ++e) {
                const double want = l > 0 ? o[e] / l : 0.0, got = get(out, (size_t)r * wide + h * HD + e);
                worst = std::fmax(worst, got == got ? std::fabs(got - want) - (QB ? std::fabs(want) / 256 : 0.0) : 1e9);
            }
        }
        for (int e = heads * HD; e < wide; ++e)              // between the rows: left as it was
            if (get(out, (size_t)r * wide + e) != 48.0) worst = 1e9;
    }
    // scores of up to 8 in fp32 (128 .. 256 terms) and sums of up to 400 weights: 2e-5 of values up to 1
    report(worst <= 2e-5, what, worst, 2e-5);
    std::free(q); std::free(out); std::free(d_lens); std::free(d_seqs); std::free(po); std::free(pml);
}

template <bool RB, bool CB, int NP>
static void rope(const char *what, int hd, int rot, bool interleaved, int heads, int kvh, int page, bool tm, bool in_place, int parts) {
    const int rows = 5, seqs = 4, per = 3, gap = 8, wide = (heads + 2 * kvh) * hd + gap;
    Pool pool(seqs * per + 1, page, seqs, per, kvh, hd, CB, tm);
    pool.table[1 * per + 0] = -7;                            // a page that does not exist: row 1 of slot 0 writes nothing
    const size_t esz = RB ? 2 : 4;
    char *in = heap<char>((size_t)rows * wide * esz), *qo = in_place ? in : heap<char>((size_t)rows * heads * hd * esz);
    auto get = [&](const char *m, size_t i) -> double { return RB ? (double)bf16_to_f32(((const uint16_t *)m)[i]) : (double)((const float *)m)[i]; };
    for (size_t i = 0; i < (size_t)rows * wide; ++i) {
        const float x = urand(3.0f);
        if (RB) ((uint16_t *)in)[i] = f32_to_bf16_rne(x); else ((float *)in)[i] = x;
    }
    std::vector<char> before(in, in + (size_t)rows * wide * esz);
    double *freq = heap<double>(rot / 2);
    for (int i = 0; i < rot / 2; ++i) freq[i] = std::pow(10000.0, -2.0 * i / rot);
    int *pos = heap<int>(rows), *slots = heap<int>(rows), *sq = heap<int>(rows);
    const int ps[rows] = {0, 131071, -5, 1000003, 77}, sl[rows] = {per * page - 1, 0, -1, 2 * page, per * page}, ss[rows] = {0, 1, 2, 3, 0};
    std::copy(ps, ps + rows, pos); std::copy(sl, sl + rows, slots); std::copy(ss, ss + rows, sq);
    const float mag = 1.25f;
    const size_t bytes = pool.count() * (CB ? 2 : 4);
    std::vector<char> k0(pool.k, pool.k + bytes), v0(pool.v, pool.v + bytes);
    RopeArgs a{pool.view(), in, in + (size_t)heads * hd * esz, in + (size_t)(heads + kvh) * hd * esz, qo, wide, wide, wide,
               in_place ? wide : heads * hd, freq, pos, slots, sq, heads, kvh, hd, rot, interleaved, parts, mag};
    emu::launch_grid([&] { k_rope_append<RB, CB, NP>(a); }, (unsigned)(rows * parts), ROPE_THREADS);
    double worst = 0.0;
    auto want = [&](int t, int h, int d) -> double {         // element d of head h (queries, keys, values one after the other)
        const char *b = before.data();
        const size_t at = (size_t)t * wide + (size_t)h * hd;
        if (h >= heads + kvh || d >= rot) return get(b, at + d);
        const int i = interleaved ? d / 2 : d % (rot / 2);
        const bool second = interleaved ? d % 2 : d >= rot / 2;
        const double x = get(b, at + (interleaved ? 2 * i : i)), y = get(b, at + (interleaved ? 2 * i + 1 : i + rot / 2)), an = ps[t] * freq[i];
        return (second ? y * std::cos(an) + x * std::sin(an) : x * std::cos(an) - y * std::sin(an)) * mag;
    };
    auto off = [&](double got, double w, bool b16) { worst = std::fmax(worst, got == got ? std::fabs(got - w) - (b16 ? std::fabs(w) / 256 : 0.0) : 1e9); };
    for (int t = 0; t < rows; ++t)
        for (int h = 0; h < heads; ++h)
            for (int d = 0; d < hd; ++d) off(get(qo, (size_t)t * (in_place ? wide : heads * hd) + h * hd + d), want(t, h, d), RB);
    for (int t = 0; t < rows; ++t) {
        int p;
        if (sl[t] < 0 || sl[t] >= per * page || !pool.real(ss[t], sl[t], &p)) continue;
        for (int h = 0; h < kvh; ++h)
            for (int d = 0; d < hd; ++d) {
                const size_t i = pool.index(p, sl[t] % page, h, d), e = CB ? 2 : 4;
                off(pool.get(pool.k, i), want(t, heads + h, d), CB);
                off(pool.get(pool.v, i), want(t, heads + kvh + h, d), CB);
                std::memcpy(pool.k + i * e, &k0[i * e], e); std::memcpy(pool.v + i * e, &v0[i * e], e);
            }
    }
    if (std::memcmp(pool.k, k0.data(), bytes) || std::memcmp(pool.v, v0.data(), bytes)) worst = 1e9;   // no other slot was touched
    // |x| + |y| <= 6, times 1.25: the fp32 turn (half an ulp of the reduced angle, of sine, cosine and three operations) is 4e-7 of it
    report(worst <= 3.1e-6, what, worst, 3.1e-6);
    if (!in_place) std::free(qo);
    std::free(in); std::free(freq); std::free(pos); std::free(slots); std::free(sq);
}

int main() {
    rope<false, true, 4>("k_rope_append fp32 rows, bf16 cache, interleaved", 128, 128, true, 4, 2, 4, true, false, 1);
    rope<true, true, 4>("k_rope_append bf16, half layout, part of the head, in place", 64, 32, false, 3, 1, 8, false, true, 2);
    rope<false, false, 1>("k_rope_append pair by pair, half layout of 31 pairs", 64, 62, false, 2, 2, 1, false, false, 3);
    rope<true, false, 1>("k_rope_append pair by pair, interleaved, hd 10", 10, 6, true, 5, 1, 2, true, true, 1);
    rope<false, true, 4>("k_rope_append without a rotation", 192, 0, true, 2, 1, 2, false, false, 1);
    attention<128, false, true, true, 4>("k_attn_paged<128, fp32, bf16, few>, splits", 1, 2, 16, true, {385, 0, 1, 129}, {0, 1, 2, 1}, 128, false);
    attention<128, true, true, true, 8>("k_attn_paged<128, bf16, bf16, few>, one split", 4, 1, 64, false, {200, 255}, {1, 0}, 256, false);
    attention<128, true, true, false, 4>("k_attn_paged<128, bf16, bf16>, pages that do not exist", 16, 1, 4, false, {70, 33, 3}, {0, 1, 2}, 128, true);
    attention<64, false, false, true, 4>("k_attn_paged<64, fp32, fp32, few>, shared sequences, no such sequence", 4, 2, 8, true, {37, 38, 39, 20}, {0, 0, 0, -1}, 32, false);
    attention<64, false, true, false, 8>("k_attn_paged<64, fp32, bf16>, 18 heads, pages of one slot", 18, 1, 1, false, {130, 17}, {0, 1}, 256, true);
    attention<64, false, true, true, 8>("k_attn_paged<64, fp32, bf16, few>, one split", 1, 4, 16, false, {1, 17, 250, 0, 129}, {0, 1, 2, 3, 4}, 256, false);
    attention<64, false, true, true, 4>("k_attn_paged<64, fp32, bf16, few>, splits", 2, 2, 16, true, {1, 17, 300, 0, 129}, {0, 1, 2, 3, 4}, 128, false);
    attention<192, true, true, true, 4>("k_attn_paged<192, bf16, bf16, few>", 2, 1, 32, true, {150}, {0}, 128, true);
    attention<256, false, false, false, 4>("k_attn_paged<256, fp32, fp32>", 5, 1, 16, false, {90, 2}, {0, 1}, 64, false);
    std::printf("%d checks failed\n", failures);
    return failures ? 1 : 0;
}
