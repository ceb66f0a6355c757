// More of the paged-cache kernels' own source on the CPU, one check per name on the command line: how near the rotary positions
// come to the formula.  (The buffers and pools are paged_cache.cpp's, its text up to the first check.)
#include "paged_pool.inc"

// Rotated fp32 queries and keys against long double.  Allowed for each: sine and cosine (with the magnitude) rounded to fp32 once,
// two products and a sum, each half a step of 2^-24, and the angle's own rounding in 64 bits: a * 2^-53.
template <int NP> static int rotation(bool interleaved, int hd, int rot, int far) {
    const int rows = 40, heads = 2, kvh = 1, page = 8, wide = (heads + 2 * kvh) * hd;
    Pool pool(rows, page, rows, 1, kvh, hd, false, true);
    float *in = heap<float>((size_t)rows * wide), *out = heap<float>((size_t)rows * heads * hd);
    double *freq = heap<double>(rot / 2);
    int *pos = heap<int>(rows), *slots = heap<int>(rows);
    for (int i = 0; i < rows * wide; ++i) in[i] = urand(3.0f);
    for (int i = 0; i < rot / 2; ++i) freq[i] = std::pow(10000.0, -2.0 * i / rot);
    for (int t = 0; t < rows; ++t) { pos[t] = t < 3 ? t : t == 3 ? far : t == 4 ? -far : (int)(rng() % (unsigned)far); slots[t] = t % page; }
    const float mag = 1.2079441f;
    RopeArgs a{pool.view(), in, in + heads * hd, in + (heads + kvh) * hd, out, wide, wide, wide, heads * hd, freq, pos, slots, nullptr,
               heads, kvh, hd, rot, interleaved, 1, mag};
    emu::launch_grid([&] { k_rope_append<false, false, NP>(a); }, (unsigned)rows, ROPE_THREADS);
    int wrong = 0;
    long double most = 0.0;
    const long double half = 0x1p-24L;
    for (int t = 0; t < rows; ++t)
        for (int h = 0; h < heads + kvh; ++h)
            for (int i = 0; i < rot / 2; ++i) {
                const int e = interleaved ? 2 * i : i, o = interleaved ? 2 * i + 1 : i + rot / 2;
                const long double x = in[(size_t)t * wide + h * hd + e], y = in[(size_t)t * wide + h * hd + o], an = (long double)pos[t] * freq[i];
                const long double c = cosl(an) * mag, s = sinl(an) * mag;
                for (int d : {e, o}) {
                    const long double xc = d == e ? x * c : y * c, ys = d == e ? -y * s : x * s, want = xc + ys;
                    const long double got = h < heads ? out[((size_t)t * heads + h) * hd + d] : (long double)pool.get(pool.k, pool.index(pool.table[t], slots[t], 0, d));
                    const long double allowed = 2.01L * half * (fabsl(xc) + fabsl(ys)) + half * fabsl(want) + 1.5L * (fabsl(x) + fabsl(y)) * (fabsl(an) + 1) * 0x1p-53L;
                    most = fmaxl(most, fabsl(got - want) / allowed);
                    wrong += !(fabsl(got - want) <= allowed);
                }
            }
    std::printf("%s, positions to %d: off by up to %.3Lf of what the roundings allow\n", interleaved ? "interleaved" : "half layout", far, most);
    std::free(in); std::free(out); std::free(freq); std::free(pos); std::free(slots);
    return wrong;
}
static int rotation_roundings() {
    return rotation<4>(true, 128, 128, 1 << 11) + rotation<4>(false, 64, 64, 1 << 17) + rotation<1>(false, 64, 62, 1 << 20) + rotation<4>(true, 64, 64, 1 << 30);
}

int main(int argc, char **argv) {
    const struct { const char *name; int (*check)(); } checks[] = {{"rotation_roundings", rotation_roundings}};
    for (const auto &c : checks)
        if (argc > 1 && !std::strcmp(argv[1], c.name)) {
            const int wrong = c.check();
            std::printf("%s: %d wrong\n", c.name, wrong);
            return wrong ? 1 : 0;
        }
    return 2;
}
