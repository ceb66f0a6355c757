// A paged key-value cache for gfx950: rotary positions with the append of new rows, and attention of new tokens
// over the cached ones.  Page p of a pool holds 2^page_shift consecutive slots of one sequence; a sequence's slot s
// is slot s % page of page page_table[sequence][s / page].
#pragma once
#include "hipdec_common.h"

struct PagedView {           // hipdec_paged_cache as the kernels take it: strides in bytes
    char *k, *v;
    long long stride_page, stride_slot, stride_head;
    const int *table;        // [n_seqs][max_pages]
    int n_pages, page_shift, n_seqs, max_pages, kv_heads;
};

// page of a sequence's slot; -1 where the table names none of the pool's pages
__device__ __forceinline__ int pg_page(const PagedView &c, int seq, int slot) {
    const int p = c.table[(size_t)seq * c.max_pages + (slot >> c.page_shift)];
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}
__device__ __forceinline__ long long pg_offset(const PagedView &c, int page, int slot) {
    return (long long)page * c.stride_page + (long long)(slot & ((1 << c.page_shift) - 1)) * c.stride_slot;
}

// ---------------------------------------------------------------- rotary positions and the append
// Row t at position m: pair i of the first `rot` elements of every query and key head turns by the angle m * freq[i]
// (pair = elements (2i, 2i + 1), or (i, i + rot / 2) in the half layout), both results scaled by `magnitude`; the
// other elements and the values pass through.  Queries go to q_out, keys and values to the row's slot of the cache.
// The angle, its sine and cosine and their products with the magnitude are 64 bits wide (a position of a million in fp32
// is off by a tenth of a radian; an angle reduced in 64 bits and rounded to fp32 by 1.9e-7, more than the turn itself); both
// are rounded to fp32 once, the turn is fp32, and each result is rounded once, to its own type.
// Measured (MI355X): 8191 rows of 32 + 16 bf16 heads of 128 (201 MB) 40.6 us, 5.0 TB/s, as much as memory gives; 1024 fp32 rows of
// 32 + 64 heads into a bf16 cache 15.4 us; one row 2.9 us, a launch.  Pair by pair, where rot / 2 is no multiple of 4 or a stride is odd, a
// thread moves 2 or 4 bytes at a time: 65 and 20.7 us.
struct RopeArgs {
    PagedView c;
    const void *q, *k, *v;
    void *q_out;
    long long q_stride, k_stride, v_stride, out_stride;      // elements between rows
    const double *freq;
    const int *pos, *slots, *seqs;                           // slots / seqs may be null: the position / the row
    int heads, kv_heads, hd, rot, interleaved, parts;
    float magnitude;
};

template <bool B16> __device__ __forceinline__ float pg_get(const void *p, long long i) {
    return B16 ? bf16_to_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}
template <bool B16, int N> __device__ __forceinline__ void pg_get_n(const void *p, long long i, float *x) {
    if (N == 1) { x[0] = pg_get<B16>(p, i); return; }
    if (B16) {
        const uint2 u = *(const uint2 *)((const uint16_t *)p + i);
        x[0] = __uint_as_float(u.x << 16); x[1] = __uint_as_float(u.x & 0xffff0000u);
        x[2] = __uint_as_float(u.y << 16); x[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
        const float4 u = *(const float4 *)((const float *)p + i);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    }
}
template <bool B16, int N> __device__ __forceinline__ void pg_put_n(void *p, long long i, const float *x) {
    if (N == 1) {
        if (B16) ((uint16_t *)p)[i] = f32_to_bf16_rne(x[0]); else ((float *)p)[i] = x[0];
        return;
    }
    if (B16) {
        uint2 u;
        u.x = f32_to_bf16_rne(x[0]) | (uint32_t)f32_to_bf16_rne(x[1]) << 16;
        u.y = f32_to_bf16_rne(x[2]) | (uint32_t)f32_to_bf16_rne(x[3]) << 16;
        *(uint2 *)((uint16_t *)p + i) = u;
    } else {
        *(float4 *)((float *)p + i) = make_float4(x[0], x[1], x[2], x[3]);
    }
}

// Sine and cosine of `a`, times `by`, rounded once.  a less whole quarter turns n (pi / 2 in two parts, the products exact) lies within
// pi / 4 of 0, where the Taylor series end with errors of 9e-12 and 4e-13; n's last two bits say which is which, and the signs.
__device__ __forceinline__ void pg_sincos(double a, double by, float &sn, float &cs) {
    const double n = rint(a * 0.63661977236758134);
    const double r = fma(n, -6.123233995736766e-17, fma(n, -1.5707963267948966, a)), z = r * r;
    double s = -2.5052108385441720e-08, c = 2.0876756987868099e-09;
    s = fma(s, z, 2.7557319223985893e-06);
    s = fma(s, z, -1.9841269841269841e-04);
    s = fma(s, z, 8.3333333333333333e-03);
    s = fma(s, z, -1.6666666666666667e-01);
    s = fma(s * z, r, r);
    c = fma(c, z, -2.7557319223985888e-07);
    c = fma(c, z, 2.4801587301587302e-05);
    c = fma(c, z, -1.3888888888888889e-03);
    c = fma(c, z, 4.1666666666666664e-02);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int q = (int)(n - 4.0 * floor(0.25 * n));
    const double p = q & 1 ? c : s, o = q & 1 ? s : c;
    sn = (float)((q & 2 ? -p : p) * by);
    cs = (float)(((q + 1) & 2 ? -o : o) * by);
}

#define ROPE_THREADS 256
// One workgroup per row and part of its heads.  Its angles are worked out once, a thread each, and shared; a thread keeps one
// unit (NP pairs) of the head and walks the heads.  NP = 4 wherever the pieces are 4 aligned elements, else 1.
template <bool RB, bool CB, int NP> __global__ __launch_bounds__(ROPE_THREADS) void k_rope_append(RopeArgs a) {
    __shared__ float s_cs[ROPE_THREADS], s_sn[ROPE_THREADS]; // (rot / 2 <= 256)
    const int units = a.hd / (2 * NP), per_pass = ROPE_THREADS / units;
    const int u = threadIdx.x % units, hg = threadIdx.x / units;
    const int t = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int m = a.pos[t];
    if ((int)threadIdx.x < a.rot / 2) pg_sincos((double)m * a.freq[threadIdx.x], (double)a.magnitude, s_sn[threadIdx.x], s_cs[threadIdx.x]);
    const int seq = a.seqs ? a.seqs[t] : t, slot = a.slots ? a.slots[t] : m;
    // a row outside the cache (a padding row: slot < 0; a slot, sequence or page that does not exist) writes nothing
    long long at = -1;
    if ((unsigned)seq < (unsigned)a.c.n_seqs && slot >= 0 && (slot >> a.c.page_shift) < a.c.max_pages) {
        const int page = pg_page(a.c, seq, slot);
        if (page >= 0) at = pg_offset(a.c, page, slot);
    }
    __syncthreads();
    if (hg >= per_pass) return;
    const bool turned = u < a.rot / (2 * NP);
    float cs[NP], sn[NP];
    if (turned) {
#pragma unroll
        for (int i = 0; i < NP; ++i) { cs[i] = s_cs[u * NP + i]; sn[i] = s_sn[u * NP + i]; }
    }
    const bool half = turned && !a.interleaved;
    const int o0 = half ? NP * u : 2 * NP * u, o1 = half ? a.rot / 2 + NP * u : 2 * NP * u + NP;
    const int H = a.heads, KV = a.kv_heads;
    for (int h = part * per_pass + hg; h < H + 2 * KV; h += a.parts * per_pass) {
        const void *src = h < H ? a.q : h < H + KV ? a.k : a.v;
        const int hh = h < H ? h : h < H + KV ? h - H : h - H - KV;
        const long long from = (long long)t * (h < H ? a.q_stride : h < H + KV ? a.k_stride : a.v_stride) + (long long)hh * a.hd;
        if (h >= H && at < 0) continue;
        const bool turn = turned && h < H + KV;
        const int p0 = h < H + KV ? o0 : 2 * NP * u, p1 = h < H + KV ? o1 : 2 * NP * u + NP;
        float x[2 * NP], y[2 * NP];
        pg_get_n<RB, NP>(src, from + p0, x);
        pg_get_n<RB, NP>(src, from + p1, x + NP);
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i) y[i] = x[i];
        if (turn) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                if (half) {
                    y[i] = x[i] * cs[i] - x[NP + i] * sn[i];
                    y[NP + i] = x[NP + i] * cs[i] + x[i] * sn[i];
                } else {
                    y[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
                    y[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
                }
            }
        }
        if (h < H) {
            const long long to = (long long)t * a.out_stride + (long long)hh * a.hd;
            pg_put_n<RB, NP>(a.q_out, to + p0, y);
            pg_put_n<RB, NP>(a.q_out, to + p1, y + NP);
        } else {
            char *base = (h < H + KV ? a.c.k : a.c.v) + at + (long long)hh * a.c.stride_head;
            pg_put_n<CB, NP>(base, p0, y);
            pg_put_n<CB, NP>(base, p1, y + NP);
        }
    }
}

// ---------------------------------------------------------------- attention of new tokens over the cache
// out[row][h] = sum_s w_s v_s, w = softmax over s < len of scale * q[row][h] . k_s, for the g = heads / kv_heads
// query heads that share a key head at once, up to sixteen of them.  A row reads its sequence's cache once (once for every 16 heads of a
// key head), so with one row per sequence the bound is the cache's bytes over HBM's rate.  Rows of one sequence (a draft's) each read
// it for themselves: 8 sequences x 8 rows over 16384 slots, 32 heads over 8, take 346 us where 8 x 1 take 101.
//
// The tile is 16 keys x 16 query heads of the matrix instructions (columns past g idle).  Scores are computed
// transposed, S^T = K Q^T, so that lane l's result registers are the scores of head l % 16 with keys 4 (l / 16) + r:
// exactly what the second product, O^T = V^T P^T on the fp32 matrix instruction, wants as its operand, with V read
// in whole rows as it lies in the cache (lane l holds 16 bytes of key 4 (l / 16) + r, and element e of them is the
// operand of one instruction).  Probabilities never leave their registers, nothing is transposed, the running
// maximum and sum of a head sit in the lanes that hold its output, and P and V enter as fp32: a bf16 cache costs no
// precision beyond its own.  The fp32 instruction has room: 64 cached numbers per 32 clocks and SIMD are 32 bytes a
// clock and CU of a bf16 cache, three times what HBM delivers.  FEW: up to four heads per key head use the 4 x 4 form
// (16 independent blocks: four heads, the values of four dim groups and one of four keys), 64 numbers in 8 clocks; the
// columns of the score tile then repeat every four, and the four lane groups keep sums over keys of their own (64 ragged
// requests 220 -> 212 us together with the smaller blocks below).
//   K of a bf16 cache goes into the bf16 instruction as it is; fp32 queries are three bf16 numbers each (24 bits),
//   bf16 queries are one.  K of an fp32 cache uses the fp32 instruction.
// Measured (MI355X, listed sizes): 64 requests of 1 .. 8192 slots, 32 heads over 8, bf16 (1.09 GB): 211 us, 5.2 TB/s; one
// request of 65536: 54.4 us, 4.9 TB/s; 64 x 4096 evenly 5.5 TB/s; a large copy reaches 4.7.
struct PagedAttn {
    PagedView c;
    const void *q;
    void *out;
    long long q_stride, out_stride;                          // elements between rows
    const int *lens, *seqs;
    int heads, g, tiles, max_len, chunk, splits;
    float sc;                                                // scale * log2(e)
    float *part_o, *part_ml;                                 // splits > 1: [row][head][split][HD], [row][head][split][2]
};

typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 pg_bf8 __attribute__((ext_vector_type(8)));

// slots that row attends to; seq: its sequence (0 where there is none of that number: no slots then)
__device__ __forceinline__ int pg_len(const PagedAttn &a, int row, int &seq) {
    seq = a.seqs ? a.seqs[row] : row;
    const int n = a.lens[row];
    if ((unsigned)seq < (unsigned)a.c.n_seqs) return min(max(n, 0), a.max_len);
    seq = 0;
    return 0;
}

// The keys and values of one block of NT x 16 slots, in registers.  (Whole vectors per load: with the words of a load as
// single variables this compiler lets go of some of them while they are still to be read.)
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t pg_u2 __attribute__((ext_vector_type(2)));
template <int HD, bool CB, int NT> struct PagedTile {
    static constexpr int KQ = HD * (CB ? 2 : 4) / 64;        // 16-byte pieces of a key per lane (4 lanes a key)
    static constexpr int NE = HD / 16;                       // elements of a value per lane (16 lanes a value)
    static constexpr int VQ = (CB ? NE / 2 : NE) / 4;        // ... in 16-byte pieces
    static constexpr bool TAIL = CB && NE % 8;               // ... and one of 8 bytes
    pg_u4 k[NT][KQ], v[NT][4][VQ ? VQ : 1];
    pg_u2 tail[NT][4];
    // element e of key r's value as fp32
    __device__ __forceinline__ float value(int t, int r, int e) const {
        const int w = CB ? e / 2 : e;
        const uint32_t u = TAIL && w >= 4 * VQ ? tail[t][r][w % 4] : v[t][r][w / 4][w % 4];
        return __uint_as_float(!CB ? u : e % 2 ? u & 0xffff0000u : u << 16);
    }
};

// Registers: a key and its value of one tile take hd * 2 (4) bytes / 64 each, for 16 lanes; with 16 keys to a block and three
// workgroups a CU the other waves cover a wave's waits better than blocks of 32 keys with two (64 ragged requests 212
// against 220 us; a second register set with the next block's loads under way gains nothing: the same bytes in flight).
constexpr int att_tiles(int hd, bool cb) { return hd * (cb ? 2 : 4) <= 128 ? 2 : 1; }
constexpr int att_groups(int hd, bool cb) { return hd * (cb ? 2 : 4) <= 256 ? 3 : hd * (cb ? 2 : 4) <= 512 ? 2 : 1; }
template <int HD, bool QB, bool CB, bool FEW, int WAVES> __global__ __launch_bounds__(64 * WAVES, WAVES == 4 ? att_groups(HD, CB) : 1) void k_attn_paged(PagedAttn a) {
    constexpr int NT = att_tiles(HD, CB);                    // key tiles of a block
    constexpr int KEYS = 16 * NT;
    using Tile = PagedTile<HD, CB, NT>;
    constexpr int KQ = Tile::KQ, NE = Tile::NE, VQ = Tile::VQ;
    constexpr int PARTS = QB ? 1 : 3;
    constexpr int QN = CB ? KQ * PARTS : KQ;
    constexpr int CE = CB && WAVES == 4 ? 8 : 4;              // value elements joined at a time
    __shared__ __align__(16) float sm_o[WAVES * 16][CE * 16 + 4];
    __shared__ float sm_m[WAVES][16], sm_l[WAVES][16];

    // (rows and heads vary fastest: consecutive workgroups go to the eight XCDs in turn, and with the splits in front
    // the XCD that gets a row's last split would be idle wherever rows are shorter than max_len: 320 against 220 us)
    const unsigned per = gridDim.x / a.splits;               // rows x units
    const int split = blockIdx.x / per, rest = blockIdx.x % per;
    const int units = a.c.kv_heads * a.tiles, row = rest / units, unit = rest % units;
    const int kvh = unit / a.tiles, g0 = (unit % a.tiles) * 16, gn = min(16, a.g - g0), head0 = kvh * a.g + g0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), col = lane & 15, grp = lane >> 4;
    const int qcol = FEW ? col & 3 : col;                    // the query head that column `col` is
    int seq;
    const int len = pg_len(a, row, seq);
    const int lo = split * a.chunk, hi = min(len, lo + a.chunk);
    // the table's entry for the slot that is key `col` of each tile (asked for without waiting for the length)
    auto entry = [&](int b, int *pg) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int s = lo + b * KEYS + 16 * t + col;
            pg[t] = s < a.max_len ? a.c.table[(size_t)seq * a.c.max_pages + (s >> a.c.page_shift)] : -1;
        }
    };
    int pg[NT], nx[NT];
    entry(wave, pg);
    entry(wave + WAVES, nx);
    if (lo >= hi) {
        if (a.splits == 1)                                   // nothing to attend to: zeros
            for (int i = threadIdx.x; i < gn * HD; i += 64 * WAVES) {
                const long long at = (long long)row * a.out_stride + (long long)head0 * HD + i;
                if (QB) ((uint16_t *)a.out)[at] = 0; else ((float *)a.out)[at] = 0.0f;
            }
        return;
    }

    // queries: column `col` of the tile, the reduction elements that this lane's pieces of a key hold
    uint4 qr[QN];
    {
        const long long at = (long long)row * a.q_stride + (long long)(head0 + (qcol < gn ? qcol : 0)) * HD;
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            if (CB) {
                const long long i = at + 32 * j + 8 * grp;
                if (QB) {
                    qr[j] = *(const uint4 *)((const uint16_t *)a.q + i);
                } else {
                    const float4 x = *(const float4 *)((const float *)a.q + i), y = *(const float4 *)((const float *)a.q + i + 4);
                    float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                    // 24 bits in three parts of 8, each the upper half of what is left: exact.  (An infinity leaves NaN in
                    // the second part, as its scores would in the softmax.)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = __builtin_amdgcn_perm(__float_as_uint(f[2 * e + 1]), __float_as_uint(f[2 * e]), 0x07060302u);
                            f[2 * e] -= __uint_as_float(w[e] << 16);
                            f[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
                        }
                        qr[p * KQ + j] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            } else {
                const long long i = at + 16 * j + 4 * grp;
                if (QB) {
                    const uint2 b = *(const uint2 *)((const uint16_t *)a.q + i);
                    qr[j] = make_uint4(b.x << 16, b.x & 0xffff0000u, b.y << 16, b.y & 0xffff0000u);
                } else {
                    qr[j] = *(const uint4 *)((const float *)a.q + i);
                }
            }
        }
        if (qcol >= gn)
#pragma unroll
            for (int j = 0; j < QN; ++j) qr[j] = make_uint4(0, 0, 0, 0);
    }

    const char *kb = a.c.k + (long long)kvh * a.c.stride_head + 16 * grp, *vb = a.c.v + (long long)kvh * a.c.stride_head;
    // entries to pages; -1: past the end, or without a page.  What is read for such a slot lies in page 0 and does
    // not count: its score becomes -inf and its value zero (it may hold a NaN).
    auto pages = [&](int b, int *pg) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (lo + b * KEYS + 16 * t + col >= hi || (unsigned)pg[t] >= (unsigned)a.c.n_pages) pg[t] = -1;
    };
    auto load_k = [&](int b, const int *pg, Tile &x) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int s = lo + b * KEYS + 16 * t + col;
            const char *p = kb + pg_offset(a.c, max(pg[t], 0), s);
#pragma unroll
            for (int j = 0; j < KQ; ++j) x.k[t][j] = *(const pg_u4 *)(p + 64 * j);
        }
    };
    auto load_v = [&](int b, const int *pg, Tile &x) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int s = lo + b * KEYS + 16 * t + 4 * grp + r;
                const int page = __shfl(pg[t], 4 * grp + r, WAVE);
                const char *p = vb + pg_offset(a.c, max(page, 0), s);
#pragma unroll
                for (int c = 0; c < VQ; ++c) x.v[t][r][c] = *(const pg_u4 *)(p + 256 * c + 16 * col);
                if (Tile::TAIL) x.tail[t][r] = *(const pg_u2 *)(p + 256 * VQ + 8 * col);
            }
    };

    pg_f4 acc[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) acc[e] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;                           // of head `col`: m the same in its four lanes, l each lane's own share
    const int blocks = (hi - lo + KEYS - 1) / KEYS;
    Tile x = {};
    int b = wave;
    if (b < blocks) {
        pages(b, pg);
        load_k(b, pg, x);
        load_v(b, pg, x);
        pages(b + WAVES, nx);
    }
    while (b < blocks) {
        pg_f4 s[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            // sums of their own for each part of the queries (fp32 cache: two): short chains, and the small ones added first
            pg_f4 sum[3] = {};
#pragma unroll
            for (int j = 0; j < KQ; ++j) {
                if (CB) {
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        sum[p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf8, x.k[t][j]),
                                                                         __builtin_bit_cast(pg_bf8, qr[p * KQ + j]), sum[p], 0, 0, 0);
                } else {
                    const pg_u4 kw = x.k[t][j];
                    const uint32_t qw[4] = {qr[j].x, qr[j].y, qr[j].z, qr[j].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sum[e % 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e]), __uint_as_float(qw[e]), sum[e % 2], 0, 0, 0);
                }
            }
            s[t] = CB && PARTS == 1 ? sum[0] : CB ? sum[0] + (sum[1] + sum[2]) : sum[0] + sum[1];
        }
        const bool more = b + WAVES < blocks;
        bool gaps = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) gaps |= __ballot(pg[t] < 0) != 0;
        if (more) load_k(b + WAVES, nx, x);
        if (gaps)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (__shfl(pg[t], 4 * grp + r, WAVE) < 0) s[t][r] = -INFINITY;
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
        top = fmaxf(top, __shfl_xor(top, 16, WAVE));
        top = fmaxf(top, __shfl_xor(top, 32, WAVE));
        const float mn = fmaxf(m, top * a.sc);
        const float ms = mn == -INFINITY ? 0.0f : mn;        // a head without a key so far: every weight is exp2(-inf) = 0
        const float fall = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        l *= fall;
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[e] *= fall;
        float p[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.sc, -ms));
                l += p[t][r];
            }
        if (gaps)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (__shfl(pg[t], 4 * grp + r, WAVE) < 0) {
#pragma unroll
                        for (int c = 0; c < VQ; ++c) x.v[t][r][c] = pg_u4{0, 0, 0, 0};
                        x.tail[t][r] = pg_u2{0, 0};
                    }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    const float f = x.value(t, r, e);
                    if (FEW) acc[e] = __builtin_amdgcn_mfma_f32_4x4x1f32(f, p[t][r], acc[e], 0, 0, 0);
                    else acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(f, p[t][r], acc[e], 0, 0, 0);
                }
        if (!more) break;
        b += WAVES;
        load_v(b, nx, x);
#pragma unroll
        for (int t = 0; t < NT; ++t) pg[t] = nx[t];
        entry(b + WAVES, nx);
        pages(b + WAVES, nx);
    }

    // the waves' shares joined in LDS and summed in a fixed order, up to 8 elements of each lane (128 dims) at a time.
    // Result row m of element e is dim m * ce + e - e0 of that part; with few heads a wave's four lane groups hold
    // sums over keys of their own, which are shares like those of the waves.
    constexpr int HEADS = FEW ? 4 : 16, SHARES = 16 * WAVES / HEADS;
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    if (lane < HEADS) { sm_m[wave][lane] = m; sm_l[wave][lane] = l; }
    const int row0 = FEW ? 4 * ((lane >> 2) & 3) : 4 * grp;
    const int mine = FEW ? (4 * wave + grp) * HEADS + qcol : wave * HEADS + col;
    float M = -INFINITY, L = 0.0f, wt[WAVES];
#pragma unroll
    for (int e0 = 0; e0 < NE; e0 += NE - e0 >= CE ? CE : 4) {
        const int ce = NE - e0 >= CE ? CE : 4;               // 16 * ce dims of every head: 4 a thread, in rounds
        const bool halves = CB && ce == 4 && e0 < NE / 8 * 8;    // of a piece of 8 elements: 4 dims of every 8
        if (e0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < ce; e += 4)
                *(float4 *)&sm_o[mine][(row0 + r) * ce + e] =
                    make_float4(acc[e0 + e][r], acc[e0 + e + 1][r], acc[e0 + e + 2][r], acc[e0 + e + 3][r]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (HEADS * 4 * ce + 64 * WAVES - 1) / (64 * WAVES); ++i) {
            const int at = i * 64 * WAVES + (int)threadIdx.x, head = at / (4 * ce), d = at % (4 * ce) * 4;
            const int dim = halves ? 16 * (e0 & ~7) + 2 * d + (e0 & 7) : 16 * e0 + d;
            if (head >= gn) continue;
            M = -INFINITY; L = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) M = fmaxf(M, sm_m[w][head]);
            const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) { wt[w] = __builtin_amdgcn_exp2f(sm_m[w][head] - ms); L = fmaf(wt[w], sm_l[w][head], L); }
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < SHARES; ++k) {
                const float4 x = *(const float4 *)&sm_o[k * HEADS + head][d];
                const float w = wt[FEW ? k / 4 : k];
                o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
            }
            if (a.splits == 1) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
                pg_put_n<QB, 4>(a.out, (long long)row * a.out_stride + (long long)(head0 + head) * HD + dim, y);
            } else {
                const size_t slot = ((size_t)row * a.heads + head0 + head) * a.splits + split;
                *(float4 *)(a.part_o + slot * HD + dim) = o;
                if (e0 == 0 && d == 0) *(float2 *)(a.part_ml + 2 * slot) = make_float2(M, L);
            }
        }
    }
}

// The splits of one row and head joined, in the order of the cache within each group of threads.
template <int HD, bool QB> __global__ __launch_bounds__(256) void k_attn_paged_join(PagedAttn a) {
    constexpr int W = HD / 4, G = 256 / W;                   // threads across a head, groups that take every G-th split
    __shared__ __align__(16) float sm[G][HD];
    __shared__ float sm_l[G], sm_top[4];
    const int row = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
    int seq;
    const int len = pg_len(a, row, seq);
    const int n = (len + a.chunk - 1) / a.chunk;
    const size_t slot0 = ((size_t)row * a.heads + h) * a.splits;
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += 256) top = fmaxf(top, a.part_ml[2 * (slot0 + i)]);
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) sm_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sm_top[0], sm_top[1]), fmaxf(sm_top[2], sm_top[3]));
    if (top == -INFINITY) top = 0.0f;
    const int grp = threadIdx.x / W, d = (threadIdx.x % W) * 4;
    if (grp < G) {
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (int i = grp; i < n; i += G) {
            const float2 ml = *(const float2 *)(a.part_ml + 2 * (slot0 + i));
            const float4 x = *(const float4 *)(a.part_o + (slot0 + i) * HD + d);
            const float w = __builtin_amdgcn_exp2f(ml.x - top);
            l = fmaf(w, ml.y, l);
            o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
        }
        *(float4 *)&sm[grp][d] = o;
        if (d == 0) sm_l[grp] = l;
    }
    __syncthreads();
    if (grp == 0) {
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
#pragma unroll
        for (int k = 0; k < G; ++k) {
            l += sm_l[k];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += sm[k][d + e];
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= inv;
        pg_put_n<QB, 4>(a.out, (long long)row * a.out_stride + (long long)h * HD + d, y);
    }
}
