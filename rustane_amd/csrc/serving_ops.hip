// The C entries of the operators on the caller's device buffers (include/hip_decode.h): argument checks, the choice
// of kernel and launch.  Nothing here allocates, waits or keeps state between calls.
#include "../../include/hip_decode.h"
#include "hipdec_paged.h"
#include "hipdec_verify.h"

#include <math.h>
#include <stdio.h>

// hip_decode.hip: sets the text hipdec_last_error(NULL) returns on this thread
extern "C" __attribute__((visibility("hidden"))) int hipdec_op_error(int code, const char *entry, const char *what);

namespace {

constexpr uint32_t kMaxPage = 65536, kMaxHeadDim = 512, kMaxVocab = 262144, kMaxDrafts = 255;
constexpr uint64_t kMaxRows = 1u << 24, kMaxLen = 1u << 30;
constexpr int kCus = 256;                                    // compute units of the one device this is built for

int refuse(const char *entry, const char *what) { return hipdec_op_error(HIPDEC_ERR_ARG, entry, what); }
int launched(const char *entry, hipError_t e) {
    if (e == hipSuccess) return HIPDEC_OK;
    (void)hipGetLastError();
    return hipdec_op_error(HIPDEC_ERR_HIP, entry, hipGetErrorString(e));
}
// The caller's stream; the handle that names the default one is that.
hipStream_t stream_of(void *stream) { return stream == (void *)hipStreamLegacy ? nullptr : (hipStream_t)stream; }
// A launch with its own error, not whatever an earlier call of the program has left behind.
template <typename A> hipError_t start(void (*kernel)(A), uint64_t grid, int threads, hipStream_t s, const A &a) {
    void *args[] = {(void *)&a};
    return hipLaunchKernel((const void *)kernel, dim3((unsigned)grid), dim3((unsigned)threads), args, 0, s);
}

// (a grid's threads are counted in 32 bits; every launch of a call is looked at before its first)
bool grid_fits(uint64_t groups, uint64_t threads) { return groups <= 0x7fffffffu && groups * threads <= 0xffffffffu; }

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Whether `p` is memory that kernels of the current device may use, and `stream` one of its streams: a host pointer,
// or a buffer of another device, would end the process inside a kernel.
const char *wrong_place(std::initializer_list<const void *> buffers, void *stream) {
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) { (void)hipGetLastError(); return "no current device"; }
    if (stream && stream != (void *)hipStreamPerThread) {    // (that one is the current device's, and no object to be asked)
        hipDevice_t of = -1;
        if (hipStreamGetDevice((hipStream_t)stream, &of) != hipSuccess) { (void)hipGetLastError(); return "not a stream"; }
        if ((int)of != dev) return "the stream is of another device than the current one";
    }
    for (const void *p : buffers) {
        if (!p) continue;
        hipPointerAttribute_t at{};
        if (hipPointerGetAttributes(&at, p) != hipSuccess) { (void)hipGetLastError(); return "a buffer is not device memory"; }
        if (at.type == hipMemoryTypeDevice ? at.device != dev : at.type != hipMemoryTypeManaged && at.type != hipMemoryTypeHost)
            return at.type == hipMemoryTypeDevice ? "a buffer is of another device than the current one" : "a buffer is not device memory";
    }
    return nullptr;
}

const char *check_cache(const hipdec_paged_cache *c) {
    if (!c->k || !c->v || !c->page_table) return "null buffer in the cache";
    if (c->kv_dtype > HIPDEC_KV_BF16) return "unknown kv_dtype";
    if (!c->n_pages || !c->kv_heads || !c->hd || !c->n_seqs || !c->max_pages) return "zero-sized cache";
    if (c->n_pages > 0x7fffffffu || c->n_seqs > kMaxRows || c->max_pages > 0x7fffffffu || c->kv_heads > 65536) return "cache too large";
    if (!c->page_size || (c->page_size & (c->page_size - 1)) || c->page_size > kMaxPage) return "page_size must be a power of two up to 65536";
    if (c->stride_page < 0 || c->stride_slot < 0 || c->stride_head < 0) return "negative stride";
    return nullptr;
}

PagedView view(const hipdec_paged_cache &c) {
    const long long e = c.kv_dtype == HIPDEC_KV_BF16 ? 2 : 4;
    PagedView v{(char *)c.k, (char *)c.v, c.stride_page * e, c.stride_slot * e, c.stride_head * e, c.page_table,
                (int)c.n_pages, 0, (int)c.n_seqs, (int)c.max_pages, (int)c.kv_heads};
    while ((1u << v.page_shift) < c.page_size) ++v.page_shift;
    return v;
}

// How the cache's length is split: keys per split (whole steps of 128, what the four waves of a workgroup take twice
// each) and splits; one split means one launch of eight-wave workgroups that write the result themselves.
//   * One workgroup per row and key head where the length is at most 256 (a step per wave; 8.9 us against 10.9 with the
//     second launch), and up to 1024 where there are enough of them for most CUs (256 workgroups: 400 keys 13.4 us
//     against 15.7).  Longer, it would win 4 % where all rows are equally long (64 x 8 heads of 4096: 185 us against
//     194), but the longest row alone sets the end where they are not (16 rows of up to 16384: 243 us against 121), and
//     the lengths are known on the device only.
//   * Else two workgroups a CU, with at most 1024 keys each: fewer leave CUs idle, more pay in the latency each starts
//     with (one request of 65536: 54.7 us, with four 59), longer ones end unevenly.
struct Split { int chunk, splits; };
Split split_of(uint64_t n_rows, uint32_t kv_heads, uint32_t g, uint64_t max_len) {
    const uint64_t units = n_rows * kv_heads * ((g + 15) / 16), steps = (max_len + 127) / 128;
    if (max_len <= 256 || (units >= 192 && max_len <= 1024)) return Split{(int)(steps ? steps : 1) * 128, 1};
    const uint64_t want = units ? (2 * kCus + units - 1) / units : 1;
    uint64_t per = (steps + want - 1) / want;
    if (per > 8) per = 8;
    return Split{(int)per * 128, (int)((steps + per - 1) / per)};
}

// Workspace for n_rows rows and max_len, and for anything smaller in either: with u key-head tiles per row, rows * splits
// is at most rows * steps / 8 where the 1024 keys decide, and rows * (2 CUs / (rows u) + 1) where the CUs do.  (No call whose
// launches fit comes near 64 bits; the largest sizes that can be asked for pass them.)
unsigned __int128 attention_bytes(uint64_t n_rows, uint32_t heads, uint32_t kv_heads, uint32_t hd, uint64_t max_len) {
    if (max_len <= 256 || !n_rows) return 0;
    const uint64_t u = (uint64_t)kv_heads * ((heads / kv_heads + 15) / 16), steps = (max_len + 127) / 128;
    uint64_t most = n_rows * ((steps + 7) / 8);
    const uint64_t by_cus = (2 * kCus + u - 1) / u + n_rows;
    if (most < by_cus) most = by_cus;
    if (most > n_rows * steps) most = n_rows * steps;
    return (unsigned __int128)(most * heads) * (hd + 2) * sizeof(float);
}

// Waves of a workgroup where one split writes the result (eight of the widest fp32 heads would not keep their registers).
constexpr int wide_waves(uint32_t hd, bool cb) { return hd * (cb ? 2 : 4) <= 512 ? 8 : 4; }
template <int HD, bool QB, bool CB, bool FEW> hipError_t go_attention(const PagedAttn &a, uint64_t grid, uint64_t joins, hipStream_t s) {
    constexpr int WIDE = wide_waves(HD, CB);
    if (a.splits == 1) return start(k_attn_paged<HD, QB, CB, FEW, WIDE>, grid, 64 * WIDE, s, a);
    const hipError_t e = start(k_attn_paged<HD, QB, CB, FEW, 4>, grid, 256, s, a);
    return e != hipSuccess ? e : start(k_attn_paged_join<HD, QB>, joins, 256, s, a);
}
template <int HD, bool QB, bool CB> hipError_t go_attention(const PagedAttn &a, uint64_t grid, uint64_t joins, hipStream_t s) {
    return a.g <= 4 ? go_attention<HD, QB, CB, true>(a, grid, joins, s) : go_attention<HD, QB, CB, false>(a, grid, joins, s);
}
template <int HD> hipError_t go_attention(bool qb, bool cb, const PagedAttn &a, uint64_t grid, uint64_t joins, hipStream_t s) {
    if (qb) return cb ? go_attention<HD, true, true>(a, grid, joins, s) : go_attention<HD, true, false>(a, grid, joins, s);
    return cb ? go_attention<HD, false, true>(a, grid, joins, s) : go_attention<HD, false, false>(a, grid, joins, s);
}

template <bool RB, bool CB> hipError_t go_rope(const RopeArgs &a, bool wide, uint64_t grid, hipStream_t s) {
    return wide ? start(k_rope_append<RB, CB, 4>, grid, ROPE_THREADS, s, a) : start(k_rope_append<RB, CB, 1>, grid, ROPE_THREADS, s, a);
}

// Logits of a row per wave: 256, 512 or 1024.  Few logits are latency, many are instructions, of which a chunk's maximum
// and sum, and reading its statistics back, are a smaller part the more logits it has: 20 rows of 32768 13.3 / 13.2 / 14.0 us, 160 rows
// 17.5 / 16.7 / 18.1, 320 rows 27.6 / 23.1 / 22.9, 512 rows 36.1 / 30.1 / 30.3, 256 rows of 131071 - / 56.6 / 52.3 (so 512 and 1024 are
// level from 10 to 17 million logits, and the border lies there).  At most 256 chunks.
struct Chunks { int per, n; };
Chunks chunks_of(uint64_t rows, uint32_t vocab) {
    const uint64_t logits = rows * vocab;
    int per = logits <= (4u << 20) ? 4 : logits <= (12u << 20) ? 8 : 16;
    while ((vocab + per * WAVE - 1) / (per * WAVE) > VF_MAX_CHUNKS) per *= 2;
    return Chunks{per, (int)((vocab + per * WAVE - 1) / (per * WAVE))};
}
uint64_t verify_bytes(uint64_t n_seqs, uint32_t max_drafts, int chunks) {
    return n_seqs * ((max_drafts + 1) * chunks * sizeof(VfStat) + chunks * sizeof(double) + sizeof(VfPlace));
}

// Workgroups of the statistics and of the decision.
struct VerifyGrids { uint64_t stats, decide; };
VerifyGrids verify_grids(uint64_t n_seqs, uint32_t max_drafts, int chunks, bool greedy) {
    const int few = (chunks + VF_STATS / WAVE - 1) / (VF_STATS / WAVE), more = (chunks + VF_DECIDE / WAVE - 1) / (VF_DECIDE / WAVE);
    return VerifyGrids{n_seqs * (max_drafts + 1) * few, greedy ? n_seqs : n_seqs * more};
}

template <bool B16, bool CAP, int PER> hipError_t go_verify(const VerifyArgs &a, hipStream_t s) {
    const VerifyGrids g = verify_grids(a.n_seqs, a.max_drafts, a.chunks, !(a.k > 0.0));
    hipError_t e = start(k_verify_stats<B16, CAP, PER>, g.stats, VF_STATS, s, a);
    if (e == hipSuccess) e = start(k_verify_decide<B16, CAP, PER>, g.decide, VF_DECIDE, s, a);
    if (e == hipSuccess && a.k > 0.0) e = start(k_verify_draw<B16, CAP, PER>, (uint64_t)a.n_seqs, WAVE, s, a);
    return e;
}
template <bool B16> hipError_t go_verify(const VerifyArgs &a, int per, hipStream_t s) {
    if (a.cap > 0.0) return per == 4 ? go_verify<B16, true, 4>(a, s) : per == 8 ? go_verify<B16, true, 8>(a, s) : go_verify<B16, true, 16>(a, s);
    return per == 4 ? go_verify<B16, false, 4>(a, s) : per == 8 ? go_verify<B16, false, 8>(a, s) : go_verify<B16, false, 16>(a, s);
}

}  // namespace

extern "C" {

int hipdec_rope_frequencies(uint32_t scaling, uint32_t rot_dim, double theta, double factor, double trained,
                            double slow_turns, double fast_turns, double *freq, float *magnitude) {
    const char *me = "hipdec_rope_frequencies";
    if (!freq || !magnitude) return refuse(me, "null buffer");
    if (scaling > HIPDEC_ROPE_PARTS) return refuse(me, "unknown scaling");
    if (rot_dim == 0 || rot_dim % 2 || rot_dim > kMaxHeadDim) return refuse(me, "rot_dim must be even, 2 .. 512");
    if (!(theta > 1.0) || !isfinite(theta)) return refuse(me, "theta must be above 1");
    if (scaling != HIPDEC_ROPE_PLAIN && (!(factor >= 1.0) || !isfinite(factor))) return refuse(me, "factor must be at least 1");
    if (scaling == HIPDEC_ROPE_BASE && rot_dim == 2) return refuse(me, "one pair cannot be scaled by its base");
    if (scaling == HIPDEC_ROPE_PARTS && (!(trained > 0.0) || !isfinite(trained) || !(slow_turns >= 0.0) || !(fast_turns > slow_turns) || !isfinite(fast_turns)))
        return refuse(me, "trained must be above 0 and fast_turns above slow_turns, which is not negative");
    if (scaling == HIPDEC_ROPE_BASE) theta *= pow(factor, (double)rot_dim / (rot_dim - 2));
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
        double f = pow(theta, -2.0 * i / rot_dim);
        if (scaling == HIPDEC_ROPE_LINEAR) f /= factor;
        if (scaling == HIPDEC_ROPE_PARTS) {
            const double turns = trained * f / 6.283185307179586477;
            const double keep = fmin(fmax((turns - slow_turns) / (fast_turns - slow_turns), 0.0), 1.0);
            f = f * keep + f / factor * (1.0 - keep);
        }
        freq[i] = f;
    }
    *magnitude = scaling == HIPDEC_ROPE_PARTS ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    return HIPDEC_OK;
}

int hipdec_rope_append_paged(const hipdec_rope *rope, const hipdec_paged_cache *cache, const hipdec_new_rows *rows,
                             void *stream) {
    const char *me = "hipdec_rope_append_paged", *bad;
    if (!rope || !cache || !rows) return refuse(me, "null argument");
    if ((bad = check_cache(cache))) return refuse(me, bad);
    if (rows->n_rows == 0) return HIPDEC_OK;
    if (!rows->d_q || !rows->d_k || !rows->d_v || !rows->d_q_out || !rows->d_positions || (rope->rot_dim && !rope->d_freq))
        return refuse(me, "null buffer");
    if (rows->dtype > HIPDEC_ROWS_BF16) return refuse(me, "unknown dtype");
    if (!rows->heads || rows->heads > 65536 || rows->n_rows > kMaxRows) return refuse(me, "heads or n_rows out of range");
    if (cache->hd % 2 || cache->hd > kMaxHeadDim) return refuse(me, "hd must be even, up to 512");
    if (rope->rot_dim % 2 || rope->rot_dim > cache->hd) return refuse(me, "rot_dim must be even, up to hd");
    if (!isfinite(rope->magnitude)) return refuse(me, "magnitude must be finite");
    const int64_t wide_q = (int64_t)rows->heads * cache->hd, wide_k = (int64_t)cache->kv_heads * cache->hd;
    if (rows->n_rows > 1 && (rows->q_stride < wide_q || rows->q_out_stride < wide_q || rows->k_stride < wide_k || rows->v_stride < wide_k))
        return refuse(me, "rows overlap: a stride is smaller than its row");
    if (rows->d_q == rows->d_q_out && rows->q_stride != rows->q_out_stride) return refuse(me, "in place, both strides must be equal");
    if ((bad = wrong_place({rows->d_q, rows->d_k, rows->d_v, rows->d_q_out, rows->d_positions, rows->d_slots, rows->d_seqs, rope->d_freq,
                            cache->k, cache->v, cache->page_table}, stream_of(stream))))
        return refuse(me, bad);

    RopeArgs a{view(*cache), rows->d_q, rows->d_k, rows->d_v, rows->d_q_out, rows->q_stride, rows->k_stride, rows->v_stride,
               rows->q_out_stride, rope->d_freq, rows->d_positions, rows->d_slots, rows->d_seqs, (int)rows->heads,
               (int)cache->kv_heads, (int)cache->hd, (int)rope->rot_dim, rope->interleaved != 0, 1, rope->magnitude};
    const int64_t strides = rows->q_stride | rows->k_stride | rows->v_stride | rows->q_out_stride | cache->stride_page |
                            cache->stride_slot | cache->stride_head;
    const bool wide = cache->hd % 8 == 0 && rope->rot_dim % 8 == 0 && strides % 4 == 0 && aligned16(rows->d_q) && aligned16(rows->d_k) &&
                      aligned16(rows->d_v) && aligned16(rows->d_q_out) && aligned16(cache->k) && aligned16(cache->v);
    // few rows: a workgroup for every pass over the heads, so that one token's heads run side by side
    const int per_pass = ROPE_THREADS / (int)(cache->hd / (wide ? 8 : 2));
    const int passes = (a.heads + 2 * a.kv_heads + per_pass - 1) / per_pass;
    a.parts = rows->n_rows * passes <= 4 * kCus ? passes : 1;
    const uint64_t grid = rows->n_rows * a.parts;
    if (!grid_fits(grid, ROPE_THREADS)) return refuse(me, "n_rows out of range");
    const bool rb = rows->dtype == HIPDEC_ROWS_BF16, cb = cache->kv_dtype == HIPDEC_KV_BF16;
    hipStream_t s = stream_of(stream);
    if (rb) return launched(me, cb ? go_rope<true, true>(a, wide, grid, s) : go_rope<true, false>(a, wide, grid, s));
    return launched(me, cb ? go_rope<false, true>(a, wide, grid, s) : go_rope<false, false>(a, wide, grid, s));
}

int hipdec_attention_paged_workspace(uint64_t n_rows, uint32_t heads, uint32_t kv_heads, uint32_t hd, uint64_t max_len,
                                     uint64_t *out_bytes) {
    const char *me = "hipdec_attention_paged_workspace";
    if (!out_bytes) return refuse(me, "null argument");
    if (!heads || !kv_heads || heads % kv_heads || heads > 65536 || hd > kMaxHeadDim || n_rows > kMaxRows || max_len > kMaxLen)
        return refuse(me, "heads, hd, n_rows or max_len out of range");
    const unsigned __int128 bytes = attention_bytes(n_rows, heads, kv_heads, hd, max_len);
    if (bytes >> 64) return refuse(me, "n_rows * heads * max_len out of range");
    *out_bytes = (uint64_t)bytes;
    return HIPDEC_OK;
}

int hipdec_attention_paged(const hipdec_paged_cache *cache, const hipdec_attention_rows *rows, void *d_workspace,
                           uint64_t workspace_bytes, void *stream) {
    const char *me = "hipdec_attention_paged", *bad;
    if (!cache || !rows) return refuse(me, "null argument");
    if ((bad = check_cache(cache))) return refuse(me, bad);
    if (rows->n_rows == 0) return HIPDEC_OK;
    if (!rows->d_q || !rows->d_out || !rows->d_lens) return refuse(me, "null buffer");
    if (rows->dtype > HIPDEC_ROWS_BF16) return refuse(me, "unknown dtype");
    if (!rows->heads || rows->heads % cache->kv_heads || rows->heads > 65536) return refuse(me, "heads must be a multiple of the cache's kv_heads");
    if (rows->n_rows > kMaxRows || rows->max_len > kMaxLen) return refuse(me, "n_rows or max_len out of range");
    if (!(rows->scale > 0.0f) || !isfinite(rows->scale * 1.44269504088896340736f)) return refuse(me, "scale must be above 0");
    if (cache->hd != 64 && cache->hd != 128 && cache->hd != 192 && cache->hd != 256)
        return hipdec_op_error(HIPDEC_ERR_UNSUPPORTED, me, "head dim must be 64, 128, 192 or 256");
    const int64_t wide = (int64_t)rows->heads * cache->hd;
    if (rows->n_rows > 1 && (rows->q_stride < wide || rows->out_stride < wide)) return refuse(me, "rows overlap: a stride is smaller than its row");
    const int64_t row_unit = rows->dtype == HIPDEC_ROWS_BF16 ? 8 : 4, kv_unit = cache->kv_dtype == HIPDEC_KV_BF16 ? 8 : 4;
    if (!aligned16(rows->d_q) || !aligned16(rows->d_out) || !aligned16(cache->k) || !aligned16(cache->v) ||
        (rows->q_stride | rows->out_stride) % row_unit || (cache->stride_page | cache->stride_slot | cache->stride_head) % kv_unit)
        return refuse(me, "queries, outputs and the cache must be 16-byte aligned, with strides of whole 16 bytes");
    if (rows->n_rows > 1 && rows->d_q == rows->d_out && rows->q_stride != rows->out_stride) return refuse(me, "in place, both strides must be equal");

    const uint64_t slots = (uint64_t)cache->max_pages * cache->page_size;
    const bool qb = rows->dtype == HIPDEC_ROWS_BF16, cb = cache->kv_dtype == HIPDEC_KV_BF16;
    const int g = (int)(rows->heads / cache->kv_heads), tiles = (g + 15) / 16;
    const Split p = split_of(rows->n_rows, cache->kv_heads, (uint32_t)g, rows->max_len);
    const uint64_t grid = rows->n_rows * cache->kv_heads * tiles * p.splits, joins = rows->n_rows * rows->heads;
    if (!grid_fits(grid, p.splits == 1 ? 64 * wide_waves(cache->hd, cb) : 256) || (p.splits > 1 && !grid_fits(joins, 256)))
        return refuse(me, "n_rows * heads * max_len out of range");
    const uint64_t need = p.splits == 1 ? 0 : rows->n_rows * rows->heads * p.splits * (cache->hd + 2) * sizeof(float);
    if (need && (!d_workspace || workspace_bytes < need || !aligned16(d_workspace)))
        return refuse(me, "workspace missing, too small (hipdec_attention_paged_workspace) or not 16-byte aligned");
    if ((bad = wrong_place({rows->d_q, rows->d_out, rows->d_lens, rows->d_seqs, cache->k, cache->v, cache->page_table,
                            need ? d_workspace : nullptr}, stream_of(stream))))
        return refuse(me, bad);

    float *po = (float *)d_workspace;
    PagedAttn a{view(*cache), rows->d_q, rows->d_out, rows->q_stride, rows->out_stride, rows->d_lens, rows->d_seqs, (int)rows->heads,
                g, tiles, (int)(rows->max_len < slots ? rows->max_len : slots), p.chunk, p.splits,
                rows->scale * 1.44269504088896340736f, po, po + rows->n_rows * rows->heads * p.splits * cache->hd};
    hipStream_t s = stream_of(stream);
    switch (cache->hd) {
    case 64: return launched(me, go_attention<64>(qb, cb, a, grid, joins, s));
    case 128: return launched(me, go_attention<128>(qb, cb, a, grid, joins, s));
    case 192: return launched(me, go_attention<192>(qb, cb, a, grid, joins, s));
    default: return launched(me, go_attention<256>(qb, cb, a, grid, joins, s));
    }
}

int hipdec_verify_drafts_workspace(uint64_t n_seqs, uint32_t max_drafts, uint32_t vocab, uint64_t *out_bytes) {
    const char *me = "hipdec_verify_drafts_workspace";
    if (!out_bytes) return refuse(me, "null argument");
    if (max_drafts > kMaxDrafts || n_seqs > kMaxRows || !vocab || vocab > kMaxVocab) return refuse(me, "n_seqs, max_drafts or vocab out of range");
    // (the most chunks any smaller call makes of a row)
    const uint32_t chunks = (vocab + 4 * WAVE - 1) / (4 * WAVE);
    *out_bytes = verify_bytes(n_seqs, max_drafts, (int)(chunks < VF_MAX_CHUNKS ? chunks : VF_MAX_CHUNKS));
    return HIPDEC_OK;
}

int hipdec_verify_drafts(const hipdec_drafts *d, void *d_workspace, uint64_t workspace_bytes, void *stream) {
    const char *me = "hipdec_verify_drafts", *bad;
    if (!d) return refuse(me, "null argument");
    if (d->n_seqs == 0) return HIPDEC_OK;
    const bool greedy = d->temperature == 0.0f;
    if (!d->d_logits || !d->d_tokens || !d->d_accepted || (d->max_drafts && !d->d_drafts) || (!greedy && !d->d_uniforms))
        return refuse(me, "null buffer");
    if (d->dtype > HIPDEC_ROWS_BF16) return refuse(me, "unknown dtype");
    if (!(d->temperature >= 0.0f) || !isfinite(d->temperature)) return refuse(me, "temperature must not be negative");
    if (!(d->softcap <= 3.4e38f)) return refuse(me, "softcap must be finite");
    if (d->max_drafts > kMaxDrafts || d->n_seqs > kMaxRows || !d->vocab || d->vocab > kMaxVocab)
        return refuse(me, "n_seqs, max_drafts or vocab out of range");
    if (d->row_stride < d->vocab || (d->d_draft_probs && d->max_drafts && d->prob_stride < d->vocab))
        return refuse(me, "rows overlap: a stride is smaller than the vocabulary");
    const uint64_t rows = d->n_seqs * (d->max_drafts + 1);
    const Chunks c = chunks_of(rows, d->vocab);
    const VerifyGrids g = verify_grids(d->n_seqs, d->max_drafts, c.n, greedy);   // (the draw's are fewer than either)
    if (!grid_fits(g.stats, VF_STATS) || !grid_fits(g.decide, VF_DECIDE)) return refuse(me, "n_seqs * max_drafts * vocab out of range");
    const uint64_t need = verify_bytes(d->n_seqs, d->max_drafts, c.n);
    if (!d_workspace || workspace_bytes < need || !aligned16(d_workspace))
        return refuse(me, "workspace missing, too small (hipdec_verify_drafts_workspace) or not 16-byte aligned");
    if ((bad = wrong_place({d->d_logits, d->d_drafts, d->d_n_drafts, d->d_draft_probs, d->d_uniforms, d->d_tokens, d->d_accepted,
                            d_workspace}, stream_of(stream))))
        return refuse(me, bad);
    VfStat *st = (VfStat *)d_workspace;
    VfPlace *places = (VfPlace *)(st + rows * c.n);
    const double log2e = 1.4426950408889634074, cap = d->softcap > 0.0f ? d->softcap : 0.0;
    const VerifyArgs a{d->d_logits, d->row_stride, d->prob_stride, d->d_drafts, d->d_n_drafts, d->d_draft_probs, d->d_uniforms,
                       (int)d->n_seqs, (int)d->max_drafts, (int)d->vocab, c.n, greedy ? 0.0 : log2e / (double)d->temperature,
                       cap, cap > 0.0 ? 2.0 * log2e / cap : 0.0, st, (double *)(places + d->n_seqs), places, d->d_tokens, d->d_accepted};
    hipStream_t s = stream_of(stream);
    return launched(me, d->dtype == HIPDEC_ROWS_BF16 ? go_verify<true>(a, c.per, s) : go_verify<false>(a, c.per, s));
}

}  // extern "C"
