// C ABI of the gfx950 decode backend (see include/hip_decode.h): model construction, weight
// conversion, hipGraph-captured decode steps and the head variants.
#include "../../include/hip_decode.h"
#include "../../include/hip_decode_debug.h"
#include "hipdec_mega.h"
#include "hipdec_lean.h"
#include "hipdec_prefill.h"
#include "hipdec_batch.h"
#include "hipdec_rows.h"
#include "hipdec_requests.h"
#include "hipdec_sample.h"

#include <math.h>
#include <cmath>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <string>
#include <vector>
#include <algorithm>
#include <map>
#include <memory>
#include <mutex>
#include <thread>
#include <unistd.h>

extern char **environ;

namespace {

// V_TOPK_S / V_STATS_S: the same step followed by the on-device draw (hipdec_sample.h)
enum Variant { V_X = 0, V_ARGMAX, V_TOPK, V_STATS, V_LOGITS, V_TOPK_S, V_STATS_S, V_COUNT };

struct WeightStore;

struct DevLayer {
    void *wqkv = nullptr, *wo = nullptr, *w13 = nullptr, *w2 = nullptr;
    void *s_qkv = nullptr, *s_wo = nullptr, *s_w13 = nullptr, *s_w2 = nullptr;
    float *g1 = nullptr, *g2 = nullptr;
    void *kc = nullptr, *vc = nullptr;
};

// Texts of failed calls without a model (hipdec_last_error(NULL)).  Creating a model, and every other entry but the operators on the
// caller's device buffers, leaves its text to the whole process: a program may create on one thread and report on another.
// An operator's text is the calling thread's own (requests on several threads may fail at once) and stands there until
// another call without a model fails on that thread.
struct CreateError {
    std::mutex mu;
    std::string text;
    CreateError &operator=(const std::string &what);
};
CreateError g_create_error;
thread_local std::string g_op_error, g_shown_error;
thread_local bool g_op_failed = false;
CreateError &CreateError::operator=(const std::string &what) {
    std::lock_guard<std::mutex> lock(mu);
    g_op_failed = false;
    text = what;
    return *this;
}

// Workspace of the chunked prompt prefill (hipdec_prefill.h), allocated at the first prefill.
struct PrefillWork {
    int rows = 0;                        // chunk capacity in prompt rows
    uint32_t *ids = nullptr;
    float *x = nullptr, *x2 = nullptr, *q = nullptr;
    uint16_t *xn_hi = nullptr, *xn_lo = nullptr, *att_hi = nullptr, *att_lo = nullptr, *gate_hi = nullptr,
             *gate_lo = nullptr;
    float *ssq = nullptr;                // [rows][chunks] sums of squares of the residual rows
    float *P = nullptr;                  // split-K partial planes
    size_t P_floats = 0;
    uint32_t *h_ids = nullptr;           // pinned
};

// State of the multi-sample decode (hipdec_batch.h): rows share cache positions [0, prefix) and
// append to their own suffix caches.
enum BatchVariant { B_LOGITS = 0, B_ARGMAX, B_TOPK, B_STATS, B_TOPK_S, B_STATS_S, B_COUNT };
struct BatchState {
    int rows = 0;                        // 0: no batch open
    size_t prefix = 0, slot = 0;
    int cap_rows = 0;                    // rows the buffers below were sized for
    size_t suf_rows = 0;                 // capacity of one row's suffix cache
    std::vector<void *> kc_suf, vc_suf;  // per layer [cap_rows][suf_rows][kv_dim]
    BatchParams *d_bp = nullptr, *h_bp = nullptr;
    float *logits = nullptr, *d_out = nullptr, *d_vals = nullptr, *d_bmax = nullptr, *d_bsum = nullptr;
    uint32_t *d_idxs = nullptr, *d_tok = nullptr;
    float *h_stage = nullptr;            // pinned, cap_rows * max(vocab, 2 * blocks * 32) floats
    size_t h_stage_floats = 0;
    bool have_logits = false;            // a step has run since hipdec_batch_begin
    hipGraphExec_t graphs[B_COUNT] = {}; // one captured step per head variant, for graph_rows rows
    uint32_t *d_ring = nullptr, *h_ring = nullptr;   // tokens of a sampled run, [steps][rows]; h_ring pinned
    size_t ring_elems = 0;
    int graph_rows = 0;
    // the layers of a step as one persistent launch (hipdec_rows.h), where the model and the row count fit
    bool rows_ready = false;             // buffers below exist and the kernel accepted its LDS size
    bool rows_off = false;               // a wait timed out: the step keeps to one kernel per product from then on
    bool rows_active = false;            // the open batch uses it
    RowsArgs rows_args{};
    void *rows_slab = nullptr;           // uncached exchange buffers (uncached_take), sized for ROWS_MAX_R rows
    size_t rows_slab_cap = 0, rows_slab_bytes = 0;
    unsigned *rows_epochs = nullptr;
    float *rows_xb = nullptr;            // per-XCD copies of the exchanged vectors (ordinary memory)
    size_t rows_xb_bytes = 0;
    void **rows_suf = nullptr;           // device table [2][L] of the suffix caches
    const void *rows_suf_seen = nullptr; // first suffix cache the table was written for
};

// State of the requests stepped together over a paged cache (hipdec_requests.h).
constexpr int kRequestRows = 32;         // rows of a step: tokens and drafts of all its sequences
struct RequestState {
    bool open = false;
    int page_shift = 0, max_pages = 0;   // pages a sequence of cfg.seq positions needs
    uint32_t max_seqs = 0, n_pages = 0;
    std::vector<void *> k, v;            // per layer [n_pages][page][kv_dim]
    std::vector<int> table;              // [max_seqs][max_pages], -1: none; d_table holds the same
    std::vector<int> free_pages;
    std::vector<long long> lens;         // positions held by each sequence, -1: not admitted
    int *d_table = nullptr, *d_rows = nullptr, *h_rows = nullptr;   // d_rows / h_rows: [5][kRequestRows] positions, slots, sequences, lengths, drafts
    double *d_freq = nullptr;
    float *qkv = nullptr, *att = nullptr, *logits = nullptr, *d_u = nullptr, *h_u = nullptr, *d_probs = nullptr;
    uint32_t *d_tok = nullptr, *h_tok = nullptr;                    // tokens of a step, then accepted counts
    void *ws_att = nullptr, *ws_ver = nullptr;
    uint64_t ws_att_bytes = 0, ws_ver_bytes = 0;
    int *d_n = nullptr;                  // draft counts, behind the rows
};

}  // namespace

// run state of the on-device sampler as the host stages it (pinned)
struct SampleHost {
    SampleParams ss;
    uint64_t rng[32];
};

struct hipdec_model {
    hipdec_config cfg{};
    hipdec_options opt{};
    int wt = WT_F32, embed_wt = WT_F32, kvbf16 = 0;
    int pf_act = PF_ACT_PAIR;            // how the chunked prefill carries activations into its GEMMs (PF_ACT_*)
    int num_cu = 256;
    hipStream_t stream = nullptr;
    std::vector<DevLayer> layers;
    void *embed = nullptr;
    float *gfinal = nullptr;
    float *x_a = nullptr, *x_b = nullptr, *q = nullptr, *att = nullptr, *gate = nullptr, *logits = nullptr,
          *x_in = nullptr, *part = nullptr;
    unsigned *counters = nullptr;
    float *rope_cos = nullptr, *rope_sin = nullptr;
    StepParams *d_sp = nullptr, *h_sp = nullptr;      // h_sp: pinned array [seq + 1]
    float *d_topk_vals = nullptr, *d_bmax = nullptr, *d_bsum = nullptr, *d_out = nullptr;
    uint32_t *d_topk_idxs = nullptr, *d_ring = nullptr;
    float *h_out = nullptr;                           // pinned staging, max(vocab, 2*blocks*32) floats
    float *d_hout = nullptr;                          // the same memory as the device sees it (nullptr: not mapped)
    size_t h_out_elems = 0;
    size_t len = 0;
    int NS = 1, blocks = 0;
    float alpha = 1.0f;
    hipGraphExec_t graphs[V_COUNT] = {};
    hipEvent_t ev0 = nullptr, ev1 = nullptr;
    hipEvent_t ev_s0 = nullptr, ev_s1 = nullptr;      // around a single step
    bool step_timed = false;
    float last_ms = 0.0f;
    // persistent one-launch-per-token step (hipdec_mega.h)
    bool mega_ok = false;
    int lean_ce = 0;                                  // != 0: the step runs k_lean<lean_ce, ...> (hipdec_lean.h) instead of k_mega
    MegaArgs mega{};
    int mega_grid = 0;
    size_t mega_lds = 0;
    unsigned *d_epochs = nullptr;
    unsigned *h_abort = nullptr, *d_abort = nullptr;  // abort flags of the persistent kernels: pinned host memory, mapped ([0] single-row, [16] multi-row)
    // The same mapped block, further on: the step parameters ([32]..) and the one-slot token ring ([48]) of a
    // single step that the host waits for.  The kernel reads its parameters from there and leaves the token there,
    // so such a step is one launch and one wait: no parameter upload in front of it, no copy behind it.
    bool direct_step = false;                         // the step just enqueued used them
    void *xslab = nullptr;                            // uncached slab holding the exchange buffers (uncached_take)
    size_t xslab_cap = 0;
    PrefillWork pf;
    BatchState bt;
    RequestState rq;
    SampleParams *d_ss = nullptr;                     // on-device sampler (hipdec_sample.h)
    uint64_t *d_rng = nullptr;                        // [32], one state per row
    SampleHost *h_samp = nullptr;                     // pinned
    std::vector<void *> allocs;
    std::shared_ptr<WeightStore> wstore;   // the weights (read-only after creation), possibly shared with other models
    std::string err;
};

namespace {

#define HCHK(expr)                                                                           \
    do {                                                                                     \
        hipError_t e_ = (expr);                                                              \
        if (e_ != hipSuccess) {                                                              \
            char b_[512];                                                                    \
            snprintf(b_, sizeof b_, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_),   \
                     __FILE__, __LINE__);                                                    \
            m->err = b_;                                                                     \
            return HIPDEC_ERR_HIP;                                                           \
        }                                                                                    \
    } while (0)

int fail(hipdec_model *m, int code, const char *msg) {
    if (m) m->err = msg; else g_create_error = msg;
    return code;
}

// Uncached device memory for the buffers workgroups exchange vectors through: stores go straight to
// the fabric and polls read from it without passing a per-XCD L2 that no other XCD shares, which
// shortens every exchange of the persistent kernel (600M step 0.797 -> 0.730 ms).  Such memory is
// never handed back to the driver while the process lives (allocations made after freeing uncached
// memory that kernels had read have been seen to hold wrong values): slabs are recycled through
// this process-wide pool, by device and power-of-two size.
struct UncachedPool {
    std::mutex mu;
    std::multimap<std::pair<int, size_t>, void *> idle;
};
UncachedPool &uncached_pool() { static UncachedPool *p = new UncachedPool(); return *p; }   // never destroyed

void *uncached_take(int device, size_t bytes, size_t *cap_out) {
    size_t cap = 64 * 1024;
    while (cap < bytes) cap <<= 1;
    *cap_out = cap;
    UncachedPool &pool = uncached_pool();
    {
        std::lock_guard<std::mutex> lock(pool.mu);
        auto it = pool.idle.find({device, cap});
        if (it != pool.idle.end()) { void *p = it->second; pool.idle.erase(it); return p; }
    }
    void *p = nullptr;
    if (hipExtMallocWithFlags(&p, cap, hipDeviceMallocUncached) != hipSuccess) { (void)hipGetLastError(); return nullptr; }
    return p;
}

void uncached_give(int device, size_t cap, void *p) {
    UncachedPool &pool = uncached_pool();
    std::lock_guard<std::mutex> lock(pool.mu);
    pool.idle.insert({{device, cap}, p});
}

// device memory of a model's weights: shared (reference-counted) by the models created from one another
// with hipdec_create_shared, freed with the last of them
struct WeightStore {
    int device = 0;
    std::vector<void *> allocs;
    ~WeightStore() {
        (void)hipSetDevice(device);
        for (void *p : allocs) (void)hipFree(p);
    }
};

template <typename T> int walloc(hipdec_model *m, T **p, size_t bytes);
template <typename T> int dalloc(hipdec_model *m, T **p, size_t bytes) {
    void *v = nullptr;
    HCHK(hipMalloc(&v, bytes ? bytes : 16));
    m->allocs.push_back(v);
    *p = (T *)v;
    return HIPDEC_OK;
}

template <typename T> int walloc(hipdec_model *m, T **p, size_t bytes) {
    void *v = nullptr;
    HCHK(hipMalloc(&v, bytes ? bytes : 16));
    m->wstore->allocs.push_back(v);
    *p = (T *)v;
    return HIPDEC_OK;
}

size_t wt_row_bytes(int wt, size_t K) {
    switch (wt) {
        case WT_F32: return K * 4;
        case WT_BF16: return K * 2;
        case WT_FP8: return K;
        default: return K / 2;
    }
}
size_t wt_scale_bytes(int wt, size_t rows, size_t K) {
    if (wt == WT_FP8) return rows * 4;
    if (wt == WT_INT4) return rows * (K / 128) * 2;
    return 0;
}

template <int WT> void launch_convert(hipStream_t s, const float *src, void *dst, void *scales, int rows, int K,
                                      int mul, int off) {
    hipLaunchKernelGGL(k_convert_rows<WT>, dim3(rows), dim3(256), 0, s, src, dst, scales, K, mul, off);
}
void convert_rows(int wt, hipStream_t s, const float *src, void *dst, void *scales, int rows, int K, int mul, int off) {
    switch (wt) {
        case WT_F32: launch_convert<WT_F32>(s, src, dst, scales, rows, K, mul, off); break;
        case WT_BF16: launch_convert<WT_BF16>(s, src, dst, scales, rows, K, mul, off); break;
        case WT_FP8: launch_convert<WT_FP8>(s, src, dst, scales, rows, K, mul, off); break;
        default: launch_convert<WT_INT4>(s, src, dst, scales, rows, K, mul, off); break;
    }
}

// host fp32 matrix -> device storage.  transpose: the host matrix is [K][O] (row = input
// channel) and is turned into out-major [O][K] first.
int load_matrix(hipdec_model *m, int wt, const float *host, int O, int K, bool transpose, float *stage_a,
                float *stage_b, void *dst, void *scales, int mul, int off) {
    HCHK(hipMemcpy(stage_a, host, (size_t)O * K * sizeof(float), hipMemcpyHostToDevice));
    const float *src = stage_a;
    if (transpose) {
        dim3 grid((O + 31) / 32, (K + 31) / 32), block(32, 8);
        hipLaunchKernelGGL(k_transpose_f32, grid, block, 0, m->stream, stage_a, stage_b, K, O);
        src = stage_b;
    }
    convert_rows(wt, m->stream, src, dst, scales, O, K, mul, off);
    HCHK(hipGetLastError());
    HCHK(hipStreamSynchronize(m->stream));
    return HIPDEC_OK;
}

// ---- one decode step, enqueued on the model's stream
template <int WT, int EPI, int KVB> void launch_gemv_t(hipdec_model *m, const GemvArgs &a) {
    int n_groups = (a.rows + 1) / 2;
    size_t lds = (size_t)a.K * sizeof(float);
    int per_cu = (int)(150 * 1024 / (lds + 64));
    if (per_cu > 8) per_cu = 8;
    if (per_cu < 1) per_cu = 1;
    int grid = (n_groups + 3) / 4;
    int cap = m->num_cu * per_cu;
    if (grid > cap) grid = cap;
    hipLaunchKernelGGL((k_gemv<WT, EPI, KVB>), dim3(grid), dim3(256), lds, m->stream, a);
}
template <int EPI> void launch_gemv(hipdec_model *m, int wt, const GemvArgs &a) {
    const int kvb = (EPI == EPI_QKV) ? m->kvbf16 : 0;
#define GEMV_CASE(W)                                                    \
    if (kvb) launch_gemv_t<W, EPI, 1>(m, a); else launch_gemv_t<W, EPI, 0>(m, a);
    switch (wt) {
        case WT_F32: GEMV_CASE(WT_F32) break;
        case WT_BF16: GEMV_CASE(WT_BF16) break;
        case WT_FP8: GEMV_CASE(WT_FP8) break;
        default: GEMV_CASE(WT_INT4) break;
    }
#undef GEMV_CASE
}

void launch_attn(hipdec_model *m, const DevLayer &L) {
    const hipdec_config &c = m->cfg;
    dim3 grid(c.heads, m->NS), block(256);
    float scale = 1.0f / sqrtf((float)c.hd);
    int gqa = c.gqa_ratio ? c.gqa_ratio : 1;
#define ATT(KVB, HD)                                                                                          \
    hipLaunchKernelGGL((k_attn_decode<KVB, HD>), grid, block, 0, m->stream, m->q, L.kc, L.vc, m->d_sp, m->part, \
                       m->counters, m->att, (int)c.kv_dim, gqa, m->NS, scale)
    if (m->kvbf16) { if (c.hd == 64) ATT(1, 64); else ATT(1, 128); }
    else { if (c.hd == 64) ATT(0, 64); else ATT(0, 128); }
#undef ATT
}

template <int WT> void launch_mega_t(hipdec_model *m, const MegaArgs &a) {
    dim3 grid(m->mega_grid), block(MEGA_THREADS);
#define MEGA2(KVB, HD, BP) hipLaunchKernelGGL((k_mega<WT, KVB, HD, BP>), grid, block, m->mega_lds, m->stream, a)
#define MEGA(KVB, HD) do { if (a.prof) MEGA2(KVB, HD, MEGA_VAR_STAMPS); else MEGA2(KVB, HD, MEGA_VAR_PLAIN); } while (0)
    if (m->kvbf16) { if (m->cfg.hd == 64) MEGA(1, 64); else MEGA(1, 128); }
    else { if (m->cfg.hd == 64) MEGA(0, 64); else MEGA(0, 128); }
#undef MEGA
#undef MEGA2
}
template <int CE> void launch_lean_t(hipdec_model *m, const MegaArgs &a) {
    dim3 grid(m->mega_grid), block(MEGA_THREADS);
#define LEAN2(KVB, HD, BP) hipLaunchKernelGGL((k_lean<CE, KVB, HD, BP>), grid, block, m->mega_lds, m->stream, a)
#define LEAN(KVB, HD) do { if (a.prof) LEAN2(KVB, HD, MEGA_VAR_STAMPS); else LEAN2(KVB, HD, MEGA_VAR_PLAIN); } while (0)
    if (m->kvbf16) { if (m->cfg.hd == 64) LEAN(1, 64); else LEAN(1, 128); }
    else { if (m->cfg.hd == 64) LEAN(0, 64); else LEAN(0, 128); }
#undef LEAN
#undef LEAN2
}
template <int CE> hipError_t lean_set_lds_t(hipdec_model *m) {
    hipError_t e = hipSuccess;
#define LEAN_ATTR(KVB, HD)                                                                                       \
    do {                                                                                                          \
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_lean<CE, KVB, HD, MEGA_VAR_PLAIN>),             \
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)m->mega_lds);                    \
        if (e == hipSuccess)                                                                                      \
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_lean<CE, KVB, HD, MEGA_VAR_STAMPS>),        \
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)m->mega_lds);                \
    } while (0)
    if (m->kvbf16) { if (m->cfg.hd == 64) LEAN_ATTR(1, 64); else LEAN_ATTR(1, 128); }
    else { if (m->cfg.hd == 64) LEAN_ATTR(0, 64); else LEAN_ATTR(0, 128); }
#undef LEAN_ATTR
    return e;
}
// chunk counts (dim / 512) the short-phase kernel is built for
constexpr bool lean_ce_built(int ce) { return ce == 1 || ce == 3; }

void launch_mega(hipdec_model *m, int do_head, int advance, bool direct = false) {
    MegaArgs a = m->mega;
    a.do_head = do_head;
    a.advance = advance;
    if (direct) {      // parameters and token slot in mapped host memory (see hipdec_model::direct_step)
        a.sp = (StepParams *)(m->d_abort + 32);
        a.ring = m->d_abort + 48;
        a.ring_cap = 1;
    }
    if (m->lean_ce) {
        if (m->lean_ce == 1) launch_lean_t<1>(m, a); else launch_lean_t<3>(m, a);
        return;
    }
    switch (m->wt) {
        case WT_F32: launch_mega_t<WT_F32>(m, a); break;
        case WT_BF16: launch_mega_t<WT_BF16>(m, a); break;
        case WT_FP8: launch_mega_t<WT_FP8>(m, a); break;
        default: launch_mega_t<WT_INT4>(m, a); break;
    }
}

template <int WT> hipError_t mega_set_lds_t(hipdec_model *m) {
    hipError_t e = hipSuccess;
#define MEGA_ATTR(KVB, HD)                                                                                       \
    do {                                                                                                          \
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_mega<WT, KVB, HD, MEGA_VAR_PLAIN>),             \
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)m->mega_lds);                    \
        if (e == hipSuccess)                                                                                      \
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_mega<WT, KVB, HD, MEGA_VAR_STAMPS>),        \
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)m->mega_lds);                \
    } while (0)
    if (m->kvbf16) { if (m->cfg.hd == 64) MEGA_ATTR(1, 64); else MEGA_ATTR(1, 128); }
    else { if (m->cfg.hd == 64) MEGA_ATTR(0, 64); else MEGA_ATTR(0, 128); }
#undef MEGA_ATTR
    return e;
}

void enqueue_step(hipdec_model *m, int variant) {
    const hipdec_config &c = m->cfg;
    const int D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, V = c.vocab;
    if (variant == V_TOPK_S || variant == V_STATS_S) {
        // the candidate / statistics step, then the draw; the drawn token becomes the next step's input
        enqueue_step(m, variant == V_TOPK_S ? V_TOPK : V_STATS);
        uint32_t *tok_out = (uint32_t *)&m->d_sp->tok;
        if (variant == V_TOPK_S)
            hipLaunchKernelGGL(k_sample_topk, dim3(1), dim3(256), 0, m->stream, m->d_topk_vals, m->d_topk_idxs, m->blocks,
                               m->d_ss, m->d_rng, tok_out, m->d_ring, (BatchParams *)nullptr);
        else
            hipLaunchKernelGGL(k_sample_fullvocab, dim3(1), dim3(256), 0, m->stream, m->logits, V, m->d_bmax, m->d_bsum,
                               m->blocks, m->d_ss, m->d_rng, tok_out, m->d_ring, (BatchParams *)nullptr);
        return;
    }
    if (m->mega_ok) {
        // the whole step in one persistent launch; with 8-bit/4-bit weights the (bf16) LM head
        // stays a separate GEMV
        const bool head_inside = (m->wt == m->embed_wt);
        if (variant == V_X) { launch_mega(m, 0, 1); return; }
        if (head_inside) {
            launch_mega(m, 1, 1);
        } else {
            launch_mega(m, 0, 0);
            GemvArgs a{};
            a.sp = m->d_sp; a.W = m->embed; a.in = m->x_a; a.gamma = m->gfinal; a.out = m->logits; a.rows = V; a.K = D;
            launch_gemv<EPI_HEAD>(m, m->embed_wt, a);
            if (variant == V_ARGMAX)
                hipLaunchKernelGGL(k_head_argmax, dim3(1), dim3(1024), 0, m->stream, m->logits, V, m->d_sp, m->d_ring,
                                   (int)c.seq);
            else
                hipLaunchKernelGGL(k_advance, dim3(1), dim3(1), 0, m->stream, m->d_sp);
        }
        if (variant == V_TOPK)
            hipLaunchKernelGGL(k_head_topk, dim3(m->blocks), dim3(256), 0, m->stream, m->logits, V, m->d_sp,
                               m->d_topk_vals, m->d_topk_idxs);
        else if (variant == V_STATS)
            hipLaunchKernelGGL(k_head_block_stats, dim3(m->blocks), dim3(256), 0, m->stream, m->logits, V, m->d_sp,
                               m->d_bmax, m->d_bsum);
        return;
    }
    if (m->embed_wt == WT_F32)
        hipLaunchKernelGGL(k_embed<WT_F32>, dim3((D + 255) / 256), dim3(256), 0, m->stream, m->embed, m->x_in,
                           m->d_sp, m->x_a, D);
    else
        hipLaunchKernelGGL(k_embed<WT_BF16>, dim3((D + 255) / 256), dim3(256), 0, m->stream, m->embed, m->x_in,
                           m->d_sp, m->x_a, D);
    for (uint32_t l = 0; l < c.nlayers; ++l) {
        const DevLayer &L = m->layers[l];
        GemvArgs a{};
        a.sp = m->d_sp; a.alpha = m->alpha; a.q_dim = Q; a.kv_dim = KV; a.hd = c.hd; a.act = m->opt.ffn_activation;
        a.rope_cos = m->rope_cos; a.rope_sin = m->rope_sin;
        // q/k/v projections + RoPE + cache append
        a.W = L.wqkv; a.scales = L.s_qkv; a.in = m->x_a; a.gamma = L.g1; a.out = m->q; a.kc = L.kc; a.vc = L.vc;
        a.rows = Q + 2 * KV; a.K = D;
        launch_gemv<EPI_QKV>(m, m->wt, a);
        launch_attn(m, L);
        // output projection + residual: x_b = x_a + alpha * (att . wo)
        a.W = L.wo; a.scales = L.s_wo; a.in = m->att; a.gamma = nullptr; a.resid = m->x_a; a.out = m->x_b;
        a.rows = D; a.K = Q;
        launch_gemv<EPI_WO>(m, m->wt, a);
        // gate/up + activation
        a.W = L.w13; a.scales = L.s_w13; a.in = m->x_b; a.gamma = L.g2; a.resid = nullptr; a.out = m->gate;
        a.rows = 2 * H; a.K = D;
        launch_gemv<EPI_W13>(m, m->wt, a);
        // down projection + residual: x_a = x_b + alpha * (gate . w2)
        a.W = L.w2; a.scales = L.s_w2; a.in = m->gate; a.gamma = nullptr; a.resid = m->x_b; a.out = m->x_a;
        a.rows = D; a.K = H;
        launch_gemv<EPI_W2>(m, m->wt, a);
    }
    if (variant == V_X) {
        hipLaunchKernelGGL(k_advance, dim3(1), dim3(1), 0, m->stream, m->d_sp);
        return;
    }
    GemvArgs a{};
    a.sp = m->d_sp; a.W = m->embed; a.in = m->x_a; a.gamma = m->gfinal; a.out = m->logits; a.rows = V; a.K = D;
    launch_gemv<EPI_HEAD>(m, m->embed_wt, a);
    switch (variant) {
        case V_ARGMAX:
            hipLaunchKernelGGL(k_head_argmax, dim3(1), dim3(1024), 0, m->stream, m->logits, V, m->d_sp, m->d_ring,
                               (int)c.seq);
            break;
        case V_TOPK:
            hipLaunchKernelGGL(k_head_topk, dim3(m->blocks), dim3(256), 0, m->stream, m->logits, V, m->d_sp,
                               m->d_topk_vals, m->d_topk_idxs);
            hipLaunchKernelGGL(k_advance, dim3(1), dim3(1), 0, m->stream, m->d_sp);
            break;
        case V_STATS:
            hipLaunchKernelGGL(k_head_block_stats, dim3(m->blocks), dim3(256), 0, m->stream, m->logits, V, m->d_sp,
                               m->d_bmax, m->d_bsum);
            hipLaunchKernelGGL(k_advance, dim3(1), dim3(1), 0, m->stream, m->d_sp);
            break;
        default:
            hipLaunchKernelGGL(k_advance, dim3(1), dim3(1), 0, m->stream, m->d_sp);
            break;
    }
}

int run_step(hipdec_model *m, int variant) {
    if (m->opt.flags & HIPDEC_FLAG_NO_GRAPH) {
        enqueue_step(m, variant);
        HCHK(hipGetLastError());
        return HIPDEC_OK;
    }
    if (!m->graphs[variant]) {
        hipGraph_t g = nullptr;
        HCHK(hipStreamBeginCapture(m->stream, hipStreamCaptureModeThreadLocal));
        enqueue_step(m, variant);
        hipError_t e = hipStreamEndCapture(m->stream, &g);
        if (e != hipSuccess || !g) { m->err = std::string("graph capture failed: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
        HCHK(hipGraphInstantiate(&m->graphs[variant], g, nullptr, nullptr, 0));
        HCHK(hipGraphDestroy(g));
    }
    HCHK(hipGraphLaunch(m->graphs[variant], m->stream));
    return HIPDEC_OK;
}

// A single step the caller waits for, on a model whose whole step (head included) is one persistent launch: the
// kernel takes its parameters from mapped host memory and writes the token there (HIPDEC_NO_DIRECT_STEP=1: the
// general way, for comparisons).
static bool direct_step_ok(const hipdec_model *m, int variant) {
    static const bool off = [] { const char *v = getenv("HIPDEC_NO_DIRECT_STEP"); return v && v[0] == '1'; }();
    if (off || !m->mega_ok || m->wt != m->embed_wt) return false;
    return variant == V_X || variant == V_ARGMAX || ((variant == V_TOPK || variant == V_STATS) && m->d_hout);
}

// upload the step parameters from pinned slot `slot`, then run one step
int step_with(hipdec_model *m, int variant, size_t slot, const StepParams &p, bool caller_waits = false) {
    static const bool no_events = [] { const char *v = getenv("HIPDEC_NO_STEP_EVENTS"); return v && v[0] == '1'; }();
    m->direct_step = false;
    if (caller_waits && direct_step_ok(m, variant)) {     // (one mapped block: only for a step that is waited for before the next)
        StepParams *hp = (StepParams *)(m->h_abort + 32);
        *hp = p;
        hp->step = 0;
        __atomic_thread_fence(__ATOMIC_RELEASE);
        if (!no_events) HCHK(hipEventRecord(m->ev_s0, m->stream));
        launch_mega(m, variant == V_X ? 0 : 1, 1, true);
        // per-block candidates / statistics straight into the pinned buffer the caller's arrays are filled from
        const StepParams *dp = (const StepParams *)(m->d_abort + 32);
        if (variant == V_TOPK)
            hipLaunchKernelGGL(k_head_topk, dim3(m->blocks), dim3(256), 0, m->stream, m->logits, (int)m->cfg.vocab, dp, m->d_hout,
                               (uint32_t *)(m->d_hout + (size_t)m->blocks * p.top_k));
        else if (variant == V_STATS)
            hipLaunchKernelGGL(k_head_block_stats, dim3(m->blocks), dim3(256), 0, m->stream, m->logits, (int)m->cfg.vocab, dp, m->d_hout,
                               m->d_hout + m->blocks);
        HCHK(hipGetLastError());
        if (!no_events) { HCHK(hipEventRecord(m->ev_s1, m->stream)); m->step_timed = true; }
        m->direct_step = true;
        return HIPDEC_OK;
    }
    m->h_sp[slot] = p;
    HCHK(hipMemcpyAsync(m->d_sp, &m->h_sp[slot], sizeof(StepParams), hipMemcpyHostToDevice, m->stream));
    if (!no_events) HCHK(hipEventRecord(m->ev_s0, m->stream));
    int rc = run_step(m, variant);
    if (rc) return rc;
    if (!no_events) { HCHK(hipEventRecord(m->ev_s1, m->stream)); m->step_timed = true; }
    return HIPDEC_OK;
}

int check_step(hipdec_model *m, uint32_t token, bool from_id) {
    if (!m) return HIPDEC_ERR_ARG;
    if (m->len >= m->cfg.seq) return fail(m, HIPDEC_ERR_FULL, "decode only supports lengths within cfg.seq");
    if (from_id && token >= m->cfg.vocab) return fail(m, HIPDEC_ERR_ARG, "token id must fit vocab");
    return HIPDEC_OK;
}

StepParams base_params(hipdec_model *m, uint32_t token) {
    StepParams p{};
    p.tok = (int)token; p.pos = (int)m->len; p.step = 0; p.top_k = 1; p.inv_t = 1.0f; p.softcap = 0.0f;
    p.use_x_in = 0; p.block_idx = 0;
    return p;
}

// stream sync after a step; a persistent-kernel wait that timed out shows up as an error here
int sync_checked(hipdec_model *m) {
    HCHK(hipStreamSynchronize(m->stream));
    // (the device time of the single step that was just waited for is worked out when hipdec_last_device_ms asks)
    if (m->mega_ok) {
        // (the kernels write the flag into mapped host memory; the wait above has made it visible)
        const unsigned flag = __atomic_load_n(&m->h_abort[0], __ATOMIC_ACQUIRE);
        if (flag) {
            __atomic_store_n(&m->h_abort[0], 0u, __ATOMIC_RELEASE);
            // The aborted step left a mix of old and new stamps in the exchange buffers and did not
            // advance the epochs, so a later step could accept its values: clear all of it and let
            // every later step take the one-kernel-per-product path (its captured graphs hold
            // persistent launches and go too).
            const hipdec_config &c = m->cfg;
            const MegaArgs &a = m->mega;
            HCHK(hipMemset(a.QKV, 0, (size_t)(c.q_dim + 2 * c.kv_dim) * 4));
            HCHK(hipMemset(a.PART, 0, (size_t)c.heads * a.ns_max * (c.hd + MEGA_PREC) * 4));
            HCHK(hipMemset(a.X2, 0, (size_t)c.dim * 4));
            HCHK(hipMemset(a.GATE, 0, (size_t)c.hidden * 4));
            HCHK(hipMemset(a.CAND, 0, (size_t)m->mega_grid * 8));
            HCHK(hipMemset(m->x_a, 0, (size_t)c.dim * 4));
            HCHK(hipMemset(m->d_epochs, 0, 16));
            m->mega_ok = false;
            m->lean_ce = 0;
            for (auto &g : m->graphs) if (g) { (void)hipGraphExecDestroy(g); g = nullptr; }
            m->err = "persistent decode kernel: a wait on another workgroup timed out (the grid needs the whole GPU to "
                     "itself); later steps use one kernel per product";
            return HIPDEC_ERR_HIP;
        }
    }
    return HIPDEC_OK;
}
#define SYNC_CHECKED(m) do { int rc_ = sync_checked(m); if (rc_ != HIPDEC_OK) return rc_; } while (0)

int softcap_out(hipdec_model *m, int start, int n, float cap, float *host_out) {
    static const bool no_direct = [] { const char *v = getenv("HIPDEC_NO_DIRECT_STEP"); return v && v[0] == '1'; }();
    if (m->d_hout && !no_direct) {
        // the kernel writes the pinned buffer itself: one launch and one wait, no copy behind it
        hipLaunchKernelGGL(k_softcap_copy, dim3((n + 255) / 256), dim3(256), 0, m->stream, m->logits, m->d_hout, start, n, cap);
        HCHK(hipGetLastError());
    } else {
        hipLaunchKernelGGL(k_softcap_copy, dim3((n + 255) / 256), dim3(256), 0, m->stream, m->logits, m->d_out, start, n, cap);
        HCHK(hipGetLastError());
        HCHK(hipMemcpyAsync(m->h_out, m->d_out, (size_t)n * sizeof(float), hipMemcpyDeviceToHost, m->stream));
    }
    SYNC_CHECKED(m);
    memcpy(host_out, m->h_out, (size_t)n * sizeof(float));
    return HIPDEC_OK;
}

// ---- chunked prompt prefill on the matrix cores (hipdec_prefill.h)
constexpr int kPrefillMaxRows = 1024;     // prompt rows per chunk
constexpr int kPrefillMinRows = 8;        // shorter prompts go through the token step

bool prefill_batched_ok(const hipdec_model *m, size_t n) {
    const hipdec_config &c = m->cfg;
    if (m->opt.flags & HIPDEC_FLAG_PREFILL_STEPS) return false;
    if (n < (size_t)kPrefillMinRows) return false;
    // (fp32 weights: chunks of at most kSkinnyRows rows, the one matrix-core GEMM that takes them)
    if (c.dim % PF_BK || c.q_dim % PF_BK || c.hidden % PF_BK) return false;
    if (m->wt == WT_INT4 && (c.dim % 128 || c.q_dim % 128 || c.hidden % 128)) return false;   // whole scale groups
    if (c.hd != 64 && c.hd != 128) return false;
    return true;
}

struct PfSplit { int splits, steps_per_split; };
constexpr int kSkinnyRows = 32;          // at most this many rows: the streaming GEMM without LDS weight tiles
constexpr int kSkinnyLdsBytes = 40 * 1024;   // dynamic LDS for the staged activation slice
// the tiled GEMM whose operands go straight into LDS (k_pf_gemm_dl): bf16 weights, enough rows to fill its
// 128 x 256 tiles, whole 64-element steps, activations as bf16 (pair or single)
constexpr int kDlMinRows = 129;
constexpr int kSkinnyI4Nt = 1;                    // 16-row weight tiles per wave of k_pf_gemm_skinny_i4 (2: 4 - 8 % slower on the 5B shapes)
constexpr int kSkinnyI4Waves = 8;                 // waves per workgroup (4: as fast at 9+ rows, 5 - 15 % slower at 8)
constexpr int kSkinnyI4Bn = 16 * kSkinnyI4Nt * kSkinnyI4Waves;   // weight rows per workgroup
// the few-row GEMM of 4-bit models: the kernel of its own (HIPDEC_NO_SKINNY_I4=1: the general few-row kernel)
bool pf_use_skinny_i4() {
    static const bool off = [] { const char *v = getenv("HIPDEC_NO_SKINNY_I4"); return v && v[0] == '1'; }();
    return !off;
}
constexpr int kSkinnyI4WgsPerCu = 3;              // workgroups per CU its K splits aim at
constexpr int kSkinnyF8Waves = 8;                 // waves per workgroup of k_pf_gemm_skinny_f8, 16 weight rows each
constexpr int kSkinnyF8Bn = 16 * kSkinnyF8Waves;
// the few-row GEMM of e4m3 models likewise (HIPDEC_NO_SKINNY_F8=1: the general few-row kernel)
bool pf_use_skinny_f8(int K) {
    static const bool off = [] { const char *v = getenv("HIPDEC_NO_SKINNY_F8"); return v && v[0] == '1'; }();
    return !off && K % 64 == 0;
}
bool pf_use_dl(int wt, int T, int K, int act) {
    static const bool off = getenv("HIPDEC_NO_DL_GEMM") != nullptr;
    return !off && wt == WT_BF16 && T >= kDlMinRows && K % PF_BKL == 0 && act != PF_ACT_F16;
}
PfSplit pf_split_k(int num_cu, int wt, int T, int N, int K, bool dl = false) {
    if (dl) {
        // One workgroup per CU, so the grid runs in rounds of num_cu workgroups and a partly filled last
        // round costs a whole one.  K splits change the round count: with s splits the work takes
        // ceil(tiles * s / num_cu) rounds of 1/s the length, plus the extra planes written and summed
        // (priced at 5 TB/s against ~1.8 us per 64-element step of a tile).
        const int tiles = ((N + PF_DL_BN - 1) / PF_DL_BN) * ((T + PF_DL_BM - 1) / PF_DL_BM);
        const int lsteps = K / PF_BKL;
        const double t_full = 1.8e-6 * lsteps, t_plane = 2.0 * T * N * 4 / 5e12;
        int best = 1;
        double best_cost = 1e30;
        for (int s = 1; s <= 8 && lsteps / s >= 4; ++s) {
            const int sps = (lsteps + s - 1) / s, ns = (lsteps + sps - 1) / sps;
            const double rounds = (double)(((size_t)tiles * ns + num_cu - 1) / num_cu);
            const double cost = rounds * t_full * sps / lsteps + (ns - 1) * t_plane;
            if (cost < best_cost * 0.97) { best_cost = cost; best = ns; }
        }
        const int sps = (lsteps + best - 1) / best;
        return PfSplit{(lsteps + sps - 1) / sps, sps};
    }
    const int nsteps = K / PF_BK;
    if (T <= kSkinnyRows && wt == WT_INT4 && pf_use_skinny_i4()) {
        // 4-bit weights: a workgroup owns kSkinnyI4Bn weight rows and every wave walks the whole K range of its
        // split; a split is a whole number of 128-element scale groups (four steps each), a multiple of four
        // of them where the staged activation slice (hi + lo) fits the LDS budget with that (the kernel then
        // reads a round's four scales of a row as one aligned load).  Aim at a few workgroups per CU.
        const int tiles = (N + kSkinnyI4Bn - 1) / kSkinnyI4Bn, groups = K / 128;
        int s = std::max(1, (kSkinnyI4WgsPerCu * num_cu + tiles - 1) / tiles);
        const int max_groups = std::min(PF_SQ_GU, std::max(1, ((kSkinnyLdsBytes / (4 * T)) - PF_SK_PAD) / 128));
        int gps = std::min(max_groups, std::max(1, (groups + s - 1) / s));
        if (gps >= 4) gps &= ~3;
        else if (max_groups >= 4) gps = 4;
        return PfSplit{(groups + gps - 1) / gps, 4 * gps};
    }
    if (T <= kSkinnyRows && wt == WT_FP8 && pf_use_skinny_f8(K)) {
        // e4m3 weights: kSkinnyF8Bn weight rows per workgroup, every wave walks the whole K range of its split, a
        // split is a whole number of 64-element blocks, at most PF_S8_GU of them (what the kernel requests at once)
        // and that many where the staged activation slice fits the LDS budget
        const int tiles = (N + kSkinnyF8Bn - 1) / kSkinnyF8Bn, blocks = K / 64;
        const int s = std::max(1, (kSkinnyI4WgsPerCu * num_cu + tiles - 1) / tiles);
        const int max_blocks = std::min(PF_S8_GU, std::max(1, ((kSkinnyLdsBytes / (4 * T)) - PF_SK_PAD) / 64));
        int bps = std::min(max_blocks, std::max(1, (blocks + s - 1) / s));
        if (max_blocks >= PF_S8_GU) bps = PF_S8_GU;
        return PfSplit{(blocks + bps - 1) / bps, 2 * bps};
    }
    if (T <= kSkinnyRows) {
        // 4 waves per workgroup share a K range; aim at ~8 waves per CU over the whole grid
        const int tiles = (N + 31) / 32;
        int s = std::max(1, (2 * num_cu) / tiles);
        s = std::min(s, std::max(1, nsteps / 8));
        // the workgroup's slice of the activation rows (hi + lo) has to fit its LDS budget
        int max_steps = std::max(1, ((kSkinnyLdsBytes / (4 * T)) - PF_SK_PAD) / PF_BK);
        if (wt == WT_INT4) max_steps = std::max(4, max_steps & ~3);   // a split covers whole scale groups (four steps each)
        s = std::max(s, (nsteps + max_steps - 1) / max_steps);
        int sps = (nsteps + s - 1) / s;
        if (wt == WT_INT4) sps = std::min(max_steps, (sps + 3) & ~3);
        return PfSplit{(nsteps + sps - 1) / sps, sps};
    }
    const int bn = PF_BN_OF(wt);
    const int tiles = ((N + bn - 1) / bn) * ((T + PF_BM - 1) / PF_BM);
    const int lsteps = (K + PF_BKL - 1) / PF_BKL;
    int s = (2 * num_cu + tiles - 1) / tiles;
    s = std::min(s, 8);
    s = std::min(s, std::max(1, lsteps / 4));
    s = std::max(s, 1);
    int sps = (lsteps + s - 1) / s;
    if (wt == WT_INT4) sps = (sps + 1) & ~1;       // a split covers whole scale groups (two steps each)
    return PfSplit{(lsteps + sps - 1) / sps, sps};
}
PfSplit pf_split_k(const hipdec_model *m, int wt, int T, int N, int K, bool dl = false) { return pf_split_k(m->num_cu, wt, T, N, K, dl); }

// What one product launches: which kernel, its grid, workgroup size and dynamic LDS, and the K splits (= planes
// written).  pf_gemm launches exactly this; hipdec_debug_gemm_plan hands it to tests, which check it against
// what the kernels assume without a GPU.
enum { PF_K_TILED = 0, PF_K_DL = 1, PF_K_FEW = 2, PF_K_FEW_I4 = 3, PF_K_FEW_F8 = 4 };
struct PfPlan { int kernel, splits, steps_per_split; unsigned gx, gy, gz, threads; size_t lds; };
PfPlan pf_plan(int num_cu, int wt, int T, int N, int K, int act) {
    if (pf_use_dl(wt, T, K, act)) {
        const PfSplit sp = pf_split_k(num_cu, wt, T, N, K, true);
        return PfPlan{PF_K_DL, sp.splits, sp.steps_per_split, (unsigned)((N + PF_DL_BN - 1) / PF_DL_BN),
                      (unsigned)((T + PF_DL_BM - 1) / PF_DL_BM), (unsigned)sp.splits, 64 * PF_DL_WAVES, 0};
    }
    const PfSplit sp = pf_split_k(num_cu, wt, T, N, K);
    // the few-row kernels stage [hi | lo][T][steps_per_split * PF_BK + PF_SK_PAD] bf16 values
    const size_t staged = (size_t)2 * T * (sp.steps_per_split * PF_BK + PF_SK_PAD) * 2;
    if (T <= kSkinnyRows && wt == WT_INT4 && pf_use_skinny_i4())
        return PfPlan{PF_K_FEW_I4, sp.splits, sp.steps_per_split, (unsigned)((N + kSkinnyI4Bn - 1) / kSkinnyI4Bn),
                      (unsigned)sp.splits, 1, 64 * kSkinnyI4Waves, staged};
    if (T <= kSkinnyRows && wt == WT_FP8 && pf_use_skinny_f8(K))
        return PfPlan{PF_K_FEW_F8, sp.splits, sp.steps_per_split, (unsigned)((N + kSkinnyF8Bn - 1) / kSkinnyF8Bn), (unsigned)sp.splits, 1,
                      64 * kSkinnyF8Waves, staged};
    if (T <= kSkinnyRows)
        return PfPlan{PF_K_FEW, sp.splits, sp.steps_per_split, (unsigned)((N + 31) / 32), (unsigned)sp.splits, 1, 256, staged};
    const int bn = PF_BN_OF(wt);
    return PfPlan{PF_K_TILED, sp.splits, sp.steps_per_split, (unsigned)((N + bn - 1) / bn), (unsigned)((T + PF_BM - 1) / PF_BM),
                  (unsigned)sp.splits, 256, 0};
}

int pf_ensure(hipdec_model *m, int T, bool with_head = false) {
    const hipdec_config &c = m->cfg;
    const size_t D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden;
    PrefillWork &w = m->pf;
    int rc;
    if (w.rows < T) {
        // (a step of samples or requests has up to kRequestRows rows, also where the window has fewer positions)
        const size_t R = std::max<size_t>(std::min<size_t>(kPrefillMaxRows, c.seq), kRequestRows);
        if ((rc = dalloc(m, &w.ids, R * 4))) return rc;
        if ((rc = dalloc(m, &w.x, R * D * 4))) return rc;
        if ((rc = dalloc(m, &w.x2, R * D * 4))) return rc;
        if ((rc = dalloc(m, &w.q, R * Q * 4))) return rc;
        if ((rc = dalloc(m, &w.xn_hi, R * D * 2))) return rc;
        if ((rc = dalloc(m, &w.xn_lo, R * D * 2))) return rc;
        if ((rc = dalloc(m, &w.att_hi, R * Q * 2))) return rc;
        if ((rc = dalloc(m, &w.att_lo, R * Q * 2))) return rc;
        if ((rc = dalloc(m, &w.gate_hi, R * H * 2))) return rc;
        if ((rc = dalloc(m, &w.gate_lo, R * H * 2))) return rc;
        if ((rc = dalloc(m, &w.ssq, R * ((D + PF_CHUNK - 1) / PF_CHUNK) * 4))) return rc;
        if (!w.h_ids) HCHK(hipHostMalloc((void **)&w.h_ids, R * 4));
        w.rows = (int)R;
    }
    size_t need = 0;
    const int dims[4][2] = {{(int)(Q + 2 * KV), (int)D}, {(int)D, (int)Q}, {(int)(2 * H), (int)D}, {(int)D, (int)H}};
    for (auto &d : dims) {
        need = std::max(need, (size_t)pf_split_k(m, m->wt, T, d[0], d[1]).splits * T * d[0]);
        if (pf_use_dl(m->wt, T, d[1], PF_ACT_PAIR))
            need = std::max(need, (size_t)pf_split_k(m, m->wt, T, d[0], d[1], true).splits * T * d[0]);
    }
    if (with_head) need = std::max(need, (size_t)pf_split_k(m, m->embed_wt, T, (int)c.vocab, (int)D).splits * T * c.vocab);
    if (need > w.P_floats) {
        if ((rc = dalloc(m, &w.P, need * 4))) return rc;
        w.P_floats = need;
    }
    return HIPDEC_OK;
}

// P[z][t][n] = sum over the z-th K slice of A[t][k] * W[n][k]; returns the number of planes
// act: PF_ACT_* of the activation arrays (the few-row kernel only takes pairs)
int pf_gemm(hipdec_model *m, int wt, const uint16_t *Ahi, const uint16_t *Alo, const void *W, const void *scales,
            int T, int N, int K, int act = PF_ACT_PAIR) {
    const PfPlan p = pf_plan(m->num_cu, wt, T, N, K, act);
    const dim3 grid(p.gx, p.gy, p.gz), block(p.threads);
    const size_t lds = p.lds;
    PfGemm g{Ahi, Alo, W, wt == WT_INT4 && p.kernel != PF_K_DL ? (const uint16_t *)scales : nullptr, m->pf.P, T, N, K, p.steps_per_split};
    switch (p.kernel) {
    case PF_K_DL:
        if (act == PF_ACT_PAIR) hipLaunchKernelGGL((k_pf_gemm_dl<true, PF_BKL, 2, PF_DL_WAVES, 1>), grid, block, 0, m->stream, g);
        else hipLaunchKernelGGL((k_pf_gemm_dl<false, PF_BKL, 3, PF_DL_WAVES, 1>), grid, block, 0, m->stream, g);
        break;
    case PF_K_FEW_I4:
        if (T <= 8) hipLaunchKernelGGL((k_pf_gemm_skinny_i4<1, true, kSkinnyI4Nt, kSkinnyI4Waves>), grid, block, lds, m->stream, g);
        else if (T <= 16) hipLaunchKernelGGL((k_pf_gemm_skinny_i4<1, false, kSkinnyI4Nt, kSkinnyI4Waves>), grid, block, lds, m->stream, g);
        else hipLaunchKernelGGL((k_pf_gemm_skinny_i4<2, false, kSkinnyI4Nt, kSkinnyI4Waves>), grid, block, lds, m->stream, g);
        break;
    case PF_K_FEW_F8:
        if (T <= 8) hipLaunchKernelGGL((k_pf_gemm_skinny_f8<1, true, kSkinnyF8Waves>), grid, block, lds, m->stream, g);
        else if (T <= 16) hipLaunchKernelGGL((k_pf_gemm_skinny_f8<1, false, kSkinnyF8Waves>), grid, block, lds, m->stream, g);
        else hipLaunchKernelGGL((k_pf_gemm_skinny_f8<2, false, kSkinnyF8Waves>), grid, block, lds, m->stream, g);
        break;
    case PF_K_FEW:
        if (wt == WT_F32) hipLaunchKernelGGL(k_pf_gemm_skinny<WT_F32>, grid, block, lds, m->stream, g);
        else if (wt == WT_BF16) hipLaunchKernelGGL(k_pf_gemm_skinny<WT_BF16>, grid, block, lds, m->stream, g);
        else if (wt == WT_FP8) hipLaunchKernelGGL(k_pf_gemm_skinny<WT_FP8>, grid, block, lds, m->stream, g);
        else hipLaunchKernelGGL(k_pf_gemm_skinny<WT_INT4>, grid, block, lds, m->stream, g);
        break;
    default:
#define PFG(WTX) do { if (act == PF_ACT_F16) hipLaunchKernelGGL((k_pf_gemm<WTX, PF_ACT_F16>), grid, block, 0, m->stream, g); \
                      else if (act == PF_ACT_BF16) hipLaunchKernelGGL((k_pf_gemm<WTX, PF_ACT_BF16>), grid, block, 0, m->stream, g); \
                      else hipLaunchKernelGGL((k_pf_gemm<WTX, PF_ACT_PAIR>), grid, block, 0, m->stream, g); } while (0)
        if (wt == WT_BF16) PFG(WT_BF16);
        else if (wt == WT_FP8) PFG(WT_FP8);
        else PFG(WT_INT4);
#undef PFG
        break;
    }
    return p.splits;
}

// launches shared by the prompt prefill and the multi-sample step
void pf_launch_embed(hipdec_model *m, int T, int f16 = 0) {
    PrefillWork &w = m->pf;
    const int D = (int)m->cfg.dim;
    dim3 grid((D + PF_CHUNK - 1) / PF_CHUNK, T), block(PF_CHUNK);
    if (m->embed_wt == WT_F32)
        hipLaunchKernelGGL(k_pf_embed<WT_F32>, grid, block, 0, m->stream, m->embed, w.ids, w.x, m->layers[0].g1, w.xn_hi,
                           w.xn_lo, w.ssq, D, f16);
    else
        hipLaunchKernelGGL(k_pf_embed<WT_BF16>, grid, block, 0, m->stream, m->embed, w.ids, w.x, m->layers[0].g1, w.xn_hi,
                           w.xn_lo, w.ssq, D, f16);
}
void pf_launch_resid(hipdec_model *m, int T, int splits, const void *wscale, const float *resid, float *out,
                     const float *gamma, int f16 = 0) {
    PrefillWork &w = m->pf;
    const int D = (int)m->cfg.dim;
    const int nch = (D + PF_CHUNK - 1) / PF_CHUNK;
    dim3 grid((nch + 3) / 4, T), block(256);
    hipLaunchKernelGGL(k_pf_resid, grid, block, 0, m->stream, w.P, splits, (size_t)T * D,
                       m->wt == WT_FP8 ? (const float *)wscale : nullptr, resid, m->alpha, out, gamma, w.xn_hi, w.xn_lo,
                       w.ssq, D, nch, f16);
}
void pf_launch_gate(hipdec_model *m, int T, int splits, const void *wscale, int f16 = 0) {
    PrefillWork &w = m->pf;
    const int D = (int)m->cfg.dim, H = (int)m->cfg.hidden;
    hipLaunchKernelGGL(k_pf_gate_epi, dim3((unsigned)((H / 4 + 255) / 256), (unsigned)T), dim3(256), 0, m->stream, w.P, splits,
                       (size_t)T * 2 * H, m->wt == WT_FP8 ? (const float *)wscale : nullptr, w.gate_hi, w.gate_lo, w.ssq,
                       (D + PF_CHUNK - 1) / PF_CHUNK, D, T, H, (int)m->opt.ffn_activation, f16);
}

// Runs prompt rows ids[0..n) at positions len .. len+n-1 through every layer, chunk by chunk; on
// return the caches hold their keys and values and *x_last points at the residual stream of the
// last row (device memory).
int prefill_batched(hipdec_model *m, const uint32_t *ids, size_t n, const float **x_last) {
    const hipdec_config &c = m->cfg;
    const int D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden;
    const int gqa = c.gqa_ratio ? c.gqa_ratio : 1;
    const float scale = 1.0f / sqrtf((float)c.hd);
    size_t done = 0;
    while (done < n) {
        const int T = (int)std::min<size_t>(n - done, m->wt == WT_F32 ? kSkinnyRows : kPrefillMaxRows);
        const int pos0 = (int)(m->len + done);
        int rc = pf_ensure(m, T);
        if (rc) return rc;
        PrefillWork &w = m->pf;
        HCHK(hipStreamSynchronize(m->stream));                  // the pinned id buffer is free again
        memcpy(w.h_ids, ids + done, (size_t)T * 4);
        HCHK(hipMemcpyAsync(w.ids, w.h_ids, (size_t)T * 4, hipMemcpyHostToDevice, m->stream));
        // how this chunk's activations travel between its kernels (the few-row GEMM only takes pairs)
        const bool tiled = T > kSkinnyRows;
        // (mode 3: the pair into the q/k/v and output projections, the hi parts alone into the two feed-forward products)
        const int act = !tiled ? PF_ACT_PAIR : m->pf_act == 3 ? PF_ACT_PAIR : m->pf_act;
        const int act_ffn = !tiled ? PF_ACT_PAIR : m->pf_act == 3 ? PF_ACT_BF16 : m->pf_act;
        const int f16 = act == PF_ACT_F16;
        pf_launch_embed(m, T, f16);
        const int nch = (D + PF_CHUNK - 1) / PF_CHUNK;
        for (uint32_t l = 0; l < c.nlayers; ++l) {
            const DevLayer &L = m->layers[l];
            const bool fp8 = m->wt == WT_FP8;
            // q/k/v projections, RoPE, cache append
            int N = Q + 2 * KV;
            int sp = pf_gemm(m, m->wt, w.xn_hi, w.xn_lo, L.wqkv, L.s_qkv, T, N, D, act);
            {
                dim3 grid((unsigned)((N / 4 + 255) / 256), (unsigned)T), block(256);
                if (m->kvbf16)
                    hipLaunchKernelGGL(k_pf_qkv_epi<1>, grid, block, 0, m->stream, w.P, sp, (size_t)T * N,
                                       fp8 ? (const float *)L.s_qkv : nullptr, w.q, L.kc, L.vc, m->rope_cos, m->rope_sin,
                                       w.ssq, nch, D, T, Q, KV, (int)c.hd, pos0);
                else
                    hipLaunchKernelGGL(k_pf_qkv_epi<0>, grid, block, 0, m->stream, w.P, sp, (size_t)T * N,
                                       fp8 ? (const float *)L.s_qkv : nullptr, w.q, L.kc, L.vc, m->rope_cos, m->rope_sin,
                                       w.ssq, nch, D, T, Q, KV, (int)c.hd, pos0);
            }
            // causal attention of the chunk's rows over positions 0 .. pos0 + t
            {
                dim3 grid((T + 31) / 32, c.heads), block(64 * PF_ATT_WAVES);
#define PFATT(KVB, HD)                                                                                             \
    hipLaunchKernelGGL((k_pf_attn<KVB, HD>), grid, block, 0, m->stream, w.q, L.kc, L.vc, w.att_hi, w.att_lo, T, Q, KV, \
                       gqa, pos0, (int)c.seq, scale, f16)
                if (m->kvbf16) { if (c.hd == 64) PFATT(1, 64); else PFATT(1, 128); }
                else { if (c.hd == 64) PFATT(0, 64); else PFATT(0, 128); }
#undef PFATT
            }
            // output projection, residual, second norm
            sp = pf_gemm(m, m->wt, w.att_hi, w.att_lo, L.wo, L.s_wo, T, D, Q, act);
            pf_launch_resid(m, T, sp, L.s_wo, w.x, w.x2, L.g2, f16);
            // gate/up, activation
            sp = pf_gemm(m, m->wt, w.xn_hi, w.xn_lo, L.w13, L.s_w13, T, 2 * H, D, act_ffn);
            pf_launch_gate(m, T, sp, L.s_w13, f16);
            // down projection, residual, next layer's first norm
            sp = pf_gemm(m, m->wt, w.gate_hi, w.gate_lo, L.w2, L.s_w2, T, D, H, act_ffn);
            pf_launch_resid(m, T, sp, L.s_w2, w.x2, w.x, l + 1 < c.nlayers ? m->layers[l + 1].g1 : nullptr, f16);
        }
        HCHK(hipGetLastError());
        *x_last = w.x + (size_t)(T - 1) * D;
        done += T;
    }
    return HIPDEC_OK;
}

// ---- multi-sample decode (hipdec_batch.h)
constexpr int kBatchMaxRows = 32;
static_assert(kBatchMaxRows <= kRequestRows, "pf_ensure makes room for both");

int batch_alloc(hipdec_model *m, int rows) {
    const hipdec_config &c = m->cfg;
    BatchState &b = m->bt;
    if (b.cap_rows >= rows) return HIPDEC_OK;
    int rc;
    const size_t esz = m->kvbf16 ? 2 : 4, V = c.vocab, blocks = (size_t)m->blocks;
    b.suf_rows = c.seq;
    b.kc_suf.assign(c.nlayers, nullptr);
    b.vc_suf.assign(c.nlayers, nullptr);
    for (uint32_t l = 0; l < c.nlayers; ++l) {
        if ((rc = dalloc(m, &b.kc_suf[l], (size_t)rows * b.suf_rows * c.kv_dim * esz))) return rc;
        if ((rc = dalloc(m, &b.vc_suf[l], (size_t)rows * b.suf_rows * c.kv_dim * esz))) return rc;
    }
    if (!b.d_bp) { if ((rc = dalloc(m, &b.d_bp, sizeof(BatchParams)))) return rc; }
    if (!b.h_bp) HCHK(hipHostMalloc((void **)&b.h_bp, sizeof(BatchParams)));
    if ((rc = dalloc(m, &b.logits, (size_t)rows * V * 4))) return rc;
    if ((rc = dalloc(m, &b.d_out, (size_t)rows * V * 4))) return rc;
    if ((rc = dalloc(m, &b.d_vals, (size_t)rows * blocks * HIPDEC_MAX_GPU_TOPK * 4))) return rc;
    if ((rc = dalloc(m, &b.d_idxs, (size_t)rows * blocks * HIPDEC_MAX_GPU_TOPK * 4))) return rc;
    if ((rc = dalloc(m, &b.d_bmax, (size_t)rows * blocks * 4))) return rc;
    if ((rc = dalloc(m, &b.d_bsum, (size_t)rows * blocks * 4))) return rc;
    if ((rc = dalloc(m, &b.d_tok, (size_t)rows * 4))) return rc;
    b.ring_elems = (size_t)rows * c.seq;
    if ((rc = dalloc(m, &b.d_ring, b.ring_elems * 4))) return rc;
    if (b.h_ring) (void)hipHostFree(b.h_ring);
    HCHK(hipHostMalloc((void **)&b.h_ring, b.ring_elems * 4));
    if (b.h_stage) (void)hipHostFree(b.h_stage);
    b.h_stage_floats = (size_t)rows * std::max(V, 2 * blocks * HIPDEC_MAX_GPU_TOPK);
    HCHK(hipHostMalloc((void **)&b.h_stage, b.h_stage_floats * 4));
    b.cap_rows = rows;
    return HIPDEC_OK;
}

// ---- the layers of a multi-row step as one persistent launch (hipdec_rows.h)
bool rows_kernel_fits(const hipdec_model *m, int R) {
    const hipdec_config &c = m->cfg;
    if (!m->mega_ok || m->bt.rows_off || m->wt != WT_BF16 || R > ROWS_MAX_R) return false;
    if (m->opt.flags & HIPDEC_FLAG_NO_MEGA) return false;
    if (const char *v = getenv("HIPDEC_NO_ROWS_KERNEL")) if (v[0] == '1') return false;
    const int G = m->mega_grid;
    const long D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, N = Q + 2 * KV;
    if (D % 256 || Q % 256 || H % 256 || N % 2) return false;
    if (D / 256 > ROWS_JA || Q / 256 > ROWS_JB || H / 256 > ROWS_JB || G % 4) return false;
    auto band = [&](long rows) { return 2 * ((rows / 2 + G - 1) / G); };          // widest band of a product with `rows` rows
    if (band(N) > 16 * ROWS_TA || band(2 * H) > 16 * ROWS_TA || band(D) > 16 * ROWS_TB) return false;
    if (std::max(std::max(N * D, 2 * H * D), std::max(D * Q, D * H)) * 2 >= (1L << 31) - 65536) return false;   // descriptors and 32-bit offsets
    if ((long)R * c.heads > G) return false;
    if (c.hd != 64 && c.hd != 128) return false;
    // (the kernel's static LDS comes on top of this: the same margin as the single-row kernel keeps)
    return rows_lds(ROWS_MAX_R, (int)D, (int)Q, (int)KV, (int)H, (int)c.nlayers, (int)c.hd, G).total <= 160 * 1024 - 2048;
}

int rows_prepare(hipdec_model *m, int R) {
    const hipdec_config &c = m->cfg;
    BatchState &b = m->bt;
    b.rows_active = false;
    if (!rows_kernel_fits(m, R)) return HIPDEC_OK;
    const int G = m->mega_grid;
    const size_t D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, REC = c.hd + MEGA_PREC;
    if (!b.rows_ready) {
        const int ns_cap = G;                                     // one row, one head: every workgroup a split
        const size_t xb[6] = {ROWS_MAX_R * D * 4, ROWS_MAX_R * D * 4, ROWS_MAX_R * (Q + 2 * KV) * 4, ROWS_MAX_R * H * 4,
                              (size_t)ns_cap * REC * 4, (size_t)G * 4};
        size_t xoff[6], total = 0;
        for (int i = 0; i < 6; ++i) { xoff[i] = total; total += (xb[i] + 255) & ~(size_t)255; }
        // (a slab taken by an earlier attempt that failed further down is used again, not taken twice)
        if (!b.rows_slab) b.rows_slab = uncached_take(m->opt.device, total, &b.rows_slab_cap);
        if (!b.rows_slab) return HIPDEC_OK;                        // no uncached memory: the step stays as it is
        b.rows_slab_bytes = total;
        char *base = (char *)b.rows_slab;
        RowsArgs &a = b.rows_args;
        a.X = (float *)(base + xoff[0]); a.X2 = (float *)(base + xoff[1]); a.QKV = (float *)(base + xoff[2]);
        a.GATE = (float *)(base + xoff[3]); a.PART = (float *)(base + xoff[4]); a.XT = (unsigned *)(base + xoff[5]);
        int rc;
        {
            // the XCDs' own copies of X, X2, GATE and the folded attention output
            const size_t cf[4] = {xb[0] / 4, xb[1] / 4, xb[3] / 4, ROWS_MAX_R * Q};
            size_t off[4], stride = 0;
            for (int i = 0; i < 4; ++i) { off[i] = stride; stride += (cf[i] + 63) & ~(size_t)63; }
            b.rows_xb_bytes = (size_t)ROWS_XCD_COPIES * stride * 4;
            if (!b.rows_xb && (rc = dalloc(m, &b.rows_xb, b.rows_xb_bytes))) return rc;
            a.XB = b.rows_xb; a.xb_stride = (int)stride; a.xb_copies = ROWS_XCD_COPIES;
            a.xb_x = (int)off[0]; a.xb_x2 = (int)off[1]; a.xb_gate = (int)off[2]; a.xb_att = (int)off[3];
        }
        if (!b.rows_epochs && (rc = dalloc(m, &b.rows_epochs, 16))) return rc;
        if (!b.rows_suf && (rc = dalloc(m, &b.rows_suf, (size_t)2 * c.nlayers * sizeof(void *)))) return rc;
        a.layers = m->mega.layers; a.gfinal = m->gfinal; a.rope_cos = m->rope_cos; a.rope_sin = m->rope_sin;
        a.kc_suf = b.rows_suf; a.vc_suf = b.rows_suf + c.nlayers;
        a.bp = b.d_bp; a.epochs = b.rows_epochs; a.abort = m->d_abort + 16;
        a.D = (int)D; a.Q = (int)Q; a.KV = (int)KV; a.H = (int)H; a.L = (int)c.nlayers; a.heads = (int)c.heads;
        a.gqa = c.gqa_ratio ? (int)c.gqa_ratio : 1; a.act = (int)m->opt.ffn_activation; a.alpha = m->alpha;
        const int lds_max = rows_lds(ROWS_MAX_R, a.D, a.Q, a.KV, a.H, a.L, (int)c.hd, G).total;
        hipError_t e;
#define ROWS_ATTR(KVB, HD)                                                                                          \
    do {                                                                                                            \
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_rows<KVB, HD, MEGA_VAR_PLAIN>),                   \
                                hipFuncAttributeMaxDynamicSharedMemorySize, lds_max);                               \
        if (e == hipSuccess)                                                                                        \
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_rows<KVB, HD, MEGA_VAR_STAMPS>),              \
                                    hipFuncAttributeMaxDynamicSharedMemorySize, lds_max);                           \
    } while (0)
        if (m->kvbf16) { if (c.hd == 64) ROWS_ATTR(1, 64); else ROWS_ATTR(1, 128); }
        else { if (c.hd == 64) ROWS_ATTR(0, 64); else ROWS_ATTR(0, 128); }
#undef ROWS_ATTR
        if (e != hipSuccess) { (void)hipGetLastError(); b.rows_off = true; return HIPDEC_OK; }
        b.rows_ready = true;
    }
    RowsArgs &a = b.rows_args;
    if (b.rows_suf_seen != b.kc_suf[0]) {                         // (the suffix caches are reallocated when the row capacity grows)
        std::vector<void *> t(2 * c.nlayers);
        for (uint32_t l = 0; l < c.nlayers; ++l) { t[l] = b.kc_suf[l]; t[c.nlayers + l] = b.vc_suf[l]; }
        HCHK(hipStreamSynchronize(m->stream));
        HCHK(hipMemcpy(b.rows_suf, t.data(), t.size() * sizeof(void *), hipMemcpyHostToDevice));
        b.rows_suf_seen = b.kc_suf[0];
    }
    // A batch starts from exchange buffers without stamps and from epoch 0 (layer 0 then expects stamp 1):
    // the row count may differ from the last batch's, and rows it did not have would carry stamps of unknown age.
    HCHK(hipMemsetAsync(b.rows_slab, 0, b.rows_slab_bytes, m->stream));
    HCHK(hipMemsetAsync(b.rows_xb, 0, b.rows_xb_bytes, m->stream));
    HCHK(hipMemsetAsync(b.rows_epochs, 0, 16, m->stream));
    a.R = R;
    a.ns_max = std::max(1, std::min(G / (R * (int)c.heads), 64));
    a.suf_rows = b.suf_rows;
    b.rows_active = true;
    return HIPDEC_OK;
}

// after a wait for the stream: a persistent multi-row launch that gave up leaves the abort flag set
int rows_check(hipdec_model *m) {
    BatchState &b = m->bt;
    if (!b.rows_active) return HIPDEC_OK;
    const unsigned flag = __atomic_load_n(&m->h_abort[16], __ATOMIC_ACQUIRE);
    if (!flag) return HIPDEC_OK;
    __atomic_store_n(&m->h_abort[16], 0u, __ATOMIC_RELEASE);
    b.rows_off = true;
    b.rows_active = false;
    for (auto &g : b.graphs) if (g) { (void)hipGraphExecDestroy(g); g = nullptr; }
    return fail(m, HIPDEC_ERR_HIP, "multi-row step kernel: a wait timed out (the batch has to be reopened; later steps use one kernel per product)");
}

void batch_enqueue(hipdec_model *m, int variant);

bool profiler_attached() {
    static const bool on = [] {
        for (const char *name : {"ROCP_TOOL_LIBRARIES", "HSA_TOOLS_LIB", "ROCP_TOOL_LIB"}) {
            const char *v = getenv(name);
            if (v && v[0]) return true;
        }
        for (char **e = environ; e && *e; ++e)                      // rocprofv3 / rocprofiler-sdk configure their tool through these
            if (!strncmp(*e, "ROCPROF_", 8) || !strncmp(*e, "ROCPROFILER_", 12)) return true;
        return false;
    }();
    return on;
}

// Everything that changes from step to step (tokens, position, sampler parameters) lives in device
// memory, so the ~210 launches of a step are captured once per (rows, head variant) and replayed.
int batch_launch(hipdec_model *m, int variant) {
    BatchState &b = m->bt;
    const int R = b.rows;
    // Replaying the step's ~210-node graph under rocprofv3's kernel trace ended once in a segmentation
    // fault inside the HIP runtime (cause not established): with a profiler tool library in the process
    // the step is launched kernel by kernel instead.  The one-launch layer kernel's graphs are a few nodes.
    if ((m->opt.flags & HIPDEC_FLAG_NO_GRAPH) || (profiler_attached() && !b.rows_active)) {
        batch_enqueue(m, variant);
        HCHK(hipGetLastError());
        return HIPDEC_OK;
    }
    if (b.graph_rows != R) {
        for (auto &g : b.graphs) if (g) { (void)hipGraphExecDestroy(g); g = nullptr; }
        b.graph_rows = R;
    }
    if (!b.graphs[variant]) {
        hipGraph_t g = nullptr;
        HCHK(hipStreamBeginCapture(m->stream, hipStreamCaptureModeThreadLocal));
        batch_enqueue(m, variant);
        hipError_t e = hipStreamEndCapture(m->stream, &g);
        if (e != hipSuccess || !g) { m->err = std::string("graph capture failed: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
        HCHK(hipGraphInstantiate(&b.graphs[variant], g, nullptr, nullptr, 0));
        HCHK(hipGraphDestroy(g));
    }
    HCHK(hipGraphLaunch(b.graphs[variant], m->stream));
    return HIPDEC_OK;
}

// one step of every open row: tokens[r] at position prefix + slot
int batch_step(hipdec_model *m, const uint32_t *tokens, int variant, uint32_t top_k, float inv_t, float softcap) {
    const hipdec_config &c = m->cfg;
    BatchState &b = m->bt;
    if (b.rows <= 0) return fail(m, HIPDEC_ERR_ARG, "no batch is open (hipdec_batch_begin)");
    if (!tokens) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if (b.prefix + b.slot >= c.seq) return fail(m, HIPDEC_ERR_FULL, "decode only supports lengths within cfg.seq");
    const int R = b.rows;
    for (int r = 0; r < R; ++r)
        if (tokens[r] >= c.vocab) return fail(m, HIPDEC_ERR_ARG, "token id must fit vocab");
    int rc = pf_ensure(m, R, true);
    if (rc) return rc;
    PrefillWork &w = m->pf;
    HCHK(hipStreamSynchronize(m->stream));                      // pinned staging is free again
    memcpy(w.h_ids, tokens, (size_t)R * 4);
    *b.h_bp = BatchParams{(int)(b.prefix + b.slot), (int)b.slot, (int)b.prefix, (int)top_k, inv_t, softcap};
    HCHK(hipMemcpyAsync(w.ids, w.h_ids, (size_t)R * 4, hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(b.d_bp, b.h_bp, sizeof(BatchParams), hipMemcpyHostToDevice, m->stream));
    HCHK(hipEventRecord(m->ev0, m->stream));
    if ((rc = batch_launch(m, variant))) return rc;
    HCHK(hipEventRecord(m->ev1, m->stream));
    b.slot += 1;
    b.have_logits = true;
    return HIPDEC_OK;
}

// the kernels of one multi-row step (no host-side state changes: safe to capture)
void batch_enqueue(hipdec_model *m, int variant) {
    const hipdec_config &c = m->cfg;
    BatchState &b = m->bt;
    PrefillWork &w = m->pf;
    const int R = b.rows;
    const int D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, V = c.vocab;
    const int gqa = c.gqa_ratio ? c.gqa_ratio : 1;
    const float scale = 1.0f / sqrtf((float)c.hd);
    pf_launch_embed(m, R);
    const int nch = (D + PF_CHUNK - 1) / PF_CHUNK;
    const bool fp8 = m->wt == WT_FP8;
    if (b.rows_active) {
        RowsArgs a = b.rows_args;
        a.x_in = w.x; a.out_hi = w.xn_hi; a.out_lo = w.xn_lo; a.out_ssq = w.ssq;
        const size_t lds = (size_t)rows_lds(R, D, Q, KV, H, (int)c.nlayers, (int)c.hd, m->mega_grid).total;
        dim3 grid(m->mega_grid), block(ROWS_THREADS);
#define ROWS_GO(KVB, HD)                                                                                            \
    do {                                                                                                            \
        if (a.prof) hipLaunchKernelGGL((k_rows<KVB, HD, MEGA_VAR_STAMPS>), grid, block, lds, m->stream, a);         \
        else hipLaunchKernelGGL((k_rows<KVB, HD, MEGA_VAR_PLAIN>), grid, block, lds, m->stream, a);                 \
    } while (0)
        if (m->kvbf16) { if (c.hd == 64) ROWS_GO(1, 64); else ROWS_GO(1, 128); }
        else { if (c.hd == 64) ROWS_GO(0, 64); else ROWS_GO(0, 128); }
#undef ROWS_GO
    }
    for (uint32_t l = 0; l < (b.rows_active ? 0u : c.nlayers); ++l) {
        const DevLayer &L = m->layers[l];
        const int N = Q + 2 * KV;
        int sp = pf_gemm(m, m->wt, w.xn_hi, w.xn_lo, L.wqkv, L.s_qkv, R, N, D);
        {
            const size_t items = (size_t)R * (N / 2);
            dim3 grid((unsigned)((items + 255) / 256)), block(256);
            if (m->kvbf16)
                hipLaunchKernelGGL(k_bd_qkv_epi<1>, grid, block, 0, m->stream, w.P, sp, (size_t)R * N,
                                   fp8 ? (const float *)L.s_qkv : nullptr, w.q, b.kc_suf[l], b.vc_suf[l], b.suf_rows,
                                   m->rope_cos, m->rope_sin, b.d_bp, w.ssq, nch, D, R, Q, KV, (int)c.hd);
            else
                hipLaunchKernelGGL(k_bd_qkv_epi<0>, grid, block, 0, m->stream, w.P, sp, (size_t)R * N,
                                   fp8 ? (const float *)L.s_qkv : nullptr, w.q, b.kc_suf[l], b.vc_suf[l], b.suf_rows,
                                   m->rope_cos, m->rope_sin, b.d_bp, w.ssq, nch, D, R, Q, KV, (int)c.hd);
        }
        {
            dim3 grid(c.heads, R), block(BD_ATT_THREADS);
#define BDATT(KVB, HD)                                                                                             \
    hipLaunchKernelGGL((k_bd_attn<KVB, HD>), grid, block, 0, m->stream, w.q, L.kc, L.vc, b.kc_suf[l], b.vc_suf[l], \
                       b.suf_rows, b.d_bp, w.att_hi, w.att_lo, Q, KV, gqa, scale)
            if (m->kvbf16) { if (c.hd == 64) BDATT(1, 64); else BDATT(1, 128); }
            else { if (c.hd == 64) BDATT(0, 64); else BDATT(0, 128); }
#undef BDATT
        }
        sp = pf_gemm(m, m->wt, w.att_hi, w.att_lo, L.wo, L.s_wo, R, D, Q);
        pf_launch_resid(m, R, sp, L.s_wo, w.x, w.x2, L.g2);
        sp = pf_gemm(m, m->wt, w.xn_hi, w.xn_lo, L.w13, L.s_w13, R, 2 * H, D);
        pf_launch_gate(m, R, sp, L.s_w13);
        sp = pf_gemm(m, m->wt, w.gate_hi, w.gate_lo, L.w2, L.s_w2, R, D, H);
        // the last layer's residual kernel prepares the final norm instead of the next layer's first one
        pf_launch_resid(m, R, sp, L.s_w2, w.x2, w.x, l + 1 < c.nlayers ? m->layers[l + 1].g1 : m->gfinal);
    }
    // tied LM head for every row (full_model.rs:419-428), then the per-row head kernel
    {
        const int sp = pf_gemm(m, m->embed_wt, w.xn_hi, w.xn_lo, m->embed, nullptr, R, V, D);
        const size_t n = (size_t)R * V;
        hipLaunchKernelGGL(k_bd_sum_planes, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, m->stream, w.P, sp, n,
                           b.logits, n, w.ssq, nch, D, V);
    }
    if (variant == B_ARGMAX)
        hipLaunchKernelGGL(k_bd_argmax, dim3(R), dim3(1024), 0, m->stream, b.logits, V, b.d_tok);
    else if (variant == B_TOPK || variant == B_TOPK_S)
        hipLaunchKernelGGL(k_bd_topk, dim3(m->blocks, R), dim3(256), 0, m->stream, b.logits, V, b.d_bp, b.d_vals, b.d_idxs);
    else if (variant == B_STATS || variant == B_STATS_S)
        hipLaunchKernelGGL(k_bd_block_stats, dim3(m->blocks, R), dim3(256), 0, m->stream, b.logits, V, b.d_bp, b.d_bmax,
                           b.d_bsum);
    // the draw on the device: each row's token goes where the next step's embedding lookup reads it
    if (variant == B_TOPK_S)
        hipLaunchKernelGGL(k_sample_topk, dim3(R), dim3(256), 0, m->stream, b.d_vals, b.d_idxs, m->blocks, m->d_ss, m->d_rng,
                           w.ids, b.d_ring, b.d_bp);
    else if (variant == B_STATS_S)
        hipLaunchKernelGGL(k_sample_fullvocab, dim3(R), dim3(256), 0, m->stream, b.logits, V, b.d_bmax, b.d_bsum, m->blocks,
                           m->d_ss, m->d_rng, w.ids, b.d_ring, b.d_bp);
}

// copies `floats` values from device memory to the caller through the pinned staging buffer
int batch_fetch(hipdec_model *m, const void *dev, void *host, size_t floats) {
    BatchState &b = m->bt;
    if (floats > b.h_stage_floats) return fail(m, HIPDEC_ERR_ARG, "internal: staging buffer too small");
    HCHK(hipMemcpyAsync(b.h_stage, dev, floats * 4, hipMemcpyDeviceToHost, m->stream));
    HCHK(hipStreamSynchronize(m->stream));
    int rc = rows_check(m);
    if (rc) return rc;
    HCHK(hipEventElapsedTime(&m->last_ms, m->ev0, m->ev1));
    m->step_timed = false;
    memcpy(host, b.h_stage, floats * 4);
    return HIPDEC_OK;
}

// ---- requests of their own prompts stepped together over a paged cache (hipdec_requests.h)
// an operator's refusal or failure as this model's
#define OPCHK(expr) do { const int rc_ = (expr); if (rc_ != HIPDEC_OK) { g_op_failed = false; return fail(m, rc_, g_op_error.c_str()); } } while (0)

hipdec_paged_cache request_cache(const hipdec_model *m, uint32_t layer) {
    const RequestState &r = m->rq;
    const hipdec_config &c = m->cfg;
    const int64_t page = (int64_t)1 << r.page_shift;
    return hipdec_paged_cache{r.k[layer], r.v[layer], m->opt.kv_dtype, (uint32_t)page, r.n_pages, c.kv_heads, c.hd, r.max_seqs,
                              (uint32_t)r.max_pages, r.d_table, page * c.kv_dim, (int64_t)c.kv_dim, (int64_t)c.hd};
}

int requests_open(hipdec_model *m, uint32_t page_size, uint32_t n_pages, uint32_t max_seqs) {
    const hipdec_config &c = m->cfg;
    RequestState &r = m->rq;
    HCHK(hipSetDevice(m->opt.device));
    while ((1u << r.page_shift) < page_size) ++r.page_shift;
    r.max_pages = (int)((c.seq + page_size - 1) >> r.page_shift);
    r.n_pages = n_pages;
    r.max_seqs = max_seqs;
    int rc;
    const size_t bytes = (size_t)n_pages * page_size * c.kv_dim * (m->kvbf16 ? 2 : 4), N = c.q_dim + 2 * c.kv_dim, R = kRequestRows;
    r.k.resize(c.nlayers, nullptr);
    r.v.resize(c.nlayers, nullptr);
    for (uint32_t l = 0; l < c.nlayers; ++l) {
        if ((rc = dalloc(m, &r.k[l], bytes))) return rc;
        if ((rc = dalloc(m, &r.v[l], bytes))) return rc;
    }
    r.table.assign((size_t)max_seqs * r.max_pages, -1);
    r.lens.assign(max_seqs, -1);
    r.free_pages.resize(n_pages);
    for (uint32_t i = 0; i < n_pages; ++i) r.free_pages[i] = (int)(n_pages - 1 - i);
    for (uint64_t rows = 1; rows <= R; ++rows) {
        uint64_t need = 0;
        for (uint64_t len = 0; len < c.seq + 128; len += 128) {
            OPCHK(hipdec_attention_paged_workspace(rows, c.heads, c.kv_heads, c.hd, len, &need));
            r.ws_att_bytes = std::max(r.ws_att_bytes, need);
        }
        for (uint32_t k = 0; rows * (k + 1) <= R; ++k) {
            OPCHK(hipdec_verify_drafts_workspace(rows, k, c.vocab, &need));
            r.ws_ver_bytes = std::max(r.ws_ver_bytes, need);
        }
    }
    if ((rc = dalloc(m, &r.d_table, r.table.size() * 4))) return rc;
    if ((rc = dalloc(m, &r.d_rows, 5 * R * 4))) return rc;
    if ((rc = dalloc(m, &r.d_n, R * 4))) return rc;
    if ((rc = dalloc(m, &r.d_freq, c.hd / 2 * sizeof(double)))) return rc;
    if ((rc = dalloc(m, &r.qkv, R * N * 4))) return rc;
    if ((rc = dalloc(m, &r.att, R * c.q_dim * 4))) return rc;
    if ((rc = dalloc(m, &r.logits, R * c.vocab * 4))) return rc;
    if ((rc = dalloc(m, &r.d_u, R * 4))) return rc;
    if ((rc = dalloc(m, &r.d_tok, 2 * R * 4))) return rc;
    if ((rc = dalloc(m, &r.ws_att, r.ws_att_bytes + 16))) return rc;
    if ((rc = dalloc(m, &r.ws_ver, r.ws_ver_bytes + 16))) return rc;
    HCHK(hipHostMalloc((void **)&r.h_rows, 6 * R * 4));
    HCHK(hipHostMalloc((void **)&r.h_u, R * 4));
    HCHK(hipHostMalloc((void **)&r.h_tok, 2 * R * 4));
    // the angles of the model's own table (theta = pos / 10000^(2i / hd) in fp32, lib.rs:1401) as frequencies
    std::vector<double> freq(c.hd / 2);
    for (size_t i = 0; i < freq.size(); ++i) freq[i] = 1.0 / (double)powf(10000.0f, 2.0f * (float)i / (float)c.hd);
    HCHK(hipMemcpy(r.d_freq, freq.data(), freq.size() * sizeof(double), hipMemcpyHostToDevice));
    HCHK(hipMemcpy(r.d_table, r.table.data(), r.table.size() * 4, hipMemcpyHostToDevice));
    r.open = true;
    return HIPDEC_OK;
}

// gives sequence q the pages of positions [0, len); the caller has checked that there are enough
void request_pages(hipdec_model *m, uint32_t q, size_t len) {
    RequestState &r = m->rq;
    int *row = &r.table[(size_t)q * r.max_pages];
    for (size_t p = 0; p << r.page_shift < len; ++p)
        if (row[p] < 0) { row[p] = r.free_pages.back(); r.free_pages.pop_back(); }
}
size_t request_pages_missing(const hipdec_model *m, uint32_t q, size_t len) {
    const RequestState &r = m->rq;
    const int *row = &r.table[(size_t)q * r.max_pages];
    size_t n = 0;
    for (size_t p = 0; p << r.page_shift < len; ++p) n += row[p] < 0;
    return n;
}
// Gives back what sequences hold beyond their lengths, whichever way the call that took pages for them ends: the pages that only
// rejected drafts were written to, and those of a step or an admission that failed.  (The device's table keeps their
// numbers behind the length, where no row looks, until the sequence's next step.  Last page first: the next one given is it.)
struct RequestTrim {
    hipdec_model *m;
    const uint32_t *seqs;
    size_t n;
    ~RequestTrim() {
        RequestState &r = m->rq;
        for (size_t i = 0; i < n; ++i) {
            int *row = &r.table[(size_t)seqs[i] * r.max_pages];
            const long long len = std::max(r.lens[seqs[i]], 0LL);
            for (int p = r.max_pages - 1; p >= 0 && (long long)p << r.page_shift >= len; --p)
                if (row[p] >= 0) { r.free_pages.push_back(row[p]); row[p] = -1; }
        }
    }
};
int request_table_up(hipdec_model *m, uint32_t q) {
    RequestState &r = m->rq;
    const size_t at = (size_t)q * r.max_pages;
    HCHK(hipMemcpyAsync(r.d_table + at, &r.table[at], (size_t)r.max_pages * 4, hipMemcpyHostToDevice, m->stream));
    return HIPDEC_OK;
}

// the layers and the head for R rows whose ids, positions, slots, sequences and lengths are on the device
int requests_forward(hipdec_model *m, int R, size_t max_len) {
    const hipdec_config &c = m->cfg;
    RequestState &r = m->rq;
    PrefillWork &w = m->pf;
    const int D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, V = c.vocab, N = Q + 2 * KV;
    const int nch = (D + PF_CHUNK - 1) / PF_CHUNK;
    const hipdec_rope rope{r.d_freq, c.hd, 1, 1.0f};
    pf_launch_embed(m, R);
    for (uint32_t l = 0; l < c.nlayers; ++l) {
        const DevLayer &L = m->layers[l];
        const hipdec_paged_cache cache = request_cache(m, l);
        int sp = pf_gemm(m, m->wt, w.xn_hi, w.xn_lo, L.wqkv, L.s_qkv, R, N, D);
        hipLaunchKernelGGL(k_rq_qkv_rows, dim3((unsigned)((N / 2 + 255) / 256), (unsigned)R), dim3(256), 0, m->stream, w.P, sp, (size_t)R * N,
                           m->wt == WT_FP8 ? (const float *)L.s_qkv : nullptr, r.qkv, w.ssq, nch, D, N);
        const hipdec_new_rows rows{r.qkv, r.qkv + Q, r.qkv + Q + KV, w.q, HIPDEC_ROWS_F32, c.heads, (uint64_t)R, N, N, N, Q,
                                   r.d_rows, r.d_rows + kRequestRows, r.d_rows + 2 * kRequestRows};
        OPCHK(hipdec_rope_append_paged(&rope, &cache, &rows, m->stream));
        const hipdec_attention_rows att{w.q, r.att, HIPDEC_ROWS_F32, c.heads, (uint64_t)R, Q, Q, r.d_rows + 3 * kRequestRows,
                                        r.d_rows + 2 * kRequestRows, max_len, 1.0f / sqrtf((float)c.hd)};
        OPCHK(hipdec_attention_paged(&cache, &att, r.ws_att, r.ws_att_bytes, m->stream));
        hipLaunchKernelGGL(k_rq_pair, dim3((unsigned)((R * Q + 255) / 256)), dim3(256), 0, m->stream, r.att, w.att_hi, w.att_lo, R * Q);
        sp = pf_gemm(m, m->wt, w.att_hi, w.att_lo, L.wo, L.s_wo, R, D, Q);
        pf_launch_resid(m, R, sp, L.s_wo, w.x, w.x2, L.g2);
        sp = pf_gemm(m, m->wt, w.xn_hi, w.xn_lo, L.w13, L.s_w13, R, 2 * H, D);
        pf_launch_gate(m, R, sp, L.s_w13);
        sp = pf_gemm(m, m->wt, w.gate_hi, w.gate_lo, L.w2, L.s_w2, R, D, H);
        pf_launch_resid(m, R, sp, L.s_w2, w.x2, w.x, l + 1 < c.nlayers ? m->layers[l + 1].g1 : m->gfinal);
    }
    const int sp = pf_gemm(m, m->embed_wt, w.xn_hi, w.xn_lo, m->embed, nullptr, R, V, D);
    const size_t n = (size_t)R * V;
    hipLaunchKernelGGL(k_bd_sum_planes, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, m->stream, w.P, sp, n, r.logits, n, w.ssq, nch, D, V);
    HCHK(hipGetLastError());
    return HIPDEC_OK;
}

// ---- sampled runs that stay on the device (hipdec_sample.h)
float sample_inv_temperature(float temperature) {              // engine/src/decode.rs:174
    const float tiny = 1.17549435e-38f;                        // f32::MIN_POSITIVE
    return 1.0f / (temperature > tiny ? temperature : tiny);
}

// The device draws are only offered where the restated expf/tanhf equal THIS host's C library (a
// different libm would make device runs and per-step host draws disagree in rare last-bit cases):
// checked once per process on 2^20 inputs each, spread over the whole range, plus the one input
// known to separate the C library's fused and unfused expf variants.
bool hostmath_matches_libm() {
    static const bool ok = [] {
        auto same = [](float a, float b) {
            uint32_t ab, bb;
            memcpy(&ab, &a, 4);
            memcpy(&bb, &b, 4);
            return ab == bb || (a != a && b != b);
        };
        auto at = [](uint32_t bits) { float x; memcpy(&x, &bits, 4); return x; };
        volatile uint32_t special = 0xc27c65d9u;                   // volatile: the C library must run, not the compiler's folder
        const float xs = at(special);
        if (!same(expf(xs), expf_as_host(xs))) return false;
        for (uint32_t i = 0; i < (1u << 20); ++i) {
            const float xe = at(0x80000000u + i * 2039u);          // -0.0 .. about -1e38
            if (!same(expf(xe), expf_as_host(xe))) return false;
            const float xt = at(i * 4093u + 7u);                   // all signs and magnitudes
            if (!same(tanhf(xt), tanhf_as_host(xt))) return false;
        }
        return true;
    }();
    return ok;
}

int sampled_args_ok(hipdec_model *m, bool topk, uint32_t top_k, float temperature, float softcap, const uint64_t *rng,
                    const uint32_t *out_tokens) {
    if (!rng || !out_tokens) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if (m->blocks > SAMPLE_MAX_BLOCKS) return fail(m, HIPDEC_ERR_UNSUPPORTED, "on-device sampling serves up to 1024 vocab blocks");
    if (!hostmath_matches_libm())
        return fail(m, HIPDEC_ERR_UNSUPPORTED, "this host's expf/tanhf differ from the ones the device sampler reproduces: use the per-step calls");
    (void)softcap;
    if (topk) {
        if (top_k == 0 || top_k > HIPDEC_MAX_GPU_TOPK) return fail(m, HIPDEC_ERR_ARG, "gpu top-k only supports k in 1..32");
    } else if (!(temperature > 0.0f)) {
        return fail(m, HIPDEC_ERR_ARG, "full-vocab sampling needs a positive temperature");
    }
    return HIPDEC_OK;
}

int sampled_run(hipdec_model *m, int variant, uint32_t token, uint32_t top_k, float temperature, float softcap,
                uint64_t *rng_state, size_t n_steps, uint32_t *out_tokens) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (n_steps == 0) return HIPDEC_OK;
    if ((rc = sampled_args_ok(m, variant == V_TOPK_S, top_k, temperature, softcap, rng_state, out_tokens))) return rc;
    if (m->bt.rows) return fail(m, HIPDEC_ERR_ARG, "a batch is open: use the *_batch calls");
    if (m->len + n_steps > m->cfg.seq) return fail(m, HIPDEC_ERR_FULL, "sampled run exceeds cfg.seq");
    StepParams p = base_params(m, token);
    p.top_k = (int)top_k; p.inv_t = sample_inv_temperature(temperature); p.softcap = softcap;
    m->h_sp[0] = p;
    m->h_samp->ss = SampleParams{temperature, softcap, (int)top_k, 0, (int)m->cfg.seq, 0u};
    m->h_samp->rng[0] = *rng_state;
    HCHK(hipMemcpyAsync(m->d_sp, &m->h_sp[0], sizeof(StepParams), hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(m->d_ss, &m->h_samp->ss, sizeof(SampleParams), hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(m->d_rng, m->h_samp->rng, sizeof(uint64_t), hipMemcpyHostToDevice, m->stream));
    HCHK(hipEventRecord(m->ev0, m->stream));
    for (size_t i = 0; i < n_steps; ++i)
        if ((rc = run_step(m, variant))) return rc;
    HCHK(hipEventRecord(m->ev1, m->stream));
    HCHK(hipMemcpyAsync(m->h_out, m->d_ring, n_steps * 4, hipMemcpyDeviceToHost, m->stream));
    HCHK(hipMemcpyAsync(m->h_samp->rng, m->d_rng, sizeof(uint64_t), hipMemcpyDeviceToHost, m->stream));
    SYNC_CHECKED(m);
    HCHK(hipEventElapsedTime(&m->last_ms, m->ev0, m->ev1));
    m->step_timed = false;
    memcpy(out_tokens, m->h_out, n_steps * 4);
    *rng_state = m->h_samp->rng[0];
    m->len += n_steps;
    return HIPDEC_OK;
}

int batch_sampled_run(hipdec_model *m, int variant, const uint32_t *tokens, uint32_t top_k, float temperature, float softcap,
                      uint64_t *rng_states, size_t n_steps, uint32_t *out_tokens) {
    if (!m) return HIPDEC_ERR_ARG;
    const hipdec_config &c = m->cfg;
    BatchState &b = m->bt;
    if (b.rows <= 0) return fail(m, HIPDEC_ERR_ARG, "no batch is open (hipdec_batch_begin)");
    if (!tokens) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if (n_steps == 0) return HIPDEC_OK;
    int rc = sampled_args_ok(m, variant == B_TOPK_S, top_k, temperature, softcap, rng_states, out_tokens);
    if (rc) return rc;
    if (b.prefix + b.slot + n_steps > c.seq) return fail(m, HIPDEC_ERR_FULL, "sampled run exceeds cfg.seq");
    const int R = b.rows;
    for (int r = 0; r < R; ++r)
        if (tokens[r] >= c.vocab) return fail(m, HIPDEC_ERR_ARG, "token id must fit vocab");
    if ((size_t)R * n_steps > b.ring_elems) return fail(m, HIPDEC_ERR_ARG, "internal: token ring too small");
    if ((rc = pf_ensure(m, R, true))) return rc;
    PrefillWork &w = m->pf;
    HCHK(hipStreamSynchronize(m->stream));                      // pinned staging is free again
    memcpy(w.h_ids, tokens, (size_t)R * 4);
    *b.h_bp = BatchParams{(int)(b.prefix + b.slot), (int)b.slot, (int)b.prefix, (int)top_k, sample_inv_temperature(temperature),
                          softcap};
    m->h_samp->ss = SampleParams{temperature, softcap, (int)top_k, 0, (int)(b.ring_elems / (size_t)R), 0u};
    memcpy(m->h_samp->rng, rng_states, (size_t)R * sizeof(uint64_t));
    HCHK(hipMemcpyAsync(w.ids, w.h_ids, (size_t)R * 4, hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(b.d_bp, b.h_bp, sizeof(BatchParams), hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(m->d_ss, &m->h_samp->ss, sizeof(SampleParams), hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(m->d_rng, m->h_samp->rng, (size_t)R * sizeof(uint64_t), hipMemcpyHostToDevice, m->stream));
    HCHK(hipEventRecord(m->ev0, m->stream));
    for (size_t i = 0; i < n_steps; ++i)
        if ((rc = batch_launch(m, variant))) return rc;
    HCHK(hipEventRecord(m->ev1, m->stream));
    HCHK(hipMemcpyAsync(b.h_ring, b.d_ring, (size_t)R * n_steps * 4, hipMemcpyDeviceToHost, m->stream));
    HCHK(hipMemcpyAsync(m->h_samp->rng, m->d_rng, (size_t)R * sizeof(uint64_t), hipMemcpyDeviceToHost, m->stream));
    HCHK(hipStreamSynchronize(m->stream));
    if ((rc = rows_check(m))) return rc;
    HCHK(hipEventElapsedTime(&m->last_ms, m->ev0, m->ev1));
    m->step_timed = false;
    memcpy(out_tokens, b.h_ring, (size_t)R * n_steps * 4);
    memcpy(rng_states, m->h_samp->rng, (size_t)R * sizeof(uint64_t));
    b.slot += n_steps;
    b.have_logits = true;
    return HIPDEC_OK;
}

// the draw kernels on caller-supplied inputs: one row, device buffers of exactly the sizes the kernels index
struct DebugDraw {
    std::vector<void *> bufs;
    ~DebugDraw() { for (void *p : bufs) (void)hipFree(p); }
    template <typename T> T *up(const T *host, size_t n, hipError_t *e) {
        void *d = nullptr;
        if (*e == hipSuccess) *e = hipMalloc(&d, n ? n * sizeof(T) : sizeof(T));
        if (*e == hipSuccess) bufs.push_back(d);
        if (*e == hipSuccess && n && host) *e = hipMemcpy(d, host, n * sizeof(T), hipMemcpyHostToDevice);
        return (T *)d;
    }
};

// a restated host function over consecutive bit patterns on the host, split over threads
template <typename F> void hostmath_host_range(uint32_t first_bits, uint64_t count, int threads, F &&per_chunk) {
    if (threads < 1) threads = 1;
    if (threads > 64) threads = 64;
    std::vector<std::thread> pool;
    const uint64_t per = (count + (uint64_t)threads - 1) / (uint64_t)threads;
    for (int t = 0; t < threads; ++t) {
        const uint64_t lo = per * (uint64_t)t, hi = std::min<uint64_t>(count, lo + per);
        if (lo >= hi) break;
        pool.emplace_back([=, &per_chunk] { per_chunk(t, first_bits + (uint32_t)lo, hi - lo); });
    }
    for (auto &th : pool) th.join();
}

}  // namespace

extern "C" {

// errors of the entries without a model that live in other files (serving_ops.hip)
__attribute__((visibility("hidden"))) int hipdec_op_error(int code, const char *entry, const char *what) {
    g_op_failed = true;
    try { g_op_error = std::string(entry) + ": " + what; } catch (...) { g_op_error.clear(); }
    return code;
}

const char *hipdec_last_error(const hipdec_model *m) {
    if (m) return m->err.c_str();
    if (g_op_failed) return g_op_error.c_str();
    try {                                                     // (a copy: another thread may fail while the caller reads)
        std::lock_guard<std::mutex> lock(g_create_error.mu);
        g_shown_error = g_create_error.text;
    } catch (...) { g_shown_error.clear(); }
    return g_shown_error.c_str();
}

void hipdec_destroy(hipdec_model *m) {
    if (!m) return;
    if (m->stream) (void)hipStreamSynchronize(m->stream);
    for (auto &g : m->graphs) if (g) (void)hipGraphExecDestroy(g);
    for (auto &g : m->bt.graphs) if (g) (void)hipGraphExecDestroy(g);
    for (void *p : m->allocs) (void)hipFree(p);
    if (m->xslab) uncached_give(m->opt.device, m->xslab_cap, m->xslab);
    if (m->bt.rows_slab) uncached_give(m->opt.device, m->bt.rows_slab_cap, m->bt.rows_slab);
    if (m->h_sp) (void)hipHostFree(m->h_sp);
    if (m->h_out) (void)hipHostFree(m->h_out);
    if (m->pf.h_ids) (void)hipHostFree(m->pf.h_ids);
    if (m->bt.h_bp) (void)hipHostFree(m->bt.h_bp);
    if (m->bt.h_stage) (void)hipHostFree(m->bt.h_stage);
    if (m->bt.h_ring) (void)hipHostFree(m->bt.h_ring);
    if (m->rq.h_rows) (void)hipHostFree(m->rq.h_rows);
    if (m->rq.h_u) (void)hipHostFree(m->rq.h_u);
    if (m->rq.h_tok) (void)hipHostFree(m->rq.h_tok);
    if (m->h_samp) (void)hipHostFree(m->h_samp);
    if (m->h_abort) (void)hipHostFree(m->h_abort);
    if (m->ev0) (void)hipEventDestroy(m->ev0);
    if (m->ev1) (void)hipEventDestroy(m->ev1);
    if (m->ev_s0) (void)hipEventDestroy(m->ev_s0);
    if (m->ev_s1) (void)hipEventDestroy(m->ev_s1);
    if (m->stream) (void)hipStreamDestroy(m->stream);
    delete m;
}

static void *noalloc_scratch();

// base != null: the new model takes base's weights (same configuration and weight format) instead of uploading any
static int create_impl(hipdec_model *m, const hipdec_layer_f32 *layers, const hipdec_head_f32 *head,
                       const hipdec_model *base = nullptr, const hipdec_packed_layer *packed = nullptr,
                       const hipdec_packed_head *phead = nullptr) {
    const hipdec_config &c = m->cfg;
    const size_t D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, V = c.vocab, S = c.seq;
    HCHK(hipSetDevice(m->opt.device));
    hipDeviceProp_t prop;
    HCHK(hipGetDeviceProperties(&prop, m->opt.device));
    m->num_cu = prop.multiProcessorCount > 0 ? prop.multiProcessorCount : 256;
    HCHK(hipStreamCreate(&m->stream));
    HCHK(hipEventCreate(&m->ev0));
    HCHK(hipEventCreate(&m->ev1));
    HCHK(hipEventCreate(&m->ev_s0));
    HCHK(hipEventCreate(&m->ev_s1));

    size_t max_elems = V * D;
    if (D * H > max_elems) max_elems = D * H;
    if (D * Q > max_elems) max_elems = D * Q;
    float *stage_a = nullptr, *stage_b = nullptr;
    if (base) {
        m->wstore = base->wstore;
    } else {
        m->wstore = std::make_shared<WeightStore>();
        m->wstore->device = m->opt.device;
        if (!packed) {                                   // (stored weights are copied as they are: nothing to stage)
            HCHK(hipMalloc((void **)&stage_a, max_elems * sizeof(float)));
            HCHK(hipMalloc((void **)&stage_b, max_elems * sizeof(float)));
        }
    }
    int rc = HIPDEC_OK;
    auto done = [&](int code) { (void)hipFree(stage_a); (void)hipFree(stage_b); return code; };

    const int wt = m->wt;
    const size_t kvsz = m->kvbf16 ? 2 : 4;
    m->layers.resize(c.nlayers);
    for (uint32_t l = 0; l < c.nlayers && rc == HIPDEC_OK; ++l) {
        DevLayer &L = m->layers[l];
#define TRY(x) do { rc = (x); if (rc != HIPDEC_OK) return done(rc); } while (0)
        if (base) {
            L = base->layers[l];                       // weight, scale and norm pointers; the caches are this model's own
            L.kc = nullptr; L.vc = nullptr;
        }
        TRY(dalloc(m, &L.kc, S * KV * kvsz));
        TRY(dalloc(m, &L.vc, S * KV * kvsz));
        HCHK(hipMemsetAsync(L.kc, 0, S * KV * kvsz, m->stream));
        HCHK(hipMemsetAsync(L.vc, 0, S * KV * kvsz, m->stream));
        if (base) continue;
        if (packed) {
            // weights as an earlier model stored them (hipdec_export_packed_*): copied, not converted
            const hipdec_packed_layer &p = packed[l];
            const size_t wb[4] = {wt_row_bytes(wt, D) * (Q + 2 * KV), wt_row_bytes(wt, Q) * D, wt_row_bytes(wt, D) * 2 * H,
                                  wt_row_bytes(wt, H) * D};
            const size_t sb[4] = {wt_scale_bytes(wt, Q + 2 * KV, D), wt_scale_bytes(wt, D, Q), wt_scale_bytes(wt, 2 * H, D),
                                  wt_scale_bytes(wt, D, H)};
            const void *wsrc[4] = {p.wqkv, p.wo, p.w13, p.w2}, *ssrc[4] = {p.s_qkv, p.s_wo, p.s_w13, p.s_w2};
            void **wdst[4] = {&L.wqkv, &L.wo, &L.w13, &L.w2}, **sdst[4] = {&L.s_qkv, &L.s_wo, &L.s_w13, &L.s_w2};
            if (!p.gamma1 || !p.gamma2) return done(fail(m, HIPDEC_ERR_ARG, "null layer weight pointer"));
            for (int i = 0; i < 4; ++i) {
                if (!wsrc[i] || (sb[i] && !ssrc[i])) return done(fail(m, HIPDEC_ERR_ARG, "null layer weight pointer"));
                TRY(walloc(m, wdst[i], wb[i]));
                HCHK(hipMemcpy(*wdst[i], wsrc[i], wb[i], hipMemcpyHostToDevice));
                TRY(walloc(m, sdst[i], sb[i]));
                if (sb[i]) HCHK(hipMemcpy(*sdst[i], ssrc[i], sb[i], hipMemcpyHostToDevice));
            }
            TRY(walloc(m, &L.g1, D * 4));
            TRY(walloc(m, &L.g2, D * 4));
            HCHK(hipMemcpy(L.g1, p.gamma1, D * 4, hipMemcpyHostToDevice));
            HCHK(hipMemcpy(L.g2, p.gamma2, D * 4, hipMemcpyHostToDevice));
            continue;
        }
        const hipdec_layer_f32 &src = layers[l];
        if (!src.wq || !src.wk || !src.wv || !src.wo || !src.w1 || !src.w3 || !src.w2 || !src.gamma1 || !src.gamma2)
            return done(fail(m, HIPDEC_ERR_ARG, "null layer weight pointer"));
        TRY(walloc(m, &L.wqkv, wt_row_bytes(wt, D) * (Q + 2 * KV)));
        TRY(walloc(m, &L.wo, wt_row_bytes(wt, Q) * D));
        TRY(walloc(m, &L.w13, wt_row_bytes(wt, D) * 2 * H));
        TRY(walloc(m, &L.w2, wt_row_bytes(wt, H) * D));
        TRY(walloc(m, &L.s_qkv, wt_scale_bytes(wt, Q + 2 * KV, D)));
        TRY(walloc(m, &L.s_wo, wt_scale_bytes(wt, D, Q)));
        TRY(walloc(m, &L.s_w13, wt_scale_bytes(wt, 2 * H, D)));
        TRY(walloc(m, &L.s_w2, wt_scale_bytes(wt, D, H)));
        TRY(walloc(m, &L.g1, D * 4));
        TRY(walloc(m, &L.g2, D * 4));
        TRY(load_matrix(m, wt, src.wq, Q, D, true, stage_a, stage_b, L.wqkv, L.s_qkv, 1, 0));
        TRY(load_matrix(m, wt, src.wk, KV, D, true, stage_a, stage_b, L.wqkv, L.s_qkv, 1, (int)Q));
        TRY(load_matrix(m, wt, src.wv, KV, D, true, stage_a, stage_b, L.wqkv, L.s_qkv, 1, (int)(Q + KV)));
        TRY(load_matrix(m, wt, src.wo, D, Q, true, stage_a, stage_b, L.wo, L.s_wo, 1, 0));
        TRY(load_matrix(m, wt, src.w1, H, D, true, stage_a, stage_b, L.w13, L.s_w13, 2, 0));
        TRY(load_matrix(m, wt, src.w3, H, D, true, stage_a, stage_b, L.w13, L.s_w13, 2, 1));
        TRY(load_matrix(m, wt, src.w2, D, H, false, stage_a, stage_b, L.w2, L.s_w2, 1, 0));
        HCHK(hipMemcpy(L.g1, src.gamma1, D * 4, hipMemcpyHostToDevice));
        HCHK(hipMemcpy(L.g2, src.gamma2, D * 4, hipMemcpyHostToDevice));
    }
    if (base) {
        m->embed = base->embed;
        m->gfinal = base->gfinal;
    } else if (packed) {
        TRY(walloc(m, &m->embed, wt_row_bytes(m->embed_wt, D) * V));
        HCHK(hipMemcpy(m->embed, phead->embed, wt_row_bytes(m->embed_wt, D) * V, hipMemcpyHostToDevice));
        TRY(walloc(m, &m->gfinal, D * 4));
        HCHK(hipMemcpy(m->gfinal, phead->gamma_final, D * 4, hipMemcpyHostToDevice));
    } else {
        TRY(walloc(m, &m->embed, wt_row_bytes(m->embed_wt, D) * V));
        TRY(load_matrix(m, m->embed_wt, head->embed, V, D, false, stage_a, stage_b, m->embed, nullptr, 1, 0));
        TRY(walloc(m, &m->gfinal, D * 4));
        HCHK(hipMemcpy(m->gfinal, head->gamma_final, D * 4, hipMemcpyHostToDevice));
    }

    m->blocks = (int)((V + HIPDEC_HEAD_BLOCK - 1) / HIPDEC_HEAD_BLOCK);
    int ns = (int)(256 / c.heads);
    if (ns < 1) ns = 1;
    if (ns > 32) ns = 32;
    m->NS = ns;
    TRY(dalloc(m, &m->x_a, D * 4));
    TRY(dalloc(m, &m->x_b, D * 4));
    TRY(dalloc(m, &m->x_in, D * 4));
    TRY(dalloc(m, &m->q, Q * 4));
    TRY(dalloc(m, &m->att, Q * 4));
    TRY(dalloc(m, &m->gate, H * 4));
    TRY(dalloc(m, &m->logits, V * 4));
    TRY(dalloc(m, &m->d_out, (V > 256 ? V : 256) * 4));
    TRY(dalloc(m, &m->part, (size_t)c.heads * ns * (c.hd + 2) * 4));
    TRY(dalloc(m, &m->counters, (size_t)c.heads * 4));
    HCHK(hipMemset(m->counters, 0, (size_t)c.heads * 4));
    TRY(dalloc(m, &m->d_sp, sizeof(StepParams)));
    HCHK(hipMemset(m->d_sp, 0, sizeof(StepParams)));
    TRY(dalloc(m, &m->d_topk_vals, (size_t)m->blocks * HIPDEC_MAX_GPU_TOPK * 4));
    TRY(dalloc(m, &m->d_topk_idxs, (size_t)m->blocks * HIPDEC_MAX_GPU_TOPK * 4));
    TRY(dalloc(m, &m->d_bmax, (size_t)m->blocks * 4));
    TRY(dalloc(m, &m->d_bsum, (size_t)m->blocks * 4));
    TRY(dalloc(m, &m->d_ring, S * 4));
    TRY(dalloc(m, &m->d_ss, sizeof(SampleParams)));
    HCHK(hipMemset(m->d_ss, 0, sizeof(SampleParams)));
    TRY(dalloc(m, &m->d_rng, sizeof(uint64_t) * 32));
    HCHK(hipHostMalloc((void **)&m->h_samp, sizeof(SampleHost), hipHostMallocDefault));
    // abort flags of the persistent kernels: host memory the device writes through a mapping, so that the
    // host needs no copy of its own to look at them after a wait for the stream
    HCHK(hipHostMalloc((void **)&m->h_abort, 256, hipHostMallocMapped));
    memset(m->h_abort, 0, 256);
    HCHK(hipHostGetDevicePointer((void **)&m->d_abort, m->h_abort, 0));
    (void)noalloc_scratch();              // (resolves this device's scratch array of hipdec_sample_fullvocab_noalloc outside any capture)
    // ---- persistent per-token kernel: exchange buffers, layer table, eligibility
    {
        const int G = m->num_cu;
        const int epl = wt == WT_F32 ? 4 : wt == WT_BF16 ? 8 : wt == WT_FP8 ? 16 : 32;
        auto tasks_of = [&](size_t rows, size_t K) {
            size_t pairs = rows / 2, npl = (pairs + G - 1) / G;
            size_t segs = (K / epl + MEGA_SEG_PIECES - 1) / MEGA_SEG_PIECES;
            return npl * segs;
        };
        const bool head_inside = (wt == m->embed_wt);
        size_t max_tasks = tasks_of(Q + 2 * KV, D);
        max_tasks = std::max(max_tasks, tasks_of(D, Q));
        max_tasks = std::max(max_tasks, tasks_of(2 * H, D));
        max_tasks = std::max(max_tasks, tasks_of(D, H));
        if (head_inside) max_tasks = std::max(max_tasks, tasks_of(V, D));
        // LDS of the persistent kernel: the staged input vector twice (even phases read D floats, odd
        // phases max(Q, H)), a small staging area (attention: one partial per wave and q / k / v of the new
        // token; odd phases: two sums per task), the residual inputs twice, the RoPE pairs and the
        // per-layer pointer table.
        const size_t lds_cap = 160 * 1024 - 2048;
        const size_t xs_floats = D + std::max(Q, H);
        const size_t xres_floats = 2 * ((D / 2 + G - 1) / G) + 2;
        const size_t rope_floats = 2 * (((Q + 2 * KV) / 2 + G - 1) / G) + 2;
        // The short-phase kernel (hipdec_lean.h) takes bf16 models whose reduction lengths are all multiples of
        // 512 and whose output / down projections are one round of four (pair, chunk) items per wave.
        const size_t odd_pairs = (D / 2 + G - 1) / G;
        const size_t lean_items = odd_pairs * (std::max(Q, H) / 512);
        const char *env_lean = getenv("HIPDEC_NO_LEAN");
        const bool lean_fits = wt == WT_BF16 && m->embed_wt == WT_BF16 && D % 512 == 0 && Q % 512 == 0 && H % 512 == 0 &&
                               lean_ce_built((int)(D / 512)) && lean_items <= (size_t)MEGA_WAVES * LEAN_ITEMS_B &&
                               !(env_lean && env_lean[0] == '1');
        // (the short-phase kernel stages LEAN_PLANES bf16 numbers per element instead of one float: sized for it when it may run)
        const size_t xs_lean_floats = lean_fits ? (xs_floats * LEAN_PLANES + 1) / 2 : 0;
        const size_t fixed_lds = (std::max(xs_floats, xs_lean_floats) + 2 * xres_floats + rope_floats) * 4 + (size_t)MEGA_LPTR * c.nlayers * sizeof(void *);
        int ns_max = G / (int)c.heads;                 // one workgroup per (split, head)
        if (ns_max > 32) ns_max = 32;
        const size_t odd_tasks = std::max(tasks_of(D, Q), tasks_of(D, H));
        const size_t stage_floats = std::max(std::max((size_t)MEGA_WAVES * (c.hd + MEGA_PREC) + 3 * c.hd, 2 * odd_tasks),
                                             lean_fits ? 2 * lean_items : (size_t)0);
        m->mega_lds = fixed_lds + stage_floats * 4;
        // Models whose output / down projections are more than one register round per wave get a second round
        // prefetched into LDS where it fits (hipdec_mega.h, issue_odd_lds): MEGA_LDS_TASKS tasks of 4 KB per wave.
        const size_t odd_rounds_w = (odd_tasks + MEGA_WAVES - 1) / MEGA_WAVES;
        const size_t lds_pf = 1024 + (size_t)MEGA_WAVES * MEGA_LDS_TASKS * 4096;
        const char *env_pf = getenv("HIPDEC_NO_LDS_PREFETCH");
        const bool lds_tasks_on = odd_rounds_w > MEGA_DEPTH_B && m->mega_lds + lds_pf <= lds_cap && !(env_pf && env_pf[0] == '1');
        if (lds_tasks_on) m->mega_lds += lds_pf;
        const char *env = getenv("HIPDEC_NO_MEGA");
        bool want = !(m->opt.flags & HIPDEC_FLAG_NO_MEGA) && !(env && env[0] == '1');
        bool fits = ns_max >= 1 && m->mega_lds <= lds_cap && (V % 2 == 0) && (int)c.heads <= G &&
                    D % 4 == 0;
        if (want && fits) {
            std::vector<MegaLayer> hl(c.nlayers);
            for (uint32_t l = 0; l < c.nlayers; ++l) {
                const DevLayer &L = m->layers[l];
                hl[l].w[0] = L.wqkv; hl[l].w[1] = L.wo; hl[l].w[2] = L.w13; hl[l].w[3] = L.w2;
                hl[l].sc[0] = L.s_qkv; hl[l].sc[1] = L.s_wo; hl[l].sc[2] = L.s_w13; hl[l].sc[3] = L.s_w2;
                hl[l].g1 = L.g1; hl[l].g2 = L.g2; hl[l].kc = L.kc; hl[l].vc = L.vc;
            }
            MegaLayer *dl = nullptr;
            TRY(dalloc(m, &dl, sizeof(MegaLayer) * c.nlayers));
            HCHK(hipMemcpy(dl, hl.data(), sizeof(MegaLayer) * c.nlayers, hipMemcpyHostToDevice));
            MegaArgs &a = m->mega;
            a.layers = dl; a.embed = m->embed; a.gfinal = m->gfinal; a.x_in = m->x_in;
            a.X = m->x_a; a.logits = m->logits; a.sp = m->d_sp; a.ring = m->d_ring; a.ring_cap = (int)S;
            // The vectors the workgroups hand to each other go into one slab of uncached device memory
            // (uncached_take); ordinary memory works too and is the fallback.
            const size_t xb[6] = {(Q + 2 * KV) * 4, (size_t)c.heads * ns_max * (c.hd + MEGA_PREC) * 4, D * 4, H * 4,
                                  (size_t)G * 8, D * 4};
            size_t xoff[6], xtotal = 0;
            for (int i = 0; i < 6; ++i) { xoff[i] = xtotal; xtotal += (xb[i] + 255) & ~(size_t)255; }
            m->xslab = uncached_take(m->opt.device, xtotal, &m->xslab_cap);
            if (m->xslab) {
                char *base = (char *)m->xslab;
                a.QKV = (float *)(base + xoff[0]); a.PART = (float *)(base + xoff[1]); a.X2 = (float *)(base + xoff[2]);
                a.GATE = (float *)(base + xoff[3]); a.CAND = (decltype(a.CAND))(base + xoff[4]);
                m->x_a = (float *)(base + xoff[5]);
                a.X = m->x_a;
            } else {
                TRY(dalloc(m, &a.QKV, xb[0]));
                TRY(dalloc(m, &a.PART, xb[1]));
                TRY(dalloc(m, &a.X2, xb[2]));
                TRY(dalloc(m, &a.GATE, xb[3]));
                TRY(dalloc(m, &a.CAND, xb[4]));
            }
            TRY(dalloc(m, &m->d_epochs, 16));
            HCHK(hipMemset(a.QKV, 0, (Q + 2 * KV) * 4));
            HCHK(hipMemset(a.PART, 0, (size_t)c.heads * ns_max * (c.hd + MEGA_PREC) * 4));
            HCHK(hipMemset(a.X2, 0, D * 4));
            HCHK(hipMemset(a.GATE, 0, H * 4));
            HCHK(hipMemset(a.CAND, 0, (size_t)G * 8));
            HCHK(hipMemset(m->d_epochs, 0, 16));
            HCHK(hipMemset(m->x_a, 0, D * 4));
            a.epochs = m->d_epochs; a.abort = m->d_abort;
            a.D = (int)D; a.Q = (int)Q; a.KV = (int)KV; a.H = (int)H; a.V = (int)V; a.L = (int)c.nlayers;
            a.hd = (int)c.hd; a.heads = (int)c.heads; a.gqa = c.gqa_ratio ? (int)c.gqa_ratio : 1;
            a.act = (int)m->opt.ffn_activation; a.ns_max = ns_max; a.seq = (int)S; a.alpha = m->alpha;
            a.stage_floats = (int)stage_floats;
            a.lds_tasks = lds_tasks_on ? MEGA_LDS_TASKS : 0;
            if (const char *pw = getenv("HIPDEC_PROF_WG")) a.prof_wg = std::max(0, std::min(G - 1, atoi(pw)));
            m->mega_grid = G;
            hipError_t e;
            switch (wt) {
                case WT_F32: e = mega_set_lds_t<WT_F32>(m); break;
                case WT_BF16: e = mega_set_lds_t<WT_BF16>(m); break;
                case WT_FP8: e = mega_set_lds_t<WT_FP8>(m); break;
                default: e = mega_set_lds_t<WT_INT4>(m); break;
            }
            m->mega_ok = (e == hipSuccess);
            if (e != hipSuccess) (void)hipGetLastError();
            if (m->mega_ok && lean_fits) {
                const hipError_t el = D / 512 == 1 ? lean_set_lds_t<1>(m) : lean_set_lds_t<3>(m);
                if (el == hipSuccess) m->lean_ce = (int)(D / 512);
                else (void)hipGetLastError();
            }
        }
        if (const char *v = getenv("HIPDEC_VERBOSE"))
            if (v[0] == '1')
                fprintf(stderr, "hipdec: persistent step kernel %s (wanted %d, fits %d, grid %d, lds %zu B, ns_max %d, tasks %zu)\n",
                        m->mega_ok ? "on" : "off", (int)want, (int)fits, G, m->mega_lds, ns_max, max_tasks);
    }
#undef TRY
    // RoPE table, theta = pos / 10000^(2i/hd) (engine/src/kernels/sdpa_fwd.rs:18-33, lib.rs:1401)
    {
        const size_t hp = c.hd / 2;
        std::vector<float> ct(S * hp), st(S * hp);
        for (size_t p = 0; p < S; ++p)
            for (size_t i = 0; i < hp; ++i) {
                float theta = (float)p / powf(10000.0f, 2.0f * (float)i / (float)c.hd);
                ct[p * hp + i] = cosf(theta);
                st[p * hp + i] = sinf(theta);
            }
        rc = dalloc(m, &m->rope_cos, S * hp * 4); if (rc) return done(rc);
        rc = dalloc(m, &m->rope_sin, S * hp * 4); if (rc) return done(rc);
        HCHK(hipMemcpy(m->rope_cos, ct.data(), S * hp * 4, hipMemcpyHostToDevice));
        HCHK(hipMemcpy(m->rope_sin, st.data(), S * hp * 4, hipMemcpyHostToDevice));
        m->mega.rope_cos = m->rope_cos;
        m->mega.rope_sin = m->rope_sin;
    }
    HCHK(hipHostMalloc((void **)&m->h_sp, sizeof(StepParams) * (S + 1), hipHostMallocDefault));
    m->h_out_elems = V > 2 * (size_t)m->blocks * HIPDEC_MAX_GPU_TOPK ? V : 2 * (size_t)m->blocks * HIPDEC_MAX_GPU_TOPK;
    if (m->h_out_elems < S) m->h_out_elems = S;
    if (m->h_out_elems < D) m->h_out_elems = D;
    HCHK(hipHostMalloc((void **)&m->h_out, m->h_out_elems * 4, hipHostMallocMapped));
    if (hipHostGetDevicePointer((void **)&m->d_hout, m->h_out, 0) != hipSuccess) { m->d_hout = nullptr; (void)hipGetLastError(); }
    SYNC_CHECKED(m);
    return done(HIPDEC_OK);
}

// the checks on a configuration that need no device (shared by model creation and hipdec_packed_sizes_of)
static int check_config(const hipdec_config &c, uint32_t weight_dtype) {
    if (!c.dim || !c.hidden || !c.heads || !c.kv_heads || !c.hd || !c.seq || !c.nlayers || !c.vocab)
        return fail(nullptr, HIPDEC_ERR_ARG, "zero-sized config field");
    if (c.q_dim != c.heads * c.hd || c.kv_dim != c.kv_heads * c.hd || c.heads % c.kv_heads != 0 ||
        (c.gqa_ratio ? c.gqa_ratio : 1) != c.heads / c.kv_heads)
        return fail(nullptr, HIPDEC_ERR_ARG, "inconsistent head geometry");
    if (weight_dtype > HIPDEC_W_INT4_G128) return fail(nullptr, HIPDEC_ERR_ARG, "unknown option value");
    if (c.hd != 64 && c.hd != 128) return fail(nullptr, HIPDEC_ERR_UNSUPPORTED, "head dim must be 64 or 128");
    const uint32_t kmul = weight_dtype == HIPDEC_W_INT4_G128 ? 128 : (weight_dtype == HIPDEC_W_FP8_E4M3 ? 16 : 8);
    if (c.dim % kmul || c.hidden % kmul || c.q_dim % kmul || c.kv_dim % 8)
        return fail(nullptr, HIPDEC_ERR_UNSUPPORTED, "dim / hidden / q_dim must be multiples of the weight load width");
    if ((size_t)(c.hidden > c.dim ? c.hidden : c.dim) * 4 > 150 * 1024)
        return fail(nullptr, HIPDEC_ERR_UNSUPPORTED, "reduction axis does not fit LDS");
    return HIPDEC_OK;
}

static int create_front(const hipdec_config *cfg, const hipdec_layer_f32 *layers, const hipdec_head_f32 *head,
                        const hipdec_packed_layer *packed, const hipdec_packed_head *phead, size_t n_layers,
                        const hipdec_options *opts, hipdec_model **out);

int hipdec_create(const hipdec_config *cfg, const hipdec_layer_f32 *layers, size_t n_layers,
                  const hipdec_head_f32 *head, const hipdec_options *opts, hipdec_model **out) {
    if (out) *out = nullptr;
    if (!cfg || !layers || !head || !out) return fail(nullptr, HIPDEC_ERR_ARG, "null argument");
    if (!head->embed || !head->gamma_final) return fail(nullptr, HIPDEC_ERR_ARG, "null head weight pointer");
    return create_front(cfg, layers, head, nullptr, nullptr, n_layers, opts, out);
}

int hipdec_create_packed(const hipdec_config *cfg, const hipdec_packed_layer *layers, size_t n_layers,
                         const hipdec_packed_head *head, const hipdec_options *opts, hipdec_model **out) {
    if (out) *out = nullptr;
    if (!cfg || !layers || !head || !out) return fail(nullptr, HIPDEC_ERR_ARG, "null argument");
    if (!head->embed || !head->gamma_final) return fail(nullptr, HIPDEC_ERR_ARG, "null head weight pointer");
    return create_front(cfg, nullptr, nullptr, layers, head, n_layers, opts, out);
}

int hipdec_packed_sizes_of(const hipdec_config *cfg, uint32_t weight_dtype, hipdec_packed_sizes *out) {
    if (!cfg || !out) return fail(nullptr, HIPDEC_ERR_ARG, "null argument");
    const int rc = check_config(*cfg, weight_dtype);
    if (rc != HIPDEC_OK) return rc;
    const hipdec_config &c = *cfg;
    const int wt = (int)weight_dtype, ewt = weight_dtype == HIPDEC_W_F32 ? WT_F32 : WT_BF16;
    const size_t D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden;
    out->wqkv = wt_row_bytes(wt, D) * (Q + 2 * KV); out->s_qkv = wt_scale_bytes(wt, Q + 2 * KV, D);
    out->wo = wt_row_bytes(wt, Q) * D;              out->s_wo = wt_scale_bytes(wt, D, Q);
    out->w13 = wt_row_bytes(wt, D) * 2 * H;         out->s_w13 = wt_scale_bytes(wt, 2 * H, D);
    out->w2 = wt_row_bytes(wt, H) * D;              out->s_w2 = wt_scale_bytes(wt, D, H);
    out->gamma = D * 4;
    out->embed = wt_row_bytes(ewt, D) * c.vocab;
    return HIPDEC_OK;
}

int hipdec_export_packed_layer(hipdec_model *m, size_t layer_idx, void *wqkv, void *wo, void *w13, void *w2, void *s_qkv,
                               void *s_wo, void *s_w13, void *s_w2, float *gamma1, float *gamma2) {
    if (!m) return HIPDEC_ERR_ARG;
    if (layer_idx >= m->layers.size()) return fail(m, HIPDEC_ERR_ARG, "layer index out of range");
    hipdec_packed_sizes z;
    int rc = hipdec_packed_sizes_of(&m->cfg, (uint32_t)m->wt, &z);
    if (rc != HIPDEC_OK) return rc;
    const DevLayer &L = m->layers[layer_idx];
    const void *src[10] = {L.wqkv, L.wo, L.w13, L.w2, L.s_qkv, L.s_wo, L.s_w13, L.s_w2, L.g1, L.g2};
    void *dst[10] = {wqkv, wo, w13, w2, s_qkv, s_wo, s_w13, s_w2, gamma1, gamma2};
    const uint64_t bytes[10] = {z.wqkv, z.wo, z.w13, z.w2, z.s_qkv, z.s_wo, z.s_w13, z.s_w2, z.gamma, z.gamma};
    HCHK(hipSetDevice(m->opt.device));
    HCHK(hipStreamSynchronize(m->stream));
    for (int i = 0; i < 10; ++i) {
        if (!bytes[i]) continue;
        if (!dst[i]) return fail(m, HIPDEC_ERR_ARG, "null output pointer");
        HCHK(hipMemcpy(dst[i], src[i], bytes[i], hipMemcpyDeviceToHost));
    }
    return HIPDEC_OK;
}

int hipdec_export_packed_head(hipdec_model *m, float *gamma_final, void *embed) {
    if (!m) return HIPDEC_ERR_ARG;
    if (!gamma_final || !embed) return fail(m, HIPDEC_ERR_ARG, "null output pointer");
    hipdec_packed_sizes z;
    int rc = hipdec_packed_sizes_of(&m->cfg, (uint32_t)m->wt, &z);
    if (rc != HIPDEC_OK) return rc;
    HCHK(hipSetDevice(m->opt.device));
    HCHK(hipStreamSynchronize(m->stream));
    HCHK(hipMemcpy(gamma_final, m->gfinal, z.gamma, hipMemcpyDeviceToHost));
    HCHK(hipMemcpy(embed, m->embed, z.embed, hipMemcpyDeviceToHost));
    return HIPDEC_OK;
}

static int create_front(const hipdec_config *cfg, const hipdec_layer_f32 *layers, const hipdec_head_f32 *head,
                        const hipdec_packed_layer *packed, const hipdec_packed_head *phead, size_t n_layers,
                        const hipdec_options *opts, hipdec_model **out) {
    if (n_layers != cfg->nlayers) return fail(nullptr, HIPDEC_ERR_ARG, "layer count does not match cfg.nlayers");
    const hipdec_config &c = *cfg;
    hipdec_options o{};
    if (opts) o = *opts;
    if (o.kv_dtype > HIPDEC_KV_BF16 || o.ffn_activation > 1) return fail(nullptr, HIPDEC_ERR_ARG, "unknown option value");
    {
        const int crc = check_config(c, o.weight_dtype);
        if (crc != HIPDEC_OK) return crc;
    }
    hipdec_model *m = new hipdec_model();
    m->cfg = c;
    // HIPDEC_NO_GRAPH=1 in the environment forces eager launches (profilers that cannot follow
    // graph replays still see every kernel)
    if (const char *e = getenv("HIPDEC_NO_GRAPH")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_NO_GRAPH;
    if (const char *e = getenv("HIPDEC_PREFILL_STEPS")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_PREFILL_STEPS;
    if (const char *e = getenv("HIPDEC_PREFILL_BF16_ACT")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_PREFILL_BF16_ACT;
    if (const char *e = getenv("HIPDEC_PREFILL_F16_ACT")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_PREFILL_F16_ACT;
    if (const char *e = getenv("HIPDEC_PREFILL_PAIR_ACT")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_PREFILL_PAIR_ACT;
    m->opt = o;
    m->wt = (int)o.weight_dtype;
    m->embed_wt = o.weight_dtype == HIPDEC_W_F32 ? WT_F32 : WT_BF16;
    m->kvbf16 = o.kv_dtype == HIPDEC_KV_BF16;
    // Prefill activations: with 8-bit or 4-bit weights and a bf16 cache the GEMMs take one fp16 number per
    // activation (half the matrix work of the pair; the weights' own rounding, 2^-4 and coarser, is far above
    // fp16's 2^-11, and such a model is judged at 5e-2 of the largest logit: measured 3e-3 from the pair at
    // 5B).  bf16 weights keep the pair whatever the cache: with fp16 activations the 600M greedy stream
    // left the CPU reference's at its 90th token (a near tie moved by differently rounded cache rows).
    // The flags override either way.
    const bool quantised = o.weight_dtype == HIPDEC_W_FP8_E4M3 || o.weight_dtype == HIPDEC_W_INT4_G128;
    m->pf_act = (o.flags & HIPDEC_FLAG_PREFILL_PAIR_ACT)   ? PF_ACT_PAIR
                : (o.flags & HIPDEC_FLAG_PREFILL_BF16_ACT) ? PF_ACT_BF16
                : (o.flags & HIPDEC_FLAG_PREFILL_F16_ACT)  ? PF_ACT_F16
                : (m->kvbf16 && quantised)                 ? PF_ACT_F16
                                                           : PF_ACT_PAIR;
    m->alpha = 1.0f / sqrtf(2.0f * (float)c.nlayers);   // lib.rs:201
    int rc = create_impl(m, layers, head, nullptr, packed, phead);
    if (rc != HIPDEC_OK) {
        g_create_error = m->err;
        hipdec_destroy(m);
        return rc;
    }
    *out = m;
    return HIPDEC_OK;
}

int hipdec_create_shared(const hipdec_model *base, uint32_t kv_dtype, uint32_t flags, hipdec_model **out) {
    if (!base || !out) return fail(nullptr, HIPDEC_ERR_ARG, "null argument");
    *out = nullptr;
    if (kv_dtype > HIPDEC_KV_BF16) return fail(nullptr, HIPDEC_ERR_ARG, "unknown kv_dtype");
    hipdec_model *m = new hipdec_model();
    m->cfg = base->cfg;
    hipdec_options o = base->opt;
    o.kv_dtype = kv_dtype;
    o.flags = flags;
    if (const char *e = getenv("HIPDEC_NO_GRAPH")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_NO_GRAPH;
    if (const char *e = getenv("HIPDEC_PREFILL_STEPS")) if (e[0] == '1') o.flags |= HIPDEC_FLAG_PREFILL_STEPS;
    m->opt = o;
    m->wt = base->wt;
    m->embed_wt = base->embed_wt;
    m->kvbf16 = kv_dtype == HIPDEC_KV_BF16;
    const bool quantised = o.weight_dtype == HIPDEC_W_FP8_E4M3 || o.weight_dtype == HIPDEC_W_INT4_G128;
    m->pf_act = (o.flags & HIPDEC_FLAG_PREFILL_PAIR_ACT)   ? PF_ACT_PAIR
                : (o.flags & HIPDEC_FLAG_PREFILL_BF16_ACT) ? PF_ACT_BF16
                : (o.flags & HIPDEC_FLAG_PREFILL_F16_ACT)  ? PF_ACT_F16
                : (m->kvbf16 && quantised)                 ? PF_ACT_F16
                                                           : PF_ACT_PAIR;
    m->alpha = base->alpha;
    const int rc = create_impl(m, nullptr, nullptr, base);
    if (rc != HIPDEC_OK) {
        g_create_error = m->err;
        hipdec_destroy(m);
        return rc;
    }
    *out = m;
    return HIPDEC_OK;
}

size_t hipdec_len(const hipdec_model *m) { return m ? m->len : 0; }

int hipdec_set_len(hipdec_model *m, size_t len) {
    if (!m) return HIPDEC_ERR_ARG;
    m->len = len < m->cfg.seq ? len : m->cfg.seq;
    return HIPDEC_OK;
}

int hipdec_set_prefill_activations(hipdec_model *m, int mode) {
    if (!m) return HIPDEC_ERR_ARG;
    if (mode < 0 || mode > 3) return fail(m, HIPDEC_ERR_ARG, "prefill activation mode must be 0 (bf16 pair), 1 (bf16), 2 (fp16) or 3 (pair into the attention products, bf16 into the feed-forward ones)");
    m->pf_act = mode;
    return HIPDEC_OK;
}

int hipdec_seed_layer_cache_from_channel_first(hipdec_model *m, size_t layer_idx, size_t live_len,
                                               const float *k_rope_cf, const float *v_cf) {
    if (!m || !k_rope_cf || !v_cf) return HIPDEC_ERR_ARG;
    if (layer_idx >= m->cfg.nlayers) return fail(m, HIPDEC_ERR_ARG, "layer_idx out of range");
    const int KV = m->cfg.kv_dim, S = m->cfg.seq;
    if (live_len > (size_t)S) live_len = S;
    float *stage = nullptr;
    HCHK(hipMalloc((void **)&stage, (size_t)KV * S * 4));
    dim3 grid((S + 31) / 32, (KV + 31) / 32), block(32, 8);
    for (int which = 0; which < 2; ++which) {
        hipError_t e = hipMemcpy(stage, which ? v_cf : k_rope_cf, (size_t)KV * S * 4, hipMemcpyHostToDevice);
        if (e != hipSuccess) { (void)hipFree(stage); m->err = hipGetErrorString(e); return HIPDEC_ERR_HIP; }
        void *dst = which ? m->layers[layer_idx].vc : m->layers[layer_idx].kc;
        if (m->kvbf16) hipLaunchKernelGGL(k_seed_cache<1>, grid, block, 0, m->stream, stage, dst, KV, S, (int)live_len);
        else hipLaunchKernelGGL(k_seed_cache<0>, grid, block, 0, m->stream, stage, dst, KV, S, (int)live_len);
        e = hipStreamSynchronize(m->stream);
        if (e != hipSuccess) { (void)hipFree(stage); m->err = hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    }
    HCHK(hipFree(stage));
    return HIPDEC_OK;
}

static int read_x(hipdec_model *m, float *x_out) {
    HCHK(hipMemcpyAsync(m->h_out, m->x_a, (size_t)m->cfg.dim * 4, hipMemcpyDeviceToHost, m->stream));
    SYNC_CHECKED(m);
    memcpy(x_out, m->h_out, (size_t)m->cfg.dim * 4);
    return HIPDEC_OK;
}

static int upload_x(hipdec_model *m, const float *x_in) {
    memcpy(m->h_out, x_in, (size_t)m->cfg.dim * 4);
    HCHK(hipMemcpyAsync(m->x_in, m->h_out, (size_t)m->cfg.dim * 4, hipMemcpyHostToDevice, m->stream));
    return HIPDEC_OK;
}

int hipdec_decode_token(hipdec_model *m, const float *x_in, float *x_out) {
    int rc = check_step(m, 0, false);
    if (rc) return rc;
    if (!x_in || !x_out) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if ((rc = upload_x(m, x_in))) return rc;
    StepParams p = base_params(m, 0);
    p.use_x_in = 1;
    if ((rc = step_with(m, V_X, 0, p, true))) return rc;
    if ((rc = read_x(m, x_out))) return rc;
    m->len += 1;
    return HIPDEC_OK;
}

int hipdec_decode_token_from_id(hipdec_model *m, uint32_t token, float *x_out) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (!x_out) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if ((rc = step_with(m, V_X, 0, base_params(m, token), true))) return rc;
    if ((rc = read_x(m, x_out))) return rc;
    m->len += 1;
    return HIPDEC_OK;
}

static int finish_argmax(hipdec_model *m, uint32_t *out_token) {
    if (m->direct_step) {
        SYNC_CHECKED(m);
        *out_token = __atomic_load_n(m->h_abort + 48, __ATOMIC_ACQUIRE);
        m->len += 1;
        return HIPDEC_OK;
    }
    HCHK(hipMemcpyAsync(m->h_out, m->d_ring, 4, hipMemcpyDeviceToHost, m->stream));
    SYNC_CHECKED(m);
    memcpy(out_token, m->h_out, 4);
    m->len += 1;
    return HIPDEC_OK;
}

int hipdec_decode_token_argmax(hipdec_model *m, const float *x_in, uint32_t *out_token) {
    int rc = check_step(m, 0, false);
    if (rc) return rc;
    if (!x_in || !out_token) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if ((rc = upload_x(m, x_in))) return rc;
    StepParams p = base_params(m, 0);
    p.use_x_in = 1;
    if ((rc = step_with(m, V_ARGMAX, 0, p, true))) return rc;
    return finish_argmax(m, out_token);
}

int hipdec_decode_token_argmax_from_id(hipdec_model *m, uint32_t token, uint32_t *out_token) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (!out_token) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if ((rc = step_with(m, V_ARGMAX, 0, base_params(m, token), true))) return rc;
    return finish_argmax(m, out_token);
}

int hipdec_decode_token_topk_from_id(hipdec_model *m, uint32_t token, uint32_t top_k, float *out_vals,
                                     uint32_t *out_idxs, size_t cap, size_t *out_count) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (top_k == 0) return fail(m, HIPDEC_ERR_ARG, "top_k must be positive");
    if (top_k > HIPDEC_MAX_GPU_TOPK) return fail(m, HIPDEC_ERR_ARG, "top_k exceeds decode top-k capacity");
    const size_t count = (size_t)m->blocks * top_k;
    if (!out_vals || !out_idxs || cap < count) return fail(m, HIPDEC_ERR_ARG, "output buffers too small for top-k candidates");
    StepParams p = base_params(m, token);
    p.top_k = (int)top_k;
    if ((rc = step_with(m, V_TOPK, 0, p, true))) return rc;
    if (!m->direct_step) {
        HCHK(hipMemcpyAsync(m->h_out, m->d_topk_vals, count * 4, hipMemcpyDeviceToHost, m->stream));
        HCHK(hipMemcpyAsync(m->h_out + count, m->d_topk_idxs, count * 4, hipMemcpyDeviceToHost, m->stream));
    }
    SYNC_CHECKED(m);
    memcpy(out_vals, m->h_out, count * 4);
    memcpy(out_idxs, m->h_out + count, count * 4);
    if (out_count) *out_count = count;
    m->len += 1;
    return HIPDEC_OK;
}

int hipdec_decode_token_block_stats_from_id(hipdec_model *m, uint32_t token, float inv_temperature, float softcap,
                                            float *out_maxes, float *out_sums, size_t cap, size_t *out_count) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    const size_t B = (size_t)m->blocks;
    if (!out_maxes || !out_sums || cap < B) return fail(m, HIPDEC_ERR_ARG, "block stats buffers too small");
    StepParams p = base_params(m, token);
    p.inv_t = inv_temperature;
    p.softcap = softcap;
    if ((rc = step_with(m, V_STATS, 0, p, true))) return rc;
    if (!m->direct_step) {
        HCHK(hipMemcpyAsync(m->h_out, m->d_bmax, B * 4, hipMemcpyDeviceToHost, m->stream));
        HCHK(hipMemcpyAsync(m->h_out + B, m->d_bsum, B * 4, hipMemcpyDeviceToHost, m->stream));
    }
    SYNC_CHECKED(m);
    memcpy(out_maxes, m->h_out, B * 4);
    memcpy(out_sums, m->h_out + B, B * 4);
    if (out_count) *out_count = B;
    m->len += 1;
    return HIPDEC_OK;
}

int hipdec_materialize_current_logits_block(hipdec_model *m, size_t block_idx, float softcap, float *out_logits,
                                            size_t cap, size_t *out_valid) {
    if (!m) return HIPDEC_ERR_ARG;
    if (block_idx >= (size_t)m->blocks) return fail(m, HIPDEC_ERR_ARG, "block_idx out of range");
    size_t start = block_idx * HIPDEC_HEAD_BLOCK;
    size_t valid = m->cfg.vocab - start;
    if (valid > HIPDEC_HEAD_BLOCK) valid = HIPDEC_HEAD_BLOCK;
    if (!out_logits || cap < valid) return fail(m, HIPDEC_ERR_ARG, "out_logits too small");
    int rc = softcap_out(m, (int)start, (int)valid, softcap, out_logits);
    if (rc) return rc;
    if (out_valid) *out_valid = valid;
    return HIPDEC_OK;
}

int hipdec_decode_logits_from_id(hipdec_model *m, uint32_t token, float softcap, float *out_logits) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (!out_logits) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if ((rc = step_with(m, V_LOGITS, 0, base_params(m, token)))) return rc;
    if ((rc = softcap_out(m, 0, (int)m->cfg.vocab, softcap, out_logits))) return rc;
    m->len += 1;
    return HIPDEC_OK;
}

int hipdec_prefill(hipdec_model *m, const uint32_t *ids, size_t n, float softcap, float *last_logits) {
    if (!m || (!ids && n)) return HIPDEC_ERR_ARG;
    if (n == 0) return HIPDEC_OK;
    if (m->len + n > m->cfg.seq) return fail(m, HIPDEC_ERR_FULL, "prefill exceeds cfg.seq");
    for (size_t i = 0; i < n; ++i)
        if (ids[i] >= m->cfg.vocab) return fail(m, HIPDEC_ERR_ARG, "token id must fit vocab");
    HCHK(hipEventRecord(m->ev0, m->stream));
    if (prefill_batched_ok(m, n)) {
        const float *x_last = nullptr;
        int rc = prefill_batched(m, ids, n, &x_last);
        if (rc) return rc;
        if (last_logits) {
            // final RMSNorm + tied LM head on the last row only (full_model.rs:419-428 computes every row)
            GemvArgs a{};
            a.sp = m->d_sp; a.W = m->embed; a.in = x_last; a.gamma = m->gfinal; a.out = m->logits;
            a.rows = (int)m->cfg.vocab; a.K = (int)m->cfg.dim;
            launch_gemv<EPI_HEAD>(m, m->embed_wt, a);
            HCHK(hipGetLastError());
        }
    } else {
        for (size_t i = 0; i < n; ++i) {
            StepParams p = base_params(m, ids[i]);
            p.pos = (int)(m->len + i);
            int variant = (i + 1 == n && last_logits) ? V_LOGITS : V_X;
            int rc = step_with(m, variant, i, p);
            if (rc) return rc;
        }
    }
    HCHK(hipEventRecord(m->ev1, m->stream));
    if (last_logits) {
        int rc = softcap_out(m, 0, (int)m->cfg.vocab, softcap, last_logits);
        if (rc) return rc;
    } else {
        SYNC_CHECKED(m);
    }
    HCHK(hipEventElapsedTime(&m->last_ms, m->ev0, m->ev1));
    m->step_timed = false;
    m->len += n;
    return HIPDEC_OK;
}

int hipdec_batch_begin(hipdec_model *m, size_t n_rows) {
    if (!m) return HIPDEC_ERR_ARG;
    if (n_rows == 0 || n_rows > (size_t)kBatchMaxRows) return fail(m, HIPDEC_ERR_ARG, "n_rows must be in 1..32");
    if (!prefill_batched_ok(m, kPrefillMinRows))
        return fail(m, HIPDEC_ERR_UNSUPPORTED, "multi-row decode needs dimensions that are multiples of 32 (128 with 4-bit weights) and a head dimension of 64 or 128");
    if (m->len >= m->cfg.seq) return fail(m, HIPDEC_ERR_FULL, "decode only supports lengths within cfg.seq");
    int rc = batch_alloc(m, (int)n_rows);
    if (rc) return rc;
    const bool was_active = m->bt.rows_active;
    if ((rc = rows_prepare(m, (int)n_rows))) return rc;
    if (was_active != m->bt.rows_active)                              // the captured steps hold the other form
        for (auto &g : m->bt.graphs) if (g) { (void)hipGraphExecDestroy(g); g = nullptr; }
    m->bt.rows = (int)n_rows;
    m->bt.prefix = m->len;
    m->bt.slot = 0;
    m->bt.have_logits = false;
    return HIPDEC_OK;
}

int hipdec_batch_end(hipdec_model *m) {
    if (!m) return HIPDEC_ERR_ARG;
    m->bt.rows = 0;
    m->bt.have_logits = false;
    return HIPDEC_OK;
}

int hipdec_batch_layers_in_one_launch(const hipdec_model *m, int *out) {
    if (!m || !out) return HIPDEC_ERR_ARG;
    *out = (m->bt.rows && m->bt.rows_active) ? 1 : 0;
    return HIPDEC_OK;
}

int hipdec_batch_steps(const hipdec_model *m, size_t *out_steps) {
    if (!m || !out_steps) return HIPDEC_ERR_ARG;
    *out_steps = m->bt.rows ? m->bt.slot : 0;
    return HIPDEC_OK;
}

int hipdec_decode_logits_from_ids_batch(hipdec_model *m, const uint32_t *tokens, float softcap, float *out_logits) {
    if (!m || !out_logits) return HIPDEC_ERR_ARG;
    int rc = batch_step(m, tokens, B_LOGITS, 1, 1.0f, 0.0f);
    if (rc) return rc;
    const size_t n = (size_t)m->bt.rows * m->cfg.vocab;
    hipLaunchKernelGGL(k_softcap_copy, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, m->stream, m->bt.logits,
                       m->bt.d_out, 0, (int)n, softcap);
    HCHK(hipGetLastError());
    return batch_fetch(m, m->bt.d_out, out_logits, n);
}

int hipdec_decode_token_argmax_from_ids_batch(hipdec_model *m, const uint32_t *tokens, uint32_t *out_tokens) {
    if (!m || !out_tokens) return HIPDEC_ERR_ARG;
    int rc = batch_step(m, tokens, B_ARGMAX, 1, 1.0f, 0.0f);
    if (rc) return rc;
    return batch_fetch(m, m->bt.d_tok, out_tokens, (size_t)m->bt.rows);
}

int hipdec_decode_token_topk_from_ids_batch(hipdec_model *m, const uint32_t *tokens, uint32_t top_k, float *out_vals,
                                            uint32_t *out_idxs, size_t cap, size_t *out_count) {
    if (!m || !out_vals || !out_idxs) return HIPDEC_ERR_ARG;
    if (top_k == 0 || top_k > HIPDEC_MAX_GPU_TOPK) return fail(m, HIPDEC_ERR_ARG, "gpu top-k only supports k in 1..32");
    const size_t per_row = (size_t)m->blocks * top_k, n = per_row * (size_t)std::max(m->bt.rows, 1);
    if (cap < n) return fail(m, HIPDEC_ERR_ARG, "top-k outputs must fit the per-block candidates of every row");
    int rc = batch_step(m, tokens, B_TOPK, top_k, 1.0f, 0.0f);
    if (rc) return rc;
    if ((rc = batch_fetch(m, m->bt.d_vals, out_vals, n))) return rc;
    if ((rc = batch_fetch(m, m->bt.d_idxs, out_idxs, n))) return rc;
    if (out_count) *out_count = per_row;
    return HIPDEC_OK;
}

int hipdec_decode_token_block_stats_from_ids_batch(hipdec_model *m, const uint32_t *tokens, float inv_temperature,
                                                   float softcap, float *out_maxes, float *out_sums, size_t cap,
                                                   size_t *out_count) {
    if (!m || !out_maxes || !out_sums) return HIPDEC_ERR_ARG;
    const size_t n = (size_t)m->blocks * (size_t)std::max(m->bt.rows, 1);
    if (cap < n) return fail(m, HIPDEC_ERR_ARG, "block stats outputs must fit the vocab blocks of every row");
    int rc = batch_step(m, tokens, B_STATS, 1, inv_temperature, softcap);
    if (rc) return rc;
    if ((rc = batch_fetch(m, m->bt.d_bmax, out_maxes, n))) return rc;
    if ((rc = batch_fetch(m, m->bt.d_bsum, out_sums, n))) return rc;
    if (out_count) *out_count = (size_t)m->blocks;
    return HIPDEC_OK;
}

int hipdec_materialize_current_logits_block_batch(hipdec_model *m, size_t row, size_t block_idx, float softcap,
                                                  float *out_logits, size_t cap, size_t *out_valid) {
    if (!m || !out_logits) return HIPDEC_ERR_ARG;
    BatchState &b = m->bt;
    if (b.rows <= 0 || !b.have_logits) return fail(m, HIPDEC_ERR_ARG, "no batched step has run");
    if (row >= (size_t)b.rows) return fail(m, HIPDEC_ERR_ARG, "row out of range");
    if (block_idx >= (size_t)m->blocks) return fail(m, HIPDEC_ERR_ARG, "block index out of range");
    const size_t V = m->cfg.vocab, start = block_idx * HIPDEC_HEAD_BLOCK;
    const size_t valid = std::min<size_t>(HIPDEC_HEAD_BLOCK, V - start);
    if (cap < valid) return fail(m, HIPDEC_ERR_ARG, "logits block output too small");
    hipLaunchKernelGGL(k_softcap_copy, dim3(1), dim3(256), 0, m->stream, b.logits + row * V, b.d_out, (int)start, (int)valid,
                       softcap);
    HCHK(hipGetLastError());
    int rc = batch_fetch(m, b.d_out, out_logits, valid);
    if (rc) return rc;
    if (out_valid) *out_valid = valid;
    return HIPDEC_OK;
}

int hipdec_requests_open(hipdec_model *m, uint32_t page_size, uint32_t n_pages, uint32_t max_seqs) {
    if (!m) return HIPDEC_ERR_ARG;
    if (m->rq.open) return fail(m, HIPDEC_ERR_ARG, "the model's pages are open already");
    if (!page_size || (page_size & (page_size - 1)) || page_size > 65536) return fail(m, HIPDEC_ERR_ARG, "page_size must be a power of two up to 65536");
    if (!n_pages || n_pages > 0x7fffffffu || !max_seqs || max_seqs > 65536) return fail(m, HIPDEC_ERR_ARG, "n_pages or max_seqs out of range");
    if (!prefill_batched_ok(m, kPrefillMinRows) || m->cfg.vocab > 262144)
        return fail(m, HIPDEC_ERR_UNSUPPORTED, "requests stepped together need dimensions that are multiples of 32 (128 with 4-bit weights), a head dimension of 64 or 128 and a vocabulary up to 262144");
    const size_t had = m->allocs.size();
    int rc;
    try { rc = requests_open(m, page_size, n_pages, max_seqs); } catch (...) { rc = fail(m, HIPDEC_ERR_HIP, "out of host memory"); }
    if (rc == HIPDEC_OK) return rc;
    // too large a pool: everything back, so that a smaller one can be opened
    RequestState &r = m->rq;
    for (; m->allocs.size() > had; m->allocs.pop_back()) (void)hipFree(m->allocs.back());
    if (r.h_rows) (void)hipHostFree(r.h_rows);
    if (r.h_u) (void)hipHostFree(r.h_u);
    if (r.h_tok) (void)hipHostFree(r.h_tok);
    r = RequestState{};
    (void)hipGetLastError();                                  // (the failed allocation's: it is reported, and must not be again)
    return rc;
}

int hipdec_requests_admit(hipdec_model *m, uint32_t seq) {
    if (!m) return HIPDEC_ERR_ARG;
    RequestState &r = m->rq;
    if (!r.open) return fail(m, HIPDEC_ERR_ARG, "no pages are open (hipdec_requests_open)");
    if (m->bt.rows) return fail(m, HIPDEC_ERR_ARG, "a batch is open");
    if (seq >= r.max_seqs || r.lens[seq] >= 0) return fail(m, HIPDEC_ERR_ARG, "sequence out of range or admitted already");
    if (request_pages_missing(m, seq, m->len) > r.free_pages.size()) return fail(m, HIPDEC_ERR_FULL, "not enough free pages");
    HCHK(hipSetDevice(m->opt.device));
    (void)hipGetLastError();                                  // (an earlier call's, not this one's launches')
    HCHK(hipStreamSynchronize(m->stream));
    const RequestTrim trim{m, &seq, 1};
    request_pages(m, seq, m->len);
    const int rc = request_table_up(m, seq);
    if (rc) return rc;
    const int pieces = (int)(m->cfg.kv_dim * (m->kvbf16 ? 2 : 4) / 16);
    if (m->len)
        for (uint32_t l = 0; l < m->cfg.nlayers; ++l) {
            const DevLayer &L = m->layers[l];
            for (int which = 0; which < 2; ++which)
                hipLaunchKernelGGL(k_rq_admit, dim3((unsigned)m->len), dim3(256), 0, m->stream, (const uint4 *)(which ? L.vc : L.kc),
                                   (uint4 *)(which ? r.v[l] : r.k[l]), r.d_table + (size_t)seq * r.max_pages, r.page_shift, pieces, (int)m->len);
        }
    HCHK(hipGetLastError());
    HCHK(hipStreamSynchronize(m->stream));
    r.lens[seq] = (long long)m->len;
    return HIPDEC_OK;
}

int hipdec_requests_release(hipdec_model *m, uint32_t seq) {
    if (!m) return HIPDEC_ERR_ARG;
    RequestState &r = m->rq;
    if (!r.open || seq >= r.max_seqs || r.lens[seq] < 0) return fail(m, HIPDEC_ERR_ARG, "no such sequence");
    int *row = &r.table[(size_t)seq * r.max_pages];
    for (int p = 0; p < r.max_pages; ++p)
        if (row[p] >= 0) { r.free_pages.push_back(row[p]); row[p] = -1; }
    r.lens[seq] = -1;
    return HIPDEC_OK;
}

int hipdec_requests_len(const hipdec_model *m, uint32_t seq, size_t *out_len, size_t *out_free_pages) {
    if (!m) return HIPDEC_ERR_ARG;
    hipdec_model *told = const_cast<hipdec_model *>(m);       // (its error text only)
    if (!m->rq.open) return fail(told, HIPDEC_ERR_ARG, "no pages are open (hipdec_requests_open)");
    if (seq >= m->rq.max_seqs || m->rq.lens[seq] < 0) return fail(told, HIPDEC_ERR_ARG, "no such sequence");
    if (out_len) *out_len = (size_t)m->rq.lens[seq];
    if (out_free_pages) *out_free_pages = m->rq.free_pages.size();
    return HIPDEC_OK;
}

int hipdec_requests_step(hipdec_model *m, size_t n_seqs, const uint32_t *seqs, const uint32_t *tokens, uint32_t max_drafts,
                         const uint32_t *n_drafts, const uint32_t *drafts, const float *draft_probs, const float *uniforms,
                         float temperature, float softcap, uint32_t *out_tokens, uint32_t *out_accepted, float *out_logits) {
    if (!m) return HIPDEC_ERR_ARG;
    const hipdec_config &c = m->cfg;
    RequestState &r = m->rq;
    if (!r.open) return fail(m, HIPDEC_ERR_ARG, "no pages are open (hipdec_requests_open)");
    if (m->bt.rows) return fail(m, HIPDEC_ERR_ARG, "a batch is open");
    if (!seqs || !tokens || !out_tokens || !out_accepted || (max_drafts && !drafts)) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if (!(temperature >= 0.0f) || !std::isfinite(temperature) || !(softcap <= 3.4e38f)) return fail(m, HIPDEC_ERR_ARG, "temperature must not be negative, softcap must be finite");
    if (temperature > 0.0f && !uniforms) return fail(m, HIPDEC_ERR_ARG, "random numbers are missing");
    const size_t K = max_drafts, S = K + 1;
    if (n_seqs == 0 || n_seqs > (size_t)kRequestRows || S > (size_t)kRequestRows || n_seqs * S > (size_t)kRequestRows)
        return fail(m, HIPDEC_ERR_ARG, "n_seqs * (max_drafts + 1) must be in 1..32");
    size_t missing = 0, max_len = 0;
    for (size_t i = 0; i < n_seqs; ++i) {
        if (seqs[i] >= r.max_seqs || r.lens[seqs[i]] < 0) return fail(m, HIPDEC_ERR_ARG, "no such sequence");
        for (size_t j = 0; j < i; ++j) if (seqs[j] == seqs[i]) return fail(m, HIPDEC_ERR_ARG, "a sequence is named twice");
        const size_t nd = n_drafts ? n_drafts[i] : K;
        if (nd > K) return fail(m, HIPDEC_ERR_ARG, "more drafts than max_drafts");
        if (tokens[i] >= c.vocab) return fail(m, HIPDEC_ERR_ARG, "token id must fit vocab");
        for (size_t j = 0; j < nd; ++j) if (drafts[i * K + j] >= c.vocab) return fail(m, HIPDEC_ERR_ARG, "token id must fit vocab");
        const size_t len = (size_t)r.lens[seqs[i]] + 1 + nd;
        if (len > c.seq) return fail(m, HIPDEC_ERR_FULL, "decode only supports lengths within cfg.seq");
        missing += request_pages_missing(m, seqs[i], len);
        max_len = std::max(max_len, len);
    }
    if (missing > r.free_pages.size()) return fail(m, HIPDEC_ERR_FULL, "not enough free pages");

    const int R = (int)(n_seqs * S);
    HCHK(hipSetDevice(m->opt.device));
    (void)hipGetLastError();                                    // (an earlier call's, not this one's launches')
    int rc = pf_ensure(m, R, true);
    if (rc) return rc;
    if (draft_probs && K && temperature > 0.0f && !r.d_probs && (rc = dalloc(m, &r.d_probs, (size_t)kRequestRows * c.vocab * 4))) return rc;
    PrefillWork &w = m->pf;
    HCHK(hipStreamSynchronize(m->stream));                      // pinned staging is free again
    const RequestTrim trim{m, seqs, n_seqs};
    int *pos = r.h_rows, *slot = pos + kRequestRows, *sq = slot + kRequestRows, *ln = sq + kRequestRows, *dr = ln + kRequestRows, *nn = dr + kRequestRows;
    for (size_t i = 0; i < n_seqs; ++i) {
        const size_t nd = n_drafts ? n_drafts[i] : K, len = (size_t)r.lens[seqs[i]];
        request_pages(m, seqs[i], len + 1 + nd);
        if ((rc = request_table_up(m, seqs[i]))) return rc;
        nn[i] = (int)nd;
        for (size_t j = 0; j < S; ++j) {
            const size_t row = i * S + j;
            const bool real = j <= nd;                          // a row behind the sequence's drafts: written nowhere, sees nothing
            w.h_ids[row] = !real ? 0 : j == 0 ? tokens[i] : drafts[i * K + j - 1];
            pos[row] = real ? (int)(len + j) : 0;
            slot[row] = real ? (int)(len + j) : -1;
            sq[row] = (int)seqs[i];
            ln[row] = real ? (int)(len + j + 1) : 0;
            if (j < K) dr[i * K + j] = j < nd ? (int)drafts[i * K + j] : -1;
            if (temperature > 0.0f) r.h_u[row] = uniforms[row];
        }
    }
    HCHK(hipMemcpyAsync(w.ids, w.h_ids, (size_t)R * 4, hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(r.d_rows, r.h_rows, 5 * kRequestRows * 4, hipMemcpyHostToDevice, m->stream));
    HCHK(hipMemcpyAsync(r.d_n, nn, n_seqs * 4, hipMemcpyHostToDevice, m->stream));
    if (temperature > 0.0f) HCHK(hipMemcpyAsync(r.d_u, r.h_u, (size_t)R * 4, hipMemcpyHostToDevice, m->stream));
    const bool probs = draft_probs && K && temperature > 0.0f;
    if (probs) HCHK(hipMemcpyAsync(r.d_probs, draft_probs, n_seqs * K * c.vocab * 4, hipMemcpyHostToDevice, m->stream));
    HCHK(hipEventRecord(m->ev0, m->stream));
    if ((rc = requests_forward(m, R, max_len))) return rc;
    const hipdec_drafts v{r.logits, HIPDEC_ROWS_F32, c.vocab, n_seqs, max_drafts, temperature, softcap, (int64_t)c.vocab, (int64_t)c.vocab,
                          r.d_rows + 4 * kRequestRows, r.d_n, probs ? r.d_probs : nullptr, r.d_u, r.d_tok, (int32_t *)r.d_tok + kRequestRows};
    OPCHK(hipdec_verify_drafts(&v, r.ws_ver, r.ws_ver_bytes, m->stream));
    HCHK(hipEventRecord(m->ev1, m->stream));
    HCHK(hipMemcpyAsync(r.h_tok, r.d_tok, 2 * kRequestRows * 4, hipMemcpyDeviceToHost, m->stream));
    if (out_logits) HCHK(hipMemcpyAsync(out_logits, r.logits, (size_t)R * c.vocab * 4, hipMemcpyDeviceToHost, m->stream));
    HCHK(hipStreamSynchronize(m->stream));
    HCHK(hipEventElapsedTime(&m->last_ms, m->ev0, m->ev1));
    m->step_timed = false;
    memcpy(out_tokens, r.h_tok, (size_t)R * 4);
    for (size_t i = 0; i < n_seqs; ++i) {
        out_accepted[i] = r.h_tok[kRequestRows + i];
        r.lens[seqs[i]] += 1 + (long long)out_accepted[i];
    }
    return HIPDEC_OK;
}

int hipdec_decode_greedy_run(hipdec_model *m, uint32_t token, size_t n_steps, uint32_t *out_tokens) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (n_steps == 0) return HIPDEC_OK;
    if (!out_tokens) return fail(m, HIPDEC_ERR_ARG, "null buffer");
    if (m->len + n_steps > m->cfg.seq) return fail(m, HIPDEC_ERR_FULL, "greedy run exceeds cfg.seq");
    m->h_sp[0] = base_params(m, token);
    HCHK(hipMemcpyAsync(m->d_sp, &m->h_sp[0], sizeof(StepParams), hipMemcpyHostToDevice, m->stream));
    HCHK(hipEventRecord(m->ev0, m->stream));
    for (size_t i = 0; i < n_steps; ++i)
        if ((rc = run_step(m, V_ARGMAX))) return rc;
    HCHK(hipEventRecord(m->ev1, m->stream));
    HCHK(hipMemcpyAsync(m->h_out, m->d_ring, n_steps * 4, hipMemcpyDeviceToHost, m->stream));
    SYNC_CHECKED(m);
    HCHK(hipEventElapsedTime(&m->last_ms, m->ev0, m->ev1));
    m->step_timed = false;
    memcpy(out_tokens, m->h_out, n_steps * 4);
    m->len += n_steps;
    return HIPDEC_OK;
}

int hipdec_decode_topk_sampled_run(hipdec_model *m, uint32_t token, uint32_t top_k, float temperature, float softcap,
                                   uint64_t *rng_state, size_t n_steps, uint32_t *out_tokens) {
    return sampled_run(m, V_TOPK_S, token, top_k, temperature, softcap, rng_state, n_steps, out_tokens);
}

int hipdec_decode_fullvocab_sampled_run(hipdec_model *m, uint32_t token, float temperature, float softcap,
                                        uint64_t *rng_state, size_t n_steps, uint32_t *out_tokens) {
    return sampled_run(m, V_STATS_S, token, 1, temperature, softcap, rng_state, n_steps, out_tokens);
}

int hipdec_decode_topk_sampled_run_batch(hipdec_model *m, const uint32_t *tokens, uint32_t top_k, float temperature,
                                         float softcap, uint64_t *rng_states, size_t n_steps, uint32_t *out_tokens) {
    return batch_sampled_run(m, B_TOPK_S, tokens, top_k, temperature, softcap, rng_states, n_steps, out_tokens);
}

int hipdec_decode_fullvocab_sampled_run_batch(hipdec_model *m, const uint32_t *tokens, float temperature, float softcap,
                                              uint64_t *rng_states, size_t n_steps, uint32_t *out_tokens) {
    return batch_sampled_run(m, B_STATS_S, tokens, 1, temperature, softcap, rng_states, n_steps, out_tokens);
}

int hipdec_debug_step_kernel(const hipdec_model *m, int *out) {
    if (!m || !out) return HIPDEC_ERR_ARG;
    *out = !m->mega_ok ? 0 : m->lean_ce ? 2 : 1;
    return HIPDEC_OK;
}

int hipdec_debug_gemm_plan(uint32_t weight_dtype, int rows, int n, int k, int num_cu, uint64_t out[8]) {
    if (!out || weight_dtype > HIPDEC_W_INT4_G128 || rows < 1 || n < 1 || k < PF_BK || k % PF_BK || num_cu < 1) return HIPDEC_ERR_ARG;
    if (weight_dtype == HIPDEC_W_INT4_G128 && k % 128) return HIPDEC_ERR_ARG;
    if (weight_dtype == HIPDEC_W_F32 && rows > kSkinnyRows) return HIPDEC_ERR_ARG;     // fp32 weights go 32 rows at a time
    const PfPlan p = pf_plan(num_cu, (int)weight_dtype, rows, n, k, PF_ACT_PAIR);
    out[0] = (uint64_t)p.kernel; out[1] = (uint64_t)p.splits; out[2] = (uint64_t)p.steps_per_split;
    out[3] = p.gx; out[4] = p.gy; out[5] = p.gz; out[6] = p.threads; out[7] = p.lds;
    return HIPDEC_OK;
}

int hipdec_debug_set_spin_limit(uint32_t check_mask, uint32_t limit) {
    const unsigned v[2] = {check_mask, limit};
    hipError_t e = hipDeviceSynchronize();
    if (e == hipSuccess) e = hipMemcpyToSymbol(HIP_SYMBOL(g_spin_ctl), v, sizeof v);
    if (e != hipSuccess) { g_create_error = std::string("hipdec_debug_set_spin_limit: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    return HIPDEC_OK;
}

int hipdec_debug_hostmath_probe(void) { return hostmath_matches_libm() ? 1 : 0; }

int hipdec_debug_sample_topk(const float *vals, const uint32_t *idxs, size_t blocks, uint32_t top_k, float temperature,
                             float softcap, uint64_t *rng_state, uint32_t *out_token) {
    if (!vals || !idxs || !rng_state || !out_token || blocks == 0 || blocks > SAMPLE_MAX_BLOCKS || top_k == 0 ||
        top_k > HIPDEC_MAX_GPU_TOPK)
        return HIPDEC_ERR_ARG;
    hipError_t e = hipSuccess;
    DebugDraw d;
    const SampleParams sp{temperature, softcap, (int)top_k, 0, 1, 0u};
    const uint32_t zero = 0;
    float *dv = d.up(vals, blocks * top_k, &e);
    uint32_t *di = d.up(idxs, blocks * top_k, &e);
    SampleParams *dsp = d.up(&sp, 1, &e);
    uint64_t *drng = d.up(rng_state, 1, &e);
    uint32_t *dtok = d.up(&zero, 1, &e), *dring = d.up(&zero, 1, &e);
    if (e == hipSuccess) {
        hipLaunchKernelGGL(k_sample_topk, dim3(1), dim3(256), 0, nullptr, dv, di, (int)blocks, dsp, drng, dtok, dring,
                           (BatchParams *)nullptr);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpy(out_token, dtok, 4, hipMemcpyDeviceToHost);
    if (e == hipSuccess) e = hipMemcpy(rng_state, drng, 8, hipMemcpyDeviceToHost);
    if (e != hipSuccess) { g_create_error = std::string("hipdec_debug_sample_topk: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    return HIPDEC_OK;
}

int hipdec_debug_sample_fullvocab(const float *logits, size_t vocab, const float *maxes, const float *sums, float temperature,
                                  float softcap, uint64_t *rng_state, uint32_t *out_token) {
    const size_t blocks = (vocab + HIPDEC_HEAD_BLOCK - 1) / HIPDEC_HEAD_BLOCK;
    if (!logits || !maxes || !sums || !rng_state || !out_token || vocab == 0 || blocks > SAMPLE_MAX_BLOCKS ||
        !(temperature > 0.0f))
        return HIPDEC_ERR_ARG;
    hipError_t e = hipSuccess;
    DebugDraw d;
    const SampleParams sp{temperature, softcap, 1, 0, 1, 0u};
    const uint32_t zero = 0;
    float *dl = d.up(logits, vocab, &e), *dm = d.up(maxes, blocks, &e), *ds = d.up(sums, blocks, &e);
    SampleParams *dsp = d.up(&sp, 1, &e);
    uint64_t *drng = d.up(rng_state, 1, &e);
    uint32_t *dtok = d.up(&zero, 1, &e), *dring = d.up(&zero, 1, &e);
    if (e == hipSuccess) {
        hipLaunchKernelGGL(k_sample_fullvocab, dim3(1), dim3(256), 0, nullptr, dl, (int)vocab, dm, ds, (int)blocks, dsp, drng,
                           dtok, dring, (BatchParams *)nullptr);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpy(out_token, dtok, 4, hipMemcpyDeviceToHost);
    if (e == hipSuccess) e = hipMemcpy(rng_state, drng, 8, hipMemcpyDeviceToHost);
    if (e != hipSuccess) { g_create_error = std::string("hipdec_debug_sample_fullvocab: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    return HIPDEC_OK;
}

// ---- the full-vocabulary draw for callers that may not allocate (see include/hip_decode.h)
// Run state of the draw kernel (SampleParams with its arrival counter at byte 0, the one-slot token
// ring at byte 64).  Every GPU the library runs on holds its own copy of this array until the process
// ends; host code reaches it only through the address hipGetSymbolAddress returns for the current device.
#define NOALLOC_SCRATCH_BYTES 256
#define NOALLOC_MAX_VOCAB ((size_t)SAMPLE_MAX_BLOCKS * HIPDEC_HEAD_BLOCK)
static __device__ __align__(256) unsigned char scratch[NOALLOC_SCRATCH_BYTES];

// (a kernel, not hipMemsetAsync: the call may be recorded into a graph)
__global__ void k_noalloc_reset(SampleParams *ss, uint32_t *ring, float temperature, float softcap) {
    ss->temperature = temperature; ss->softcap = softcap; ss->top_k = 1; ss->step = 0; ss->ring_cap = 1; ss->done = 0u;
    *ring = 0u;
}

static std::mutex g_scratch_mu;
static void *g_scratch_ptr[64] = {};      // by device ordinal

// This device's copy of the array, looked up once per device (hipGetSymbolAddress may load the code object,
// which must not happen under stream capture: hipdec_create* call this, so a process that has created a
// model on the device can record the entry point below into a graph from its first call on).
static void *noalloc_scratch() {
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) { (void)hipGetLastError(); return nullptr; }
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    if (!g_scratch_ptr[dev]) {
        void *p = nullptr;
        if (hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)) == hipSuccess) g_scratch_ptr[dev] = p;
        else (void)hipGetLastError();
    }
    return g_scratch_ptr[dev];
}

int hipdec_sample_fullvocab_noalloc(const float *d_logits, size_t vocab, const float *d_maxes, const float *d_sums,
                                    float temperature, float softcap, uint64_t *d_rng_state, uint32_t *d_out_token,
                                    void *stream) {
    if (!d_logits || !d_maxes || !d_sums || !d_rng_state || !d_out_token || vocab == 0 || !(temperature > 0.0f)) {
        g_create_error = "hipdec_sample_fullvocab_noalloc: null buffer, empty vocabulary or non-positive temperature";
        return HIPDEC_ERR_ARG;
    }
    if (vocab > NOALLOC_MAX_VOCAB) {
        g_create_error = "hipdec_sample_fullvocab_noalloc: vocab exceeds the 262144 rows (1024 blocks of 256) this entry point serves";
        return HIPDEC_ERR_ARG;
    }
    hipError_t e = hipSuccess;
    void *base = noalloc_scratch();
    if (!base) {
        g_create_error = "hipdec_sample_fullvocab_noalloc: no scratch array for the current device";
        return HIPDEC_ERR_UNSUPPORTED;
    }
    if (e == hipSuccess) {
        SampleParams *ss = (SampleParams *)base;
        uint32_t *ring = (uint32_t *)((unsigned char *)base + 64);
        const int blocks = (int)((vocab + HIPDEC_HEAD_BLOCK - 1) / HIPDEC_HEAD_BLOCK);
        hipStream_t s = (hipStream_t)stream;
        hipLaunchKernelGGL(k_noalloc_reset, dim3(1), dim3(1), 0, s, ss, ring, temperature, softcap);
        hipLaunchKernelGGL(k_sample_fullvocab, dim3(1), dim3(256), 0, s, d_logits, (int)vocab, d_maxes, d_sums, blocks, ss,
                           d_rng_state, d_out_token, ring, (BatchParams *)nullptr);
        e = hipGetLastError();
    }
    if (e != hipSuccess) { g_create_error = std::string("hipdec_sample_fullvocab_noalloc: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    return HIPDEC_OK;
}

int hipdec_debug_hostmath_eval(int fn, const float *in, float *out, size_t n, int on_device) {
    if (!in || !out || (fn != HOSTMATH_EXPF && fn != HOSTMATH_TANHF)) return HIPDEC_ERR_ARG;
    if (!on_device) {
        for (size_t i = 0; i < n; ++i) out[i] = hostmath_eval(fn, in[i]);
        return HIPDEC_OK;
    }
    if (n == 0) return HIPDEC_OK;
    float *d_in = nullptr, *d_out = nullptr;
    hipError_t e = hipMalloc((void **)&d_in, n * 4);
    if (e == hipSuccess) e = hipMalloc((void **)&d_out, n * 4);
    if (e == hipSuccess) e = hipMemcpy(d_in, in, n * 4, hipMemcpyHostToDevice);
    if (e == hipSuccess) {
        hipLaunchKernelGGL(k_hostmath_eval, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, nullptr, fn, d_in, d_out, n);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpy(out, d_out, n * 4, hipMemcpyDeviceToHost);
    if (d_in) (void)hipFree(d_in);
    if (d_out) (void)hipFree(d_out);
    if (e != hipSuccess) { g_create_error = std::string("hipdec_debug_hostmath_eval: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    return HIPDEC_OK;
}

int hipdec_debug_hostmath_checksum(int fn, uint32_t first_bits, uint64_t count, int on_device, int host_threads,
                                   uint64_t *out) {
    if (!out || count > (1ull << 32) || (uint64_t)first_bits + count > (1ull << 32)) return HIPDEC_ERR_ARG;
    if (fn != HOSTMATH_EXPF && fn != HOSTMATH_TANHF) return HIPDEC_ERR_ARG;
    if (!on_device) {
        uint64_t parts[64] = {};
        hostmath_host_range(first_bits, count, host_threads, [&](int t, uint32_t lo, uint64_t n) {
            uint64_t acc = 0;
            for (uint64_t i = 0; i < n; ++i) acc += hostmath_mix(fn, lo + (uint32_t)i);
            parts[t] = acc;
        });
        uint64_t total = 0;
        for (uint64_t v : parts) total += v;
        *out = total;
        return HIPDEC_OK;
    }
    unsigned long long *d_acc = nullptr, h_acc = 0;
    hipError_t e = hipMalloc((void **)&d_acc, 8);
    if (e == hipSuccess) e = hipMemset(d_acc, 0, 8);
    if (e == hipSuccess && count) {
        hipLaunchKernelGGL(k_hostmath_checksum, dim3(4096), dim3(256), 0, nullptr, fn, first_bits, count, d_acc);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpy(&h_acc, d_acc, 8, hipMemcpyDeviceToHost);
    if (d_acc) (void)hipFree(d_acc);
    if (e != hipSuccess) { g_create_error = std::string("hipdec_debug_hostmath_checksum: ") + hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    *out = (uint64_t)h_acc;
    return HIPDEC_OK;
}

int hipdec_debug_hostmath_count_mismatch(int fn, uint32_t first_bits, uint64_t count, int host_threads,
                                         uint64_t *out_mismatches) {
    if (!out_mismatches || count > (1ull << 32) || (uint64_t)first_bits + count > (1ull << 32)) return HIPDEC_ERR_ARG;
    if (fn != HOSTMATH_EXPF && fn != HOSTMATH_TANHF) return HIPDEC_ERR_ARG;
    uint64_t parts[64] = {};
    hostmath_host_range(first_bits, count, host_threads, [&](int t, uint32_t lo, uint64_t n) {
        uint64_t bad = 0;
        for (uint64_t i = 0; i < n; ++i) {
            const uint32_t bits = lo + (uint32_t)i;
            float x;
            memcpy(&x, &bits, 4);
            const float a = fn == HOSTMATH_TANHF ? tanhf(x) : expf(x), b = hostmath_eval(fn, x);
            uint32_t ab, bb;
            memcpy(&ab, &a, 4);
            memcpy(&bb, &b, 4);
            if (ab != bb && !(a != a && b != b)) ++bad;           // any two NaNs agree
        }
        parts[t] = bad;
    });
    uint64_t total = 0;
    for (uint64_t v : parts) total += v;
    *out_mismatches = total;
    return HIPDEC_OK;
}

int hipdec_last_device_ms(const hipdec_model *m, float *out_ms) {
    if (!m || !out_ms) return HIPDEC_ERR_ARG;
    if (m->step_timed) {
        hipdec_model *mm = const_cast<hipdec_model *>(m);
        mm->step_timed = false;
        if (hipEventElapsedTime(&mm->last_ms, m->ev_s0, m->ev_s1) != hipSuccess) { (void)hipGetLastError(); mm->last_ms = 0.0f; }
    }
    *out_ms = m->last_ms;
    return HIPDEC_OK;
}

int hipdec_bytes_per_token(const hipdec_model *m, size_t kv_len, uint64_t *out_bytes) {
    if (!m || !out_bytes) return HIPDEC_ERR_ARG;
    const hipdec_config &c = m->cfg;
    const uint64_t D = c.dim, Q = c.q_dim, KV = c.kv_dim, H = c.hidden, V = c.vocab, L = c.nlayers;
    auto mat = [&](int wt, uint64_t rows, uint64_t K) { return (uint64_t)wt_row_bytes(wt, K) * rows + wt_scale_bytes(wt, rows, K); };
    uint64_t per_layer = mat(m->wt, Q + 2 * KV, D) + mat(m->wt, D, Q) + mat(m->wt, 2 * H, D) + mat(m->wt, D, H);
    uint64_t kvsz = m->kvbf16 ? 2 : 4;
    uint64_t b = L * per_layer + mat(m->embed_wt, V, D) + wt_row_bytes(m->embed_wt, D) + (2 * L + 1) * D * 4 +
                 L * 2 * (uint64_t)kv_len * KV * kvsz + L * 2 * KV * kvsz;
    *out_bytes = b;
    return HIPDEC_OK;
}

int hipdec_debug_calibration_copy(size_t bytes, int reps) {
    if (bytes < 16 || reps < 1) return HIPDEC_ERR_ARG;
    uint4 *src = nullptr, *dst = nullptr;
    if (hipMalloc((void **)&src, bytes) != hipSuccess) return HIPDEC_ERR_HIP;
    if (hipMalloc((void **)&dst, bytes) != hipSuccess) { (void)hipFree(src); return HIPDEC_ERR_HIP; }
    (void)hipMemset(src, 1, bytes);
    (void)hipMemset(dst, 0, bytes);
    for (int i = 0; i < reps; ++i)
        hipLaunchKernelGGL(k_calib_copy, dim3(2048), dim3(256), 0, nullptr, src, dst, bytes / 16);
    hipError_t e = hipDeviceSynchronize();
    (void)hipFree(src);
    (void)hipFree(dst);
    return e == hipSuccess ? HIPDEC_OK : HIPDEC_ERR_HIP;
}

int hipdec_debug_step_profile(hipdec_model *m, uint32_t token, uint64_t *out, size_t cap, size_t *out_count) {
    int rc = check_step(m, token, true);
    if (rc) return rc;
    if (!m->mega_ok) return fail(m, HIPDEC_ERR_UNSUPPORTED, "persistent step kernel is off");
    const size_t n = (size_t)(m->cfg.nlayers + 1) * MEGA_PROF_SLOTS;
    if (!out || cap < n) return fail(m, HIPDEC_ERR_ARG, "profile buffer too small");
    unsigned long long *d = nullptr;
    HCHK(hipMalloc((void **)&d, n * 8));
    HCHK(hipMemset(d, 0, n * 8));
    m->h_sp[0] = base_params(m, token);
    HCHK(hipMemcpyAsync(m->d_sp, &m->h_sp[0], sizeof(StepParams), hipMemcpyHostToDevice, m->stream));
    m->mega.prof = d;
    launch_mega(m, m->wt == m->embed_wt ? 1 : 0, 1);
    m->mega.prof = nullptr;
    rc = sync_checked(m);
    if (rc == HIPDEC_OK) {
        hipError_t e = hipMemcpy(out, d, n * 8, hipMemcpyDeviceToHost);
        if (e != hipSuccess) { m->err = hipGetErrorString(e); rc = HIPDEC_ERR_HIP; }
    }
    (void)hipFree(d);
    if (rc) return rc;
    if (out_count) *out_count = n;
    m->len += 1;
    return HIPDEC_OK;
}

int hipdec_debug_batch_step_profile(hipdec_model *m, const uint32_t *tokens, uint64_t *out, size_t cap, size_t *out_count) {
    if (!m) return HIPDEC_ERR_ARG;
    BatchState &b = m->bt;
    if (b.rows <= 0 || !b.rows_active) return fail(m, HIPDEC_ERR_UNSUPPORTED, "the open batch does not run its layers as one launch");
    const size_t n = (size_t)(m->cfg.nlayers + 1) * ROWS_PROF_SLOTS;
    if (!out || cap < n) return fail(m, HIPDEC_ERR_ARG, "profile buffer too small");
    unsigned long long *d = nullptr;
    HCHK(hipMalloc((void **)&d, n * 8));
    HCHK(hipMemset(d, 0, n * 8));
    const uint32_t saved = m->opt.flags;
    m->opt.flags |= HIPDEC_FLAG_NO_GRAPH;                    // (a captured step holds the plain build)
    b.rows_args.prof = d;
    int rc = batch_step(m, tokens, B_ARGMAX, 1, 1.0f, 0.0f);
    b.rows_args.prof = nullptr;
    m->opt.flags = saved;
    if (rc == HIPDEC_OK) {
        hipError_t e = hipStreamSynchronize(m->stream);
        if (e == hipSuccess) e = hipMemcpy(out, d, n * 8, hipMemcpyDeviceToHost);
        if (e != hipSuccess) { m->err = hipGetErrorString(e); rc = HIPDEC_ERR_HIP; }
        if (rc == HIPDEC_OK) rc = rows_check(m);
    }
    (void)hipFree(d);
    if (rc) return rc;
    if (out_count) *out_count = n;
    return HIPDEC_OK;
}

int hipdec_export_weight(hipdec_model *m, size_t layer_idx, uint32_t which, float *out, size_t cap) {
    if (!m || !out) return HIPDEC_ERR_ARG;
    const hipdec_config &c = m->cfg;
    const void *src = nullptr, *sc = nullptr;
    size_t rows = 0, K = 0;
    int wt = m->wt;
    if (which == 4) { src = m->embed; rows = c.vocab; K = c.dim; wt = m->embed_wt; }
    else {
        if (layer_idx >= c.nlayers) return fail(m, HIPDEC_ERR_ARG, "layer_idx out of range");
        const DevLayer &L = m->layers[layer_idx];
        switch (which) {
            case 0: src = L.wqkv; sc = L.s_qkv; rows = c.q_dim + 2 * c.kv_dim; K = c.dim; break;
            case 1: src = L.wo; sc = L.s_wo; rows = c.dim; K = c.q_dim; break;
            case 2: src = L.w13; sc = L.s_w13; rows = 2 * c.hidden; K = c.dim; break;
            case 3: src = L.w2; sc = L.s_w2; rows = c.dim; K = c.hidden; break;
            default: return fail(m, HIPDEC_ERR_ARG, "unknown weight selector");
        }
    }
    if (cap < rows * K) return fail(m, HIPDEC_ERR_ARG, "export buffer too small");
    float *tmp = nullptr;
    HCHK(hipMalloc((void **)&tmp, rows * K * 4));
    switch (wt) {
        case WT_F32: hipLaunchKernelGGL(k_export_rows<WT_F32>, dim3(rows), dim3(256), 0, m->stream, src, sc, tmp, (int)K); break;
        case WT_BF16: hipLaunchKernelGGL(k_export_rows<WT_BF16>, dim3(rows), dim3(256), 0, m->stream, src, sc, tmp, (int)K); break;
        case WT_FP8: hipLaunchKernelGGL(k_export_rows<WT_FP8>, dim3(rows), dim3(256), 0, m->stream, src, sc, tmp, (int)K); break;
        default: hipLaunchKernelGGL(k_export_rows<WT_INT4>, dim3(rows), dim3(256), 0, m->stream, src, sc, tmp, (int)K); break;
    }
    hipError_t e = hipStreamSynchronize(m->stream);
    if (e == hipSuccess) e = hipMemcpy(out, tmp, rows * K * 4, hipMemcpyDeviceToHost);
    (void)hipFree(tmp);
    if (e != hipSuccess) { m->err = hipGetErrorString(e); return HIPDEC_ERR_HIP; }
    return HIPDEC_OK;
}

}  // extern "C"
