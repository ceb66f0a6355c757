// What the paged-cache and draft-verification kernels need of the GPU beyond emu.h: shuffles from any lane, ballots,
// the fp32 matrix instructions, double-precision shuffles and the bit-level conversions.  All of them meet at the
// wave's barrier: the kernels call them under wave-uniform control flow.
#pragma once
#include "emu.h"
#include <algorithm>
#include <cmath>

namespace emu {
// What the lanes of one wave exchange: two sets of slots in turn, so that one meeting per exchange is enough (a lane
// writes a set again only behind the next meeting, which every reader of it has reached by then).
struct Exchange {
    uint64_t slot[2][64];
    std::atomic<int> count{0};
    std::atomic<unsigned> turn{0};
    void meet() {
        const unsigned t = turn.load(std::memory_order_acquire);
        if (count.fetch_add(1, std::memory_order_acq_rel) == 63) {
            count.store(0, std::memory_order_relaxed);
            turn.store(t + 1, std::memory_order_release);
        } else {
            while (turn.load(std::memory_order_acquire) == t) std::this_thread::yield();
        }
    }
    // every lane's value, as the lane's own view of this exchange
    template <class T> const uint64_t *share(int lane, T v) {
        const unsigned set = turn.load(std::memory_order_acquire) & 1;
        slot[set][lane] = 0;
        std::memcpy(&slot[set][lane], &v, sizeof(T));
        meet();
        return slot[set];
    }
};
inline Exchange g_exchange[16];                              // (one workgroup runs at a time)
template <class T> inline const uint64_t *share(T v) {
    static_assert(sizeof(T) <= 8, "");
    return g_exchange[tl_thread.x >> 6].share(lane(), v);
}
template <class T> inline T of_bits(uint64_t u) { T r; std::memcpy(&r, &u, sizeof(T)); return r; }
template <class T> inline T from_lane(T v, int src) { return of_bits<T>(share(v)[src & 63]); }
inline uint64_t ballot(bool p) {
    const uint64_t *all = share((uint32_t)p);
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= all[i] << i;
    return r;
}
// v_mfma_f32_16x16x4_f32: D = A (16 x 4) . B (4 x 16) + C.  Lane l supplies A[l % 16][l / 16] and B[l / 16][l % 16];
// register r of lane l holds D[4 * (l / 16) + r][l % 16].
template <class V4> inline V4 mfma_16x16x4(float a, float b, V4 c) {
    const uint64_t *all = share((uint64_t)float_as_uint(a) | (uint64_t)float_as_uint(b) << 32);
    const int l = lane();
    V4 d = c;
    for (int r = 0; r < 4; ++r)
        for (int k = 0; k < 4; ++k)
            d[r] = std::fmaf(uint_as_float((uint32_t)all[16 * k + 4 * (l / 16) + r]), uint_as_float((uint32_t)(all[16 * k + l % 16] >> 32)), d[r]);
    return d;
}
// v_mfma_f32_4x4x1_16b_f32: sixteen products of 4 x 1 by 1 x 4.  Lane l supplies A[l % 4] and B[l % 4] of block l / 4;
// register r of lane l holds D[r][l % 4] of that block.
template <class V4> inline V4 mfma_4x4x1(float a, float b, V4 c) {
    const uint64_t *all = share(a);
    V4 d = c;
    for (int r = 0; r < 4; ++r) d[r] = std::fmaf(uint_as_float((uint32_t)all[lane() / 4 * 4 + r]), b, d[r]);
    return d;
}
template <class B8, class V4> inline V4 mfma_bf16(B8 a, B8 b, V4 c) {
    // (D = A (16 x 32) . B (32 x 16) + C as in emu.h, four exchanges of 16-byte operands)
    uint64_t aw[2], bw[2], ar[2][64], br[2][64];
    std::memcpy(aw, &a, 16);
    std::memcpy(bw, &b, 16);
    for (int i = 0; i < 2; ++i) {
        std::memcpy(ar[i], share(aw[i]), sizeof ar[i]);
        std::memcpy(br[i], share(bw[i]), sizeof br[i]);
    }
    const int l = lane();
    V4 d = c;
    for (int r = 0; r < 4; ++r) {
        double s = 0.0;
        for (int k = 0; k < 32; ++k) {
            const int row = (k / 8) * 16 + 4 * (l / 16) + r, col = (k / 8) * 16 + l % 16, half = k % 8 / 4, sh = 16 * (k % 4);
            s += (double)bf16_to_float((uint16_t)(ar[half][row] >> sh)) * (double)bf16_to_float((uint16_t)(br[half][col] >> sh));
        }
        d[r] = (float)((double)c[r] + s);
    }
    return d;
}
// body() as every thread of every workgroup of a grid of x workgroups, one workgroup after the other on one set of threads
// (kernels without dynamic LDS)
template <class F> inline void launch_grid(F body, unsigned x, unsigned threads) {
    Block blk((int)threads, 0);
    std::vector<std::thread> ts;
    ts.reserve(threads);
    for (unsigned t = 0; t < threads; ++t)
        ts.emplace_back([&, t] {
            tl_thread = dim3{t, 0, 0}; tl_grid = dim3{x, 1, 1}; tl_blockdim = dim3{threads, 1, 1}; tl_blk = &blk;
            for (unsigned b = 0; b < x; ++b) {
                tl_block = dim3{b, 0, 0};
                body();
                blk.bar.wait();
            }
        });
    for (auto &th : ts) th.join();
}
inline int lo_int(double d) { uint64_t u; std::memcpy(&u, &d, 8); return (int)(uint32_t)u; }
inline int hi_int(double d) { uint64_t u; std::memcpy(&u, &d, 8); return (int)(uint32_t)(u >> 32); }
inline double of_ints(int hi, int lo) { const uint64_t u = (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo; double d; std::memcpy(&d, &u, 8); return d; }
}  // namespace emu

#undef __builtin_amdgcn_mfma_f32_16x16x32_bf16
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) emu::mfma_bf16((a), (b), (c))
#define __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, x, y, z) emu::mfma_16x16x4((a), (b), (c))
#define __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, c, x, y, z) emu::mfma_4x4x1((a), (b), (c))
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_rcp(x) (1.0 / (x))
#undef __shfl_xor
#define __shfl_xor(v, m, w) emu::from_lane((v), emu::lane() ^ (m))
#define __shfl(v, s, w) emu::from_lane((v), (s))
#define __shfl_up(v, d, w) emu::from_lane((v), emu::lane() >= (d) ? emu::lane() - (d) : emu::lane())
#define __ffsll(x) __builtin_ffsll((long long)(x))
#define __clzll(x) __builtin_clzll((unsigned long long)(x))
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_readlane(v, l) emu::from_lane((v), (l))
#define __ballot(p) emu::ballot(p)
#define __double2loint(d) emu::lo_int(d)
#define __double2hiint(d) emu::hi_int(d)
#define __hiloint2double(h, l) emu::of_ints((h), (l))
static inline void sincospif(float x, float *s, float *c) { *s = (float)std::sin(M_PI * (double)x); *c = (float)std::cos(M_PI * (double)x); }
static inline int atomicMin(int *p, int v) { int o = __atomic_load_n(p, __ATOMIC_SEQ_CST); while (v < o && !__atomic_compare_exchange_n(p, &o, v, false, __ATOMIC_SEQ_CST, __ATOMIC_SEQ_CST)) {} return o; }
static inline int atomicMax(int *p, int v) { int o = __atomic_load_n(p, __ATOMIC_SEQ_CST); while (v > o && !__atomic_compare_exchange_n(p, &o, v, false, __ATOMIC_SEQ_CST, __ATOMIC_SEQ_CST)) {} return o; }
static inline float wave_max(float v) { for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, WAVE)); return v; }
static inline bool better(float v, uint32_t i, float bv, uint32_t bi) { return v > bv || (v == bv && i < bi); }
static inline void wave_argbest(float &v, uint32_t &i) {
    for (int o = 32; o > 0; o >>= 1) {
        const float ov = __shfl_xor(v, o, WAVE);
        const uint32_t oi = __shfl_xor(i, o, WAVE);
        if (better(ov, oi, v, i)) { v = ov; i = oi; }
    }
}
// (the data-parallel moves of hipdec_common.h: running sum, a lane's value everywhere, the lane before's, the largest)
static inline double wave_scan_f64(double v) {
    const double mine = v;
    double r = 0.0;
    uint64_t all[64];
    std::memcpy(all, emu::share(mine), sizeof all);
    for (int i = 0; i <= emu::lane(); ++i) r += emu::of_bits<double>(all[i]);
    return r;
}
static inline double wave_read_f64(double v, int lane) { return emu::from_lane(v, lane); }
static inline double wave_before_f64(double v) { const double r = emu::from_lane(v, emu::lane() ? emu::lane() - 1 : 0); return emu::lane() ? r : 0.0; }
static inline float wave_max_dpp(float v) { return wave_max(v); }
