// batchattn_tc.cuh -- the shared prefix's part of kllm_batch_attention on the
// 5th-generation tensor cores, for 128 query rows at a time.
//
// All sequences' query heads of one kv head read the same keys, so a block
// takes 128 rows (sequence, head) against a range of the prefix:
//   scores  S[128][BN] = Q . K^T     two fp16 terms of q, keys as fp16
//   weights P = 2^(S - m)            back into S's columns, two fp16 terms
//   output  O[128][HD] = P . V       values as fp16, transposed
// tile by tile of BN positions.  Codes of 8 bits are exact in fp16; an fp32 key
// or value is brought to [2^13, 2^14) by a power of two of its own and taken as
// two fp16 terms (22 bits).  Keys' scales go to the scores, values' to the
// weights.  O does not stay in tensor memory: the tensor core cuts its sums off
// instead of rounding them, so each tile's O is added to fp32 registers, which
// is also where the running maximum's corrections and the unit of the tile's
// weights come in.
//
// Warps: two groups of four that take the tiles' softmax in turn (a row per
// thread) and each keep half of O's columns; four that bring keys and values
// from global memory to fp16 operands in shared memory, the next tile's loads
// in flight in registers (fp32: four for keys and four for values, the next
// tile's copies in flight in shared memory, since two terms to make of each
// number leave no time to wait); one that issues the products.  Warps whose
// rows lie behind the last leave their part of a tile alone.
// A tile's weights are relative to the tile's own maximum, so that the two
// groups need nothing of one another; the running maximum is applied where O
// is added up.  S/P and O have two buffers each, keys and values two (8 bits)
// or one; S of the next tile is issued before P.V of this one, so that the
// tensor cores work while the softmax does.  Every wait is bounded; one that
// gives up leaves NaN in the part's sums and ST_WAIT_TIMEOUT in the status word
// (where there is one).  The issuing warp sees all of its products end before
// the block gives its memory back, on that path too.
//
// Bound: of a tile of 128 positions of 8 bits (16.8 MFLOP with two terms) the
// products take some 1900 cycles (the tensor pipe is active 27 % of the
// kernel's time), the bytes 1600 of an SM's share of the memory's; a tile takes
// some 5700: of the two groups' 11400 each, 1400 are the maxima's, 4800 the
// weights', 1200 O's, the rest waiting for products that wait for weights.
// Taking the weights four rows a lane (a quarter of the scales' reads), their
// first terms without a conversion back, or their loads a step ahead measured
// the same; 16 softmax warps were a third slower (80 registers).  256 rows x
// 16384 positions of 8 kv heads of 128, e4m3, two tiles of rows: 75 us in all
// (17.2 GFLOP: 0.23 PFLOP/s, 0.46 as issued in two terms).  An fp32 tile's
// keys' conversion and the three products of its scores follow one another (one
// buffer of keys: two, with the queries in tensor memory, measured the same),
// and its weights wait for the values' scales.  24 rows x 4000 positions of 32
// kv heads of 128, fp32: 62 us (131 MB, 2.1 TB/s); 52 before keys and values
// had scales of their own.
#pragma once

#include "batchattn.cuh"
#include "umma.cuh"

namespace kllm {
namespace {

constexpr int BT_SOFT = 8;                                       // warps
constexpr int BT_ROWS = 128, BT_RING = 8;

template <int HD, int FMT>
struct BtGeom {
    static constexpr bool F32 = FMT == KLLM_KV_F32;
    static constexpr int FEED = F32 ? 8 : 4;                     // warps
    static constexpr int ST = F32 ? 1 : 2;                       // buffers of keys, of values
    static constexpr int THREADS = 32 * (BT_SOFT + FEED + 1);
    static constexpr int BN = F32 ? 64 : 128;                    // positions of a tile
    static constexpr int KT = F32 ? 2 : 1;                       // terms of a key or value
    static constexpr int KB = HD > 64 ? HD / 64 : 1;             // 64-dim blocks of Q and K
    static constexpr int VB = BN / 64;                           // 64-position blocks of V^T
    static constexpr int Q_TERM = KB * BT_ROWS * 128;
    static constexpr int K_TERM = KB * BN * 128, V_TERM = VB * HD * 128;
    static constexpr int K_STAGE = KT * K_TERM, V_STAGE = KT * V_TERM;
    static constexpr int Q_AT = 0, K_AT = 2 * Q_TERM, V_AT = K_AT + ST * K_STAGE;
    static constexpr int RAW_AT = V_AT + ST * V_STAGE, RAW = F32 ? BN * HD * 4 : 0;      // fp32 keys, values
    static constexpr int END = RAW_AT + 2 * RAW;
    static constexpr int S_COLS = BN, O_COLS = HD < 32 ? 32 : HD;
    static constexpr int COLS = 2 * (S_COLS + O_COLS) > 256 ? 512 : 2 * (S_COLS + O_COLS) > 128 ? 256 : 128;
};

struct BtShared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2];
    uint64_t sc_full[BT_RING], m_full[BT_RING], vs_full[BT_RING];
    uint32_t tmem;
    int dead;
    uint2 range[2][4];
    float vscale[BT_RING];               // what the tile's pv are in units of
    int spread[BT_RING];                 // whether its value scales lie far apart
    float rowfac[BT_ROWS];
    // a tile's maximum and sum of weights per row, and what O of the tile is in units of
    float mt[BT_RING][BT_ROWS], lt[BT_RING][BT_ROWS], ot[BT_RING][BT_ROWS];
    alignas(16) float ks[BT_RING][128], pv[BT_RING][128];
    alignas(16) float vu[64];            // fp32: the scales of the tile's values
};

template <int HD, int FMT>
constexpr size_t bt_smem() {
    return 1024 + BtGeom<HD, FMT>::END + sizeof(BtShared);
}

// Wait for phase `parity`; false when it, or another warp's wait, gave up (with
// a limit of 0, as soon as it would have to wait).
__device__ __forceinline__ bool bt_wait(uint64_t *bar, uint32_t parity, int *dead, unsigned long long limit) {
    if (limit ? mbar_try_wait(bar, parity) : mbar_test_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer();
    do {
        if (*(volatile int *)dead) return false;
        if (globaltimer() - t0 >= limit) {
            *(volatile int *)dead = 1;
            return false;
        }
    } while (!mbar_try_wait(bar, parity));
    return true;
}

// Two columns' scores times their keys' scales, and the maximum with them.
__device__ __forceinline__ float bt_max16(const uint32_t (&x)[16], const float4 *ks, float mx, bool cut,
                                          int n) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float4 k = ks[e];
        float2 a = __fmul2_rn(make_float2(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1])),
                              make_float2(k.x, k.y));
        float2 b = __fmul2_rn(make_float2(__uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3])),
                              make_float2(k.z, k.w));
        if (cut) {
            if (4 * e >= n) a.x = -INFINITY;
            if (4 * e + 1 >= n) a.y = -INFINITY;
            if (4 * e + 2 >= n) b.x = -INFINITY;
            if (4 * e + 3 >= n) b.y = -INFINITY;
        }
        mx = fmaxf(mx, fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y)));
    }
    return mx;
}

// The largest p times its value's scale of 16 columns, and `most`.
__device__ __forceinline__ float bt_most16(const uint32_t (&x)[16], const float *ks, const float *pv,
                                           float fac, float ref, float most, int n) {
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (e < n) most = fmaxf(most, ba_ex2(__fmaf_rn(__uint_as_float(x[e]) * ks[e], fac, -ref)) * fabsf(pv[e]));
    return most;
}

// 16 columns' weights p = 2^(score - ref) to the tensor memory: the fp16 terms
// of p times their values' scales (SPREAD: and times `up`), the first in
// columns at.., the second 8 columns behind.  Returns the weights' sum with
// them.
template <bool SPREAD>
__device__ __forceinline__ float2 bt_exp16(const uint32_t (&x)[16], const float4 *ks, const float4 *pv,
                                           float fac, float ref, float up, float2 sum, bool cut, int n,
                                           uint32_t at) {
    const float2 f = make_float2(fac, fac), r = make_float2(-ref, -ref), minus = make_float2(-1.f, -1.f);
#pragma unroll
    for (int q = 0; q < 2; q++) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float4 k = ks[2 * q + e], v = pv[2 * q + e];
            const uint32_t *s = x + 8 * q + 4 * e;
            const float2 a = __ffma2_rn(
                __fmul2_rn(make_float2(__uint_as_float(s[0]), __uint_as_float(s[1])), make_float2(k.x, k.y)), f, r);
            const float2 b = __ffma2_rn(
                __fmul2_rn(make_float2(__uint_as_float(s[2]), __uint_as_float(s[3])), make_float2(k.z, k.w)), f, r);
            float2 p = make_float2(ba_ex2(a.x), ba_ex2(a.y)), w = make_float2(ba_ex2(b.x), ba_ex2(b.y));
            if (cut) {
                if (8 * q + 4 * e >= n) p.x = 0.f;
                if (8 * q + 4 * e + 1 >= n) p.y = 0.f;
                if (8 * q + 4 * e + 2 >= n) w.x = 0.f;
                if (8 * q + 4 * e + 3 >= n) w.y = 0.f;
            }
            sum = __fadd2_rn(sum, __fadd2_rn(p, w));
            p = __fmul2_rn(p, make_float2(v.x, v.y));
            w = __fmul2_rn(w, make_float2(v.z, v.w));
            if (SPREAD) p.x *= up, p.y *= up, w.x *= up, w.y *= up;
            const __half2 ph = __float22half2_rn(p), wh = __float22half2_rn(w);
            const __half2 pl = __float22half2_rn(__ffma2_rn(__half22float2(ph), minus, p));
            const __half2 wl = __float22half2_rn(__ffma2_rn(__half22float2(wh), minus, w));
            hi[2 * e] = *reinterpret_cast<const uint32_t *>(&ph);
            hi[2 * e + 1] = *reinterpret_cast<const uint32_t *>(&wh);
            lo[2 * e] = *reinterpret_cast<const uint32_t *>(&pl);
            lo[2 * e + 1] = *reinterpret_cast<const uint32_t *>(&wl);
        }
        tmem_st4(at + 4 * q, hi);
        tmem_st4(at + 8 + 4 * q, lo);
    }
    return sum;
}

// The softmax of one row of a tile, its scores in columns at..: first their
// maximum (before fac); the first 16 columns are on their way to `first` then.
template <int BN, bool CUT>
__device__ __forceinline__ float bt_top(uint32_t at, const float4 *ks, int n, uint32_t (&first)[16]) {
    uint32_t s1[16];
    float mx = -INFINITY;
    tmem_ld16(at, first);
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
        tmem_wait_ld16(first);
        tmem_ld16(at + c + 16, s1);
        mx = bt_max16(first, ks + c / 4, mx, CUT, n - c);
        tmem_wait_ld16(s1);
        tmem_ld16(at + (c + 32) % BN, first);       // behind the last, the first again
        mx = bt_max16(s1, ks + c / 4 + 4, mx, CUT, n - c - 16);
    }
    return mx;
}

// Then the weights relative to the maximum, in log2 *m, and their sum; their two
// terms take the columns of their scores, 8 columns each for 16 positions.  pv
// is in units of *unit.  The weights times pv have to be fp16 numbers, whose
// terms end at 2^-24: with pv all near 2^13 that is far below the row's largest.
// Where they lie apart (SPREAD), a row whose large values have no weight would
// be left with nothing, so its own largest p pv is found first and brought to
// [2^13, 2^14) (a third pass; *unit changes with it).  With every tile's scales
// apart: 64 sequences x 16384 e4m3 99 us for 74, 24 x 4000 fp32 105 for 92.
template <int BN, bool CUT, bool SPREAD>
__device__ __forceinline__ void bt_weights(uint32_t at, const float4 *ks, const float4 *pv, float fac, int n,
                                           float mx, uint32_t (&s0)[16], float *m, float *sum, float *unit) {
    const float top = mx * fac, ref = top == -INFINITY ? 0.f : top;
    float up = 1.f;
    if constexpr (SPREAD) {
        float most = 0.f;
#pragma unroll 1
        for (int c = 0; c < BN; c += 16) {
            tmem_wait_ld16(s0);
            most = bt_most16(s0, reinterpret_cast<const float *>(ks) + c, reinterpret_cast<const float *>(pv) + c,
                             fac, ref, most, n - c);
            tmem_ld16(at + (c + 16) % BN, s0);
        }
        most = ba_pow2(most);
        up = 0x1p13f / most;
        *unit *= most * 0x1p-13f;
    }
    float2 t = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int c = 0; c < BN; c += 16) {
        tmem_wait_ld16(s0);
        t = bt_exp16<SPREAD>(s0, ks + c / 4, pv + c / 4, fac, ref, up, t, CUT, n - c, at + c);
        if (c + 16 < BN) tmem_ld16(at + c + 16, s0);
    }
    *m = top;
    *sum = t.x + t.y;
}

// 16 bytes at row r, 16-byte chunk c of a 128-byte-swizzled tile
__device__ __forceinline__ uint8_t *bt_at(uint8_t *tile, int r, int c) {
    return tile + r * 128 + ((c ^ (r & 7)) << 4);
}

template <int BAR>
__device__ __forceinline__ void bt_feed_bar() {
    asm volatile("bar.sync %0, 128;" ::"n"(BAR) : "memory");
}

// How a tile's value scales (four feeding warps, one or none, that is 0, a
// thread; all call it) go to pv: times `by`, in units of `unit`.  Near one
// another, the largest to [2^13, 2^14); with one 2^10 times another, as they are.
struct BtScales {
    float by, unit;
    bool spread;
};
template <int BAR>
__device__ __forceinline__ BtScales bt_feed_scales(float s, uint2 *range) {
    const uint32_t b = __float_as_uint(s) & 0x7fffffffu;
    // (zeros, one below which is the largest number, do not count for the smallest)
    uint2 r = make_uint2(__reduce_max_sync(0xffffffffu, b), __reduce_min_sync(0xffffffffu, b - 1u));
    if ((threadIdx.x & 31) == 0) range[threadIdx.x >> 5 & 3] = r;
    bt_feed_bar<BAR>();
#pragma unroll
    for (int i = 0; i < 4; i++) r.x = max(r.x, range[i].x), r.y = min(r.y, range[i].y);
    BtScales o = {1.f, 1.f, (int)(r.x >> 23) - (int)((r.y + 1u) >> 23) > 10};
    if (!o.spread) {
        const float most = ba_pow2(__uint_as_float(r.x));
        o.by = 0x1p13f / most;
        o.unit = most * 0x1p-13f;
    }
    return o;
}

// Whether all of a role's THREADS threads say yes (so that they leave their
// loop together); the feeding warps' barriers are 2 and 5, the softmax warps' 3.
template <int THREADS, int BAR = 3>
__device__ __forceinline__ bool bt_all(bool yes) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.and.pred p, %3, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)yes), "n"(THREADS), "n"(BAR)
        : "memory");
    return all != 0;
}

// What a feeding thread (of 128) holds of a tile of 8-bit codes: K, 16 codes
// (16 bytes) of every RPP-th row; V, DV dims of 8 positions in a row.
template <int HD>
struct BtFeed8 {
    static constexpr int LPR = HD / 16, RPP = 128 / LPR, NK = 128 / RPP, DV = HD / 8;
    uint32_t k[NK][4], v[8][DV / 4];
    float ks, vs;

    __device__ __forceinline__ void load_k(const uint8_t *kb, const float *ksc, const float *vsc, int j0,
                                           int n) {
        const int t = threadIdx.x - 32 * BT_SOFT;
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const int r = p * RPP + t / LPR;
            ba_fetch(k[p], kb + (long long)(j0 + r) * HD + 16 * (t % LPR), r < n);
        }
        uint32_t x[1], y[1];
        ba_fetch(x, ksc + j0 + t, t < n);
        ba_fetch(y, vsc + j0 + t, t < n);
        ks = __uint_as_float(x[0]), vs = __uint_as_float(y[0]);
    }
    __device__ __forceinline__ void load_v(const uint8_t *vb, int j0, int n) {
        const int t = threadIdx.x - 32 * BT_SOFT;
        const int pg = (t & 7) | ((t >> 5) & 1) << 3, dg = ((t >> 3) & 3) | (t >> 6) << 2;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = pg * 8 + j;
            ba_fetch(v[j], vb + (long long)(j0 + r) * HD + dg * DV, r < n);
        }
    }
    template <int FMT>
    __device__ __forceinline__ void store_k(uint8_t *tile) const {
        const int t = threadIdx.x - 32 * BT_SOFT;
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const int r = p * RPP + t / LPR, i = t % LPR, blk = i >> 2, c = 2 * (i & 3);
            uint32_t u[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t x = FMT == KLLM_KV_I8 ? k[p][e] ^ 0x80808080u : k[p][e];
                u[2 * e] = ba_codes<FMT, 0>(x);
                u[2 * e + 1] = ba_codes<FMT, 1>(x);
            }
            // the lanes of the second block of dims store their odd chunk first: a row's eight
            // lanes then touch eight different banks' worth
            uint8_t *b = tile + blk * (128 * 128);
            const bool s = blk & 1;
            *reinterpret_cast<uint4 *>(bt_at(b, r, c + s)) =
                make_uint4(s ? u[4] : u[0], s ? u[5] : u[1], s ? u[6] : u[2], s ? u[7] : u[3]);
            *reinterpret_cast<uint4 *>(bt_at(b, r, c + 1 - s)) =
                make_uint4(s ? u[0] : u[4], s ? u[1] : u[5], s ? u[2] : u[6], s ? u[3] : u[7]);
        }
    }
    template <int FMT>
    __device__ __forceinline__ void store_v(uint8_t *tile) const {
        const int t = threadIdx.x - 32 * BT_SOFT;
        const int pg = (t & 7) | ((t >> 5) & 1) << 3, dg = ((t >> 3) & 3) | (t >> 6) << 2;
        uint8_t *b = tile + (pg >> 3) * (HD * 128);
#pragma unroll
        for (int q = 0; q < DV / 4; q++) {
            uint32_t h[4][4];      // [dim][positions 2 i, 2 i + 1]
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t x = v[2 * i][q], y = v[2 * i + 1][q];
                if (FMT == KLLM_KV_I8) x ^= 0x80808080u, y ^= 0x80808080u;
                const uint32_t a = ba_prmt(x, y, 0x5140), c = ba_prmt(x, y, 0x7362);
                h[0][i] = ba_codes<FMT, 0>(a);
                h[1][i] = ba_codes<FMT, 1>(a);
                h[2][i] = ba_codes<FMT, 0>(c);
                h[3][i] = ba_codes<FMT, 1>(c);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                *reinterpret_cast<uint4 *>(bt_at(b, dg * DV + 4 * q + e, pg & 7)) =
                    make_uint4(h[e][0], h[e][1], h[e][2], h[e][3]);
        }
    }
};

// The same of an fp32 tile of 64 positions, which comes to shared memory as it
// is, copied by the threads that will read it (no barrier, few registers):
// K, 16-byte pieces in a row; V, the pieces of four dims of 8 positions, moved
// within a row by the position so that eight lanes' reads meet eight banks.
template <int HD>
struct BtFeed32 {
    static constexpr int PIECES = HD / 4, NK = 64 * PIECES / 128, ITEMS = 8 * PIECES, NV = (ITEMS + 127) / 128;
    uint8_t *raw_k, *raw_v;

    static __device__ __forceinline__ int thread() { return threadIdx.x & 127; }
    static __device__ __forceinline__ float most(float4 x) {
        return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    }
    __device__ __forceinline__ float4 *v_at(int row, int dg) const {
        return reinterpret_cast<float4 *>(raw_v) + row * PIECES + (dg ^ ((row >> 3) & 7));
    }
    __device__ __forceinline__ void load_k(const uint8_t *kb, int j0, int n) {
#pragma unroll 4
        for (int e = 0; e < NK; e++) {
            const int q = e * 128 + thread(), bytes = q / PIECES < n ? 16 : 0;
            ba_cp16(smem_u32(raw_k + 16 * q), kb + (bytes ? (long long)j0 * HD * 4 + 16 * q : 0), bytes);
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t *vb, int j0, int n) {
#pragma unroll
        for (int e = 0; e < NV; e++) {
            const int t = e * 128 + thread(), pg = t & 7, dg = t >> 3;
            if (t < ITEMS)
#pragma unroll 4
                for (int j = 0; j < 8; j++) {
                    const int r = pg * 8 + j, bytes = r < n ? 16 : 0;
                    ba_cp16(smem_u32(v_at(r, dg)), vb + (bytes ? ((long long)(j0 + r) * HD + 4 * dg) * 4 : 0), bytes);
                }
        }
    }
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
    // the 64 rows from j0 on towards L2
    static __device__ __forceinline__ void prefetch(const uint8_t *b, int j0, int n) {
        for (int o = thread() * 128; o < n * HD * 4; o += 128 * 128) prefetch_l2_line(b + (long long)j0 * HD * 4 + o);
    }
    // The power of two that brings a key to [2^13, 2^14) is its own; the inverse takes part in the scores
    // as an 8-bit key's scale does.  A key's pieces are in PIECES lanes of a warp, of which lane e works
    // it out for the warp's e-th keys and returns it.
    __device__ __forceinline__ float scale_k(float *scale) const {
        float mine = 0.f;
#pragma unroll 8
        for (int e = 0; e < NK; e++) {
            float m = most(reinterpret_cast<const float4 *>(raw_k)[e * 128 + thread()]);
            if constexpr (PIECES == 32) m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
            else
#pragma unroll
                for (int o = PIECES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (thread() % PIECES == e) mine = m;
        }
        mine = ba_pow2(mine);
        const int e = thread() % PIECES;
        if (e < NK) scale[e * (128 / PIECES) + thread() / PIECES] = mine * 0x1p-13f;
        return 0x1p13f / mine;
    }
    // The same of the values: their scales to `scale` (0 for a row of zeros, NaN for one that is not
    // finite); returns this thread's, or 0.  (All four warps' copies are there: this reads whole rows.)
    __device__ __forceinline__ float scale_v(float *scale) const {
        float mine = 0.f;
#pragma unroll 8
        for (int e = 0; e < NK; e++) {
            const float4 x = reinterpret_cast<const float4 *>(raw_v)[e * 128 + thread()];
            float m = max_nan(max_nan(fabsf(x.x), fabsf(x.y)), max_nan(fabsf(x.z), fabsf(x.w)));
            if constexpr (PIECES == 32) m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
            else
#pragma unroll
                for (int o = PIECES / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (thread() % PIECES == e) mine = m;
        }
        const int e = thread() % PIECES;
        if (e >= NK) return 0.f;
        mine = mine < INFINITY ? mine > 0.f ? ba_pow2(mine) * 0x1p-13f : 0.f : __uint_as_float(0x7fffffffu);
        scale[e * (128 / PIECES) + thread() / PIECES] = mine;
        return mine;
    }
    static __device__ __forceinline__ float max_nan(float a, float b) {
        float c;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
        return c;
    }
    __device__ __forceinline__ void store_k(uint8_t *tile, int term, float mine) const {
#pragma unroll 8
        for (int e = 0; e < NK; e++) {
            const int q = e * 128 + thread(), r = q / PIECES, i = q % PIECES, blk = i >> 4;
            const float4 x = reinterpret_cast<const float4 *>(raw_k)[q];
            const float f = __shfl_sync(0xffffffffu, mine, e, PIECES);
            uint2 h, l;
            ba_split(x.x * f, x.y * f, &h.x, &l.x);
            ba_split(x.z * f, x.w * f, &h.y, &l.y);
            uint8_t *a = bt_at(tile + blk * (64 * 128), r, (i & 15) >> 1) + 8 * (i & 1);
            *reinterpret_cast<uint2 *>(a) = h;
            *reinterpret_cast<uint2 *>(a + term) = l;
        }
    }
    __device__ __forceinline__ void store_v(uint8_t *tile, int term, const float *scale) const {
#pragma unroll 1
        for (int e = 0; e < NV; e++) {
            const int t = e * 128 + thread(), pg = t & 7, dg = t >> 3;
            if (t >= ITEMS) break;
            uint32_t h[4][4], l[4][4];      // [dim][positions 2 i, 2 i + 1]
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 x = *v_at(pg * 8 + 2 * i, dg), y = *v_at(pg * 8 + 2 * i + 1, dg);
                // (the inverse of a power of two; of 0 it is 2^127, of NaN some number: p is NaN then)
                const float2 s = *reinterpret_cast<const float2 *>(scale + pg * 8 + 2 * i);
                const float f = __uint_as_float(0x7f000000u - __float_as_uint(s.x));
                const float g = __uint_as_float(0x7f000000u - __float_as_uint(s.y));
                ba_split(x.x * f, y.x * g, &h[0][i], &l[0][i]);
                ba_split(x.y * f, y.y * g, &h[1][i], &l[1][i]);
                ba_split(x.z * f, y.z * g, &h[2][i], &l[2][i]);
                ba_split(x.w * f, y.w * g, &h[3][i], &l[3][i]);
            }
#pragma unroll
            for (int d = 0; d < 4; d++) {
                uint8_t *a = bt_at(tile, 4 * dg + d, pg);
                *reinterpret_cast<uint4 *>(a) = make_uint4(h[d][0], h[d][1], h[d][2], h[d][3]);
                *reinterpret_cast<uint4 *>(a + term) = make_uint4(l[d][0], l[d][1], l[d][2], l[d][3]);
            }
        }
    }
};

// grid: (kv head, tile of 128 rows, part) of the prefix
template <int HD, int FMT>
__global__ void __launch_bounds__((BtGeom<HD, FMT>::THREADS), 1)
k_ba_prefix(const BaArgs a) {
    using G = BtGeom<HD, FMT>;
    constexpr bool F32 = G::F32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    BtShared &sh = *reinterpret_cast<BtShared *>(smem + G::END);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    int b = blockIdx.x;
    const int part = b % a.pre.parts;
    b /= a.pre.parts;
    const int tile = b % a.tiles_pre, kvh = b / a.tiles_pre;
    const int p0 = part * a.pre.chunk, p1 = p0 + min(a.prefix_len - p0, a.pre.chunk);
    const int nt = (p1 - p0 + G::BN - 1) / G::BN;
    const int n_rows = a.n_seq * a.groups;

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.k_full[i], 128);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], 128);
            mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 128);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.o_empty[i], 32 * BT_SOFT);
        }
        for (int i = 0; i < BT_RING; i++) {
            mbar_init(&sh.sc_full[i], 128);
            mbar_init(&sh.m_full[i], 128);
            mbar_init(&sh.vs_full[i], 128);
        }
        sh.dead = 0;
        mbar_fence_init();
    }
    if (warp == BT_SOFT + G::FEED) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sh.tmem)), "r"(G::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // A softmax warp's 16 rows of the tile, row k of them by lane k: (k / RPW, k % RPW) is its place
    // in a loop of 16 / RPW turns, HD / 4 lanes a row (small loops: code that runs once costs its
    // own fetch).
    constexpr int LPR = HD / 4, RPW = 32 / LPR;
    const int my_row = ((lane % 16 / RPW) * BT_SOFT + warp) * RPW + lane % RPW, sub = lane / LPR, dim = 4 * (lane % LPR);
    const int R = tile * BT_ROWS + my_row, R_seq = R / a.groups, R_head = kvh * a.groups + R % a.groups;
    const uint32_t have = __ballot_sync(0xffffffffu, R < n_rows && lane < 16);
    // Rows of the tile, to the next 32: warps without any leave S, P and O as they are (a row of them
    // needs nothing of another).
    const int there = min(BT_ROWS, (n_rows - tile * BT_ROWS + 31) / 32 * 32), turns = there / (8 * RPW);
    // The queries, raw into the place of keys and values, then times scale * log2(e), brought to
    // [2^13, 2^14) by a power of two, in two fp16 terms.
    if (warp < BT_SOFT) {
        const long long q_at = (long long)R_seq * a.q_stride + (long long)R_head * HD;
        float *raw = reinterpret_cast<float *>(smem + G::K_AT);
#pragma unroll 4
        for (int e = 0; e < turns; e++) {
            const int k = e * RPW + sub, r = (e * BT_SOFT + warp) * RPW + sub;
            const long long at = __shfl_sync(0xffffffffu, q_at, k);
            const uint32_t d = smem_u32(raw + r * HD + dim);
            const int bytes = have >> k & 1;
            const float *q = a.q + (bytes ? at + dim : 0);
            if (a.q_vec) {
                ba_cp16(d, q, 16 * bytes);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) ba_cp4(d + 4 * i, q + (bytes ? i : 0), 4 * bytes);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // (each lane reads what it copied)
#pragma unroll 2
        for (int e = 0; e < turns; e++) {
            const int r = (e * BT_SOFT + warp) * RPW + sub, i = dim / 4;
            const float4 x = *reinterpret_cast<const float4 *>(raw + r * HD + dim);
            const float4 y = make_float4(x.x * a.qk, x.y * a.qk, x.z * a.qk, x.w * a.qk);
            float m = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float up = ba_pow2(m), f = 0x1p13f / up;
            if (i == 0) sh.rowfac[r] = up * 0x1p-13f;
            uint2 h, l;
            ba_split(y.x * f, y.y * f, &h.x, &l.x);
            ba_split(y.z * f, y.w * f, &h.y, &l.y);
            uint8_t *t = bt_at(smem + G::Q_AT + (i >> 4) * (BT_ROWS * 128), r, (i & 15) >> 1) + 8 * (i & 1);
            *reinterpret_cast<uint2 *>(t) = h;
            *reinterpret_cast<uint2 *>(t + G::Q_TERM) = l;
        }
        fence_async_shared();
    } else if (warp < BT_SOFT + G::FEED) {
        // the first tile's rows towards L2 meanwhile
        const long long at = (long long)kvh * a.pre.max_pos + p0;
        constexpr int ROW = HD * (F32 ? 4 : 1);
        const int bytes = min(G::BN, p1 - p0) * ROW;
        for (int o = (tid - 32 * BT_SOFT) * 128; o < bytes; o += 32 * G::FEED * 128) {
            prefetch_l2_line(static_cast<const uint8_t *>(a.pre.k) + at * ROW + o);
            prefetch_l2_line(static_cast<const uint8_t *>(a.pre.v) + at * ROW + o);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    auto s_cols = [&](int t) { return tmem + (uint32_t)((t & 1) * G::S_COLS); };
    auto o_cols = [&](int t) { return tmem + (uint32_t)(2 * G::S_COLS + (t & 1) * G::O_COLS); };
    const long long row0 = (long long)kvh * a.pre.max_pos;
    const int parts = a.pre.parts + a.own.parts;
    // where row r of this tile leaves its part
    auto part_of = [&](int r) {
        const int R = tile * BT_ROWS + r;
        return ((long long)(R / a.groups) * a.nh + kvh * a.groups + R % a.groups) * parts + part;
    };

    if (warp < BT_SOFT) {
        // --------------------------------------------- softmax and output --
        const int group = warp >> 2, r = 32 * (warp & 3) + lane;
        constexpr int NC = HD / 2;                 // columns of O of this thread
        const int c0 = group * NC;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const bool rows_here = 32 * (warp & 3) < there;
        const float fac = sh.rowfac[r];
        float m_run = -INFINITY, l_run = 0.f, acc[NC];
#pragma unroll
        for (int e = 0; e < NC; e++) acc[e] = 0.f;
        bool ok = true;
        // the weights of tile t
        auto soft = [&](int t) {
            const int ring = t & (BT_RING - 1), n = min(G::BN, p1 - p0 - t * G::BN);
            ok = __all_sync(0xffffffffu, ok && bt_wait(&sh.sc_full[ring], (t / BT_RING) & 1, &sh.dead, a.wait_ns) &&
                                             (!F32 || bt_wait(&sh.vs_full[ring], (t / BT_RING) & 1, &sh.dead, a.wait_ns)) &&
                                             bt_wait(&sh.s_full[t & 1], (t / 2) & 1, &sh.dead, a.wait_ns));
            if (!ok) return;
            tc_fence_after();
            const float4 *ks = reinterpret_cast<const float4 *>(sh.ks[ring]);
            const float4 *pv = reinterpret_cast<const float4 *>(sh.pv[ring]);
            const uint32_t at = s_cols(t) + lanes;
            uint32_t first[16];
            float mx = 0.f;
            if (rows_here) mx = n == G::BN ? bt_top<G::BN, false>(at, ks, n, first) : bt_top<G::BN, true>(at, ks, n, first);
            if (rows_here) {
                float m, sum, unit = sh.vscale[ring];
                if (sh.spread[ring]) bt_weights<G::BN, true, true>(at, ks, pv, fac, n, mx, first, &m, &sum, &unit);
                else if (n == G::BN) bt_weights<G::BN, false, false>(at, ks, pv, fac, n, mx, first, &m, &sum, &unit);
                else bt_weights<G::BN, true, false>(at, ks, pv, fac, n, mx, first, &m, &sum, &unit);
                sh.mt[ring][r] = m;
                sh.lt[ring][r] = sum;
                sh.ot[ring][r] = unit;
                tmem_wait_st();
            }
            tc_fence_before();
            mbar_arrive(&sh.p_full[t & 1]);
            mbar_arrive(&sh.m_full[ring]);
        };
        // tile t's output to the registers
        auto add = [&](int t) {
            const int ring = t & (BT_RING - 1);
            ok = __all_sync(0xffffffffu, ok && bt_wait(&sh.m_full[ring], (t / BT_RING) & 1, &sh.dead, a.wait_ns) &&
                                             bt_wait(&sh.o_full[t & 1], (t / 2) & 1, &sh.dead, a.wait_ns));
            if (!ok) return;
            tc_fence_after();
            if (rows_here) {
                const float m = sh.mt[ring][r], m_new = fmaxf(m_run, m), ref = m_new == -INFINITY ? 0.f : m_new;
                const float corr = ba_ex2(m_run - ref), w = ba_ex2(m - ref), f = w * sh.ot[ring][r];
                l_run = l_run * corr + sh.lt[ring][r] * w;
                m_run = m_new;
#pragma unroll
                for (int c = 0; c < NC / 16; c++) {
                    uint32_t v[16];
                    tmem_ld16(o_cols(t) + lanes + c0 + 16 * c, v);
                    tmem_wait_ld16(v);
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        acc[16 * c + e] = fmaf(__uint_as_float(v[e]), f, acc[16 * c + e] * corr);
                }
            }
            tc_fence_before();
            mbar_arrive(&sh.o_empty[t & 1]);
        };
        for (int t = group; t < nt + 2; t += 2) {
            if (t < nt && ok) soft(t);
            if (t >= 2 && ok) add(t - 2);
            if (t >= 1 && t - 1 < nt && ok) add(t - 1);
        }
        // The rows' sums to memory, by way of the operands' place (all products are done), so that a
        // warp writes whole rows.
        constexpr int PITCH = HD + 4;
        static_assert(BT_ROWS * PITCH * 4 <= G::V_AT, "rows of fp32 in the place of Q and K");
        float *rows = reinterpret_cast<float *>(smem);
        ok = bt_all<32 * BT_SOFT>(ok);
        if (!ok && a.status && tid == 0) atomicOr(a.status, ST_WAIT_TIMEOUT);
#pragma unroll
        for (int e = 0; e < NC / 4; e++)
            if (rows_here) *reinterpret_cast<float4 *>(rows + r * PITCH + c0 + 4 * e) =
                make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
        bt_all<32 * BT_SOFT>(true);
        const float nan = __uint_as_float(0x7fffffffu);
        const long long part_at = ((long long)R_seq * a.nh + R_head) * parts + part;
#pragma unroll 4
        for (int e = 0; e < turns; e++) {
            const int k = e * RPW + sub, q = (e * BT_SOFT + warp) * RPW + sub;
            const long long at = __shfl_sync(0xffffffffu, part_at, k);
            const float4 v = *reinterpret_cast<const float4 *>(rows + q * PITCH + dim);
            if (have >> k & 1)
                *reinterpret_cast<float4 *>(a.part_o + at * HD + dim) = ok ? v : make_float4(nan, nan, nan, nan);
        }
        if (group == 0 && tile * BT_ROWS + r < n_rows)
            *reinterpret_cast<float2 *>(a.part_ml + 2 * part_of(r)) =
                ok ? make_float2(m_run, l_run) : make_float2(nan, nan);
    } else if (warp < BT_SOFT + G::FEED) {
        // --------------------------------------------------------- feeding --
        // Before the scales of a tile are written: the scores of tile t - ST are done.  They were issued
        // behind the output of tile t - 4 or a later one, which waited for all to be done with that of
        // tile t - 6; so the ring's slot, tile t - 8's, is free.  (fp32 keys' are written before that wait:
        // then the scores of tile t - 2 are done, issued behind the output of tile t - 4, as above.)
        const int f = tid & 127;
        const uint8_t *kb = static_cast<const uint8_t *>(a.pre.k) + row0 * HD * (F32 ? 4 : 1);
        const uint8_t *vb = static_cast<const uint8_t *>(a.pre.v) + row0 * HD * (F32 ? 4 : 1);
        bool ok = true;
        auto left = [&](int t) { return min(G::BN, p1 - p0 - t * G::BN); };
        if constexpr (F32) {
            // four warps bring keys, four values
            BtFeed32<HD> x = {smem + G::RAW_AT, smem + G::RAW_AT + G::RAW};
            uint8_t *kt = smem + G::K_AT, *vt = smem + G::V_AT;
            if (warp < BT_SOFT + 4) {
                x.load_k(kb, p0, left(0));
                for (int t = 0; t < nt; t++) {
                    const int ring = t & (BT_RING - 1);
                    if (t + 1 < nt) x.prefetch(kb, p0 + (t + 1) * G::BN, left(t + 1));
                    x.wait();
                    const float up = x.scale_k(sh.ks[ring]);      // (a free slot: above)
                    if (t) ok = bt_wait(&sh.k_empty[0], (t & 1) ^ 1, &sh.dead, a.wait_ns);
                    if (!bt_all<128, 2>(ok)) break;
                    x.store_k(kt, G::K_TERM, up);
                    fence_async_shared();
                    mbar_arrive(&sh.k_full[0]);
                    mbar_arrive(&sh.sc_full[ring]);
                    if (t + 1 < nt) x.load_k(kb, p0 + (t + 1) * G::BN, left(t + 1));
                }
            } else {
                x.load_v(vb, p0, left(0));
                for (int t = 0; t < nt; t++) {
                    const int ring = t & (BT_RING - 1);
                    if (t + 1 < nt) x.prefetch(vb, p0 + (t + 1) * G::BN, left(t + 1));
                    x.wait();
                    bt_feed_bar<4>();
                    // (the ring's slot is free: the output of tile t - 2 is done, issued when all were done
                    // with that of tile t - 4)
                    const BtScales vs = bt_feed_scales<4>(x.scale_v(sh.vu), sh.range[1]);
                    if (f < G::BN) sh.pv[ring][f] = sh.vu[f] * vs.by;
                    if (f == 0) sh.vscale[ring] = vs.unit, sh.spread[ring] = vs.spread;
                    mbar_arrive(&sh.vs_full[ring]);
                    if (t) ok = bt_wait(&sh.v_empty[0], (t & 1) ^ 1, &sh.dead, a.wait_ns);
                    if (!bt_all<128, 5>(ok)) break;
                    x.store_v(vt, G::V_TERM, sh.vu);
                    fence_async_shared();
                    mbar_arrive(&sh.v_full[0]);
                    if (t + 1 < nt) x.load_v(vb, p0 + (t + 1) * G::BN, left(t + 1));
                }
            }
            x.wait();      // (nothing of it comes after the block)
        } else {
            const float *ksc = a.pre.ks + row0, *vsc = a.pre.vs + row0;
            BtFeed8<HD> x;
            x.load_k(kb, ksc, vsc, p0, left(0));
            x.load_v(vb, p0, left(0));
            for (int t = 0; t < nt; t++) {
                const int st = t & 1, ring = t & (BT_RING - 1);
                const uint32_t free_parity = ((t / 2) & 1) ^ 1;
                if (t >= 2) ok = ok && bt_wait(&sh.k_empty[st], free_parity, &sh.dead, a.wait_ns);
                if (!bt_all<128, 2>(ok)) break;
                x.template store_k<FMT>(smem + G::K_AT + st * G::K_STAGE);
                const BtScales vs = bt_feed_scales<1>(x.vs, sh.range[st]);
                sh.ks[ring][f] = x.ks, sh.pv[ring][f] = x.vs * vs.by;
                if (f == 0) sh.vscale[ring] = vs.unit, sh.spread[ring] = vs.spread;
                fence_async_shared();
                mbar_arrive(&sh.k_full[st]);
                mbar_arrive(&sh.sc_full[ring]);
                if (t + 1 < nt) x.load_k(kb, ksc, vsc, p0 + (t + 1) * G::BN, left(t + 1));
                if (t >= 2) ok = bt_wait(&sh.v_empty[st], free_parity, &sh.dead, a.wait_ns);
                if (ok) {
                    x.template store_v<FMT>(smem + G::V_AT + st * G::V_STAGE);
                    fence_async_shared();
                    mbar_arrive(&sh.v_full[st]);
                }
                if (t + 1 < nt) x.load_v(vb, p0 + (t + 1) * G::BN, left(t + 1));
            }
        }
    } else if (lane == 0) {
        // -------------------------------------------------------- products --
        constexpr uint32_t s_idesc = umma_idesc_f16(128, G::BN), o_idesc = umma_idesc_f16(128, HD);
        const uint32_t qa = smem_u32(smem + G::Q_AT);
        auto scores = [&](int t) {
            const uint32_t kt = smem_u32(smem + G::K_AT + t % G::ST * G::K_STAGE), d = s_cols(t);
            uint32_t acc = 0;
            // small terms first
#pragma unroll
            for (int c = (F32 ? 2 : 1); c >= 0; c--) {
                const uint32_t q = qa + (c == 1 ? G::Q_TERM : 0), k = kt + (c == 2 ? G::K_TERM : 0);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {
                    umma_f16_ss(d, umma_desc_sw128(q + (ks >> 2) * (BT_ROWS * 128) + 32 * (ks & 3)),
                                umma_desc_sw128(k + (ks >> 2) * (G::BN * 128) + 32 * (ks & 3)), s_idesc, acc);
                    acc = 1;
                }
            }
            umma_commit(&sh.s_full[t & 1]);
            umma_commit(&sh.k_empty[t % G::ST]);
        };
        auto output = [&](int t) {
            const uint32_t vt = smem_u32(smem + G::V_AT + t % G::ST * G::V_STAGE), d = o_cols(t), p = s_cols(t);
            uint32_t acc = 0;
#pragma unroll
            for (int c = (F32 ? 2 : 1); c >= 0; c--) {
                const uint32_t v = vt + (c == 2 ? G::V_TERM : 0);
#pragma unroll
                for (int ks = 0; ks < G::BN / 16; ks++) {
                    umma_f16_ts(d, p + 16 * ks + (c == 1 ? 8 : 0),
                                umma_desc_sw128(v + (ks >> 2) * (HD * 128) + 32 * (ks & 3)), o_idesc, acc);
                    acc = 1;
                }
            }
            umma_commit(&sh.o_full[t & 1]);
            umma_commit(&sh.v_empty[t % G::ST]);
        };
        // S of the next tile ahead of O of this one: the tensor cores work while the softmax does.
        bool ok = true;
        int n_s = 0, n_o = 0;      // tiles whose scores, outputs were issued
        for (int t = 0; t <= nt && ok; t++) {
            if (t < nt) {
                ok = bt_wait(&sh.k_full[t % G::ST], (t / G::ST) & 1, &sh.dead, a.wait_ns);
                tc_fence_after();
                if (ok) scores(t), n_s++;
            }
            const int u = t - 1;
            if (u < 0 || !ok) continue;
            ok = bt_wait(&sh.p_full[u & 1], (u / 2) & 1, &sh.dead, a.wait_ns) &&
                 bt_wait(&sh.v_full[u % G::ST], (u / G::ST) & 1, &sh.dead, a.wait_ns) &&
                 (u < 2 || bt_wait(&sh.o_empty[u & 1], ((u / 2) & 1) ^ 1, &sh.dead, a.wait_ns));
            tc_fence_after();
            if (ok) output(u), n_o++;
        }
        // Products and their arrivals are over before the memory that they write is given back (they wait
        // for nothing themselves, so this ends, given up or not).
        auto drain = [](uint64_t *bar, int buffers, int n) {
            for (int b = 0; b < buffers; b++)
                if (n > b) mbar_wait(&bar[b], (n - b - 1) / buffers & 1, nullptr);
        };
        drain(sh.s_full, 2, n_s);
        drain(sh.k_empty, G::ST, n_s);
        drain(sh.o_full, 2, n_o);
        drain(sh.v_empty, G::ST, n_o);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == BT_SOFT + G::FEED) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::COLS)
                     : "memory");
    }
}

}  // namespace
}  // namespace kllm
