// batchattn_tc.cuh -- the shared prefix's part of kllm_batch_attention on the
// 5th-generation tensor cores, for 128 query rows at a time.
//
// All sequences' query heads of one kv head read the same keys, so a block
// takes 128 rows (sequence, head) against a range of the prefix:
//   scores  S[128][BN] = Q . K^T     two fp16 terms of q, keys as fp16
//   weights P = 2^(S - m)            back into S's columns, two fp16 terms
//   output  O[128][HD] = P . V       values as fp16, transposed
// tile by tile of BN positions.  Codes of 8 bits are exact in fp16; an fp32
// tile is brought to [2^13, 2^14) by a power of two and taken as two fp16
// terms (22 bits).  O does not stay in tensor memory: the tensor core cuts
// its sums off instead of rounding them, so each tile's O is added to fp32
// registers, which is also where the running maximum's corrections and the
// tile's value scale come in.
//
// 21 warps: 4 softmax (a row per thread), 8 that keep O (a row and half the
// columns per thread), 8 that bring keys and values from global memory to
// fp16 operands in shared memory (next tile's loads in flight in registers),
// one that issues the products.  Keys, values, S/P and O have two buffers
// each; S of the next tile is issued before P.V of this one, so that the
// tensor cores work while the softmax does.  Every wait is bounded; one that
// gives up leaves NaN in the part's sums.
//
// Bound: products.  With two terms a tile of 128 positions of 8 bits takes
// 16.8 MFLOP, 1.5 us at the tensor cores' rate, where its bytes take 0.8 us
// of an SM's share of the memory's; fp32 tiles take three products (25
// MFLOP, 2.3 us per 128 positions) against 2.9 us of bytes.
#pragma once

#include "batchattn.cuh"
#include "umma.cuh"

namespace kllm {
namespace {

constexpr int BT_SOFT = 4, BT_OUT = 8, BT_FEED = 8;              // warps
constexpr int BT_THREADS = 32 * (BT_SOFT + BT_OUT + BT_FEED + 1);
constexpr int BT_ROWS = 128, BT_RING = 8;

template <int HD, int FMT>
struct BtGeom {
    static constexpr bool F32 = FMT == KLLM_KV_F32;
    static constexpr int BN = F32 ? 64 : 128;                    // positions of a tile
    static constexpr int KT = F32 ? 2 : 1;                       // terms of a key or value
    static constexpr int KB = HD > 64 ? HD / 64 : 1;             // 64-dim blocks of Q and K
    static constexpr int VB = BN / 64;                           // 64-position blocks of V^T
    static constexpr int Q_TERM = KB * BT_ROWS * 128;
    static constexpr int K_TERM = KB * BN * 128, V_TERM = VB * HD * 128;
    static constexpr int K_STAGE = KT * K_TERM, V_STAGE = KT * V_TERM;
    static constexpr int Q_AT = 0, K_AT = 2 * Q_TERM, V_AT = K_AT + 2 * K_STAGE;
    static constexpr int END = V_AT + 2 * V_STAGE;
    static constexpr int S_COLS = BN, O_COLS = HD < 32 ? 32 : HD;
    static constexpr int COLS = 2 * (S_COLS + O_COLS) > 256 ? 512 : 2 * (S_COLS + O_COLS) > 128 ? 256 : 128;
};

struct BtShared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2];
    uint64_t sc_full[BT_RING];
    uint32_t tmem;
    int dead;
    float wmax[2][BT_FEED];
    float vscale[BT_RING];               // what O of the tile is in units of
    float rowfac[BT_ROWS];
    float corr[BT_RING][BT_ROWS];
    alignas(16) float ks[BT_RING][128], pv[BT_RING][128];
};

template <int HD, int FMT>
constexpr size_t bt_smem() {
    return 1024 + BtGeom<HD, FMT>::END + sizeof(BtShared);
}

// Wait for phase `parity`; false when it, or another warp's wait, gave up.
__device__ __forceinline__ bool bt_wait(uint64_t *bar, uint32_t parity, int *dead) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity)) {
        if (*(volatile int *)dead) return false;
        if (globaltimer() - t0 > kWaitLimitNs) {
            *(volatile int *)dead = 1;
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ float bt_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes at row r, 16-byte chunk c of a 128-byte-swizzled tile
__device__ __forceinline__ uint8_t *bt_at(uint8_t *tile, int r, int c) {
    return tile + r * 128 + ((c ^ (r & 7)) << 4);
}

// the largest |x| of the feeding warps' threads (all call it)
__device__ __forceinline__ float bt_feed_max(float m, float *wmax) {
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int w = (threadIdx.x >> 5) - BT_SOFT - BT_OUT;
    if ((threadIdx.x & 31) == 0) wmax[w] = m;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * BT_FEED) : "memory");
#pragma unroll
    for (int i = 0; i < BT_FEED; i++) m = fmaxf(m, wmax[i]);
    return m;
}

// whether all feeding threads say yes: they leave their loop together
__device__ __forceinline__ bool bt_feed_all(bool yes) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.and.pred p, 2, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)yes), "n"(32 * BT_FEED)
        : "memory");
    return all != 0;
}

// What a feeding thread holds of a tile of 8-bit codes: K, 16 codes (16 bytes)
// of each of BN / rows-a-pass rows; V, DV dims of 8 positions in a row.
template <int HD>
struct BtFeed8 {
    static constexpr int LPR = HD / 16, RPP = 32 * BT_FEED / LPR, NK = (128 + RPP - 1) / RPP;
    static constexpr int DV = HD / 16 < 4 ? 4 : HD / 16, ITEMS = 16 * (HD / DV);
    uint4 k[NK];
    uint32_t v[8][DV / 4];
    float ks, vs;

    __device__ __forceinline__ void load_k(const uint8_t *kb, const float *ksc, const float *vsc, int j0,
                                           int n) {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const int r = p * RPP + t / LPR;
            k[p] = make_uint4(0, 0, 0, 0);
            if (r < n) k[p] = __ldg(reinterpret_cast<const uint4 *>(kb + (long long)(j0 + r) * HD) + t % LPR);
        }
        ks = vs = 0.f;
        if (t < n) ks = __ldg(ksc + j0 + t), vs = __ldg(vsc + j0 + t);
    }
    __device__ __forceinline__ void load_v(const uint8_t *vb, int j0, int n) {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
        if (t >= ITEMS) return;
        const int pg = (t & 7) | ((t >> 5) & 1) << 3, dg = ((t >> 3) & 3) | (t >> 6) << 2;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = pg * 8 + j;
            ba_ld<DV>(v[j], vb + (long long)(j0 + r) * HD + dg * DV, r < n);
        }
    }
    template <int FMT>
    __device__ __forceinline__ void store_k(uint8_t *tile) const {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const int r = p * RPP + t / LPR, i = t % LPR, blk = i >> 2, c = 2 * (i & 3);
            if (RPP * NK > 128 && r >= 128) continue;
            const uint32_t w[4] = {k[p].x, k[p].y, k[p].z, k[p].w};
            uint4 o[2];
            uint32_t *u = reinterpret_cast<uint32_t *>(o);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t x = FMT == KLLM_KV_I8 ? w[e] ^ 0x80808080u : w[e];
                u[2 * e] = ba_codes<FMT, 0>(x);
                u[2 * e + 1] = ba_codes<FMT, 1>(x);
            }
            // the lanes of the second block of dims store their odd chunk first: a row's eight
            // lanes then touch eight different banks' worth
            uint8_t *b = tile + blk * (128 * 128);
            const int s = blk & 1;
            *reinterpret_cast<uint4 *>(bt_at(b, r, c + s)) = o[s];
            *reinterpret_cast<uint4 *>(bt_at(b, r, c + 1 - s)) = o[1 - s];
        }
    }
    template <int FMT>
    __device__ __forceinline__ void store_v(uint8_t *tile) const {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
        if (t >= ITEMS) return;
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

// The same of an fp32 tile of 64 positions: K, four dims of rows in turn; V, four
// dims of 8 positions in a row.
template <int HD>
struct BtFeed32 {
    static constexpr int LPR = HD / 4, RPP = 32 * BT_FEED / LPR, NK = (64 + RPP - 1) / RPP;
    static constexpr int ITEMS = 8 * (HD / 4);
    float4 k[NK], v[8];

    __device__ __forceinline__ void load_k(const uint8_t *kb, int j0, int n) {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const int r = p * RPP + t / LPR;
            k[p] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < n)
                k[p] = __ldg(reinterpret_cast<const float4 *>(kb + (long long)(j0 + r) * HD * 4) + t % LPR);
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t *vb, int j0, int n) {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
        const int pg = t & 7, dg = t >> 3;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = pg * 8 + j;
            v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t < ITEMS && r < n)
                v[j] = __ldg(reinterpret_cast<const float4 *>(vb + (long long)(j0 + r) * HD * 4) + dg);
        }
    }
    static __device__ __forceinline__ float most(float4 x) {
        return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    }
    __device__ __forceinline__ float max_k() const {
        float m = 0.f;
#pragma unroll
        for (int p = 0; p < NK; p++) m = fmaxf(m, most(k[p]));
        return m;
    }
    __device__ __forceinline__ float max_v() const {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, most(v[j]));
        return m;
    }
    __device__ __forceinline__ void store_k(uint8_t *tile, int term, float f) const {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const int r = p * RPP + t / LPR, i = t % LPR, blk = i >> 4;
            if (RPP * NK > 64 && r >= 64) continue;
            uint2 h, l;
            ba_split(k[p].x * f, k[p].y * f, &h.x, &l.x);
            ba_split(k[p].z * f, k[p].w * f, &h.y, &l.y);
            uint8_t *a = bt_at(tile + blk * (64 * 128), r, (i & 15) >> 1) + 8 * (i & 1);
            *reinterpret_cast<uint2 *>(a) = h;
            *reinterpret_cast<uint2 *>(a + term) = l;
        }
    }
    __device__ __forceinline__ void store_v(uint8_t *tile, int term, float f) const {
        const int t = threadIdx.x - 32 * (BT_SOFT + BT_OUT);
        if (t >= ITEMS) return;
        const int pg = t & 7, dg = t >> 3;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint4 h, l;
            auto x = [&](int j) { return (e == 0 ? v[j].x : e == 1 ? v[j].y : e == 2 ? v[j].z : v[j].w) * f; };
            ba_split(x(0), x(1), &h.x, &l.x);
            ba_split(x(2), x(3), &h.y, &l.y);
            ba_split(x(4), x(5), &h.z, &l.z);
            ba_split(x(6), x(7), &h.w, &l.w);
            uint8_t *a = bt_at(tile, 4 * dg + e, pg);
            *reinterpret_cast<uint4 *>(a) = h;
            *reinterpret_cast<uint4 *>(a + term) = l;
        }
    }
};

// grid: (kv head, tile of 128 rows, part) of the prefix
template <int HD, int FMT>
__global__ void __launch_bounds__(BT_THREADS, 1)
k_ba_prefix(const BaArgs a) {
    using G = BtGeom<HD, FMT>;
    constexpr bool F32 = G::F32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    BtShared &sh = *reinterpret_cast<BtShared *>(smem + G::END);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int b = blockIdx.x;
    const int part = b % a.pre.parts;
    b /= a.pre.parts;
    const int tile = b % a.tiles_pre, kvh = b / a.tiles_pre;
    const int p0 = part * a.pre.chunk, p1 = min(a.prefix_len, p0 + a.pre.chunk);
    const int nt = (p1 - p0 + G::BN - 1) / G::BN;
    const int n_rows = a.n_seq * a.groups;

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.k_full[i], 32 * BT_FEED);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], 32 * BT_FEED);
            mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 32 * BT_SOFT);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.o_empty[i], 32 * BT_OUT);
        }
        for (int i = 0; i < BT_RING; i++) mbar_init(&sh.sc_full[i], 32 * BT_FEED);
        sh.dead = 0;
        mbar_fence_init();
    }
    if (warp == BT_SOFT + BT_OUT + BT_FEED) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sh.tmem)), "r"(G::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The queries: LPR lanes a row, four dims each.  q times scale * log2(e), brought to
    // [2^13, 2^14) by a power of two, in two fp16 terms.
    {
        constexpr int LPR = HD / 4, RPW = 32 / LPR, WARPS = BT_THREADS / 32;
#pragma unroll 2
        for (int r0 = warp * RPW; r0 < BT_ROWS; r0 += WARPS * RPW) {
            const int r = r0 + lane / LPR, i = lane % LPR, R = tile * BT_ROWS + r;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (R < n_rows && r < BT_ROWS) {
                const float *q = a.q + (long long)(R / a.groups) * a.q_stride +
                                 (long long)(kvh * a.groups + R % a.groups) * HD + 4 * i;
                x = make_float4(q[0] * a.qk, q[1] * a.qk, q[2] * a.qk, q[3] * a.qk);
            }
            float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float up = ba_pow2(m), f = 0x1p14f / up;
            if (r < BT_ROWS) {
                if (i == 0) sh.rowfac[r] = up * 0x1p-14f;
                uint2 h, l;
                ba_split(x.x * f, x.y * f, &h.x, &l.x);
                ba_split(x.z * f, x.w * f, &h.y, &l.y);
                uint8_t *t = bt_at(smem + G::Q_AT + (i >> 4) * (BT_ROWS * 128), r, (i & 15) >> 1) + 8 * (i & 1);
                *reinterpret_cast<uint2 *>(t) = h;
                *reinterpret_cast<uint2 *>(t + G::Q_TERM) = l;
            }
        }
        fence_async_shared();
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
        // ------------------------------------------------------- softmax --
        const int r = 32 * warp + lane;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        const float fac = sh.rowfac[r];
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        for (int t = 0; t < nt; t++) {
            const int ring = t & (BT_RING - 1), n = min(G::BN, p1 - p0 - t * G::BN);
            ok = __all_sync(0xffffffffu, bt_wait(&sh.sc_full[ring], (t / BT_RING) & 1, &sh.dead) &&
                                             bt_wait(&sh.s_full[t & 1], (t / 2) & 1, &sh.dead));
            if (!ok) break;
            tc_fence_after();
            const float4 *ks = reinterpret_cast<const float4 *>(sh.ks[ring]);
            const float4 *pv = reinterpret_cast<const float4 *>(sh.pv[ring]);
            float mx = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < G::BN / 32; c++) {
                float s[32];
                tmem_ld32(s_cols(t) + lanes + 32 * c, s);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float4 k = ks[8 * c + e];
                    s[4 * e] *= k.x, s[4 * e + 1] *= k.y, s[4 * e + 2] *= k.z, s[4 * e + 3] *= k.w;
                }
                if (32 * c + 32 > n) {
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (32 * c + e >= n) s[e] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 32; e++) mx = fmaxf(mx, s[e]);
            }
            const float m_new = fmaxf(m_run, mx * fac);
            const float corr = m_run == -INFINITY ? 0.f : bt_ex2(m_run - m_new);
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            m_run = m_new;
            sh.corr[ring][r] = corr;
            float sum = 0.f;
            // 16 positions at a time: their two terms take the columns of their scores, 8 each
#pragma unroll 1
            for (int c = 0; c < G::BN / 16; c++) {
                float s[16];
                tmem_ld16(s_cols(t) + lanes + 16 * c, s);
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float4 k = ks[4 * c + e], v = pv[4 * c + e];
                    float p[4] = {bt_ex2(fmaf(s[4 * e] * k.x, fac, -ref)), bt_ex2(fmaf(s[4 * e + 1] * k.y, fac, -ref)),
                                  bt_ex2(fmaf(s[4 * e + 2] * k.z, fac, -ref)),
                                  bt_ex2(fmaf(s[4 * e + 3] * k.w, fac, -ref))};
                    if (16 * c + 16 > n) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (16 * c + 4 * e + i >= n) p[i] = 0.f;
                    }
                    sum += (p[0] + p[1]) + (p[2] + p[3]);
                    ba_split(p[0] * v.x, p[1] * v.y, &hi[2 * e], &lo[2 * e]);
                    ba_split(p[2] * v.z, p[3] * v.w, &hi[2 * e + 1], &lo[2 * e + 1]);
                }
                tmem_st8(s_cols(t) + lanes + 16 * c, hi);
                tmem_st8(s_cols(t) + lanes + 16 * c + 8, lo);
            }
            tmem_wait_st();
            l_run = l_run * corr + sum;
            tc_fence_before();
            mbar_arrive(&sh.p_full[t & 1]);
        }
        if (tile * BT_ROWS + r < n_rows) {
            const long long o = 2 * part_of(r);
            a.part_ml[o] = ok ? m_run : __uint_as_float(0x7fffffffu);
            a.part_ml[o + 1] = ok ? l_run : __uint_as_float(0x7fffffffu);
        }
    } else if (warp < BT_SOFT + BT_OUT) {
        // -------------------------------------------------------- output --
        const int w = warp - BT_SOFT, r = 32 * (w & 3) + lane;
        constexpr int NC = HD / 2;                 // columns of this thread
        const int c0 = (w >> 2) * NC;
        const uint32_t lanes = (uint32_t)(32 * (w & 3)) << 16;
        float acc[NC];
#pragma unroll
        for (int e = 0; e < NC; e++) acc[e] = 0.f;
        bool ok = true;
        for (int t = 0; t < nt; t++) {
            const int ring = t & (BT_RING - 1);
            ok = __all_sync(0xffffffffu, bt_wait(&sh.o_full[t & 1], (t / 2) & 1, &sh.dead));
            if (!ok) break;
            tc_fence_after();
            const float corr = sh.corr[ring][r], vs = sh.vscale[ring];
#pragma unroll
            for (int c = 0; c < NC / 16; c++) {
                float v[16];
                tmem_ld16(o_cols(t) + lanes + c0 + 16 * c, v);
#pragma unroll
                for (int e = 0; e < 16; e++) acc[16 * c + e] = fmaf(v[e], vs, acc[16 * c + e] * corr);
            }
            tc_fence_before();
            mbar_arrive(&sh.o_empty[t & 1]);
        }
        if (tile * BT_ROWS + r < n_rows) {
            float4 *o = reinterpret_cast<float4 *>(a.part_o + part_of(r) * HD + c0);
            const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
            for (int e = 0; e < NC / 4; e++)
                o[e] = ok ? make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3])
                          : make_float4(nan, nan, nan, nan);
        }
    } else if (warp < BT_SOFT + BT_OUT + BT_FEED) {
        // --------------------------------------------------------- feeding --
        const int f = tid - 32 * (BT_SOFT + BT_OUT);
        const uint8_t *kb = static_cast<const uint8_t *>(a.pre.k) + row0 * HD * (F32 ? 4 : 1);
        const uint8_t *vb = static_cast<const uint8_t *>(a.pre.v) + row0 * HD * (F32 ? 4 : 1);
        const float *ksc = F32 ? nullptr : a.pre.ks + row0, *vsc = F32 ? nullptr : a.pre.vs + row0;
        std::conditional_t<F32, BtFeed32<HD>, BtFeed8<HD>> x;
        auto load_k = [&](int t) {
            if constexpr (F32) x.load_k(kb, p0 + t * G::BN, p1 - p0 - t * G::BN);
            else x.load_k(kb, ksc, vsc, p0 + t * G::BN, min(128, p1 - p0 - t * G::BN));
        };
        auto load_v = [&](int t) { x.load_v(vb, p0 + t * G::BN, p1 - p0 - t * G::BN); };
        load_k(0);
        load_v(0);
        bool ok = true;
        for (int t = 0; t < nt; t++) {
            const int st = t & 1, ring = t & (BT_RING - 1);
            const uint32_t free_parity = ((t / 2) & 1) ^ 1;
            uint8_t *kt = smem + G::K_AT + st * G::K_STAGE, *vt = smem + G::V_AT + st * G::V_STAGE;
            // The keys of tile t - 2 are done: its scores were issued behind the output of tile t - 4,
            // which waited for the output warps to be done with tile t - 6, so the ring's slot is
            // free too.
            if (t >= 2) ok = ok && bt_wait(&sh.k_empty[st], free_parity, &sh.dead);
            if (!bt_feed_all(ok)) break;
            float vscale;
            if constexpr (F32) {
                const float km = ba_pow2(bt_feed_max(x.max_k(), sh.wmax[0]));
                const float vm = ba_pow2(bt_feed_max(x.max_v(), sh.wmax[1]));
                x.store_k(kt, G::K_TERM, 0x1p14f / km);
                if (f < G::BN) sh.ks[ring][f] = km * 0x1p-14f, sh.pv[ring][f] = 0x1p14f;
                vscale = vm;
            } else {
                x.template store_k<FMT>(kt);
                const float vm = ba_pow2(bt_feed_max(f < 128 ? fabsf(x.vs) : 0.f, sh.wmax[st]));
                if (f < G::BN) sh.ks[ring][f] = x.ks, sh.pv[ring][f] = x.vs * (0x1p14f / vm);
                vscale = vm;
            }
            if (f == 0) sh.vscale[ring] = F32 ? vscale * 0x1p-14f * 0x1p-14f : vscale * 0x1p-14f;
            fence_async_shared();
            mbar_arrive(&sh.k_full[st]);
            mbar_arrive(&sh.sc_full[ring]);
            if (t + 1 < nt) load_k(t + 1);
            if (t >= 2) ok = bt_wait(&sh.v_empty[st], free_parity, &sh.dead);
            if (ok) {
                if constexpr (F32) x.store_v(vt, G::V_TERM, 0x1p14f / vscale);
                else x.template store_v<FMT>(vt);
                fence_async_shared();
                mbar_arrive(&sh.v_full[st]);
            }
            if (t + 1 < nt) load_v(t + 1);
        }
    } else if (lane == 0) {
        // -------------------------------------------------------- products --
        constexpr uint32_t s_idesc = umma_idesc_f16(128, G::BN), o_idesc = umma_idesc_f16(128, HD);
        const uint32_t qa = smem_u32(smem + G::Q_AT);
        auto scores = [&](int t) {
            const uint32_t kt = smem_u32(smem + G::K_AT + (t & 1) * G::K_STAGE), d = s_cols(t);
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
            umma_commit(&sh.k_empty[t & 1]);
        };
        auto output = [&](int t) {
            const uint32_t vt = smem_u32(smem + G::V_AT + (t & 1) * G::V_STAGE), d = o_cols(t), p = s_cols(t);
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
            umma_commit(&sh.v_empty[t & 1]);
        };
        bool ok = bt_wait(&sh.k_full[0], 0, &sh.dead);
        tc_fence_after();
        if (ok) scores(0);
        for (int t = 0; t < nt && ok; t++) {
            if (t + 1 < nt) {
                ok = bt_wait(&sh.k_full[(t + 1) & 1], ((t + 1) / 2) & 1, &sh.dead);
                tc_fence_after();
                if (!ok) break;
                scores(t + 1);
            }
            ok = bt_wait(&sh.p_full[t & 1], (t / 2) & 1, &sh.dead) &&
                 bt_wait(&sh.v_full[t & 1], (t / 2) & 1, &sh.dead) &&
                 (t < 2 || bt_wait(&sh.o_empty[t & 1], ((t / 2) & 1) ^ 1, &sh.dead));
            tc_fence_after();
            if (ok) output(t);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == BT_SOFT + BT_OUT + BT_FEED) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::COLS)
                     : "memory");
    }
}

}  // namespace
}  // namespace kllm
