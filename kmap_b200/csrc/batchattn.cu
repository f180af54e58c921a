// batchattn.cu -- decode attention of a batch whose sequences share a prefix
// (kllm_batch_attention): one query token per sequence over the prefix's
// positions, read once for all sequences, and the sequence's own.
//
// Both are cut into ranges of positions ("parts"); a part's block leaves its
// running maximum m, its sum l and its unnormalised sum of p v per query
// row, and a row's parts are joined by the block of its own positions (where
// they are one part) or by k_ba_merge:
//     M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
// k_ba_part takes four or eight query rows; batchattn_tc.cuh 128, of a prefix.
//
// Products of fp32 queries and weights run on the tensor cores without
// losing them to 16 bits: a row of q (and of p) is split into two terms,
// hi = rn(x), lo = rn(x - hi), and both go through one product as two columns
// of the same operand.  Codes of 8 bits are exact in fp16; fp32 rows run as two tf32 terms each.
// Scores carry scale * log2(e) * (the key row's scale); a weight carries the
// value row's scale, times a power of two that brings a query row's largest
// p times scale so far to 2^14: p's fp16 terms, which end at 2^-24, stay in
// range and lose nothing that counts beside it, whatever the scales of values
// without weight are.
#include <algorithm>
#include <mutex>

#include "batchattn.cuh"
#include "batchattn_tc.cuh"
#include "rows.cuh"
#include "serve.cuh"
#include "sm100.cuh"

namespace kllm {
namespace {

// tf32 terms: x to the nearest of 11 significand bits, and the rest, which the
// product cuts to 11: it has either sign, so the cuts do not lean one way, and
// a NaN stays in it.
__device__ __forceinline__ void ba_split32(float x, uint32_t *hi, uint32_t *lo) {
    *hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    *lo = __float_as_uint(x - __uint_as_float(*hi));
}

// A warp's ring of key and value rows in shared memory: each stage holds
// PT positions (and their scales), copied 16 bytes at a time by the warp's own
// lanes, so no warp waits for another.  16-byte pieces are permuted within a
// row by the row's number (ba_turn) so that the fragments' reads, by four
// lanes a key row and eight lanes a value row, meet no bank twice (head dim
// 128 and fp32; at most twice for 8-bit rows below 128 bytes).
template <int HD, int FMT>
struct BaRing {
    static constexpr bool F32 = FMT == KLLM_KV_F32;
    static constexpr int PT = F32 ? 16 : 32;             // positions of a turn
    static constexpr int WARPS = F32 ? 2 : 4;            // of a block
    static constexpr int ROW = HD * (F32 ? 4 : 1);       // bytes
    static constexpr int PIECES = ROW / 16;              // of a row
    static constexpr int KV = PT * ROW;                  // bytes of a stage's keys, or values
    static constexpr int STAGE = 2 * KV + (F32 ? 0 : 2 * PT * 4);
    static constexpr int STAGES = ROW >= 128 ? 2 : 3;
    static constexpr int RINGS = WARPS * STAGES * STAGE;
    // the join of the warps takes the rings' place
    static constexpr int JOIN = WARPS * 8 * (HD + 2) * 4;
    static constexpr int SMEM = RINGS > JOIN ? RINGS : JOIN;
};

template <int HD, int FMT>
__device__ __forceinline__ int ba_turn(int row) {
    if constexpr (FMT == KLLM_KV_F32) return ((row & 1) << 2) | (row & 2);
    else return HD == 128 ? row & 7 : HD == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
}

// an 8 x 8 matrix of 16-bit values, a row in four lanes, transposed
__device__ __forceinline__ uint32_t ba_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The output of row (seq, h), by one warp, VEC = HD / 32 dims a lane: the join
// of n parts from `at` on and, where `one`, one more (its maximum m, sum l and
// o).
template <int HD>
__device__ __forceinline__ void ba_join(const BaArgs &a, long long at, int n, bool one, float m, float l,
                                        float (&o)[HD / 32], int seq, int h, int lane) {
    constexpr int VEC = HD / 32;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + at;
    const float *po = a.part_o + at * HD + VEC * lane;
    // the first 32 parts' statistics, a part a lane
    float2 mine = make_float2(-INFINITY, 0.f);
    if (lane < n) mine = ml[lane];
    float M = fmaxf(m, mine.x);
    for (int p = lane + 32; p < n; p += 32) M = fmaxf(M, ml[p].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float ref = M == -INFINITY ? 0.f : M;
    // (a part whose scores are all -infinity has no finite sums to give: NaN, as in one pass)
    const bool none = m == -INFINITY && l == 0.f;
    const float w0 = none ? 0.f : exp2f(m - ref);
    float L = l * w0;
#pragma unroll
    for (int e = 0; e < VEC; e++) o[e] *= w0;
    for (int p0 = 0; p0 < n; p0 += 32) {
        if (p0) mine = p0 + lane < n ? ml[p0 + lane] : make_float2(-INFINITY, 0.f);
        const float w = p0 + lane < n ? exp2f(mine.x - ref) : 0.f;
        float s = p0 + lane < n ? mine.y * w : 0.f;
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        L += s;
        const int c = min(32, n - p0);
#pragma unroll 8
        for (int p = 0; p < c; p++) {
            const float wp = __shfl_sync(0xffffffffu, w, p);
            float v[VEC];
            bd_load<VEC>(po + (long long)(p0 + p) * HD, v);
#pragma unroll
            for (int e = 0; e < VEC; e++) o[e] = fmaf(wp, v[e], o[e]);
        }
    }
    const bool empty = n == 0 && !one;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float v = empty ? 0.f : o[e] / L;
        if (a.terms_out)
            bd_emit(v, ((size_t)seq * a.nh + h) * HD + VEC * lane + e, a.terms, (size_t)a.n_seq * a.nh * HD,
                    a.terms_out);
        else
            a.out[(long long)seq * a.out_stride + (long long)h * HD + VEC * lane + e] = v;
    }
}

// One part of 4 NB query rows of one kv head.  grid: the prefix's (kv head,
// row tile, part), then the sequences' (sequence, kv head, row tile, part);
// the block's warps take turns at PT positions, each with its next turn on its
// way into its ring.
//
// The keys are the products' 16-row side, four query rows in two terms each
// its 8 columns: scores [16 positions][row, term], so that lane 4 g + i has
// row i's scores of positions g and g + 8, both terms.  The weights' two terms,
// as 16-bit pairs, are transposed within the warp into the other product's
// 8 columns: output [16 dims][row, term] = V^T [16 dims][16 positions] . P.
template <int HD, int FMT, int NB>
__global__ void __launch_bounds__(32 * BaRing<HD, FMT>::WARPS, BaRing<HD, FMT>::F32 ? 3 : NB == 1 ? 3 : 2)
k_ba_part(const BaArgs a) {
    using G = BaRing<HD, FMT>;
    constexpr bool F32 = G::F32;
    constexpr int W = G::WARPS, RT = 4 * NB, NT = G::PT / 16, DT = HD / 16;
    extern __shared__ __align__(128) uint8_t ring[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
    // which item
    int b = blockIdx.x, kvh, seq = 0, tile, part;
    const bool pre = b < a.blocks_pre;
    pdl_launch_dependents();
    if (pre) {
        part = b % a.pre.parts, b /= a.pre.parts;
        tile = b % a.tiles_pre, kvh = b / a.tiles_pre;
    } else {
        b -= a.blocks_pre;
        part = b % a.own.parts, b /= a.own.parts;
        tile = b % a.tiles_own, b /= a.tiles_own;
        kvh = b % a.nkv, seq = b / a.nkv;
    }
    // the queries, on their way while the length is read (row 0's for rows past the last)
    const int n_rows = pre ? a.n_seq * a.groups : a.groups;
    float qx[NB][HD / 4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        int row = tile * RT + 4 * nb + (g >> 1);
        row = row < n_rows ? row : 0;
        const int qs = pre ? row / a.groups : seq, qh = kvh * a.groups + (pre ? row % a.groups : row);
        const float *qp = a.q + (long long)qs * a.q_stride + (long long)qh * HD + (F32 ? 4 * i : i * (HD / 4));
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            const float *p = qp + (F32 ? 16 : 4) * d;
            float4 x;
            if (a.q_vec) x = __ldg(reinterpret_cast<const float4 *>(p));
            else x = make_float4(p[0], p[1], p[2], p[3]);
            qx[nb][4 * d] = x.x, qx[nb][4 * d + 1] = x.y, qx[nb][4 * d + 2] = x.z, qx[nb][4 * d + 3] = x.w;
        }
    }
    const int own = pre ? 0 : a.own_len[seq], len = pre ? a.prefix_len : min(own, a.own_cap);
    const BaSide &S = pre ? a.pre : a.own;
    const int p0 = part * S.chunk, p1 = p0 + max(min(len - p0, S.chunk), 0);
    const bool join = a.join && !pre;
    if ((p0 >= p1 && !join) || own < 0) {
        pdl_wait();
        return;
    }
    // cache rows of this (sequence, kv head)
    const long long at = (long long)seq * S.seq_stride + (long long)kvh * S.max_pos * HD;
    const uint8_t *kb = static_cast<const uint8_t *>(S.k) + at * (F32 ? 4 : 1);
    const uint8_t *vb = static_cast<const uint8_t *>(S.v) + at * (F32 ? 4 : 1);
    const long long sat = (long long)seq * S.scale_stride + (long long)kvh * S.max_pos;
    uint8_t *mine = ring + warp * G::STAGES * G::STAGE;
    const uint32_t mine_at = (uint32_t)__cvta_generic_to_shared(mine);
    // turn n of this warp: positions p0 + (W n + warp) PT ..
    const int turns = (p1 - p0 + G::PT - 1) / G::PT;
    const int n_turns = (turns - warp + W - 1) / W;
    // each lane copies the same pieces of every stage: rows r0, r0 + RS, .. (ba_turn repeats with them)
    constexpr int RS = 32 / G::PIECES > 0 ? 32 / G::PIECES : 1, CS = G::PIECES > 32 ? G::PIECES / 32 : 1;
    const int r0 = lane / G::PIECES, c0 = lane % G::PIECES;
    auto fetch = [&](int n) {
        if (n < n_turns) {
            const int j0 = p0 + (W * n + warp) * G::PT, left = p1 - j0;
            const uint32_t st = mine_at + (n % G::STAGES) * G::STAGE;
            const uint8_t *ks = kb + (long long)j0 * G::ROW, *vs = vb + (long long)j0 * G::ROW;
#pragma unroll
            for (int e = 0; e < G::PT / RS; e++) {
                const int r = r0 + e * RS;
                const int bytes = r < left ? 16 : 0, row = r < left ? r : 0;
#pragma unroll
                for (int q = 0; q < CS; q++) {
                    const int c = c0 + 32 * q;
                    const uint32_t d = st + r * G::ROW + ((c ^ ba_turn<HD, FMT>(r)) << 4);
                    ba_cp16(d, ks + row * G::ROW + 16 * c, bytes);
                    ba_cp16(d + G::KV, vs + row * G::ROW + 16 * c, bytes);
                }
            }
            if constexpr (!F32) {
                const int bytes = lane < left ? 4 : 0, row = lane < left ? lane : 0;
                ba_cp4(st + 2 * G::KV + 4 * lane, S.ks + sat + j0 + row, bytes);
                ba_cp4(st + 2 * G::KV + 4 * (G::PT + lane), S.vs + sat + j0 + row, bytes);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int n = 0; n < G::STAGES - 1; n++) fetch(n);
    // the queries' column of this lane: row g / 2's term g % 2
    uint32_t qb[NB][F32 ? HD / 8 : HD / 16][2];
    float fac[NB];       // of row i's scores
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const bool have = tile * RT + 4 * nb + (g >> 1) < n_rows, low = g & 1;
        if (!have)
#pragma unroll
            for (int d = 0; d < HD / 4; d++) qx[nb][d] = 0.f;
        if constexpr (F32) {
            fac[nb] = a.qk;
#pragma unroll
            for (int d = 0; d < HD / 4; d++) {
                uint32_t h, l;
                ba_split32(qx[nb][d], &h, &l);
                qb[nb][d >> 1][d & 1] = low ? l : h;
            }
        } else {
            // the row brought to [2^13, 2^14) by a power of two
            float m = 0.f;
#pragma unroll
            for (int d = 0; d < HD / 4; d++) m = fmaxf(m, fabsf(qx[nb][d]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const float up = ba_pow2(m), f = 0x1p13f / up;
            fac[nb] = __shfl_sync(0xffffffffu, a.qk * up * 0x1p-13f, 8 * i);
#pragma unroll
            for (int ks = 0; ks < HD / 16; ks++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    uint32_t h, l;
                    ba_split(qx[nb][4 * ks + 2 * e] * f, qx[nb][4 * ks + 2 * e + 1] * f, &h, &l);
                    qb[nb][ks][e] = low ? l : h;
                }
        }
    }
    // of row 4 nb + i: maximum and sum; 8-bit: the largest log2 of a weight times its value's scale (to
    // within a few 2^-20), and o in units of 2^-up
    float m_run[NB], l_run[NB], w_run[NB], o[NB][DT][4];
    int up[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        m_run[nb] = w_run[nb] = -INFINITY, l_run[nb] = 0.f, up[nb] = 14;
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[nb][t][e] = 0.f;
    }

#pragma unroll 1
    for (int turn = 0; turn < n_turns; turn++) {
        const int left = p1 - p0 - (W * turn + warp) * G::PT;
        asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 2) : "memory");
        __syncwarp();
        fetch(turn + G::STAGES - 1);
        const uint8_t *kt = mine + (turn % G::STAGES) * G::STAGE, *vt = kt + G::KV;
        const float *ksc = reinterpret_cast<const float *>(kt + 2 * G::KV), *vsc = ksc + G::PT;
        float s[NB][NT][2];   // log2 scores of row 4 nb + i, positions 16 t + g + {0, 8}
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float c[NB][4], d[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int e = 0; e < 4; e++) c[nb][e] = d[nb][e] = 0.f;
            const int r = 16 * t + g;             // this lane reads key rows r and r + 8
            const int tn = ba_turn<HD, FMT>(r);   // (the same of both)
            if constexpr (F32) {
#pragma unroll
                for (int u = 0; u < HD / 16; u++) {
                    const uint8_t *p = kt + r * G::ROW + (((4 * u + i) ^ tn) << 4);
                    const float4 x = *reinterpret_cast<const float4 *>(p);
                    const float4 y = *reinterpret_cast<const float4 *>(p + 8 * G::ROW);
                    uint32_t h[2][4], l[2][4];
                    ba_split32(x.x, &h[0][0], &l[0][0]);
                    ba_split32(y.x, &h[0][1], &l[0][1]);
                    ba_split32(x.y, &h[0][2], &l[0][2]);
                    ba_split32(y.y, &h[0][3], &l[0][3]);
                    ba_split32(x.z, &h[1][0], &l[1][0]);
                    ba_split32(y.z, &h[1][1], &l[1][1]);
                    ba_split32(x.w, &h[1][2], &l[1][2]);
                    ba_split32(y.w, &h[1][3], &l[1][3]);
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            ba_mma_tf32(c[nb], h[e], qb[nb][2 * u + e][0], qb[nb][2 * u + e][1]);
                            ba_mma_tf32(d[nb], l[e], qb[nb][2 * u + e][0], qb[nb][2 * u + e][1]);
                        }
                }
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        s[nb][t][e] = (c[nb][2 * e] + ((c[nb][2 * e + 1] + d[nb][2 * e]) + d[nb][2 * e + 1])) * fac[nb];
            } else {
                uint32_t kw[2][HD / 16];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint8_t *p = kt + (r + 8 * e) * G::ROW;
                    if constexpr (HD == 128) {
                        *reinterpret_cast<uint4 *>(kw[e]) = *reinterpret_cast<const uint4 *>(p + (((2 * i) ^ tn) << 4));
                        *reinterpret_cast<uint4 *>(kw[e] + 4) =
                            *reinterpret_cast<const uint4 *>(p + (((2 * i + 1) ^ tn) << 4));
                    } else if constexpr (HD == 64) {
                        *reinterpret_cast<uint4 *>(kw[e]) = *reinterpret_cast<const uint4 *>(p + ((i ^ tn) << 4));
                    } else {
                        *reinterpret_cast<uint2 *>(kw[e]) =
                            *reinterpret_cast<const uint2 *>(p + (((i >> 1) ^ tn) << 4) + 8 * (i & 1));
                    }
                }
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {
                    const uint32_t x = FMT == KLLM_KV_I8 ? kw[0][ks] ^ 0x80808080u : kw[0][ks];
                    const uint32_t y = FMT == KLLM_KV_I8 ? kw[1][ks] ^ 0x80808080u : kw[1][ks];
                    const uint32_t ka[4] = {ba_codes<FMT, 0>(x), ba_codes<FMT, 0>(y), ba_codes<FMT, 1>(x),
                                            ba_codes<FMT, 1>(y)};
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
                        ba_mma_f16(ks & 1 ? d[nb] : c[nb], ka, qb[nb][ks][0], qb[nb][ks][1]);
                }
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        s[nb][t][e] = ((c[nb][2 * e] + d[nb][2 * e]) + (c[nb][2 * e + 1] + d[nb][2 * e + 1])) *
                                      (ksc[r + 8 * e] * fac[nb]);
            }
            if (left < G::PT) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (r + 8 * e >= left) s[nb][t][e] = -INFINITY;
            }
        }
        float vs[NT][2], lv[NT][2];      // the values' scales and their log2
        if constexpr (!F32) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    vs[t][e] = vsc[16 * t + g + 8 * e];
                    lv[t][e] = ba_lg2(fabsf(vs[t][e]));
                }
        }
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float mx = m_run[nb], wx = w_run[nb];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                mx = fmaxf(mx, fmaxf(s[nb][t][0], s[nb][t][1]));
                if constexpr (!F32) wx = fmaxf(wx, fmaxf(s[nb][t][0] + lv[t][0], s[nb][t][1] + lv[t][1]));
            }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                if constexpr (!F32) wx = fmaxf(wx, __shfl_xor_sync(0xffffffffu, wx, x));
            }
            const float ref = mx == -INFINITY ? 0.f : mx, corr = ba_ex2(m_run[nb] - ref);
            float corr_o = corr;
            if constexpr (!F32) {
                // (an append's scales lie between 2^-109 and 2^120)
                const int to = wx == -INFINITY ? up[nb] : 14 + min(max(__float2int_rn(ref - wx), -126), 112);
                corr_o *= ba_exp2i(min(max(to - up[nb], -126), 126));
                up[nb] = to;
                w_run[nb] = wx;
            }
            if (__any_sync(0xffffffffu, corr != 1.f || corr_o != 1.f)) {
                l_run[nb] *= corr;
#pragma unroll
                for (int t = 0; t < DT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[nb][t][e] *= corr_o;
            }
            m_run[nb] = mx;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                s[nb][t][0] = ba_ex2(s[nb][t][0] - ref);
                s[nb][t][1] = ba_ex2(s[nb][t][1] - ref);
                l_run[nb] += s[nb][t][0] + s[nb][t][1];
            }
        }
        // P.V
        if constexpr (F32) {
            constexpr int T8 = G::PT / 8;      // by 8 positions: rows i and i + 4 of them
            uint32_t pb[T8][NB][2];
#pragma unroll
            for (int t = 0; t < T8; t++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float p = __shfl_sync(0xffffffffu, s[nb][t >> 1][t & 1], 4 * (i + 4 * e) + (g >> 1));
                        uint32_t h, l;
                        ba_split32(p, &h, &l);
                        pb[t][nb][e] = g & 1 ? l : h;
                    }
            // (the turn's sum by itself: the tensor core cuts its sums off, always towards zero, and o would
            // lose some 2^-25 of itself with each product)
#pragma unroll
            for (int u = 0; u < HD / 32; u++) {
                float d[NB][2][4] = {};
#pragma unroll
                for (int t = 0; t < T8; t++) {
                    const int r = 8 * t + i, tn = ba_turn<HD, FMT>(r);      // (the same of r + 4)
                    const uint8_t *p = vt + r * G::ROW + (((8 * u + g) ^ tn) << 4);
                    const float4 x = *reinterpret_cast<const float4 *>(p);
                    const float4 y = *reinterpret_cast<const float4 *>(p + 4 * G::ROW);
                    uint32_t h[2][4], l[2][4];
                    ba_split32(x.x, &h[0][0], &l[0][0]);
                    ba_split32(x.y, &h[0][1], &l[0][1]);
                    ba_split32(y.x, &h[0][2], &l[0][2]);
                    ba_split32(y.y, &h[0][3], &l[0][3]);
                    ba_split32(x.z, &h[1][0], &l[1][0]);
                    ba_split32(x.w, &h[1][1], &l[1][1]);
                    ba_split32(y.z, &h[1][2], &l[1][2]);
                    ba_split32(y.w, &h[1][3], &l[1][3]);
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            ba_mma_tf32(d[nb][e], l[e], pb[t][nb][0], pb[t][nb][1]);
                            ba_mma_tf32(d[nb][e], h[e], pb[t][nb][0], pb[t][nb][1]);
                        }
                }
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int c = 0; c < 4; c++) o[nb][2 * u + e][c] += d[nb][e][c];
            }
        } else {
#pragma unroll
            for (int t = 0; t < NT; t++) {   // 16 positions
                uint32_t pb[NB][2];
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float p = s[nb][t][e] * vs[t][e] * ba_exp2i(up[nb]);
                        const float h = __half2float(__float2half_rn(p));
                        pb[nb][e] = ba_transpose(ba_h2(h, p - h));
                    }
                uint32_t vw[4][HD / 32];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int r = 16 * t + 2 * i + (e & 1) + 8 * (e >> 1);
                    const int tn = ba_turn<HD, FMT>(r);
                    if constexpr (HD == 128)
                        *reinterpret_cast<uint4 *>(vw[e]) =
                            *reinterpret_cast<const uint4 *>(vt + r * G::ROW + ((g ^ tn) << 4));
                    else if constexpr (HD == 64)
                        *reinterpret_cast<uint2 *>(vw[e]) = *reinterpret_cast<const uint2 *>(
                            vt + r * G::ROW + (((g >> 1) ^ tn) << 4) + 8 * (g & 1));
                    else
                        vw[e][0] = *reinterpret_cast<const uint32_t *>(
                            vt + r * G::ROW + (((g >> 2) ^ tn) << 4) + 4 * (g & 3));
                    if constexpr (FMT == KLLM_KV_I8)
#pragma unroll
                        for (int w = 0; w < HD / 32; w++) vw[e][w] ^= 0x80808080u;
                }
#pragma unroll
                for (int w = 0; w < HD / 32; w++) {
                    const uint32_t x01 = ba_prmt(vw[0][w], vw[1][w], 0x5140);
                    const uint32_t x23 = ba_prmt(vw[0][w], vw[1][w], 0x7362);
                    const uint32_t y01 = ba_prmt(vw[2][w], vw[3][w], 0x5140);
                    const uint32_t y23 = ba_prmt(vw[2][w], vw[3][w], 0x7362);
                    const uint32_t va[4] = {ba_codes<FMT, 0>(x01), ba_codes<FMT, 1>(x01), ba_codes<FMT, 0>(y01),
                                            ba_codes<FMT, 1>(y01)};
                    const uint32_t wa[4] = {ba_codes<FMT, 0>(x23), ba_codes<FMT, 1>(x23), ba_codes<FMT, 0>(y23),
                                            ba_codes<FMT, 1>(y23)};
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) {
                        ba_mma_f16(o[nb][2 * w], va, pb[nb][0], pb[nb][1]);
                        ba_mma_f16(o[nb][2 * w + 1], wa, pb[nb][0], pb[nb][1]);
                    }
                }
            }
        }
        __syncwarp();      // the stage may be filled again
    }
    // join the warps, in warp order, where the rings were
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float(*sm_o)[8][HD] = reinterpret_cast<float(*)[8][HD]>(ring);
    float(*sm_ml)[8][2] = reinterpret_cast<float(*)[8][2]>(ring + W * 8 * HD * sizeof(float));
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l_run[nb] += __shfl_xor_sync(0xffffffffu, l_run[nb], x);
        if (g == 0) {
            sm_ml[warp][4 * nb + i][0] = m_run[nb];
            sm_ml[warp][4 * nb + i][1] = l_run[nb];
        }
    }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const int rr = 4 * nb + i;
        float M = sm_ml[0][rr][0];
#pragma unroll
        for (int w = 1; w < W; w++) M = fmaxf(M, sm_ml[w][rr][0]);
        float f = m_run[nb] == -INFINITY ? 0.f : exp2f(m_run[nb] - M);
        if constexpr (!F32) f *= ba_exp2i(-up[nb]);
#pragma unroll
        for (int t = 0; t < DT; t++) {
            // dims of rows g and g + 8 of tile t
            const int d = F32 ? 32 * (t >> 1) + 4 * g + 2 * (t & 1) : g * (HD / 8) + 2 * t;
            *reinterpret_cast<float2 *>(&sm_o[warp][rr][d]) =
                make_float2((o[nb][t][0] + o[nb][t][1]) * f, (o[nb][t][2] + o[nb][t][3]) * f);
        }
    }
    __syncthreads();
    const int parts = a.pre.parts + a.own.parts, pi = pre ? part : a.pre.parts + part;
    // a warp takes a row: its part's maximum and sum, VEC dims a lane
    constexpr int VEC = HD / 32;
    // (dependent launches: the join below, and the one in k_ba_merge, wait for this
    // launch alone, so none of its blocks ends before the launch before does)
    if (!join) pdl_wait();
    for (int rr = warp; rr < RT; rr += W) {
        const int R = tile * RT + rr;
        if (R >= n_rows) break;
        const int rs = pre ? R / a.groups : seq, rh = kvh * a.groups + (pre ? R % a.groups : R);
        float m = sm_ml[0][rr][0], l = 0.f, v[VEC];
#pragma unroll
        for (int w = 1; w < W; w++) m = fmaxf(m, sm_ml[w][rr][0]);
#pragma unroll
        for (int w = 0; w < W; w++)
            if (sm_ml[w][rr][0] != -INFINITY) l += sm_ml[w][rr][1] * exp2f(sm_ml[w][rr][0] - m);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            v[e] = sm_o[0][rr][VEC * lane + e];
#pragma unroll
            for (int w = 1; w < W; w++) v[e] += sm_o[w][rr][VEC * lane + e];
        }
        const long long at = ((long long)rs * a.nh + rh) * parts;
        if (join) {
            pdl_wait();
            ba_join<HD>(a, at, a.pre.parts, p1 > p0, m, l, v, rs, rh, lane);
        } else {
            float *o = a.part_o + (at + pi) * HD + VEC * lane;
#pragma unroll
            for (int e = 0; e < VEC; e++) o[e] = v[e];
            if (lane == 0) a.part_ml[2 * (at + pi)] = m, a.part_ml[2 * (at + pi) + 1] = l;
        }
    }
    if (join) pdl_wait();
}

// Rows whose parts lie in memory, one warp per row.
template <int HD>
__global__ void __launch_bounds__(128)
k_ba_merge(const BaArgs a) {
    const int R = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (R >= a.n_seq * a.nh) return;
    const int seq = R / a.nh, h = R % a.nh;
    pdl_wait();
    const int own = a.own_len ? a.own_len[seq] : 0, len = min(own, a.own_cap);
    if (own < 0) return;
    const int n = a.pre.parts + (len > 0 ? (len + a.own.chunk - 1) / a.own.chunk : 0);
    float v[HD / 32] = {};
    ba_join<HD>(a, (long long)R * (a.pre.parts + a.own.parts), n, false, -INFINITY, 0.f, v,
                seq, h, lane);
}

// How a call is cut.
struct BaCut {
    int tiles_pre = 0, tiles_own = 0, own_cap = 0;
    int parts_pre = 0, chunk_pre = 0, parts_own = 0, chunk_own = 0;
    bool wide = false;      // the prefix by 128-row tiles
    int nb = 1, nb_pre = 1; // a tile's query rows over four
    bool join = false;      // own positions in one part, joined where they are computed
    size_t rows = 0, bytes = 0;
    long long pre_blocks = 0, own_blocks = 0;
};

// Most positions of a range: what the kernels and the cut count in 32 bits, with room for a piece's rounding.
constexpr int BA_POSITIONS = 0x7ffffc00;

// len positions (at most BA_POSITIONS) in n pieces of a multiple of 128, or fewer.
void ba_pieces(int len, int n, int *parts, int *chunk) {
    *chunk = ((len - 1) / n + 128) / 128 * 128;
    *parts = (len - 1) / *chunk + 1;
}

// `items` ranges of up to len positions into parts of at least 128 positions
// (a turn of each warp), as many as give every SM its two blocks twice over,
// and of at most 512 where the lengths are only bounds (blocks past a length
// end at once, the others even out), else 2048: with 8 bits a warp's sums pass
// through the tensor core with every 16 positions, which cuts off half a unit
// of 2^-23 in the mean, always towards zero (over 14,500 positions a warp, 2^-16).
void ba_split_range(long long items, int len, bool bound, int *parts, int *chunk) {
    const long long want = std::max<long long>(1, (148 * 4 + items - 1) / items);
    const long long most = (len + 127) / 128, least = (len - 1) / (bound ? 512 : 2048) + 1;
    ba_pieces(len, (int)std::min(std::max(want, least), most), parts, chunk);
}

BaCut ba_cut(const kllm_batch_attn &a) {
    const kllm_kv_cache *c = a.prefix ? a.prefix : a.own;
    BaCut x;
    const int groups = a.n_heads / c->n_kv;
    x.nb = groups > 4 ? 2 : 1;
    const int tile = 4 * x.nb;
    x.own_cap = a.own ? std::min(a.max_len, a.own->max_pos) : 0;
    const int pre = a.prefix ? a.prefix_len : 0;
    if (pre > 0) {
        const long long rows = (long long)a.n_seq * groups;
        // The 128-row tiles have a start of some 12 us and little time per row, the narrow tiles 6 us and
        // theirs per row: which ends first goes with positions x rows x kv heads, and 24 rows leave the
        // wide tiles too empty.  Measured, narrow and wide, in us (with one own position each):
        //   e4m3    head dim 128, 32 kv heads: 32 rows x 2000  36.0 35.4, 48 x 1000  35.6 36.1, 64 x 1000
        //           44 42, 64 x 4000  81 59, 24 x 4000  39 43; 8 kv heads: 32 x 4000  16.5 19.4, 48 x 4000
        //           24 21; head dim 64, 4 kv heads: 256 x 500  14.1 15.5, 192 x 1000  12.8 14.1, 256 x 1000
        //           15.9 14.1, 128 x 1000  12.6 14.1, 32 x 1000  7.9 12.4
        //   fp32    head dim 128, 32 kv heads: 16 x 4000  60 76, 24 x 4000  92 76, 24 x 1000  31 32, 32 x
        //           1000  43 35; head dim 64, 4 kv heads: 128 x 1000  16 19, 192 x 1000  23 19
        const long long work = c->n_kv * rows * pre;
        x.wide = c->format == KLLM_KV_F32 ? rows >= 24 && work >= 1000000
                                          : rows >= 32 && work >= 12000ll * c->head_dim;
        // fp32 tiles are read once per tile: eight rows as soon as there are more than four (24 rows x 4000
        // as above: 91 us, 96 in tiles of four)
        x.nb_pre = c->format == KLLM_KV_F32 ? (rows > 4 ? 2 : 1) : x.nb;
        const int t = x.wide ? BT_ROWS : 4 * x.nb_pre;
        x.tiles_pre = (int)((rows + t - 1) / t);
        const long long items = (long long)c->n_kv * x.tiles_pre;
        if (x.wide) {
            // one block an SM: as many parts as fill them once
            ba_pieces(pre, (int)std::min<long long>(std::max<long long>(148 / items, 1), (pre + 127) / 128),
                      &x.parts_pre, &x.chunk_pre);
        } else {
            ba_split_range(items, pre, false, &x.parts_pre, &x.chunk_pre);
        }
    }
    if (x.own_cap > 0) {
        x.tiles_own = (groups + tile - 1) / tile;
        const long long items = (long long)a.n_seq * c->n_kv * x.tiles_own;
        // One part, joined where it is computed (no launch for the join), where a block's keys are few, or
        // the blocks as many as they are KB: measured, more parts and one, in us, after 64 positions of a
        // prefix: head dim 128, 8 kv heads of int8, 512 positions: 1 sequence 7.4 8.2, 8 sequences 9.8
        // 8.8, 48 19 16; 1000: 8 sequences 11.5 11.7, 16 14.7 12.1; 128: 1 sequence 6.3 5.6; 32 kv heads of
        // fp32, 64: 6.9 6.3; 256: 1 sequence 8.8 11.7, 8 19.8 12.2; 1000: 4 19 33, 16 54 57.  Above 1024
        // positions lengths differ enough for parts to even them out.
        const long long kb = (long long)x.own_cap * c->head_dim * (c->format == KLLM_KV_F32 ? 4 : 1) / 1024;
        if (kb <= 32 || (x.own_cap <= 1024 && items >= kb)) {
            x.parts_own = 1;
            x.chunk_own = x.own_cap;
            x.join = true;
        } else {
            ba_split_range(items, x.own_cap, true, &x.parts_own, &x.chunk_own);
        }
    }
    x.pre_blocks = (long long)c->n_kv * x.tiles_pre * x.parts_pre;
    x.own_blocks = (long long)a.n_seq * c->n_kv * x.tiles_own * x.parts_own;
    x.rows = (size_t)a.n_seq * a.n_heads;
    const size_t parts = x.parts_pre + x.parts_own;
    x.bytes = ((x.rows * parts * 2 * 4 + 15) / 16 * 16) + x.rows * parts * c->head_dim * 4 + 16;
    return x;
}

// Whether the call can be run, and its cut.
bool ba_ok(const char *who, const kllm_batch_attn *a, BaCut *x) {
    if (!a || a->n_seq < 1 || a->n_heads < 1 || !a->q || (!a->prefix && !a->own)) {
        set_error("%s: invalid arguments", who);
        return false;
    }
    if (a->prefix && !kv_cache_ok(who, a->prefix)) return false;
    if (a->own && !kv_cache_ok(who, a->own)) return false;
    if (a->prefix && a->own &&
        (a->prefix->format != a->own->format || a->prefix->n_kv != a->own->n_kv ||
         a->prefix->head_dim != a->own->head_dim)) {
        set_error("%s: the two caches differ in format, kv heads or head dim", who);
        return false;
    }
    if (a->prefix_len < 0 || (a->prefix ? a->prefix_len > a->prefix->max_pos : a->prefix_len > 0)) {
        set_error("%s: a prefix of %d positions outside its cache", who, a->prefix_len);
        return false;
    }
    if (a->own && (!a->own_len || a->own->n_seq < a->n_seq || a->max_len < 0)) {
        set_error("%s: own cache of %d sequences for %d, lengths %s, max_len %d", who, a->own->n_seq,
                  a->n_seq, a->own_len ? "given" : "NULL", a->max_len);
        return false;
    }
    const kllm_kv_cache *c = a->prefix ? a->prefix : a->own;
    if (a->n_heads % c->n_kv) {
        set_error("%s: %d heads on %d kv heads", who, a->n_heads, c->n_kv);
        return false;
    }
    if (a->n_seq > 1 && a->q_stride < (long long)a->n_heads * c->head_dim) {
        set_error("%s: q_stride %lld for %d heads of %d", who, a->q_stride, a->n_heads, c->head_dim);
        return false;
    }
    const int own = a->own ? std::min(a->max_len, a->own->max_pos) : 0;
    if ((long long)a->n_seq * a->n_heads > 0x7fffffffll || std::max(a->prefix_len, own) > BA_POSITIONS) {
        set_error("%s: %d sequences of %d heads, %d positions of a prefix and %d of their own are more than "
                  "32 bits count", who, a->n_seq, a->n_heads, a->prefix_len, own);
        return false;
    }
    *x = ba_cut(*a);
    if (x->pre_blocks + x->own_blocks > 0x7fffffffll) {
        set_error("%s: %lld blocks", who, x->pre_blocks + x->own_blocks);
        return false;
    }
    return true;
}

// A kernel's shared-memory limit, raised once per device.
template <auto KERNEL>
bool ba_prepare(size_t smem) {
    static std::mutex mu;
    static bool ready[64] = {};
    int dev = 0;
    if (!KLLM_CUDA(cudaGetDevice(&dev))) return false;
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 64 && ready[dev]) return true;
    if (!KLLM_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)))
        return false;
    if (dev < 64) ready[dev] = true;
    return true;
}

template <int HD, int FMT>
bool ba_launch(cudaStream_t s, const BatchAttention &call, const BaCut &x) {
    const kllm_batch_attn &a = call.a;
    const kllm_kv_cache *c = a.prefix ? a.prefix : a.own;
    BaArgs k = {};
    auto side = [](const kllm_kv_cache *c, int parts, int chunk) {
        BaSide d = {};
        if (c) d = {c->k, c->v, c->k_scale, c->v_scale, c->seq_stride, c->scale_stride, c->max_pos, 0, 1};
        d.parts = parts;
        d.chunk = std::max(chunk, 1);
        return d;
    };
    k.pre = side(a.prefix, x.parts_pre, x.chunk_pre);
    k.own = side(a.own, x.parts_own, x.chunk_own);
    k.q = a.q;
    k.q_stride = a.q_stride;
    k.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.n_seq == 1 || a.q_stride % 4 == 0);
    k.own_len = a.own ? a.own_len : nullptr;
    k.n_seq = a.n_seq;
    k.nh = a.n_heads;
    k.nkv = c->n_kv;
    k.groups = a.n_heads / c->n_kv;
    k.prefix_len = x.parts_pre ? a.prefix_len : 0;
    k.own_cap = x.own_cap;
    k.tiles_pre = std::max(x.tiles_pre, 1);
    k.tiles_own = std::max(x.tiles_own, 1);
    k.qk = (float)((double)a.scale * 1.4426950408889634);
    k.part_ml = static_cast<float *>(a.workspace);
    const size_t parts = x.parts_pre + x.parts_own;
    k.part_o = reinterpret_cast<float *>(static_cast<char *>(a.workspace) +
                                         (x.rows * parts * 2 * 4 + 15) / 16 * 16);
    k.join = x.join;
    k.out = a.out;
    k.out_stride = a.out_stride;
    k.terms = call.terms;
    k.terms_out = call.terms_out;
    k.status = call.status;
    k.wait_ns = call.wait_ns;
    // Each launch but the first may start beside the one before, and waits
    // for it where it needs it: the sequences' blocks before they join or end,
    // k_ba_merge at once.
    bool first = true;
    auto launch = [&](auto kernel, unsigned grid, unsigned block, size_t smem, auto... args) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(block);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = first ? 0 : 1;
        first = false;
        g_launches++;
        return KLLM_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    };
    if (x.wide) {
        constexpr size_t smem = bt_smem<HD, FMT>();
        if (!ba_prepare<k_ba_prefix<HD, FMT>>(smem) ||
            !launch(k_ba_prefix<HD, FMT>, (unsigned)x.pre_blocks, BtGeom<HD, FMT>::THREADS, smem, k))
            return false;
    }
    auto part = [&](long long pre, long long own) {
        using G = BaRing<HD, FMT>;
        if (pre + own == 0) return true;
        k.blocks_pre = (int)pre;
        auto go = [&](auto nb) {
            constexpr auto kernel = k_ba_part<HD, FMT, decltype(nb)::value>;
            return ba_prepare<kernel>(G::SMEM) && launch(kernel, (unsigned)(pre + own), 32 * G::WARPS, G::SMEM, k);
        };
        return (pre ? x.nb_pre : x.nb) == 1 ? go(std::integral_constant<int, 1>())
                                            : go(std::integral_constant<int, 2>());
    };
    const long long narrow = x.wide ? 0 : x.pre_blocks;
    if (x.join || x.nb != x.nb_pre ? !part(narrow, 0) || !part(0, x.own_blocks) : !part(narrow, x.own_blocks))
        return false;
    if (!x.join && !launch(k_ba_merge<HD>, (unsigned)((x.rows + 3) / 4), 128, 0, k)) return false;
    return KLLM_CUDA(cudaGetLastError());
}

}  // namespace

bool batch_attention(cudaStream_t s, const BatchAttention &b) {
    const char *who = "kllm_batch_attention";
    const kllm_batch_attn &a = b.a;
    BaCut x;
    if (!ba_ok(who, &a, &x)) return false;
    if (!a.out && !b.terms_out) {
        set_error("%s: invalid arguments", who);
        return false;
    }
    const kllm_kv_cache *c = a.prefix ? a.prefix : a.own;
    if (!b.terms_out && a.n_seq > 1 && a.out_stride < (long long)a.n_heads * c->head_dim) {
        set_error("%s: out_stride %lld for %d heads of %d", who, a.out_stride, a.n_heads, c->head_dim);
        return false;
    }
    if (!a.workspace || a.workspace_bytes < x.bytes || (reinterpret_cast<uintptr_t>(a.workspace) & 15)) {
        set_error("%s: %zu bytes of workspace on 16 bytes needed, %zu given", who, x.bytes,
                  a.workspace ? a.workspace_bytes : (size_t)0);
        return false;
    }
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return c->format == KLLM_KV_F32 ? ba_launch<HD, KLLM_KV_F32>(s, b, x)
             : c->format == KLLM_KV_I8  ? ba_launch<HD, KLLM_KV_I8>(s, b, x)
                                        : ba_launch<HD, KLLM_KV_E4M3>(s, b, x);
    };
    return c->head_dim == 32 ? go(std::integral_constant<int, 32>())
         : c->head_dim == 64 ? go(std::integral_constant<int, 64>())
                             : go(std::integral_constant<int, 128>());
}

}  // namespace kllm

using namespace kllm;

extern "C" size_t kllm_batch_attention_workspace(const kllm_batch_attn *a) {
    BaCut x;
    return ba_ok("kllm_batch_attention_workspace", a, &x) ? x.bytes : 0;
}

extern "C" int kllm_batch_attention(const kllm_batch_attn *a, void *stream) {
    if (!a) {
        set_error("kllm_batch_attention: invalid arguments");
        return -1;
    }
    BatchAttention b;
    b.a = *a;
    return batch_attention((cudaStream_t)stream, b) ? 0 : -1;
}
