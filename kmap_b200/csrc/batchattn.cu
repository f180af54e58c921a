// batchattn.cu -- decode attention of a batch whose sequences share a prefix
// (kllm_batch_attention): one query token per sequence over the prefix's
// positions, read once for all sequences, and the sequence's own.
//
// Both are cut into ranges of positions ("parts"); a part's block leaves its
// running maximum m, its sum l and its unnormalised sum of p v per query
// row, and k_ba_merge joins a row's parts:
//     M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
//
// Products of fp32 queries and weights run on the tensor cores without
// losing them to 16 bits: a row of q (and of p) is split into two terms,
// hi = rn(x), lo = rn(x - hi), and both go through one product as two rows
// of the same 16-row operand, so a tile is eight query rows by both terms.
// Codes of 8 bits are exact in fp16; fp32 rows run as two tf32 terms each.
// Scores carry scale * log2(e) * (the key row's scale); a weight carries the
// value row's scale over the largest scale met so far (a power of two), so
// p's fp16 terms stay in range whatever the scales are.
#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "batchattn.cuh"
#include "batchattn_tc.cuh"
#include "rows.cuh"
#include "serve.cuh"
#include "sm100.cuh"

namespace kllm {
namespace {

// tf32 terms: the upper 11 significand bits, and the rest (13 bits, of which
// the product takes 11)
__device__ __forceinline__ void ba_split32(float x, uint32_t *hi, uint32_t *lo) {
    *hi = __float_as_uint(x) & 0xffffe000u;
    *lo = __float_as_uint(x - __uint_as_float(*hi));
}

// A warp's ring of key and value rows in shared memory: each stage holds
// PT positions (and their scales), copied 16 bytes at a time by the warp's own
// lanes, so no warp waits for another.  16-byte pieces are permuted within a
// row by the row's number (ba_turn) so that the fragments' reads, by four
// lanes a key row and eight lanes a value row, meet no bank twice.
template <int HD, int FMT>
struct BaRing {
    static constexpr bool F32 = FMT == KLLM_KV_F32;
    static constexpr int PT = F32 ? 16 : 32;             // positions of a turn
    static constexpr int ROW = HD * (F32 ? 4 : 1);       // bytes
    static constexpr int PIECES = ROW / 16;              // of a row
    static constexpr int KV = PT * ROW;                  // bytes of a stage's keys, or values
    static constexpr int STAGE = 2 * KV + (F32 ? 0 : 2 * PT * 4);
    static constexpr int STAGES = F32 ? (HD == 128 ? 2 : 3) : HD == 128 ? 3 : 4;
    static constexpr int SMEM = BA_WARPS * STAGES * STAGE;
    // the join of the warps (in the rings' place) must fit
    static_assert(SMEM >= BA_WARPS * BA_ROWS * (HD + 2) * 4, "ring below the join's size");
};

template <int HD, int FMT>
__device__ __forceinline__ int ba_turn(int row) {
    if constexpr (FMT == KLLM_KV_F32) return (row & 6) ^ ((row & 1) << 2);
    else return HD == 128 ? row & 7 : HD == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
}

__device__ __forceinline__ void ba_cp16(uint32_t dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void ba_cp4(uint32_t dst, const void *src, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0)
                 : "memory");
}

// One part of eight query rows of one kv head.  grid: the prefix's
// (kv head, row tile, part), then the sequences' (sequence, kv head, row tile,
// part); four warps take turns at blocks of PT positions, each with the next
// blocks on their way into its ring.
template <int HD, int FMT>
__global__ void __launch_bounds__(BA_THREADS, 2)
k_ba_part(const BaArgs a) {
    using G = BaRing<HD, FMT>;
    constexpr bool F32 = G::F32;
    constexpr int NT = G::PT / 8;           // 8-position tiles per turn
    extern __shared__ __align__(128) uint8_t ring[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
    // which item
    int b = blockIdx.x, kvh, seq = 0, tile, part, len;
    const int n_pre = a.wide ? 0 : a.nkv * a.tiles_pre * a.pre.parts;
    const bool pre = b < n_pre;
    if (pre) {
        part = b % a.pre.parts, b /= a.pre.parts;
        tile = b % a.tiles_pre, kvh = b / a.tiles_pre;
        len = a.prefix_len;
    } else {
        b -= n_pre;
        part = b % a.own.parts, b /= a.own.parts;
        tile = b % a.tiles_own, b /= a.tiles_own;
        kvh = b % a.nkv, seq = b / a.nkv;
        len = ba_len(a.own_len, a.own_cap, seq);
    }
    const BaSide &S = pre ? a.pre : a.own;
    const int p0 = part * S.chunk, p1 = min(len, p0 + S.chunk);
    if (p0 >= p1) {
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
    // turn n of this warp: positions p0 + (4 n + warp) PT ..
    const int turns = (p1 - p0 + G::PT - 1) / G::PT;
    const int n_turns = (turns - warp + BA_WARPS - 1) / BA_WARPS;
    auto fetch = [&](int n) {
        if (n < n_turns) {
            const int j0 = p0 + (BA_WARPS * n + warp) * G::PT;
            const uint32_t st = mine_at + (n % G::STAGES) * G::STAGE;
#pragma unroll
            for (int e = 0; e < G::PT * G::PIECES / 32; e++) {
                const int q = e * 32 + lane, r = q / G::PIECES, c = q % G::PIECES;
                const uint32_t d = st + r * G::ROW + ((c ^ ba_turn<HD, FMT>(r)) << 4);
                const long long off = (long long)(j0 + r) * G::ROW + 16 * c;
                const bool in = j0 + r < p1;
                ba_cp16(d, kb + (in ? off : 0), in);
                ba_cp16(d + G::KV, vb + (in ? off : 0), in);
            }
            if constexpr (!F32) {
                const bool in = j0 + lane < p1;
                ba_cp4(st + 2 * G::KV + 4 * lane, S.ks + sat + (in ? j0 + lane : 0), in);
                ba_cp4(st + 2 * G::KV + 4 * (G::PT + lane), S.vs + sat + (in ? j0 + lane : 0), in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int n = 0; n < G::STAGES - 1; n++) fetch(n);
    // this lane's query row
    const int n_rows = pre ? a.n_seq * a.groups : a.groups, row = tile * BA_ROWS + g;
    const int qs = pre ? row / a.groups : seq, qh = kvh * a.groups + (pre ? row % a.groups : row);
    const bool have = row < n_rows;
    const float *qp = a.q + (long long)qs * a.q_stride + (long long)qh * HD;
    uint32_t qa[F32 ? HD / 8 : HD / 16][4];
    float rowfac = a.qk;
    if constexpr (F32) {
#pragma unroll
        for (int u = 0; u < HD / 16; u++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int d = 16 * u + 4 * i + 2 * e;
                const float x = have ? qp[d] : 0.f, y = have ? qp[d + 1] : 0.f;
                ba_split32(x, &qa[2 * u + e][0], &qa[2 * u + e][1]);
                ba_split32(y, &qa[2 * u + e][2], &qa[2 * u + e][3]);
            }
    } else {
        // the row brought to [2^13, 2^14) by a power of two
        float m = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 4; d++) m = fmaxf(m, have ? fabsf(qp[i * (HD / 4) + d]) : 0.f);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float up = ba_pow2(m), f = 0x1p14f / up;
        rowfac = a.qk * up * 0x1p-14f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ks++) {
            const int d = i * (HD / 4) + 4 * ks;
            const float x0 = have ? qp[d] * f : 0.f, x1 = have ? qp[d + 1] * f : 0.f;
            const float x2 = have ? qp[d + 2] * f : 0.f, x3 = have ? qp[d + 3] * f : 0.f;
            ba_split(x0, x1, &qa[ks][0], &qa[ks][1]);
            ba_split(x2, x3, &qa[ks][2], &qa[ks][3]);
        }
    }
    float m_run = -INFINITY, l_run = 0.f, sv = 0x1p-110f;   // sv: value scale in use (8-bit)
    float o[HD / 8][4];
#pragma unroll
    for (int t = 0; t < HD / 8; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[t][e] = 0.f;

#pragma unroll 1
    for (int turn = 0; turn < n_turns; turn++) {
        const int j0 = p0 + (BA_WARPS * turn + warp) * G::PT;
        asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 2) : "memory");
        __syncwarp();
        fetch(turn + G::STAGES - 1);
        const uint8_t *kt = mine + (turn % G::STAGES) * G::STAGE, *vt = kt + G::KV;
        const float *ksc = reinterpret_cast<const float *>(kt + 2 * G::KV), *vsc = ksc + G::PT;
        float s[NT][2];   // log2 scores of row g, positions j0 + 8 t + 2 i + {0, 1}
        float vs[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            const int r = 8 * t + g;              // the key row this lane reads
            if constexpr (F32) {
                float cl[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < HD / 16; u++) {
                    const float4 k = *reinterpret_cast<const float4 *>(
                        kt + r * G::ROW + (((4 * u + i) ^ ba_turn<HD, FMT>(r)) << 4));
                    uint32_t h[4], l[4];
                    ba_split32(k.x, &h[0], &l[0]);
                    ba_split32(k.y, &h[1], &l[1]);
                    ba_split32(k.z, &h[2], &l[2]);
                    ba_split32(k.w, &h[3], &l[3]);
                    ba_mma_tf32(c, qa[2 * u], h[0], h[1]);
                    ba_mma_tf32(cl, qa[2 * u], l[0], l[1]);
                    ba_mma_tf32(c, qa[2 * u + 1], h[2], h[3]);
                    ba_mma_tf32(cl, qa[2 * u + 1], l[2], l[3]);
                }
                s[t][0] = (c[0] + ((c[2] + cl[0]) + cl[2])) * rowfac;
                s[t][1] = (c[1] + ((c[3] + cl[1]) + cl[3])) * rowfac;
            } else {
                uint32_t kw[HD / 16];
                if constexpr (HD == 128) {
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        *reinterpret_cast<uint4 *>(kw + 4 * e) = *reinterpret_cast<const uint4 *>(
                            kt + r * G::ROW + (((2 * i + e) ^ ba_turn<HD, FMT>(r)) << 4));
                } else if constexpr (HD == 64) {
                    *reinterpret_cast<uint4 *>(kw) =
                        *reinterpret_cast<const uint4 *>(kt + r * G::ROW + ((i ^ ba_turn<HD, FMT>(r)) << 4));
                } else {
                    *reinterpret_cast<uint2 *>(kw) = *reinterpret_cast<const uint2 *>(
                        kt + r * G::ROW + (((i >> 1) ^ ba_turn<HD, FMT>(r)) << 4) + 8 * (i & 1));
                }
                float d[4] = {0.f, 0.f, 0.f, 0.f};      // two chains
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {
                    const uint32_t w = FMT == KLLM_KV_I8 ? kw[ks] ^ 0x80808080u : kw[ks];
                    ba_mma_f16(ks & 1 ? d : c, qa[ks], ba_codes<FMT, 0>(w), ba_codes<FMT, 1>(w));
                }
                const float2 k2 = *reinterpret_cast<const float2 *>(ksc + 8 * t + 2 * i);
                const float2 v2 = *reinterpret_cast<const float2 *>(vsc + 8 * t + 2 * i);
                vs[t][0] = v2.x, vs[t][1] = v2.y;
                s[t][0] = ((c[0] + d[0]) + (c[2] + d[2])) * (k2.x * rowfac);
                s[t][1] = ((c[1] + d[1]) + (c[3] + d[3])) * (k2.y * rowfac);
            }
            if (j0 + 8 * t + 2 * i >= p1) s[t][0] = -INFINITY;
            if (j0 + 8 * t + 2 * i + 1 >= p1) s[t][1] = -INFINITY;
        }
        float mx = m_run, svx = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            mx = fmaxf(mx, fmaxf(s[t][0], s[t][1]));
            if constexpr (!F32) svx = fmaxf(svx, fmaxf(fabsf(vs[t][0]), fabsf(vs[t][1])));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        float corr = m_run == -INFINITY ? 0.f : exp2f(m_run - mx);
        float isv = 1.f;
        l_run *= corr;
        if constexpr (!F32) {
            svx = fmaxf(svx, __shfl_xor_sync(0xffffffffu, svx, 1));
            svx = fmaxf(svx, __shfl_xor_sync(0xffffffffu, svx, 2));
            const float svn = fmaxf(sv, ba_pow2(svx));   // the same in every lane of the warp
            corr *= sv / svn;
            sv = svn;
            isv = 0x1p14f / svn;
        }
        if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
            for (int t = 0; t < HD / 8; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[t][e] *= corr;
        }
        m_run = mx;
        const float mref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            s[t][0] = exp2f(s[t][0] - mref);
            s[t][1] = exp2f(s[t][1] - mref);
            l_run += s[t][0] + s[t][1];
        }
        // P.V
        if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                uint32_t pa[4];
                ba_split32(s[t][0], &pa[0], &pa[1]);
                ba_split32(s[t][1], &pa[2], &pa[3]);
                const int r = 8 * t + 2 * i;
#pragma unroll
                for (int u = 0; u < HD / 32; u++) {
                    const float4 v0 = *reinterpret_cast<const float4 *>(
                        vt + r * G::ROW + (((8 * u + g) ^ ba_turn<HD, FMT>(r)) << 4));
                    const float4 v1 = *reinterpret_cast<const float4 *>(
                        vt + (r + 1) * G::ROW + (((8 * u + g) ^ ba_turn<HD, FMT>(r + 1)) << 4));
                    const float x[4] = {v0.x, v0.y, v0.z, v0.w}, y[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t h0, l0, h1, l1;
                        ba_split32(x[e], &h0, &l0);
                        ba_split32(y[e], &h1, &l1);
                        ba_mma_tf32(o[4 * u + e], pa, l0, l1);
                        ba_mma_tf32(o[4 * u + e], pa, h0, h1);
                    }
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < NT; t += 2) {   // 16 positions
                uint32_t pa[4];
                ba_split(s[t][0] * (vs[t][0] * isv), s[t][1] * (vs[t][1] * isv), &pa[0], &pa[1]);
                ba_split(s[t + 1][0] * (vs[t + 1][0] * isv), s[t + 1][1] * (vs[t + 1][1] * isv),
                         &pa[2], &pa[3]);
                uint32_t vw[4][HD / 32];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int r = 8 * t + 2 * i + (e & 1) + 8 * (e >> 1);
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
                    ba_mma_f16(o[4 * w], pa, ba_codes<FMT, 0>(x01), ba_codes<FMT, 0>(y01));
                    ba_mma_f16(o[4 * w + 1], pa, ba_codes<FMT, 1>(x01), ba_codes<FMT, 1>(y01));
                    ba_mma_f16(o[4 * w + 2], pa, ba_codes<FMT, 0>(x23), ba_codes<FMT, 0>(y23));
                    ba_mma_f16(o[4 * w + 3], pa, ba_codes<FMT, 1>(x23), ba_codes<FMT, 1>(y23));
                }
            }
        }
        __syncwarp();      // the stage may be filled again
    }
    // join the four warps, in warp order, where the rings were
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float(*sm_o)[BA_ROWS][HD] = reinterpret_cast<float(*)[BA_ROWS][HD]>(ring);
    float(*sm_ml)[BA_ROWS][2] =
        reinterpret_cast<float(*)[BA_ROWS][2]>(ring + BA_WARPS * BA_ROWS * HD * sizeof(float));
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (i == 0) {
        sm_ml[warp][g][0] = m_run;
        sm_ml[warp][g][1] = l_run;
    }
    __syncthreads();
    float M = sm_ml[0][g][0];
#pragma unroll
    for (int w = 1; w < BA_WARPS; w++) M = fmaxf(M, sm_ml[w][g][0]);
    float f = m_run == -INFINITY ? 0.f : exp2f(m_run - M);
    if constexpr (!F32) f *= sv * 0x1p-14f;
#pragma unroll
    for (int t = 0; t < HD / 8; t++) {
        // dims of columns 2 i and 2 i + 1 of tile t
        const int d0 = F32 ? 32 * (t / 4) + 4 * (2 * i) + t % 4 : 2 * i * (HD / 8) + t;
        const int d1 = F32 ? d0 + 4 : d0 + HD / 8;
        sm_o[warp][g][d0] = (o[t][0] + o[t][2]) * f;
        sm_o[warp][g][d1] = (o[t][1] + o[t][3]) * f;
    }
    __syncthreads();
    const int parts = a.pre.parts + a.own.parts, pi = pre ? part : a.pre.parts + part;
    for (int x = tid; x < BA_ROWS * HD; x += BA_THREADS) {
        const int rr = x / HD, d = x % HD, R = tile * BA_ROWS + rr;
        if (R >= n_rows) break;
        const int rs = pre ? R / a.groups : seq, rh = kvh * a.groups + (pre ? R % a.groups : R);
        const long long out = ((long long)rs * a.nh + rh) * parts + pi;
        a.part_o[out * HD + d] = (sm_o[0][rr][d] + sm_o[1][rr][d]) + (sm_o[2][rr][d] + sm_o[3][rr][d]);
        if (d == 0) {
            float mm = sm_ml[0][rr][0], l = 0.f;
            for (int w = 1; w < BA_WARPS; w++) mm = fmaxf(mm, sm_ml[w][rr][0]);
            for (int w = 0; w < BA_WARPS; w++)
                if (sm_ml[w][rr][0] != -INFINITY) l += sm_ml[w][rr][1] * exp2f(sm_ml[w][rr][0] - mm);
            a.part_ml[2 * out] = mm;
            a.part_ml[2 * out + 1] = l;
        }
    }
    // done only when the launch before (the prefix's) is: the join waits for this one alone
    pdl_wait();
}

// Row (sequence, head) of the output from its parts, one warp per row.
template <int HD>
__global__ void __launch_bounds__(128)
k_ba_merge(const float *__restrict__ part_ml, const float *__restrict__ part_o, int parts_pre,
           int parts_own, int chunk_own, const int *__restrict__ own_len, int own_cap, int n_seq,
           int nh, float *__restrict__ out, long long out_stride, int terms, void *terms_out) {
    constexpr int VEC = HD / 32;
    const int R = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (R >= n_seq * nh) return;       // (the launch's completion needs no wait of this warp)
    const int seq = R / nh, h = R % nh, parts = parts_pre + parts_own;
    pdl_wait();
    if (own_len && own_len[seq] < 0) return;
    const int len = ba_len(own_len, own_cap, seq);
    const int n = parts_pre + (len > 0 ? (len + chunk_own - 1) / chunk_own : 0);
    const float *ml = part_ml + (long long)R * parts * 2, *po = part_o + (long long)R * parts * HD;
    float M = -INFINITY;
    for (int p = lane; p < n; p += 32) M = fmaxf(M, ml[2 * p]);
#pragma unroll
    for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    float L = 0.f, acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) acc[e] = 0.f;
    for (int p0 = 0; p0 < n; p0 += 32) {
        float w = 0.f, l = 0.f;
        if (p0 + lane < n) {
            const float m = ml[2 * (p0 + lane)];
            w = m == -INFINITY && M != -INFINITY ? 0.f : exp2f(m - M);
            l = ml[2 * (p0 + lane) + 1] * w;
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        L += l;
        const int c = min(32, n - p0);
#pragma unroll 4
        for (int p = 0; p < c; p++) {
            const float wp = __shfl_sync(0xffffffffu, w, p);
            float v[VEC];
            bd_load<VEC>(po + (long long)(p0 + p) * HD + VEC * lane, v);
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[e] = fmaf(wp, v[e], acc[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float v = n ? acc[e] / L : 0.f;
        if (terms_out)
            bd_emit(v, (size_t)R * HD + VEC * lane + e, terms, (size_t)n_seq * nh * HD, terms_out);
        else
            out[(long long)seq * out_stride + (long long)h * HD + VEC * lane + e] = v;
    }
}

// How a call is cut.
struct BaCut {
    int tiles_pre = 0, tiles_own = 0, own_cap = 0;
    int parts_pre = 0, chunk_pre = 0, parts_own = 0, chunk_own = 0;
    bool wide = false;      // the prefix by 128-row tiles
    size_t rows = 0, bytes = 0;
};

// `items` ranges of up to len positions into parts of at least 128 positions
// (a turn of each warp), as many as give every SM its two blocks twice over,
// and of at most 512 where the lengths are only bounds (blocks past a length
// end at once, the others even out).
void ba_split_range(long long items, int len, bool bound, int *parts, int *chunk) {
    const long long want = std::max<long long>(1, (148 * 4 + items - 1) / items);
    const long long most = (len + 127) / 128, least = bound ? (len + 511) / 512 : 1;
    const int n = (int)std::min(std::max(want, least), most);
    *chunk = ((len + n - 1) / n + 127) / 128 * 128;
    *parts = (len + *chunk - 1) / *chunk;
}

BaCut ba_cut(const kllm_batch_attn &a) {
    const kllm_kv_cache *c = a.prefix ? a.prefix : a.own;
    BaCut x;
    const int groups = a.n_heads / c->n_kv;
    x.own_cap = a.own ? std::min(a.max_len, a.own->max_pos) : 0;
    const int pre = a.prefix ? a.prefix_len : 0;
    if (pre > 0) {
        const long long rows = (long long)a.n_seq * groups;
        x.wide = rows >= 32 && pre >= 256;
        x.tiles_pre = (int)((rows + (x.wide ? BT_ROWS : BA_ROWS) - 1) / (x.wide ? BT_ROWS : BA_ROWS));
        const long long items = (long long)c->n_kv * x.tiles_pre;
        if (x.wide) {
            // one block an SM: as many parts as fill them once
            const int n = (int)std::min<long long>(std::max<long long>(148 / items, 1), (pre + 127) / 128);
            x.chunk_pre = ((pre + n - 1) / n + 127) / 128 * 128;
            x.parts_pre = (pre + x.chunk_pre - 1) / x.chunk_pre;
        } else {
            ba_split_range(items, pre, false, &x.parts_pre, &x.chunk_pre);
        }
    }
    if (x.own_cap > 0) {
        x.tiles_own = (groups + BA_ROWS - 1) / BA_ROWS;
        ba_split_range((long long)a.n_seq * c->n_kv * x.tiles_own, x.own_cap, true, &x.parts_own,
                       &x.chunk_own);
    }
    x.rows = (size_t)a.n_seq * a.n_heads;
    const size_t parts = x.parts_pre + x.parts_own;
    x.bytes = ((x.rows * parts * 2 * 4 + 15) / 16 * 16) + x.rows * parts * c->head_dim * 4 + 16;
    return x;
}

bool ba_ok(const char *who, const kllm_batch_attn *a) {
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
    return true;
}

// A kernel's shared-memory limit, raised once per device.
bool ba_prepare(const void *kernel, size_t smem) {
    static std::mutex mu;
    static std::set<std::pair<int, const void *>> done;
    int dev = 0;
    if (!KLLM_CUDA(cudaGetDevice(&dev))) return false;
    std::lock_guard<std::mutex> lk(mu);
    if (done.count({dev, kernel})) return true;
    if (!KLLM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)))
        return false;
    done.insert({dev, kernel});
    return true;
}

template <int HD, int FMT>
bool ba_launch(cudaStream_t s, const kllm_batch_attn &a, const BaCut &x, int terms, void *terms_out) {
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
    k.wide = x.wide;
    const long long pre_blocks = (long long)k.nkv * x.tiles_pre * x.parts_pre;
    const long long blocks = (x.wide ? 0 : pre_blocks) +
                             (long long)a.n_seq * k.nkv * x.tiles_own * x.parts_own;
    if (pre_blocks > 0x7fffffffll || blocks > 0x7fffffffll || x.rows > 0x7fffffffull) {
        set_error("kllm_batch_attention: %lld blocks", blocks);
        return false;
    }
    // each launch but the first may start while the one before drains; the
    // join waits for the parts' launch, which ends only when the prefix's has
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
        auto kernel = k_ba_prefix<HD, FMT>;
        constexpr size_t smem = bt_smem<HD, FMT>();
        if (!ba_prepare(reinterpret_cast<const void *>(kernel), smem) ||
            !launch(kernel, (unsigned)pre_blocks, BtGeom<HD, FMT>::THREADS, smem, k))
            return false;
    }
    if (blocks) {
        auto kernel = k_ba_part<HD, FMT>;
        constexpr size_t smem = BaRing<HD, FMT>::SMEM;
        if (!ba_prepare(reinterpret_cast<const void *>(kernel), smem) ||
            !launch(kernel, (unsigned)blocks, BA_THREADS, smem, k))
            return false;
    }
    if (!launch(k_ba_merge<HD>, (unsigned)((x.rows + 3) / 4), 128, 0, (const float *)k.part_ml,
                (const float *)k.part_o, x.parts_pre, x.parts_own, k.own.chunk, k.own_len, x.own_cap,
                a.n_seq, a.n_heads, a.out, a.out_stride, terms, terms_out))
        return false;
    return KLLM_CUDA(cudaGetLastError());
}

}  // namespace

bool batch_attention(cudaStream_t s, const kllm_batch_attn &a, int terms, void *terms_out) {
    const char *who = "kllm_batch_attention";
    if (!ba_ok(who, &a)) return false;
    if (!a.out && !terms_out) {
        set_error("%s: invalid arguments", who);
        return false;
    }
    const kllm_kv_cache *c = a.prefix ? a.prefix : a.own;
    if (!terms_out && a.n_seq > 1 && a.out_stride < (long long)a.n_heads * c->head_dim) {
        set_error("%s: out_stride %lld for %d heads of %d", who, a.out_stride, a.n_heads, c->head_dim);
        return false;
    }
    const BaCut x = ba_cut(a);
    if (!a.workspace || a.workspace_bytes < x.bytes || (reinterpret_cast<uintptr_t>(a.workspace) & 15)) {
        set_error("%s: %zu bytes of workspace on 16 bytes needed, %zu given", who, x.bytes,
                  a.workspace ? a.workspace_bytes : (size_t)0);
        return false;
    }
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return c->format == KLLM_KV_F32 ? ba_launch<HD, KLLM_KV_F32>(s, a, x, terms, terms_out)
             : c->format == KLLM_KV_I8  ? ba_launch<HD, KLLM_KV_I8>(s, a, x, terms, terms_out)
                                        : ba_launch<HD, KLLM_KV_E4M3>(s, a, x, terms, terms_out);
    };
    return c->head_dim == 32 ? go(std::integral_constant<int, 32>())
         : c->head_dim == 64 ? go(std::integral_constant<int, 64>())
                             : go(std::integral_constant<int, 128>());
}

}  // namespace kllm

using namespace kllm;

extern "C" size_t kllm_batch_attention_workspace(const kllm_batch_attn *a) {
    return ba_ok("kllm_batch_attention_workspace", a) ? ba_cut(*a).bytes : 0;
}

extern "C" int kllm_batch_attention(const kllm_batch_attn *a, void *stream) {
    if (!a) {
        set_error("kllm_batch_attention: invalid arguments");
        return -1;
    }
    return batch_attention((cudaStream_t)stream, *a, 0, nullptr) ? 0 : -1;
}
