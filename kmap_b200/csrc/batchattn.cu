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

namespace kllm {
namespace {

// tf32 terms: the upper 11 significand bits, and the rest (13 bits, of which
// the product takes 11)
__device__ __forceinline__ void ba_split32(float x, uint32_t *hi, uint32_t *lo) {
    *hi = __float_as_uint(x) & 0xffffe000u;
    *lo = __float_as_uint(x - __uint_as_float(*hi));
}

// One part of eight query rows of one kv head.  grid: the prefix's
// (kv head, row tile, part), then the sequences' (sequence, kv head, row tile,
// part); four warps take turns at blocks of 8 NT positions.
template <int HD, int FMT>
__global__ void __launch_bounds__(BA_THREADS, FMT == KLLM_KV_F32 ? 2 : 3)
k_ba_part(const BaArgs a) {
    constexpr bool F32 = FMT == KLLM_KV_F32;
    constexpr int NT = F32 ? 2 : 4;         // 8-position tiles per turn
    __shared__ float sm_o[BA_WARPS][BA_ROWS][HD];
    __shared__ float sm_ml[BA_WARPS][BA_ROWS][2];
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
    if (p0 >= p1) return;
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
    // cache rows of this (sequence, kv head)
    constexpr int ES = F32 ? 4 : 1;
    const long long at = (long long)seq * S.seq_stride + (long long)kvh * S.max_pos * HD;
    const uint8_t *kb = static_cast<const uint8_t *>(S.k) + at * ES;
    const uint8_t *vb = static_cast<const uint8_t *>(S.v) + at * ES;
    const float *ksc = F32 ? nullptr : S.ks + (long long)seq * S.scale_stride + (long long)kvh * S.max_pos;
    const float *vsc = F32 ? nullptr : S.vs + (long long)seq * S.scale_stride + (long long)kvh * S.max_pos;
    float m_run = -INFINITY, l_run = 0.f, sv = 0x1p-110f;   // sv: value scale in use (8-bit)
    float o[HD / 8][4];
#pragma unroll
    for (int t = 0; t < HD / 8; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[t][e] = 0.f;

    for (int j0 = p0 + warp * 8 * NT; j0 < p1; j0 += BA_WARPS * 8 * NT) {
        float s[NT][2];   // log2 scores of row g, positions j0 + 8 t + 2 i + {0, 1}
        float vs[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            const int jk = j0 + 8 * t + g;        // the key row this lane loads
            const bool in = jk < p1;
            if constexpr (F32) {
                float4 kw[HD / 16];
#pragma unroll
                for (int u = 0; u < HD / 16; u++)
                    ba_ld<16>(reinterpret_cast<uint32_t *>(&kw[u]),
                              kb + ((long long)jk * HD + 16 * u + 4 * i) * 4, in);
                float cl[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < HD / 16; u++) {
                    uint32_t h[4], l[4];
                    ba_split32(kw[u].x, &h[0], &l[0]);
                    ba_split32(kw[u].y, &h[1], &l[1]);
                    ba_split32(kw[u].z, &h[2], &l[2]);
                    ba_split32(kw[u].w, &h[3], &l[3]);
                    ba_mma_tf32(c, qa[2 * u], h[0], h[1]);
                    ba_mma_tf32(cl, qa[2 * u], l[0], l[1]);
                    ba_mma_tf32(c, qa[2 * u + 1], h[2], h[3]);
                    ba_mma_tf32(cl, qa[2 * u + 1], l[2], l[3]);
                }
                s[t][0] = (c[0] + ((c[2] + cl[0]) + cl[2])) * rowfac;
                s[t][1] = (c[1] + ((c[3] + cl[1]) + cl[3])) * rowfac;
            } else {
                uint32_t kw[HD / 16];
                ba_ld<HD / 4>(kw, kb + (long long)jk * HD + i * (HD / 4), in);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {
                    const uint32_t w = FMT == KLLM_KV_I8 ? kw[ks] ^ 0x80808080u : kw[ks];
                    ba_mma_f16(c, qa[ks], ba_codes<FMT, 0>(w), ba_codes<FMT, 1>(w));
                }
                const int j = j0 + 8 * t + 2 * i;
                const float k0 = j < p1 ? __ldg(ksc + j) : 0.f, k1 = j + 1 < p1 ? __ldg(ksc + j + 1) : 0.f;
                vs[t][0] = j < p1 ? __ldg(vsc + j) : 0.f;
                vs[t][1] = j + 1 < p1 ? __ldg(vsc + j + 1) : 0.f;
                s[t][0] = (c[0] + c[2]) * (k0 * rowfac);
                s[t][1] = (c[1] + c[3]) * (k1 * rowfac);
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
                const int jv = j0 + 8 * t + 2 * i;
#pragma unroll
                for (int u = 0; u < HD / 32; u++) {
                    float4 v0, v1;
                    ba_ld<16>(reinterpret_cast<uint32_t *>(&v0), vb + ((long long)jv * HD + 32 * u + 4 * g) * 4,
                              jv < p1);
                    ba_ld<16>(reinterpret_cast<uint32_t *>(&v1),
                              vb + ((long long)(jv + 1) * HD + 32 * u + 4 * g) * 4, jv + 1 < p1);
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
                const int jv = j0 + 8 * t + 2 * i;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = jv + (e & 1) + 8 * (e >> 1);
                    ba_ld<HD / 8>(vw[e], vb + (long long)j * HD + g * (HD / 8), j < p1);
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
    }
    // join the four warps, in warp order
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
}

// Row (sequence, head) of the output from its parts, one warp per row.
template <int HD>
__global__ void __launch_bounds__(128)
k_ba_merge(const float *__restrict__ part_ml, const float *__restrict__ part_o, int parts_pre,
           int parts_own, int chunk_own, const int *__restrict__ own_len, int own_cap, int n_seq,
           int nh, float *__restrict__ out, long long out_stride, int terms, void *terms_out) {
    constexpr int VEC = HD / 32;
    const int R = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (R >= n_seq * nh) return;
    const int seq = R / nh, h = R % nh, parts = parts_pre + parts_own;
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

// How a call is cut: enough blocks for three per SM, at least 128 positions each.
struct BaCut {
    int tiles_pre = 0, tiles_own = 0, own_cap = 0;
    int parts_pre = 0, chunk_pre = 0, parts_own = 0, chunk_own = 0;
    bool wide = false;      // the prefix by 128-row tiles
    size_t rows = 0, bytes = 0;
};

void ba_split_range(long long items, int len, int *parts, int *chunk) {
    const long long want = std::max<long long>(1, (148 * 3 + items - 1) / items);
    const long long most = (len + 127) / 128;
    const int n = (int)std::min(want, most);
    *chunk = ((len + n - 1) / n + 31) / 32 * 32;
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
            ba_split_range(items, pre, &x.parts_pre, &x.chunk_pre);
        }
    }
    if (x.own_cap > 0) {
        x.tiles_own = (groups + BA_ROWS - 1) / BA_ROWS;
        ba_split_range((long long)a.n_seq * c->n_kv * x.tiles_own, x.own_cap, &x.parts_own, &x.chunk_own);
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
    if (x.wide) {
        if (!ba_prepare(reinterpret_cast<const void *>(k_ba_prefix<HD, FMT>), bt_smem<HD, FMT>())) return false;
        k_ba_prefix<HD, FMT><<<(unsigned)pre_blocks, BtGeom<HD, FMT>::THREADS, bt_smem<HD, FMT>(), s>>>(k);
        g_launches++;
    }
    if (blocks) {
        k_ba_part<HD, FMT><<<(unsigned)blocks, BA_THREADS, 0, s>>>(k);
        g_launches++;
    }
    k_ba_merge<HD><<<(unsigned)((x.rows + 3) / 4), 128, 0, s>>>(
        k.part_ml, k.part_o, x.parts_pre, x.parts_own, k.own.chunk, k.own_len, x.own_cap, a.n_seq,
        a.n_heads, a.out, a.out_stride, terms, terms_out);
    g_launches++;
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
