// sample.cu -- one token per row of logits, drawn with a given uniform number
// under temperature, top-k, top-p and min-p (kllm_sample).
//
// The definition orders a row's tokens by (logit descending, index
// ascending) and keeps a prefix of that order; no row is sorted here.  Weights
// are 2^-40 fixed point, w = rn(2^40 exp((x - max) / T)), so their sums are
// exact integers whatever the order of the additions: atomics and the split
// over blocks cannot change a result.
//
// A cluster of up to eight blocks takes a row, each a contiguous slice that
// it loads once into shared memory, each warp a contiguous part of that.
//   1. the row's maximum;
//   2. a histogram of the row over 1024 ranges of the distance to the
//      maximum (each 3 % of weight wide): a count and, in the low bits, where
//      in the range its tokens lie, so that a range's mass is known to 0.2 %;
//   3. from it the range in which top-k, or top-p, ends;
//   4a. few tokens up to there (512): they go to one block, whose threads
//      take one each, and count the tokens and the mass before theirs, then
//      the kept mass up to theirs in index order: top-k, top-p, min-p and the
//      draw in two loops over the list;
//   4b. many: the prefix's last logit tau, and how many of the tokens that
//      equal it are kept.  One pass collects the tokens of the ranges that
//      the boundary can lie in and sums the weights before them; histograms
//      over the collected tokens' keys (order-preserving integers) close in
//      on one key; then the kept mass of every warp's part, and the draw by
//      the warp that holds it.  Passes take four tokens a lane at a time, for
//      the weights' chains to overlap, and skip what no lane wants.
// Histograms are summed over the cluster by every block for itself
// (distributed shared memory): one cluster barrier a step.
//
// Bound: a row's 4 vocab bytes are read once; past that, some 30 instructions
// a weight, a weight a token where all are needed (top-p alone, plain
// temperature) and another for the kept ones, between barriers that wait for a
// row's slowest warp: two blocks an SM use 43 % of the issue slots, and the
// barriers are the longest stall.  Few rows wait for the chain of dependent
// steps.  Measured: 1 row of 32000 tokens 17 us, 32 rows of 128256 (a mix of
// settings) 45 us, 128 rows of 128256 with top-p and many equal logits 192 to
// 208 us (0.3 TB/s, in step 4b).
#include <cooperative_groups.h>
#include <float.h>

#include <algorithm>
#include <mutex>

#include "rows.cuh"
#include "serve.cuh"

namespace kllm {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_CL = 8;
constexpr int SA_BINS = 1024, SA_FINE = 512;       // ranges of step 2; keys of step 4b
constexpr int SA_RPT = SA_BINS / SA_THREADS, SA_FPT = SA_FINE / SA_THREADS;   // of each per thread
constexpr int SA_LIST = 512;                       // most tokens of step 4a
constexpr int SA_LPT = SA_LIST / SA_THREADS;
constexpr int SA_NEAR = 2048;                      // most collected tokens of a block in step 4b
constexpr float SA_OCTAVES = 41.5f;                // weights below 2^-41 of the largest are zero
constexpr int SA_VOCAB = 1 << 22;                  // sums stay below 2^62
constexpr size_t SA_CACHE = 180 * 1024;            // slice bytes that are kept on chip
static_assert(SA_RPT == 2 && SA_FPT == 1, "loads of 8 bytes per thread");

// Order-preserving integer of a logit (no NaN); one for both zeros.
__device__ __forceinline__ uint32_t sa_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sa_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^-(j / 32) as fractions of 2^32
__constant__ uint32_t sa_tab[32] = {
    0xffffffffu, 0xfa83b2dbu, 0xf5257d15u, 0xefe4b99cu, 0xeac0c6e8u, 0xe5b906e7u, 0xe0ccdeecu,
    0xdbfbb798u, 0xd744fccbu, 0xd2a81d92u, 0xce248c15u, 0xc9b9bd86u, 0xc5672a11u, 0xc12c4ccau,
    0xbd08a39fu, 0xb8fbaf47u, 0xb504f334u, 0xb123f582u, 0xad583eeau, 0xa9a15ab5u, 0xa5fed6aau,
    0xa2704303u, 0x9ef53261u, 0x9b8d39bau, 0x9837f052u, 0x94f4efa9u, 0x91c3d374u, 0x8ea4398bu,
    0x8b95c1e4u, 0x88980e81u, 0x85aac368u, 0x82cd8699u};

struct SaShared {
    alignas(16) uint32_t coarse[SA_BINS];          // counts, and below them positions
    alignas(16) u64 fine[2][SA_FINE + 2];          // + the exact mass before the ranges
    union {
        alignas(16) ulonglong2 list[SA_LIST];      // 4a: (key, ~index) and weight
        int near[SA_NEAR];                         // 4b: places of the collected tokens
    };
    uint32_t tab[32];                              // 2^-(j / 32), 32-bit fractions
    float top[SA_CL];
    u64 mass[SA_CL], total[SA_CL];                 // written by the blocks of the cluster
    int ties[SA_CL];
    u64 wsum[SA_WARPS], wabove[SA_WARPS];
    double wlo[SA_WARPS], whi[SA_WARPS], goal_lo, goal_hi;
    int wtie[SA_WARPS];
    u64 sel_before, sel_amount;
    int sel_bin, sel_upto, lo_bin, hi_bin, icut, n_list, n_near;
};

__device__ __forceinline__ u64 sa_warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Exclusive sum over the block's threads, and the whole in *all.
template <class T>
__device__ __forceinline__ T sa_scan(T v, T *wsum, T *all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();                  // wsum is free
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    T before = inc - v, sum = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; w++) {
        const T t = wsum[w];
        if (w < warp) before += t;
        sum += t;
    }
    *all = sum;
    return before;
}

// Every block gets the sum over the cluster of what its warps' lanes 0 left in
// wsum; `to` are the cluster's words.
__device__ __forceinline__ u64 sa_cluster_sum(cg::cluster_group &cl, SaShared &sh,
                                              u64 (SaShared::*to)[SA_CL], const u64 *wsum, u64 extra) {
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank();
    __syncthreads();
    if (threadIdx.x < C) {
        u64 t = extra;
#pragma unroll
        for (int w = 0; w < SA_WARPS; w++) t += wsum[w];
        (cl.map_shared_rank(&sh, threadIdx.x)->*to)[c] = t;
    }
    cl.sync();
    u64 t = 0;
#pragma unroll
    for (int k = 0; k < SA_CL; k++)
        if (k < C) t += (sh.*to)[k];
    return t;
}

// The upper set of the order that is kept: logits above tau, and of those that
// equal it the first `ties` in index order (all of them unless `cut`).
struct SaKept {
    float tau;
    uint32_t key;
    u64 ties;
    bool cut;
};

// The row's weights: its maximum, log2(e) / T, units per logit (2^q_bits to a
// range of step 2).
struct SaScale {
    float m, unit;
    int q_bits;
    double md, mw, lt;      // the maximum, wide(it), log2(e) / T in wide's units
    const uint32_t *tab;    // sa_tab in shared memory

    // A float times 2^-896, exactly: its exponent and fraction bits in a double's place, where zero and
    // the subnormals are what they were too (a double's conversion from a float is slow).  -infinity
    // becomes -2^128 times that.
    static __device__ __forceinline__ double wide(float x) {
        const uint32_t b = __float_as_uint(x);
        return __hiloint2double((int)(((b & 0x7fffffffu) >> 3) | (b & 0x80000000u)), (int)(b << 29));
    }

    // Distance to the maximum in units.
    __device__ __forceinline__ float dist(float x) const { return (m - x) * unit; }
    __device__ __forceinline__ float units(int range) const { return (float)(range << q_bits); }

    // Weight of a logit, 2^-40 fixed point: t = (m - x) log2(e) / T in double precision, its whole
    // part n and a fraction of 32 bits by one addition (conversions from and to 64 bits are slow):
    // the sum of t and 1.5 * 2^20 has n in its upper word and the fraction in its lower.
    // 2^-fraction is a table's 2^-(j / 32), one word a bank, times 1 - z (c1 - z (c2 - z c3)), the
    // polynomial that meets 2^-z at the Chebyshev nodes of [0, 1/32), all as 32-bit fractions
    // (relative error below 2^-29); the shift by n and the rounding are one addition of 2^52.
    // No branch: several tokens' chains overlap.
    __device__ __forceinline__ u64 weight(float x) const {
        const double y = fma(mw - wide(x), lt, 0x1.8p20);
        const uint32_t n = min((uint32_t)__double2hiint(y) - 0x41380000u, 63u);
        const uint32_t lo = (uint32_t)__double2loint(y), z = lo & 0x07ffffffu, t = tab[lo >> 27];
        uint32_t q = 0x3d7f23e8u - __umulhi(z, 0x0e181d25u);
        q = 0xb17217d1u - __umulhi(z, q);
        const uint32_t f = t - __umulhi(t, __umulhi(z, q));
        const double v = __hiloint2double(0x43300000, (int)f) - 0x1p52;        // f as a double
        const double r = fma(v, __hiloint2double((int)((1031u - n) << 20), 0), 0x1p52);   // f 2^(8 - n)
        return (u64)(__double2hiint(r) & 0xfffff) << 32 | (uint32_t)__double2loint(r);
    }
};

// A block's slice of the row.
template <bool CACHED>
struct SaSlice {
    float *cache;           // the slice in shared memory (CACHED), -infinity behind its end
    const float *g;         // in global memory
    int nz;
    long long plane;
    int first, n;           // index of its first token, tokens
    int wper, i0;           // tokens per warp (a multiple of 128), this warp's first

    // a logit, NaN as -infinity, +infinity as the largest number
    static __device__ __forceinline__ float tame(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (CACHED) return cache[i];
        return i < n ? tame(bd_sum(g, nz, plane, i)) : -INFINITY;
    }
    __device__ __forceinline__ float4 at4(int i) const {
        if constexpr (CACHED) return *reinterpret_cast<const float4 *>(cache + i);
        return make_float4(at(i), at(i + 1), at(i + 2), at(i + 3));
    }
    // f(x, i, in) with four tokens in a row of this lane, the first one's place in the slice and
    // whether each is `wanted` (never -infinity), where any of the warp's is.
    template <class P, class F>
    __device__ __forceinline__ void each4(P &&wanted, F &&f) const {
        int i = i0 + 4 * (threadIdx.x & 31);
        const int end = min(i0 + wper, n);      // (the warp's: the same for its lanes)
#pragma unroll 1
        for (int j = i0; j < end; j += 128, i += 128) {
            const float4 v = at4(i);
            const float x[4] = {v.x, v.y, v.z, v.w};
            bool in[4];
#pragma unroll
            for (int e = 0; e < 4; e++) in[e] = wanted(x[e], i + e);
            if (__any_sync(0xffffffffu, (in[0] || in[1]) || (in[2] || in[3]))) f(x, i, in);
        }
    }
    // f(x, i) for the tokens of a lane's share of the warp's part, when each lane takes a run of
    // them (lanes start at different places of theirs: few bank conflicts)
    template <class F>
    __device__ __forceinline__ void run4(F &&f) const {
        const int lane = threadIdx.x & 31, len = wper / 128, base = i0 + lane * 4 * len;
        int q = lane % len;
#pragma unroll 2
        for (int e = 0; e < len; e++) {
            const float4 v = at4(base + 4 * q);
            f(v.x, base + 4 * q), f(v.y, base + 4 * q + 1), f(v.z, base + 4 * q + 2), f(v.w, base + 4 * q + 3);
            q = q + 1 < len ? q + 1 : 0;
        }
    }
};

// Places of the flagged ones of a warp's four tokens a lane in a block's list:
// one addition to its length for all of them.  Called by the whole warp.
__device__ __forceinline__ void sa_append(int *length, const bool (&in)[4], int (&at)[4]) {
    const int lane = threadIdx.x & 31;
    const unsigned below = (1u << lane) - 1u;
    unsigned b[4];
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        b[e] = __ballot_sync(0xffffffffu, in[e]);
        at[e] = n + __popc(b[e] & below);
        n += __popc(b[e]);
    }
    int first = 0;
    if (lane == 0) first = atomicAdd(length, n);
    first = __shfl_sync(0xffffffffu, first, 0);
#pragma unroll
    for (int e = 0; e < 4; e++) at[e] += first;
}

// What a pass over the collected tokens does: f(x, i) for each, or, where a
// block had more of them than it can hold, for every token of its slice that
// the ranges [flo, fhi) hold.
template <bool CACHED, class F>
__device__ __forceinline__ void sa_near(const SaShared &sh, const SaScale &sc, const SaSlice<CACHED> &sl,
                                        float flo, float fhi, F &&f) {
    const int n = sh.n_near;
    if (n <= SA_NEAR) {
        for (int q = threadIdx.x; q < n; q += SA_THREADS) {
            const int i = sh.near[q];
            f(sl.at(i), i);
        }
    } else {
        sl.each4(
            [&](float x, int) {
                const float t = sc.dist(x);
                return t < fhi && t >= flo;
            },
            [&](const float (&x)[4], int i, const bool (&in)[4]) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (in[e]) f(x[e], i + e);
            });
    }
}

// The boundary's key, among the tokens that `in` keeps (limited): with MASS
// that of the last token whose mass before is < frac times their whole mass,
// else of the one with `count` - 1 before it; it lies in ranges
// [lo_bin, hi_bin], the tokens themselves in those up to `last`.  `above` is
// the amount before the boundary's ranges (MASS: summed here, and left per
// warp in sh.wabove).
template <bool MASS, bool CACHED>
__device__ SaKept sa_narrow(cg::cluster_group &cl, SaShared &sh, const SaScale &sc,
                            const SaSlice<CACHED> &sl, const SaKept &in, bool limited, int lo_bin,
                            int hi_bin, int last, u64 above, u64 count, double frac, int &buf) {
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank(), tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    // the ranges' keys, a little to the safe side
    const double step = (double)(1 << sc.q_bits) / (double)sc.unit;
    const double xh = lo_bin ? sc.md - (double)lo_bin * step * (1 - 1e-6) : sc.md;
    const double xl = sc.md - (double)(hi_bin + 1) * step * (1 + 1e-6);
    uint32_t khi = sa_key(lo_bin ? fminf(__double2float_ru(xh), sc.m) : sc.m);
    uint32_t klo = sa_key(__double2float_rd(xl));
    const float flo = sc.units(lo_bin), fhi = sc.units(hi_bin + 1);
    const float tau = limited ? in.tau : -INFINITY;
    // collect (tau's own ties are added once, below)
    if (tid == 0) sh.n_near = 0;
    __syncthreads();
    u64 a = 0, all_mass = 0;
    const float fend = MASS ? sc.units(last + 1) : fhi;
    sl.each4(
        [&](float x, int) {
            const float t = sc.dist(x);
            return t < fend && (MASS || t >= flo) && x > tau;
        },
        [&](const float (&x)[4], int i, const bool (&in)[4]) {
            bool near[4];
            int at[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float t = sc.dist(x[e]);
                near[e] = in[e] && t >= flo && t < fhi;
                if (MASS) {
                    u64 w = sc.weight(x[e]);
                    if (!in[e]) w = 0;      // (-infinity's is not zero at every temperature)
                    all_mass += w;
                    if (t < flo) a += w;
                }
            }
            if (!__any_sync(0xffffffffu, (near[0] || near[1]) || (near[2] || near[3]))) return;
            sa_append(&sh.n_near, near, at);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (near[e] && at[e] < SA_NEAR) sh.near[at[e]] = i + e;
        });
    if (MASS) {
        a = sa_warp_sum(a);
        all_mass = sa_warp_sum(all_mass);
        if (lane == 0) sh.wabove[warp] = a, sh.wsum[warp] = all_mass;
    }
    double goal = 0;
    SaKept out;
    for (int level = 0; level < 6; level++) {
        int shift = 0;
        while (((khi - klo) >> shift) >= (uint32_t)SA_FINE) shift++;
        u64 *hist = sh.fine[buf];
        for (int b = tid; b < SA_FINE; b += SA_THREADS) hist[b] = 0;
        __syncthreads();
        sa_near(sh, sc, sl, flo, fhi, [&](float x, int) {
            const uint32_t k = sa_key(x);
            if (!(x > tau) || k < klo || k > khi) return;
            const u64 w = MASS ? sc.weight(x) : 1ull;
            if (w) atomicAdd(&hist[(khi - k) >> shift], w);
        });
        __syncthreads();
        if (tid == 0) {
            if (MASS && level == 0) {
                u64 t = 0, t2 = 0;
#pragma unroll
                for (int w = 0; w < SA_WARPS; w++) t += sh.wabove[w], t2 += sh.wsum[w];
                if (c == 0 && limited) t2 += sc.weight(in.tau) * in.ties;
                hist[SA_FINE] = t;
                hist[SA_FINE + 1] = t2;
            }
            // the kept ties at tau, once for the cluster
            if (c == 0 && limited) {
                const float t = sc.dist(in.tau);
                if (t >= flo && t < fhi && in.key >= klo && in.key <= khi)
                    hist[(khi - in.key) >> shift] += MASS ? sc.weight(in.tau) * in.ties : in.ties;
            }
        }
        cl.sync();
        u64 mine[SA_FPT] = {};
#pragma unroll
        for (int k = 0; k < SA_CL; k++)
            if (k < C) {
                mine[0] += cl.map_shared_rank(&sh, k)->fine[buf][tid];
            }
        if (MASS && level == 0) {
            u64 t = 0, t2 = 0;
            if (lane < C) {
                const u64 *h = cl.map_shared_rank(&sh, lane)->fine[buf];
                t = h[SA_FINE];
                t2 = h[SA_FINE + 1];
            }
            above = sa_warp_sum(t);
            goal = frac * (double)sa_warp_sum(t2);
        }
        buf ^= 1;
        u64 all;
        u64 before = above + sa_scan<u64>(mine[0], sh.wsum, &all);
        const u64 end = above + all;
        auto keep = [&](u64 b) { return MASS ? (double)b < goal || b == 0 : b < count; };
        // one thread: the last non-empty range that starts before the boundary
#pragma unroll
        for (int e = 0; e < SA_FPT; e++) {
            if (mine[e] && keep(before) && (before + mine[e] == end || !keep(before + mine[e]))) {
                sh.sel_bin = SA_FPT * tid + e;
                sh.sel_before = before;
                sh.sel_amount = mine[e];
            }
            before += mine[e];
        }
        __syncthreads();
        const uint32_t bin = (uint32_t)sh.sel_bin;
        above = sh.sel_before;
        const uint32_t top = khi - (bin << shift);
        if (shift == 0) {
            out.key = top;
            out.tau = sa_value(top);
            const u64 w = MASS ? sc.weight(out.tau) : 1ull, n = sh.sel_amount / (w ? w : 1ull);
            u64 lo = 1;
            if constexpr (MASS) {
                // the first number of ties whose mass reaches the goal
                u64 hi = n;
                while (lo < hi) {
                    const u64 mid = (lo + hi) / 2;
                    if ((double)(above + mid * w) < goal) lo = mid + 1;
                    else hi = mid;
                }
            } else {
                lo = min(n, count - above);
            }
            out.ties = lo;
            out.cut = lo < n || (limited && in.cut && out.key == in.key);
            break;
        }
        const uint32_t bottom = top - ((1u << shift) - 1u);
        if (bottom > klo && bottom <= top) klo = bottom;
        khi = top;
    }
    return out;
}

// Step 4a, in block 0: the n tokens of sh.list, SA_LPT per thread.  `whole`: the
// mass that top-p is a part of, 0: that of what top-k leaves of the list.
__device__ void sa_list(SaShared &sh, const SaScale &sc, int n, int k, float p, u64 whole, u64 wmin,
                        float u, int *token) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 id[SA_LPT], w[SA_LPT], before[SA_LPT];
    int rank[SA_LPT];
    bool keep[SA_LPT];
#pragma unroll
    for (int e = 0; e < SA_LPT; e++) {
        const int q = e * SA_THREADS + tid;
        id[e] = w[e] = before[e] = 0;
        rank[e] = 0;
        if (q < n) {
            id[e] = sh.list[q].x;
            w[e] = sc.weight(sa_value((uint32_t)(id[e] >> 32)));
            sh.list[q].y = w[e];
        }
    }
    __syncthreads();
    if (warp * 32 < n)
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const ulonglong2 t = sh.list[j];
#pragma unroll
            for (int e = 0; e < SA_LPT; e++)
                if (t.x > id[e]) before[e] += t.y, rank[e]++;
        }
    auto sum = [&](bool (&in)[SA_LPT]) {
        u64 v = 0;
#pragma unroll
        for (int e = 0; e < SA_LPT; e++) v += in[e] ? w[e] : 0;
        v = sa_warp_sum(v);
        __syncthreads();
        if (lane == 0) sh.wsum[warp] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < SA_WARPS; i++) t += sh.wsum[i];
        return t;
    };
#pragma unroll
    for (int e = 0; e < SA_LPT; e++) keep[e] = e * SA_THREADS + tid < n && (k <= 0 || rank[e] < k);
    if (p < 1.f) {
        const double goal = (double)p * (double)(whole ? whole : sum(keep));
#pragma unroll
        for (int e = 0; e < SA_LPT; e++) keep[e] = keep[e] && ((double)before[e] < goal || rank[e] == 0);
    }
#pragma unroll
    for (int e = 0; e < SA_LPT; e++) keep[e] = keep[e] && (w[e] >= wmin || rank[e] == 0);
    const double goal = (double)u * (double)sum(keep);
#pragma unroll
    for (int e = 0; e < SA_LPT; e++)
        if (e * SA_THREADS + tid < n) sh.list[e * SA_THREADS + tid].y = keep[e] ? w[e] : 0;
    __syncthreads();
    if (warp * 32 < n) {
        u64 to[SA_LPT] = {};       // kept mass of indexes up to this one: ~index from ~0 down
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const ulonglong2 t = sh.list[j];
#pragma unroll
            for (int e = 0; e < SA_LPT; e++)
                if ((uint32_t)t.x >= (uint32_t)id[e]) to[e] += t.y;
        }
#pragma unroll
        for (int e = 0; e < SA_LPT; e++)
            if (keep[e] && w[e] && (double)to[e] > goal && (double)(to[e] - w[e]) <= goal)
                *token = (int)(0xffffffffu - (uint32_t)id[e]);
    }
}

template <bool CACHED>
__global__ void __launch_bounds__(SA_THREADS, 2)
k_sample(const kllm_sample_rows a, int nz, long long plane, int per, int wper, int pos_bits,
         int q_bits, bool vec) {
    extern __shared__ __align__(16) float cache[];
    __shared__ SaShared sh;
    cg::cluster_group cl = cg::this_cluster();
    // (a block's shared memory is there for the others once it has started: waited for ahead of step 1's
    // first access)
    cl.barrier_arrive();
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank();
    const int r = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    SaSlice<CACHED> sl;
    sl.cache = cache;
    sl.first = min(c * per, a.vocab);
    sl.n = min(per, a.vocab - sl.first);
    sl.g = a.logits + (long long)r * a.row_stride + sl.first;
    sl.nz = nz;
    sl.plane = plane;
    sl.wper = wper;
    sl.i0 = warp * wper;
    const float T = a.temperature ? a.temperature[r] : 1.f;
    const int topk = a.top_k ? a.top_k[r] : 0;
    const float topp = a.top_p ? a.top_p[r] : 1.f;
    const float minp = a.min_p ? a.min_p[r] : 0.f;
    float u = a.u[r];
    u = u > 0.f ? fminf(u, 1.f - 0x1p-24f) : 0.f;

    // 1. load the slice; its largest
    float top = -INFINITY;
    if (tid == 0) sh.n_list = 0;
    if (tid < 32) sh.tab[tid] = sa_tab[tid];
    for (int b = tid; b < SA_BINS; b += SA_THREADS) sh.coarse[b] = 0;
#pragma unroll 4
    for (int j = 0; j < wper; j += 128) {
        const int i = sl.i0 + j + 4 * lane;
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (vec && i < sl.n) {      // (n is a multiple of four then)
            v = __ldg(reinterpret_cast<const float4 *>(sl.g + i));
        } else if (!vec) {
            if (i < sl.n) v.x = bd_sum(sl.g, nz, plane, i);
            if (i + 1 < sl.n) v.y = bd_sum(sl.g, nz, plane, i + 1);
            if (i + 2 < sl.n) v.z = bd_sum(sl.g, nz, plane, i + 2);
            if (i + 3 < sl.n) v.w = bd_sum(sl.g, nz, plane, i + 3);
        }
        v.x = sl.tame(v.x), v.y = sl.tame(v.y), v.z = sl.tame(v.z), v.w = sl.tame(v.w);
        if (CACHED) *reinterpret_cast<float4 *>(cache + i) = v;
        top = fmaxf(top, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sh.wlo[warp] = (double)top;
    __syncthreads();
    cl.barrier_wait();
    if (tid < C) {
        double b = sh.wlo[0];
#pragma unroll
        for (int w = 1; w < SA_WARPS; w++) b = fmax(b, sh.wlo[w]);
        cl.map_shared_rank(&sh, tid)->top[c] = (float)b;
    }
    cl.sync();
#pragma unroll
    for (int k = 0; k < SA_CL; k++)
        if (k < C) top = fmaxf(top, sh.top[k]);
    SaScale sc;
    sc.m = top;
    sc.tab = sh.tab;
    if (T <= 0.f || sc.m == -INFINITY) {
        // the first maximum
        int at = 0x7fffffff;
        sl.each4([&](float x, int i) { return x == top && i < sl.n; },
                 [&](const float (&)[4], int i, const bool (&in)[4]) {
#pragma unroll
                     for (int e = 0; e < 4; e++)
                         if (in[e]) at = min(at, sl.first + i + e);
                 });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) sh.wtie[warp] = at;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < SA_WARPS; w++) at = min(at, sh.wtie[w]);
            cl.map_shared_rank(&sh, 0)->ties[c] = at;
        }
        cl.sync();
        if (c == 0 && tid == 0) {
            for (int k = 0; k < C; k++) at = min(at, sh.ties[k]);
            const float x0 = bd_sum(a.logits + (long long)r * a.row_stride, nz, plane, 0);
            a.tokens[r] = x0 != x0 || top == -INFINITY ? 0 : at;
        }
        return;     // the last barrier is behind every remote access
    }
    sc.md = (double)sc.m;
    sc.mw = SaScale::wide(sc.m);
    const double lt = 1.4426950408889634 / (double)(T == T ? fminf(fmaxf(T, 1e-30f), 1e30f) : 1.f);
    sc.lt = lt * 0x1p896;
    sc.q_bits = q_bits;
    sc.unit = (float)(lt * (double)(SA_BINS << q_bits) / (double)SA_OCTAVES);
    const float f_all = sc.units(SA_BINS);      // weights are zero from here on
    // min-p: a bound on the weight, which the largest always meets
    u64 wmin = 1;
    if (minp > 0.f)
        wmin = min(max(1ull, (u64)ceil((double)fminf(minp, 1.f) * 0x1p40)), sc.weight(sc.m));
    const bool use_k = topk > 0 && topk < a.vocab, use_p = topp < 1.f;
    SaKept kept = {-INFINITY, 0, 0, false};
    bool above_known = false, limited = false;      // limited: top-k cuts
    float tau_k = -INFINITY;
    int buf = 0, p_lo = 0, p_hi = 0;
    if (use_k || use_p) {
        // 2. counts, and positions in units that cannot carry into them
        const uint32_t pos_mask = (1u << pos_bits) - 1u;
        const double Q = (double)(1 << q_bits);
        sl.each4([&](float x, int) { return sc.dist(x) < f_all; },
                 [&](const float (&x)[4], int, const bool (&in)[4]) {
#pragma unroll
                     for (int e = 0; e < 4; e++) {
                         const uint32_t t = (uint32_t)(int)sc.dist(x[e]);
                         if (in[e])
                             atomicAdd(&sh.coarse[t >> q_bits],
                                       (1u << pos_bits) + (t & ((1u << q_bits) - 1u)));
                     }
                 });
        cl.sync();
        uint32_t cnt[SA_RPT] = {}, pos[SA_RPT] = {};
#pragma unroll
        for (int k = 0; k < SA_CL; k++)
            if (k < C) {
                const uint2 v = reinterpret_cast<const uint2 *>(cl.map_shared_rank(&sh, k)->coarse)[tid];
                const uint32_t w[SA_RPT] = {v.x, v.y};
#pragma unroll
                for (int j = 0; j < SA_RPT; j++) cnt[j] += w[j] >> pos_bits, pos[j] += w[j] & pos_mask;
            }
        // 3. the last range that top-k leaves (with fewer tokens that carry
        // weight it cuts nothing)
        uint32_t all;
        uint32_t from[SA_RPT + 1];
        from[0] = sa_scan<uint32_t>(cnt[0] + cnt[1], reinterpret_cast<uint32_t *>(sh.wsum), &all);
#pragma unroll
        for (int j = 0; j < SA_RPT; j++) from[j + 1] = from[j] + cnt[j];
        int last = SA_BINS - 1, upto = (int)all;
        u64 k_before = 0;
        limited = use_k && all > (uint32_t)topk;
        if (limited) {
#pragma unroll
            for (int j = 0; j < SA_RPT; j++)
                if (from[j] < (uint32_t)topk && from[j + 1] >= (uint32_t)topk) {
                    sh.sel_bin = SA_RPT * tid + j;
                    sh.sel_before = from[j];
                    sh.sel_upto = (int)from[j + 1];
                }
            __syncthreads();
            last = sh.sel_bin;
            upto = sh.sel_upto;
            k_before = sh.sel_before;
        }
        p_hi = last;
        if (use_p) {
            // Bounds of the mass up to each range: a range's tokens weigh
            // e^(-d f) of its upper edge, f in [0, 1) their place in it and d its
            // width, 1 - d f <= e^(-d f) <= 1 - d f + d^2 / 2.
            constexpr double d = (double)SA_OCTAVES / SA_BINS * 0.6931471805599453;
            double lo[SA_RPT + 1], hi[SA_RPT + 1];
            lo[0] = hi[0] = 0;
#pragma unroll
            for (int j = 0; j < SA_RPT; j++) {
                const double edge = 0x1p40 * (double)exp2f(-(float)(SA_RPT * tid + j) * (SA_OCTAVES / SA_BINS));
                const double n = cnt[j], s = (double)pos[j] / Q;
                lo[j + 1] = lo[j] + edge * (1 - 1e-5) * (n * (1 - d / Q) - s * d) - n;
                hi[j + 1] = hi[j] + edge * (1 + 1e-5) * (n * (1 + d * d / 2) - s * d) + n;
            }
            double sum;
            const double blo = sa_scan<double>(lo[SA_RPT], sh.wlo, &sum), bhi = sa_scan<double>(hi[SA_RPT], sh.whi, &sum);
#pragma unroll
            for (int j = 0; j <= SA_RPT; j++) lo[j] += blo, hi[j] += bhi;
            if (tid == 0) sh.lo_bin = 0, sh.hi_bin = last;
#pragma unroll
            for (int j = 0; j < SA_RPT; j++)
                if (SA_RPT * tid + j == last) {
                    // what top-k leaves of the last range is anything from nothing to all
                    sh.goal_lo = (double)topp * (limited ? lo[j] : lo[j + 1]) * (1 - 1e-9);
                    sh.goal_hi = (double)topp * hi[j + 1] * (1 + 1e-9);
                }
            __syncthreads();
            const double goal_lo = topp > 0.f ? sh.goal_lo : 0.0, goal_hi = topp > 0.f ? sh.goal_hi : 0.0;
#pragma unroll
            for (int j = 0; j < SA_RPT; j++) {
                const int b = SA_RPT * tid + j;
                // the boundary lies in or behind the last range that surely starts before
                // the goal, and before the first that surely starts behind it
                if (b <= last && cnt[j] && hi[j] < goal_lo) atomicMax(&sh.lo_bin, b);
                if (b <= last && b > 0 && lo[j] > goal_hi) atomicMin(&sh.hi_bin, b - 1);
            }
            __syncthreads();
            p_lo = sh.lo_bin;
            p_hi = max(sh.hi_bin, p_lo);
            if (!limited) {
#pragma unroll
                for (int j = 0; j < SA_RPT; j++)
                    if (SA_RPT * tid + j == p_hi) sh.sel_upto = (int)from[j + 1];
                __syncthreads();
                upto = sh.sel_upto;
            }
        }
        // (top-p after top-k: its whole mass is that of all that top-k leaves)
        if (upto <= SA_LIST) {
            // 4a. the tokens up to the last range to block 0, whatever the order;
            // where top-k cuts nothing the whole mass beside them
            const bool mass = use_p && !limited;
            const float fhi = sc.units((mass ? p_hi : last) + 1), fend = mass ? f_all : fhi;
            u64 sum = 0;
            sl.each4([&](float x, int) { return sc.dist(x) < fend; },
                     [&](const float (&x)[4], int i, const bool (&in)[4]) {
                         bool near[4];
                         int at[4];
#pragma unroll
                         for (int e = 0; e < 4; e++) {
                             near[e] = in[e] && sc.dist(x[e]) < fhi;
                             if (mass && in[e]) sum += sc.weight(x[e]);
                         }
                         if (!__any_sync(0xffffffffu, near[0] || near[1] || near[2] || near[3])) return;
                         sa_append(&sh.n_list, near, at);
#pragma unroll
                         for (int e = 0; e < 4; e++)
                             if (near[e])
                                 sh.list[at[e]].x =
                                     (u64)sa_key(x[e]) << 32 | (0xffffffffu - (uint32_t)(sl.first + i + e));
                     });
            u64 total = 0;
            if (mass) {
                sum = sa_warp_sum(sum);
                if (lane == 0) sh.wabove[warp] = sum;
                total = sa_cluster_sum(cl, sh, &SaShared::total, sh.wabove, 0);
            }
            if (!mass) cl.sync();
            int n = 0;
            if (c == 0) {
                n = sh.n_list;
                for (int k = 1; k < C; k++) {
                    const SaShared *o = cl.map_shared_rank(&sh, k);
                    const int m = o->n_list;
                    for (int i = tid; i < m; i += SA_THREADS) sh.list[n + i].x = o->list[i].x;
                    n += m;
                }
            }
            cl.sync();      // the other blocks may leave
            if (c == 0)
                sa_list(sh, sc, n, limited ? topk : 0, use_p ? topp : 1.f, total, wmin, u, &a.tokens[r]);
            return;
        }
        // 4b. the boundary's key
        if (limited) {
            kept = sa_narrow<false>(cl, sh, sc, sl, kept, false, last, last, last, k_before, (u64)topk,
                                    0.0, buf);
            tau_k = kept.tau;
        }
        if (use_p) {
            kept = sa_narrow<true>(cl, sh, sc, sl, kept, limited, p_lo, p_hi, last, 0, 0, (double)topp, buf);
            above_known = wmin <= 1;
        }
    }
    // where the kept ties end: the index of the last of them
    // (where nothing cuts, tau is -infinity and none of those is kept)
    int icut = kept.tau == -INFINITY ? -1 : 0x7fffffff;
    if (kept.cut) {
        int n = 0;
        sl.each4([&](float x, int) { return x == kept.tau; },
                 [&](const float (&)[4], int, const bool (&in)[4]) {
                     n += in[0] + in[1] + in[2] + in[3];
                 });
        const int nw = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) sh.wtie[warp] = nw;
        __syncthreads();
        if (tid < C) {
            int t = 0;
#pragma unroll
            for (int w = 0; w < SA_WARPS; w++) t += sh.wtie[w];
            cl.map_shared_rank(&sh, tid)->ties[c] = t;
        }
        cl.sync();
        u64 before = 0;
        for (int q = 0; q < c; q++) before += sh.ties[q];
        for (int w = 0; w < warp; w++) before += sh.wtie[w];
        if (before < kept.ties && before + nw >= kept.ties) {
            // the (kept.ties - before)-th tie of this warp's part
            const int need = (int)(kept.ties - before);
            const int len = sl.wper / 32;
            int have = 0;
            sl.run4([&](float x, int) { have += x == kept.tau; });
            int upto = have;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int who = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
            int left = need - __shfl_sync(0xffffffffu, upto - have, who);
            for (int e = 0; e < len; e += 32) {
                const int i = sl.i0 + who * len + e + lane;
                unsigned b = __ballot_sync(0xffffffffu, e + lane < len && sl.at(i) == kept.tau);
                if (left <= __popc(b)) {
                    for (; left > 1; left--) b &= b - 1;
                    if (lane < C)
                        cl.map_shared_rank(&sh, lane)->icut = sl.first + sl.i0 + who * len + e + __ffs(b) - 1;
                    break;
                }
                left -= __popc(b);
            }
        }
        cl.sync();
        icut = sh.icut;
    }
    auto keeps = [&](float x, int i) {
        return x > kept.tau || (x == kept.tau && sl.first + i <= icut);
    };
    auto mass_of = [&](float x, int i) -> u64 {
        const u64 w = sc.weight(x);
        return w >= wmin && keeps(x, i) ? w : 0;
    };
    u64 sum;
    if (above_known) {
        // step 4b left the mass before its ranges; the collected tokens', and
        // those of top-k's own last logit where top-p stopped there
        __syncthreads();
        if (lane == 0) sh.wsum[warp] = sh.wabove[warp];
        __syncthreads();
        sa_near(sh, sc, sl, sc.units(p_lo), sc.units(p_hi + 1), [&](float x, int i) {
            if (x > tau_k && keeps(x, i)) atomicAdd(&sh.wsum[i / sl.wper], sc.weight(x));
        });
        if (limited && kept.tau <= tau_k)
            sl.each4([&](float x, int i) { return x == tau_k && keeps(x, i); },
                     [&](const float (&)[4], int, const bool (&in)[4]) {
                         atomicAdd(&sh.wsum[warp], (u64)(in[0] + in[1] + in[2] + in[3]) * sc.weight(tau_k));
                     });
        __syncthreads();
        sum = sh.wsum[warp];
    } else {
        sum = 0;
        sl.each4([&](float x, int i) { return keeps(x, i) && sc.dist(x) < f_all; },
                 [&](const float (&x)[4], int, const bool (&in)[4]) {
#pragma unroll
                     for (int e = 0; e < 4; e++) {
                         const u64 w = sc.weight(x[e]);
                         if (in[e] && w >= wmin) sum += w;
                     }
                 });
        sum = sa_warp_sum(sum);
    }
    __syncthreads();
    if (lane == 0) sh.wsum[warp] = sum;
    const u64 total = sa_cluster_sum(cl, sh, &SaShared::mass, sh.wsum, 0);
    u64 before = 0;
    for (int q = 0; q < c; q++) before += sh.mass[q];
    for (int w = 0; w < warp; w++) before += sh.wsum[w];
    const double goal = (double)u * (double)total;
    if ((double)before <= goal && (double)(before + sum) > goal) {
        // The token lies in this warp's part: each lane sums a run of tokens, then the run
        // that holds it is taken apart.
        const int len = sl.wper / 32;
        u64 part = 0;
        sl.run4([&](float x, int i) {
            if (keeps(x, i)) part += mass_of(x, i);
        });
        u64 inc = part;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, (double)(before + inc) > goal);
        const int who = __ffs(hit) - 1;
        before += __shfl_sync(0xffffffffu, inc - part, who);
        for (int e0 = 0; e0 < len; e0 += 32) {
            const int i = sl.i0 + who * len + e0 + lane;
            u64 w = 0;
            if (e0 + lane < len) {
                const float x = sl.at(i);
                if (keeps(x, i)) w = mass_of(x, i);
            }
            inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned at = __ballot_sync(0xffffffffu, (double)(before + inc) > goal);
            if (at) {
                if (lane == 0) a.tokens[r] = sl.first + sl.i0 + who * len + e0 + __ffs(at) - 1;
                break;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}

}  // namespace

bool sample_rows(cudaStream_t s, const kllm_sample_rows &r, int nz, long long plane) {
    // A row's blocks: at least 2048 tokens each (1 row of 1000 tokens: 13.2 us with one, 16.1 with eight;
    // of 16000: 19.5, 16.6 with two, 15.7 with four, 16.5 with eight), and fewer where all rows' are more
    // than one an SM, a block's fixed work being that of some 2000 tokens (128 rows of 32000: 81 us with
    // one, 38 with two, 47 with four, 68 with eight; 32 rows: 64, 35, 26, 29), but slices of 64 KB at
    // most, two blocks an SM (128 rows of 128256: 128 us with eight, 172 with four).
    int C = SA_CL;
    while (C > 1 && r.vocab <= C * 2048) C /= 2;
    auto cost = [&](int c) { return std::max(148ll, (long long)r.rows * c) * (2000 + r.vocab / c); };
    while (C > 1 && r.vocab / (C / 2) <= 16384 && cost(C / 2) < cost(C)) C /= 2;
    const int per = ((r.vocab + C - 1) / C + 3) / 4 * 4;
    const int wper = ((per + SA_WARPS - 1) / SA_WARPS + 127) / 128 * 128;
    const size_t slice = (size_t)wper * SA_WARPS * 4;
    const bool cached = slice <= SA_CACHE;
    // a range's word: a slice's count above the sum of its tokens' positions, q_bits each
    int pos_bits = 31, q_bits = 0;
    while ((1ll << (32 - pos_bits)) <= per) pos_bits--;
    while (((2ll << q_bits) - 1) * per < (1ll << pos_bits) && q_bits < 8) q_bits++;
    const bool vec = nz == 1 && r.vocab % 4 == 0 && (r.rows == 1 || r.row_stride % 4 == 0) &&
                     (reinterpret_cast<uintptr_t>(r.logits) & 15) == 0;
    static bool ready[64] = {};
    static std::mutex mu;
    int dev = 0;
    if (!KLLM_CUDA(cudaGetDevice(&dev))) return false;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 64 || !ready[dev]) {
            if (!KLLM_CUDA(cudaFuncSetAttribute(k_sample<true>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                (int)SA_CACHE)))
                return false;
            if (dev < 64) ready[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(r.rows * C));
    cfg.blockDim = dim3(SA_THREADS);
    cfg.dynamicSmemBytes = cached ? slice : 0;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (!KLLM_CUDA(cudaLaunchKernelEx(&cfg, cached ? k_sample<true> : k_sample<false>, r, nz, plane, per,
                                      wper, pos_bits, q_bits, vec))) return false;
    g_launches++;
    return KLLM_CUDA(cudaGetLastError());
}

}  // namespace kllm

using namespace kllm;

extern "C" int kllm_sample(const kllm_sample_rows *r, void *stream) {
    if (!r || r->rows < 0 || r->rows > (1 << 24) || r->vocab < 1 || !r->logits || !r->u || !r->tokens ||
        (r->rows > 1 && r->row_stride < r->vocab)) {
        set_error("kllm_sample: invalid arguments");
        return -1;
    }
    if (r->vocab > SA_VOCAB) {
        set_error("kllm_sample: %d tokens (at most %d)", r->vocab, SA_VOCAB);
        return -1;
    }
    if (r->rows == 0) return 0;
    return sample_rows((cudaStream_t)stream, *r, 1, 0) ? 0 : -1;
}
