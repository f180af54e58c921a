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
//      for top-p alone the exact whole mass beside it;
//   3. from it the range in which top-k, or top-p, ends;
//   4a. few tokens up to there (512): they go to one block, whose threads
//      take one each, and count the tokens and the mass before theirs, then
//      the kept mass up to theirs in index order: top-k, top-p, min-p and the
//      draw in two loops over the list;
//   4b. many: the prefix's last logit tau, and how many of the tokens that
//      equal it are kept, from histograms over the keys (order-preserving
//      integers) of the ranges that the boundary can lie in, until one key is
//      left; then the kept mass of every warp's part, and the draw by the
//      warp that holds it.  Each lane keeps a mask of its tokens up to the
//      boundary's range, so that these passes touch no others.
// Histograms are summed over the cluster by every block for itself
// (distributed shared memory): one cluster barrier a step.
//
// Bound: a row's 4 vocab bytes are read once; past that the weights take 15
// double-precision operations a token where all are needed (top-p alone, plain
// temperature), and few rows wait for the chain of dependent steps.
#include <cooperative_groups.h>

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
constexpr int SA_LIST = SA_THREADS;                // most tokens of step 4a
constexpr float SA_OCTAVES = 41.5f;                // weights below 2^-41 of the largest are zero
constexpr int SA_VOCAB = 1 << 22;                  // sums stay below 2^62
constexpr size_t SA_CACHE = 180 * 1024;            // slice bytes that are kept on chip
static_assert(SA_BINS == 2 * SA_THREADS && SA_FINE == SA_THREADS, "one thread per two ranges, per key");

// Order-preserving integer of a logit (no NaN); one for both zeros.
__device__ __forceinline__ uint32_t sa_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sa_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct SaShared {
    alignas(16) uint32_t coarse[SA_BINS];          // counts, and below them positions
    alignas(16) u64 fine[2][SA_FINE + 2];          // + the exact mass before the ranges
    alignas(16) ulonglong2 list[SA_LIST];          // (key, ~index) and weight
    u64 best[SA_CL], mass[SA_CL], total[SA_CL];    // written by the blocks of the cluster
    int ties[SA_CL];
    u64 wsum[SA_WARPS], wabove[SA_WARPS];
    double wlo[SA_WARPS], whi[SA_WARPS];
    int wtie[SA_WARPS];
    u64 sel_before, sel_amount;
    int sel_bin, sel_upto, lo_bin, hi_bin, icut, n_list;
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

// The row's weights: its maximum, log2(e) / T, ranges per logit.
struct SaScale {
    float m, binf;
    double md, lt;

    // Range of the distance to the maximum, as a number (no NaN unless x is
    // -infinity under T = infinity).
    __device__ __forceinline__ float range(float x) const { return x == m ? 0.f : (m - x) * binf; }

    // Weight of a logit, 2^-40 fixed point.  2^-t = 2^-n 2^f, n the integer next to t, with 2^f
    // on [-1/2, 1/2] as the polynomial of degree 9 that meets it at the Chebyshev nodes (relative
    // error 2^-45.6); both roundings to integers are additions of a power of two, since
    // conversions from and to 64 bits run at a quarter of the additions' rate.  No branch: several
    // tokens' chains overlap.
    __device__ __forceinline__ u64 weight(float x) const {
        // a normal float's bits as a double's; the others are converted
        const uint32_t b = __float_as_uint(x);
        double xd = __hiloint2double((int)((((b & 0x7fffffffu) >> 3) + 0x38000000u) | (b & 0x80000000u)),
                                     (int)(b << 29));
        if ((b & 0x7f800000u) == 0) xd = (double)x;
        const double t = (md - xd) * lt;
        const double magic = 0x1.8p52;
        const double y = t + magic;
        const double f = (y - magic) - t;
        double p = 1.0205905413765595794e-7;
        p = fma(p, f, 1.325964524488711024e-6);
        p = fma(p, f, 0.000015252672924850736404);
        p = fma(p, f, 0.00015403433751251008921);
        p = fma(p, f, 0.0013333558200794592645);
        p = fma(p, f, 0.0096181291939343133551);
        p = fma(p, f, 0.055504108664651672007);
        p = fma(p, f, 0.2402265069564033974);
        p = fma(p, f, 0.69314718055994615897);
        p = fma(p, f, 1.0000000000000134868);
        const int n = __double2loint(y);
        const double r = __hiloint2double(__double2hiint(p) + ((40 - n) << 20), __double2loint(p)) + 0x1p52;
        const u64 w = (u64)__double_as_longlong(r) & 0xfffffffffffffull;
        return x == m ? 1ull << 40 : t < (double)SA_OCTAVES && x != -INFINITY ? w : 0ull;
    }
};

// A block's slice of the row.
template <bool CACHED>
struct SaSlice {
    float *cache;           // the slice in shared memory (CACHED)
    const float *g;         // in global memory
    int nz;
    long long plane;
    int first;              // index of its first token
    int i0, i1, steps;      // this warp's part, and its 32-token steps
    int per_bit;            // steps a bit of a lane's mask stands for

    // a logit of the slice, NaN as -infinity
    __device__ __forceinline__ float at(int i) const {
        if constexpr (CACHED) return cache[i];
        const float x = bd_sum(g, nz, plane, i);
        return x != x ? -INFINITY : x;
    }
    // f(x, i) for this lane's tokens in the steps of the mask
    template <class F>
    __device__ __forceinline__ void each(uint32_t mask, F &&f) const {
        const int lane = threadIdx.x & 31;
        while (mask) {
            const int b = __ffs(mask) - 1;
            mask &= mask - 1;
            for (int j = b * per_bit; j < (b + 1) * per_bit; j++) {
                const int i = i0 + 32 * j + lane;
                if (i < i1) f(at(i), i);
            }
        }
    }
};

// Narrows the keys of ranges [lo_bin, hi_bin] until the boundary's key is
// found, among the tokens that `in` keeps (limited): with MASS the last token
// whose mass before is < goal, else the one with `count` - 1 before it.
// `above` is the amount before the ranges (MASS: found by the first pass, and
// left per warp in sh.wabove).
template <bool MASS, bool CACHED>
__device__ SaKept sa_narrow(cg::cluster_group &cl, SaShared &sh, const SaScale &sc,
                            const SaSlice<CACHED> &sl, uint32_t mask, const SaKept &in, bool limited,
                            int lo_bin, int hi_bin, u64 above, u64 count, double goal, int &buf) {
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank(), tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    // the ranges' keys, a little to the safe side
    const double step = 1.0 / (double)sc.binf;
    const double xh = lo_bin ? sc.md - (double)lo_bin * step * (1 - 1e-6) : sc.md;
    const double xl = sc.md - (double)(hi_bin + 1) * step * (1 + 1e-6);
    uint32_t khi = sa_key(lo_bin ? fminf(__double2float_ru(xh), sc.m) : sc.m);
    uint32_t klo = sa_key(__double2float_rd(xl));
    const float flo = (float)lo_bin, fhi = (float)(hi_bin + 1);
    const float tau = limited ? in.tau : -INFINITY;
    SaKept out;
    for (int level = 0; level < 6; level++) {
        int shift = 0;
        while (((khi - klo) >> shift) >= (uint32_t)SA_FINE) shift++;
        u64 *hist = sh.fine[buf];
        hist[tid] = 0;
        __syncthreads();
        u64 a = 0;
        sl.each(mask, [&](float x, int) {
            const float t = sc.range(x);
            // tau's own ties are added once, below
            if (!(t < fhi) || (limited && !(x > tau))) return;
            if (t < flo) {
                if (MASS && level == 0) a += sc.weight(x);
                return;
            }
            const uint32_t k = sa_key(x);
            if (k < klo || k > khi) return;
            const u64 w = MASS ? sc.weight(x) : 1ull;
            if (w) atomicAdd(&hist[(khi - k) >> shift], w);
        });
        if (MASS && level == 0) {
            a = sa_warp_sum(a);
            if (lane == 0) sh.wabove[warp] = a;
        }
        __syncthreads();
        if (tid == 0) {
            if (MASS && level == 0) {
                u64 t = 0;
#pragma unroll
                for (int w = 0; w < SA_WARPS; w++) t += sh.wabove[w];
                hist[SA_FINE] = t;
            }
            // the kept ties at tau, once for the cluster
            if (c == 0 && limited) {
                const float t = sc.range(in.tau);
                if (t >= flo && t < fhi && in.key >= klo && in.key <= khi)
                    hist[(khi - in.key) >> shift] += MASS ? sc.weight(in.tau) * in.ties : in.ties;
            }
        }
        cl.sync();
        u64 mine = 0, amass = 0;
#pragma unroll
        for (int k = 0; k < SA_CL; k++)
            if (k < C) mine += cl.map_shared_rank(&sh, k)->fine[buf][tid];
        if (MASS && level == 0) {
            if (lane < C) amass = cl.map_shared_rank(&sh, lane)->fine[buf][SA_FINE];
            above = sa_warp_sum(amass);
        }
        buf ^= 1;
        u64 all;
        const u64 before = above + sa_scan<u64>(mine, sh.wsum, &all), end = above + all;
        auto keep = [&](u64 b) { return MASS ? (double)b < goal || b == 0 : b < count; };
        // one thread: the last non-empty range that starts before the boundary
        if (mine && keep(before) && (before + mine == end || !keep(before + mine))) {
            sh.sel_bin = tid;
            sh.sel_before = before;
            sh.sel_amount = mine;
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

// Step 4a, in block 0: the n tokens of sh.list, one per thread.  `whole`: the
// mass that top-p is a part of, 0: that of what top-k leaves of the list.
__device__ void sa_list(SaShared &sh, const SaScale &sc, int n, int k, float p, u64 whole, u64 wmin,
                        float u, int *token) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 id = 0, w = 0, before = 0;
    int rank = 0;
    if (tid < n) {
        id = sh.list[tid].x;
        w = sc.weight(sa_value((uint32_t)(id >> 32)));
        sh.list[tid].y = w;
    }
    __syncthreads();
    if (warp * 32 < n)
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const ulonglong2 t = sh.list[j];
            if (t.x > id) before += t.y, rank++;
        }
    // (an id is 0 only past the list)
    bool keep = tid < n && (k <= 0 || rank < k);
    auto sum = [&](u64 v) {
        v = sa_warp_sum(v);
        __syncthreads();
        if (lane == 0) sh.wsum[warp] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < SA_WARPS; i++) t += sh.wsum[i];
        return t;
    };
    if (p < 1.f) {
        const double goal = (double)p * (double)(whole ? whole : sum(keep ? w : 0));
        keep = keep && ((double)before < goal || rank == 0);
    }
    keep = keep && (w >= wmin || rank == 0);
    const double goal = (double)u * (double)sum(keep ? w : 0);
    if (tid < n) sh.list[tid].y = keep ? w : 0;
    __syncthreads();
    if (warp * 32 < n) {
        u64 to = 0;       // kept mass of indexes up to this one: ~index from ~0 down
        const uint32_t mine = (uint32_t)id;
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const ulonglong2 t = sh.list[j];
            if ((uint32_t)t.x >= mine) to += t.y;
        }
        if (keep && w && (double)to > goal && (double)(to - w) <= goal)
            *token = (int)(0xffffffffu - mine);
    }
}

template <bool CACHED>
__global__ void __launch_bounds__(SA_THREADS, 2)
k_sample(const kllm_sample_rows a, int nz, long long plane, int per) {
    extern __shared__ float cache[];
    __shared__ SaShared sh;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank();
    const int r = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    SaSlice<CACHED> sl;
    sl.cache = cache;
    sl.first = min(c * per, a.vocab);
    const int n_slice = min(per, a.vocab - sl.first);
    sl.g = a.logits + (long long)r * a.row_stride + sl.first;
    sl.nz = nz;
    sl.plane = plane;
    const int wper = ((n_slice + SA_WARPS - 1) / SA_WARPS + 31) / 32 * 32;
    sl.i0 = min(warp * wper, n_slice);
    sl.i1 = min(sl.i0 + wper, n_slice);
    sl.steps = (sl.i1 - sl.i0 + 31) / 32;
    sl.per_bit = (wper / 32 + 31) / 32;
    const float T = a.temperature ? a.temperature[r] : 1.f;
    const int topk = a.top_k ? a.top_k[r] : 0;
    const float topp = a.top_p ? a.top_p[r] : 1.f;
    const float minp = a.min_p ? a.min_p[r] : 0.f;
    float u = a.u[r];
    u = u > 0.f ? fminf(u, 1.f - 0x1p-24f) : 0.f;

    // 1. load the slice; its largest (key, first index)
    u64 best = 0;
    if (tid == 0) sh.n_list = 0;
    for (int b = tid; b < SA_BINS; b += SA_THREADS) sh.coarse[b] = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < sl.steps; j0 += 8) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = sl.i0 + 32 * (j0 + e) + lane;
            x[e] = -INFINITY;
            if (i < sl.i1) x[e] = nz == 1 ? __ldg(sl.g + i) : bd_sum(sl.g, nz, plane, i);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = sl.i0 + 32 * (j0 + e) + lane;
            if (i >= sl.i1) continue;
            if (x[e] != x[e]) x[e] = -INFINITY;
            if (CACHED) cache[i] = x[e];
            best = max(best, (u64)sa_key(x[e]) << 32 | (0xffffffffu - (uint32_t)(sl.first + i)));
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.wsum[warp] = best;
    __syncthreads();
    if (tid < C) {
        u64 b = 0;
#pragma unroll
        for (int w = 0; w < SA_WARPS; w++) b = max(b, sh.wsum[w]);
        cl.map_shared_rank(&sh, tid)->best[c] = b;
    }
    cl.sync();
    best = 0;
#pragma unroll
    for (int k = 0; k < SA_CL; k++)
        if (k < C) best = max(best, sh.best[k]);
    SaScale sc;
    sc.m = sa_value((uint32_t)(best >> 32));
    if (T <= 0.f || sc.m == -INFINITY) {
        if (c == 0 && tid == 0) {
            const float x0 = bd_sum(a.logits + (long long)r * a.row_stride, nz, plane, 0);
            a.tokens[r] = x0 != x0 || sc.m == -INFINITY ? 0 : (int)(0xffffffffu - (uint32_t)best);
        }
        return;     // the last barrier is behind every remote access
    }
    sc.md = (double)sc.m;
    sc.lt = 1.4426950408889634 / (double)(T == T ? T : 1.f);
    sc.binf = (float)(sc.lt * ((double)SA_BINS / SA_OCTAVES));
    // min-p: a bound on the weight
    u64 wmin = 1;
    if (minp > 0.f) wmin = max(1ull, (u64)ceil((double)fminf(minp, 1.f) * 0x1p40));
    const bool use_k = topk > 0 && topk < a.vocab, use_p = topp < 1.f;
    SaKept kept = {-INFINITY, 0, 0, false};
    uint32_t mask = sl.steps ? 0xffffffffu >> (32 - (sl.steps + sl.per_bit - 1) / sl.per_bit) : 0u;
    bool above_known = false;
    int buf = 0, p_lo = 0;
    if (use_k || use_p) {
        // 2. counts, and positions in units that cannot carry into them
        int bits = 32;
        while (bits > 1 && (1u << (bits - 1)) > (uint32_t)per) bits--;     // 2^bits > per
        const int pos_bits = 32 - bits;
        const uint32_t pos_mask = (1u << pos_bits) - 1u, Q = max(pos_mask / (uint32_t)per, 1u);
        const bool mass = use_p && !use_k;
        u64 sum = 0;
#pragma unroll 1
        for (int j0 = 0; j0 < sl.steps; j0 += 4) {
            float x[4], t[4];
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = sl.i0 + 32 * (j0 + e) + lane;
                x[e] = i < sl.i1 ? sl.at(i) : -INFINITY;
                t[e] = sc.range(x[e]);
                any = any || t[e] < (float)SA_BINS;
                if (x[e] > -INFINITY && t[e] < (float)SA_BINS) {
                    const int b = (int)t[e];
                    atomicAdd(&sh.coarse[b],
                              (1u << pos_bits) + (uint32_t)((t[e] - (float)b) * (float)Q));
                }
            }
            if (mass && __any_sync(0xffffffffu, any))
                sum += (sc.weight(x[0]) + sc.weight(x[1])) + (sc.weight(x[2]) + sc.weight(x[3]));
        }
        u64 total = 0;
        if (mass) {
            sum = sa_warp_sum(sum);
            if (lane == 0) sh.wabove[warp] = sum;
            total = sa_cluster_sum(cl, sh, &SaShared::total, sh.wabove, 0);
        } else {
            cl.sync();
        }
        uint32_t cnt[2] = {}, pos[2] = {};
#pragma unroll
        for (int k = 0; k < SA_CL; k++)
            if (k < C) {
                const uint2 v = reinterpret_cast<const uint2 *>(cl.map_shared_rank(&sh, k)->coarse)[tid];
                cnt[0] += v.x >> pos_bits, pos[0] += v.x & pos_mask;
                cnt[1] += v.y >> pos_bits, pos[1] += v.y & pos_mask;
            }
        // 3. the last range that top-k leaves (with fewer tokens that carry
        // weight it cuts nothing)
        uint32_t all;
        const uint32_t first = sa_scan<uint32_t>(cnt[0] + cnt[1], reinterpret_cast<uint32_t *>(sh.wsum), &all);
        const uint32_t from[3] = {first, first + cnt[0], first + cnt[0] + cnt[1]};
        int last = SA_BINS - 1, upto = (int)all;
        const bool limited = use_k && all > (uint32_t)topk;
        if (limited) {
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (from[j] < (uint32_t)topk && from[j + 1] >= (uint32_t)topk) {
                    sh.sel_bin = 2 * tid + j;
                    sh.sel_before = from[j];
                    sh.sel_upto = (int)from[j + 1];
                }
            __syncthreads();
            last = sh.sel_bin;
            upto = sh.sel_upto;
        }
        // bounds of the mass before each range: a range's tokens weigh
        // e^(-d f) of its upper edge, f in [0, 1) their place in it and d its
        // width, 1 - d f <= e^(-d f) <= 1 - d f + d^2 / 2
        int p_hi = last;
        double goal = 0;
        auto bracket = [&]() {
            goal = (double)topp * (double)total;
            constexpr double d = (double)SA_OCTAVES / SA_BINS * 0.6931471805599453;
            double lo[2], hi[2], slo = 0, shi = 0;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const double edge = 0x1p40 * (double)exp2f(-(float)(2 * tid + j) * (SA_OCTAVES / SA_BINS));
                const double n = cnt[j], s = (double)pos[j] / Q;
                lo[j] = slo, hi[j] = shi;        // before range j, within the thread
                slo += edge * (1 - 1e-5) * (n * (1 - d / Q) - s * d) - n;
                shi += edge * (1 + 1e-5) * (n * (1 + d * d / 2) - s * d) + n;
            }
            double sum;
            const double blo = sa_scan<double>(slo, sh.wlo, &sum), bhi = sa_scan<double>(shi, sh.whi, &sum);
            if (tid == 0) sh.lo_bin = 0, sh.hi_bin = last;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int b = 2 * tid + j;
                // the boundary lies in or behind the last range that surely starts before
                // the goal, and before the first that surely starts behind it
                if (b <= last && cnt[j] && bhi + hi[j] < goal * (1 - 1e-9)) atomicMax(&sh.lo_bin, b);
                if (b <= last && b > 0 && blo + lo[j] > goal * (1 + 1e-9)) atomicMin(&sh.hi_bin, b - 1);
            }
            __syncthreads();
            p_lo = sh.lo_bin;
            p_hi = max(sh.hi_bin, p_lo);
            if (2 * tid == p_hi) sh.sel_upto = (int)from[1];
            if (2 * tid + 1 == p_hi) sh.sel_upto = (int)from[2];
            __syncthreads();
            upto = min(upto, sh.sel_upto);
        };
        // top-p alone: nothing behind its own ranges is looked at again (top-p
        // after top-k: its whole mass has still to be summed)
        if (mass) bracket();
        // the lanes' tokens up to the last range
        {
            const float fhi = (float)((mass ? p_hi : last) + 1);
            uint32_t mk = 0;
#pragma unroll 4
            for (int j = 0; j < sl.steps; j++) {
                const int i = sl.i0 + 32 * j + lane;
                const float x = i < sl.i1 ? sl.at(i) : -INFINITY;
                if (x > -INFINITY && sc.range(x) < fhi) mk |= 1u << (sl.per_bit == 1 ? j : j / sl.per_bit);
            }
            mask = mk;
            if (upto <= SA_LIST) {
                // 4a. to block 0, whatever the order
                sl.each(mask, [&](float x, int i) {
                    if (x > -INFINITY && sc.range(x) < fhi)
                        sh.list[atomicAdd(&sh.n_list, 1)].x =
                            (u64)sa_key(x) << 32 | (0xffffffffu - (uint32_t)(sl.first + i));
                });
                cl.sync();
                int n = 0, have = 0;
                if (c == 0) {
                    have = sh.n_list;
                    n = have;
                    for (int k = 1; k < C; k++) {
                        const SaShared *o = cl.map_shared_rank(&sh, k);
                        const int m = o->n_list;
                        for (int i = tid; i < m; i += SA_THREADS) sh.list[n + i].x = o->list[i].x;
                        n += m;
                    }
                }
                cl.sync();      // the other blocks may leave
                if (c == 0)
                    sa_list(sh, sc, n, limited ? topk : 0, use_p ? topp : 1.f, total, wmin, u,
                            &a.tokens[r]);
                return;
            }
        }
        // 4b. the boundary's key
        if (limited) {
            kept = sa_narrow<false>(cl, sh, sc, sl, mask, kept, false, last, last, sh.sel_before,
                                    (u64)topk, 0.0, buf);
        }
        if (use_p) {
            if (!mass) {
                // the exact mass of what top-k leaves
                u64 t = 0;
                sl.each(mask, [&](float x, int) {
                    if (x > kept.tau) t += sc.weight(x);
                });
                t = sa_warp_sum(t);
                if (lane == 0) sh.wabove[warp] = t;
                const u64 extra = c == 0 && limited ? sc.weight(kept.tau) * kept.ties : 0ull;
                total = sa_cluster_sum(cl, sh, &SaShared::total, sh.wabove, extra);
                bracket();
            }
            kept = sa_narrow<true>(cl, sh, sc, sl, mask, kept, limited, p_lo, p_hi, 0, 0, goal, buf);
            above_known = wmin <= 1;
        }
    }
    // where the kept ties end: the index of the last of them
    int icut = 0x7fffffff;
    if (kept.cut) {
        int n = 0;
        sl.each(mask, [&](float x, int) { n += x == kept.tau; });
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
            int need = (int)(kept.ties - before);
#pragma unroll 4
            for (int j = 0; j < sl.steps; j++) {
                const int i = sl.i0 + 32 * j + lane;
                unsigned b = __ballot_sync(0xffffffffu, i < sl.i1 && sl.at(i) == kept.tau);
                const int cnt = __popc(b);
                if (need > 0 && need <= cnt) {
                    for (int k = need; k > 1; k--) b &= b - 1;
                    if (lane < C)
                        cl.map_shared_rank(&sh, lane)->icut = sl.first + sl.i0 + 32 * j + __ffs(b) - 1;
                }
                need -= cnt;
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
    u64 sum = 0;
    if (above_known) {      // the mass before step 4b's ranges is there
        const float flo = (float)p_lo;
        sl.each(mask, [&](float x, int i) {
            if (keeps(x, i) && !(sc.range(x) < flo)) sum += sc.weight(x);
        });
        sum = sa_warp_sum(sum) + sh.wabove[warp];
    } else if (use_k || use_p) {
        sl.each(mask, [&](float x, int i) {
            if (keeps(x, i)) sum += mass_of(x, i);
        });
        sum = sa_warp_sum(sum);
    } else {
#pragma unroll 1
        for (int j0 = 0; j0 < sl.steps; j0 += 4) {
            float x[4];
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = sl.i0 + 32 * (j0 + e) + lane;
                x[e] = i < sl.i1 ? sl.at(i) : -INFINITY;
                any = any || sc.range(x[e]) < (float)SA_BINS;
            }
            if (__any_sync(0xffffffffu, any))
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u64 w = sc.weight(x[e]);
                    sum += w >= wmin ? w : 0;
                }
        }
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
        // The token lies in this warp's part: each lane sums `steps` tokens in
        // a row (read from a place that turns with the lane: no two on one
        // bank), then the lane that holds it is taken apart.
        const int len = sl.steps, base = sl.i0 + lane * len;
        u64 part = 0;
#pragma unroll 4
        for (int e = 0; e < len; e++) {
            const int q = e + lane % len, i = base + (q < len ? q : q - len);
            if (i < sl.i1) {
                const float x = sl.at(i);
                if (keeps(x, i)) part += mass_of(x, i);
            }
        }
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
            if (e0 + lane < len && i < sl.i1) {
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
    int C = SA_CL;
    while (C > 1 && r.vocab <= C * 2048) C /= 2;
    const int per = ((r.vocab + C - 1) / C + 3) / 4 * 4;
    const bool cached = (size_t)per * 4 <= SA_CACHE;
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
    cfg.dynamicSmemBytes = cached ? (size_t)per * 4 : 0;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (!KLLM_CUDA(cudaLaunchKernelEx(&cfg, cached ? k_sample<true> : k_sample<false>, r, nz, plane, per))) return false;
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
