// sample.cu -- one token per row of logits, drawn with a given uniform number
// under temperature, top-k, top-p and min-p (kllm_sample).
//
// The definition orders a row's tokens by (logit descending, index
// ascending) and keeps a prefix of that order; nothing here sorts.  The
// prefix is described by its last logit tau (as an order-preserving integer
// key) and how many of the tokens that equal tau it holds, and top-k and
// top-p both find it the same way: a histogram over 2048 ranges of the
// distance to the maximum, the range the boundary falls into, then
// histograms over that range's keys until one key is left (two more as a
// rule).  Weights are 2^-40 fixed point, w = rn(2^40 exp((x - max) / T)), so
// their sums are exact integers whatever the order of the additions: atomics
// and the split over blocks cannot change a result.  The draw runs over the
// kept weights in index order.
//
// A cluster of up to eight blocks takes a row, each a contiguous slice that
// it loads once into shared memory; maxima, histograms and sums meet through
// distributed shared memory.  Bound: the row's 4 vocab bytes; in practice
// the latency of the dependent passes over the slice.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

#include "rows.cuh"
#include "serve.cuh"

namespace kllm {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 2048, SA_CL = 8;
constexpr int SA_VOCAB = 1 << 22;                  // sums stay below 2^62
constexpr size_t SA_CACHE = 180 * 1024;            // slice bytes that are kept on chip

// Order-preserving integer of a logit; NaN counts as -infinity.
__device__ __forceinline__ uint32_t sa_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);   // one key for both zeros
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sa_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct SaShared {
    u64 hist[SA_BINS];           // this block's histogram
    u64 wsum[SA_WARPS];
    u64 seg_total[SA_CL];        // written by the blocks of the cluster
    u64 best[SA_CL];             // largest (key, ~index) of each slice
    u64 cand_before[SA_CL];
    int cand_bin[SA_CL];
    u64 mass[SA_CL];             // kept mass of each slice
    uint32_t klo[SA_CL], khi[SA_CL];
    int ties[SA_CL];
    int icut, token;
    uint32_t rlo, rhi;
    int wtie[SA_WARPS];
};

__device__ __forceinline__ u64 sa_warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The upper set of the order that is kept: keys above tau, and the first
// `ties` (in index order) of those that equal it.
struct SaKept {
    uint32_t tau;
    u64 ties;
};

struct SaRow {
    const float *src;       // the slice: shared memory, or the row in global memory
    const float *g;         // the slice in global memory
    int nz;
    long long plane;
    int n, first;           // tokens of the slice, index of its first
    bool cached;
    float m;                // the row's maximum
    double lt;              // log2(e) / T
    float binf;             // ranges per logit

    __device__ __forceinline__ float at(int i) const {
        if (cached || nz == 1) return src[i];
        return bd_sum(g, nz, plane, i);
    }
    // weight of a logit, 2^-40 fixed point
    __device__ __forceinline__ u64 weight(float x) const {
        if (x == m) return 1ull << 40;
        const double t = ((double)m - (double)x) * lt;
        if (!(t < 41.5)) return 0;
        return (u64)__double2ll_rn(exp2(40.0 - t));
    }
    // range of the distance to the maximum, SA_BINS where the weight is zero
    __device__ __forceinline__ int bin(float x) const {
        if (x == m) return 0;
        const float t = (m - x) * binf;
        return t < (float)SA_BINS ? (int)t : SA_BINS;
    }
};

// Finds the prefix of the order that a rule keeps, among the tokens of
// `in`: with MASS those whose mass before is < frac * (mass of `in`), else
// the first `count`.  All blocks of the cluster return the same.
template <bool MASS>
__device__ SaKept sa_select(cg::cluster_group &cl, SaShared &sh, const SaRow &row, SaKept in,
                            u64 count, double frac) {
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank(), tid = threadIdx.x;
    const int seg = SA_BINS / C;
    u64 above = 0, total = 0;
    uint32_t klo = 0, khi = 0;
    int shift = -1;                     // below 0: ranges of the distance
    for (int level = 0; level < 8; level++) {
        for (int b = tid; b < SA_BINS; b += SA_THREADS) sh.hist[b] = 0;
        if (tid == 0) sh.rlo = 0xffffffffu, sh.rhi = 0;
        __syncthreads();
        for (int i = tid; i < row.n; i += SA_THREADS) {
            const float x = row.at(i);
            const uint32_t k = sa_key(x);
            if (k <= in.tau) continue;      // tau's own ties are added once, below
            int b;
            if (shift < 0) {
                b = row.bin(x);
                if (b >= SA_BINS) continue;
            } else {
                if (k < klo || k > khi) continue;
                b = (int)((khi - k) >> shift);
            }
            const u64 w = MASS ? row.weight(x) : 1ull;
            if (w) atomicAdd(&sh.hist[b], w);
        }
        __syncthreads();
        // the kept ties at tau: block 0 adds them where they belong
        if (c == 0 && tid == 0 && in.tau) {
            const float x = sa_value(in.tau);
            const u64 w = MASS ? row.weight(x) * in.ties : in.ties;
            int b = -1;
            if (shift < 0) {
                b = row.bin(x);
            } else if (in.tau >= klo && in.tau <= khi) {
                b = (int)((khi - in.tau) >> shift);
            }
            if (b >= 0 && b < SA_BINS && w) sh.hist[b] += w;
        }
        cl.sync();
        // this block's segment of the ranges, summed over the cluster
        u64 mine[SA_BINS / SA_THREADS], s = 0;
        const int per = (seg + SA_THREADS - 1) / SA_THREADS;
#pragma unroll
        for (int e = 0; e < SA_BINS / SA_THREADS; e++) {
            mine[e] = 0;
            const int b = tid * per + e;
            if (e < per && b < seg)
                for (int k = 0; k < C; k++) mine[e] += cl.map_shared_rank(&sh, k)->hist[c * seg + b];
            s += mine[e];
        }
        // inclusive sums over the threads
        u64 inc = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, inc, o);
            if ((tid & 31) >= o) inc += v;
        }
        if ((tid & 31) == 31) sh.wsum[tid >> 5] = inc;
        __syncthreads();
        u64 before = inc - s;
        for (int w = 0; w < (tid >> 5); w++) before += sh.wsum[w];
        if (tid == SA_THREADS - 1)
            for (int k = 0; k < C; k++) cl.map_shared_rank(&sh, k)->seg_total[c] = before + s;
        if (tid == 0) sh.cand_bin[c] = -1;
        cl.sync();
        u64 base = above, all = 0;
        for (int k = 0; k < C; k++) {
            if (k < c) base += sh.seg_total[k];
            all += sh.seg_total[k];
        }
        if (level == 0) total = all;
        const double goal = frac * (double)total;
        // the last non-empty range that starts before the goal
        before += base;
        int last = -1;
        u64 last_before = 0;
#pragma unroll
        for (int e = 0; e < SA_BINS / SA_THREADS; e++) {
            const bool keep = MASS ? (double)before < goal || before == 0 : before < count;
            if (mine[e] && keep) last = c * seg + tid * per + e, last_before = before;
            before += mine[e];
        }
        // later threads hold later ranges: the largest wins
        const int wl = __reduce_max_sync(0xffffffffu, last);
        if (last >= 0 && last == wl) atomicMax(&sh.cand_bin[c], last);
        __syncthreads();
        if (last >= 0 && last == sh.cand_bin[c]) {
            for (int k = 0; k < C; k++)
                if (k != c) {
                    cl.map_shared_rank(&sh, k)->cand_bin[c] = last;
                    cl.map_shared_rank(&sh, k)->cand_before[c] = last_before;
                }
            sh.cand_before[c] = last_before;
        } else if (tid == 0 && sh.cand_bin[c] < 0) {
            for (int k = 0; k < C; k++)
                if (k != c) cl.map_shared_rank(&sh, k)->cand_bin[c] = -1;
        }
        cl.sync();
        int bin = -1;
        for (int k = 0; k < C; k++)
            if (sh.cand_bin[k] >= 0) bin = sh.cand_bin[k], above = sh.cand_before[k];
        if (bin < 0) return in;             // no weight at all beyond the first: nothing to cut
        if (shift == 0) {                   // one key left
            klo = khi = khi - (uint32_t)bin;
            break;
        }
        if (shift < 0) {
            // the keys of the range: from the data
            uint32_t lo = 0xffffffffu, hi = 0;
            for (int i = tid; i < row.n; i += SA_THREADS) {
                const float x = row.at(i);
                if (row.bin(x) != bin) continue;
                const uint32_t k = sa_key(x);
                if (k < in.tau) continue;
                lo = min(lo, k), hi = max(hi, k);
            }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            if ((tid & 31) == 0) {
                atomicMin(&sh.rlo, lo);
                atomicMax(&sh.rhi, hi);
            }
            __syncthreads();
            if (tid < C) {
                cl.map_shared_rank(&sh, tid)->klo[c] = sh.rlo;
                cl.map_shared_rank(&sh, tid)->khi[c] = sh.rhi;
            }
            cl.sync();
            klo = 0xffffffffu, khi = 0;
            for (int k = 0; k < C; k++) klo = min(klo, sh.klo[k]), khi = max(khi, sh.khi[k]);
        } else {
            const uint32_t top = khi - ((uint32_t)bin << shift);
            const uint32_t bottom = top - ((1u << shift) - 1u);
            klo = bottom > klo && bottom <= top ? bottom : klo;
            khi = top;
        }
        shift = 0;
        while (((khi - klo) >> shift) >= SA_BINS) shift++;
    }
    // the ties of the boundary key
    SaKept out;
    out.tau = klo;
    int n = 0;
    if (out.tau == in.tau) {
        out.ties = in.ties;
    } else {
        for (int i = tid; i < row.n; i += SA_THREADS) n += sa_key(row.at(i)) == out.tau;
        n = __reduce_add_sync(0xffffffffu, n);
        if ((tid & 31) == 0) sh.wtie[tid >> 5] = n;
        __syncthreads();
        if (tid < C) {
            int t = 0;
            for (int w = 0; w < SA_WARPS; w++) t += sh.wtie[w];
            cl.map_shared_rank(&sh, tid)->ties[c] = t;
        }
        cl.sync();
        u64 t = 0;
        for (int k = 0; k < C; k++) t += sh.ties[k];
        out.ties = t;
    }
    if constexpr (MASS) {
        const u64 w = row.weight(sa_value(out.tau));
        const double goal = frac * (double)total;
        // the first number of ties whose mass reaches the goal
        u64 lo = 1, hi = out.ties;
        while (lo < hi) {
            const u64 mid = (lo + hi) / 2;
            if ((double)(above + mid * w) < goal) lo = mid + 1;
            else hi = mid;
        }
        out.ties = lo;
    } else {
        out.ties = min(out.ties, count - above);
    }
    cl.sync();   // the shared words are free again
    return out;
}

__global__ void __launch_bounds__(SA_THREADS)
k_sample(const kllm_sample_rows a, int nz, long long plane, int per, int cached) {
    extern __shared__ float cache[];
    __shared__ SaShared sh;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), c = (int)cl.block_rank();
    const int r = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float *g = a.logits + (long long)r * a.row_stride;
    SaRow row;
    row.first = min(c * per, a.vocab);
    row.n = min(per, a.vocab - row.first);
    row.g = row.src = g + row.first;
    row.nz = nz;
    row.plane = plane;
    row.cached = false;
    // load the slice; its largest (key, first index)
    u64 best = 0;
    for (int i = tid; i < row.n; i += SA_THREADS) {
        const float x = row.at(i);
        if (cached) cache[i] = x;
        best = max(best, (u64)sa_key(x) << 32 | (0xffffffffu - (uint32_t)(row.first + i)));
    }
    if (cached) row.src = cache, row.cached = true;
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.wsum[warp] = best;
    __syncthreads();
    if (tid < C) {
        u64 b = 0;
        for (int w = 0; w < SA_WARPS; w++) b = max(b, sh.wsum[w]);
        cl.map_shared_rank(&sh, tid)->best[c] = b;
    }
    cl.sync();
    best = 0;
    for (int k = 0; k < C; k++) best = max(best, sh.best[k]);
    row.m = sa_value((uint32_t)(best >> 32));
    const int first_max = (int)(0xffffffffu - (uint32_t)best);
    const float T = a.temperature ? a.temperature[r] : 1.f;
    const bool greedy = T <= 0.f;
    if (greedy || row.m == -INFINITY) {
        if (c == 0 && tid == 0) {
            const float x0 = bd_sum(a.logits + (long long)r * a.row_stride, nz, plane, 0);
            a.tokens[r] = x0 != x0 || row.m == -INFINITY ? 0 : first_max;
        }
        cl.sync();
        return;
    }
    row.lt = 1.4426950408889634 / (double)(T == T ? T : 1.f);
    row.binf = (float)(row.lt * (SA_BINS / 41.5));
    SaKept kept{0u, ~0ull};     // everything (no token has key 0)
    const int k = a.top_k ? a.top_k[r] : 0;
    if (k > 0 && k < a.vocab) kept = sa_select<false>(cl, sh, row, kept, (u64)k, 0.0);
    const float p = a.top_p ? a.top_p[r] : 1.f;
    if (p < 1.f) kept = sa_select<true>(cl, sh, row, kept, 0, (double)p);
    // min-p: a bound on the weight
    u64 wmin = 1;
    if (a.min_p) {
        const float mp = a.min_p[r];
        if (mp > 0.f) wmin = max(1ull, (u64)ceil((double)fminf(mp, 1.f) * 0x1p40));
    }
    // contiguous parts of the slice per warp, in index order
    const int wper = ((row.n + SA_WARPS - 1) / SA_WARPS + 31) / 32 * 32;
    const int i0 = min(warp * wper, row.n), i1 = min(i0 + wper, row.n);
    // where the kept ties end: the index of the last of them
    int icut = 0x7fffffff;
    if (kept.tau) {
        int n = 0;
        for (int i = i0 + lane; i < i1; i += 32) n += sa_key(row.at(i)) == kept.tau;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) sh.wtie[warp] = n;
        if (tid == 0) sh.icut = 0x7fffffff;
        __syncthreads();
        if (tid < C) {
            int t = 0;
            for (int w = 0; w < SA_WARPS; w++) t += sh.wtie[w];
            cl.map_shared_rank(&sh, tid)->ties[c] = t;
        }
        cl.sync();
        u64 before = 0;
        for (int q = 0; q < c; q++) before += sh.ties[q];
        for (int w = 0; w < warp; w++) before += sh.wtie[w];
        if (before < kept.ties && before + n >= kept.ties) {
            // the (kept.ties - before)-th tie of this warp's part
            int need = (int)(kept.ties - before);
            for (int i = i0; i < i1; i += 32) {
                const bool t = i + lane < i1 && sa_key(row.at(i + lane)) == kept.tau;
                unsigned b = __ballot_sync(0xffffffffu, t);
                const int cnt = __popc(b);
                if (need <= cnt) {
                    for (; need > 1; need--) b &= b - 1;
                    if (lane < C) cl.map_shared_rank(&sh, lane)->icut = row.first + i + __ffs(b) - 1;
                    break;
                }
                need -= cnt;
            }
        }
        cl.sync();
        icut = sh.icut;
    }
    auto mass_of = [&](int i) -> u64 {
        const float x = row.at(i);
        const uint32_t key = sa_key(x);
        if (key < kept.tau || (key == kept.tau && row.first + i > icut)) return 0;
        const u64 w = row.weight(x);
        return w >= wmin ? w : 0;
    };
    u64 sum = 0;
    for (int i = i0 + lane; i < i1; i += 32) sum += mass_of(i);
    sum = sa_warp_sum(sum);
    if (lane == 0) sh.wsum[warp] = sum;
    __syncthreads();
    if (tid < C) {
        u64 t = 0;
        for (int w = 0; w < SA_WARPS; w++) t += sh.wsum[w];
        cl.map_shared_rank(&sh, tid)->mass[c] = t;
    }
    cl.sync();
    u64 total = 0, before = 0;
    for (int q = 0; q < C; q++) {
        if (q < c) before += sh.mass[q];
        total += sh.mass[q];
    }
    for (int w = 0; w < warp; w++) before += sh.wsum[w];
    float u = a.u[r];
    u = u > 0.f ? fminf(u, 1.f - 0x1p-24f) : 0.f;
    const double goal = (double)u * (double)total;
    if ((double)before <= goal && (double)(before + sum) > goal) {
        // the token lies in this warp's part
        for (int i = i0; i < i1; i += 32) {
            const u64 w = i + lane < i1 ? mass_of(i + lane) : 0;
            u64 inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, (double)(before + inc) > goal);
            if (hit) {
                if (lane == 0) a.tokens[r] = row.first + i + __ffs(hit) - 1;
                break;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    cl.sync();   // no block leaves while another may read its shared memory
}

}  // namespace

bool sample_rows(cudaStream_t s, const kllm_sample_rows &r, int nz, long long plane) {
    int C = SA_CL;
    while (C > 1 && r.vocab <= C * 2048) C /= 2;
    const int per = ((r.vocab + C - 1) / C + 3) / 4 * 4;
    const bool cached = (size_t)per * 4 <= SA_CACHE;
    const size_t smem = cached ? (size_t)per * 4 : 0;
    static bool ready[64] = {};
    static std::mutex mu;
    int dev = 0;
    if (!KLLM_CUDA(cudaGetDevice(&dev))) return false;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 64 || !ready[dev]) {
            if (!KLLM_CUDA(cudaFuncSetAttribute(k_sample, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                (int)SA_CACHE)))
                return false;
            if (dev < 64) ready[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(r.rows * C));
    cfg.blockDim = dim3(SA_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (!KLLM_CUDA(cudaLaunchKernelEx(&cfg, k_sample, r, nz, plane, per, (int)cached))) return false;
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
