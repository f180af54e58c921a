// kvcache.cu -- the key/value cache that is quantised as it is written
// (kllm_kv_append) and read back as fp32 (kllm_kv_read).
//
// A row is the head_dim values of one (position, head).  With a = max |x_i|
// (at least 2^-100, so a row of zeros needs no case of its own) and Q the
// largest code, code_i = rn(fl(x_i * fl(Q / a))) and scale = fl(a / Q): one
// division per row, one product per value, every step rounded to nearest, so
// that any implementation of those words stores the same codes (the scale is
// held down to where Q times it is still finite).  q and k are
// turned first, with the tape's float arithmetic (rotate-half RoPE:
// fl(fl(y cos) + fl(y' sin))).
//
// Bound by memory, 8-bit appends by instructions: each value is loaded once and
// leaves as one byte.  A row lives in head_dim / 4 lanes, four values each, so
// its loads (16 bytes a lane) and its code stores (4 bytes a lane) are whole
// 128-byte lines; the rotation's partner values and the row's maximum come by
// shuffles.
// Measured: 4095 positions of 32 heads of 128, 8 bits: appended in 70 us
// (307 MB, 4.4 TB/s: instructions, 76 % of the issue slots; the rotation, the
// maximum over a row's lanes, the division and the codes), read back in 28 us
// (169 MB, 6.0 TB/s); fp32 65 us (407 MB, 6.3 TB/s) and 43 us (268 MB, 6.2).
// 32 rows of 48 heads: 3.9 us for both, two launches.
#include <cuda_fp8.h>
#include <float.h>

#include "serve.cuh"

namespace kllm {
namespace {

constexpr int KV_THREADS = 256;

__device__ __forceinline__ float4 kv_load4(const float *p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const float4 *>(p));
    return make_float4(p[0], p[1], p[2], p[3]);
}

// Four values of one row: the sum of nz planes in range order.
__device__ __forceinline__ float4 kv_source(const float *p, bool vec, int nz, long long plane) {
    float4 a = kv_load4(p, vec);
    for (int z = 1; z < nz; z++) {
        const float4 b = kv_load4(p + z * plane, vec);
        a.x = __fadd_rn(a.x, b.x);
        a.y = __fadd_rn(a.y, b.y);
        a.z = __fadd_rn(a.z, b.z);
        a.w = __fadd_rn(a.w, b.w);
    }
    return a;
}

// Where row r lives: its sequence and position, or false outside the cache.
__device__ __forceinline__ bool kv_place(const kllm_kv_cache &c, const int *seq, const int *pos,
                                         int pos0, int r, int *s, long long *p) {
    *s = seq ? seq[r] : pos ? r : 0;
    *p = (long long)pos0 + (pos ? pos[r] : r);
    return *s >= 0 && *s < c.n_seq && *p >= 0 && *p < c.max_pos;
}

template <int FMT>
__device__ __forceinline__ uint32_t kv_codes(float4 y) {
    if constexpr (FMT == KLLM_KV_I8) {
        const int a = __float2int_rn(y.x), b = __float2int_rn(y.y), c = __float2int_rn(y.z),
                  d = __float2int_rn(y.w);
        return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 |
               (uint32_t)d << 24;
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y.x, y.y), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y.z, y.w), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}

// A warp takes U x (128 / HD) consecutive heads of one row, of q (rotated
// into q_out), then k (rotated, stored), then v (stored).
// grid: rows x any number of blocks over the heads.
template <int HD, int FMT, int U>
__global__ void __launch_bounds__(KV_THREADS)
k_kv_append(const kllm_kv_cache c, const kllm_kv_rows a, int nz, long long plane, bool vec) {
    constexpr int LPR = HD / 4, HPW = 32 / LPR;   // lanes per head row, head rows per warp
    const int r = blockIdx.x, lane = threadIdx.x & 31, sub = lane / LPR, d = 4 * (lane % LPR);
    const int heads = a.n_heads + 2 * c.n_kv;
    const int h0 = (blockIdx.y * (KV_THREADS / 32) + (threadIdx.x >> 5)) * (U * HPW);
    if (h0 >= heads) return;
    int s;
    long long p;
    if (!kv_place(c, a.seq, a.pos, a.pos0, r, &s, &p)) return;
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool rope = a.rope_cos != nullptr;
    if (rope) {
        const long long ang = p + a.rope_offset;
        if (ang < 0 || ang >= a.rope_rows) return;
        const float *cp = a.rope_cos + ang * HD + d, *sp = a.rope_sin + ang * HD + d;
        cs = kv_load4(cp, vec);
        sn = kv_load4(sp, vec);
    }
    float4 x[U];
    // where head h of the row's q, k and v would be, h counted through all three
    const int hk = a.n_heads, hv = a.n_heads + c.n_kv;
    const long long row = (long long)r * a.row_stride + d;
    const float *bq = a.q + row, *bk = a.k + row - hk * a.head_stride, *bv = a.v + row - hv * a.head_stride;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW + sub;
        x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < heads) x[u] = kv_source((h < hk ? bq : h < hv ? bk : bv) + h * a.head_stride, vec, nz, plane);
    }
    // (what no row of the warp needs is left out)
    uint32_t most[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW + sub;
        const bool turned = rope && h < a.n_heads + c.n_kv;
        float4 y = x[u];
        if (__any_sync(0xffffffffu, turned)) {
            // the partner values live half a row of lanes away
            float4 o;
            o.x = __shfl_xor_sync(0xffffffffu, y.x, LPR / 2);
            o.y = __shfl_xor_sync(0xffffffffu, y.y, LPR / 2);
            o.z = __shfl_xor_sync(0xffffffffu, y.z, LPR / 2);
            o.w = __shfl_xor_sync(0xffffffffu, y.w, LPR / 2);
            if (d < HD / 2) o = make_float4(-o.x, -o.y, -o.z, -o.w);
            if (turned) {
                y.x = __fadd_rn(__fmul_rn(y.x, cs.x), __fmul_rn(o.x, sn.x));
                y.y = __fadd_rn(__fmul_rn(y.y, cs.y), __fmul_rn(o.y, sn.y));
                y.z = __fadd_rn(__fmul_rn(y.z, cs.z), __fmul_rn(o.z, sn.z));
                y.w = __fadd_rn(__fmul_rn(y.w, cs.w), __fmul_rn(o.w, sn.w));
            }
            x[u] = y;
        }
        // the row's maximum, by bit patterns: an infinity or a NaN wins
        if (FMT != KLLM_KV_F32 && __any_sync(0xffffffffu, h >= a.n_heads)) {
            uint32_t m =
                max(max(__float_as_uint(y.x) & 0x7fffffffu, __float_as_uint(y.y) & 0x7fffffffu),
                    max(__float_as_uint(y.z) & 0x7fffffffu, __float_as_uint(y.w) & 0x7fffffffu));
#pragma unroll
            for (int o2 = LPR / 2; o2; o2 >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o2));
            most[u] = m;
        } else {
            most[u] = 0;
        }
    }
    // Row k of the warp's U HPW by lane k: its two divisions, once for all of them, and its scale.
    float inv = 0.f;
    constexpr float Q = FMT == KLLM_KV_I8 ? 127.f : 448.f;
    if constexpr (FMT != KLLM_KV_F32) {
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t t = __shfl_sync(0xffffffffu, most[u], lane % HPW * LPR);
            if (lane / HPW == u) m = t;
        }
        const bool fine = m < 0x7f800000u;
        const float amax = fmaxf(__uint_as_float(m), 0x1p-100f);
        inv = fine ? __fdiv_rn(Q, amax) : 0.f;
        const int h = h0 + lane - a.n_heads;
        if (lane < U * HPW && h >= 0 && h < 2 * c.n_kv)
            (h < c.n_kv ? c.k_scale : c.v_scale)[(long long)s * c.scale_stride +
                                                 (long long)(h < c.n_kv ? h : h - c.n_kv) * c.max_pos + p] =
                fine ? fminf(__fdiv_rn(amax, Q), __fdiv_rz(FLT_MAX, Q)) : __uint_as_float(0x7fffffffu);
    }
    constexpr int ES = FMT == KLLM_KV_F32 ? 4 : 1;
    const long long head = (long long)c.max_pos * HD * ES, at = ((long long)s * c.seq_stride + p * HD + d) * ES;
    uint8_t *dk = static_cast<uint8_t *>(c.k) + at - hk * head, *dv = static_cast<uint8_t *>(c.v) + at - hv * head;
    float *dq = a.q_out + (long long)r * a.n_heads * HD + d;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW + sub;
        const float f = FMT == KLLM_KV_F32 ? 0.f : __shfl_sync(0xffffffffu, inv, u * HPW + sub);
        if (h >= heads) continue;
        const float4 y = x[u];
        if (h < a.n_heads) {
            float *q = dq + h * HD;
            if (vec) {
                *reinterpret_cast<float4 *>(q) = y;
            } else {
                q[0] = y.x, q[1] = y.y, q[2] = y.z, q[3] = y.w;
            }
            continue;
        }
        uint8_t *dst = (h < hv ? dk : dv) + h * head;
        if constexpr (FMT == KLLM_KV_F32) {
            *reinterpret_cast<float4 *>(dst) = y;
        } else {
            // (f is 0 for a row that is not finite: its codes are zeros, and NaN * 0 is none)
            const uint32_t codes = kv_codes<FMT>(make_float4(__fmul_rn(y.x, f), __fmul_rn(y.y, f),
                                                             __fmul_rn(y.z, f), __fmul_rn(y.w, f)));
            *reinterpret_cast<uint32_t *>(dst) = f == 0.f ? 0u : codes;
        }
    }
}

template <int FMT>
__device__ __forceinline__ float4 kv_values(uint32_t w, float sc) {
    float4 y;
    if constexpr (FMT == KLLM_KV_I8) {
        y = make_float4((float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16),
                        (float)(int8_t)(w >> 24));
    } else {
        const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
        const float2 b = __half22float2(
            __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
        y = make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__fmul_rn(y.x, sc), __fmul_rn(y.y, sc), __fmul_rn(y.z, sc),
                       __fmul_rn(y.w, sc));
}

// A warp takes U x (128 / HD) consecutive heads of one row, of k, then v.
template <int HD, int FMT, int U>
__global__ void __launch_bounds__(KV_THREADS)
k_kv_read(const kllm_kv_cache c, const int *__restrict__ seq, const int *__restrict__ pos, int pos0,
          float *__restrict__ ko, float *__restrict__ vo, long long row_stride,
          long long head_stride, bool vec) {
    constexpr int LPR = HD / 4, HPW = 32 / LPR;
    const int r = blockIdx.x, lane = threadIdx.x & 31, sub = lane / LPR, d = 4 * (lane % LPR);
    const int h0 = (blockIdx.y * (KV_THREADS / 32) + (threadIdx.x >> 5)) * (U * HPW);
    int s;
    long long p;
    if (h0 >= 2 * c.n_kv || !kv_place(c, seq, pos, pos0, r, &s, &p)) return;
    float4 y[U];
    uint32_t w[U];
    float sc[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW + sub;
        if (h >= 2 * c.n_kv) continue;
        const bool isk = h < c.n_kv;
        const long long row = (long long)(isk ? h : h - c.n_kv) * c.max_pos + p;
        const void *src = isk ? c.k : c.v;
        if constexpr (FMT == KLLM_KV_F32) {
            y[u] = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(src) +
                                                          (long long)s * c.seq_stride + row * HD + d));
        } else {
            w[u] = __ldg(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(src) +
                                                            (long long)s * c.seq_stride + row * HD + d));
            sc[u] = __ldg((isk ? c.k_scale : c.v_scale) + (long long)s * c.scale_stride + row);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW + sub;
        if (h >= 2 * c.n_kv) continue;
        if constexpr (FMT != KLLM_KV_F32) y[u] = kv_values<FMT>(w[u], sc[u]);
        float *o = (h < c.n_kv ? ko : vo) + (long long)r * row_stride +
                   (long long)(h < c.n_kv ? h : h - c.n_kv) * head_stride + d;
        if (vec) {
            *reinterpret_cast<float4 *>(o) = y[u];
        } else {
            o[0] = y[u].x, o[1] = y[u].y, o[2] = y[u].z, o[3] = y[u].w;
        }
    }
}

bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int HD, int FMT>
bool append_launch(cudaStream_t s, const KvAppend &a, bool vec) {
    const int heads = a.r.n_heads + 2 * a.c.n_kv, per = KV_THREADS / 32 * (128 / HD);
    // few rows: as many warps as there are head rows (latency); many rows:
    // four head rows' loads in flight per warp, the angles loaded once for
    // them.  Append and read together, one and four, in us: 96 head rows of
    // 128 (8 bits), 32 rows 4.8 5.4, 64 rows 6.4 5.8, 1000 rows 45 26; 48 of
    // 128 (fp32), 64 rows 4.2 4.4, 200 rows 5.7 5.1; 40 of 64 (8 bits), 200
    // rows 5.0 5.2, 400 rows 6.2 5.5.
    if ((long long)a.r.rows * heads <= 148ll * 4 * per) {
        k_kv_append<HD, FMT, 1><<<dim3(a.r.rows, (heads + per - 1) / per), KV_THREADS, 0, s>>>(
            a.c, a.r, a.nz, a.plane, vec);
    } else {
        k_kv_append<HD, FMT, 4><<<dim3(a.r.rows, (heads + 4 * per - 1) / (4 * per)), KV_THREADS, 0,
                                  s>>>(a.c, a.r, a.nz, a.plane, vec);
    }
    g_launches++;
    return KLLM_CUDA(cudaGetLastError());
}

template <int HD, int FMT>
bool read_launch(cudaStream_t s, const kllm_kv_cache &c, int rows, const int *seq, const int *pos,
                 int pos0, float *k, float *v, long long row_stride, long long head_stride,
                 bool vec) {
    const int heads = 2 * c.n_kv, per = KV_THREADS / 32 * (128 / HD);
    if ((long long)rows * heads <= 148ll * 4 * per)      // (as append_launch)
        k_kv_read<HD, FMT, 1><<<dim3(rows, (heads + per - 1) / per), KV_THREADS, 0, s>>>(
            c, seq, pos, pos0, k, v, row_stride, head_stride, vec);
    else
        k_kv_read<HD, FMT, 4><<<dim3(rows, (heads + 4 * per - 1) / (4 * per)), KV_THREADS, 0, s>>>(
            c, seq, pos, pos0, k, v, row_stride, head_stride, vec);
    g_launches++;
    return KLLM_CUDA(cudaGetLastError());
}

template <int HD, class F>
bool by_format(int fmt, F &&f) {
    return fmt == KLLM_KV_F32 ? f(std::integral_constant<int, KLLM_KV_F32>())
         : fmt == KLLM_KV_I8  ? f(std::integral_constant<int, KLLM_KV_I8>())
                              : f(std::integral_constant<int, KLLM_KV_E4M3>());
}

}  // namespace

bool kv_cache_ok(const char *who, const kllm_kv_cache *c) {
    if (!c || c->format < KLLM_KV_F32 || c->format > KLLM_KV_E4M3) {
        set_error("%s: no cache, or an unknown format", who);
        return false;
    }
    if (c->n_seq < 1 || c->n_kv < 1 || c->n_kv > 65535 || c->max_pos < 1 ||
        (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)) {
        set_error("%s: cache of %d sequences, %d kv heads of %d, %d positions (head dims 32, 64, 128)",
                  who, c->n_seq, c->n_kv, c->head_dim, c->max_pos);
        return false;
    }
    const bool f32 = c->format == KLLM_KV_F32;
    if (!c->k || !c->v || (!f32 && (!c->k_scale || !c->v_scale))) {
        set_error("%s: a cache pointer is NULL", who);
        return false;
    }
    const long long seq = (long long)c->n_kv * c->max_pos;
    if (!on16(c->k) || !on16(c->v) || c->seq_stride % (f32 ? 4 : 16) ||
        (!f32 && ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3))) {
        set_error("%s: cache rows must start on 16 bytes, scales on 4", who);
        return false;
    }
    if (c->n_seq > 1 && (c->seq_stride < seq * c->head_dim || (!f32 && c->scale_stride < seq))) {
        set_error("%s: sequences %lld elements and %lld scales apart overlap", who, c->seq_stride,
                  c->scale_stride);
        return false;
    }
    return true;
}

bool kv_append(cudaStream_t s, const KvAppend &a) {
    const kllm_kv_rows &r = a.r;
    // 16-byte loads and stores where every row of q, k, v and the angles allows them
    const bool vec = on16(r.q) && on16(r.k) && on16(r.v) && on16(r.q_out) && on16(r.rope_cos) &&
                     on16(r.rope_sin) && r.row_stride % 4 == 0 && r.head_stride % 4 == 0 &&
                     a.plane % 4 == 0;
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return by_format<HD>(a.c.format, [&](auto f) {
            return append_launch<HD, decltype(f)::value>(s, a, vec);
        });
    };
    return a.c.head_dim == 32 ? go(std::integral_constant<int, 32>())
         : a.c.head_dim == 64 ? go(std::integral_constant<int, 64>())
                              : go(std::integral_constant<int, 128>());
}

bool kv_read(cudaStream_t s, const kllm_kv_cache &c, int rows, const int *seq, const int *pos,
             int pos0, float *k, float *v, long long row_stride, long long head_stride) {
    const bool vec = on16(k) && on16(v) && row_stride % 4 == 0 && head_stride % 4 == 0;
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return by_format<HD>(c.format, [&](auto f) {
            return read_launch<HD, decltype(f)::value>(s, c, rows, seq, pos, pos0, k, v, row_stride,
                                                       head_stride, vec);
        });
    };
    return c.head_dim == 32 ? go(std::integral_constant<int, 32>())
         : c.head_dim == 64 ? go(std::integral_constant<int, 64>())
                            : go(std::integral_constant<int, 128>());
}

}  // namespace kllm

using namespace kllm;

extern "C" int kllm_kv_append(const kllm_kv_cache *cache, const kllm_kv_rows *rows, void *stream) {
    if (!kv_cache_ok("kllm_kv_append", cache)) return -1;
    if (!rows || rows->rows < 0 || rows->n_heads < 0 || rows->n_heads > 65535 || !rows->k ||
        !rows->v || (rows->n_heads && (!rows->q || !rows->q_out))) {
        set_error("kllm_kv_append: invalid arguments");
        return -1;
    }
    if (!rows->rope_cos != !rows->rope_sin || (rows->rope_cos && rows->rope_rows < 1)) {
        set_error("kllm_kv_append: rope_cos and rope_sin come together, with rope_rows rows");
        return -1;
    }
    if (rows->seq && !rows->pos) {
        set_error("kllm_kv_append: seq without pos");
        return -1;
    }
    if (rows->rows == 0) return 0;
    KvAppend a;
    a.c = *cache;
    a.r = *rows;
    return kv_append((cudaStream_t)stream, a) ? 0 : -1;
}

extern "C" int kllm_kv_read(const kllm_kv_cache *cache, int rows, const int *seq, const int *pos,
                            int pos0, float *k, float *v, long long row_stride,
                            long long head_stride, void *stream) {
    if (!kv_cache_ok("kllm_kv_read", cache)) return -1;
    if (rows < 0 || !k || !v) {
        set_error("kllm_kv_read: invalid arguments");
        return -1;
    }
    if (seq && !pos) {
        set_error("kllm_kv_read: seq without pos");
        return -1;
    }
    if (rows == 0) return 0;
    return kv_read((cudaStream_t)stream, *cache, rows, seq, pos, pos0, k, v, row_stride, head_stride)
               ? 0
               : -1;
}
