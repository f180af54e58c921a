// batchattn.cuh -- what the kernels of the shared-prefix attention have in
// common (batchattn.cu: a few rows at a time; batchattn_tc.cuh: 128).
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace kllm {
namespace {

struct BaSide {
    const void *k, *v;
    const float *ks, *vs;
    long long seq_stride, scale_stride;
    int max_pos;      // rows of a (sequence, head)
    int parts, chunk; // ranges of `chunk` positions
};

struct BaArgs {
    BaSide pre, own;
    const float *q;
    long long q_stride;
    bool q_vec;                 // rows of q start on 16 bytes
    const int *own_len;
    int n_seq, nh, nkv, groups, prefix_len, own_cap;
    int tiles_pre, tiles_own;   // row tiles: of n_seq * groups, of groups
    int blocks_pre;             // of this launch: the first take the prefix's items, the rest the sequences'
    bool join;                  // the sequences' blocks join their rows' parts and write the output
    float qk;                   // scale * log2(e)
    float *part_ml, *part_o;    // [n_seq * nh][parts][2], [n_seq * nh][parts][HD]
    float *out;
    long long out_stride;
    int terms;                  // as bd_emit
    void *terms_out;
    int *status;                // gets ST_WAIT_TIMEOUT when a wait gives up (may be null)
    unsigned long long wait_ns; // bound of each wait
};

__device__ __forceinline__ uint32_t ba_prmt(uint32_t a, uint32_t b, uint32_t sel) {
    return __byte_perm(a, b, sel);
}

__device__ __forceinline__ uint32_t ba_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float ba_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float ba_lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^n, n from -126 to 127
__device__ __forceinline__ float ba_exp2i(int n) { return __int_as_float((n + 127) << 23); }

// hi and lo fp16 terms of a pair
__device__ __forceinline__ void ba_split(float a, float b, uint32_t *hi, uint32_t *lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    *hi = *reinterpret_cast<const uint32_t *>(&h);
    *lo = ba_h2(a - f.x, b - f.y);
}

// the two codes of each half of a word, (c0, c1) or (c2, c3), as fp16
template <int FMT, int HALF>
__device__ __forceinline__ uint32_t ba_codes(uint32_t w) {
    if constexpr (FMT == KLLM_KV_I8) {
        // w holds code + 128: the fp16 with bits 0x6400 + u is 1024 + u
        const uint32_t u = ba_prmt(w, 0x64646464u, HALF ? 0x4342 : 0x4140);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&u),
                                  __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        uint32_t d;
        const uint16_t c = (uint16_t)(HALF ? w >> 16 : w & 0xffffu);
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(c));
        return d;
    }
}

__device__ __forceinline__ void ba_mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                           uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ba_mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The power of two that |x| lies above (to 2^126, which goes for all larger
// numbers too): x times its inverse and 2^13 is below 2^15.
__device__ __forceinline__ float ba_pow2(float x) {
    const float c = fminf(fmaxf(x, 0x1p-110f), 0x1p126f);
    return __uint_as_float(__float_as_uint(c) & 0x7f800000u);
}

// Loads that stay where they are written (ahead of their use, which the
// compiler would rather load at), zeros where `in` is false.
__device__ __forceinline__ void ba_fetch(uint32_t (&w)[4], const void *p, bool in) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %5, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(w[0]), "=&r"(w[1]), "=&r"(w[2]), "=&r"(w[3])
        : "l"(p), "r"((uint32_t)in));
}
__device__ __forceinline__ void ba_fetch(uint32_t (&w)[2], const void *p, bool in) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
        "@p ld.global.nc.v2.u32 {%0, %1}, [%2];\n\t}"
        : "=&r"(w[0]), "=&r"(w[1])
        : "l"(p), "r"((uint32_t)in));
}
__device__ __forceinline__ void ba_fetch(uint32_t (&w)[1], const void *p, bool in) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "mov.u32 %0, 0;\n\t"
        "@p ld.global.nc.u32 %0, [%1];\n\t}"
        : "=&r"(w[0])
        : "l"(p), "r"((uint32_t)in));
}

// Asynchronous copies to shared memory, zeros past `bytes`.
__device__ __forceinline__ void ba_cp16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void ba_cp4(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}

}  // namespace
}  // namespace kllm
