// rows.cuh -- what the row kernels of the batched decode share: reading a
// GEMM's output, writing the next one's input, row loads.
#pragma once

#include <cuda_bf16.h>

namespace kllm {

// One element of a GEMM output: the sum of its nz K-range partial tiles,
// part[z * plane + i], in range order (nz = 1: the output itself).
__device__ __forceinline__ float bd_sum(const float *__restrict__ part, int nz, size_t plane,
                                        size_t i) {
    float a = part[i];
    for (int z = 1; z < nz; z++) a = __fadd_rn(a, part[(size_t)z * plane + i]);
    return a;
}

// One element of the next GEMM's input: fp32 (terms 0), or the bf16 terms
// hi = bf16(v), mid = bf16(v - hi), lo = bf16(v - hi - mid), term t at
// t * plane + i.
__device__ __forceinline__ void bd_emit(float v, size_t i, int terms, size_t plane,
                                        void *__restrict__ xs) {
    if (!terms) {
        reinterpret_cast<float *>(xs)[i] = v;
        return;
    }
    __nv_bfloat16 *o = reinterpret_cast<__nv_bfloat16 *>(xs);
    float r = v;
    for (int t = 0; t < terms; t++) {
        const __nv_bfloat16 b = __float2bfloat16_rn(r);
        o[(size_t)t * plane + i] = b;
        r = __fsub_rn(r, __bfloat162float(b));
    }
}

template <int VEC>
__device__ __forceinline__ void bd_load(const float *p, float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(p);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else if constexpr (VEC == 2) {
        const float2 t = *reinterpret_cast<const float2 *>(p);
        v[0] = t.x, v[1] = t.y;
    } else {
        v[0] = *p;
    }
}

}  // namespace kllm
