// serve.cuh -- internal entry points of the batch serving operators, shared
// by their C ABI (include/kllm_cuda.h) and the batched decode (plan.cu).
#pragma once

#include "common.cuh"
#include "sm100.cuh"

namespace kllm {

// ------------------------------------------------ kvcache.cu: the cache ----

// What kllm_kv_append runs, with rows that may come as the K-range partial
// tiles of a GEMM: each value of q, k and v is the sum of nz planes, `plane`
// floats apart, in range order.
struct KvAppend {
    kllm_kv_cache c;
    kllm_kv_rows r;
    int nz = 1;
    long long plane = 0;
};

bool kv_cache_ok(const char *who, const kllm_kv_cache *c);
bool kv_append(cudaStream_t s, const KvAppend &a);
bool kv_read(cudaStream_t s, const kllm_kv_cache &c, int rows, const int *seq, const int *pos,
             int pos0, float *k, float *v, long long row_stride, long long head_stride);

// ------------------------------------------- batchattn.cu: attention -------

// What kllm_batch_attention runs.  The output may be written as the next
// GEMM's input: fp32 rows (terms 0, `out` as the struct has it), or `terms`
// bf16 terms of the exact split in planes of n_seq * n_heads * head_dim
// (rows.cuh, bd_emit).  A wait that takes longer than wait_ns gives up, leaves
// NaN in the rows it was for and ST_WAIT_TIMEOUT in *status (may be null).
struct BatchAttention {
    kllm_batch_attn a;
    int terms = 0;
    void *terms_out = nullptr;
    int *status = nullptr;
    unsigned long long wait_ns = kWaitLimitNs;
};

bool batch_attention(cudaStream_t s, const BatchAttention &b);

// ------------------------------------------------- sample.cu: the draw -----

// kllm_sample, its logits as the sum of nz planes (as KvAppend).
bool sample_rows(cudaStream_t s, const kllm_sample_rows &r, int nz, long long plane);

}  // namespace kllm
