/*
 * kllm_cuda.h -- extensions of the kllm C ABI that the B200 executor adds
 * next to the drop-in surface of tape_runner.h.
 *
 * None of these exists in the reference runtime (csrc/tape_runner.h); each
 * comment says which reference behaviour it complements.  All functions are
 * plain C: pointers and sizes only.
 */
#ifndef KLLM_CUDA_H
#define KLLM_CUDA_H

#include <stddef.h>
#include <stdint.h>

#include "tape_runner.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- errors --
 * The reference has no error reporting (void functions, exit(1) in the
 * loaders, processor_infer* always return 0: _tape_runner.c:1587,1762).
 * Here every failure is recorded per thread and the call returns. */

/* Message of the first error recorded on this thread since the last clear,
 * or NULL when there is none. */
const char *kllm_last_error(void);
void kllm_clear_error(void);

/* Version string of this library. */
const char *kllm_version(void);

/* Number of CUDA devices visible to this process (0 without a GPU). */
int kllm_device_count(void);

/* Device used by contexts created afterwards on this thread (default: the
 * CUDA current device).  Returns 0, or -1 for an invalid ordinal. */
int kllm_set_device(int device);

/* tape_run with a status: 0 on success, non-zero on error
 * (complements _tape_runner.c:665, which cannot fail). */
int kllm_tape_run(TapeCtx *ctx);

/* Kernels launched by this process so far (all contexts). */
long long kllm_launch_count(void);

/* --------------------------------------------------- inference options --
 * processor_infer / processor_infer_bytes keep the reference signatures;
 * these settings ride on the context. */
enum {
    KLLM_MODE_AUTO = 0,     /* fused decode plan when the tape matches the
                               compiler's LLaMA template, else per-op */
    KLLM_MODE_GENERIC = 1,  /* per-op device execution of every instruction
                               (same loop structure as the reference) */
    KLLM_MODE_FUSED = 2     /* fused plan or an error */
};

/* Summation order of the fused decode step's TT-GEMVs. */
enum {
    KLLM_ORDER_EXACT = 0,   /* the reference's chunked order: every MATMUL_TT
                               result is bit-identical to _tape_runner.c's */
    KLLM_ORDER_FAST = 1     /* K split finer across warps (decode only): same
                               tokens and logits within the decode tolerance,
                               more parallelism in the narrow projections; one
                               GPU only (a column-sharded context builds the
                               exact order) */
};

typedef struct {
    int mode;                /* KLLM_MODE_* */
    float *logits_out;       /* optional host buffer: the logits row after
                                every tape step, [logits_rows][vocab] */
    int logits_rows;         /* capacity of logits_out in rows */
    int use_graphs;          /* replay each step as a CUDA graph (fused) */
    int order;               /* KLLM_ORDER_*, fused decode step */
    int prefill;             /* 1: the prompt's positions but the last run as one
                                batched pass (TT-GEMMs, kllm_tt_gemm) instead of
                                one tape step each (persistent plan, one GPU, no
                                logits_out); 0: the default, step by step */
    int reserved[6];
} kllm_infer_opts;

typedef struct {
    int fused;               /* 1 when the fused plan ran */
    int steps;               /* tape steps run (prompt + generated) */
    double prefill_ms;       /* device time of the prompt steps */
    double decode_ms;        /* device time of the generation steps */
    double total_ms;         /* wall time inside the call */
    long long launches;      /* kernels launched inside the call */
    int step_kernel;         /* fused: 1 = one persistent kernel per tape step,
                                0 = the per-kernel plan */
    int stream_values;       /* persistent step: what the weight streams hold,
                                0 = codebook table slots, 1 = bf16 values,
                                2 = fp16 values (exact codebooks only) */
    int shared_prefix;       /* kllm_infer_batch_ex: prompt positions that were
                                computed and held once for all sequences */
    int reserved[5];
} kllm_infer_stats;

void kllm_default_infer_opts(kllm_infer_opts *o);
int kllm_set_infer_opts(TapeCtx *ctx, const kllm_infer_opts *o);
int kllm_get_infer_stats(TapeCtx *ctx, kllm_infer_stats *s);

/* Whether processor_infer takes the fused decode plan for this tape: 1
 * when the tape is the kllm compiler's LLaMA decode template
 * (kllm_compile.c:1143-1385) for these dimensions and slot maps, 0 when not
 * (the first mismatch is written to why), -1 on bad arguments.  Host only;
 * needs no GPU. */
int kllm_plan_match(TapeCtx *ctx, int vocab_size, int hidden_dim, int head_dim,
                    int token_embed_slot, int rope_cos_slot, int rope_sin_slot,
                    const int *kv_in_slots, const int *kv_out_slots, int logits_slot,
                    int n_layers, int num_kv_heads, char *why, int why_len);

/* Build the fused decode plan now (weights to the device layout, buffers)
 * for contexts of up to max_pos positions, instead of at the first
 * processor_infer call.  Same model arguments as processor_infer.  0 on
 * success, -1 (kllm_last_error) when the tape does not match the template. */
int kllm_plan_prepare(TapeCtx *ctx, const float *embed_table, int vocab_size, int hidden_dim,
                      const float *rope_cos, const float *rope_sin, int head_dim,
                      int token_embed_slot, int rope_cos_slot, int rope_sin_slot,
                      const int *kv_in_slots, const int *kv_out_slots, int logits_slot,
                      int n_layers, int num_kv_heads, int max_pos);

/* ----------------------------------------------- column-sharded decode -----
 * One process per GPU.  Rank r of `world` stores and multiplies every
 * world-th column group of each TT matrix (N is sharded, K and the
 * codebooks are not), and stores its results into every rank's copy of the
 * activations over NVLink peer memory inside the decode kernel; each output
 * column's arithmetic is unchanged, so results equal the 1-GPU run.
 * Sequence: kllm_shard_set (before the plan exists), kllm_plan_prepare,
 * kllm_shard_export on every rank, exchange the blocks (any transport,
 * e.g. torch.distributed), kllm_shard_connect with all blocks in rank
 * order, then processor_infer on every rank with the same arguments.  The
 * reference has no multi-GPU path. */
int kllm_shard_set(TapeCtx *ctx, int rank, int world);
/* This rank's block (CUDA IPC handles); *len gets its size. */
int kllm_shard_export(TapeCtx *ctx, void *out, size_t cap, size_t *len);
/* world blocks of per_rank bytes each, in rank order. */
int kllm_shard_connect(TapeCtx *ctx, const void *all, size_t per_rank);

/* ----------------------------------------------------------- TT-GEMV -----
 * y[r][n] = sum_k fl(x[r][k] * codebook[idx[k][n]]) in the accumulation
 * order of the reference TT-GEMV (_tape_runner.c:495-663): K is cut into
 * T = min(8, ceil(K/128)) chunks (the first K%T chunks one row longer),
 * each chunk is summed row by row from 0.0f, and the chunk sums are added
 * in chunk order.  Results are bit-identical to the reference for every
 * input.  idx is uint16 row-major [K][N]; codebook has n_codes floats.
 *
 * Device-pointer form: all pointers are device memory of the calling
 * thread's device; stream is a cudaStream_t (NULL = default stream).  Every
 * index must be < n_codes (not checked here: the caller owns the data).
 * Uses a per-device scratch buffer for the chunk partials, grown on demand
 * with cudaMalloc.  Returns 0 or non-zero on error (see kllm_last_error). */
int kllm_tt_gemv(const float *x, int rows, const float *codebook, int n_codes,
                 const uint16_t *idx, int K, int N, float *y, void *stream);

/* Host-buffer form of the same product: checks every index against
 * n_codes, copies x, codebook and idx to the device, runs, copies y back
 * (synchronous). */
int kllm_tt_gemv_host(const float *x, int rows, const float *codebook,
                      int n_codes, const uint16_t *idx, int K, int N, float *y);

/* TT-GEMM: the same product for many rows at once (prefill: every prompt
 * position against one MATMUL_TT weight), each row bit-identical to
 * kllm_tt_gemv of that row (the reference order of _tape_runner.c:474-663 per
 * row).  x is [rows][K] and y [rows][N], device memory; the decoded weight
 * tile is reused across 64 rows, so this form is bound by the FP32 pipes
 * rather than by the index stream.  Allocates nothing.  Every index must be
 * < n_codes; rows <= 4194240.  Returns 0 or non-zero (kllm_last_error). */
int kllm_tt_gemm(const float *x, int rows, const float *codebook, int n_codes,
                 const uint16_t *idx, int K, int N, float *y, void *stream);

/* TT-GEMM on the tensor cores (the same product as kllm_tt_gemm, replacing
 * the per-row MATMUL_TT loop of _tape_runner.c:804-811 for prefill), for
 * matrices whose codebook entries are all bf16 numbers: x is split into
 * `terms` (2 or 3) bf16 terms (hi, mid, lo; 3 terms carry all 24 significand
 * bits of a normal fp32), each weight is exact in bf16, and the products
 * accumulate in fp32 in tensor memory.  Results agree with kllm_tt_gemm to
 * fp32 rounding in a different summation order, not bit for bit.  K must be
 * a multiple of 64 and N of 128; the codebook is checked (a device-to-host
 * copy) and a codebook with any non-bf16 entry is an error.  Allocates and
 * frees its bf16 operands on the stream.  Returns 0 or non-zero
 * (kllm_last_error). */
int kllm_tt_gemm_tc(const float *x, int rows, const float *codebook, int n_codes,
                    const uint16_t *idx, int K, int N, float *y, int terms, void *stream);

/* Allocation-free form of kllm_tt_gemv for one row (x is [K], y is [N]).
 * No counterpart in the reference runtime.  For callers that may not
 * allocate device memory -- code running during CUDA graph capture, plugins
 * whose host framework owns the device memory pool, fixed-footprint
 * real-time hosts -- it keeps its scratch in a fixed array inside the
 * library's device image instead of growing one with cudaMalloc: N is at
 * most 65536 (2 MiB of partial rows per device, held until exit); larger N
 * is rejected with an error.  The first call on a device looks up the
 * array's device address and should come before any stream capture.  Calls
 * whose kernels overlap on the GPU share the array and race.  Same result,
 * bit for bit, as kllm_tt_gemv; every index must be < n_codes. */
int kllm_tt_gemv_noalloc(const float *x, const float *codebook, int n_codes,
                         const uint16_t *idx, int K, int N, float *y, void *stream);

/* ------------------------------------------------ batch serving operators --
 * What a batch that answers one prompt many times needs next to the greedy
 * decode above: key/value caches in 8 bits, attention that reads a prefix
 * which all sequences share once, and tokens drawn from the logits.  None has
 * a counterpart in the reference (its caches are fp32, its attention one
 * sequence's, its pick the first maximum: _tape_runner.c:1602-1763).
 *
 * All pointers inside these structs are device memory of the calling
 * thread's current device unless marked "host"; the structs themselves are
 * host memory and may go away after the call.  Every call launches on
 * `stream` (a cudaStream_t, NULL = default stream), allocates nothing, never
 * waits, and may be captured into a CUDA graph.  Returns 0, or non-zero
 * with kllm_last_error() set and nothing launched. */
enum {
    KLLM_KV_F32 = 0,    /* fp32 as it is, no scales */
    KLLM_KV_I8 = 1,     /* 8-bit integers -127..127 and one scale per row */
    KLLM_KV_E4M3 = 2    /* 8-bit floats (4 exponent, 3 fraction bits) and one
                           scale per row */
};

/* A cache of keys and values: n_seq sequences of up to max_pos positions, a
 * row of head_dim values per (sequence, kv head, position).
 * k, v: [n_seq][n_kv][max_pos][head_dim] floats or codes, sequences
 * seq_stride elements apart; k_scale, v_scale: [n_seq][n_kv][max_pos] floats,
 * sequences scale_stride apart (unused for KLLM_KV_F32).
 * A row x is stored as code_i = rn(fl(x_i * fl(Q / a))) and scale = fl(a / Q),
 * a = max(max |x_i|, 2^-100), Q = 127 (I8) or 448 (E4M3), ties to even (the
 * scale at most the largest with Q * scale finite), and stands for the values
 * fl(code_i * scale).  A row that holds an infinity or
 * a NaN is stored as zeros with a NaN scale: it reads back as NaN.
 * head_dim is 32, 64 or 128; k and v start on 16 bytes and seq_stride is a
 * multiple of 16 elements (4 for KLLM_KV_F32). */
typedef struct {
    int format;              /* KLLM_KV_* */
    int n_seq, n_kv, head_dim, max_pos;
    void *k, *v;
    float *k_scale, *v_scale;
    long long seq_stride, scale_stride;
} kllm_kv_cache;

/* New rows for a cache.  Row r goes to position pos0 + pos[r] of sequence
 * seq[r] (seq NULL: of sequence r); with pos NULL the rows are consecutive
 * positions pos0 + r of sequence 0 (a prompt).  A row whose position or
 * sequence lies outside the cache (a negative one among them: padding) is
 * skipped whole.  Two rows must not name the same place.
 * Head h of row r of q, k and v starts row_stride * r + head_stride * h
 * floats after q, k and v; k and v are required, n_heads = 0 leaves q out.
 * With rope_cos and rope_sin
 * ([rope_rows][head_dim]) q and k are turned as the tape does it
 * (rotate-half, fp32) by the angles of row position + rope_offset; a row
 * whose angles lie outside the tables is skipped. */
typedef struct {
    int rows;
    int n_heads;             /* query heads, 0: no q */
    int pos0;
    int rope_rows, rope_offset;
    const int *seq, *pos;
    const float *q, *k, *v;
    long long row_stride, head_stride;
    float *q_out;            /* [rows][n_heads][head_dim] */
    const float *rope_cos, *rope_sin;   /* both or neither */
} kllm_kv_rows;

/* Turn q and k, quantise k and v and write them into the cache: one kernel. */
int kllm_kv_append(const kllm_kv_cache *cache, const kllm_kv_rows *rows, void *stream);

/* Read rows of a cache back as fp32: row r (placed by seq, pos, pos0 as for
 * kllm_kv_rows) to k and v, head h of it at row_stride * r + head_stride * h.
 * Rows that lie outside the cache are left as they were. */
int kllm_kv_read(const kllm_kv_cache *cache, int rows, const int *seq, const int *pos, int pos0,
                 float *k, float *v, long long row_stride, long long head_stride, void *stream);

/* Attention of one query token per sequence (a decode step) over a prefix
 * that all sequences share and each sequence's own positions:
 *   out[i][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),
 *   s_j = scale * q[i][h] . k_j
 * for j over the prefix's first prefix_len positions, then the first
 * own_len[i] positions of sequence i.  Query head h uses kv head
 * h / (n_heads / n_kv).  The prefix (sequence 0 of `prefix`) is read once
 * for all sequences.  prefix may be NULL (prefix_len 0), own may be NULL
 * (every own length 0); where both are given their formats, n_kv and
 * head_dim agree.  Results are fp32 with fp32 sums in an order of their own.
 *   own_len[i] < 0      a padding row: out[i] is left as it was
 *   own_len[i] > own->max_pos or max_len: the smaller of those is taken
 *   no position at all  out[i] is zeros
 * Scores are fp32 numbers (one past their range is an infinity); a row none of
 * whose scores is above -infinity is NaN.
 * A row of q that holds an infinity or a NaN gets NaN, and so does every row
 * that sees a position whose fp32 key or value is not finite (of a value, in
 * its dim at least), or whose scale is NaN; no other row changes by it.
 * q, p and fp32 keys and values are taken
 * to 22 bits; numbers of a row of q, of a key or of a value that lie far below
 * the largest of the same head_dim numbers keep 2^-38 of that one at least.
 * Other positions and rows do not matter for that.  Keys of 2^100 and more, and
 * scores and |v| times the positions past fp32's range, may become infinities
 * or NaN.
 * n_seq * n_heads and the positions (prefix_len, the smaller of max_len and
 * own->max_pos) are at most 2^31 - 1024.
 * max_len is an upper bound of the own lengths (it sizes the launch, so a
 * captured graph serves every length up to it).  Positions past the lengths
 * are not read.  workspace: kllm_batch_attention_workspace(a) bytes on 16
 * bytes; calls that overlap on the GPU need one each.  Waits inside the call
 * are bounded (2 s); should one give up, its rows are NaN. */
typedef struct {
    int n_seq, n_heads;
    int prefix_len, max_len;
    float scale;
    const float *q;          /* [n_seq], rows of n_heads * head_dim, q_stride floats apart */
    long long q_stride;
    const kllm_kv_cache *prefix, *own;   /* host */
    const int *own_len;      /* [n_seq] */
    float *out;              /* as q */
    long long out_stride;
    void *workspace;
    size_t workspace_bytes;
} kllm_batch_attn;

/* Bytes of workspace the call needs, or 0 with kllm_last_error() set for a
 * call that kllm_batch_attention would refuse.  The workspace, its size, out
 * and out_stride are not looked at. */
size_t kllm_batch_attention_workspace(const kllm_batch_attn *a);
int kllm_batch_attention(const kllm_batch_attn *a, void *stream);

/* One token per row of logits, drawn with a given uniform number:
 *   w_i  = exp((x_i - max x) / temperature), NaN logits as -infinity
 *   kept = the first top_k of the order (x descending, index ascending);
 *          of those, each whose mass of w before it is < top_p times theirs;
 *          of those, each with w_i >= min_p (the first of the order always)
 *   token = the first index whose running sum of kept w, in index order,
 *           exceeds u times their whole sum
 * top_k <= 0, top_p >= 1 and min_p <= 0 turn a rule off; temperature <= 0
 * picks the first maximum, by the rule of the greedy decode (a NaN at index
 * 0 picks 0).  Where no logit is above -infinity the token is 0; +infinity
 * counts as the largest number; temperatures are taken into [1e-30, 1e30], u
 * into [0, 1); NaN
 * settings are refused nowhere and turn their rule off (u: 0).
 * Weights are 2^-40 fixed point, their sums exact integers: a row's token
 * does not depend on the launch or on the other rows.  vocab is at most
 * 2^22.  Settings are one per row; a NULL array turns the rule off
 * (temperature: 1, u: required). */
typedef struct {
    int rows, vocab;
    const float *logits;     /* rows of vocab floats, row_stride apart */
    long long row_stride;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p;
    const float *u;
    int *tokens;             /* [rows] */
} kllm_sample_rows;

int kllm_sample(const kllm_sample_rows *rows, void *stream);

/* ------------------------------------------------------------- chips -----
 * Chip directory loader: the same files, read the same way, as the
 * reference CLI's static chip_load (csrc/kllm.c:152-388): processor.json,
 * tables/<name>.bin, bpe/<files>, circuit/tape.bin + slots.bin + const_<slot>*.bin.
 * The loader validates what the reference trusts (file sizes against
 * slots.bin, the 276-byte record size, slot ids in processor.json) and
 * returns NULL with kllm_last_error() set instead of exiting. */
typedef struct kllm_chip kllm_chip;

kllm_chip *kllm_chip_open(const char *chip_dir);
void kllm_chip_close(kllm_chip *chip);
TapeCtx *kllm_chip_ctx(kllm_chip *chip);

/* info[0..17] = vocab_size, hidden_dim, num_layers, num_kv_heads, head_dim,
 * max_seq_len, eos_token_id, logits_slot, token_embed_slot, rope_cos_slot,
 * rope_sin_slot, n_slots, n_instrs, bos_token_id, hash table_size,
 * max_piece_len, num_merges, num_special. */
int kllm_chip_info(kllm_chip *chip, int *info);

/* processor_infer with the chip's tables and slot maps (what kllm.c passes,
 * csrc/kllm.c:566-584, minus the BPE). */
int kllm_chip_infer(kllm_chip *chip, const int *prompt, int prompt_len, int max_new,
                    int eos_token_id, int *out_tokens, int *out_len);

/* Batched greedy decode of nseq independent sequences on one GPU -- the
 * reference has no counterpart: its processor_infer (_tape_runner.c:
 * 1602-1763) runs one sequence; this runs that loop for all of them at
 * once, each with its own KV cache and position.  prompts holds the
 * sequences' token IDs back to back (prompt_lens[i] each); out receives
 * nseq x max_new tokens (row i: sequence i's greedy tokens, computed for all
 * max_new steps), out_lens[i] the number before sequence i's first `eos`
 * (the reference would stop there; pass -1 for none).  Prompts go through
 * the batched prompt pass, then each step is one GEMM per projection over
 * the nseq rows: on the tensor cores when every codebook entry is a bf16
 * number and nseq <= 128 (a tolerance result), else -- or with
 * KLLM_BATCH_TC=0 in the environment -- the exact TT-GEMM, each row
 * bit-identical to the TT-GEMV.  The context must not be column-sharded.
 * Returns 0 or non-zero (kllm_last_error); kllm_get_infer_stats gives the
 * prompt and decode device times. */
int kllm_infer_batch(TapeCtx *ctx, const int *prompts, const int *prompt_lens, int nseq,
                     int max_new, int eos, int *out, int *out_lens);
/* The same on a loaded chip (prepares its fused plan first). */
int kllm_chip_infer_batch(kllm_chip *chip, const int *prompts, const int *prompt_lens, int nseq,
                          int max_new, int eos, int *out, int *out_lens);

/* Options of kllm_infer_batch_ex (zeros: what kllm_infer_batch does).  All
 * pointers are host memory. */
typedef struct {
    int kv_format;           /* KLLM_KV_* of the sequences' caches and the prefix */
    int share_prefix;        /* 1: the prompts' longest common prefix is computed
                                and held once (every prompt keeps its last
                                token) */
    const float *temperature;   /* [nseq] each, as kllm_sample; NULL: off */
    const int *top_k;
    const float *top_p, *min_p;
    const float *u;          /* [nseq][max_new] uniform numbers in [0, 1), one
                                per generated token; NULL: greedy */
    int reserved[8];
} kllm_batch_opts;

/* kllm_infer_batch with a prefix that the sequences share, caches in 8 bits
 * and drawn tokens (kllm_kv_append, kllm_batch_attention and kllm_sample in
 * the captured step).  With 8-bit caches every decoded position attends to
 * the stored values; a prompt's own positions see fp32 values among
 * themselves and the stored ones of the prefix.  The prompt passes use the
 * context's single-sequence cache.  Head dims 32, 64 and 128. */
int kllm_infer_batch_ex(TapeCtx *ctx, const int *prompts, const int *prompt_lens, int nseq,
                        int max_new, int eos, const kllm_batch_opts *opts, int *out, int *out_lens);
int kllm_chip_infer_batch_ex(kllm_chip *chip, const int *prompts, const int *prompt_lens, int nseq,
                             int max_new, int eos, const kllm_batch_opts *opts, int *out,
                             int *out_lens);

/* kllm_plan_prepare with the chip's tables, for its max_seq_len. */
int kllm_chip_plan_prepare(kllm_chip *chip);

/* processor_infer_bytes with the chip's ROMs, as `kllm infer` calls it
 * (csrc/kllm.c:566-584); max_seq_tokens <= 0 means the chip's max_seq_len. */
int kllm_chip_infer_bytes(kllm_chip *chip, const uint8_t *input, int input_len, int max_new,
                          int max_seq_tokens, token_callback_fn cb, void *user_data,
                          int *total_generated);

/* bpe_encode / bpe_decode with the chip's ROMs. */
int kllm_chip_encode(kllm_chip *chip, const uint8_t *bytes, int len, int max_tokens,
                     int32_t *out_ids);
int kllm_chip_decode(kllm_chip *chip, const int32_t *ids, int n, int max_bytes,
                     int skip_leading_space, uint8_t *out_bytes);

#ifdef __cplusplus
}
#endif

#endif /* KLLM_CUDA_H */
