/*
 * tensorshrink_b200 — C ABI of the B200 (sm_100a) QuantLinear hot path.
 *
 * Plain pointers and sizes only: every pointer argument named "device" is a
 * CUDA device address on the current device, and `stream` is a cudaStream_t
 * passed as void* (NULL = legacy default stream). No entry point allocates
 * device memory; scratch comes from caller-provided workspaces whose sizes
 * the *_workspace_size() functions report. All launches are asynchronous on
 * `stream`. Functions return TS_OK (0) or a negative ts_status; the message
 * of the last failure on the calling thread is in ts_last_error().
 *
 * Packed-weight layout is the reference's `QuantLinear` buffer layout,
 * unchanged (tensorshrink codec.py:102-151, modules.py:337-448):
 *   packed   uint8 [rows, padded_cols*bits/8]; 4-bit: byte = c[2j] | c[2j+1]<<4;
 *            2-bit: byte = c[4j] | c[4j+1]<<2 | c[4j+2]<<4 | c[4j+3]<<6; 8-bit raw.
 *   scale/gmin fp16 [rows, n_groups]   (or the double-quantized form:
 *   dq_*_codes uint8 flattened row-major over [rows, n_groups], one
 *   (meta_scale, meta_min) fp16 pair per dq_group_size entries).
 *   codebook fp32 [1<<bits] (NF / Lloyd-Max levels) or NULL.
 *   outliers: row-sorted int32 row/col, fp16 delta, plus CSR row offsets.
 * Reconstruction: w[r,c] = cb?[code] * scale[r,g] + gmin[r,g] (+ delta at
 * outlier positions), g = c / group_size.
 */
#ifndef TENSORSHRINK_B200_H
#define TENSORSHRINK_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define TS_API __attribute__((visibility("default")))
#else
#define TS_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef enum ts_dtype {
  TS_F16 = 0,
  TS_BF16 = 1,
  TS_F32 = 2
} ts_dtype;

typedef enum ts_status {
  TS_OK = 0,
  TS_ERR_INVALID = -1,     /* bad argument (shape, pointer, alignment) */
  TS_ERR_UNSUPPORTED = -2, /* valid but not covered (bit width, dtype) */
  TS_ERR_CUDA = -3,        /* a CUDA runtime call failed */
  TS_ERR_WORKSPACE = -4,   /* workspace missing or too small */
  TS_ERR_TIMEOUT = -5      /* a bounded wait in a kernel ran out (ts_qlinear_status) */
} ts_status;

/* One quantized weight matrix as resident on the device (QuantLinear's
 * buffers). Exactly one of {scale,gmin} / {dq_*} is set. */
typedef struct ts_qweight {
  int64_t rows;             /* out_features (N) */
  int64_t cols;             /* in_features (K), unpadded */
  int64_t padded_cols;      /* cols rounded up to a multiple of group_size */
  int64_t n_groups;         /* padded_cols / group_size */
  int64_t packed_row_bytes; /* row stride of `packed` in bytes */
  int32_t bits;             /* 2, 4 or 8 */
  int32_t group_size;
  const uint8_t* packed;
  const uint16_t* scale;    /* fp16 [rows, n_groups] or NULL */
  const uint16_t* gmin;     /* fp16 [rows, n_groups] or NULL */
  const uint8_t* dq_scale_codes;
  const uint16_t* dq_scale_meta; /* fp16 [n_super, 2] */
  const uint8_t* dq_gmin_codes;
  const uint16_t* dq_gmin_meta;
  int32_t dq_group_size;
  int32_t reserved0;
  const float* codebook;    /* fp32 [1<<bits] or NULL */
  int64_t n_outliers;
  const int32_t* outlier_row_ptr; /* [rows+1] CSR offsets into the tables */
  const int32_t* outlier_row;     /* row-sorted */
  const int32_t* outlier_col;
  const uint16_t* outlier_delta;  /* fp16 */
} ts_qweight;

/* ---------------------------------------------------------------------------
 * Fused dequant-GEMM:  out[M, rows] = x[M, cols] . W^T (+ outliers) (+ bias)
 *
 * Replaces triton_kernels.py:714-945 `fused_quantized_linear` (and, for
 * M > 64, the modules.py:898-922 dequantize_weight + F.linear path). Same
 * arguments in the same meaning; the output is written directly in
 * `out_dtype` (fp16, bf16 or fp32) instead of an fp32 pool buffer plus a
 * cast, and outliers are folded into the kernel's epilogue through the CSR
 * row offsets instead of an atomic post-pass.
 * x: device [M, cols] rows `x_row_stride` elements apart, fp16 or bf16.
 * bias: device [rows] in `bias_dtype`, or NULL. out: device [M, rows].
 * workspace: device memory of ts_qlinear_workspace_size() bytes, zero-filled
 * before its first use; calls leave it zeroed again. Calls that run
 * concurrently must use distinct workspaces.
 */
TS_API size_t ts_qlinear_workspace_size(const ts_qweight* w, int64_t M);

TS_API int ts_qlinear(const ts_qweight* w, const void* x, int x_dtype, int64_t M,
               int64_t x_row_stride, const void* bias, int bias_dtype, void* out,
               int out_dtype, int64_t out_row_stride, void* workspace,
               size_t workspace_bytes, void* stream);

/*
 * Gated MLP projection: out = (silu(gate) * up) . W^T (+ outliers)(+ bias),
 * with gate_up [M, 2 * cols] holding gate in columns [0, cols) and up in
 * [cols, 2 cols) (the output of a fused gate/up projection). silu(gate) and
 * the product are rounded to x_dtype as the unfused F.silu(gate) * up
 * rounds them. Decode-sized calls only (the decode kernel computes the
 * product while staging the activations): TS_ERR_UNSUPPORTED otherwise,
 * and the caller runs the product and ts_qlinear. Replaces the
 * `F.silu(gate) * up` elementwise pass in front of the reference's down
 * projection (the reference has no fused form). Workspace as ts_qlinear.
 */
TS_API int ts_qlinear_gated(const ts_qweight* w, const void* gate_up, int x_dtype, int64_t M,
               int64_t x_row_stride, const void* bias, int bias_dtype, void* out,
               int out_dtype, int64_t out_row_stride, void* workspace,
               size_t workspace_bytes, void* stream);

/*
 * One layer of a fused decode call. The reference runs each of these as a
 * QuantLinear.forward (modules.py:819-940) between plain torch ops of its
 * model (RMSNorm in front, the residual add behind); here they are folded
 * into the decode kernel:
 *   flags & TS_OP_GATED:   x rows hold [gate | up] (2 * cols): the input is
 *                          silu(gate) * up (as ts_qlinear_gated);
 *   flags & TS_OP_RMSNORM: x rows are fp32 (x_dtype TS_F32): the input is
 *                          F.rms_norm(x, norm_weight, norm_eps) rounded to
 *                          act_dtype, each token's mean square reduced in the
 *                          kernel;
 *   residual != NULL:      fp32 [M, rows] added to the result (may alias out).
 * act_dtype: the activation dtype the staged input is rounded to (fp16/bf16;
 * x_dtype for plain 16-bit inputs).
 */
#define TS_OP_GATED 1
#define TS_OP_RMSNORM 2
typedef struct ts_qlinear_op {
  const ts_qweight* w;
  const void* x;
  int64_t x_row_stride;
  int32_t x_dtype;
  int32_t flags;
  const void* bias;
  int32_t bias_dtype;
  int32_t out_dtype;
  void* out;
  int64_t out_row_stride;
  const float* norm_weight;
  float norm_eps;
  int32_t act_dtype;
  const float* residual;
  int64_t residual_row_stride;
} ts_qlinear_op;

/*
 * One fused layer call (decode-sized M; TS_ERR_UNSUPPORTED for calls the
 * decode kernel does not take: then run the unfused ops and ts_qlinear).
 * A call with no flags and no residual is ts_qlinear. Workspace as ts_qlinear.
 */
TS_API int ts_qlinear_ex(const ts_qlinear_op* op, int64_t M, void* workspace, size_t workspace_bytes,
                         void* stream);

/*
 * A chain of n_ops layers where op i + 1 reads what op i wrote (an MLP:
 * gate_up then the gated down projection; or consecutive blocks). Results
 * equal n_ops ts_qlinear_ex calls in stream order; every op is validated
 * before any runs. persistent = 0: one decode launch per layer (each starts
 * streaming its weights while the previous one finishes, by programmatic
 * dependent launch). persistent != 0, when every layer takes the decode
 * kernel in one pass with the same code layout (bits, group size, codebook,
 * double quant) and n_ops <= ts_qlinear_chain_max(): ONE launch, in which
 * layer i + 1 waits (bounded) on a grid-wide counter for layer i while the
 * weight tiles of the following layers already stream into shared memory.
 * The workspace must cover ts_qlinear_workspace_size() of every layer.
 */
TS_API int ts_qlinear_chain(const ts_qlinear_op* ops, int n_ops, int64_t M, int persistent, void* workspace,
                            size_t workspace_bytes, void* stream);
TS_API int ts_qlinear_chain_max(void);

/*
 * Allocation-free variant of ts_qlinear (no counterpart in the reference):
 * same arguments minus the workspace. The decode kernel's scratch lives in a
 * fixed per-device array of ts_qlinear_noalloc_max_scratch() bytes (512 KiB)
 * inside the library, for callers that cannot allocate device memory. A
 * call that takes the decode kernel (fewer than 65 tokens, or a layout the
 * tensor-core kernel does not cover) with a weight whose
 * ts_qlinear_workspace_size() exceeds that returns TS_ERR_UNSUPPORTED. The
 * first call on each device loads the array there and must happen before
 * any stream capture. Calls that may overlap on one device race on the
 * shared array and must be serialized.
 */
TS_API size_t ts_qlinear_noalloc_max_scratch(void);

TS_API int ts_qlinear_noalloc(const ts_qweight* w, const void* x, int x_dtype, int64_t M,
               int64_t x_row_stride, const void* bias, int bias_dtype, void* out,
               int out_dtype, int64_t out_row_stride, void* stream);

/*
 * Device error status of the qlinear kernels. Every barrier wait inside the
 * kernels is bounded (2 s); a wait that runs out makes the kernel unwind
 * (its results are then invalid) and records a code in the workspace's flag
 * (decode kernel) or in a per-device flag (tensor-core kernel). This call
 * synchronizes `stream`, reads both flags and returns TS_OK when neither is
 * set, else TS_ERR_TIMEOUT with the codes in ts_last_error(). With
 * clear != 0 it also resets the flags and the workspace's row-block
 * counters, so the workspace is usable again. workspace == NULL checks the
 * ts_qlinear_noalloc scratch array instead. No counterpart in the reference
 * (its Triton kernels have no waits).
 */
TS_API int ts_qlinear_status(void* workspace, size_t workspace_bytes, int clear, void* stream);

/* Test hook: the next qlinear kernel launch on the calling thread runs with
 * its copy producer disabled and every barrier wait limited to
 * `wait_limit_ns` (at most 2 s), so its first waits run out and the kernel
 * reports TS_ERR_TIMEOUT through ts_qlinear_status. Nothing faults or hangs:
 * the kernel returns within a few wait limits. */
TS_API int ts_test_inject_stall(uint64_t wait_limit_ns);

/* Standalone outlier correction into an fp32 result:
 *   out[m, row[k]] += x[m, col[k]] * delta[k]   for every k (any order).
 * Replaces triton_kernels.py:948-991 `apply_outlier_correction` (the path the
 * reference takes for unsorted or very large outlier tables). */
TS_API int ts_apply_outlier_correction(float* out, int64_t M, int64_t N, int64_t out_row_stride,
                                const void* x, int x_dtype, int64_t x_row_stride,
                                const int32_t* row, const int32_t* col,
                                const uint16_t* delta, int64_t n_outliers, void* stream);

/* QuantLinear outlier tables from a container's outlier stream.
 * Replaces the host decode of container.py:142-153 `_decode_outliers` plus
 * the table build of modules.py:414-448, 649-715. Inputs: the weight
 * (packed codes and metadata set; outlier fields ignored) and the stream as
 * stored: row deltas and columns as unsigned 16- or 32-bit integers
 * (index_bytes), values fp16, n entries, rows non-decreasing. Outputs
 * (device): int32 rows (prefix sums of the deltas) and columns, fp16 deltas
 * f16(value - (cb?[code] * scale + gmin)) in fp32 with the double-quant
 * metadata reconstructed in fp32, and CSR offsets row_ptr[rows + 1].
 * *bad_flag (device int) is set to 1 when an entry lies outside the weight. */
TS_API int ts_outlier_tables_from_stream(const ts_qweight* w, const void* row_delta, const void* col,
                                         int index_bytes, const uint16_t* val, int64_t n, int32_t* row_out,
                                         int32_t* col_out, uint16_t* delta_out, int32_t* row_ptr_out,
                                         int* bad_flag, void* stream);

/* ---------------------------------------------------------------------------
 * One-shot all-reduce over NVLink peer memory for tensor-parallel layers.
 * Replaces, for the row-parallel partial sums, the torch.distributed
 * all_reduce the reference's multi-GPU path would use (the reference itself
 * has no tensor parallelism; its layers run on one device).
 * Each rank allocates one exchange buffer (ts_peer_alloc, zeroed; bytes from
 * ts_peer_buffer_bytes), shares its CUDA IPC handle (ts_ipc_get_handle, 64
 * bytes) and maps the others (ts_ipc_open). ts_allreduce_oneshot then sums
 * `n` floats of `in` over the ranks (rank order, identical on every rank)
 * plus an optional `residual`, into `out` (which may alias either). Every
 * rank must make the same sequence of calls with the same n; n <= cap.
 * Waits for peers are bounded (2 s); on expiry *err_flag (device int) is
 * set to a non-zero code and the output is invalid.
 */
TS_API size_t ts_peer_buffer_bytes(int world, int64_t cap);
TS_API int ts_peer_alloc(int world, int64_t cap, void** ptr);
TS_API int ts_peer_free(void* ptr);
TS_API int ts_ipc_get_handle(void* ptr, void* handle_out);
TS_API int ts_ipc_open(const void* handle, void** ptr);
TS_API int ts_ipc_close(void* ptr);
TS_API int ts_allreduce_oneshot(void* const* peer_bufs, int rank, int world, int64_t cap, const float* in,
                                const float* residual, float* out, int64_t n, int* err_flag, void* stream);

/*
 * Decode-step attention of the Llama-shaped decoder used to measure decode
 * tok/s (no counterpart in the reference, whose models keep their own
 * attention): for each of `batch` sequences, rotary embedding of the new q
 * and k (rope_cos / rope_sin: fp32 [max_seq, head_dim / 2]), append of k and
 * v to the bf16 caches at position *pos (device int64), and grouped-query
 * attention over cache positions [0, min(attn_len, *pos + 1)).
 * qkv: bf16 [batch, (n_q + 2 n_kv) head_dim] (q heads, then k, then v);
 * caches: bf16 [batch][n_kv][max_seq][head_dim] with the given element
 * strides; out: bf16 [batch, n_q head_dim].
 */
TS_API int ts_decode_attention(const void* qkv, int64_t qkv_row_stride, int batch, int n_q, int n_kv,
                               int head_dim, const int64_t* pos, const float* rope_cos, const float* rope_sin,
                               void* k_cache, void* v_cache, int64_t cache_batch_stride,
                               int64_t cache_head_stride, int attn_len, int max_seq, void* out,
                               int64_t out_row_stride, void* stream);

/* ---------------------------------------------------------------------------
 * Paged key-value cache for sequences of unequal length (no counterpart in
 * the reference, whose models keep their own caches).
 *
 * k_pages / v_pages: fp16 or bf16 [num_pages, n_kv, page_size, head_dim] with
 * the given element strides, the same for both (multiples of 8; rows of
 * head_dim contiguous; a token-major pool is a choice of strides). Slot s of
 * sequence b lies in page page_table[b * table_stride + s / page_size] at
 * offset s % page_size; entries outside [0, num_pages) have no memory and
 * are never touched. seq_lens[b] counts the cached tokens of sequence b; a
 * negative count marks a sequence that takes no part in a call. scores
 * (fp32) and slot_pos (int32), both contiguous [num_pages, n_kv, page_size]
 * or NULL, hold each slot's accumulated attention weight and its token's
 * position; ts_paged_evict needs both. head_dim: a multiple of 16 up to 256.
 */
typedef struct ts_paged_cache {
  void* k_pages;
  void* v_pages;
  int64_t page_stride, head_stride, token_stride;
  const int32_t* page_table;  /* device [batch, max_pages] */
  int64_t table_stride;
  int32_t* seq_lens;          /* device [batch] */
  float* scores;
  int32_t* slot_pos;
  int32_t dtype;              /* TS_F16 or TS_BF16 */
  int32_t batch, n_kv, head_dim, page_size, num_pages, max_pages;
  int32_t reserved0;
} ts_paged_cache;

/*
 * Stores `tokens` new tokens per sequence in slots seq_lens[b] + t (n_new,
 * device [batch] or NULL, gives a smaller count per sequence). k / v:
 * [batch, tokens, n_kv, head_dim] in the cache's type with element strides
 * (sequence, token, head). With rotary tables (fp32 [rope_rows, head_dim / 2])
 * keys are rotated to position first[b] + t (first: device int64, or NULL for
 * the slot's number). scores (fp32 [batch, n_kv, tokens], strides (sequence,
 * head, token)) initialise the slots' scores, 0 without. Tokens without a
 * slot, a page or a rotary row are dropped. seq_lens is not changed.
 */
TS_API int ts_paged_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                           int tokens, const int32_t* n_new, const ts_paged_cache* cache, const int64_t* first,
                           const float* rope_cos, const float* rope_sin, int64_t rope_rows, const float* scores,
                           const int64_t* score_strides, void* stream);

/*
 * One decode step of grouped-query attention: for each sequence, q and k of
 * the new token are rotated to positions[b] (no rotation without tables), k
 * and v stored in slot seq_lens[b], and every query head attends over slots
 * [0, seq_lens[b]] with scores scale * q.k. With accumulate != 0 each slot's
 * score grows by the weights that the kv head's query heads gave it (the new
 * slot's starts from 0; it is set to 0 too when nothing is accumulated);
 * sequences must not share pages then, as one of two additions to the same score
 * would be lost. A
 * sequence whose count is negative, that has no page left for the token, or
 * whose position has no rotary row answers with zeros and stores nothing.
 * seq_lens is not changed. qkv, out as in ts_decode_attention, in the
 * cache's type. workspace: zero-filled once; its first
 * ts_serving_counter_bytes() are zero again after every call and the rest is scratch (one workspace may serve all
 * ts_paged_* and ts_fp4_* calls of a stream). A call's kernels pass data to
 * one another through it: host threads that launch on one stream need a
 * workspace each, or a lock around each call.
 */
TS_API size_t ts_paged_attention_workspace_size(const ts_paged_cache* cache, int n_q, int accumulate);
TS_API int ts_paged_decode_attention(const void* qkv, int64_t qkv_row_stride, int n_q, const ts_paged_cache* cache,
                                     const int64_t* positions, const float* rope_cos, const float* rope_sin,
                                     int64_t rope_rows, float scale, int accumulate, void* out,
                                     int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Cuts every sequence longer than `budget` back to `budget` slots per kv
 * head: the slots of the `recent` newest positions stay, then those of the
 * largest scores (equal scores: the lowest slot; NaN counts as -inf). Kept
 * slots at or behind `budget` move into the holes before it, both in
 * ascending order, and seq_lens becomes `budget`. A sequence's pages must
 * not be shared with another one. Workspace as ts_paged_decode_attention.
 */
TS_API size_t ts_paged_evict_workspace_size(const ts_paged_cache* cache, int budget);
TS_API int ts_paged_evict(const ts_paged_cache* cache, int budget, int recent, void* workspace,
                          size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * A paged key-value cache held in 8 bits. Pages hold codes [num_pages, n_kv,
 * page_size, head_dim] (strides in elements = bytes), `block` neighbouring slots of
 * a kv head share an fp32 scale: scales are contiguous [num_pages, n_kv, page_size /
 * block], value = code * scale. page_size and block are multiples of 16, and
 * block divides page_size. Everything else is as in ts_paged_cache.
 */
typedef enum ts_cache_code {
  TS_CACHE_INT8 = 0,    /* signed integers, -127 .. 127 */
  TS_CACHE_E4M3 = 1     /* 8-bit floating point, largest value 448 */
} ts_cache_code;

typedef struct ts_paged_cache8 {
  void* k_pages;
  void* v_pages;
  int64_t page_stride, head_stride, token_stride;
  float* k_scales;
  float* v_scales;
  const int32_t* page_table;  /* device [batch, max_pages] */
  int64_t table_stride;
  int32_t* seq_lens;          /* device [batch] */
  int32_t code;               /* ts_cache_code */
  int32_t batch, n_kv, head_dim, page_size, num_pages, max_pages, block;
} ts_paged_cache8;

/*
 * Stores new tokens of each sequence in slots seq_lens[b] + t. k / v:
 * [batch, tokens, n_kv, head_dim] of fp16 or bf16 with element strides (sequence,
 * token, head) or, with offsets (device int32 [batch + 1]), packed: sequence b's
 * tokens are rows offsets[b] to offsets[b + 1] of `tokens` in all, and the sequence
 * stride is not used. n_new (device int32 [batch], or NULL): a smaller count per
 * sequence. Rotation as ts_paged_append, k rounded to its type before it is
 * quantised. For every block of slots that gets tokens, with a = max|new values|
 * and q = 127 (TS_CACHE_INT8) or 448, in fp32:
 *   need = max(a * fp32(1 / q), 2^-100)
 *   scale = need                          the block holds no earlier tokens
 *         = old                           need <= |old|
 *         = max(need, 1.25 |old|)         otherwise; earlier codes become
 *                                         round(code * (old / scale))
 *   code = round(x * (1 / scale)), to nearest even, within +-q
 * An infinity or a NaN among a block's values makes its scale NaN (and stays
 * until the block begins anew); the new codes are 0 then. Tokens without a slot, a page or a
 * rotary row are dropped. seq_lens is not changed; codes of slots behind the last token are left alone.
 */
TS_API int ts_paged8_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                            int kv_dtype, int64_t tokens, const int32_t* offsets, const int32_t* n_new,
                            const ts_paged_cache8* cache, const int64_t* first, const float* rope_cos,
                            const float* rope_sin, int64_t rope_rows, void* stream);

/* The values of all pages, k and v contiguous [num_pages, n_kv, page_size,
 * head_dim] of out_dtype, rounded once from the fp32 product code * scale. */
TS_API int ts_paged8_dequantize(const ts_paged_cache8* cache, void* k, void* v, int out_dtype, void* stream);

/*
 * Attention of one query token per sequence over its cached tokens, slots [0,
 * seq_lens[b]): q [batch, n_q * head_dim] fp16 or bf16, out alike. With tables q is
 * rotated to positions[b]; a position without a rotary row, like a sequence
 * without tokens, answers with zeros. Slots without a page do not count. out may be q
 * (of a projection's output: its query columns), and overlaps it in no other way.
 * Workspace as ts_paged_decode_attention.
 */
TS_API size_t ts_paged8_attention_workspace_size(const ts_paged_cache8* cache, int n_q);
TS_API int ts_paged8_attention(const void* q, int q_dtype, int64_t q_row_stride, int n_q, const ts_paged_cache8* cache,
                               const int64_t* positions, const float* rope_cos, const float* rope_sin,
                               int64_t rope_rows, float scale, void* out, int64_t out_row_stride, void* workspace,
                               size_t workspace_bytes, void* stream);

/*
 * ts_paged_decode_attention for this cache: the new token's k and v (from qkv,
 * [batch, (n_q + 2 n_kv) * head_dim]) are stored by ts_paged8_append, and
 * every query head attends over slots [0, seq_lens[b]]. Workspace as above.
 */
TS_API int ts_paged8_decode_attention(const void* qkv, int qkv_dtype, int64_t qkv_row_stride, int n_q,
                                      const ts_paged_cache8* cache, const int64_t* positions, const float* rope_cos,
                                      const float* rope_sin, int64_t rope_rows, float scale, void* out,
                                      int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream);

/* ts_int8_status for the 8-bit attention's flag. */
TS_API int ts_paged8_status(int clear, void* stream);

/* ---------------------------------------------------------------------------
 * Norms of queries and keys for each head, and their rotation.
 *
 * x [tokens, (n_q + 2 n_kv) * head_dim] (fp16 or bf16, rows 16-byte aligned):
 * query heads, key heads, value heads. Query and key heads become
 *   y = x * rsqrt(mean(x^2) + eps) * w        (w: q_weight or k_weight, [head_dim]
 *                                             of weight_dtype; NULL: y = x)
 *   (y1 c - y2 s, y1 s + y2 c)                with tables, at positions[t]
 * in fp32, rounded once; values are copied. out may be x, and overlaps it in no other way. With a cache (16
 * bits, x's type) key and value heads also go to slot slots[t] (device int64: page *
 * page_size + offset) of its pages, whose score and position are set; a slot outside
 * the pool is not written. A token whose position has no rotary row gets
 * zeros and is not stored.
 */
TS_API int ts_qk_norm_rope(const void* x, int dtype, int64_t x_row_stride, int64_t tokens, int n_q, int n_kv, int head_dim,
                           const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                           const int64_t* positions, const float* rope_cos, const float* rope_sin, int64_t rope_rows,
                           void* out, int64_t out_row_stride, const ts_paged_cache* cache, const int64_t* slots,
                           void* stream);

/* ---------------------------------------------------------------------------
 * Page tables from request lengths. The pool is a stack of page numbers:
 * free_pages[0 .. n_free[0]) of `capacity` are free, the last one is taken first.
 */
typedef struct ts_page_pool {
  int32_t* free_pages;   /* device [capacity] */
  int32_t* n_free;       /* device [1] */
  int32_t capacity;
  int32_t reserved0;
} ts_page_pool;

typedef struct ts_page_table {
  int32_t* table;        /* device [batch, max_pages] */
  int64_t table_stride;
  int32_t* seq_lens;     /* device [batch] */
  int32_t batch, max_pages, page_size, num_pages;
} ts_page_table;

/*
 * Pages for n_new[b] (device; negative counts as 0) tokens behind each sequence's
 * cached ones. An entry of the table that these tokens need and that names no page of
 * [0, num_pages) gets one from the pool; sequences are served in order, all
 * or nothing, until one needs more pages than are left: it and those behind
 * it that need any get none. granted[b]: n_new[b], or 0 for a sequence that was
 * not served, is out of use (negative seq_lens) or would pass the table's end. offsets
 * [batch + 1]: where each sequence's tokens start in a packed batch of all n_new. For
 * token t < capacity `tokens` of the packed batch: sequences[t] (-1 behind the
 * last), slots[t] = page * page_size + offset (-1 without a page), positions[t] =
 * (first[b], or without first the slot's number in the sequence) of a token with a slot, 0
 * otherwise. seq_lens is not changed. There is no workspace.
 */
TS_API int ts_paged_reserve(const ts_page_pool* pool, const ts_page_table* table, const int32_t* n_new,
                            const int64_t* first, int64_t tokens, int32_t* granted, int32_t* offsets, int64_t* slots,
                            int64_t* positions, int32_t* sequences, void* stream);

/*
 * Cuts sequences back: where keep[b] (device) is not negative, seq_lens[b]
 * becomes min(seq_lens[b], keep[b]) and the pages that it no longer needs go to the
 * pool, in order of the sequences and of their pages; their entries become
 * -1. Sequences must not share such pages.
 */
TS_API int ts_paged_release(const ts_page_pool* pool, const ts_page_table* table, const int32_t* keep, void* stream);

/* ---------------------------------------------------------------------------
 * Microscaled 4-bit floating point. Elements are E2M1, the even column in a
 * byte's low nibble, columns padded with zeros to a multiple of 64:
 *   TS_NVFP4  blocks of 16 columns with an E4M3 scale s and one fp32 scale g
 *             of the tensor: value = e2m1 * (s * g)
 *   TS_MXFP4  blocks of 32 columns with an E8M0 scale: value = e2m1 * 2^(s - 127)
 * codes: [rows, padded_cols / 2]. scales: tiles of 128 rows x 4 blocks, 512
 * bytes each, the tiles of a row of tiles one after another; the byte of
 * (row r, block j) within its tile is (r % 32) * 16 + (r % 128) / 32 * 4 + j % 4.
 * Bytes of rows behind the last one are never read.
 */
typedef enum ts_fp4_format {
  TS_NVFP4 = 0,
  TS_MXFP4 = 1
} ts_fp4_format;

typedef struct ts_fp4_tensor {
  uint8_t* codes;        /* device, 16-byte aligned */
  uint8_t* scales;       /* device, 16-byte aligned */
  float* global_scale;   /* device [1] (TS_NVFP4), or NULL (counts as 1) */
  int64_t rows, cols;
  int32_t format;
  int32_t reserved0;
} ts_fp4_tensor;

/*
 * Quantises x [rows, cols] (fp16, bf16 or fp32) into t. TS_NVFP4:
 *   s = e4m3(min(max|block| * (1 / (6 g)), 448)),  e2m1(x * (1 / (s g)))
 * with every operation rounded to fp32 and both conversions to nearest even
 * (saturating); g is t->global_scale[0], which find_scale != 0 first sets to
 * max(max|x| * fp32(1 / 2688), 2^-100) over the finite elements. TS_MXFP4:
 *   s = 2^(floor(log2 max|block|) - 2), at least 2^-127;  e2m1(x / s)
 * A block that holds an infinity or a NaN gets a NaN scale and zero codes.
 * A given g outside [2^-100, 2^118] counts as the nearer bound, a NaN as the
 * lower. workspace (as of ts_paged_decode_attention): needed when find_scale is
 * set, ts_fp4_quantize_workspace_size() bytes.
 */
TS_API size_t ts_fp4_scales_bytes(int64_t rows, int64_t cols, int format);
TS_API size_t ts_fp4_quantize_workspace_size(void);
TS_API int ts_fp4_quantize(const void* x, int x_dtype, int64_t x_row_stride, const ts_fp4_tensor* t, int find_scale,
                           void* workspace, size_t workspace_bytes, void* stream);

/* The values of t in out_dtype, rounded once from e2m1 * fp32(s * g). */
TS_API int ts_fp4_dequantize(const ts_fp4_tensor* t, void* out, int out_dtype, int64_t out_row_stride, void* stream);

/*
 * out[M, N] = a . b^T (+ bias) for a [M, K] and b [N, K] of one format on the
 * block-scaled tensor cores, fp32 sums: ga * gb * sum + bias, rounded once
 * to out_dtype. Workspace as ts_paged_decode_attention.
 */
TS_API size_t ts_fp4_matmul_workspace_size(int64_t M, int64_t N, int64_t K, int format);
TS_API int ts_fp4_matmul(const ts_fp4_tensor* a, const ts_fp4_tensor* b, const void* bias, int bias_dtype, void* out,
                         int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                         void* stream);

/*
 * out[M, N] = x . w^T (+ bias): ts_fp4_quantize of x [M, cols] (with the given
 * device scale x_scale for TS_NVFP4, NULL: 1), then ts_fp4_matmul, bit for
 * bit; a few tokens in one kernel, more by way of the workspace.
 */
TS_API size_t ts_fp4_linear_workspace_size(int64_t M, int64_t N, int64_t K, int format);
TS_API int ts_fp4_linear(const void* x, int x_dtype, int64_t M, int64_t x_row_stride, float* x_scale,
                         const ts_fp4_tensor* w, const void* bias, int bias_dtype, void* out, int out_dtype,
                         int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * 8-bit integers with a scale per row: value = code * scale[row]. Codes of a
 * row lie on 16 bytes, `row_stride` bytes from the next row's; cols at most
 * 131072 (a product's sums are 32-bit integers).
 */
typedef struct ts_int8_tensor {
  int8_t* codes;         /* device, 16-byte aligned */
  int64_t row_stride;    /* a multiple of 16, at least cols rounded up to 16 */
  float* scales;         /* device [rows] */
  int64_t rows, cols;
} ts_int8_tensor;

/*
 * Quantises x [rows, cols] (fp16, bf16 or fp32) into t:
 *   scale = max(max|row| * fp32(1 / 127), 2^-100),  code = rint(x * (1 / scale))
 * with every operation rounded to fp32; columns up to the next multiple of 16
 * get codes of 0. A row that holds an infinity or a NaN gets the scale NaN and
 * codes of 0.
 */
TS_API int ts_int8_quantize(const void* x, int x_dtype, int64_t x_row_stride, const ts_int8_tensor* t, void* stream);

/* The values of t in out_dtype, rounded once from the fp32 product code * scale. */
TS_API int ts_int8_dequantize(const ts_int8_tensor* t, void* out, int out_dtype, int64_t out_row_stride, void* stream);

/*
 * out[M, N] = a . b^T (+ bias) for a [M, K] and b [N, K] on the integer tensor
 * cores: exact 32-bit sums, then (sum * smaller scale) * larger scale + bias in fp32,
 * rounded once to out_dtype. Workspace as ts_paged_decode_attention.
 */
TS_API size_t ts_int8_matmul_workspace_size(int64_t M, int64_t N, int64_t K);
TS_API int ts_int8_matmul(const ts_int8_tensor* a, const ts_int8_tensor* b, const void* bias, int bias_dtype, void* out,
                          int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream);

/* out[M, N] = x . w^T (+ bias): ts_int8_quantize of x [M, cols], then ts_int8_matmul,
 * bit for bit; by way of the workspace, or for one or two short tokens in one
 * kernel. out does not overlap x. */
TS_API size_t ts_int8_linear_workspace_size(int64_t M, int64_t N, int64_t K);
TS_API int ts_int8_linear(const void* x, int x_dtype, int64_t M, int64_t x_row_stride, const ts_int8_tensor* w,
                          const void* bias, int bias_dtype, void* out, int out_dtype, int64_t out_row_stride,
                          void* workspace, size_t workspace_bytes, void* stream);

/* ts_fp4_status for the int8 product's flag (the workspace's counters are the
 * caller's to zero). */
TS_API int ts_int8_status(int clear, void* stream);

/* Bytes at a serving workspace's start that hold counters: zero before the
 * first call and between calls. */
TS_API size_t ts_serving_counter_bytes(void);

/* ts_qlinear_status for the fp4 product (a per-device flag); with clear the
 * counters at the workspace's start are zeroed too (workspace may be NULL): no
 * call that uses it may be in flight on another stream then. Waits for
 * `stream`; covers its calls and those that other streams have finished. */
TS_API int ts_fp4_status(void* workspace, size_t workspace_bytes, int clear, void* stream);

/* Dense reconstruction W[rows, cols] in `out_dtype`.
 * Replaces triton_kernels.py:1114-1186 `dequantize_weight` (which covers only
 * 4/8-bit; this covers 2/4/8 and the double-quantized metadata). With
 * apply_outliers != 0 the outlier positions get base + delta, computed in
 * fp32, as modules.py:912-919 does before its F.linear. */
TS_API int ts_dequantize_weight(const ts_qweight* w, void* out, int out_dtype, int64_t out_row_stride,
                         int apply_outliers, void* stream);

/* ---------------------------------------------------------------------------
 * GPU quantize + pack (GOAP), replacing gpu_quantize.py:52-166
 * `quantize_tensor_gpu` and the tensor work of codec.py:453-675
 * `quantize_tensor`: top-k |w| outlier extraction and clamp, per-group affine
 * parameters, uniform / codebook / Lloyd-Max code assignment, bit packing,
 * double quantization of scale/gmin, and QuantLinear's row-sorted outlier
 * tables with their fp16 deltas (modules.py:414-448, 649-715).
 * Bit-identical to the reference codec on the same input, except that ties
 * at the top-k threshold keep the lowest flat indices.
 */
typedef enum ts_qmode {
  TS_QMODE_UNIFORM = 0,  /* round-half-even on the integer grid */
  TS_QMODE_CODEBOOK = 1, /* nearest entry of a given sorted fp32 codebook (NF) */
  TS_QMODE_LLOYD = 2     /* fit a Lloyd-Max codebook on the device, then assign */
} ts_qmode;

typedef struct ts_quant_params {
  int64_t rows, cols;
  int32_t bits, group_size;
  int64_t k_outliers;        /* codec.py:530: max(1, int(n*frac)) or 0 */
  int32_t double_quant;      /* 0/1 */
  int32_t dq_group_size;
  int32_t mode;              /* ts_qmode */
  int32_t lloyd_iters;       /* codec.py:258 default 12 */
  const float* codebook;     /* device fp32 [1<<bits], sorted (TS_QMODE_CODEBOOK) */
  const int64_t* lloyd_sample; /* device flat indices into the padded
                                  [rows, padded_cols] grid, or NULL = all */
  int64_t lloyd_n_sample;
} ts_quant_params;

typedef struct ts_quant_outputs {
  uint8_t* packed;           /* [rows, padded_cols*bits/8] */
  uint16_t* scale;           /* fp16 [rows, n_groups]; DQ-reconstructed when double_quant */
  uint16_t* gmin;
  uint8_t* dq_scale_codes;   /* [n_super*dq_group_size] (double_quant only) */
  uint16_t* dq_scale_meta;   /* fp16 [n_super, 2] */
  uint8_t* dq_gmin_codes;
  uint16_t* dq_gmin_meta;
  float* codebook_out;       /* fp32 [1<<bits]: levels the codes were assigned
                                against (Lloyd: the fitted levels), or NULL */
  uint16_t* codebook_f16;    /* fp16 [1<<bits] stored codebook (Lloyd-Max: required;
                                codebook mode: optional, and when given the
                                outlier deltas are taken against these fp16
                                levels, as for a companded weight), or NULL */
  int32_t* outlier_idx;      /* [k] flat indices, ascending */
  uint16_t* outlier_val;     /* fp16 [k] original values */
  int32_t* outlier_row;      /* [k] row-sorted (ascending flat index order) */
  int32_t* outlier_col;
  uint16_t* outlier_delta;   /* fp16 [k] val - base */
  int32_t* outlier_row_ptr;  /* [rows+1] */
  float* threshold;          /* [1] clipping magnitude (0 when no outliers), or NULL */
} ts_quant_outputs;

TS_API size_t ts_quantize_workspace_size(const ts_quant_params* p);

TS_API int ts_quantize_pack(const void* w, int w_dtype, const ts_quant_params* p,
                     const ts_quant_outputs* o, void* workspace, size_t workspace_bytes,
                     void* stream);

/* Lloyd-Max 1-D fit on device values, codec.py:320-361 (on a given sample):
 * levels_out = sorted fp32 [n_levels] after `iters` Lloyd iterations started
 * from linspace(min, max). */
TS_API size_t ts_lloyd_fit_workspace_size(int64_t n, int n_levels);
TS_API int ts_lloyd_fit(const float* values, int64_t n, int n_levels, int iters, float* levels_out,
                 void* workspace, size_t workspace_bytes, void* stream);

/* Diagnostics. */
TS_API const char* ts_last_error(void);
TS_API const char* ts_version(void);
/* Number of kernels this library launched on the calling thread since the
 * last reset (bench bookkeeping). */
TS_API int64_t ts_launch_count(int reset);

#ifdef __cplusplus
}
#endif

#endif /* TENSORSHRINK_B200_H */
