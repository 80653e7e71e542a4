/*
 * mote_hip.h: C ABI of libmote_hip.so, the MI355X (gfx950) implementation of
 * Mote's Q4_0 quantized-linear path, RMSNorm and RoPE, of the attention between
 * them, and of the MLP of a mixture of experts.
 *
 * Conventions (all of them those of the reference's Rust FFI,
 * crates/mote-backend-hip/src/ffi.rs:8-13): pointers are untyped device
 * pointers, streams are opaque `void*` hipStream_t handles, every launch is
 * asynchronous on the given stream, the caller owns every buffer, and the
 * return value is an `int` status where 0 means success.
 *
 * Symbols marked [reference] keep the exact signature, argument meaning and
 * status codes of the reference export they replace (file:line cited).
 * Symbols marked [new] have no counterpart in the reference.
 */
#ifndef MOTE_HIP_H
#define MOTE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- HIP runtime wrappers ------------------------------------------------ */
/* [reference] crates/mote-backend-hip/src/hipblaslt_shim.cpp:259-324, bound at
 * crates/mote-backend-hip/src/ffi.rs:42-61.  Raw hipError_t; -1 for a null
 * out-parameter.  mote_hip_stream_create also allocates the stream's 64 MiB
 * split-K scratch (so split-K linears on it allocate nothing up to that
 * size) and, where memory allows, 64 MiB of prompt scratch;
 * mote_hip_stream_destroy does not wait for the stream, and frees the scratch
 * once the work queued before it has completed.
 *
 * Prompt scratch: linears on the many-token tiles (more than 64 tokens, and
 * fewer where those tiles are the faster ones) never allocate.  On a stream made
 * by mote_hip_stream_create, outside graph capture, they may divide K over
 * workgroups whose partial sums meet in the stream's prompt scratch (Q4_K keeps
 * its activation sums there too).  Under capture, and on any other stream, they
 * use no scratch: Q4_K, Q6_K, Q8_0 and Q4_0 prompts then run over all of K in one
 * workgroup per tile, equal to the tolerance but not bit for bit to the divided
 * call, and up to twice as slow where K is long and the tiles are few.  So a
 * graph of such calls holds no memory of the library's: it may be replayed on
 * any stream, beside other graphs and eager calls, and after its capture stream
 * is gone. */
int mote_hip_get_device_count(int* count);
int mote_hip_set_device(int ordinal);
int mote_hip_malloc(void** pointer, size_t bytes);
int mote_hip_free(void* pointer);
int mote_hip_memcpy_host_to_device(void* destination, const void* source, size_t bytes);
int mote_hip_memcpy_device_to_host(void* destination, const void* source, size_t bytes);
int mote_hip_stream_create(void** stream);
int mote_hip_stream_destroy(void* stream);
int mote_hip_stream_synchronize(void* stream);
int mote_hip_mem_get_info(size_t* free_bytes, size_t* total_bytes);

/* ---- Q4_0 quantized linear ------------------------------------------------ */
/* [reference] crates/mote-backend-hip/src/quantized_linear.hip:56-91, bound at
 * crates/mote-backend-hip/src/ffi.rs:287-326.
 * output[rows, N] (f16) = input[rows, K] (f16) x weights[N, K]^T (GGML Q4_0,
 * rows of K/32 blocks of 18 bytes), f32 accumulation, one f16 rounding.
 * Status: null pointer or K % 32 != 0 -> 1 (hipErrorInvalidValue);
 * rows == 0 or N == 0 -> 0, nothing launched; rows * N > UINT_MAX -> 9
 * (hipErrorInvalidConfiguration); K == 0 launches and writes zeros; else the
 * launch status.  K above 2^31 - 1 (64-bit sizes, as in the reference) runs
 * per-element products over K parts of each output, added in part order, with
 * the partials in the stream's split-K scratch.  Output must not alias the
 * inputs. */
int mote_hip_quantized_linear_q4_0_f16(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);

/* [new] Same as above with an f32 output [rows, N] (the reference oracle's
 * output type, crates/mote-reference/src/quantized.rs:89-144). */
int mote_hip_quantized_linear_q4_0_f32(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);

/* [new] No counterpart in the reference.  mote_hip_quantized_linear_q4_0_f32
 * for callers that cannot allocate device memory (code under HIP graph
 * capture, serving loops or harnesses that forbid hipMalloc): the same
 * arguments, checks, statuses, plans and kernels (prompts in the stream's
 * prompt scratch included), but the split-K partial
 * tiles (1-64 tokens where K exceeds one K slice) go to the library's static
 * 16 MiB device array instead of a per-stream buffer the library allocates;
 * nothing is allocated on any call.  Every call on one GPU shares that
 * array, and it keeps the last call's contents: calls that overlap in time on
 * one GPU (several streams or threads) race.  A problem whose partial tiles
 * need more than 16 MiB (M x N x K-parts x 4 bytes) returns 2
 * (hipErrorOutOfMemory) before any launch; K above 2^31 - 1 keeps its K-part
 * partials there too. */
int mote_hip_quantized_linear_q4_0_f32_no_alloc(const void* input, const void* weights, void* output,
                                                uint64_t rows, uint64_t output_features,
                                                uint64_t input_features, void* stream);

/* [new] Fused gate/up projection: output[rows, N] (f32) =
 * silu(input . gate^T) * (input . up^T), silu(z) = z / (1 + e^-z); gate and up
 * are Q4_0 [N, K].  up_weights == NULL means gate_weights is the concatenated
 * [2N, K] matrix with the gate rows first.  Status codes as above. */
int mote_hip_q4_0_gate_up_silu_f32(const void* input, const void* gate_weights,
                                   const void* up_weights, void* output, uint64_t rows,
                                   uint64_t output_features, uint64_t input_features,
                                   void* stream);

/* [new] Q8_0 weight-only linear, the next format of the path: the reference
 * decodes Q8_0 in its oracle (crates/mote-reference/src/quantized.rs:191-195,
 * 34-byte blocks: f16 scale + 32 int8, value v * d) but has no HIP kernel for
 * it.  Weights are raw GGML Q8_0 bytes [N, K] (2-byte aligned at least);
 * arguments, outputs and status codes as for the Q4_0 entry points above. */
int mote_hip_quantized_linear_q8_0_f16(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);
int mote_hip_quantized_linear_q8_0_f32(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);

/* [new] On-device Q4_0 decode of rows x K elements to f32, bit-identical to
 * dequantize_quantized_row (crates/mote-reference/src/quantized.rs:58-74).
 * Status: null or K % 32 != 0 -> 1; empty -> 0. */
int mote_hip_dequantize_q4_0_f32(const void* weights, void* output, uint64_t rows,
                                 uint64_t input_features, void* stream);

/* ---- K-quants: Q4_K and Q6_K (256-element super-blocks) ------------------ */
/* [new] The reference defines only their geometry
 * (crates/mote-types/src/lib.rs:39-74: Q4_K 256 elements in 144 bytes,
 * 4-byte aligned; Q6_K 256 in 210 bytes, 2-byte aligned; the GGML
 * ggml-common.h layouts) and plans their block-dot path
 * (docs/roadmap.md:26-27); it has no kernel, no FFI and no oracle for them
 * (crates/mote-reference/src/quantized.rs:154-156).  These follow the
 * Q4_0 entry points' arguments and statuses, with blocks of 256 elements:
 * null pointer, K % 256 != 0, weights below the format's alignment, an odd
 * input address or an output below its element alignment -> 1; rows == 0 or
 * N == 0 -> 0; rows * N > UINT_MAX or K > 2^31 - 1 -> 9; K == 0 writes zeros.
 * output[rows, N] = input[rows, K] (f16) x weights[N, K]^T, f32
 * accumulation, one final rounding for the f16 output. */
int mote_hip_quantized_linear_q4_k_f16(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);
int mote_hip_quantized_linear_q4_k_f32(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);
int mote_hip_quantized_linear_q6_k_f16(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);
int mote_hip_quantized_linear_q6_k_f32(const void* input, const void* weights, void* output,
                                       uint64_t rows, uint64_t output_features,
                                       uint64_t input_features, void* stream);

/* [new] A Q8_0, Q4_K or Q6_K linear (format: the GGML type 8, 12 or 14) on one
 * form of the many-token tiles: tile_rows 64, 96 or 128, K divided into k_parts
 * (0: one part, no scratch; Q4_K then not on 128 rows).  The linears choose
 * among these themselves; tests use it to run each on the same problem.  K a
 * multiple of 256 up to 2^22, input and weights (Q6_K: 2-byte) 16-byte aligned;
 * 1 for anything else, 801 (hipErrorNotSupported) where the stream has no
 * prompt scratch for it, else the launch status. */
int mote_hip_prompt_linear_tiles(int format, const void* input, const void* weights, void* output,
                                 uint64_t rows, uint64_t output_features, uint64_t input_features,
                                 int output_f16, int tile_rows, int k_parts, void* stream);

/* [new] On-device decode of rows x K elements to f32 (output 4-byte
 * aligned), bit-identical to GGML's dequantize_row_q4_K / dequantize_row_q6_K.
 * Status: null, K % 256 != 0 or misaligned -> 1; empty -> 0. */
int mote_hip_dequantize_q4_k_f32(const void* weights, void* output, uint64_t rows,
                                 uint64_t input_features, void* stream);
int mote_hip_dequantize_q6_k_f32(const void* weights, void* output, uint64_t rows,
                                 uint64_t input_features, void* stream);

/* ---- Q4_0 dispatch context (per-(M, N, K) plan cache) -------------------- */
/* [new] Handle pattern of the reference's hipBLASLt plan cache
 * (crates/mote-backend-hip/src/hipblaslt_shim.cpp:326-408): create / destroy
 * / last_error, a mutex-guarded map from (M, N, K, op, output type) to the
 * kernel variant, chosen on first use by a shape heuristic or, with autotune
 * on, by timing every eligible variant and the heuristic's own pick on the
 * caller's stream.  Statuses are
 * hipError_t values; on failure last_error describes the cause. */
int mote_q4_0_dispatch_create(void** handle);
void mote_q4_0_dispatch_destroy(void* handle);
const char* mote_q4_0_dispatch_last_error(void* handle);
int mote_q4_0_dispatch_set_autotune(void* handle, int enabled);
/* Split K (K parts of one tile computed by different workgroups): enabled,
 * the tiles kernel adds the parts itself, the last workgroup of a tile to
 * finish summing them in part order (write-through partial stores and a
 * per-tile arrival counter); disabled (the default, faster on MI355X), a
 * second kernel adds them in the same order.  Results are bit-identical. */
int mote_q4_0_dispatch_set_splitk_fold(void* handle, int enabled);
/* Forces one variant by name (NULL or "" clears); tests use it to run every
 * kernel on the same problem.  A forced Q4_0 prompt variant runs its own tiles
 * over all of K, where the unforced one may choose 128-row tiles over K parts;
 * "name/P" (128-row multi-pair linear tiles, P = 2 to 8) runs it over P parts.
 * The multi-pair Q8_0 names run the exact-integer tiles of their own choice
 * where K is a multiple of 256. */
int mote_q4_0_dispatch_force_variant(void* handle, const char* name);
int mote_q4_0_dispatch_linear(void* handle, const void* input, const void* weights,
                              void* output, uint64_t rows, uint64_t output_features,
                              uint64_t input_features, int output_f16, void* stream);
int mote_q4_0_dispatch_gate_up_silu(void* handle, const void* input, const void* gate_weights,
                                    const void* up_weights, void* output, uint64_t rows,
                                    uint64_t output_features, uint64_t input_features,
                                    int output_f16, void* stream);
/* The Q8_0 linear through the same context (its own plans and variants). */
int mote_q4_0_dispatch_linear_q8_0(void* handle, const void* input, const void* weights,
                                   void* output, uint64_t rows, uint64_t output_features,
                                   uint64_t input_features, int output_f16, void* stream);
/* Name of the cached variant for a problem (gate_up_op: 0 linear, 1 gate/up,
 * 2 Q8_0 linear); hipErrorNotFound (500) when the problem has not run yet. */
int mote_q4_0_dispatch_plan(void* handle, uint64_t rows, uint64_t output_features,
                            uint64_t input_features, int gate_up_op, int output_f16,
                            char* name, size_t capacity);
/* The variant the context would plan for a problem with 256-byte aligned
 * operands (op: 0 linear, 1 gate/up, 2 Q8_0 linear): the forced variant, else
 * the shape heuristic's choice ("wide_k" for K above 2^31 - 1, which a forced
 * variant cannot run).  Host only: nothing is launched or cached, and no
 * device is needed.  hipErrorInvalidValue (1) for an empty or unsupported
 * shape, hipErrorNotFound (500) when no variant fits. */
int mote_q4_0_dispatch_select(void* handle, uint64_t rows, uint64_t output_features,
                              uint64_t input_features, int op, char* name, size_t capacity);
/* No counterpart in the reference (for the plan-table benchmark, bench.py
 * --plan-table): the comma-separated names of the variants the autotuner
 * would time for a problem with 256-byte aligned operands, the rule-based
 * heuristic's pick included.  Host only.  hipErrorInvalidValue (1) for an
 * empty or unsupported shape or a buffer too small for the list. */
int mote_q4_0_dispatch_candidates(void* handle, uint64_t rows, uint64_t output_features,
                                  uint64_t input_features, int op, char* names, size_t capacity);
int mote_q4_0_variant_count(void);
const char* mote_q4_0_variant_name(int index);

/* ---- Dense F16 x F16 -> F32 matmul (hipBLASLt) ---------------------------- */
/* [reference] crates/mote-backend-hip/src/hipblaslt_shim.cpp:326-408, bound at
 * crates/mote-backend-hip/src/ffi.rs:329-417 for matmul_f16_f32
 * (crates/mote-backend-hip/src/matmul.rs:10-52).  Row-major C[m, n] (f32) =
 * A[m, k] B[k, n] (f16), f32 accumulation, on `stream`, with a caller-owned
 * workspace (the reference passes 32 MiB).  A context caches one plan per
 * (m, n, k); the first call for a shape times hipBLASLt's heuristic
 * candidates on the stream (synchronising it) and keeps the fastest.
 * Statuses: 0; -1 for a null argument or an internal error; hipBLAS
 * statuses from the library; -1000 - hipError for HIP runtime failures;
 * last_error describes the most recent failure ("" after a success).
 * m == 0 or n == 0 returns 0 without a launch; k == 0 writes zeros. */
int mote_hipblaslt_create(void** handle);
void mote_hipblaslt_destroy(void* handle);
const char* mote_hipblaslt_last_error(void* handle);
int mote_hipblaslt_matmul_f16_f32(void* handle, uint64_t m, uint64_t n, uint64_t k, const void* lhs,
                                  const void* rhs, void* output, void* workspace, size_t workspace_bytes,
                                  void* stream);

/* ---- RMSNorm and fused add + RMSNorm -------------------------------------- */
/* [reference] crates/mote-backend-hip/src/rms_norm.hip:68-98, bound at
 * crates/mote-backend-hip/src/ffi.rs:120-161.  f16 [rows, hidden] in/out,
 * f16 weight [hidden], f32 arithmetic.  -1 for null pointers or rows >
 * UINT32_MAX; rows == 0 or hidden == 0 -> 0 without a launch. */
int mote_hip_rms_norm_f16(const void* input, const void* weight, void* output, uint64_t rows,
                          uint64_t hidden_size, float epsilon, void* stream);

/* [reference] crates/mote-backend-hip/src/fused_add_rms_norm.hip:99-138,
 * bound at crates/mote-backend-hip/src/ffi.rs:163-219.  s = input + residual
 * in f32; output = f16(s * rsqrt(mean(s^2) + eps) * weight); residual <-
 * f16(s).  input may alias output; output == residual, a non-finite or
 * negative epsilon, null pointers or rows > UINT32_MAX -> -1. */
int mote_hip_fused_add_rms_norm_f16(const void* input, void* residual, const void* weight,
                                    void* output, uint64_t rows, uint64_t hidden_size,
                                    float epsilon, void* stream);

/* ---- RoPE ------------------------------------------------------------------ */
/* [reference] crates/mote-backend-hip/src/rope.hip:99-150, bound at
 * crates/mote-backend-hip/src/ffi.rs:221-285.  f16 [tokens, heads, head_dim]
 * in/out (may alias), f32 cos/sin [tokens, rotary_dim / 2]; layout 0 =
 * half-split (pairs j, j + R/2), 1 = interleaved (2j, 2j + 1); the tail past
 * rotary_dim is copied.  -1 for null input/output/stream, null cos/sin with
 * rotary_dim > 0, an unknown layout, an odd or oversized rotary_dim, or
 * tokens * heads > UINT32_MAX; any zero dimension -> 0 without a launch. */
int mote_hip_rope_f16(const void* input, const void* cos, const void* sin, void* output,
                      uint64_t tokens, uint64_t heads, uint64_t head_dim, uint64_t rotary_dim,
                      uint32_t layout, void* stream);

/* [new] q and k rotated in one launch with the shared cos/sin rows; same
 * semantics and status codes as mote_hip_rope_f16 applied to each tensor. */
int mote_hip_rope_qk_f16(const void* q_input, const void* k_input, const void* cos,
                         const void* sin, void* q_output, void* k_output, uint64_t tokens,
                         uint64_t q_heads, uint64_t k_heads, uint64_t head_dim,
                         uint64_t rotary_dim, uint32_t layout, void* stream);

/* [new] cos/sin tables [tokens, rotary_dim / 2] from int64 positions:
 * inv_j = theta^(-2j / rotary_dim), angle = position * inv_j, computed in
 * binary64 and rounded to binary32.  -1 for null pointers, an odd rotary_dim
 * or theta <= 0. */
int mote_hip_rope_tables_f32(const void* positions, void* cos_out, void* sin_out,
                             uint64_t tokens, uint64_t rotary_dim, double theta, void* stream);

/* ---- Attention over packed prompts ----------------------------------------- */
/* [new] No counterpart in the reference.  Sequences of different lengths lie one
 * behind the other: sequence s has query rows query_offsets[s] up to
 * query_offsets[s + 1] and key rows key_offsets[s] up to key_offsets[s + 1]
 * (int32, sequences + 1 of each, on the device, ascending from 0 to query_tokens
 * and key_tokens; key_offsets NULL: the query offsets).  q and output are f16
 * rows of q_heads x head_dim, k and v of kv_heads x head_dim, a row `stride`
 * elements after the one before; query head h reads key head
 * h / (q_heads / kv_heads).  Query i of a sequence with n queries and t keys has
 * position i + t - n: with causal = 1 it sees the keys up to its position, and
 * with window > 0 only the last `window` of those; with causal = 0 all t keys
 * (window must be 0).  output = softmax(scale q k^T) v over the keys seen, in f32
 * with one f16 rounding (the weights of the second product are rounded to f16);
 * a query that sees none, or only scores of -infinity, gets zeros.  Keys and values
 * that a query does not see do not touch its output, whatever they hold; of those it
 * sees, a NaN shows as NaN and an infinity as an infinity or NaN.  max_keys: at least the longest
 * sequence's keys (it only chooses how the work is divided).
 * Few rows over many keys are computed in parts that a second launch joins, in
 * `workspace` (16-byte aligned, at least the bytes that
 * mote_hip_prompt_attention_workspace says for the same sizes, which may be 0);
 * it holds nothing between calls.  The output may be q itself (same stride), and
 * must not overlap k or v.  Offsets that run past the rows there are cut to them;
 * output rows that no sequence owns are left as they are.
 * Nothing is allocated, and a call can be captured.
 * Status: 0; -1 for a null pointer (key_offsets, and a workspace of which 0 bytes
 * are needed, excepted), an odd f16 or misaligned offsets address, head_dim not a
 * multiple of 8 or above 256, q_heads not a multiple of kv_heads or above 65535,
 * an output stride below q_heads x head_dim, a scale that is not finite and
 * positive, causal other than 0 or 1, a window without causal, key_offsets NULL
 * with key_tokens other than query_tokens, more than 2^30 rows or sequences or
 * 2^32 - 1 query rows x heads, too small a workspace; the launch status.  No sequence, query, head or dimension: 0 without
 * a launch. */
int mote_hip_prompt_attention_workspace(uint64_t sequences, uint64_t query_tokens, uint64_t key_tokens,
                                        uint64_t max_keys, uint64_t q_heads, uint64_t kv_heads,
                                        uint64_t head_dim, size_t* bytes);
int mote_hip_prompt_attention_f16(const void* q, const void* k, const void* v, void* output,
                                  const void* query_offsets, const void* key_offsets, uint64_t sequences,
                                  uint64_t query_tokens, uint64_t key_tokens, uint64_t max_keys,
                                  uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim, uint64_t q_stride,
                                  uint64_t k_stride, uint64_t v_stride, uint64_t output_stride, float scale,
                                  int causal, uint64_t window, void* workspace, size_t workspace_bytes,
                                  void* stream);

/* ---- Keys and values in 8 bits ----------------------------------------------- */
/* [new] No counterpart in the reference.  The cache is cache_blocks blocks of 32
 * tokens; sequence s's tokens 32 b .. 32 b + 31 are in block
 * block_table[s x table_blocks + b] (int32).  With P = head_dim rounded up to a
 * multiple of 32, `cache` is uint8 [cache_blocks][kv_heads][2][32 P] (planes of
 * keys and of values, 16-byte aligned) and `scales` float
 * [cache_blocks][kv_heads][2], not negative; byte u of a plane stands for (u - 128) x
 * its scale.
 * With c = d / 32, element (token t of the block, dimension d) is byte
 *   keys:   [c][(d % 32) / 8][t % 16][t / 16][d % 8]                of [P/32][4][16][2][8]
 *   values: [c][(t % 16) / 4][d % 16][(d % 32) / 16][4 (t/16) + t%4]  of the same.
 *
 * append: rows offsets[s] up to offsets[s + 1] of k and v (f16, kv_heads x
 * head_dim, `stride` elements apart) become sequence s's tokens from
 * positions[s] on (int32).  A plane's scale is the largest magnitude of its
 * tokens over 127, a byte 128 + the rounded quotient (ties to even).  Tokens
 * that join a block begun earlier (positions[s] not a multiple of 32) keep its
 * scale unless one needs a larger one; the block's bytes are then rounded again
 * to the larger scale.  A block written from its first token on starts anew,
 * whatever it held, with bytes of 128 in the slots not written.  An infinity or NaN makes its plane's scale NaN, so that
 * every read of the plane shows it, until the block starts anew.  Blocks shared
 * by sequences must not be appended to.
 *
 * read: the same rows the other way: tokens of sequence s from positions[s] on,
 * as many as its rows, to k and v, (u - 128) x scale rounded to f16.
 *
 * Tokens past the table, and those of blocks whose number is not below
 * cache_blocks, are left out.  Nothing is allocated, and a call can be captured.
 * Status: 0; -1 for a null pointer, an odd f16 address, int32 or float arrays off
 * their alignment, a cache off the 16-byte grid, head_dim not a multiple of 8 or
 * above 256, more than 65535 heads, 2^30 tokens or sequences or 2^25 blocks of a
 * sequence (for read, a stride below kv_heads x head_dim); the launch status.  No sequence,
 * token, head or dimension: 0 without a launch. */
int mote_hip_kv_cache_append_q8(const void* k, const void* v, const void* offsets, const void* positions,
                                const void* block_table, void* cache, void* scales, uint64_t sequences,
                                uint64_t tokens, uint64_t kv_heads, uint64_t head_dim, uint64_t k_stride,
                                uint64_t v_stride, uint64_t table_blocks, uint64_t cache_blocks, void* stream);
int mote_hip_kv_cache_read_q8_f16(const void* cache, const void* scales, const void* offsets,
                                  const void* positions, const void* block_table, void* k, void* v,
                                  uint64_t sequences, uint64_t tokens, uint64_t kv_heads, uint64_t head_dim,
                                  uint64_t k_stride, uint64_t v_stride, uint64_t table_blocks,
                                  uint64_t cache_blocks, void* stream);

/* [new] Attention of the last tokens of each sequence over the cache: sequence s
 * holds lengths[s] tokens (int32, its queries' own included), and its n query
 * rows, query_offsets[s] up to query_offsets[s + 1] (NULL: row s alone), are the
 * last n of them: query i has position lengths[s] - n + i and sees the tokens up
 * to it, with window > 0 only the last `window` of those.  Formula, heads,
 * strides, types, rows that see nothing, workspace and statuses as for the prompt
 * attention above, with the cache's values (u - 128) x scale for k and v; the
 * cache's own requirements as for append.  max_queries: at least the largest n
 * (the output rows of a sequence's queries past it, like those that no sequence
 * owns, are left as they are); max_context: at least the largest length (it
 * only chooses how the work is divided).  query_offsets NULL needs query_tokens =
 * sequences and max_queries = 1.  Blocks whose number is not below cache_blocks
 * count as not there.  A plane whose scale is NaN makes every query NaN that
 * sees one of its tokens.  Nothing is allocated, and a call can be captured.
 * Status -1 also for max_queries x q_heads from 2^31 on and for more than 2^32 - 1
 * workgroups, of which a sequence takes at most one for each key head, 16 rows
 * (queries x heads of the key head) and part. */
int mote_hip_cache_attention_workspace(uint64_t sequences, uint64_t query_tokens, uint64_t max_queries,
                                       uint64_t max_context, uint64_t q_heads, uint64_t kv_heads,
                                       uint64_t head_dim, size_t* bytes);
int mote_hip_cache_attention_q8_f16(const void* q, const void* cache, const void* scales,
                                    const void* query_offsets, const void* lengths, const void* block_table,
                                    void* output, uint64_t sequences, uint64_t query_tokens,
                                    uint64_t max_queries, uint64_t max_context, uint64_t q_heads,
                                    uint64_t kv_heads, uint64_t head_dim, uint64_t q_stride,
                                    uint64_t output_stride, uint64_t table_blocks, uint64_t cache_blocks,
                                    float scale, uint64_t window, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* ---- Microscaled formats ----------------------------------------------------- */
/* [new] No counterpart in the reference.  Rows of `features` elements (a multiple of
 * 32) in blocks of 32 with a scale each.  With Kp = features rounded up to a multiple
 * of 128, `values` is uint8 [rows][Kp bits / 8] (16-byte aligned) and `scales` uint8
 * [rows][Kp / 32]; what of a row lies past `features` is zeros.  A scale byte b
 * stands for 2^(b - 127), 255 for not a number.  bits = 4: E2M1, code c (its top bit
 * the sign) for 0, 0.5, 1, 1.5, 2, 3, 4, 6; bits = 6: E2M3, 0 to 1.875 in eighths, to
 * 3.75 in quarters, to 7.5 in halves.  Element i of a block is bits (bits x i) up to (bits x
 * (i + 1)) of its 4 x bits bytes, lowest first.  Block n's first 16 bytes are at 16 n of its
 * row, its other 8 (bits = 6) at Kp / 2 + 8 n.  (4-bit rows of a multiple of 128
 * elements are those of the published MXFP4 format, two elements a byte, the first in the
 * low half.)
 *
 * quantize: rows `input_stride` elements apart.  Scale 2^(floor(log2 m) - 2), m the
 * block's largest magnitude, at least 2^-127; elements rounded to the nearest, ties to
 * the even code, held to +-6 or +-7.5.  A block of zeros has scale byte 0; one with an infinity or
 * NaN has 255 and zeros.  Writes the padding too.
 * dequantize: element x 2^(b - 127) rounded once to the output's type, to rows
 * `output_stride` apart; what lies between the rows is left as it is.  Neither works in place.
 * Status: 0; -1 for a null pointer, bits other than 4 or 6, features not a multiple of
 * 32 or above 2^24, a stride below features or above 2^40, more than 2^31 rows or 2^32 - 257 blocks
 * (padding included), values off the 16-byte grid, f16 or f32 off their alignment; the
 * launch status.  No row or feature: 0 without a launch. */
int mote_hip_mx_quantize_f16(const void* input, void* values, void* scales, uint64_t rows, uint64_t features,
                             uint64_t input_stride, int bits, void* stream);
int mote_hip_mx_quantize_f32(const void* input, void* values, void* scales, uint64_t rows, uint64_t features,
                             uint64_t input_stride, int bits, void* stream);
int mote_hip_mx_dequantize_f16(const void* values, const void* scales, void* output, uint64_t rows,
                               uint64_t features, uint64_t output_stride, int bits, void* stream);
int mote_hip_mx_dequantize_f32(const void* values, const void* scales, void* output, uint64_t rows,
                               uint64_t features, uint64_t output_stride, int bits, void* stream);

/* [new] output[rows, N] = input[rows, K] x weights[N, K]^T, the weights in 4 bits, the
 * input in input_bits (4 or 6), f32 accumulation, one rounding to the output's type.  A
 * scale that is not a number shows as NaN in the outputs of its row.
 * Status: 0; -1 for a null pointer, input_bits other than 4 or 6, K not a multiple of
 * 32, K or N above 2^24, more than 2^30 rows, values off the 16-byte grid or scales off the 4-byte
 * one, an output off its alignment, more work than one launch holds (2^36 outputs where K is
 * at most 384, 2^40 else, each side counted in whole tiles of up to 256); the launch status.
 * rows == 0 or N == 0: 0 without a launch; K == 0 writes zeros.  Output must not alias the inputs.
 * Nothing is allocated, and a call can be captured. */
int mote_hip_mx_linear_f16(const void* input_values, const void* input_scales, const void* weight_values,
                           const void* weight_scales, void* output, uint64_t rows, uint64_t output_features,
                           uint64_t input_features, int input_bits, void* stream);
int mote_hip_mx_linear_f32(const void* input_values, const void* input_scales, const void* weight_values,
                           const void* weight_scales, void* output, uint64_t rows, uint64_t output_features,
                           uint64_t input_features, int input_bits, void* stream);

/* ---- Experts -------------------------------------------------------------------- */
/* [new] No counterpart in the reference.  The `top` experts of each token: logits
 * [tokens, experts] -> ids (int32) and weights (float), [tokens, top] each, the best first.
 * score 0: softmax over the experts; 1: sigmoid.  The choice is by score + bias[expert]
 * (float), by the logit where bias is NULL, for both scores grow with it; equal choices go by the logit,
 * then the lowest index first; the bias is not in the weights.
 * With top_groups < groups the experts are `groups` runs of experts / groups; a group's
 * worth is the sum of its group_best (1 or 2) best choices, as many as it has, and only the experts of
 * the top_groups best groups are chosen.  weights = scale x score, divided by the chosen
 * scores' sum with renormalize = 1 (0 where that is 0).  An expert whose logit, or whose score +
 * bias, is infinite or NaN takes no part (a logit that is, not in the softmax either);
 * where fewer than `top` are left the ids are -1 and the weights 0, so a row of
 * -infinity is a token without experts.  Scores are held in 64 bits: choices of different biases, and
 * worths, that differ by less than 2^-50 (of the larger, or of 1) can come in either order; a score under 2^-1022,
 * of a softmax's logit 708 below the largest or a sigmoid's below -708, can be 0 in the weights and in the worth of two.
 * Status: 0; -1 for a null pointer (bias excepted), logits, bias, ids or weights off
 * their alignment, score or renormalize other than 0 or 1, group_best other than 1 or 2, a scale that is
 * not finite, more than 1024 experts, top above 64 or above the experts that the groups leave, groups that do not
 * divide the experts or top_groups not in 1 .. groups, more than 2^26 - 4 tokens
 * or 2^30 pairs; the launch status.  No token, expert or top: 0 without a launch. */
int mote_hip_route_experts_f16(const void* logits, const void* bias, void* ids, void* weights, uint64_t tokens,
                               uint64_t experts, uint64_t top, int score, uint64_t groups, uint64_t top_groups,
                               int group_best, int renormalize, float scale, void* stream);
int mote_hip_route_experts_f32(const void* logits, const void* bias, void* ids, void* weights, uint64_t tokens,
                               uint64_t experts, uint64_t top, int score, uint64_t groups, uint64_t top_groups,
                               int group_best, int renormalize, float scale, void* stream);

/* [new] The plan of the experts' products: the pairs (token t, choice j), numbered
 * top x t + j, in the order of their experts and within one of their numbers.  rows (int32
 * [tokens x top]): the pairs; expert e has rows offsets[e] up to offsets[e + 1] (int32
 * [experts + 1]).  A pair whose id is not in 0 .. experts - 1 has no row; the rows
 * past offsets[experts] are -1.  None of the arrays may overlap another.
 * Status: 0; -1 for a null pointer, int32 arrays off their alignment, more than 1024
 * experts, top above 64, 2^30 pairs or tokens; the launch status.  No expert: 0 without a launch. */
int mote_hip_plan_experts(const void* ids, void* offsets, void* rows, uint64_t tokens, uint64_t top,
                          uint64_t experts, void* stream);

/* [new] The experts' gate and up projections: row i of output (f16 [tokens x top, inner]) is,
 * for the pair rows[i] of token t and expert e, silu(x_t Wg_e^T) (x_t Wu_e^T), in f32 with one
 * rounding; x [tokens, hidden] in input_bits, weights 4-bit rows [experts][2 inner] of
 * `hidden`, an expert's gate rows first.  Rows past offsets[experts] are left as they are.
 *
 * The down projection: output[t] (f16 [tokens, hidden]) = the sum over j of pair_weights[t, j]
 * h_(t, j) W_e^T, in the order of j in f32 (a pair that the plan leaves out adds nothing; a
 * token with none gets zeros); row i of the input (h, `inner` elements in input_bits) is that of pair
 * rows[i], weights 4-bit rows [experts][hidden] of `inner`.  The pairs' products meet in `workspace`
 * (16-byte aligned, at least the bytes that mote_hip_experts_down_workspace says for the same
 * sizes); it holds nothing between calls, and calls that overlap need their own.  ids and
 * plan must belong together.
 *
 * Offsets that run past the pairs are cut to them, and a row that names no pair reads
 * token 0 or is left out.  Outputs and workspace must not alias inputs.  Nothing is allocated, and a
 * call can be captured.
 * Status: 0; -1 for a null pointer (a workspace of which 0 bytes are needed excepted), operands as for
 * mx_linear, int32 or float arrays off their alignment, hidden or inner not a multiple of 32 or
 * above 2^24, more than 1024 experts, top above 64, 2^30 pairs or tokens, too small a
 * workspace, more work than one launch holds; the launch status.  No output: 0 without a launch. */
int mote_hip_experts_gate_up_silu_mx_f16(const void* input_values, const void* input_scales,
                                         const void* weight_values, const void* weight_scales, const void* offsets,
                                         const void* rows, void* output, uint64_t tokens, uint64_t top,
                                         uint64_t experts, uint64_t hidden, uint64_t inner, int input_bits,
                                         void* stream);
int mote_hip_experts_down_workspace(uint64_t tokens, uint64_t top, uint64_t experts, uint64_t hidden, uint64_t inner,
                                    size_t* bytes);
int mote_hip_experts_down_mx_f16(const void* input_values, const void* input_scales, const void* weight_values,
                                 const void* weight_scales, const void* ids, const void* offsets, const void* rows,
                                 const void* pair_weights, void* output, uint64_t tokens, uint64_t top,
                                 uint64_t experts, uint64_t hidden, uint64_t inner, int input_bits, void* workspace,
                                 size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MOTE_HIP_H */
