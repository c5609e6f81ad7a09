/*
 * include/prima_b200.h — C ABI of libprima_b200.so, the B200-native (sm_100a) quantized-decode hot path of prima.cpp.
 *
 * Plain pointers and sizes only; no torch / ggml types.  All functions return 0 on success, a cudaError_t (>0) for
 * CUDA failures or a negative PB200_E* code for argument errors; nothing throws or aborts across the ABI.
 * Device pointers are raw CUDA device addresses, `stream` is a cudaStream_t passed as void* (NULL = default stream).
 *
 * What each entry point replaces in the reference (paths within its project):
 *   pb200_mul_mat_vec*      ggml_cuda_mul_mat -> ggml_cuda_op_mul_mat_vec_q -> mul_mat_vec_q<type,1>
 *                           ggml/src/ggml-cuda.cu:1883-1948, ggml-cuda/mmvq.cu:55-202, vecdotq.cuh:357-787
 *                           (+ the per-call quantize_row_q8_1_cuda, quantize.cu:129-141); CPU semantics:
 *                           ggml_compute_forward_mul_mat ggml/src/ggml.c:12377-12600
 *   pb200_quantize_act      quantize_q8_1 quantize.cu:4-38; CPU: quantize_row_q8_K_ref ggml-quants.c:3785-3822
 *   pb200_rms_norm          ggml_cuda_op_rms_norm norm.cu:206-224; CPU ggml.c:11950-11996
 *   pb200_rope              ggml_cuda_op_rope rope.cu:188-271; CPU ggml.c:14143-14266
 *   pb200_soft_max          ggml_cuda_op_soft_max softmax.cu:170-206; CPU ggml.c:13783-13880
 *   pb200_attn_decode       FA-off attention chain: ggml_cuda_mul_mat_batched_cublas x2 + soft_max + cont,
 *                           ggml-cuda.cu:1737-1881; graph src/llama.cpp:10032-10165
 *   pb200_mul_mat_q         ggml_cuda_op_mul_mat_q mmq.cu:3-98 -> mul_mat_q<type,...> mmq.cuh:2583-2650 (+ quantize_mmq_q8_1_cuda
 *                           quantize.cu:143-169): the batched / prefill product, here on tcgen05 + TMEM
 *   pb200_get_rows          ggml_cuda_op_get_rows getrows.cu (k-quant rows are unsupported there, ggml-cuda.cu:3033-3047)
 *   pb200_model_* / pb200_decode*   the per-token loop ggml_backend_cuda_graph_compute ggml-cuda.cu:2508-2778 over the
 *                           graph of build_llama / build_qwen2 (src/llama.cpp:11000-11216, 12736-12916) — one fused,
 *                           CUDA-graph-replayed launch sequence instead of ~30 launches per layer
 *   (the ggml-backend plugin that exposes the same kernels through ggml_backend_reg/device/buffer vtables is
 *    include/ggml_b200.h)
 */
#ifndef PRIMA_B200_H
#define PRIMA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PB200_API __attribute__((visibility("default")))

/* enum ggml_type values used on this path (ggml/include/ggml.h:356-395) */
enum { PB200_TYPE_F32 = 0, PB200_TYPE_F16 = 1, PB200_TYPE_Q5_1 = 7, PB200_TYPE_Q8_0 = 8, PB200_TYPE_Q4_K = 12, PB200_TYPE_Q5_K = 13, PB200_TYPE_Q6_K = 14,
       PB200_TYPE_BF16 = 30 /* dense weights of the layer-list family */ };

enum { PB200_EINVAL = -1, PB200_ENOMEM = -2, PB200_ENOTSUP = -3, PB200_ESTATE = -4, PB200_EABORTED = -5 };

/* ---- library ---- */
PB200_API const char * pb200_version(void);
PB200_API const char * pb200_error_string(int code);
PB200_API int          pb200_device_count(void);
PB200_API int          pb200_sm_count(void);              /* of the current device */
PB200_API int64_t      pb200_row_bytes(int type, int64_t k);   /* ggml_row_size */
PB200_API uint64_t     pb200_kernel_launches(void);       /* kernels launched by this library since load (bench `gpu_launches`) */
PB200_API void         pb200_kernel_launches_add(uint64_t n);   /* a host that replays a CUDA graph of this library's launches accounts for them here */

/* ---- single ops, device buffers ---- */
/* workspace for the quantized activation of length k (any mode): bytes to allocate */
PB200_API size_t pb200_act_workspace_bytes(int64_t k);
/* x[k] f32 -> activation workspace in the format the CPU backend uses for weight type wtype (q8_K / q8_0 / q8_1) */
PB200_API int pb200_quantize_act(int wtype, const float * x, int64_t k, void * act_ws, void * stream);
/* y[n] = W[n][k] . x   with W raw GGUF blocks of `type`; act_ws from pb200_quantize_act(type, x, k).
 * W must be 16-byte aligned and its allocation padded to a multiple of 16 bytes (+16): the kernel moves whole 16-byte units and
 * may read up to 15 bytes past the last row (Q6_K / Q8_0 rows are not multiples of 16 bytes).  ggml-backend buffers of the B200
 * plugin and pb200_model_set_tensor pad for you. */
PB200_API int pb200_mul_mat_vec_q(int type, const void * W, int64_t n, int64_t k, const void * act_ws, float * y,
                                  const float * bias, const float * resid, void * stream);
/* convenience: quantize + mul_mat_vec in one call (what ggml_cuda_mul_mat does for ne11 == 1).  y may lie over x. */
PB200_API int pb200_mul_mat_vec(int type, const void * W, int64_t n, int64_t k, const float * x, float * y, void * act_ws, void * stream);
/* up to 3 matrices sharing one activation, one fused launch (q|k|v, gate|up) */
PB200_API int pb200_mul_mat_vec_fused(int nmat, const int * types, const void * const * W, const int64_t * n, int64_t k,
                                      const void * act_ws, float * const * y, void * stream);
/* HOST buffers end to end (H2D of x, quantize, GEMV, D2H of y, synchronised): W must already be on the device */
PB200_API int pb200_mul_mat_vec_host(int type, const void * W_dev, int64_t n, int64_t k, const float * x_host, float * y_host);

/* profiling: while a buffer is set, k_gemv_kquant runs its instrumented instantiation: launch i writes row (i % slots) of
 * dev_buf (rows of 4096 u64), CTA c its 8 entries [8c .. 8c+7]: [0..5] %globaltimer (ns) at CTA start / ring fill issued /
 * dependency resolved (griddepcontrol.wait returned) / activation in registers / first tile landed / done, [6], [7] clock64 at
 * the first and last stamp.  NULL or slots = 0 switches back to the uninstrumented kernel. */
PB200_API int pb200_debug_set_trace(void * dev_buf, int slots);
/* Every in-kernel wait is bounded (~1 s of SM clocks).  A wait that gives up ends its launch quickly with invalid results and
 * the call that synchronises on it (pb200_decode, pb200_synchronize, pb200_prefill) returns PB200_EABORTED once; the flag
 * re-arms, later calls are unaffected.  Callers that only use the single-op entry points on their own streams poll this after
 * synchronising: returns 1 (and clears the flag) if any launch of this process gave up since the last call. */
PB200_API int pb200_aborted(void);

PB200_API int pb200_rms_norm(const float * x, float * y, int64_t n, int64_t nrows, float eps, void * stream);
PB200_API int pb200_rope(const float * x, float * y, int64_t n_tokens, int n_head, int head_dim, int n_dims, int mode, const int32_t * pos,
                         float freq_base, float freq_scale, float ext_factor, float attn_factor, float beta_fast, float beta_slow,
                         int n_ctx_orig, const float * freq_factors, void * stream);
/* The tokens of a prompt with heads of 128: q [T][n_head][128] rotated in place, rope(k) and v as f16 to rows pos[t] of caches [.][n_head_kv][128].
 * PB200_ENOTSUP for rotated sizes that are no multiple of 8 and arrays that are not 16-byte aligned. */
PB200_API int pb200_rope_kv_prompt(float * q, const float * k, const float * v, void * kcache, void * vcache, int64_t n_tokens, int n_head, int n_head_kv, int n_dims,
                                   int mode, const int32_t * pos, float freq_base, float freq_scale, float ext_factor, float attn_factor, float beta_fast,
                                   float beta_slow, int n_ctx_orig, const float * freq_factors, void * stream);
PB200_API int pb200_soft_max(const float * x, const float * mask, float * y, int64_t ncols, int64_t nrows, int64_t mask_rows, float scale, void * stream);
PB200_API int pb200_silu_mul(const float * gate, const float * up, float * y, int64_t n, void * stream);
/* element-wise glue of the graph (binbcast.cu / unary.cu / cpy.cu): y = a (+|*) b[i % nb]  (op 0 add, 1 mul); y = silu(x);
 * 4-D strided copy f32 -> f32|f16 (byte strides; dst logical order) — CPY / CONT / DUP incl. the transposed V-cache store */
PB200_API int pb200_binary(int op, const float * a, const float * b, float * y, int64_t n, int64_t nb, void * stream);
PB200_API int pb200_silu(const float * x, float * y, int64_t n, void * stream);
PB200_API int pb200_copy_strided(const void * src_f32, void * dst, int dst_is_f16, const int64_t * ne, const int64_t * src_strides,
                                 const int64_t * dst_strides, void * stream);
/* d[i0,i1,i2,i3] = sum_k a_f16[k,i0,i2/r2,i3/r3] * f16(b[k,i1,i2,i3]) — the FA-off KQ / KQV products (ggml-cuda.cu:1737-1881), byte strides */
PB200_API int pb200_mul_mat_f16(const void * a_f16, const float * b_f32, float * d, int64_t k, const int64_t * ne, int64_t r2, int64_t r3,
                                const int64_t * a_strides, const int64_t * b_strides, const int64_t * d_strides, void * stream);
/* batched (prefill) product: dst[t][n] = sum_k W[n][k] * x[t][k] (+ bias[n]) (+ resid[t][n]); W: n rows of k-quant blocks
 * (Q4_K/Q5_K/Q6_K with k % 256 == 0, or Q8_0/Q5_1 with k % 64 == 0), x: t rows of ldx floats, dst / resid: t rows of n floats, resid must not alias dst; W and x 16-byte aligned, ldx % 4 == 0.  Activations are quantized like the CPU backend does for that weight type (q8_K, or q8_0/q8_1 per 32 values),
 * then both operands run as fp16 on the tensor cores with fp32 accumulation.  ws: pb200_mul_mat_q_workspace_bytes(k, t). */
PB200_API size_t pb200_mul_mat_q_workspace_bytes(int64_t k, int64_t t);
PB200_API int pb200_mul_mat_q(int type, const void * W, int64_t n, int64_t k, const float * x, int64_t ldx, int64_t t, float * dst,
                              const float * bias, const float * resid, void * ws, void * stream);
PB200_API int pb200_get_rows(int type, const void * table, int64_t k, const int32_t * ids, int64_t n_ids, float * y, void * stream);
/* decode attention over an f16 KV cache laid out [n_ctx][n_head_kv*head_dim]; n_kv = *pos_dev + 1 */
PB200_API int pb200_attn_decode(const float * q, const void * k_cache_f16, const void * v_cache_f16, float * out, int n_head, int n_head_kv,
                                int head_dim, const int32_t * pos_dev, int n_ctx, float scale, void * stream);
/* prompt-processing attention: n_tok query rows q[t][n_head][head_dim]; token t attends to cache rows [0, pos_dev[t]] (its own
 * K/V row already stored); n_kv_max >= max(pos_dev) + 1.  Same FA-off arithmetic per row as pb200_attn_decode. */
PB200_API int pb200_attn_prefill(const float * q, const void * k_cache_f16, const void * v_cache_f16, float * out, int n_head, int n_head_kv,
                                 int head_dim, const int32_t * pos_dev, int n_tok, int n_kv_max, float scale, void * stream);

/* GGML_OP_FLASH_ATTN_EXT (ggml_cuda_flash_attn_ext, ggml-cuda/fattn.cu:298-345; CPU ggml.c:15538-15748) with f16 K / V:
 * dst[D][n_head][n_tokens] = softmax(scale * K q + slope * mask) . V per (token, head); online softmax split over the KV range and
 * merged (flash_attn_combine_results, fattn-common.cuh:519-561).  Byte strides: q_nb = {nb1 (token), nb2 (head)}, k_nb / v_nb =
 * {nb1 (cell), nb2 (kv head)}; mask f16 [n_kv] rows of mask_nb1 bytes or NULL; max_bias = ALiBi, logit_softcap = Gemma-2 style cap. */
PB200_API int pb200_flash_attn_ext(const float * q, const void * k_f16, const void * v_f16, const void * mask_f16, float * dst, int head_dim, int n_tokens,
                                   int n_head, int n_head_kv, int n_kv, const int64_t * q_nb, const int64_t * k_nb, const int64_t * v_nb, int64_t mask_nb1,
                                   float scale, float max_bias, float logit_softcap, void * stream);

/* ---- a cache of 4-bit keys and values in pages ----
 * A page holds 64 cells of every layer and kv head; sequences have lists of pages (tables), in any order, and may share them.  Page i lies at pages + i *
 * pb200_kv4_page_bytes: chunks [n_layer][n_head_kv], each 64 key rows and 64 value rows of head_dim numbers in 4 bits, with a scale (f16 of 8 significant bits) for
 * every 32 of them: 144 bytes for a cell's key and value of 128 (f16: 512).  A number is (n - 8) * scale; scale = the block's number of largest magnitude / -8
 * (of several, the first), rounded to 8 bits, n = round(x / scale) + 8 in 0 .. 15.  NaN counts as 0, magnitudes beyond 21760 as 21760: a cache holds numbers only.
 * csrc/kv4.cuh says where the bits lie.  head_dim 64 or 128 (others: PB200_ENOTSUP).  pages: device memory at a 16-byte boundary, which the caller owns.
 * Numbers in device memory (cells, tables, lengths) are checked by the kernels: what names no cell of the cache is not stored, read as a cell that nobody sees.
 * Calls are ordered by their streams alone; nothing is kept from one to the next but in the cache. */
enum { PB200_KV4_CELLS = 64 };
typedef struct pb200_kv4_cache {
    void *  pages;
    int64_t n_pages;
    int32_t n_layer, n_head_kv, head_dim, _pad;
} pb200_kv4_cache;
/* rotation as in pb200_rope, the angles in 64 bits; n_dims a multiple of 8 (others: PB200_ENOTSUP), 0: none; mode 0: neighbouring pairs, 2: halves */
typedef struct pb200_rope_args {
    int32_t n_dims, mode, n_ctx_orig;
    float   freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow;
    const float * freq_factors;   /* device [n_dims / 2], or NULL */
} pb200_rope_args;
PB200_API size_t pb200_kv4_page_bytes(int n_layer, int n_head_kv, int head_dim);   /* 0: not supported */
/* The rows of n_tokens tokens, one launch: queries and keys normed per head (x / sqrt(mean(x^2) + eps) * weight, weights f32 [head_dim] at 16 bytes, either may be NULL),
 * rotated by the token's position, queries to q_out (which may be q), keys and values into cell cells[t] = page * 64 + cell of the layer (negative: not stored; no two tokens
 * have the same).  type: PB200_TYPE_F32, F16 or BF16 of q, q_out, k and v; rows of ld* numbers (a multiple of 4), heads next to each other, at 4 numbers' boundaries.
 * n_head 0: keys and values alone.  q_out lies over q (with its stride) or over nothing that the call reads; rows may lie between each other where strides are equal, as in a joint
 * buffer (ranges of other strides have to lie apart). */
PB200_API int pb200_kv4_append(const pb200_kv4_cache * cache, int layer, int type, const void * q, int64_t ldq, void * q_out, int64_t ldq_out, const void * k, int64_t ldk,
                               const void * v, int64_t ldv, int64_t n_tokens, int n_head, const int64_t * cells, const int32_t * pos, const float * q_norm, const float * k_norm,
                               float eps, const pb200_rope_args * rope, void * stream);
/* the numbers that n cells hold, rows [n_head_kv][head_dim] of a type (F32 and F16 hold them exactly); k or v may be NULL; a cell outside of the cache leaves its rows as they were */
PB200_API int pb200_kv4_load(const pb200_kv4_cache * cache, int layer, int type, const int64_t * cells, int64_t n, void * k, int64_t ldk, void * v, int64_t ldv, void * stream);
/* Attention of a ragged batch.  The queries of sequence s are the rows q_start[s] .. q_start[s+1]-1 of q (device [n_seq + 1], rising), the last kv_len[s] cells' own: query i of n
 * stands at position p = kv_len[s] - n + i and sees the cells 0 .. p; with window > 0 those of the last `window` positions and the first keep_first.  Cell j is cell j % 64 of
 * page table[s * table_ld + j / 64].  out[t][head] = sum of softmax(scale q k) v over what it sees, zeros if that is nothing; rows outside q_start[0] .. q_start[n_seq]-1, and
 * queries beyond the first max_q of a sequence, stay as they were.  n_tokens: rows of q and out; max_q: the most queries of one sequence.  q, out: rows of [n_head][head_dim] of the
 * type as in pb200_kv4_append, whose rows may lie between each other in the same way, but have no number in common.
 * Precision.  Scores: 32 bits, up to 4e7 of them.  q: F16 and BF16 as it is, F32 22 bits of a number or 2^-39 of its row's largest.  Weights: F32 22 bits or 2^-39 of the row's largest weight, F16 and BF16 11 bits or 2^-34;
 * BF16 with few rows (up to 48 queries x heads of a group) 11 bits of a weight and of its product with its block's scale, or 2^-39 of the largest weight, 2^-36 of it in what they add to the
 * output, both times the largest value in the sequence's pages / 8 where that is more than 1.  Sums: 32 bits; prompts' are the tensor core's, which cuts off what it adds to:
 * F32 for 256 cells at a time (1e-6 of the output's norm, whatever the length), 16 bits for all (2e-4 at 131 000 cells, which is F16's own rounding).
 * PB200_ENOTSUP where pages, heads and tiles of rows do not fit 31 bits.
 * ws: pb200_kv4_attn_workspace_bytes, zeroed once by the caller, for calls that follow one another (one per stream, also of graphs that may run at the same time). */
PB200_API size_t pb200_kv4_attn_workspace_bytes(int n_head, int n_head_kv, int head_dim);
PB200_API int pb200_kv4_attn(const pb200_kv4_cache * cache, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start,
                             const int32_t * kv_len, const int32_t * table, int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, void * ws,
                             size_t ws_bytes, void * stream);
/* The same, and lse[t * ld_lse + head] = the natural logarithm of the sum of exp(scale q k) over what the query sees (f32; -inf where that is nothing). */
PB200_API int pb200_kv4_attn_lse(const pb200_kv4_cache * cache, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start,
                                 const int32_t * kv_len, const int32_t * table, int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, float * lse,
                                 int64_t ld_lse, void * ws, size_t ws_bytes, void * stream);
/* Attention of a batch whose sequences come in groups with a prefix in common, whose pages are kept once.  Group g has the sequences group_start[g] .. group_start[g+1]-1 (device
 * [n_group + 1], rising; sequences outside of group_start[0] .. group_start[n_group]-1 have no prefix), whose queries all see the prefix_len[g] cells of row g of prefix_table (as table's,
 * prefix_ld pages a row) in front of their own, which are those of pb200_kv4_attn without a window: kv_len counts them alone, and rotations count from the prefix's start.  A prefix may end
 * inside a page, and ends with its row of the table at the latest.  Sequences with few rows (up to 48 queries x heads of a group, 32 in F32) have the prefix's pages read once for all of the group,
 * by a kernel of its own, where that saves enough pages; where it does not (a few sequences, a short prefix), and for sequences with many rows, each reads them in front of its own.  Which, goes by lengths and
 * groups on the device, so that a graph follows them; max_q and n_tokens, if they are more than there is, may cost time.
 * lse: as in pb200_kv4_attn_lse, or NULL.  Precision: as in pb200_kv4_attn, of one sequence with all the cells; a prefix that is read once has a prompt's: in F16 and BF16 weights of 11 bits and
 * sums of the tensor core's (F16: 2.8e-4 of the output's norm where 32-bit operations have 2.1e-4).  A prefix and the cells behind it lie within 2^30, groups within 2^24.
 * ws: pb200_kv4_attn_shared_workspace_bytes, zeroed once, as pb200_kv4_attn's, for which it serves, too. */
PB200_API size_t pb200_kv4_attn_shared_workspace_bytes(int n_head, int n_head_kv, int head_dim, int64_t n_tokens);
PB200_API int pb200_kv4_attn_shared(const pb200_kv4_cache * cache, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start,
                                    const int32_t * kv_len, const int32_t * table, int64_t table_ld, int n_group, const int32_t * group_start, const int32_t * prefix_len,
                                    const int32_t * prefix_table, int64_t prefix_ld, int64_t n_tokens, int max_q, float scale, float * lse, int64_t ld_lse, void * ws, size_t ws_bytes,
                                    void * stream);
/* What the cells are worth: sums[s * ld_sums + j] = decay * old[s * ld_old + j] + the weights of cell j, exp(scale q k - lse), added up over the queries of sequence s that see it and all heads,
 * for j below kv_len[s] and ld_sums; other sums stay as they were.  The arguments as in pb200_kv4_attn, lse as pb200_kv4_attn_lse gives it.  q_start may name the last few queries of a prompt
 * alone: their positions are the last ones.  old: NULL counts as zeros (and is not read with a decay of 0); sums may lie over old (with its stride), otherwise apart from it.
 * Precision: scores and sums in 32 bits (q: F16 and BF16 as it is, F32 22 bits of a number).  Equal calls give equal bits. */
PB200_API int pb200_kv4_weigh(const pb200_kv4_cache * cache, int layer, int type, const void * q, int64_t ldq, int n_head, int n_seq, const int32_t * q_start, const int32_t * kv_len,
                              const int32_t * table, int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, const float * lse, int64_t ld_lse, float decay,
                              const float * old, int64_t ld_old, float * sums, int64_t ld_sums, void * stream);
/* Which cells a sequence keeps, for pb200_kv4_compact: of its len = kv_len[s] cells (max_len and ld_sums at most) count[s] = min(len, budget[s], ld_index): the last keep_last, the first keep_first
 * (as far as count[s] goes, the last ones first), and of those between the ones with the largest sums, of equal ones the lowest; a sum that is no number counts as -inf, -0 as 0.
 * index[s * ld_index + i]: the i-th, ascending; kept (or NULL)[s * ld_kept + i]: its sum, for the compacted sequence.  What lies behind count[s] stays as it was.  kept lies apart from sums. */
PB200_API int pb200_kv4_select(int n_seq, const float * sums, int64_t ld_sums, const int32_t * kv_len, int max_len, const int32_t * budget, int keep_first, int keep_last, int32_t * index,
                               int64_t ld_index, int32_t * count, float * kept, int64_t ld_kept, void * stream);
/* Copies of whole pages, all layers: page src[i] to page dst[i] (HOST arrays, not needed after the call).  A sequence that forks shares its full pages with the new one, and
 * copies the last, which both go on writing.  PB200_EINVAL where a page is written twice, or written and read. */
PB200_API int pb200_kv4_copy_pages(const pb200_kv4_cache * cache, const int32_t * src, const int32_t * dst, int n, void * stream);
/* Cells that a sequence keeps, to pages of their own, all layers: cell index[s * index_ld + i] of table row s becomes cell i of row s of `to`, i < count[s] and
 * max_count (device arrays).  Bits are moved as they are: keys stay rotated for the positions that they had.  Pages of `to` are none of the pages that are read, and of one sequence each;
 * their other cells stay as they were.  Behind it the old pages are free. */
PB200_API int pb200_kv4_compact(const pb200_kv4_cache * cache, int n_seq, const int32_t * table, int64_t table_ld, const int32_t * to, int64_t to_ld, const int32_t * index,
                                int64_t index_ld, const int32_t * count, int max_count, void * stream);

/* ---- verification of drafted tokens ----
 * Sequence s has the drafts start[s] .. start[s+1]-1 (device [n_seq + 1], rising from 0 to n_drafts): tokens and, in rows of n_vocab logits of a type (PB200_TYPE_F32, F16 or BF16; any stride), what
 * the draft model had: row i of `draft` for draft i, or draft NULL: the tokens come from elsewhere, as if with probability 1.  target: for each of its drafts and for the token behind the last one
 * a row: start[s] + s .. start[s+1] + s.  p and q: softmax of logits times inv_temp[s] (NULL: 1; infinite: all on the largest, of several the lowest; 0: even over all finite logits).
 * Draft x with its number u = u_accept[i] is accepted where u q(x) < p(x), p and q by sums in 32 bits: to 1e-6 as a rule, 1e-5 at most (vocabularies of up to 200 000); n_accepted[s]: how many are, up to the first that is not.  Behind them comes a token drawn by u_draw[s]: with weights
 * w = max(p - q, 0) of the first that is not accepted (p, where these are all 0), with p behind the last: the lowest i with w_0 + .. + w_i > u_draw[s] * (sum of w), in 64 bits.
 * out[s * ld_out + ..]: the accepted tokens and that one (as far as ld_out goes; what lies behind stays as it was).  kv_len_out[s] = kv_len[s] less the drafts that were not accepted (both NULL:
 * not wanted; may be the same): the cells of these are free.  Logits that are no number count as -inf, +inf takes all weight; tokens outside the vocabulary are not accepted; weights below 2^-960
 * of a row's largest count as 0; where a row has no weights at all, or inv_temp[s] is below 0 or no number, the token is -1.  Numbers u lie in [0, 1).
 * ws: pb200_verify_drafts_workspace_bytes, for calls that follow one another. */
PB200_API size_t pb200_verify_drafts_workspace_bytes(int64_t n_drafts);
PB200_API int pb200_verify_drafts(int type, const void * target, int64_t ld_target, const void * draft, int64_t ld_draft, int n_vocab, int n_seq, const int32_t * start, int64_t n_drafts,
                                  const int32_t * tokens, const float * inv_temp, const float * u_accept, const float * u_draw, int32_t * n_accepted, int32_t * out, int64_t ld_out,
                                  const int32_t * kv_len, int32_t * kv_len_out, void * ws, size_t ws_bytes, void * stream);

/* ---- fused decode launches (what the engine is made of), for graph-level fusion in a host such as the ggml-backend plugin ---- */
typedef struct pb200_gemv_mat {
    int32_t type;          /* k-quant type of W (Q4_K / Q5_K / Q6_K) */
    int32_t _pad;
    const void * W;        /* [n][k] raw GGUF blocks, 16-byte aligned (padding rule above) */
    int64_t n;
    float * y;             /* [n]  y = W . act (+ add[row]) */
    const float * add;     /* optional [n]: bias or residual added in the epilogue (ggml ADD node folded in) */
} pb200_gemv_mat;
/* Up to 3 matrices sharing one activation of length k (k % 256 == 0, k <= 28672), ONE launch.  prologue:
 *   0  act_ws already holds the q8_K activation (pb200_quantize_act, or pb200_attn_ggml with act_ws_out)
 *   1  act = q8_K( rms_norm(in0, eps) * in1 )     ggml RMS_NORM + MUL by the norm weight   (llm_build_norm, src/llama.cpp:9772-9802)
 *   2  act = q8_K( silu(in0) * in1 )              ggml UNARY(SILU) + MUL                    (llm_build_ffn, src/llama.cpp:9858-9907)
 * computed once, distributed over the launch's CTAs (one in-kernel grid barrier); norms of up to 3840 entries by every CTA for itself, unless
 * a y lies over in0 or in1 (which it may).  Left in act_ws either way.  sync_ws: 16 bytes of zero-initialised
 * device memory owned by the caller (barrier state, self-resetting; one per stream).  pdl != 0: the launch may start while the
 * previous kernel of the stream drains (programmatic dependent launch); its inputs are read only after that kernel has completed.
 * Returns PB200_ENOTSUP for types / shapes outside the fast kernel (callers fall back to the single ops). */
PB200_API int pb200_gemv_fused(int nmat, const pb200_gemv_mat * mats, int64_t k, void * act_ws, int prologue, const float * in0, const float * in1,
                               float eps, void * sync_ws, int pdl, void * stream);
/* One token of the reference graph's FA-off attention chain as ONE launch (llm_build_kv_store + llm_build_kqv, src/llama.cpp:9673-9718,
 * 10032-10165): rope(q), rope(k) -> f16 K row into cell kv_head of k_cache [cell][n_head_kv*128]; v -> f16 into column kv_head of the
 * TRANSPOSED v cache [n_head_kv*128][vt_stride]; out[h] = softmax(scale * K q_h + mask) . V over n_cells cells (multiple of 32, mask f32
 * [n_cells], -inf = not visible).  head_dim 128, n_head even.  act_ws_out (optional): also leaves q8_K(out) there for the following
 * mat-vec.  kv_head_dev (optional): the cell is read from this device word instead of kv_head, so a CUDA graph that captured the launch can
 * be replayed for the next token.  rope op parameters as in pb200_rope.  Returns PB200_ENOTSUP for shapes it does not handle. */
PB200_API int pb200_attn_ggml(const float * q, const float * k, const float * v, void * k_cache_f16, void * v_cache_t_f16, int64_t vt_stride, float * out,
                              void * act_ws_out, int n_head, int n_head_kv, int head_dim, const int32_t * pos_dev, int n_cells, int kv_head,
                              const int32_t * kv_head_dev, const float * mask, int n_dims, int mode, float freq_base, float freq_scale, float ext_factor, float attn_factor,
                              float beta_fast, float beta_slow, int n_ctx_orig, const float * freq_factors, float scale, int pdl, void * stream);

/* ---- decode engine (one model shard per process / GPU) ---- */
typedef struct pb200_hparams {
    int32_t n_layer, n_embd, n_head, n_head_kv, head_dim, n_ff, n_vocab, n_ctx;
    int32_t rope_mode;        /* 0 = NORM (llama), 2 = NEOX (qwen2) */
    int32_t n_ctx_orig;
    float   rope_freq_base, rope_freq_scale, rms_eps;
} pb200_hparams;

typedef struct pb200_model pb200_model;

/* layers [layer_begin, layer_end) live on this device (prima's layer window, src/llama.cpp:3838-3883);
 * with_embd / with_head: whether token_embd and output_norm+output live here (first / last pipeline stage) */
PB200_API pb200_model * pb200_model_create(const pb200_hparams * hp, int device, int layer_begin, int layer_end, int with_embd, int with_head);
PB200_API void          pb200_model_free(pb200_model * m);
/* tensor names follow GGUF: "token_embd.weight", "output_norm.weight", "output.weight", "rope_freqs.weight",
 * "blk.%d.{attn_norm,attn_q,attn_k,attn_v,attn_output,ffn_norm,ffn_gate,ffn_up,ffn_down}.weight", "blk.%d.attn_{q,k,v}.bias".
 * data: HOST pointer to raw GGUF bytes (exactly ggml_nbytes) — the same bytes llm_load_tensors hands to set_tensor. */
PB200_API int pb200_model_set_tensor(pb200_model * m, const char * name, int type, const void * host_data, size_t nbytes);
/* The same without the copy: reserves the tensor's device memory and returns its address in *dev_ptr (NULL with return 0: the tensor
 * belongs to another stage) for hosts that stream the bytes themselves (pb200_model_load_gguf does). */
PB200_API int pb200_model_tensor_alloc(pb200_model * m, const char * name, int type, size_t nbytes, void ** dev_ptr);
/* GGUF file -> finalized model shard (replaces gguf_init_from_file + llm_load_hparams + llm_load_tensors' per-tensor
 * synchronous set_tensor, ggml-cuda.cu:464-487, for this path): v2 / v3 containers, architectures "llama" and "qwen2", tensors kept in
 * their raw block layout; the file is streamed through two pinned 64-MiB buffers with cudaMemcpyAsync so reading chunk i+1 overlaps the
 * PCIe copy of chunk i.  layer_end < 0: to the last layer; with_embd / with_head < 0: derived from the window; n_ctx <= 0:
 * min(trained context, 4096).  seconds / bytes_loaded (optional) report the load.  pb200_gguf_probe only parses (no CUDA): hyper-parameters,
 * tensor count, bytes of the data section, architecture string (16 bytes). */
PB200_API int pb200_model_load_gguf(const char * path, int device, int layer_begin, int layer_end, int n_ctx, int with_embd, int with_head,
                                    pb200_model ** out, double * seconds, int64_t * bytes_loaded);
PB200_API int pb200_gguf_probe(const char * path, pb200_hparams * hp, int32_t * n_tensors, int64_t * data_bytes, char * arch_out16);
/* random-init weights generated on the device with the Q4_K_M (ftype 0) or Q5_K_M (ftype 1) type mixture of
 * llama_tensor_get_type (src/llama.cpp:19271-19556); for benchmarking without a checkpoint */
PB200_API int pb200_model_synth(pb200_model * m, int ftype, uint64_t seed);
PB200_API int pb200_model_finalize(pb200_model * m);     /* allocate KV cache + activations, capture the CUDA graph */
/* device address, size and ggml type of a tensor this shard holds (GGUF names as in pb200_model_set_tensor): lets a host copy
 * weights device-to-device, e.g. bench.py moving the synthetic model into the ggml-backend buffers of the plugin */
PB200_API int pb200_model_tensor_device(pb200_model * m, const char * name, const void ** dev_ptr, size_t * nbytes, int * type);
PB200_API int64_t pb200_model_weight_bytes(const pb200_model * m);    /* algorithmic bytes read per decoded token on this shard */
/* Prompt processing (prefill): n_tokens tokens at positions pos0 .. pos0+n_tokens-1 through all layers as one batch — the
 * reference's llama_decode with a multi-token ubatch (ne11 > 1: ggml_cuda_op_mul_mat_q, mmq.cu:3-98; attention
 * ggml-cuda.cu:1737-1881).  Mat-muls on the tensor cores (pb200_mul_mat_q), attention over the K/V rows just stored.  The KV
 * cache is left exactly as n_tokens pb200_decode calls would leave it up to fp16-rounding differences in the mat-muls;
 * logits of the LAST token go to logits_host (may be NULL).  Models created with with_embd and first_layer == 0 only. */
PB200_API int pb200_prefill(pb200_model * m, const int32_t * tokens_host, int32_t n_tokens, int32_t pos0, float * logits_host);
/* Prompt processing on a pipeline shard (prima's layer windows, src/llama.cpp:3838-3883, 17825-18029): ONE ubatch of n_tokens <= 512 through
 * the layers of this model object.  The stage that holds the embedding takes tokens_host (hidden_in_dev ignored); every other stage takes
 * the previous stage's hidden states hidden_in_dev [n_tokens][n_embd] f32 in device memory (not modified).  The stage's output hidden
 * states stay on the device at pb200_prefill_hidden_device(m) until the next prefill call (the caller ships them to the next stage, e.g.
 * with ncclSend on the model stream); the stage with the head also computes the last token's logits.  synchronize = 0: everything is
 * only enqueued on the model stream (micro-batched pipelines keep several ubatches in flight across the stages); logits_host requires
 * synchronize != 0.  K/V rows pos0 .. pos0+n_tokens-1 of this shard's layers are written like pb200_prefill writes them. */
PB200_API int pb200_prefill_stage(pb200_model * m, const int32_t * tokens_host, const float * hidden_in_dev, int32_t n_tokens, int32_t pos0,
                                  float * logits_host, int32_t synchronize);
PB200_API float * pb200_prefill_hidden_device(pb200_model * m);
PB200_API int pb200_kv_clear(pb200_model * m);

/* one decode step, HOST in/out (the llama_decode-equivalent call): token id + position in, n_vocab logits out.
 * On a pipeline stage without the embedding / head the hidden state is exchanged through pb200_hidden_* instead. */
PB200_API int pb200_decode(pb200_model * m, int32_t token, int32_t pos, float * logits_host);
/* device-resident variant: enqueue one step on the model stream, no host copies, no synchronisation */
PB200_API int pb200_decode_async(pb200_model * m, int32_t token, int32_t pos);
PB200_API int pb200_synchronize(pb200_model * m);
/* Several independent sequences per shard (each with its own KV cache, token and position slot): what keeps every stage of the layer
 * pipeline busy — prima's piped ring with one token per stage in flight (src/llama.cpp:17825-18029, 18299-18387).  Set before finalize. */
PB200_API int pb200_model_set_n_seq(pb200_model * m, int n_seq);
PB200_API int pb200_decode_seq_async(pb200_model * m, int seq, int32_t token, int32_t pos);   /* pb200_decode_async on slot seq */
/* one step of slot seq with token id and position taken from device memory (written by a hand-off, pb200_set_tokpos_seq or
 * pb200_argmax_seq); nothing crosses the host.  advance_pos != 0: the slot's position is incremented afterwards. */
PB200_API int pb200_step_seq_dev(pb200_model * m, int seq, int advance_pos);
PB200_API int pb200_set_tokpos_seq(pb200_model * m, int seq, int32_t token, int32_t pos);
/* greedy sampling on the device (ggml-cuda/argmax.cu:7): argmax of the slot's logits -> pb200_sample_device(m, seq); feed_back != 0 on a
 * shard that also holds the embedding writes it into the slot's token as well (single-GPU generation without a host round trip) */
PB200_API int pb200_argmax_seq(pb200_model * m, int seq, int feed_back);
PB200_API int32_t * pb200_token_device(pb200_model * m, int seq);    /* int32[2]: {token, position} of the slot */
PB200_API int32_t * pb200_sample_device(pb200_model * m, int seq);   /* int32: greedy token of the slot's last step */
PB200_API float * pb200_logits_device(pb200_model * m);      /* [n_vocab] f32 */
PB200_API float * pb200_hidden_in_device(pb200_model * m);   /* [n_embd] f32: input of layer_begin (written by the previous stage) */
PB200_API float * pb200_hidden_out_device(pb200_model * m);  /* [n_embd] f32: output of layer_end-1 */
PB200_API void *  pb200_stream(pb200_model * m);
PB200_API int pb200_get_hidden(pb200_model * m, float * hidden_host);   /* copies hidden_out to the host (tests) */
/* one step with CUDA events around every GEMV launch (direct launches): summed GEMV device time, the algorithmic
 * weight bytes those launches read, their count and the whole-step time — the live roofline measurement of bench.py */
PB200_API int pb200_profile_step(pb200_model * m, int32_t token, int32_t pos, double * gemv_ms, int64_t * gemv_bytes, int32_t * gemv_launches, double * step_ms);
PB200_API int pb200_set_hidden(pb200_model * m, const float * hidden_host);   /* host -> hidden_in (tests, host-staged hand-off) */
PB200_API int pb200_debug_read(pb200_model * m, const char * name, float * host, int64_t n);   /* white-box tests: q,k,v,att,g,u,x_a,x_b,xn,logits; prompt_q,_k,_v,_g,_u of the last prompt's last layer */
PB200_API int pb200_set_use_graph(pb200_model * m, int on);             /* CUDA-graph replay on/off (default on) */

/* dense product, device buffers: C[t][n] = alpha * sum_k A[t][k] W[n][k] (+ bias[n]) (+ resid[t][n]); A [T][K] and W [N][K] row-major of `type`
 * (PB200_TYPE_F32: true fp32; PB200_TYPE_BF16: bf16 operands, fp32 accumulation: tcgen05 tensor cores for more than 4 tokens when K and
 * the strides are multiples of 8, a weight-streaming kernel for fewer); C, bias, resid f32; resid may alias C; strides in elements */
PB200_API int pb200_dense(int type, const void * A, int64_t lda, const void * W, int64_t ldw, float * C, int64_t ldc, int T, int N, int K,
                          const float * bias, const float * resid, int64_t ldr, float alpha, void * stream);

/* ---- architectures ----
 * Two families share the model object: 0 = one fixed transformer graph over k-quant GGUF weights ("llama", "qwen2":
 * pb200_model_create / pb200_model_load_gguf), 1 = layer list: a configuration file lists the layers, each with a sequence mixer
 * (windowed attention with kept first tokens, a Mamba-2 state-space mixer, linear attention with a fixed decay per head, softmax attention
 * over a low-rank latent, a WKV mixer, or an attention branch beside a gated linear recurrence) and an optional feed-forward (gated,
 * squared-ReLU or xIELU, dense or a routed mixture of experts), over dense f32 / bf16
 * weights ("Vamidra", "Mumizen", "Sapudra", "Zevedra", "Ruvuvik": pb200_model_create_from_config / pb200_model_load_dir).  pb200_arch_family: -1 for an unknown name. */
PB200_API int          pb200_arch_count(void);
PB200_API const char * pb200_arch_name(int i);
PB200_API int          pb200_arch_family(const char * name);

/* ---- layer-list family ----
 * config_json: the text of the model's configuration file; its "architecture" selects the design.  compute_type: PB200_TYPE_BF16 (dense
 * products on bf16 operands with fp32 accumulation; norms, the residual stream and all recurrent state stay fp32; attention takes fp32
 * queries, keys, values and softmax weights and accumulates in fp32, in prompts beyond 16 tokens with every operand as two f16 numbers,
 * 22 bits and more) or PB200_TYPE_F32 (everything in true fp32).  A row of a batch does not depend on what the others hold; how many they
 * are may change the order of its fp32 sums.  n_ctx: the most positions one sequence can have where a layer has to keep all of
 * them; a windowed attention layer keeps keep_first + window rows per sequence whatever its length.  n_seq: sequence slots
 * (<= 0: as many as 8 GiB of state hold, 4 .. 256).  Tensors arrive through pb200_model_set_tensor under their checkpoint names with
 * type PB200_TYPE_BF16 or PB200_TYPE_F32 (converted to what the model computes in); then pb200_model_finalize.  pb200_model_synth
 * fills every tensor with random values instead (benchmarks). */
PB200_API pb200_model * pb200_model_create_from_config(const char * config_json, int compute_type, int device, int n_ctx, int n_seq);
/* <dir>/config.json + <dir>/model.safetensors -> finalized model */
PB200_API int pb200_model_load_dir(const char * dir, int compute_type, int device, int n_ctx, int n_seq, pb200_model ** out);
PB200_API int pb200_model_get_hparams(const pb200_model * m, pb200_hparams * out);   /* n_layer, n_embd, n_vocab, n_ctx are set for every family */
PB200_API int pb200_model_n_seq(const pb200_model * m);

/* Sequence slots.  A slot holds everything a sequence carries from token to token (attention rows, convolution inputs, recurrent
 * state); pb200_seq_alloc hands out a free slot in the empty state (>= 0, or PB200_ENOMEM), pb200_seq_free gives it back. */
PB200_API int pb200_seq_alloc(pb200_model * m);
PB200_API int pb200_seq_free(pb200_model * m, int slot);
PB200_API int pb200_seq_length(pb200_model * m, int slot);   /* tokens the slot has seen; < 0: free slot */

/* One step of a ragged batch: entry e appends n_tokens tokens to sequence slot seq (continuing at the slot's length) and asks for the
 * logits at the token indices want[0..n_want) of its tokens.  logits_host receives the wanted rows, [sum n_want][n_vocab] f32, in the
 * order of the entries and of want; greedy_host (optional) receives per entry the arg-max token of the logits after its last token.
 * Entries that start a sequence run together as one prompt batch; entries that continue one advance token by token, all of them
 * batched per token.  The logits of a position do not depend on what else is in the batch beyond fp32 rounding. */
typedef struct pb200_batch_entry {
    int32_t seq;
    int32_t n_tokens;
    const int32_t * tokens;
    int32_t n_want;
    const int32_t * want;
} pb200_batch_entry;
/* Page-locked host memory for logits_host, out of a pool of bounded size that a layer-list model takes from the system as blocks are asked for and holds until its end:
 * the rows arrive in it without a copy through a staging buffer (as in any page-locked memory of the caller's).  NULL: the pool has no room, or there is no memory that can
 * be page-locked; use any other memory.  A block stays valid until it is given back, also beyond the model's end.  Both calls may come from any thread. */
PB200_API void * pb200_result_take(pb200_model * m, size_t bytes);
PB200_API int    pb200_result_give(void * block);
PB200_API int pb200_batch_step(pb200_model * m, int n_entries, const pb200_batch_entry * entries, float * logits_host, int32_t * greedy_host);
/* white-box tests: on != 0 keeps the residual stream after every layer run of the next batches; read it with
 * pb200_debug_read(m, "layers", host, runs * tokens * n_embd) */
PB200_API int pb200_debug_tap_layers(pb200_model * m, int on);
/* measurement: on != 0 records CUDA events around every launch of the next batches; pb200_debug_read(m, "profile", host, 10) returns the
 * device milliseconds of the last batch per category: dense products, attention, convolution, scan, norms, element-wise, output head,
 * [7] total, [8] routed experts, [9] the small steps around latent attention.  Events serialise nothing but forbid overlap between launches; leave it off when timing whole steps. */
PB200_API int pb200_debug_profile(pb200_model * m, int on);

#ifdef __cplusplus
}
#endif
#endif /* PRIMA_B200_H */
