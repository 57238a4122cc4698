/*
 * superl8_b200 -- C ABI of the rotary positions and of the paged int8 K/V cache: rotate, append,
 * attend, read back.  Included by superl8_b200.h, whose conventions hold here too: device pointers,
 * sizes and a CUDA stream; nothing allocates; launches are asynchronous; SL8_OK or SL8_ERR_*.
 */
#ifndef SUPERL8_B200_PAGED_H_
#define SUPERL8_B200_PAGED_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions ---------------------------------------------------- */

/*
 * Rotary positions on q [B, Hq, S, D] and k [B, Hkv, S, D] (either may be NULL), one launch for both:
 * channel pair i < rot / 2 of a row turns by  t = pos[axis(i)] * inv_freq[i],
 *   y_a = a cos t - b sin t,  y_b = b cos t + a sin t,
 * (a, b) = channels (i, i + rot / 2), or (2 i, 2 i + 1) with interleaved != 0; channels from rot on are
 * copied.  positions: int32 or int64 (pos_is_64), element strides per axis, sequence and token (0 where
 * shared); freq_axis: uint8 [rot / 2], the axis of every frequency (time / height / width; NULL = axis 0;
 * values past n_axes - 1 read the last axis).  The angle is formed in 64 bits and reduced before sin / cos,
 * so positions up to 2^31 lose nothing; inv_freq must be
 * finite (a frequency of NaN or infinity does not turn).  inverse != 0 turns by -t: the gradient, and the inverse.
 * dtype fp16 / bf16 / fp32 (arithmetic in fp32, one rounding); D and rot even, rot <= D; strides are in
 * elements, the channel dimension is contiguous; x and y may be the same tensor.  No counterpart on the
 * reference's attention path (its `rope` is a separate glue kernel).
 */
typedef struct sl8_rope_params {
  const void* q; void* q_out; const void* k; void* k_out;
  int64_t q_stride_b, q_stride_h, q_stride_s, q_out_stride_b, q_out_stride_h, q_out_stride_s;
  int64_t k_stride_b, k_stride_h, k_stride_s, k_out_stride_b, k_out_stride_h, k_out_stride_s;
  const void* positions;
  int64_t pos_stride_axis, pos_stride_b, pos_stride_s;
  const float* inv_freq;
  const uint8_t* freq_axis;
  int32_t B, Hq, Hkv, S, D, rot;
  int32_t dtype; int32_t pos_is_64; int32_t n_axes; int32_t interleaved; int32_t inverse;
} sl8_rope_params;
int sl8_rope(const sl8_rope_params* p, void* stream);

/* ---- paged int8 K/V cache ------------------------------------------------ */

/*
 * A cache of pages: page_size (16, 32, 64, 128 or 256) tokens of every KV head.  A page of one head has ONE
 * scale for K and one for V; the values it stands for are code * scale.  A page whose V scale is 0
 * holds nothing (a zeroed pool is empty).  block_table[b * table_stride + j] is the page of tokens
 * [j * page_size, (j + 1) * page_size) of sequence b; entries outside [0, num_pages) are pages that the
 * cache does not have: their tokens are neither stored nor seen.  context_lens[b]: tokens of sequence b in
 * the cache, those of the current step included; tokens past max_pages * page_size do not exist.
 * D in {32, 64, 128, 256}.  Replaces the reference's per-token-scale paged cache
 * (superl8/ops.py:730-918) with block scales that can be kept while tokens arrive one at a time.
 */
typedef struct sl8_paged_cache {
  int8_t* k; int8_t* v;              /* [num_pages, Hkv, page_size, D] */
  float* k_scale; float* v_scale;    /* [num_pages, Hkv] */
  const int32_t* block_table;        /* [B, max_pages] */
  int64_t table_stride;
  const int32_t* context_lens;       /* [B] */
  int32_t num_pages, Hkv, page_size, D, max_pages;
} sl8_paged_cache;

/*
 * Stores the last new_lens[b] tokens of every sequence (M for all where new_lens is NULL): row i of k_new /
 * v_new [B, Hkv, M, D] is the token at place context_lens[b] - new_lens[b] + i (a negative place is not
 * stored).  K is rotated on the way (rot > 0; as sl8_rope, positions [axes, B, M], NULL = the token's
 * place), and so is q [B, Hq, M, D] into q_out (nullable; rows past new_lens[b] become zeros).
 * Per touched page and head:  scale' = max(scale, max|x_new| * (1 / 127), 2^-40), with scale = 0 where the
 * page holds no older token;  code = rint(x / scale');  older codes become rint(code * scale / scale') when
 * the scale grew (each growth moves an older value by at most half a step).  Codes behind the sequence's
 * end are left as they were.  A NaN or infinity makes its page's scale NaN or infinite: what attends to it
 * is NaN.  A page that is written to may be named once only, by one sequence.  fp16 / bf16, rot % 16 == 0, rows
 * 16-byte aligned.
 */
typedef struct sl8_append_params {
  const void* k_new; const void* v_new;
  const void* q; void* q_out;
  int64_t k_stride_b, k_stride_h, k_stride_s, v_stride_b, v_stride_h, v_stride_s;
  int64_t q_stride_b, q_stride_h, q_stride_s, q_out_stride_b, q_out_stride_h, q_out_stride_s;
  const int32_t* new_lens;
  const void* positions;
  int64_t pos_stride_axis, pos_stride_b, pos_stride_s;
  const float* inv_freq;
  const uint8_t* freq_axis;
  int32_t B, Hq, M, rot;
  int32_t dtype; int32_t pos_is_64; int32_t n_axes; int32_t interleaved;
} sl8_append_params;
int sl8_kv_append_paged(const sl8_paged_cache* cache, const sl8_append_params* p, void* stream);

/*
 * The cache's values as 16-bit tensors: k_out / v_out [B, Hkv, count, D] (dtype fp16 / bf16), row j =
 * token first[b] + j (first NULL: 0); zeros where the sequence has no such token.
 */
int sl8_kv_read_paged(const sl8_paged_cache* cache, int32_t B, const int32_t* first, int32_t count, int dtype,
                      void* k_out, void* v_out, void* stream);

/*
 * Attention over the paged cache: out = softmax(scale * q . K^T) V with K = code * scale, V = code * scale.
 * q, out [B, Hq, M, D] fp16 or bf16 (element strides, channels contiguous, rows 16-byte aligned).  Row i of
 * sequence b is the token at place context_lens[b] - query_lens[b] + i (query_lens NULL: M); rows past
 * query_lens[b] give zeros, so does a row that sees no key.  causal != 0: it sees the keys up to its own
 * place, else all of the context; window_left >= 0: only keys in (place - window_left, ...].
 * max_context_len (host): an upper bound of context_lens that sizes the launch and the workspace (keys at or
 * past it are not seen); <= 0 = max_pages * page_size.
 * Two kernels: a split one that streams the pages once per 64 query rows of a KV head (32 at D = 256; rows =
 * M * Hq / Hkv: decode, drafted tokens), and a tensor-memory one over a dense copy of the codes in the workspace
 * (D 64 / 128 / 256, scale >= 0, else SL8_ERR_UNSUPPORTED when asked for).  SL8_BACKEND_AUTO takes the split one
 * up to 64 rows, and above whichever it estimates to be faster.
 * workspace: sl8_attn_paged_workspace() bytes, 16-byte aligned, any contents; it serves one call at a time.
 */
typedef struct sl8_paged_attn_params {
  const void* q; void* out;
  int64_t q_stride_b, q_stride_h, q_stride_s, out_stride_b, out_stride_h, out_stride_s;
  const int32_t* query_lens;
  int32_t B, Hq, M;
  int32_t dtype; int32_t causal; int32_t window_left; int32_t max_context_len;
  float softmax_scale;
  int32_t backend;        /* SL8_BACKEND_AUTO, SL8_BACKEND_MMA (split), SL8_BACKEND_TCGEN05 (tensor memory) */
} sl8_paged_attn_params;
size_t sl8_attn_paged_workspace(const sl8_paged_cache* cache, const sl8_paged_attn_params* p);
int sl8_attn_paged(const sl8_paged_cache* cache, const sl8_paged_attn_params* p, void* workspace,
                   size_t workspace_bytes, void* stream);

/* Synchronises the stream and returns the status of these kernels' bounded waits on the current
 * device since the last call (SL8_OK or SL8_ERR_DEVICE_TIMEOUT), and clears it. */
int sl8_paged_status(void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SUPERL8_B200_PAGED_H_ */
