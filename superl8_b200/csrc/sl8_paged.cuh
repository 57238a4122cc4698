// What the attention kernels over the paged cache share: their arguments and what a sequence asks for.
#pragma once
#include "sl8_common.cuh"

namespace sl8 {

// A V scale below the smallest normal number marks a page that holds nothing (pages are written with 2^-40 at least).
constexpr float kLeastScale = 1.17549435e-38f;

struct PagedArgs {
  const void* q;
  int64_t q_sb, q_sh, q_ss;
  void* out;
  int64_t o_sb, o_sh, o_ss;
  const int8_t *k, *v;
  const float *ks, *vs;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* query_lens;
  float* part_o;      // [2 * blocks][rows_per_unit][D]
  float* part_ml;     // [2 * blocks][rows_per_unit][2]
  int B, Hq, Hkv, M, G, rows;              // rows = M * G query rows per (sequence, KV head)
  int page_shift, num_pages, max_tokens;   // max_tokens: what the table can name and the caller lets be seen
  int causal, window, bf16;
  int row_warps;      // warps that share a key but hold other rows (1 or 2)
  int rows_per_unit, row_units;            // rows = up to row_units * rows_per_unit
  int blocks;         // blocks that share the line of all units (or a unit, in a cluster)
  int chunk_shift;    // log2 of the keys of a chunk
  float scale_log2;   // softmax_scale * log2 e
};

// A sequence: tokens that can be seen, its query tokens, and the place of query token 0.
struct Seq {
  int len, n, place;
  int first_chunk, chunks;   // chunks of 2^chunk_shift keys that some query can see
};

__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int b) {
  Seq s;
  const int context = max(__ldg(a.lens + b), 0);
  s.n = a.query_lens ? min(max(__ldg(a.query_lens + b), 0), a.M) : a.M;
  s.len = min(context, a.max_tokens);
  s.place = context - s.n;
  int64_t lo = 0;
  if (a.window >= 0) lo = max((int64_t)0, (int64_t)s.place - a.window + 1);
  s.first_chunk = (int)(lo >> a.chunk_shift);
  s.chunks = (s.n > 0 && lo < s.len) ? (int)(((int64_t)s.len + (1 << a.chunk_shift) - 1) >> a.chunk_shift) - s.first_chunk : 0;
  return s;
}

}  // namespace sl8

// Many query rows per KV head (paged_prefill.cu): workspace it needs (0: it does not serve the call), and the
// launch.  `workspace` is 1024-byte aligned.
size_t sl8_paged_prefill_workspace(const sl8::PagedArgs& a, int D);
double sl8_paged_prefill_us(const sl8::PagedArgs& a, int D);
int sl8_paged_prefill(const sl8::PagedArgs& a, int D, void* workspace, size_t workspace_bytes, cudaStream_t stream);
int sl8_paged_prefill_status(void* stream);
