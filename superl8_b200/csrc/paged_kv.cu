// The paged int8 K/V cache: appending new tokens (with the position rotation of K and Q on the way) and
// reading sequences back as 16-bit values.
//
// Cache: codes int8 [pages, Hkv, page_size, D], scales fp32 [pages, Hkv], one for K and one for V of every
// page and KV head; a value is code * scale.  block_table [B, max_pages] names the page of every page_size
// tokens of a sequence.
//
// Append: block (page of a sequence, head, K or V).  All new tokens of a page meet in one block, so its
// scale needs no atomics and nothing depends on an order:
//   scale' = max(scale, max|new| / 127, 2^-40)   (scale = 0 where the page holds no older token),
//   code   = rint(x / scale'),   older codes -> rint(code * scale / scale')  when scale' > scale.
// An append that does not raise the scale leaves the older codes alone; one that does adds at most half a
// step of the new scale to them.  The largest |x| is compared as bits, so NaN and infinity reach the scale
// (as NaN, and from there every value of the page) instead of vanishing in a maximum.  Bound by HBM for prompts
// (2 D bytes read, D written per token, head and tensor), by launch and three dependent loads
// (length -> page -> scale) for single tokens.
//
// Measured (8 KV heads of 128, 32 heads of Q rotated as well): a prompt of 4096 tokens in bf16 26.5 us (9 us
// without Q; the rotation's instructions and the loads' latency bound it, HBM would take 10), one token of
// each of 128 sequences 5.1 us.  Reading the prompt back as 16-bit values takes 7.7 us.
#include "sl8_rope.cuh"

namespace sl8 {
namespace {

constexpr float kScaleFloor = 9.094947017729282e-13f;   // 2^-40: no page of a stored token has scale 0
constexpr float kMagic = 12582912.f;                    // 1.5 * 2^23: adding it rounds to an integer (low byte = code)

struct PoolArgs {
  const void* x;              // new K or V
  int64_t x_sb, x_sh, x_ss;
  int8_t* codes;
  float* scale;
};

struct AppendArgs {
  PoolArgs k, v;
  const void* q;              // nullable
  void* q_out;
  int64_t q_sb, q_sh, q_ss, qo_sb, qo_sh, qo_ss;
  RopeFreq f;                 // half = 0: no rotation; positions null: the token's place in the sequence
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;        // tokens in the cache with the new ones
  const int32_t* new_lens;    // nullable: M
  int B, Hq, Hkv, M, D, page_shift, max_pages, num_pages, interleaved;
  int page_slots;             // pages one sequence's new tokens can touch
  uint32_t kv_units;          // (sequence, page, head): blocks that store K, and as many that store V
  int q_heads_per_block, q_head_groups;
};

__device__ __forceinline__ int new_count(const AppendArgs& a, int b) {
  return a.new_lens ? min(max(__ldg(a.new_lens + b), 0), a.M) : a.M;
}

// Angles of 8 frequencies for new token i of sequence b whose place in the sequence is `place`.
__device__ __forceinline__ void append_angles(const AppendArgs& a, const unsigned long long* table, int i0, int b, int i, int place,
                                              float (&c)[8], float (&s)[8]) {
  if (a.f.positions) {
    rope_angles<8>(a.f, table, i0, b, i, c, s);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float2 cc, ss;
      rope_angle2(place, table[i0 + e], place, table[i0 + e + 1], cc, ss);
      c[e] = cc.x; c[e + 1] = cc.y;
      s[e] = ss.x; s[e + 1] = ss.y;
    }
  }
}

__device__ __forceinline__ uint32_t pack_codes(const float* x, float inv) {
  const float2 inv2 = make_float2(inv, inv), magic2 = make_float2(kMagic, kMagic);
  const float2 a = __ffma2_rn(make_float2(x[0], x[1]), inv2, magic2), b = __ffma2_rn(make_float2(x[2], x[3]), inv2, magic2);
  return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                     __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

__device__ __forceinline__ void store_codes(int8_t* row, int2 at, const float (&u)[8], const float (&w)[8], float inv) {
  *reinterpret_cast<uint2*>(row + at.x) = make_uint2(pack_codes(u, inv), pack_codes(u + 4, inv));
  *reinterpret_cast<uint2*>(row + at.y) = make_uint2(pack_codes(w, inv), pack_codes(w + 4, inv));
}

// Largest magnitude of 16 values; a NaN stays (max.NaN), unlike in fmaxf.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t abs_bits(const float (&u)[8], const float (&w)[8]) {
  float m = max3_abs(u[0], u[1], w[0]), k = max3_abs(w[1], u[2], w[2]);
#pragma unroll
  for (int e = 3; e < 7; e += 2) {
    m = max3_abs(m, u[e], u[e + 1]);
    k = max3_abs(k, w[e], w[e + 1]);
  }
  return __float_as_uint(max3_abs(max3_abs(m, u[7], w[7]), k, k)) & 0x7fffffffu;
}

// Older codes of a page meet its larger scale.
__device__ __forceinline__ void requantise(int8_t* codes, int bytes, float ratio, int tid, int threads) {
  for (int i = tid; i < bytes / 16; i += threads) {
    uint4 p = reinterpret_cast<uint4*>(codes)[i];
    uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)(w[n] >> (8 * e));
      w[n] = pack_codes(x, ratio);
    }
    reinterpret_cast<uint4*>(codes)[i] = p;
  }
}

// The role of a block that stores K or V: one page of one sequence and one head of one of the two.
// NIT > 0: items (16 channels of a token) per thread, held in registers between the maximum and the
// codes; NIT = 0: any number, read twice (the second time from L1 / L2).
template <typename T, int NIT, bool IS_K>
__device__ void append_page(const AppendArgs& a, uint32_t unit, uint32_t* red, const unsigned long long* table) {
  const uint32_t rest = unit / (uint32_t)a.Hkv;
  const int h = (int)(unit - rest * a.Hkv);
  const int b = (int)(rest / (uint32_t)a.page_slots), slot = (int)(rest - (uint32_t)b * a.page_slots);
  const int len = __ldg(a.lens + b), n = new_count(a, b);
  const int page_size = 1 << a.page_shift;
  const int64_t start = (int64_t)len - n;                          // place of new token 0 (negative: not stored)
  const int first_page = (int)(max(start, (int64_t)0) >> a.page_shift);
  const int page_no = first_page + slot;
  const int64_t lo = (int64_t)page_no << a.page_shift;             // first token of the page
  const int t0 = (int)max((int64_t)0, start - lo);                 // new tokens fill [t0, t1) of the page
  const int t1 = (int)min((int64_t)page_size, (int64_t)len - lo);
  if (n == 0 || t1 <= t0 || page_no >= a.max_pages) return;
  const int page = __ldg(a.table + b * a.table_stride + page_no);
  if (page < 0 || page >= a.num_pages) return;                     // a page the cache does not have: nothing is stored

  const PoolArgs& pool = IS_K ? a.k : a.v;
  const int per_row = a.D / 16, row_shift = __ffs(per_row) - 1;    // D is a power of two
  const int items = (t1 - t0) * per_row;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int i_first = (int)(lo + t0 - start);                      // new-token index of place t0
  const bool interleaved = a.interleaved != 0;
  const int64_t ph = (int64_t)page * a.Hkv + h;
  int8_t* const codes = pool.codes + ph * page_size * a.D;
  const T* x = reinterpret_cast<const T*>(pool.x) + b * pool.x_sb + h * pool.x_sh + i_first * pool.x_ss;
  const float old = t0 > 0 ? pool.scale[ph] : 0.f;

  // an item's 16 values, rotated
  auto fetch = [&](int item, float (&u)[8], float (&w)[8]) {
    const int row = item >> row_shift, j = item & (per_row - 1);
    const bool turn = IS_K && j * 8 < a.f.half;
    const int2 at = IS_K ? rope_item<8>(j, a.f.half, interleaved) : make_int2(16 * j, 16 * j + 8);
    const Piece<T, 8> p0 = piece_load<T, 8>(x + row * pool.x_ss + at.x), p1 = piece_load<T, 8>(x + row * pool.x_ss + at.y);
    float c[8], s[8];
    if (turn) append_angles(a, table, j * 8, b, i_first + row, (int)lo + t0 + row, c, s);
    p0.get(u);
    p1.get(w);
    if (turn) rope_turn<8>(u, w, c, s, interleaved);
  };
  auto put = [&](int item, const float (&u)[8], const float (&w)[8], float inv) {
    const int row = item >> row_shift, j = item & (per_row - 1);
    const int2 at = IS_K ? rope_item<8>(j, a.f.half, interleaved) : make_int2(16 * j, 16 * j + 8);
    store_codes(codes + (int64_t)(t0 + row) * a.D, at, u, w, inv);
  };
  constexpr int KEEP = NIT > 0 ? NIT : 1;
  float u[KEEP][8], w[KEEP][8];
  uint32_t top = 0;
  if (NIT > 0) {
#pragma unroll
    for (int it = 0; it < KEEP; ++it)
      if (tid + it * threads < items) {
        fetch(tid + it * threads, u[it], w[it]);
        top = max(top, abs_bits(u[it], w[it]));
      }
  } else {
    for (int item = tid; item < items; item += threads) {
      fetch(item, u[0], w[0]);
      top = max(top, abs_bits(u[0], w[0]));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (threads > 32) {
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int i = 0; i < threads / 32; ++i) top = max(top, red[i]);
  } else {
    __syncwarp();
  }
  // as bits again: a NaN scale stays, and an infinite one becomes NaN, so that no product of its codes can hide
  // the page behind a weight of exp(-inf)
  uint32_t bits = max(__float_as_uint(old) & 0x7fffffffu, __float_as_uint(__fdiv_rn(__uint_as_float(top), 127.f)));
  if (bits >= 0x7f800000u) bits = 0x7fffffffu;
  const float now = __uint_as_float(max(bits, __float_as_uint(kScaleFloor)));
  const float inv = 1.f / now;
  if (NIT > 0) {
#pragma unroll
    for (int it = 0; it < KEEP; ++it)
      if (tid + it * threads < items) put(tid + it * threads, u[it], w[it], inv);
  } else {
    for (int item = tid; item < items; item += threads) {
      fetch(item, u[0], w[0]);
      put(item, u[0], w[0], inv);
    }
  }
  if (t0 > 0 && now != old) requantise(codes, t0 * a.D, __fdiv_rn(old, now), tid, threads);
  // the other threads of a wide block have read the old scale: they passed the barrier above
  if (tid == 0) pool.scale[ph] = now;
}

// The role of a block that rotates Q: as rope.cu, rows past new_lens are written as zeros.
template <typename T>
__device__ void append_query(const AppendArgs& a, uint32_t block, const unsigned long long* table) {
  const uint32_t rest = block / (uint32_t)a.q_head_groups;
  const int group = (int)(block - rest * a.q_head_groups);
  const int per_row = a.D / 16, row_shift = __ffs(per_row) - 1;
  const uint32_t item = rest * blockDim.x + threadIdx.x, token = item >> row_shift;   // the host keeps them below 2^32
  if (token >= (uint32_t)a.B * (uint32_t)a.M) return;
  const int j = (int)(item & (per_row - 1));
  const int b = (int)(token / (uint32_t)a.M), i = (int)(token - (uint32_t)b * a.M);
  const int n = new_count(a, b);
  const bool real = i < n, turn = real && j * 8 < a.f.half;
  const int2 at = rope_item<8>(j, a.f.half, a.interleaved != 0);
  const int h0 = group * a.q_heads_per_block, h1 = min(a.Hq, h0 + a.q_heads_per_block);
  const T* x = reinterpret_cast<const T*>(a.q) + b * a.q_sb + i * a.q_ss + h0 * a.q_sh;
  T* y = reinterpret_cast<T*>(a.q_out) + b * a.qo_sb + i * a.qo_ss + h0 * a.qo_sh;
  float c[8], s[8];
  if (turn) append_angles(a, table, j * 8, b, i, __ldg(a.lens + b) - n + i, c, s);
#pragma unroll 2
  for (int h = h0; h < h1; ++h) {
    Piece<T, 8> p0, p1;
    p0.zero();
    p1.zero();
    if (real) {
      p0 = piece_load<T, 8>(x + at.x);
      p1 = piece_load<T, 8>(x + at.y);
    }
    if (turn) {
      float u[8], w[8];
      p0.get(u);
      p1.get(w);
      rope_turn<8>(u, w, c, s, a.interleaved != 0);
      p0.put(u);
      p1.put(w);
    }
    p0.store(y + at.x);
    p1.store(y + at.y);
    x += a.q_sh;
    y += a.qo_sh;
  }
}

template <typename T, int NIT>
__global__ void __launch_bounds__(256, 4) append_kernel(const AppendArgs a) {
  __shared__ uint32_t red[8];
  __shared__ unsigned long long table[128];   // D <= 256
  const uint32_t block = blockIdx.x;
  const bool v_role = block >= a.kv_units && block < 2 * a.kv_units;
  if (a.f.half > 0 && !v_role) {
    rope_table(table, a.f);
    if (blockDim.x > 32) __syncthreads(); else __syncwarp();
  }
  if (block < a.kv_units) append_page<T, NIT, true>(a, block, red, table);
  else if (v_role) append_page<T, NIT, false>(a, block - a.kv_units, red, table);
  else append_query<T>(a, block - 2 * a.kv_units, table);
}

template <typename T>
int launch_append(AppendArgs a, cudaStream_t stream) {
  const int page_size = 1 << a.page_shift;
  const int rows = a.M < page_size ? a.M : page_size;
  const int items = rows * (a.D / 16);
  // One warp serves a single token; a full page of 64 x 128 takes 256 threads with two items each.  Above
  // 512 items (pages of 128 x 128 and larger) the rows are read twice instead of held.
  int threads = 32;
  while (threads < 256 && threads < items) threads *= 2;
  const int nit = (items + threads - 1) / threads;
  a.page_slots = (a.M + page_size - 2) / page_size + 1;
  if (a.page_slots > a.max_pages) a.page_slots = a.max_pages;
  const int64_t kv_units = (int64_t)a.B * a.page_slots * a.Hkv;
  int64_t q_blocks = 0;
  if (a.q) {
    // the heads of a block share the angles: at least four of them unless that leaves SMs idle
    const int64_t gx = ((int64_t)a.B * a.M * (a.D / 16) + threads - 1) / threads;
    int64_t groups = (kNumSms * 16 + gx - 1) / gx, most = (a.Hq + 3) / 4;
    if (gx * most < kNumSms * 8) most = a.Hq;
    if (groups > most) groups = most;
    a.q_heads_per_block = (int)((a.Hq + groups - 1) / groups);
    a.q_head_groups = (a.Hq + a.q_heads_per_block - 1) / a.q_heads_per_block;
    q_blocks = gx * a.q_head_groups;
  }
  const int64_t blocks = 2 * kv_units + q_blocks;
  if (blocks == 0) return SL8_OK;
  if (blocks > 0x7fffffffll || (int64_t)a.B * a.M * (a.D / 16) + threads > 0xffffffffll) return SL8_ERR_TOO_LARGE;
  a.kv_units = (uint32_t)kv_units;
  if (nit <= 1) append_kernel<T, 1><<<(unsigned)blocks, threads, 0, stream>>>(a);
  else if (nit == 2) append_kernel<T, 2><<<(unsigned)blocks, threads, 0, stream>>>(a);
  else append_kernel<T, 0><<<(unsigned)blocks, threads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SL8_OK : SL8_ERR_CUDA;
}

struct ReadArgs {
  const int8_t *k, *v;
  const float *ks, *vs;
  void *k_out, *v_out;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* first;      // nullable: 0
  int Hkv, count, D, page_shift, max_pages, num_pages;
};

// 16 codes -> 16 values; a thread's piece of a row for K and the same piece for V.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  const int per_row = a.D / 16, row_shift = __ffs(per_row) - 1;
  const uint32_t item = blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(item >> row_shift), j = (int)(item & (per_row - 1)), h = blockIdx.y, b = blockIdx.z;
  if (i >= a.count) return;
  const int64_t row = ((int64_t)b * a.Hkv + h) * a.count + i;
  const int64_t token = (a.first ? (int64_t)__ldg(a.first + b) : 0) + i;
  int page = -1;
  if (token >= 0 && token < __ldg(a.lens + b) && (token >> a.page_shift) < a.max_pages)
    page = __ldg(a.table + b * a.table_stride + (token >> a.page_shift));
  uint4 kc = make_uint4(0, 0, 0, 0), vc = kc;
  float ks = 0.f, vs = 0.f;
  if (page >= 0 && page < a.num_pages) {
    const int64_t ph = (int64_t)page * a.Hkv + h;
    const int64_t at = ((ph << a.page_shift) + (token & ((1 << a.page_shift) - 1))) * a.D + 16 * j;
    kc = *reinterpret_cast<const uint4*>(a.k + at);
    vc = *reinterpret_cast<const uint4*>(a.v + at);
    ks = __ldg(a.ks + ph);
    vs = __ldg(a.vs + ph);
  }
  auto put = [&](const uint4& p, float scale, void* out) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
    uint4 o[2];
    uint32_t* y = reinterpret_cast<uint32_t*>(o);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)(w[n] >> (8 * e)) * scale;
      y[2 * n] = pack2<T>(x[0], x[1]);
      y[2 * n + 1] = pack2<T>(x[2], x[3]);
    }
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(out) + row * a.D + 16 * j);
    dst[0] = o[0];
    dst[1] = o[1];
  };
  put(kc, ks, a.k_out);
  put(vc, vs, a.v_out);
}

int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (1 << s)) return s;
  return -1;
}

bool rows16(const void* x, int64_t sb, int64_t sh, int64_t ss) {
  return aligned16(x) && sb % 8 == 0 && sh % 8 == 0 && ss % 8 == 0;
}

int cache_checks(const sl8_paged_cache* c) {
  if (c->D != 32 && c->D != 64 && c->D != 128 && c->D != 256) return SL8_ERR_BAD_HEAD_DIM;
  if (c->num_pages < 0 || c->Hkv < 0 || c->max_pages < 0 || page_shift_of(c->page_size) < 0) return SL8_ERR_BAD_SHAPE;
  return SL8_OK;
}

int cache_pointers(const sl8_paged_cache* c) {
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->block_table || !c->context_lens) return SL8_ERR_NULL;
  return aligned16(c->k) && aligned16(c->v) ? SL8_OK : SL8_ERR_MISALIGNED;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" int sl8_kv_append_paged(const sl8_paged_cache* c, const sl8_append_params* p, void* stream) {
  if (c == nullptr || p == nullptr) return SL8_ERR_NULL;
  int rc = cache_checks(c);
  if (rc != SL8_OK) return rc;
  if (p->B < 0 || p->Hq < 0 || p->M < 0 || p->n_axes < 1) return SL8_ERR_BAD_SHAPE;
  if (p->rot < 0 || p->rot > c->D || p->rot % 16 != 0) return SL8_ERR_BAD_SHAPE;
  if (p->dtype != SL8_F16 && p->dtype != SL8_BF16) return SL8_ERR_BAD_DTYPE;
  if (p->M > 0x40000000) return SL8_ERR_TOO_LARGE;
  if ((int64_t)p->B * p->M == 0 || c->Hkv == 0) return SL8_OK;
  if (!p->k_new || !p->v_new || (p->rot > 0 && !p->inv_freq) || (p->q && !p->q_out)) return SL8_ERR_NULL;
  // an empty pool or table stores nothing but still rotates Q
  const bool store = c->num_pages > 0 && c->max_pages > 0;
  if (store) {
    rc = cache_pointers(c);
    if (rc != SL8_OK) return rc;
  } else if (!c->context_lens) {
    return SL8_ERR_NULL;
  }
  if (!rows16(p->k_new, p->k_stride_b, p->k_stride_h, p->k_stride_s) || !rows16(p->v_new, p->v_stride_b, p->v_stride_h, p->v_stride_s))
    return SL8_ERR_MISALIGNED;
  if (p->q && (!rows16(p->q, p->q_stride_b, p->q_stride_h, p->q_stride_s) ||
               !rows16(p->q_out, p->q_out_stride_b, p->q_out_stride_h, p->q_out_stride_s)))
    return SL8_ERR_MISALIGNED;
  AppendArgs a{};
  a.k = PoolArgs{p->k_new, p->k_stride_b, p->k_stride_h, p->k_stride_s, c->k, c->k_scale};
  a.v = PoolArgs{p->v_new, p->v_stride_b, p->v_stride_h, p->v_stride_s, c->v, c->v_scale};
  a.q = p->Hq > 0 ? p->q : nullptr;
  a.q_out = p->q_out;
  a.q_sb = p->q_stride_b; a.q_sh = p->q_stride_h; a.q_ss = p->q_stride_s;
  a.qo_sb = p->q_out_stride_b; a.qo_sh = p->q_out_stride_h; a.qo_ss = p->q_out_stride_s;
  a.f = RopeFreq{p->positions, p->pos_stride_axis, p->pos_stride_b, p->pos_stride_s, p->inv_freq,
                 p->n_axes > 1 ? p->freq_axis : nullptr, p->pos_is_64 != 0, p->n_axes, p->rot / 2, 1.f};
  a.table = c->block_table; a.table_stride = c->table_stride; a.lens = c->context_lens; a.new_lens = p->new_lens;
  a.B = p->B; a.Hq = p->Hq; a.Hkv = c->Hkv; a.M = p->M; a.D = c->D; a.page_shift = page_shift_of(c->page_size);
  a.max_pages = store ? c->max_pages : 0; a.num_pages = c->num_pages; a.interleaved = p->interleaved;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p->dtype == SL8_F16 ? launch_append<__half>(a, s) : launch_append<__nv_bfloat16>(a, s);
}

extern "C" int sl8_kv_read_paged(const sl8_paged_cache* c, int32_t B, const int32_t* first, int32_t count, int dtype, void* k_out,
                                 void* v_out, void* stream) {
  if (c == nullptr) return SL8_ERR_NULL;
  int rc = cache_checks(c);
  if (rc != SL8_OK) return rc;
  if (B < 0 || count < 0) return SL8_ERR_BAD_SHAPE;
  if (dtype != SL8_F16 && dtype != SL8_BF16) return SL8_ERR_BAD_DTYPE;
  const int64_t rows = (int64_t)B * c->Hkv * count;
  if (rows == 0) return SL8_OK;
  if (!k_out || !v_out) return SL8_ERR_NULL;
  if (!aligned16(k_out) || !aligned16(v_out)) return SL8_ERR_MISALIGNED;
  const bool held = c->num_pages > 0 && c->max_pages > 0;
  if (held) {
    rc = cache_pointers(c);
    if (rc != SL8_OK) return rc;
  } else if (!c->context_lens) {
    return SL8_ERR_NULL;
  }
  ReadArgs a{c->k, c->v, c->k_scale, c->v_scale, k_out, v_out, c->block_table, c->table_stride, c->context_lens, first,
             c->Hkv, count, c->D, page_shift_of(c->page_size), held ? c->max_pages : 0, c->num_pages};
  const int64_t gx = ((int64_t)count * (c->D / 16) + 255) / 256;
  if (gx * 256 > 0xffffffffll || c->Hkv > 65535 || B > 65535) return SL8_ERR_TOO_LARGE;
  const dim3 blocks((unsigned)gx, (unsigned)c->Hkv, (unsigned)B);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == SL8_F16) read_kernel<__half><<<blocks, 256, 0, s>>>(a);
  else read_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? SL8_OK : SL8_ERR_CUDA;
}
