// Attention of one or several query tokens per sequence over the paged int8 cache (one scale per page and
// KV head): out = softmax(scale q.K^T) V with K = code_k s_k, V = code_v s_v.
//
// Mathematics.  s_k is constant over a page, so logit = (q . code_k) s_k, and s_v moves into the exponent:
//   w_n = exp2(logit_n + log2 s_v(n) - M),  M = running maximum of the exponent,
//   O = sum_n w_n code_v(n),  l = sum_n w_n / s_v(n),  out = O / l.
// w lies in (0, 1], so its rounding to fp16 for the P.V product loses 2^-12 of each term whatever the pages'
// scales are.  q is split into two int8 planes, q = (128 hi + lo) qs with |128 hi + lo| <= 16256 per row
// (half a step is 2^-15 of the row's largest value: finer than bf16, at fp16's level for the values that
// matter), so K's codes enter the integer MMA as they lie in memory and only V's are widened.
//
// What bounds it: HBM, 2 D bytes per key and KV head.  All query rows that share a KV head (the GQA group
// times the query tokens) are served by one pass over its keys, with keys on the M axis of the MMA (16 per
// warp and step) and 8 query rows on the N axis, so a group of 8 heads wastes nothing.  Every warp streams
// its own 16-key chunks (a chunk never crosses a page: page sizes are multiples of 16) through a private
// ring of cp.async stages: no barrier inside the loop, 160 KB in flight per SM.
//
// Split.  The chunks of all (sequence, KV head) units form one line, cut into equal ranges, one per block
// of a one-block-per-SM grid, whatever the lengths are; a unit that lies in one range is finished there,
// the others leave (O, M, l) partials that a second kernel joins.  The loads run ahead across unit
// boundaries, so merging a unit's warps does not drain the ring.
#include "sl8_common.cuh"
#include "sl8_mma.cuh"

#include <atomic>

namespace sl8 {
namespace {

constexpr int kPaWarps = 8;
constexpr int kPaThreads = 32 * kPaWarps;
constexpr int kChunk = 16;      // keys per warp and step

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
  int page_shift, num_pages, max_pages;
  int causal, window, bf16;
  int row_warps;      // warps that share a key but hold other rows (1, 2, 4)
  int rows_per_unit, row_units;            // rows = up to row_units * rows_per_unit
  int blocks;         // blocks of the split kernel
  float scale_log2;   // softmax_scale * log2 e
};

// What a sequence asks for: tokens that exist, its query tokens, the first 16-key chunk a query can see.
struct Seq {
  int len, n, first_chunk, chunks;
  int place;   // of query token 0
};

__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int b) {
  Seq s;
  const int context = __ldg(a.lens + b);
  s.n = a.query_lens ? min(max(__ldg(a.query_lens + b), 0), a.M) : a.M;
  const int64_t held = (int64_t)a.max_pages << a.page_shift;
  s.len = (int)min((int64_t)max(context, 0), held);
  s.place = max(context, 0) - s.n;
  int64_t lo = 0;
  if (a.window >= 0) lo = max((int64_t)0, (int64_t)s.place - a.window + 1);
  s.first_chunk = (int)(lo / kChunk);
  s.chunks = (s.n > 0 && lo < s.len) ? (s.len + kChunk - 1) / kChunk - s.first_chunk : 0;
  return s;
}

// Block-wide: chunks of all units together, and those of the sequences before `upto`.
// `find` >= 0 (a place on the line) also yields the sequence that holds it.
struct Line {
  long long total, before;
  int b;   // sequence that holds `find`
};

__device__ Line line_of(const PagedArgs& a, int upto, int units, long long (*red)[2]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long sum = 0, pre = 0;
  for (int b = tid; b < a.B; b += kPaThreads) {
    const long long c = seq_of(a, b).chunks;
    sum += c;
    if (b < upto) pre += c;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    pre += __shfl_xor_sync(0xffffffffu, pre, o);
  }
  if (lane == 0) { red[warp][0] = sum; red[warp][1] = pre; }
  __syncthreads();
  Line l{0, 0, 0};
  for (int w = 0; w < kPaWarps; ++w) { l.total += red[w][0]; l.before += red[w][1]; }
  l.total *= units;
  l.before *= units;
  return l;
}

// Chunks per block: equal shares, whole rounds of the block's warps.
__device__ __forceinline__ long long share_of(long long total, int blocks) {
  const long long per = (total + blocks - 1) / blocks;
  return max((long long)kPaWarps, (per + kPaWarps - 1) / kPaWarps * kPaWarps);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 16-byte piece `c` of row `r` of a [16][D] byte tile: pieces are exchanged within 128 bytes so that the
// eight rows of an ldmatrix lie in eight different bank groups.
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  constexpr int SH = D >= 128 ? 0 : (D == 64 ? 1 : 2);
  constexpr int MASK = D >= 128 ? 7 : D / 16 - 1;
  return r * D + ((c ^ ((r >> SH) & MASK)) << 4);
}

template <int D, int NG>
struct PaCfg {
  static constexpr int SLOT = 2 * kChunk * D + 16;                       // K rows, V rows, the two scales
  static constexpr int STAGES = D == 256 ? 2 : (D == 128 ? 5 : (D == 64 ? 10 : 16));
  static constexpr int RING = kPaWarps * STAGES * SLOT;
  static constexpr int BUF_ROW = D + 8;                                  // floats per row of the merge buffer
  static constexpr int BUF = kPaWarps * 8 * BUF_ROW * 4;
  static constexpr int Q_GROUP = D * 16;                                 // two int8 planes of 8 rows, fragment order
  static constexpr int ML = kPaWarps * NG * 8 * 8;
  static constexpr int GROUPS = D == 256 ? 4 : 8;                        // row groups of 8 a block may hold
  static constexpr int smem(int row_warps) { return RING + BUF + ML + row_warps * NG * (Q_GROUP + 32); }
  static_assert(smem(GROUPS / NG) <= 226 * 1024, "over the shared memory of an SM");
};

template <int D, int NG>
__global__ void __launch_bounds__(kPaThreads, 1) paged_split_kernel(const PagedArgs a) {
  using C = PaCfg<D, NG>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long red[kPaWarps][2];
  __shared__ int s_start[3];
  float* buf = reinterpret_cast<float*>(smem + C::RING);
  float2* ml = reinterpret_cast<float2*>(smem + C::RING + C::BUF);       // [warp][NG * 8]
  uint4* qf = reinterpret_cast<uint4*>(smem + C::RING + C::BUF + C::ML); // [group][D / 32][lane]
  float* qs = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(qf) + a.row_warps * NG * C::Q_GROUP);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int key_warps = kPaWarps / a.row_warps;
  const int rw = warp / key_warps, kw = warp - rw * key_warps;
  const int units = a.Hkv * a.row_units;                                 // of one sequence

  // ---- this block's range of the line ----
  const Line line = line_of(a, 0, units, red);
  const long long per = share_of(line.total, a.blocks);
  const long long c0 = per * blockIdx.x;
  const long long c1 = min(line.total, c0 + per);
  if (c0 >= c1) return;
  if (warp == 0) {
    // the sequence that holds c0: a warp walks the batch 32 at a time
    long long at = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + lane;
      const long long own = b < a.B ? (long long)seq_of(a, b).chunks * units : 0;
      long long inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const long long begin = at + inc - own;
      if (own > 0 && begin <= c0 && c0 < begin + own) {
        const int chunks = (int)(own / units);
        s_start[0] = b;
        s_start[1] = (int)((c0 - begin) / chunks);
        s_start[2] = (int)((c0 - begin) % chunks);
      }
      at += __shfl_sync(0xffffffffu, inc, 31);
      if (at > c0) break;
    }
  }
  __syncthreads();

  // ---- the loads' cursor: this warp's next chunk, running ahead of the compute cursor ----
  struct Cursor {
    int b, u, c, cend;
    long long left;    // chunks of the block's range behind this segment
    Seq s;
  };
  auto open = [&](Cursor& x, int c_begin) {
    x.cend = (int)min((long long)x.s.chunks, c_begin + x.left);
    x.left -= x.cend - c_begin;
    x.c = c_begin + kw;
  };
  auto next_unit = [&](Cursor& x) {   // only while x.left > 0: there is a unit with chunks ahead
    if (++x.u == units) {
      x.u = 0;
      do { x.s = seq_of(a, ++x.b); } while (x.s.chunks == 0);
    }
    open(x, 0);
  };
  Cursor cur;
  cur.b = s_start[0]; cur.u = s_start[1];
  cur.s = seq_of(a, cur.b);
  cur.left = c1 - c0;
  int c_begin = s_start[2];
  open(cur, c_begin);

  uint8_t* ring = smem + warp * C::STAGES * C::SLOT;
  const uint32_t ring_addr = smem_u32(ring);
  Cursor ahead = cur;
  bool more = true;
  int page = -1;
  auto find_page = [&]() {   // the page of the cursor's chunk, asked for one step before it is needed
    while (ahead.c >= ahead.cend) {
      if (ahead.left <= 0) { more = false; return; }
      next_unit(ahead);
    }
    page = __ldg(a.table + ahead.b * a.table_stride + ((int64_t)(ahead.s.first_chunk + ahead.c) * kChunk >> a.page_shift));
  };
  find_page();
  auto issue = [&](int slot) {
    if (more) {
      const bool held = page >= 0 && page < a.num_pages;   // otherwise zeros, and a scale of 0: nothing is seen
      const int64_t ph = held ? (int64_t)page * a.Hkv + ahead.u / a.row_units : 0;
      const int in_page = ((ahead.s.first_chunk + ahead.c) * kChunk) & ((1 << a.page_shift) - 1);
      const int64_t at = ((ph << a.page_shift) + (held ? in_page : 0)) * D;
      const uint32_t dst = ring_addr + slot * C::SLOT;
      const int n16 = held ? 16 : 0, n4 = held ? 4 : 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int idx = lane + 32 * i, r = idx / (D / 16), c = idx % (D / 16);
        cp_async16(dst + tile_offset<D>(r, c), a.k + at + 16 * idx, n16);
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int idx = lane + 32 * i, r = idx / (D / 16), c = idx % (D / 16);
        cp_async16(dst + kChunk * D + tile_offset<D>(r, c), a.v + at + 16 * idx, n16);
      }
      if (lane < 2) cp_async4(dst + 2 * kChunk * D + 4 * lane, (lane ? a.vs : a.ks) + ph, n4);
      ahead.c += key_warps;
      find_page();
    }
    cp_async_commit();
  };
  int slot_in = 0, slot_out = 0;
#pragma unroll 1
  for (int i = 0; i < C::STAGES - 1; ++i) issue(i);
  slot_in = C::STAGES - 1;

  float o[NG][D / 16][4];
  while (true) {
    // ================= one segment: chunks [c_begin, cur.cend) of unit (cur.b, cur.u) =================
    const int hkv = cur.u / a.row_units, row0 = (cur.u % a.row_units) * a.rows_per_unit;
    const Seq s = cur.s;
    // ---- Q of the segment: two int8 planes in fragment order ----
    for (int grp = warp; grp < a.row_warps * NG; grp += kPaWarps) {
      const int r = row0 + grp * 8 + g;
      const int i = r / a.G, head = hkv * a.G + r % a.G;
      const bool live = r < a.rows && i < s.n;
      const uint2* src = reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(a.q) + cur.b * a.q_sb + head * a.q_sh + i * a.q_ss);
      float x[D / 32][2][4];
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 p = live ? __ldg(src + 8 * w + 4 * h + t) : make_uint2(0, 0);
          const float2 u0 = a.bf16 ? unpack2<__nv_bfloat16>(p.x) : unpack2<__half>(p.x);
          const float2 u1 = a.bf16 ? unpack2<__nv_bfloat16>(p.y) : unpack2<__half>(p.y);
          x[w][h][0] = u0.x; x[w][h][1] = u0.y; x[w][h][2] = u1.x; x[w][h][3] = u1.y;
#pragma unroll
          for (int e = 0; e < 4; ++e)   // as bits: a NaN stays the largest
            top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(x[w][h][e]) & 0x7fffffffu));
        }
      }
      uint32_t bits = __float_as_uint(top);
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
      bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
      top = __uint_as_float(bits);
      const float inv = top < 1e-30f ? 0.f : 16256.f / top;   // a row of zeros has logits of zero
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int q16 = __float2int_rn(x[w][h][e] * inv);
            const int q_hi = (q16 + 64) >> 7;
            hi[h] |= (uint32_t)(q_hi & 255) << (8 * e);
            lo[h] |= (uint32_t)((q16 - 128 * q_hi) & 255) << (8 * e);
          }
        qf[(grp * (D / 32) + w) * 32 + lane] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
      }
      if (t == 0) qs[grp * 8 + g] = top * (1.f / 16256.f) * a.scale_log2;
    }
    __syncthreads();

    // ---- the segment's rows of this warp ----
    float row_scale[NG][2], m_run[NG][2], l_run[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_scale[ng][e] = qs[(rw * NG + ng) * 8 + 2 * t + e];
        m_run[ng][e] = kNegSentinel;
        l_run[ng][e] = 0.f;
      }
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[ng][d][0] = o[ng][d][1] = o[ng][d][2] = o[ng][d][3] = 0.f;
    // keys every valid row of the warp sees: [all_from, all_to)
    const int r_first = row0 + rw * NG * 8;
    const int i_first = r_first / a.G, i_last = min(s.n, (min(a.rows, r_first + NG * 8) - 1) / a.G + 1) - 1;
    const int all_to = a.causal ? min(s.len, s.place + i_first + 1) : s.len;
    const int all_from = a.window >= 0 ? s.place + i_last - a.window + 1 : 0;

    for (int c = cur.c; c < cur.cend; c += key_warps) {
      issue(slot_in);
      slot_in = slot_in + 1 == C::STAGES ? 0 : slot_in + 1;
      cp_async_wait<C::STAGES - 1>();
      __syncwarp();
      const uint32_t kbase = ring_addr + slot_out * C::SLOT, vbase = kbase + kChunk * D;
      const float2 scales = *reinterpret_cast<const float2*>(ring + slot_out * C::SLOT + 2 * kChunk * D);
      slot_out = slot_out + 1 == C::STAGES ? 0 : slot_out + 1;
      if (scales.y == 0.f) { __syncwarp(); continue; }        // a page that holds nothing
      const int key0 = (s.first_chunk + c) * kChunk;
      const bool whole = key0 + kChunk <= all_to && key0 >= all_from;
      const float lv = log2f(scales.y), iv = 1.f / scales.y;

      uint32_t kf[D / 32][4];
#pragma unroll
      for (int w = 0; w < D / 32; ++w)
        ldmatrix_x4(kf[w], kbase + tile_offset<D>((lane & 7) + ((lane >> 3) & 1) * 8, 2 * w + (lane >> 4)));
      uint32_t pb[NG][2];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        // ---- S^T = K . Q^T: keys g, g + 8, rows 2t, 2t + 1 ----
        int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          const uint4 q4 = qf[((rw * NG + ng) * (D / 32) + w) * 32 + lane];
          mma_s8_16832(hi, kf[w], q4.x, q4.y);
          mma_s8_16832(lo, kf[w], q4.z, q4.w);
        }
        float x[4], mx[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf((float)(hi[e] * 128 + lo[e]), row_scale[ng][e & 1] * scales.x, lv);
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = (r_first + ng * 8 + 2 * t + (e & 1)) / a.G, place = s.place + i, key = key0 + g + 8 * (e >> 1);
            const bool seen = key < s.len && (!a.causal || key <= place) && (a.window < 0 || key > place - a.window);
            if (!seen) x[e] = -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(x[e], x[e + 2]);
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
        }
        const bool grown = mx[0] > m_run[ng][0] || mx[1] > m_run[ng][1];
        if (__any_sync(0xffffffffu, grown)) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m = fmaxf(m_run[ng][e], mx[e]);
            f[e] = ex2_approx(m_run[ng][e] - m);
            m_run[ng][e] = m;
            l_run[ng][e] *= f[e];
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[ng][d][0] *= f[0];
            o[ng][d][1] *= f[1];
            o[ng][d][2] *= f[0];
            o[ng][d][3] *= f[1];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = ex2_approx(x[e] - m_run[ng][e & 1]);
        l_run[ng][0] = fmaf(x[0] + x[2], iv, l_run[ng][0]);
        l_run[ng][1] = fmaf(x[1] + x[3], iv, l_run[ng][1]);
        pb[ng][0] = transpose8x8(pack2<__half>(x[0], x[1]));
        pb[ng][1] = transpose8x8(pack2<__half>(x[2], x[3]));
      }
      // ---- O^T += V^T . P^T.  A transposing ldmatrix hands out byte pairs of two neighbouring channels for
      // keys 2t, 2t + 1; widened exactly ((b ^ 0x80) | 0x6400 is 1152 + b), channel 2g feeds row g of the
      // tile and channel 2g + 1 row g + 8 ----
      const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
      auto widen = [&](uint32_t x, uint32_t sel) -> uint32_t {
        const uint32_t u = __byte_perm(x, 0x64646464u, sel);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), bias);
        return *reinterpret_cast<const uint32_t*>(&h);
      };
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        uint32_t r[4];
        ldmatrix_x4_trans(r, vbase + tile_offset<D>((lane & 7) + ((lane >> 3) & 1) * 8, 2 * w + (lane >> 4)));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t y0 = r[2 * half] ^ 0x80808080u, y1 = r[2 * half + 1] ^ 0x80808080u;
          const uint32_t va[4] = {widen(y0, 0x4240u), widen(y0, 0x4341u), widen(y1, 0x4240u), widen(y1, 0x4341u)};
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) mma_f16_16816(o[ng][2 * w + half], va, pb[ng][0], pb[ng][1]);
        }
      }
      __syncwarp();
    }

    // ================= join the key warps and write =================
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[ng][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) ml[warp * NG * 8 + ng * 8 + 2 * t + e] = make_float2(m_run[ng][e], l);
      }
    __syncthreads();
    const bool complete = c_begin == 0 && cur.cend == s.chunks;
    const int64_t part = (2ll * blockIdx.x + (c_begin == 0)) * a.rows_per_unit;
#pragma unroll
    for (int ng = 0; ng < NG; ++ng) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m = kNegSentinel;
        for (int w = 0; w < key_warps; ++w) m = fmaxf(m, ml[(rw * key_warps + w) * NG * 8 + ng * 8 + 2 * t + e].x);
        f[e] = ex2_approx(m_run[ng][e] - m);
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        float* dst = buf + (warp * 8 + 2 * t) * C::BUF_ROW + 16 * d + 2 * g;
        *reinterpret_cast<float2*>(dst) = make_float2(o[ng][d][0] * f[0], o[ng][d][2] * f[0]);
        *reinterpret_cast<float2*>(dst + C::BUF_ROW) = make_float2(o[ng][d][1] * f[1], o[ng][d][3] * f[1]);
      }
      __syncthreads();
      for (int idx = kw * 32 + lane; idx < 2 * D; idx += key_warps * 32) {
        const int row = idx / (D / 4), d4 = idx % (D / 4);
        float m = kNegSentinel, l = 0.f;
        for (int w = 0; w < key_warps; ++w) m = fmaxf(m, ml[(rw * key_warps + w) * NG * 8 + ng * 8 + row].x);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < key_warps; ++w) {
          const float2 one = ml[(rw * key_warps + w) * NG * 8 + ng * 8 + row];
          l += one.y * ex2_approx(one.x - m);
          const float4 x = *reinterpret_cast<const float4*>(buf + ((rw * key_warps + w) * 8 + row) * C::BUF_ROW + 4 * d4);
          sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
        }
        const int r_local = (rw * NG + ng) * 8 + row, r = row0 + r_local;
        if (complete) {
          if (r < a.rows) {
            const int i = r / a.G, head = hkv * a.G + r % a.G;
            const float inv = (i < s.n && l != 0.f) ? 1.f / l : 0.f;
            if (inv == 0.f) sum = make_float4(0.f, 0.f, 0.f, 0.f);
            uint2 y;
            if (a.bf16) y = make_uint2(pack2<__nv_bfloat16>(sum.x * inv, sum.y * inv), pack2<__nv_bfloat16>(sum.z * inv, sum.w * inv));
            else y = make_uint2(pack2<__half>(sum.x * inv, sum.y * inv), pack2<__half>(sum.z * inv, sum.w * inv));
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + cur.b * a.o_sb + head * a.o_sh + i * a.o_ss + 4 * d4) = y;
          }
        } else {
          *reinterpret_cast<float4*>(a.part_o + (part + r_local) * D + 4 * d4) = sum;
          if (d4 == 0) *reinterpret_cast<float2*>(a.part_ml + (part + r_local) * 2) = make_float2(m, l);
        }
      }
      __syncthreads();
    }
    if (cur.left <= 0) break;
    next_unit(cur);
    c_begin = 0;
  }
  cp_async_wait<0>();
}

// Joins the partials of the units that more than one block worked on, and writes the zeros of sequences
// without keys or queries.  One block per unit, one warp per row at a time.
template <int D>
__global__ void __launch_bounds__(kPaThreads) paged_join_kernel(const PagedArgs a) {
  __shared__ long long red[kPaWarps][2];
  const int units = a.Hkv * a.row_units;
  const int b = blockIdx.x / units, u = blockIdx.x - b * units;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Line line = line_of(a, b, units, red);
  const Seq s = seq_of(a, b);
  const long long per = share_of(line.total, a.blocks);
  const long long g0 = line.before + (long long)u * s.chunks;
  const long long i0 = g0 / per, i1 = s.chunks > 0 ? (g0 + s.chunks - 1) / per : i0;
  // every block waits, also one with nothing to do: a grid that ended before the split kernel would let
  // the stream's next kernel start beside it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (s.chunks > 0 && i0 == i1) return;            // finished by its block
  const int hkv = u / a.row_units, row0 = (u % a.row_units) * a.rows_per_unit;
  constexpr int PER = D / 32;                       // channels per lane
  for (int r_local = warp; r_local < a.rows_per_unit && row0 + r_local < a.rows; r_local += kPaWarps) {
    const int r = row0 + r_local, i = r / a.G, head = hkv * a.G + r % a.G;
    float sum[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) sum[e] = 0.f;
    float l = 0.f;
    if (s.chunks > 0 && i < s.n) {
      // partial n: block i0 + n, its slot 1 where it began the unit (n = 0), else slot 0
      float m = kNegSentinel;
      const int parts = (int)(i1 - i0 + 1);
      auto row_of = [&](int n) { return (2 * (i0 + n) + (n == 0)) * a.rows_per_unit + r_local; };
      for (int n = lane; n < parts; n += 32) m = fmaxf(m, a.part_ml[row_of(n) * 2]);
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll 4
      for (int n = 0; n < parts; ++n) {
        const float2 one = *reinterpret_cast<const float2*>(a.part_ml + row_of(n) * 2);
        const float f = ex2_approx(one.x - m);
        l = fmaf(one.y, f, l);
        const float* src = a.part_o + row_of(n) * D + PER * lane;
#pragma unroll
        for (int e = 0; e < PER; ++e) sum[e] = fmaf(src[e], f, sum[e]);
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + b * a.o_sb + head * a.o_sh + i * a.o_ss + PER * lane;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const float y = inv == 0.f ? 0.f : sum[e] * inv;
      if (a.bf16) reinterpret_cast<__nv_bfloat16*>(dst)[e] = __float2bfloat16_rn(y);
      else reinterpret_cast<__half*>(dst)[e] = __float2half_rn(y);
    }
  }
}

int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (1 << s)) return s;
  return -1;
}

// Rows that one unit serves: 8 per group of the MMA's N axis, groups per warp (NG), warps with other rows.
struct Plan {
  int ng, row_warps, row_units, rows_per_unit, blocks;
};

Plan plan_of(const sl8_paged_cache& c, const sl8_paged_attn_params& p) {
  Plan x{};
  const int64_t rows = (int64_t)p.M * (p.Hq / c.Hkv);
  const int most = c.D == 256 ? 2 : 4;            // accumulators: D / 4 * NG registers a thread
  x.ng = rows <= 8 ? 1 : (rows <= 16 ? 2 : most);
  x.row_warps = 1;
  const int groups = c.D == 256 ? 4 : 8;          // PaCfg::GROUPS
  while (x.row_warps * x.ng * 8 < rows && x.row_warps * x.ng < groups) x.row_warps *= 2;
  x.rows_per_unit = x.row_warps * x.ng * 8;
  x.row_units = (int)((rows + x.rows_per_unit - 1) / x.rows_per_unit);
  const int64_t held = (int64_t)c.max_pages * c.page_size;
  const int64_t longest = p.max_context_len > 0 && p.max_context_len < held ? p.max_context_len : held;
  const int64_t chunks = (longest + kChunk - 1) / kChunk * p.B * c.Hkv * x.row_units;
  const int64_t want = (chunks + kPaWarps - 1) / kPaWarps;
  x.blocks = (int)(want < 1 ? 1 : (want > kNumSms ? kNumSms : want));
  return x;
}

int paged_checks(const sl8_paged_cache* c, const sl8_paged_attn_params* p) {
  if (c == nullptr || p == nullptr) return SL8_ERR_NULL;
  if (c->D != 32 && c->D != 64 && c->D != 128 && c->D != 256) return SL8_ERR_BAD_HEAD_DIM;
  if (p->dtype != SL8_F16 && p->dtype != SL8_BF16) return SL8_ERR_BAD_DTYPE;
  if (c->num_pages < 0 || c->Hkv < 0 || c->max_pages < 0 || page_shift_of(c->page_size) < 0) return SL8_ERR_BAD_SHAPE;
  if (p->B < 0 || p->Hq < 0 || p->M < 0) return SL8_ERR_BAD_SHAPE;
  if (p->Hq > 0 && (c->Hkv == 0 || p->Hq % c->Hkv != 0)) return SL8_ERR_BAD_SHAPE;
  return SL8_OK;
}

template <int D, int NG>
int launch_paged(const PagedArgs& a, cudaStream_t stream) {
  static std::atomic<bool> allowed[64];
  int dev = 0;
  SL8_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !allowed[dev].load()) {
    SL8_CUDA_TRY(cudaFuncSetAttribute(paged_split_kernel<D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      PaCfg<D, NG>::smem(PaCfg<D, NG>::GROUPS / NG)));
    if (dev < 64) allowed[dev].store(true);
  }
  const int smem = PaCfg<D, NG>::smem(a.row_warps);
  paged_split_kernel<D, NG><<<a.blocks, kPaThreads, smem, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return SL8_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.row_units));
  cfg.blockDim = dim3(kPaThreads);
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  SL8_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, a));
  return SL8_OK;
}

template <int D>
int launch_paged_rows(const PagedArgs& a, int ng, cudaStream_t stream) {
  switch (ng) {
    case 1: return launch_paged<D, 1>(a, stream);
    case 2: return launch_paged<D, 2>(a, stream);
    default:
      if constexpr (D == 256) return SL8_ERR_UNSUPPORTED;
      else return launch_paged<D, 4>(a, stream);
  }
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_attn_paged_workspace(const sl8_paged_cache* c, const sl8_paged_attn_params* p) {
  if (paged_checks(c, p) != SL8_OK || (int64_t)p->B * p->Hq * p->M == 0) return 256;
  const Plan x = plan_of(*c, *p);
  return 256 + (size_t)2 * x.blocks * x.rows_per_unit * (c->D + 2) * sizeof(float);
}

extern "C" int sl8_attn_paged(const sl8_paged_cache* c, const sl8_paged_attn_params* p, void* workspace, size_t workspace_bytes,
                              void* stream) {
  int rc = paged_checks(c, p);
  if (rc != SL8_OK) return rc;
  if ((int64_t)p->B * p->Hq * p->M == 0) return SL8_OK;
  if (!p->q || !p->out || !c->context_lens) return SL8_ERR_NULL;
  const bool held = c->num_pages > 0 && c->max_pages > 0;
  if (held && (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->block_table)) return SL8_ERR_NULL;
  if (!aligned16(p->q) || !aligned16(p->out) || (held && (!aligned16(c->k) || !aligned16(c->v)))) return SL8_ERR_MISALIGNED;
  if (p->q_stride_b % 8 || p->q_stride_h % 8 || p->q_stride_s % 8 || p->out_stride_b % 8 || p->out_stride_h % 8 || p->out_stride_s % 8)
    return SL8_ERR_MISALIGNED;
  if (workspace == nullptr || workspace_bytes < sl8_attn_paged_workspace(c, p)) return SL8_ERR_WORKSPACE;
  if (!aligned16(workspace)) return SL8_ERR_MISALIGNED;
  const Plan x = plan_of(*c, *p);
  if ((int64_t)p->B * c->Hkv * x.row_units > 0x7fffffffll) return SL8_ERR_TOO_LARGE;
  PagedArgs a{};
  a.q = p->q; a.q_sb = p->q_stride_b; a.q_sh = p->q_stride_h; a.q_ss = p->q_stride_s;
  a.out = p->out; a.o_sb = p->out_stride_b; a.o_sh = p->out_stride_h; a.o_ss = p->out_stride_s;
  a.k = c->k; a.v = c->v; a.ks = c->k_scale; a.vs = c->v_scale;
  a.table = c->block_table; a.table_stride = c->table_stride; a.lens = c->context_lens; a.query_lens = p->query_lens;
  a.part_o = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + 256);
  a.part_ml = a.part_o + (size_t)2 * x.blocks * x.rows_per_unit * c->D;
  a.B = p->B; a.Hq = p->Hq; a.Hkv = c->Hkv; a.M = p->M; a.G = p->Hq / c->Hkv; a.rows = p->M * a.G;
  a.page_shift = page_shift_of(c->page_size); a.num_pages = c->num_pages; a.max_pages = held ? c->max_pages : 0;
  a.causal = p->causal; a.window = p->window_left; a.bf16 = p->dtype == SL8_BF16;
  a.row_warps = x.row_warps; a.rows_per_unit = x.rows_per_unit; a.row_units = x.row_units; a.blocks = x.blocks;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (c->D) {
    case 32: return launch_paged_rows<32>(a, x.ng, s);
    case 64: return launch_paged_rows<64>(a, x.ng, s);
    case 128: return launch_paged_rows<128>(a, x.ng, s);
    default: return launch_paged_rows<256>(a, x.ng, s);
  }
}
