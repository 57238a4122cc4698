// Attention of one or several query tokens per sequence over the paged int8 cache (one scale per page and
// KV head): out = softmax(scale q.K^T) V with K = code_k s_k, V = code_v s_v.
//
// Mathematics.  s_k is constant over a page, so logit = (q . code_k) s_k, and s_v moves into the exponent:
//   w_n = exp2(logit_n + log2 s_v(n) - M),  M = running maximum of the exponent,
//   O = sum_n w_n code_v(n),  l = sum_n w_n / s_v(n),  out = O / l.
// w stays below 2^8, so its rounding to fp16 for the P.V product loses 2^-11 of each term at most whatever the
// pages' scales are.  q is split into two int8 planes, q = (128 hi + lo) qs with |128 hi + lo| <= 16256 per row
// (half a step is 2^-15 of the row's largest value: finer than bf16, at fp16's level for the values that
// matter), so K's codes enter the integer MMA as they lie in memory and only V's are widened.
//
// What bounds it: HBM, 2 D bytes per key and KV head.  All query rows that share a KV head (the GQA group
// times the query tokens) are served by one pass over its keys, with keys on the M axis of the MMA (tiles
// of 16) and 8 query rows on the N axis, so a group of 8 heads wastes nothing.  Every warp streams
// its own chunks of 32 or 16 keys (a 16-key tile never crosses a page: page sizes are multiples of 16) through
// a private ring of TMA stages: no barrier between warps inside the loop, 128 KB in flight per SM.
//
// Split.  The chunks of all (sequence, KV head) units form one line, cut into equal ranges, one per block
// of a one-block-per-SM grid, whatever the lengths are; a unit that lies in one range is finished there,
// the others leave (O, M, l) partials that a second kernel joins.  The loads run ahead across unit
// boundaries, so merging a unit's warps does not drain the ring.  Few or short units are instead given a
// cluster of up to 8 blocks each, joined over distributed shared memory: one launch and no partials.
//
// Measured (D = 128, heads 64 : 8).  One token of 64 sequences of 1024 ... 32768 keys: 341-353 us, 6.3-6.5 TB/s
// (HBM bound).  Five tokens of 16 sequences of up to 8192 keys: 72 us where HBM would take 24; the rows are 40 per
// unit, so every 16-key tile is multiplied five times and the eight warps' instruction latency bounds it.
// One token of one sequence of 1024 keys: 7.6 us in clusters, a chain of launch, length, page, tile and join.
#include "sl8_paged.cuh"
#include "sl8_mma.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace sl8 {
namespace {

__device__ int g_paged_wait_status;   // raised by an expired wait; zero when the library is loaded

constexpr int kPaWarps = 8;
constexpr int kPaThreads = 32 * kPaWarps;

// The line: the chunks of all units, sequence by sequence (the host bounds it below 2^31).  Every thread owns
// a run of ceil(B / threads) sequences; returns the line's length and the place where the run begins.
struct Line {
  unsigned total, begin;
  int b0, b1;
};

__device__ Line line_of(const PagedArgs& a, int units, unsigned* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (a.B + kPaThreads - 1) / kPaThreads;
  Line l;
  l.b0 = min(a.B, tid * run);
  l.b1 = min(a.B, l.b0 + run);
  unsigned own = 0;
  for (int b = l.b0; b < l.b1; ++b) own += seq_of(a, b).chunks;
  own *= units;
  unsigned inc = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  l.total = 0;
  l.begin = inc - own;
#pragma unroll
  for (int w = 0; w < kPaWarps; ++w) {
    if (w == warp) l.begin += l.total;
    l.total += red[w];
  }
  return l;
}

// The unit and the chunk in it that lie at place c of the line (every c < total is found by one thread).
__device__ __forceinline__ void locate(const PagedArgs& a, const Line& line, int units, unsigned c, int (&found)[3]) {
  unsigned at = line.begin;
  if (at > c) return;
  for (int b = line.b0; b < line.b1; ++b) {
    const unsigned chunks = seq_of(a, b).chunks, own = chunks * units;
    if (c >= at && c - at < own) {
      found[0] = b;
      found[1] = (int)((c - at) / chunks);
      found[2] = (int)((c - at) % chunks);
    }
    at += own;
  }
}

// Chunks per block: equal shares, in whole rounds of the block's warps, or, where the units are shorter than that
// on average, in whole units of the average's next power of two (256 units of 16 keys: one or two units per block
// instead of eight on a few blocks).
__device__ __forceinline__ unsigned share_of(const PagedArgs& a, int units, unsigned total) {
  const unsigned per = (total + a.blocks - 1) / a.blocks;
  unsigned round = 1;
  while (round < (unsigned)kPaWarps && (uint64_t)round * units * a.B < total) round *= 2;
  return max(round, (per + round - 1) / round * round);
}

__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async4(void* dst, const void* src, int bytes) {   // 0 bytes: zero
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Where 16-byte piece `c` of row `r` of a 16-key tile lies in shared memory: sub-tiles of at most 128 bytes a
// row, as the copy engine's swizzle leaves them (the eight rows of an ldmatrix in eight different bank groups).
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  constexpr int ROW = D < 128 ? D : 128, SW = D >= 128 ? 3 : (D == 64 ? 2 : 1);
  return (c / (ROW / 16)) * (16 * ROW) + swizzle_offset<SW>(r * ROW + (c % (ROW / 16)) * 16);
}

// Keys per warp and step: 32 (two 16-key tiles share the maximum, the rescaling and the loop) where the
// accumulators leave the registers for it and the ring the space, else 16.
__host__ __device__ constexpr int chunk_shift_of(int D, int ng) { return D == 256 || (D == 128 && ng == 4) ? 4 : 5; }

// Most groups of 8 query rows a warp can accumulate: D / 4 registers a thread each.
__host__ __device__ constexpr int groups_of(int D) { return D == 256 ? 2 : 4; }

template <int D, int NG>
struct PaCfg {
  static constexpr int SHIFT = chunk_shift_of(D, NG);
  static constexpr int TILES = (1 << SHIFT) / 16;                        // 16-key tiles per chunk
  static constexpr int TILE = 2 * 16 * D;                                // K rows, V rows
  static constexpr int SLOT = TILES * TILE;
  static constexpr int SUBS = D <= 128 ? 1 : D / 128, ROW = D / SUBS;    // sub-tiles of at most 128 bytes a row
  // What streams at the HBM's rate (one group) wants 128 KB in flight; more groups take longer per step than a
  // load takes, and give the space to the join.
  static constexpr int STAGES = D == 256 ? 2 : (D == 128 ? (TILES == 2 ? (NG == 1 ? 3 : 2) : 4) : (D == 64 ? 5 : 8));
  static constexpr int RING = kPaWarps * STAGES * SLOT;
  static constexpr int SIDE = kPaWarps * STAGES * (TILES * 8 + 8);       // the tiles' scales, the slots' barriers
  // The join of a group of rows: every fragment (float4 a lane) of the other key warps' accumulators.  Two such
  // buffers where several groups follow one another and the space is there.
  static constexpr int FRAGS = D / 16, BUF_ONE = FRAGS * (kPaWarps - 1) * 512;
  static constexpr int BUFS = NG > 1 && D < 256 ? 2 : 1, BUF = BUFS * BUF_ONE;
  static constexpr int Q_GROUP = D * 16;                                 // two int8 planes of 8 rows, fragment order
  static constexpr int ROW_WARPS = NG == groups_of(D) ? 2 : 1;           // most warps with rows of their own
  static constexpr int ML = (kPaWarps + ROW_WARPS) * NG * 8 * 8;         // per warp and row, and per row
  static constexpr bool Q_REGS = NG * D <= 256;                          // fragments of Q held in registers
  static constexpr int smem(int row_warps) { return 1024 + RING + SIDE + BUF + ML + row_warps * NG * (Q_GROUP + 32); }
  static_assert(smem(ROW_WARPS) <= 227 * 1024 - 256, "over the shared memory of an SM");
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ float2 cluster_load2(const float2* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_load4(const float* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr(p, rank))
               : "memory");
  return v;
}

// Four channels of output row r of a unit: sum / l, zeros where the row has no query or saw no key.
__device__ __forceinline__ void store_row(const PagedArgs& a, int b, int hkv, int r, int n, int ch, float4 sum, float l) {
  const int i = r / a.G, head = hkv * a.G + r - i * a.G;
  const float inv = (i < n && l != 0.f) ? 1.f / l : 0.f;
  if (inv == 0.f) sum = make_float4(0.f, 0.f, 0.f, 0.f);
  uint2 y;
  if (a.bf16) y = make_uint2(pack2<__nv_bfloat16>(sum.x * inv, sum.y * inv), pack2<__nv_bfloat16>(sum.z * inv, sum.w * inv));
  else y = make_uint2(pack2<__half>(sum.x * inv, sum.y * inv), pack2<__half>(sum.z * inv, sum.w * inv));
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + b * a.o_sb + head * a.o_sh + i * a.o_ss + ch) = y;
}

// A row's reference M moves only when a logit passes it by this much (in powers of two): the weights stay
// below 2^8, far inside fp16, and the accumulators are hardly ever rescaled.
constexpr float kSlack = 8.f;

// CLUSTER: the blocks of a thread-block cluster share one unit and join through distributed shared memory,
// so no second kernel follows; otherwise the block takes its range of the line.
template <int D, int NG, bool CLUSTER>
__global__ void __launch_bounds__(kPaThreads, 1) paged_split_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                    const __grid_constant__ CUtensorMap v_map,
                                                                    const __grid_constant__ PagedArgs a) {
  using C = PaCfg<D, NG>;
  constexpr int T = C::TILES, KEYS = 1 << C::SHIFT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ unsigned red[kPaWarps];
  __shared__ int s_start[3];
  float4* buf = reinterpret_cast<float4*>(smem + C::RING);               // [fragment][other key warp][lane]
  float2* ml = reinterpret_cast<float2*>(smem + C::RING + C::BUF);       // [warp][NG * 8]
  float2* joint = ml + kPaWarps * NG * 8;                                // [row_warps * NG * 8]: reference, sum
  uint4* qf = reinterpret_cast<uint4*>(smem + C::RING + C::BUF + C::ML); // [group][D / 32][lane]
  float2* side = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(qf) + a.row_warps * NG * (C::Q_GROUP + 32));
  float* qs = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(qf) + a.row_warps * NG * C::Q_GROUP);

  if constexpr (!CLUSTER) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int key_warps = kPaWarps / a.row_warps;
  const int rw = warp / key_warps, kw = warp - rw * key_warps;
  const int units = a.Hkv * a.row_units;                                 // of one sequence
  // this warp's ring, and beside it the scales of every tile and a barrier per slot
  uint8_t* const ring = smem + warp * C::STAGES * C::SLOT;
  float2* const scales_at = side + warp * C::STAGES * T;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(side + kPaWarps * C::STAGES * T) + warp * C::STAGES;
  if (lane == 0) {
    if (warp == 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
#pragma unroll
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&bars[i], T);
    mbar_fence_init();
  }
  __syncwarp();

  // ---- the two cursors of a warp: compute, and the loads that run ahead of it across units ----
  struct Cursor {
    int b, u, c, cend;
    int left;          // chunks of the block's range behind this segment
    Seq s;
  };
  auto open = [&](Cursor& x, int c_begin) {
    x.cend = min(x.s.chunks, c_begin + x.left);
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
  int c_begin;
  if constexpr (CLUSTER) {
    // equal shares of the unit; a block without one still joins
    const int unit = blockIdx.x / a.blocks, rank = blockIdx.x - unit * a.blocks;
    cur.b = unit / units;
    cur.u = unit - cur.b * units;
    cur.s = seq_of(a, cur.b);
    const int per = (cur.s.chunks + a.blocks - 1) / a.blocks;
    c_begin = min(cur.s.chunks, rank * per);
    cur.left = min(per, cur.s.chunks - c_begin);
  } else {
    const Line line = line_of(a, units, red);
    const unsigned per = share_of(a, units, line.total);
    const unsigned c0 = min(line.total, per * blockIdx.x);
    const unsigned c1 = min(line.total, c0 + per);
    if (c0 >= c1) return;
    locate(a, line, units, c0, s_start);
    __syncthreads();
    cur.b = s_start[0]; cur.u = s_start[1];
    cur.s = seq_of(a, cur.b);
    cur.left = (int)(c1 - c0);
    c_begin = s_start[2];
  }
  open(cur, c_begin);

  // Q of a segment comes in two steps: the values (asked for early, a row per four lanes of its group's warp) and
  // their two int8 planes in fragment order.
  uint2 q_raw[D / 32][2];
  auto load_q = [&](const Cursor& x) {
    if (warp >= a.row_warps * NG) return;
    const int head0 = x.u / a.row_units, r = (x.u - head0 * a.row_units) * a.rows_per_unit + warp * 8 + g;
    const int i = r / a.G, head = head0 * a.G + r - i * a.G;
    const bool live = r < a.rows && i < x.s.n;
    const uint2* src = reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(a.q) + x.b * a.q_sb + head * a.q_sh + i * a.q_ss);
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) q_raw[w][h] = live ? __ldg(src + 8 * w + 4 * h + t) : make_uint2(0, 0);
  };
  auto split_q = [&]() {
    if (warp >= a.row_warps * NG) return;
    auto value = [&](uint32_t x) { return a.bf16 ? unpack2<__nv_bfloat16>(x) : unpack2<__half>(x); };
    uint32_t bits = 0;   // the largest magnitude, compared as bits: a NaN stays the largest
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 u0 = value(q_raw[w][h].x), u1 = value(q_raw[w][h].y);
        bits = max(bits, max(__float_as_uint(u0.x) & 0x7fffffffu, __float_as_uint(u0.y) & 0x7fffffffu));
        bits = max(bits, max(__float_as_uint(u1.x) & 0x7fffffffu, __float_as_uint(u1.y) & 0x7fffffffu));
      }
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
    const float top = __uint_as_float(bits);
    const float inv = top < 1e-30f ? 0.f : 16256.f / top;   // a row of zeros has logits of zero
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 u0 = value(q_raw[w][h].x), u1 = value(q_raw[w][h].y);
        const float v[4] = {u0.x, u0.y, u1.x, u1.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int q16 = __float2int_rn(v[e] * inv);
          const int q_hi = (q16 + 64) >> 7;
          hi[h] |= (uint32_t)(q_hi & 255) << (8 * e);
          lo[h] |= (uint32_t)((q16 - 128 * q_hi) & 255) << (8 * e);
        }
      }
      qf[(warp * (D / 32) + w) * 32 + lane] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
    }
    if (t == 0) qs[warp * 8 + g] = top * (1.f / 16256.f) * a.scale_log2;
  };
  load_q(cur);

  // Loads of a chunk: lane 16 h asks the copy engine for tile h (each tile has its own page), and for its scales
  // with two four-byte copies.
  const int l_tile = T == 2 ? lane >> 4 : 0;
  const bool loader = (lane & 15) == 0 && lane < 16 * T;
  Cursor ahead = cur;
  const int32_t* a_row = a.table + ahead.b * a.table_stride;
  int a_head = ahead.u / a.row_units;
  int a_tok = 0, page = -1;
  const int page_mask = (1 << a.page_shift) - 1;
  auto find_page = [&]() {   // the page of this lane's tile, asked for one step before it is needed
    a_tok = (ahead.s.first_chunk + ahead.c) * KEYS + 16 * l_tile;
    page = loader && a_tok < ahead.s.len ? __ldg(a_row + (a_tok >> a.page_shift)) : -1;
  };
  auto seek = [&]() {        // the next segment with a chunk for this warp; none: c stays at or past cend
    while (ahead.c >= ahead.cend && ahead.left > 0) {
      next_unit(ahead);
      a_row = a.table + ahead.b * a.table_stride;
      a_head = ahead.u / a.row_units;
    }
    if (ahead.c < ahead.cend) find_page();
  };
  auto seek_or_find = [&]() { if (ahead.c < ahead.cend) find_page(); else seek(); };
  // the first chunks' table entries come together: lane i of a half asks for the i-th chunk's
  int early = -1;
  {
    const int c = ahead.c + (lane & 15) * key_warps, tok = (ahead.s.first_chunk + c) * KEYS + 16 * l_tile;
    if ((lane & 15) < C::STAGES - 1 && c < ahead.cend && tok < ahead.s.len) early = __ldg(a_row + (tok >> a.page_shift));
  }
  auto load = [&](int slot) {   // chunk ahead.c of this segment into `slot`
    if (loader) {
      const bool held = (unsigned)page < (unsigned)a.num_pages;
      const int ph = held ? page * a.Hkv + a_head : 0, row = a_tok & page_mask;
      float2* sc = scales_at + slot * T + l_tile;                // a missing page: scales of 0, nothing is seen
      cp_async4(&sc->x, a.ks + ph, held ? 4 : 0);
      cp_async4(&sc->y, a.vs + ph, held ? 4 : 0);
      if (held) {
        uint8_t* dst = ring + slot * C::SLOT + l_tile * C::TILE;
        mbar_expect_tx(&bars[slot], C::TILE);
#pragma unroll
        for (int i = 0; i < C::SUBS; ++i) {
          tma_load_3d(dst + i * 16 * C::ROW, &k_map, &bars[slot], i * C::ROW, row, ph);
          tma_load_3d(dst + 16 * D + i * 16 * C::ROW, &v_map, &bars[slot], i * C::ROW, row, ph);
        }
      } else {
        mbar_arrive(&bars[slot]);
      }
    }
  };
  auto issue = [&](int slot) {
    if (ahead.c < ahead.cend) {
      load(slot);
      ahead.c += key_warps;
      seek_or_find();
    }
    cp_async_commit();
  };
  bool first = true;            // the first chunks, as far as this segment has them
#pragma unroll 1
  for (int i = 0; i < C::STAGES - 1; ++i) {
    const int entry = __shfl_sync(0xffffffffu, early, (lane & 16) + i);
    if (first && ahead.c < ahead.cend) {
      page = loader ? entry : -1;
      a_tok = (ahead.s.first_chunk + ahead.c) * KEYS + 16 * l_tile;
      load(i);
      ahead.c += key_warps;
      cp_async_commit();
    } else {
      if (first) seek();
      first = false;
      issue(i);
    }
  }
  if (first) seek_or_find();
  int slot_in = C::STAGES - 1, slot_out = 0;
  uint32_t parity = 0;       // of slot_out's current use
  bool ok = true;            // false once a bounded wait has expired: the block runs on without waiting
  const uint32_t ring_addr = smem_u32(ring);

  // ldmatrix rows and pieces of this lane: K tiles [key][channel] and, transposing, V
  const int m_row = (lane & 7) + ((lane >> 3) & 1) * 8, m_piece = lane >> 4;

  float o[NG][D / 16][4];
  while (true) {
    // ================= one segment: chunks [c_begin, cur.cend) of unit (cur.b, cur.u) =================
    const int hkv = cur.u / a.row_units, row0 = (cur.u - hkv * a.row_units) * a.rows_per_unit;
    const Seq s = cur.s;
    split_q();
    __syncthreads();

    // ---- the segment's rows of this warp ----
    float row_scale[NG][2], m_run[NG][2], l_run[NG][2];
    uint4 qr[C::Q_REGS ? NG : 1][C::Q_REGS ? D / 32 : 1];
    const uint4* my_q = qf + rw * NG * (D / 32) * 32 + lane;
#pragma unroll
    for (int ng = 0; ng < NG; ++ng) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_scale[ng][e] = qs[(rw * NG + ng) * 8 + 2 * t + e];
        m_run[ng][e] = kNegSentinel;
        l_run[ng][e] = 0.f;
      }
      if constexpr (C::Q_REGS) {
#pragma unroll
        for (int w = 0; w < D / 32; ++w) qr[ng][w] = my_q[(ng * (D / 32) + w) * 32];
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[ng][d][0] = o[ng][d][1] = o[ng][d][2] = o[ng][d][3] = 0.f;
    }
    // keys every valid row of the warp sees: [all_from, all_to)
    const int r_first = row0 + rw * NG * 8;
    const int i_first = r_first / a.G, i_last = min(s.n, (min(a.rows, r_first + NG * 8) - 1) / a.G + 1) - 1;
    const int all_to = a.causal ? min(s.len, s.place + i_first + 1) : s.len;
    const int all_from = a.window >= 0 ? s.place + i_last - a.window + 1 : 0;

    for (int c = cur.c; c < cur.cend; c += key_warps) {
      issue(slot_in);
      slot_in = slot_in + 1 == C::STAGES ? 0 : slot_in + 1;
      cp_async_wait<C::STAGES - 1>();
      if (ok) ok = mbar_wait(&bars[slot_out], parity, &g_paged_wait_status);
      __syncwarp();
      const uint32_t base = ring_addr + slot_out * C::SLOT;
      const float2* here = scales_at + slot_out * T;
      if (++slot_out == C::STAGES) { slot_out = 0; parity ^= 1u; }
      const int key0 = (s.first_chunk + c) * KEYS;
      const bool whole = key0 + KEYS <= all_to && key0 >= all_from;
      // A page that holds nothing: log2 0 = -inf hides its keys.  NaN passes through lv to the rows that see the
      // page; its 1 / s_v is 0, so that weights of 0 stay 0 in the other rows' sums.
      float ks[T], lv[T], iv[T];
#pragma unroll
      for (int h = 0; h < T; ++h) {
        const float2 scales = here[h];
        const bool holds = scales.y >= kLeastScale;
        ks[h] = holds ? scales.x : 0.f;
        lv[h] = lg2_approx(scales.y);
        iv[h] = holds ? rcp_approx(scales.y) : 0.f;
      }

      // ---- S^T = K . Q^T: keys g, g + 8 of a tile, rows 2t, 2t + 1.  Groups, planes (and both tiles, while the
      // registers last) step through the channels together: four to eight independent accumulations hide the
      // MMA's latency ----
      constexpr int TOGETHER = NG <= 2 ? T : 1;
      float x[T][NG][4];
#pragma unroll
      for (int h0 = 0; h0 < T; h0 += TOGETHER) {
        int hi[TOGETHER][NG][4], lo[TOGETHER][NG][4];
#pragma unroll
        for (int h = 0; h < TOGETHER; ++h)
#pragma unroll
          for (int ng = 0; ng < NG; ++ng)
#pragma unroll
            for (int e = 0; e < 4; ++e) hi[h][ng][e] = lo[h][ng][e] = 0;
        uint32_t kf[TOGETHER][D / 32][4];
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int h = 0; h < TOGETHER; ++h)
            ldmatrix_x4(kf[h][w], base + (h0 + h) * C::TILE + tile_offset<D>(m_row, 2 * w + m_piece));
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) {
            uint4 q4;
            if constexpr (C::Q_REGS) q4 = qr[ng][w];
            else q4 = my_q[(ng * (D / 32) + w) * 32];
#pragma unroll
            for (int h = 0; h < TOGETHER; ++h) {
              mma_s8_16832(hi[h][ng], kf[h][w], q4.x, q4.y);
              mma_s8_16832(lo[h][ng], kf[h][w], q4.z, q4.w);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < TOGETHER; ++h)
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) {
            const float f0 = row_scale[ng][0] * ks[h0 + h], f1 = row_scale[ng][1] * ks[h0 + h];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[h0 + h][ng][e] = fmaf((float)(hi[h][ng][e] * 128 + lo[h][ng][e]), e & 1 ? f1 : f0, lv[h0 + h]);
          }
      }
      if (!whole) {
#pragma unroll
        for (int ng = 0; ng < NG; ++ng)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int place = s.place + (r_first + ng * 8 + 2 * t + e) / a.G;
            const int to = a.causal ? min(s.len, place + 1) : s.len, from = a.window >= 0 ? place - a.window + 1 : 0;
#pragma unroll
            for (int h = 0; h < T; ++h)
#pragma unroll
              for (int k8 = 0; k8 < 2; ++k8) {
                const int key = key0 + 16 * h + 8 * k8 + g;
                if (key >= to || key < from) x[h][ng][2 * k8 + e] = -INFINITY;
              }
          }
      }
      // ---- reference, weights, row sums ----
      float mx[NG][2];
      bool grown = false;
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[ng][e] = fmaxf(x[0][ng][e], x[0][ng][e + 2]);
          if constexpr (T == 2) mx[ng][e] = max3f(mx[ng][e], x[1][ng][e], x[1][ng][e + 2]);
          grown |= mx[ng][e] > m_run[ng][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = mx[ng][e];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float m = fmaxf(m_run[ng][e], top);
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
      }
      uint32_t pb[NG][T][2];
#pragma unroll
      for (int h = 0; h < T; ++h)
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[h][ng][e] = ex2_approx(x[h][ng][e] - m_run[ng][e & 1]);
          l_run[ng][0] = fmaf(x[h][ng][0] + x[h][ng][2], iv[h], l_run[ng][0]);
          l_run[ng][1] = fmaf(x[h][ng][1] + x[h][ng][3], iv[h], l_run[ng][1]);
          pb[ng][h][0] = pack2<__half>(x[h][ng][0], x[h][ng][1]);
          pb[ng][h][1] = pack2<__half>(x[h][ng][2], x[h][ng][3]);
        }
#pragma unroll
      for (int h = 0; h < T; ++h)
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) {
          pb[ng][h][0] = transpose8x8(pb[ng][h][0]);
          pb[ng][h][1] = transpose8x8(pb[ng][h][1]);
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
      for (int h = 0; h < T; ++h) {
        uint32_t r[D / 32][4];
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
          ldmatrix_x4_trans(r[w], base + h * C::TILE + 16 * D + tile_offset<D>(m_row, 2 * w + m_piece));
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t y0 = r[w][2 * half] ^ 0x80808080u, y1 = r[w][2 * half + 1] ^ 0x80808080u;
            const uint32_t va[4] = {widen(y0, 0x4240u), widen(y0, 0x4341u), widen(y1, 0x4240u), widen(y1, 0x4341u)};
#pragma unroll
            for (int ng = 0; ng < NG; ++ng) mma_f16_16816(o[ng][2 * w + half], va, pb[ng][h][0], pb[ng][h][1]);
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
    const bool complete = !CLUSTER && c_begin == 0 && cur.cend == s.chunks;
    // of a cluster's block, in the ring: every chunk has been consumed
    float* const res_o = reinterpret_cast<float*>(smem);                 // [rows_per_unit][D]
    float2* const res_ml = reinterpret_cast<float2*>(res_o + a.rows_per_unit * D);
    const int64_t part = (2ll * blockIdx.x + (c_begin == 0)) * a.rows_per_unit;
    // per row: the weight of every key warp, and the joint reference and sum (a thread per row and key warp)
    if (tid < a.rows_per_unit * key_warps) {
      const int idx = tid / key_warps, w = tid - idx * key_warps, w_row = idx / (NG * 8);
      float2* mine = ml + (w_row * key_warps + w) * NG * 8 + (idx - w_row * NG * 8);
      const float2 one = *mine;
      float m = one.x;
      for (int o2 = key_warps / 2; o2; o2 >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o2));
      const float f = ex2_approx(one.x - m);
      float l = one.y * f;
      for (int o2 = key_warps / 2; o2; o2 >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o2);
      mine->x = f;
      if (w == 0) joint[idx] = make_float2(m, l);
    }
    __syncthreads();
    // where this thread's rows go: 2 t + e of every group
    uint16_t* out_at[NG][2];
    float inv[NG][2];
    float2 both[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r_local = (rw * NG + ng) * 8 + 2 * t + e, r = row0 + r_local, i = r / a.G, head = hkv * a.G + r - i * a.G;
        both[ng][e] = joint[r_local];
        inv[ng][e] = (i < s.n && both[ng][e].y != 0.f) ? 1.f / both[ng][e].y : 0.f;
        out_at[ng][e] = r < a.rows ? reinterpret_cast<uint16_t*>(a.out) + cur.b * a.o_sb + head * a.o_sh + i * a.o_ss : nullptr;
      }
    auto put = [&](int ng, int e, int ch, float y0, float y1) {   // two channels of a row
      const int r_local = (rw * NG + ng) * 8 + 2 * t + e;
      if constexpr (CLUSTER) {
        *reinterpret_cast<float2*>(res_o + r_local * D + ch) = make_float2(y0, y1);
        if (ch == 0) res_ml[r_local] = both[ng][e];
      } else if (complete) {
        if (out_at[ng][e] != nullptr) {
          const float f = inv[ng][e];
          y0 = f == 0.f ? 0.f : y0 * f;
          y1 = f == 0.f ? 0.f : y1 * f;
          *reinterpret_cast<uint32_t*>(out_at[ng][e] + ch) = a.bf16 ? pack2<__nv_bfloat16>(y0, y1) : pack2<__half>(y0, y1);
        }
      } else {
        *reinterpret_cast<float2*>(a.part_o + (part + r_local) * D + ch) = make_float2(y0, y1);
        if (ch == 0) *reinterpret_cast<float2*>(a.part_ml + (part + r_local) * 2) = both[ng][e];
      }
    };
    // a fragment is summed and written by one warp: d % key_warps (warps without one only hand theirs over)
    auto join_groups = [&](auto key_warps_c) {
      constexpr int KW = decltype(key_warps_c)::value, OWN = (C::FRAGS + KW - 1) / KW;
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        float4* here = buf + (C::BUFS == 2 ? (ng & 1) * (C::BUF_ONE / 16) : 0) + rw * C::FRAGS * (KW - 1) * 32 + lane;
        const float f0 = ml[warp * NG * 8 + ng * 8 + 2 * t].x, f1 = ml[warp * NG * 8 + ng * 8 + 2 * t + 1].x;
        float4 own[OWN];
#pragma unroll
        for (int d = 0; d < C::FRAGS; ++d) {
          const float4 x = make_float4(o[ng][d][0] * f0, o[ng][d][1] * f1, o[ng][d][2] * f0, o[ng][d][3] * f1);
          if (d % KW == kw) own[d / KW] = x;
          else here[(d * (KW - 1) + (kw < d % KW ? kw : kw - 1)) * 32] = x;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
          const int d = k * KW + kw;
          if (d < C::FRAGS) {
            float4 x = own[k];
#pragma unroll
            for (int w = 0; w < KW - 1; ++w) {
              const float4 y = here[(d * (KW - 1) + w) * 32];
              x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) put(ng, e, 16 * d + 2 * g, e ? x.y : x.x, e ? x.w : x.z);
          }
        }
        if (C::BUFS == 1 && ng + 1 < NG) __syncthreads();
      }
    };
    if (C::ROW_WARPS == 2 && a.row_warps == 2) join_groups(std::integral_constant<int, kPaWarps / 2>{});
    else join_groups(std::integral_constant<int, kPaWarps>{});
    if constexpr (CLUSTER) {
      cluster_sync();
      const int rank = blockIdx.x % a.blocks;
      for (int idx = rank * kPaThreads + tid; idx < a.rows_per_unit * (D / 4); idx += a.blocks * kPaThreads) {
        const int r_local = idx / (D / 4), ch = idx % (D / 4) * 4, r = row0 + r_local;
        if (r >= a.rows) break;
        float m = kNegSentinel, l = 0.f;
        for (int c = 0; c < a.blocks; ++c) m = fmaxf(m, cluster_load2(res_ml + r_local, c).x);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < a.blocks; ++c) {
          const float2 one = cluster_load2(res_ml + r_local, c);
          const float f = ex2_approx(one.x - m);
          const float4 x = cluster_load4(res_o + r_local * D + ch, c);
          l = fmaf(one.y, f, l);
          sum.x = fmaf(x.x, f, sum.x); sum.y = fmaf(x.y, f, sum.y); sum.z = fmaf(x.z, f, sum.z); sum.w = fmaf(x.w, f, sum.w);
        }
        store_row(a, cur.b, hkv, r, s.n, ch, sum, l);
      }
      cluster_sync();   // a block's shared memory outlives its readers
      break;
    } else {
      if (cur.left <= 0) break;
      next_unit(cur);
      load_q(cur);
      c_begin = 0;
    }
  }
  if (!ok) {   // an expired wait: this warp's copies in flight land before its shared memory goes away
    for (int i = 0; i < C::STAGES; ++i)
      for (uint32_t ph = 0; ph < 2; ++ph) mbar_wait_quiet(&bars[i], ph, 10000000ull);
  }
}

// Behind the split kernel, with its grid: block i joins the partials of the unit that begins in range i and ends
// behind it (at most one), a warp per row, and writes the zeros of every sequence without keys or queries.
template <int D>
__global__ void __launch_bounds__(kPaThreads, 1) paged_join_kernel(const PagedArgs a) {
  __shared__ unsigned red[kPaWarps];
  __shared__ int s_last[3];
  const int units = a.Hkv * a.row_units;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Line line = line_of(a, units, red);
  const unsigned per = share_of(a, units, line.total);
  const unsigned c0 = min(line.total, per * blockIdx.x), c1 = min(line.total, c0 + per);
  if (c0 < c1) locate(a, line, units, c1 - 1, s_last);
  __syncthreads();
  for (int b = blockIdx.x; b < a.B; b += a.blocks) {
    if (seq_of(a, b).chunks > 0) continue;
    for (int64_t idx = threadIdx.x; idx < (int64_t)a.Hq * a.M * (D / 4); idx += kPaThreads) {
      const int ch = (int)(idx % (D / 4)) * 4, head = (int)(idx / (D / 4) % a.Hq), i = (int)(idx / (D / 4) / a.Hq);
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + b * a.o_sb + head * a.o_sh + i * a.o_ss + ch) = make_uint2(0, 0);
    }
  }
  // every block waits, also one with nothing to do: a grid that ended before the split kernel would let
  // the stream's next kernel start beside it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 >= c1) return;
  const int b = s_last[0], u = s_last[1];
  const Seq s = seq_of(a, b);
  const unsigned back = s_last[2];                            // chunks of the unit before c1 - 1
  if (back > c1 - 1 - c0 || (int)back == s.chunks - 1) return;   // it began in an earlier range, or ends in this one
  const unsigned i0 = blockIdx.x, i1 = (c1 - 1 - back + s.chunks - 1) / per;
  const int hkv = u / a.row_units, row0 = (u - hkv * a.row_units) * a.rows_per_unit;
  const int parts = (int)(i1 - i0 + 1);
  constexpr int PER = D >= 128 ? 4 : D / 32;                  // channels per lane and pass
  for (int r_local = warp; r_local < a.rows_per_unit && row0 + r_local < a.rows; r_local += kPaWarps) {
    const int r = row0 + r_local;
    // partial n: block i0 + n, its slot 1 where it began the unit (n = 0), else slot 0
    auto row_of = [&](int n) { return (int64_t)(2 * (i0 + n) + (n == 0)) * a.rows_per_unit + r_local; };
    float m = kNegSentinel;
    for (int n = lane; n < parts; n += 32) m = fmaxf(m, a.part_ml[row_of(n) * 2]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += 32 * PER) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll 8
      for (int n = 0; n < parts; ++n) {
        const float2 one = *reinterpret_cast<const float2*>(a.part_ml + row_of(n) * 2);
        const float* src = a.part_o + row_of(n) * D + d0 + PER * lane;
        float x[4];
        if constexpr (PER == 4) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else if constexpr (PER == 2) {
          const float2 v = *reinterpret_cast<const float2*>(src);
          x[0] = v.x; x[1] = v.y;
        } else {
          x[0] = *src;
        }
        const float f = ex2_approx(one.x - m);
        l = fmaf(one.y, f, l);
#pragma unroll
        for (int e = 0; e < PER; ++e) sum[e] = fmaf(x[e], f, sum[e]);
      }
      if constexpr (PER == 4) {
        store_row(a, b, hkv, r, s.n, d0 + 4 * lane, make_float4(sum[0], sum[1], sum[2], sum[3]), l);
      } else {
        // four channels from the neighbouring lanes
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z0 = __shfl_sync(0xffffffffu, sum[0], (4 * lane + e) / PER & 31);
          const float z1 = __shfl_sync(0xffffffffu, sum[PER - 1], (4 * lane + e) / PER & 31);
          y[e] = PER == 1 || e % 2 == 0 ? z0 : z1;
        }
        if (lane < D / 4) store_row(a, b, hkv, r, s.n, 4 * lane, make_float4(y[0], y[1], y[2], y[3]), l);
      }
    }
  }
}

// Rows that one unit of the split kernel serves: 8 per group of the MMA's N axis, groups per warp (NG), warps
// with other rows.
struct Plan {
  int ng, row_warps, row_units, rows_per_unit, chunk_shift;
  bool cluster;           // blocks = blocks per unit, else of the whole grid
  int blocks;
  size_t prefill_bytes;   // > 0: paged_prefill.cu serves the call, with this workspace
};

// Rows per (sequence, KV head) from which the tensor-memory kernel may serve a call: up to 32 the split kernel makes
// one pass with half the work per key that its estimate below counts.
constexpr int kPrefillRows = 33;

int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (1 << s)) return s;
  return -1;
}

constexpr int kJoinSteps = 4, kClusterSteps = 8;

PagedArgs args_of(const sl8_paged_cache& c, const sl8_paged_attn_params& p) {
  PagedArgs a{};
  a.q = p.q; a.q_sb = p.q_stride_b; a.q_sh = p.q_stride_h; a.q_ss = p.q_stride_s;
  a.out = p.out; a.o_sb = p.out_stride_b; a.o_sh = p.out_stride_h; a.o_ss = p.out_stride_s;
  a.k = c.k; a.v = c.v; a.ks = c.k_scale; a.vs = c.v_scale;
  a.table = c.block_table; a.table_stride = c.table_stride; a.lens = c.context_lens; a.query_lens = p.query_lens;
  a.B = p.B; a.Hq = p.Hq; a.Hkv = c.Hkv; a.M = p.M; a.G = p.Hq / c.Hkv; a.rows = p.M * a.G;
  a.page_shift = page_shift_of(c.page_size); a.num_pages = c.num_pages;
  int64_t tokens = c.num_pages > 0 ? (int64_t)c.max_pages * c.page_size : 0;
  if (p.max_context_len > 0 && p.max_context_len < tokens) tokens = p.max_context_len;
  a.max_tokens = (int)(tokens < 0x7fffff00 ? tokens : 0x7fffff00);   // tile ends stay in 32 bits
  a.causal = p.causal; a.window = p.window_left < 0x40000000 ? p.window_left : -1; a.bf16 = p.dtype == SL8_BF16;
  a.scale_log2 = p.softmax_scale * 1.4426950408889634f;
  return a;
}

Plan plan_of(const PagedArgs& a, int D, int backend) {
  Plan x{};
  x.ng = std::min(groups_of(D), (a.rows + 7) / 8);
  x.row_warps = a.rows > 8 * groups_of(D) ? 2 : 1;   // PaCfg::ROW_WARPS
  x.rows_per_unit = x.row_warps * x.ng * 8;
  x.row_units = (a.rows + x.rows_per_unit - 1) / x.rows_per_unit;
  x.chunk_shift = chunk_shift_of(D, x.ng);
  // Few units of few chunks: a cluster per unit, up to eight blocks with a chunk per warp at least, as long as
  // all clusters run at once (of eight blocks, fifteen or sixteen do, depending on which SMs a GPU has, and one too
  // many doubles the time: 16 units of 4096 keys 18 us, 12 in clusters of four; so fourteen) and the chunks per warp
  // are at most kJoinSteps more than the line would give: joining through global memory costs as much as that many
  // steps (8 heads of 128, 4096 keys: 9.9 us in clusters, 14.5 on the line).  Above kClusterSteps a ragged batch
  // would wait for its longest sequence, which the line does not.
  const int64_t units = (int64_t)a.B * a.Hkv * x.row_units, keys = 1 << x.chunk_shift;
  const int64_t longest = ((int64_t)a.max_tokens + keys - 1) / keys, key_warps = kPaWarps / x.row_warps;
  int per_unit = 1;
  while (per_unit < 8 && units * per_unit * 2 <= (per_unit == 4 ? 112 : 128) && (int64_t)per_unit * key_warps < longest) per_unit *= 2;
  const int64_t steps = (longest + per_unit * key_warps - 1) / (per_unit * key_warps);
  const int64_t line_steps = (longest * units + kNumSms * key_warps - 1) / (kNumSms * key_warps);
  const bool cluster = units * per_unit <= kNumSms && steps <= kClusterSteps && steps <= line_steps + kJoinSteps;
  if (backend == SL8_BACKEND_TCGEN05 || (backend == SL8_BACKEND_AUTO && a.rows >= kPrefillRows)) {
    // The tensor-memory kernel takes the call when its estimate is lower.  The split kernel's: 0.09, 0.17 and 0.17 ns
    // per key, KV head and pass at D = 64, 128 (64 rows a pass) and 256 (32), and 6.7, 9.5 and 8.8 us per unit that a
    // block begins, joins or leaves.  Over 439 calls (40 ... 1024 rows, 8 ... 512 units, 16 ... 16384 keys) the choice
    // costs 0.2 % over the faster kernel's time on average and 20 % at most (64 rows of 512 units of 4096 keys: 414
    // against 492 us); the two differ by up to three times either way (64 rows of 8 units of 16384 keys: 71 against
    // 197 us, 72 rows of 512 units of 16 keys: 81 against 24 us).
    const double unit_us = D <= 64 ? 6.7 : (D == 128 ? 9.5 : 8.8), begun = std::max(1.0, (double)units / kNumSms);
    const double split_us = 4.0 + (cluster ? 1.0 : begun + 1.5) * unit_us +
                            (double)units * a.max_tokens * (D <= 64 ? 0.09e-3 : 0.17e-3);
    const size_t bytes = sl8_paged_prefill_workspace(a, D);
    if (bytes > 0 && (backend == SL8_BACKEND_TCGEN05 || sl8_paged_prefill_us(a, D) < split_us)) {
      x.prefill_bytes = bytes;
      return x;
    }
  }
  if (cluster) {
    x.cluster = true;
    x.blocks = per_unit;
    return x;
  }
  const int64_t chunks = (((int64_t)a.max_tokens + (1 << x.chunk_shift) - 1) >> x.chunk_shift) * a.B * a.Hkv * x.row_units;
  x.blocks = (int)(chunks < 1 ? 1 : (chunks > kNumSms ? kNumSms : chunks));
  return x;
}

int paged_checks(const sl8_paged_cache* c, const sl8_paged_attn_params* p) {
  if (c == nullptr || p == nullptr) return SL8_ERR_NULL;
  if (c->D != 32 && c->D != 64 && c->D != 128 && c->D != 256) return SL8_ERR_BAD_HEAD_DIM;
  if (p->dtype != SL8_F16 && p->dtype != SL8_BF16) return SL8_ERR_BAD_DTYPE;
  if (c->num_pages < 0 || c->Hkv < 0 || c->max_pages < 0 || page_shift_of(c->page_size) < 0) return SL8_ERR_BAD_SHAPE;
  if (p->B < 0 || p->Hq < 0 || p->M < 0) return SL8_ERR_BAD_SHAPE;
  if (p->backend != SL8_BACKEND_AUTO && p->backend != SL8_BACKEND_MMA && p->backend != SL8_BACKEND_TCGEN05) return SL8_ERR_UNSUPPORTED;
  if (p->Hq > 0 && (c->Hkv == 0 || p->Hq % c->Hkv != 0)) return SL8_ERR_BAD_SHAPE;
  return SL8_OK;
}

template <int D, int NG, bool CLUSTER>
int allow_smem() {
  static std::atomic<bool> allowed[64];
  int dev = 0;
  SL8_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && allowed[dev].load()) return SL8_OK;
  SL8_CUDA_TRY(cudaFuncSetAttribute(paged_split_kernel<D, NG, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    PaCfg<D, NG>::smem(PaCfg<D, NG>::ROW_WARPS)));
  if (dev < 64) allowed[dev].store(true);
  return SL8_OK;
}

template <int D, int NG>
int launch_paged(const PagedArgs& a, bool cluster, cudaStream_t stream) {
  using C = PaCfg<D, NG>;
  CUtensorMap k_map{}, v_map{};   // boxes of one tile; an empty pool is never read
  if (a.max_tokens > 0) {
    const uint64_t page_heads = (uint64_t)a.num_pages * a.Hkv;
    int rc = sl8_make_tmap_3d(&k_map, a.k, 1, D, 1u << a.page_shift, page_heads, C::ROW, 16, C::ROW);
    if (rc == SL8_OK) rc = sl8_make_tmap_3d(&v_map, a.v, 1, D, 1u << a.page_shift, page_heads, C::ROW, 16, C::ROW);
    if (rc != SL8_OK) return rc;
  }
  const int smem = PaCfg<D, NG>::smem(a.row_warps);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cfg.blockDim = dim3(kPaThreads);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cluster) {
    const int rc = allow_smem<D, NG, true>();
    if (rc != SL8_OK) return rc;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)a.blocks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.row_units * a.blocks));
    cfg.dynamicSmemBytes = smem;
    SL8_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_split_kernel<D, NG, true>, k_map, v_map, a));
    return SL8_OK;
  }
  const int rc = allow_smem<D, NG, false>();
  if (rc != SL8_OK) return rc;
  paged_split_kernel<D, NG, false><<<a.blocks, kPaThreads, smem, stream>>>(k_map, v_map, a);
  if (cudaGetLastError() != cudaSuccess) return SL8_ERR_CUDA;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)a.blocks);
  SL8_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, a));
  return SL8_OK;
}

template <int D>
int launch_paged_rows(const PagedArgs& a, int ng, bool cluster, cudaStream_t stream) {
  switch (ng) {
    case 1: return launch_paged<D, 1>(a, cluster, stream);
    case 2: return launch_paged<D, 2>(a, cluster, stream);
    case 3:
      if constexpr (D == 256) return SL8_ERR_UNSUPPORTED;
      else return launch_paged<D, 3>(a, cluster, stream);
    default:
      if constexpr (D == 256) return SL8_ERR_UNSUPPORTED;
      else return launch_paged<D, 4>(a, cluster, stream);
  }
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_attn_paged_workspace(const sl8_paged_cache* c, const sl8_paged_attn_params* p) {
  if (paged_checks(c, p) != SL8_OK || (int64_t)p->B * p->Hq * p->M == 0) return 1024;
  const Plan x = plan_of(args_of(*c, *p), c->D, p->backend);
  if (x.prefill_bytes > 0) return 1024 + x.prefill_bytes;
  if (x.cluster) return 1024;
  return 1024 + (size_t)2 * x.blocks * x.rows_per_unit * (c->D + 2) * sizeof(float);
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
  if ((int64_t)p->M * (p->Hq / c->Hkv) > 0x40000000ll) return SL8_ERR_TOO_LARGE;
  PagedArgs a = args_of(*c, *p);
  const Plan x = plan_of(a, c->D, p->backend);
  // (without a key there is nothing for the tensor-memory kernel: the split one writes the zeros)
  if (p->backend == SL8_BACKEND_TCGEN05 && x.prefill_bytes == 0 && a.max_tokens > 0) return SL8_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < sl8_attn_paged_workspace(c, p)) return SL8_ERR_WORKSPACE;
  if (!aligned16(workspace)) return SL8_ERR_MISALIGNED;
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 1023) & ~uintptr_t(1023));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  a.chunk_shift = x.chunk_shift;
  if (x.prefill_bytes > 0) return sl8_paged_prefill(a, c->D, ws, x.prefill_bytes, s);
  if ((int64_t)c->num_pages * c->Hkv > 0x7fffffffll) return SL8_ERR_TOO_LARGE;
  // the line of all chunks is counted in 32 bits; its length is bounded by what can be seen
  const int64_t most = ((int64_t)a.max_tokens + 31) / 16 * p->B * c->Hkv * x.row_units;
  if ((int64_t)p->B * c->Hkv * x.row_units > 0x7fffffffll || most > 0x7fffffffll) return SL8_ERR_TOO_LARGE;
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = a.part_o + (size_t)2 * x.blocks * x.rows_per_unit * c->D;
  a.row_warps = x.row_warps; a.rows_per_unit = x.rows_per_unit; a.row_units = x.row_units; a.blocks = x.blocks;
  switch (c->D) {
    case 32: return launch_paged_rows<32>(a, x.ng, x.cluster, s);
    case 64: return launch_paged_rows<64>(a, x.ng, x.cluster, s);
    case 128: return launch_paged_rows<128>(a, x.ng, x.cluster, s);
    default: return launch_paged_rows<256>(a, x.ng, x.cluster, s);
  }
}

extern "C" int sl8_paged_status(void* stream) {
  void* word = nullptr;
  SL8_CUDA_TRY(cudaGetSymbolAddress(&word, g_paged_wait_status));
  const int rc = sl8_read_device_status(word, stream);
  const int prefill = sl8_paged_prefill_status(stream);
  return rc != SL8_OK ? rc : prefill;
}
