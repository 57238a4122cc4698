// Attention of many query rows over the paged int8 cache (a prompt's next piece, or its whole): tensor bound.
//
// Two kernels.  The first widens the codes that a group of (sequence, KV head) units can see to dense 16-bit
// integers -- exact, |code| <= 127 -- and lists, per 16 keys (a page is a multiple of 16), the two numbers the
// scales come down to: f = s_k * softmax_scale * log2 e and lv = log2 s_v.  The second is a flash-attention
// kernel on the tensor-memory path with
//   x_n = (q . code_k) f_n + lv_n,   w_n = 2^(x_n - M),   O += w_n code_v(n),   l += w_n / s_v(n),
// so neither K's nor V's scale is ever rounded into a 16-bit operand; P = w is (2^-11 of each weight: fp16 also
// under bf16 queries, since w stays below 2^8 and V's codes are exact in either type), and the output.  f and lv are constant over 16 columns: the sweep over the logits is the
// 16-bit forward kernel's, with one multiply-add per logit.
//
// Why a dense copy: a unit's keys are read by rows / 128 blocks (32 for 1024 tokens of 4 heads per KV head),
// and widening in each of them would cost more issue slots than the softmax has to spare.  The copy (4 D bytes
// per key) is made for as many units at a time as fit kGroupBytes, which keeps most of it in L2, or as fill the
// GPU with row tiles, up to kMostBytes.
//
// Block = 128 query rows (token-major over the heads of one KV head) x 64-key tiles, six warps as in
// fwd_tcgen05.cu: four softmax warps (one row per thread), a TMA producer, an MMA issuer; two blocks per SM
// share the tensor pipe (D = 256: one).  Every wait is bounded; an expired one raises the status word that
// sl8_paged_status reads.
//
// Measured (D = 128, heads 32 : 8, fp16): 1024 query tokens at the end of 9216 keys, two sequences: copy 24.5 us,
// attention 262-269 us = 880 TFLOP/s.  The softmax warps' chain bounds it, as in the 16-bit forward, and the
// grid is 1.73 waves of resident blocks.
#include "sl8_paged.cuh"
#include "sl8_softmax.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace sl8 {
namespace {

constexpr int kTM = 128, kTN = 64;
constexpr int kSoftmaxWarps = 4, kProducerWarp = 4, kMmaWarp = 5;
constexpr int kThreads = 192;
constexpr int kScaleStages = 4;
constexpr size_t kGroupBytes = 192u << 20, kMostBytes = 2048u << 20;   // dense copies made at a time (one unit at least)

__device__ int g_paged_status;               // zero when the library is loaded

// ---- the dense copy -----------------------------------------------------------------------

struct WidenArgs {
  PagedArgs a;
  void* k;              // [units][n_pad][D] of the query type
  __half* v;            // fp16
  float2* scales;       // [units][n_pad / 16]: f, lv
  int unit0, n_pad;
};

// A block widens 64 keys of one unit; keys behind the sequence's end in the last tile become zeros with
// lv = -inf, tiles behind it are not touched (no block reads them).
template <int D, typename VT>
__global__ void __launch_bounds__(256) paged_widen_kernel(const WidenArgs w) {
  const PagedArgs& a = w.a;
  const int unit = w.unit0 + blockIdx.y, b = unit / a.Hkv, h = unit - b * a.Hkv;
  const int n0 = blockIdx.x * kTN;
  const Seq s = seq_of(a, b);
  if (n0 >= s.len || s.n == 0) return;
  if (a.window >= 0 && n0 + kTN <= s.place - a.window + 1) return;   // no query sees them
  constexpr int PER_ROW = D / 16;
#pragma unroll
  for (int it = 0; it < kTN * PER_ROW / 256 + (kTN * PER_ROW % 256 != 0); ++it) {
    const int idx = threadIdx.x + 256 * it;
    if (idx >= kTN * PER_ROW) break;
    const int i = idx / PER_ROW, j = idx - i * PER_ROW, n = n0 + i;
    int page = -1;
    if (n < s.len) page = __ldg(a.table + b * a.table_stride + (n >> a.page_shift));
    uint4 kc = make_uint4(0, 0, 0, 0), vc = kc;
    float f = 0.f, lv = -INFINITY;
    if ((unsigned)page < (unsigned)a.num_pages) {
      const int64_t ph = (int64_t)page * a.Hkv + h;
      const int64_t at = ((ph << a.page_shift) + (n & ((1 << a.page_shift) - 1))) * D + 16 * j;
      kc = *reinterpret_cast<const uint4*>(a.k + at);
      vc = *reinterpret_cast<const uint4*>(a.v + at);
      const float vs = __ldg(a.vs + ph);
      if (!(vs < kLeastScale)) {   // a page that holds nothing keeps f = 0 and lv = -inf; NaN passes
        f = __ldg(a.ks + ph) * a.scale_log2;
        lv = log2f(vs);
      }
    }
    if (i % 16 == 0 && j == 0) w.scales[((int64_t)blockIdx.y * w.n_pad + n) / 16] = make_float2(f, lv);
    auto put = [&](const uint4& p, auto* out) {
      using T = std::remove_pointer_t<decltype(out)>;
      const uint32_t c[4] = {p.x, p.y, p.z, p.w};
      uint4 o[2];
      uint32_t* y = reinterpret_cast<uint32_t*>(o);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[2 * e] = pack2<T>((float)(int8_t)c[e], (float)(int8_t)(c[e] >> 8));
        y[2 * e + 1] = pack2<T>((float)(int8_t)(c[e] >> 16), (float)(int8_t)(c[e] >> 24));
      }
      uint4* dst = reinterpret_cast<uint4*>(out + ((int64_t)blockIdx.y * w.n_pad + n) * D + 16 * j);
      dst[0] = o[0];
      dst[1] = o[1];
    };
    put(kc, reinterpret_cast<VT*>(w.k));
    put(vc, w.v);
  }
}

// ---- the sweep ----------------------------------------------------------------------------

// One pass over the 64 logits of this thread's row, as softmax_pass (sl8_softmax.cuh) with f and lv per 16
// columns (sc: four float2).  FIRST && MASK leaves the finished x in r (the second pass then takes them as
// they are); otherwise r stays as the accumulators.  mx: the largest x; sum: of w / s_v.
template <bool MASK, bool FIRST>
__device__ __forceinline__ void paged_sweep(uint32_t (&r)[kTN], const float2* sc, float neg_m, int n_block, int to, int from,
                                            uint32_t t_p, float& mx, float& sum) {
  constexpr int G = 4, NG = kTN / 2 / G;      // pairs per group, groups; two groups share a scale
  const float2 neg_m2 = make_float2(neg_m, neg_m), one2 = make_float2(1.f, 1.f);
  mx = -INFINITY;
  sum = 0.f;
  float mx0 = -INFINITY, mx1 = -INFINITY;
  float2 sum_a = make_float2(0.f, 0.f), sum_b = sum_a;
  float2 x[2][G];
  uint32_t pk[16];
  auto prep = [&](int g, float2 (&xo)[G]) {
    const float2 s = sc[g / 2];
    float2 p[G];
#pragma unroll
    for (int u = 0; u < G; ++u) p[u] = bits2(r[2 * (g * G + u)], r[2 * (g * G + u) + 1]);
    if (FIRST && MASK) {
#pragma unroll
      for (int u = 0; u < G; ++u) {
        p[u] = __ffma2_rn(p[u], make_float2(s.x, s.x), make_float2(s.y, s.y));
        const int n = n_block + 2 * (g * G + u);
        p[u].x = (n < to && n >= from) ? p[u].x : -INFINITY;
        p[u].y = (n + 1 < to && n + 1 >= from) ? p[u].y : -INFINITY;
        r[2 * (g * G + u)] = __float_as_uint(p[u].x);
        r[2 * (g * G + u) + 1] = __float_as_uint(p[u].y);
      }
    }
    if (FIRST) {
#pragma unroll
      for (int u = 0; u < G; u += 2) {
        mx0 = max3f(mx0, p[u].x, p[u].y);
        mx1 = max3f(mx1, p[u + 1].x, p[u + 1].y);
      }
      if (!MASK && (g & 1)) {   // f >= 0: the largest accumulator of the 16 gives the largest x
        mx = fmaxf(mx, fmaf(fmaxf(mx0, mx1), s.x, s.y));
        mx0 = mx1 = -INFINITY;
      }
    }
    if (MASK) {
#pragma unroll
      for (int u = 0; u < G; ++u) xo[u] = __ffma2_rn(p[u], one2, neg_m2);
    } else {
      const float c = s.y + neg_m;
#pragma unroll
      for (int u = 0; u < G; ++u) xo[u] = __ffma2_rn(p[u], make_float2(s.x, s.x), make_float2(c, c));
    }
  };
  prep(0, x[0]);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float2(&xc)[G] = x[g & 1];
#pragma unroll
    for (int u = 0; u < G; ++u) xc[u] = make_float2(ex2_issue(xc[u].x), ex2_issue(xc[u].y));
    if (g + 1 < NG) prep(g + 1, x[(g + 1) & 1]);
#pragma unroll
    for (int u = 0; u < G; u += 2) {
      sum_a = add2(sum_a, xc[u]);
      sum_b = add2(sum_b, xc[u + 1]);
    }
    if (g & 1) {
      const float2 st = add2(sum_a, sum_b);
      const float lv = sc[g / 2].y;
      // lv = NaN: rows that see the keys have NaN weights, the others' zeros stay zeros
      sum = fmaf(st.x + st.y, lv > -INFINITY ? ex2_approx(-lv) : 0.f, sum);
      sum_a = sum_b = make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < G; ++u) pk[(g * G + u) & 15] = pack2<__half>(xc[u].x, xc[u].y);
    if (((g + 1) * G) % 16 == 0) tc_st16(t_p + 16 * (((g + 1) * G) / 16 - 1), pk);
  }
  if (FIRST && MASK) mx = fmaxf(mx0, mx1);
}

// ---- attention ----------------------------------------------------------------------------

template <int D>
struct Cfg {
  static constexpr int SUBS = D / 64;                     // sub-tiles of 64 channels (128 bytes a row)
  static constexpr int Q_SUB = kTM * 128, KV_SUB = kTN * 128;
  static constexpr int Q_TILE = SUBS * Q_SUB, KV_TILE = SUBS * KV_SUB;
  static constexpr int OFF_Q = 0, OFF_K = Q_TILE, OFF_V = OFF_K + 2 * KV_TILE;
  static constexpr int OFF_SC = OFF_V + 2 * KV_TILE;      // kScaleStages x 4 float2
  static constexpr int OFF_BAR = OFF_SC + kScaleStages * 32;
  static constexpr int NEED = OFF_BAR + 512 + 1024;
  static constexpr int SMEM = NEED < 78 * 1024 ? 78 * 1024 : NEED;   // at most two blocks per SM: TMEM_COLS each
  static constexpr uint32_t TMEM_COLS = D <= 128 ? 256 : 512;
  static constexpr uint32_t COL_S = 0, COL_O = 128;
};

enum Bar { O_DONE = 0, PV_DONE, S_FULL = PV_DONE + 2, P_FULL = S_FULL + 2, K_FULL = P_FULL + 2, V_FULL = K_FULL + 2,
           SC_EMPTY = V_FULL + 2, NUM_BARS = SC_EMPTY + kScaleStages };

struct PrefillArgs {
  PagedArgs a;
  const float2* scales;
  int unit0, n_pad;
};

template <int D, typename VT>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) paged_prefill_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                                    const __grid_constant__ CUtensorMap v_map,
                                                                                    const __grid_constant__ PrefillArgs w) {
  using C = Cfg<D>;
  const PagedArgs& a = w.a;
  int* status = &g_paged_status;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float2* sc_smem = reinterpret_cast<float2*>(smem + C::OFF_SC);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NUM_BARS);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = w.unit0 + blockIdx.y, b = unit / a.Hkv, hkv = unit - b * a.Hkv;
  const Seq s = seq_of(a, b);
  // long rows first: a causal tile's keys end with its last row
  const int r0 = (gridDim.x - 1 - blockIdx.x) * kTM, r1 = min(a.rows, r0 + kTM);
  const int i_first = r0 / a.G, i_last = min(s.n, (r1 - 1) / a.G + 1) - 1;     // query tokens of the tile
  const int n_end = a.causal ? max(0, min(s.len, s.place + i_last + 1)) : s.len;
  const int n_begin = a.window >= 0 ? (int)(max((int64_t)0, (int64_t)s.place + i_first - a.window + 1) / kTN * kTN) : 0;
  const int ntiles = (i_first < s.n && n_end > n_begin) ? (n_end - n_begin + kTN - 1) / kTN : 0;
  auto out_row = [&](int r) {
    const int i = r / a.G;
    return reinterpret_cast<VT*>(a.out) + b * a.o_sb + (int64_t)(hkv * a.G + r - i * a.G) * a.o_sh + i * a.o_ss;
  };
  if (ntiles == 0) {
    for (int idx = threadIdx.x; idx < (r1 - r0) * (D / 8); idx += kThreads)
      *reinterpret_cast<uint4*>(out_row(r0 + idx / (D / 8)) + idx % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(&bars[O_DONE], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[PV_DONE + i], 1);
      mbar_init(&bars[S_FULL + i], 2);             // the MMA commit and the tile's scales
      mbar_init(&bars[P_FULL + i], kSoftmaxWarps);
      mbar_init(&bars[K_FULL + i], 1);
      mbar_init(&bars[V_FULL + i], 1);
    }
    for (int i = 0; i < kScaleStages; ++i) mbar_init(&bars[SC_EMPTY + i], kSoftmaxWarps);
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    tc_alloc(tmem_slot, C::TMEM_COLS);
    tc_relinquish();
    tc_fence_before();
  }
  // Q: any strides, so plain loads into the swizzled layout of a TMA tile; rows without a query are zeros
  for (int idx = threadIdx.x; idx < kTM * (D / 8); idx += kThreads) {
    const int row = idx / (D / 8), c = idx % (D / 8), r = r0 + row, i = r / a.G;
    uint4 p = make_uint4(0, 0, 0, 0);
    if (r < r1 && i < s.n)
      p = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const VT*>(a.q) + b * a.q_sb + (int64_t)(hkv * a.G + r - i * a.G) * a.q_sh +
                                               i * a.q_ss + 8 * c));
    *reinterpret_cast<uint4*>(smem + C::OFF_Q + (c >> 3) * C::Q_SUB + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = p;
  }
  fence_proxy_async_smem();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  bool ok = true;

  if (warp == kProducerWarp) {
    // ======================= producer: K two tiles ahead, V, the scales through registers =======================
    const float2* sc_row = w.scales + (int64_t)blockIdx.y * (w.n_pad / 16);
    if (lane == 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
    auto load_k = [&](int t) -> bool {   // lane 0 only
      const int ks = t & 1;
      if (t >= 2 && !mbar_wait(&bars[S_FULL + ks], ((t >> 1) - 1) & 1, status)) return false;
      mbar_expect_tx(&bars[K_FULL + ks], C::KV_TILE);
#pragma unroll
      for (int c = 0; c < C::SUBS; ++c)
        tma_load_3d(smem + C::OFF_K + ks * C::KV_TILE + c * C::KV_SUB, &k_map, &bars[K_FULL + ks], 64 * c, n_begin + t * kTN, blockIdx.y);
      return true;
    };
    if (lane == 0) {
      ok = load_k(0);
      if (ok && ntiles > 1) ok = load_k(1);
    }
    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    auto fetch = [&](int t) { return (lane < 4 && t < ntiles) ? __ldg(sc_row + (n_begin + t * kTN) / 16 + lane) : make_float2(0.f, 0.f); };
    float2 s0 = fetch(0), s1 = fetch(1), s2 = fetch(2);
    for (int j = 0; j < ntiles && ok; ++j) {
      const int ss = j % kScaleStages;
      if (j >= kScaleStages) ok = mbar_wait(&bars[SC_EMPTY + ss], ((j / kScaleStages) - 1) & 1, status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane < 4) sc_smem[ss * 4 + lane] = s0;
      s0 = s1;
      s1 = s2;
      s2 = fetch(j + 3);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[S_FULL + (j & 1)]);
        if (j + 2 < ntiles) ok = load_k(j + 2);
        if (ok && j >= 2) ok = mbar_wait(&bars[PV_DONE + (j & 1)], ((j >> 1) - 1) & 1, status);
        if (ok) {
          mbar_expect_tx(&bars[V_FULL + (j & 1)], C::KV_TILE);
#pragma unroll
          for (int c = 0; c < C::SUBS; ++c)
            tma_load_3d(smem + C::OFF_V + (j & 1) * C::KV_TILE + c * C::KV_SUB, &v_map, &bars[V_FULL + (j & 1)], 64 * c, n_begin + j * kTN,
                        blockIdx.y);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    }
  } else if (warp == kMmaWarp) {
    // ======================= issuer: QK_0, QK_1, then P.V_j, QK_{j+2} =======================
    constexpr uint32_t fmt = std::is_same<VT, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc_qk = umma_idesc(1, fmt, fmt, 0, 0, kTM, kTN);
    const uint32_t idesc_pv = umma_idesc(1, 0, 0, 0, 1, kTM, D);   // P and V are fp16
    const uint64_t dq = umma_smem_desc(smem_u32(smem + C::OFF_Q), 16, 1024, kUmmaSw128);
    const uint64_t dk = umma_smem_desc(smem_u32(smem + C::OFF_K), 16, 1024, kUmmaSw128);
    const uint64_t dv = umma_smem_desc(smem_u32(smem + C::OFF_V), C::KV_SUB, 1024, kUmmaSw128);
    auto issue_qk = [&](int t, int buf) -> bool {
      if (!__all_sync(0xffffffffu, mbar_wait(&bars[K_FULL + buf], (t >> 1) & 1, status))) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t sub = k / 4, within = 32 * (k % 4);
          tc_mma_f16_ss(tmem + C::COL_S + kTN * buf, umma_desc_advance(dq, sub * C::Q_SUB + within),
                        umma_desc_advance(dk, buf * C::KV_TILE + sub * C::KV_SUB + within), idesc_qk, k > 0 ? 1u : 0u);
        }
        tc_commit(&bars[S_FULL + buf]);
      }
      __syncwarp();
      return true;
    };
    ok = issue_qk(0, 0);
    if (ok && ntiles > 1) ok = issue_qk(1, 1);
    for (int j = 0; j < ntiles && ok; ++j) {
      const int u = j & 1;
      const uint32_t par = (j >> 1) & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars[P_FULL + u], par, status));
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars[V_FULL + u], par, status));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kTN / 16; ++k)
          tc_mma_f16_ts(tmem + C::COL_O, tmem + C::COL_S + kTN * u + 8 * k, umma_desc_advance(dv, u * C::KV_TILE + k * 2048), idesc_pv,
                        (j > 0 || k > 0) ? 1u : 0u);
        tc_commit(&bars[PV_DONE + u]);
      }
      __syncwarp();
      if (j + 2 < ntiles) ok = issue_qk(j + 2, u);
      if (j == ntiles - 1 && elect_one()) tc_commit(&bars[O_DONE]);
      __syncwarp();
    }
  } else {
    // ======================= softmax: thread = query row =======================
    const int row = 32 * warp + lane, r = r0 + row;
    const int place = s.place + r / a.G;
    const int to = a.causal ? min(s.len, place + 1) : s.len;
    const int from = a.window >= 0 ? (int)max((int64_t)0, (int64_t)place - a.window + 1) : 0;
    // keys that every row of the tile sees
    const int all_to = a.causal ? min(s.len, s.place + i_first + 1) : s.len;
    const int all_from = a.window >= 0 ? (int)max((int64_t)0, (int64_t)s.place + (r1 - 1) / a.G - a.window + 1) : 0;
    const uint32_t t_row = tmem + ((uint32_t)(32 * warp) << 16);
    const uint32_t t_o = t_row + C::COL_O;
    float m_run = -INFINITY, l_run = 0.f;
    uint32_t acc[kTN];     // live across the loop's back edge: the next tile's logits are loaded early
    bool loaded = false;
    for (int j = 0; j < ntiles; ++j) {
      const int n_block = n_begin + j * kTN, ss = j % kScaleStages;
      const uint32_t t_s = t_row + C::COL_S + kTN * (j & 1);
      if (!loaded) {
        ok = mbar_wait(&bars[S_FULL + (j & 1)], (j >> 1) & 1, status);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) tc_ld32(t_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&acc[32 * c]));
      }
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 2; ++c) tc_regs_ready(*reinterpret_cast<uint32_t(*)[32]>(&acc[32 * c]));
      float2 sc[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 p = *reinterpret_cast<const float4*>(sc_smem + ss * 4 + 2 * i);
        sc[2 * i] = make_float2(p.x, p.y);
        sc[2 * i + 1] = make_float2(p.z, p.w);
      }
      const bool masked = n_block + kTN > all_to || n_block < all_from;
      float mx, psum;
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      if (masked) paged_sweep<true, true>(acc, sc, neg_m, n_block, to, from, t_s, mx, psum);
      else paged_sweep<false, true>(acc, sc, neg_m, n_block, to, from, t_s, mx, psum);
      const bool grow = m_run == -INFINITY ? mx > -INFINITY : mx > m_run + kLazyRescaleLog2;
      float resc = 1.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = fmaxf(m_run, mx);
        resc = exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
        m_run = m_new;
        if (j > 0) {   // O *= resc once the previous P.V has landed
          ok = mbar_wait(&bars[PV_DONE + ((j - 1) & 1)], ((j - 1) >> 1) & 1, status);
          if (!ok) break;
          tc_fence_after();
          const float2 resc2 = make_float2(resc, resc);
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tc_ld32(t_o + 32 * c, o);
            tc_wait_ld();
            tc_regs_ready(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 t = mul2(bits2(o[2 * i], o[2 * i + 1]), resc2);
              o[2 * i] = __float_as_uint(t.x);
              o[2 * i + 1] = __float_as_uint(t.y);
            }
            tc_st32(t_o + 32 * c, o);
          }
        }
        tc_wait_st();   // the speculative P is done before P is stored again
        float unused;
        const float again = m_run == -INFINITY ? 0.f : -m_run;
        if (masked) paged_sweep<true, false>(acc, sc, again, n_block, to, from, t_s, unused, psum);
        else paged_sweep<false, false>(acc, sc, again, n_block, to, from, t_s, unused, psum);
      }
      l_run = l_run * resc + psum;
      loaded = false;
      if (j + 1 < ntiles && __all_sync(0xffffffffu, mbar_test(&bars[S_FULL + ((j + 1) & 1)], ((j + 1) >> 1) & 1))) {
        tc_fence_after();
        const uint32_t t_n = t_row + C::COL_S + kTN * ((j + 1) & 1);
#pragma unroll
        for (int c = 0; c < 2; ++c) tc_ld32(t_n + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&acc[32 * c]));
        loaded = true;
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[P_FULL + (j & 1)]);
        mbar_arrive(&bars[SC_EMPTY + ss]);
      }
    }
    if (ok) ok = mbar_wait(&bars[O_DONE], 0, status);
    if (ok) {
      tc_fence_after();
      const float inv = (r < r1 && r / a.G < s.n && l_run != 0.f) ? 1.f / l_run : 0.f;
      VT* dst = out_row(min(r, r1 - 1));
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tc_ld32(t_o + 32 * c, o);
        tc_wait_ld();
        tc_regs_ready(o);
        if (r < r1) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = inv == 0.f ? 0.f : __uint_as_float(o[8 * v + e]) * inv;
            *reinterpret_cast<uint4*>(dst + 32 * c + 8 * v) =
                make_uint4(pack2<VT>(y[0], y[1]), pack2<VT>(y[2], y[3]), pack2<VT>(y[4], y[5]), pack2<VT>(y[6], y[7]));
          }
        }
      }
    }
    tc_fence_before();
  }
  // every role arrives here, on success and behind an expired wait
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tc_dealloc(tmem, C::TMEM_COLS);
  }
}

// Blocks that run at once.
int slots_of(int D) { return D <= 128 ? 2 * kNumSms : kNumSms; }

// Keys a dense copy is laid out for, and units copied at a time.
struct Group {
  int n_pad;
  int64_t units;
  size_t unit_bytes, scale_bytes;   // per unit: one of K / V, and the scales
};

Group group_of(const PagedArgs& a, int D) {
  Group g;
  g.n_pad = (int)(((int64_t)a.max_tokens + kTN - 1) / kTN * kTN);
  g.unit_bytes = (size_t)g.n_pad * D * 2;
  g.scale_bytes = (size_t)g.n_pad / 16 * sizeof(float2);
  const int64_t all = (int64_t)a.B * a.Hkv, tiles = (a.rows + kTM - 1) / kTM;
  const size_t both = std::max<size_t>(2 * g.unit_bytes, 1);
  const int64_t wanted = std::min<int64_t>((slots_of(D) + tiles - 1) / tiles, kMostBytes / both);
  g.units = std::max<int64_t>(1, std::min(std::min(all, std::max<int64_t>(kGroupBytes / both, wanted)), (int64_t)65535));
  return g;
}

size_t align1k(size_t x) { return (x + 1023) / 1024 * 1024; }

template <int D, typename VT>
int launch_prefill(const PagedArgs& a, uint8_t* ws, cudaStream_t stream) {
  using C = Cfg<D>;
  const Group g = group_of(a, D);
  uint8_t* k = ws;
  uint8_t* v = k + align1k(g.units * g.unit_bytes);
  float2* scales = reinterpret_cast<float2*>(v + align1k(g.units * g.unit_bytes));
  static std::atomic<bool> allowed[64];
  int dev = 0;
  SL8_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !allowed[dev].load()) {
    SL8_CUDA_TRY(cudaFuncSetAttribute(paged_prefill_kernel<D, VT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    if (dev < 64) allowed[dev].store(true);
  }
  CUtensorMap k_map, v_map;
  int rc = sl8_make_tmap_3d(&k_map, k, 2, D, g.n_pad, g.units, 64, kTN, 128);
  if (rc == SL8_OK) rc = sl8_make_tmap_3d(&v_map, v, 2, D, g.n_pad, g.units, 64, kTN, 128);
  if (rc != SL8_OK) return rc;
  const int64_t all = (int64_t)a.B * a.Hkv;
  for (int64_t u0 = 0; u0 < all; u0 += g.units) {
    const unsigned units = (unsigned)std::min(g.units, all - u0);
    const WidenArgs wa{a, k, reinterpret_cast<__half*>(v), scales, (int)u0, g.n_pad};
    paged_widen_kernel<D, VT><<<dim3(g.n_pad / kTN, units), 256, 0, stream>>>(wa);
    const PrefillArgs pa{a, scales, (int)u0, g.n_pad};
    paged_prefill_kernel<D, VT><<<dim3((a.rows + kTM - 1) / kTM, units), kThreads, C::SMEM, stream>>>(k_map, v_map, pa);
    if (cudaGetLastError() != cudaSuccess) return SL8_ERR_CUDA;
  }
  return SL8_OK;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

size_t sl8_paged_prefill_workspace(const PagedArgs& a, int D) {
  if (D != 64 && D != 128 && D != 256) return 0;
  if (a.scale_log2 < 0.f || a.max_tokens <= 0) return 0;   // the sweep takes a group's maximum before it is scaled
  const Group g = group_of(a, D);
  return 2 * align1k(g.units * g.unit_bytes) + align1k(g.units * g.scale_bytes);
}

// Estimated time: every wave of blocks walks the longest context (0.67, 0.83 and 1.2 us per 64-key tile at
// D = 64, 128 and 256, two blocks per SM except at 256) behind 4 us of set-up, and the copy moves 6 D bytes per key,
// Q and the result 4 D per row, at 6 TB/s.
double sl8_paged_prefill_us(const PagedArgs& a, int D) {
  const Group g = group_of(a, D);
  const int64_t all = (int64_t)a.B * a.Hkv, tiles = (a.rows + kTM - 1) / kTM;
  const int64_t waves = (all / g.units) * ((g.units * tiles + slots_of(D) - 1) / slots_of(D)) +
                        (all % g.units * tiles + slots_of(D) - 1) / slots_of(D);
  const double tile_us = D == 64 ? 0.67 : (D == 128 ? 0.83 : 1.2);
  return (D == 256 ? 9.0 : 5.0) + (double)waves * ((double)g.n_pad / kTN * tile_us + 4.0) + (double)all * g.n_pad * 6 * D / 6e6 +
         (double)all * a.rows * 4 * D / 6e6;
}

int sl8_paged_prefill(const PagedArgs& a, int D, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (workspace == nullptr || workspace_bytes < sl8_paged_prefill_workspace(a, D)) return SL8_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  switch (D) {
    case 64: return a.bf16 ? launch_prefill<64, __nv_bfloat16>(a, ws, stream) : launch_prefill<64, __half>(a, ws, stream);
    case 128: return a.bf16 ? launch_prefill<128, __nv_bfloat16>(a, ws, stream) : launch_prefill<128, __half>(a, ws, stream);
    case 256: return a.bf16 ? launch_prefill<256, __nv_bfloat16>(a, ws, stream) : launch_prefill<256, __half>(a, ws, stream);
  }
  return SL8_ERR_UNSUPPORTED;
}

int sl8_paged_prefill_status(void* stream) {
  void* word = nullptr;
  SL8_CUDA_TRY(cudaGetSymbolAddress(&word, g_paged_status));
  return sl8_read_device_status(word, stream);
}
