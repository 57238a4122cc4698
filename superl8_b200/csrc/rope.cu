// Rotary positions with one or several axes on q and k (one launch for both), and the gradient,
// which is the rotation by the opposite angle.
//
// HBM bound: every element is read once and written once, 2 e bytes.  A thread owns one item -- 2 VEC
// channels of one token that pair with one another -- works out its VEC angles once and walks the
// heads with them, so the angles (fixed-point products and two short series, sl8_rope.cuh) are shared by
// all heads of a block's group and the loads of four heads are in flight together.
//
// Measured: 4 x 8192 tokens of 72 heads of 128 in fp16, 189 us = 6.4 TB/s (what a plain copy reaches is 6.5);
// with the angles from the math library's sine and cosine it was 283 us, bound by their instructions.
#include "sl8_rope.cuh"

namespace sl8 {
namespace {

struct RopeTensor {
  const void* x;
  void* y;
  int64_t x_sb, x_sh, x_ss, y_sb, y_sh, y_ss;
};

struct RopeArgs {
  RopeTensor q, k;
  RopeFreq f;
  uint32_t tokens;   // B * S
  int S, Hq, H, items, heads_per_block, interleaved;   // H = Hq + Hkv
};

constexpr int kRopeThreads = 256;

// U heads in flight per thread; four blocks per SM where an item's pieces leave the registers for it.
template <typename T, int VEC>
struct RopeCfg {
  static constexpr int BYTES = sizeof(T) * VEC;
  static constexpr int U = BYTES > 16 ? 2 : 4;
  static constexpr int BLOCKS = BYTES > 16 ? 2 : 3;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kRopeThreads, RopeCfg<T, VEC>::BLOCKS) rope_kernel(const RopeArgs a) {
  constexpr int U = RopeCfg<T, VEC>::U;
  extern __shared__ unsigned long long table[];
  const uint32_t item = blockIdx.x * kRopeThreads + threadIdx.x;   // the host keeps them below 2^32
  const uint32_t token = item / (uint32_t)a.items;
  const bool real = token < a.tokens;
  const int j = (int)(item - token * a.items);
  const int64_t b = token / (uint32_t)a.S, s = token - b * a.S;
  const bool turn = j * VEC < a.f.half;
  const bool interleaved = a.interleaved != 0;
  const int2 at = rope_item<VEC>(j, a.f.half, interleaved);
  const int h0 = blockIdx.y * a.heads_per_block, h1 = min(a.H, h0 + a.heads_per_block);

  rope_table(table, a.f);
  __syncthreads();
  if (!real) return;
  float c[VEC], sn[VEC];
  if (turn) rope_angles<VEC>(a.f, table, j * VEC, b, s, c, sn);

  auto heads = [&](const RopeTensor& t, int from, int to) {
    const T* x = reinterpret_cast<const T*>(t.x) + b * t.x_sb + s * t.x_ss + from * t.x_sh;
    T* y = reinterpret_cast<T*>(t.y) + b * t.y_sb + s * t.y_ss + from * t.y_sh;
    auto one = [&](Piece<T, VEC>& p0, Piece<T, VEC>& p1, T* dst) {
      if (turn) {
        float u[VEC], w[VEC];
        p0.get(u);
        p1.get(w);
        rope_turn<VEC>(u, w, c, sn, interleaved);
        p0.put(u);
        p1.put(w);
      }
      p0.store(dst + at.x);
      p1.store(dst + at.y);
    };
    int n = to - from;
    for (; n >= U; n -= U) {
      Piece<T, VEC> p0[U], p1[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        p0[i] = piece_load<T, VEC>(x + i * t.x_sh + at.x);
        p1[i] = piece_load<T, VEC>(x + i * t.x_sh + at.y);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) one(p0[i], p1[i], y + i * t.y_sh);
      x += U * t.x_sh;
      y += U * t.y_sh;
    }
    for (; n > 0; --n) {
      Piece<T, VEC> p0 = piece_load<T, VEC>(x + at.x), p1 = piece_load<T, VEC>(x + at.y);
      one(p0, p1, y);
      x += t.x_sh;
      y += t.y_sh;
    }
  };
  if (h0 < a.Hq) heads(a.q, h0, min(h1, a.Hq));
  if (h1 > a.Hq) heads(a.k, max(h0, a.Hq) - a.Hq, h1 - a.Hq);
}

template <typename T, int VEC>
int launch_rope(RopeArgs a, int D, cudaStream_t stream) {
  a.items = D / (2 * VEC);
  const int64_t gx = ((int64_t)a.tokens * a.items + kRopeThreads - 1) / kRopeThreads;
  if (gx * kRopeThreads > 0xffffffffll) return SL8_ERR_TOO_LARGE;
  // A block's heads share the angles (as much work as four heads' products): at least four of them, unless
  // that leaves SMs idle, and few enough for six waves of blocks.
  int64_t groups = (kNumSms * 18 + gx - 1) / gx, most = (a.H + 3) / 4;
  if (gx * most < kNumSms * 3) most = a.H;
  if (groups > most) groups = most;
  a.heads_per_block = (int)((a.H + groups - 1) / groups);
  const unsigned gy = (unsigned)((a.H + a.heads_per_block - 1) / a.heads_per_block);
  if (gy > 65535u) return SL8_ERR_TOO_LARGE;
  rope_kernel<T, VEC><<<dim3((unsigned)gx, gy), kRopeThreads, a.f.half * 8, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SL8_OK : SL8_ERR_CUDA;
}

template <typename T>
int launch_rope_vec(const RopeArgs& a, int D, int vec, cudaStream_t stream) {
  switch (vec) {
    case 8: return launch_rope<T, 8>(a, D, stream);
    case 4: return launch_rope<T, 4>(a, D, stream);
    case 2: return launch_rope<T, 2>(a, D, stream);
    default: return launch_rope<T, 1>(a, D, stream);
  }
}

// Largest piece (elements) that keeps every row's pieces whole and aligned.
int piece_size(const sl8_rope_params& p, int elem) {
  for (int vec = 8; vec > 1; vec /= 2) {
    const int64_t bytes = (int64_t)vec * elem > 16 ? 16 : (int64_t)vec * elem;
    bool ok = (p.rot / 2) % vec == 0 && p.D % (2 * vec) == 0;
    auto fits = [&](const void* x, int64_t sb, int64_t sh, int64_t ss) {
      return x == nullptr || (reinterpret_cast<uintptr_t>(x) % bytes == 0 && sb * elem % bytes == 0 && sh * elem % bytes == 0 &&
                              ss * elem % bytes == 0);
    };
    ok = ok && fits(p.q, p.q_stride_b, p.q_stride_h, p.q_stride_s) && fits(p.q_out, p.q_out_stride_b, p.q_out_stride_h, p.q_out_stride_s) &&
         fits(p.k, p.k_stride_b, p.k_stride_h, p.k_stride_s) && fits(p.k_out, p.k_out_stride_b, p.k_out_stride_h, p.k_out_stride_s);
    if (ok) return vec;
  }
  return 1;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" int sl8_rope(const sl8_rope_params* p, void* stream) {
  if (p == nullptr) return SL8_ERR_NULL;
  if (p->B < 0 || p->Hq < 0 || p->Hkv < 0 || p->S < 0 || p->n_axes < 1) return SL8_ERR_BAD_SHAPE;
  if (p->D < 2 || p->D > 8192 || p->D % 2 != 0 || p->rot < 0 || p->rot > p->D || p->rot % 2 != 0) return SL8_ERR_BAD_SHAPE;
  if (p->dtype != SL8_F16 && p->dtype != SL8_BF16 && p->dtype != SL8_F32) return SL8_ERR_BAD_DTYPE;
  const int Hq = p->q ? p->Hq : 0, Hkv = p->k ? p->Hkv : 0;
  if ((int64_t)p->B * p->S * (Hq + Hkv) == 0) return SL8_OK;
  if ((Hq && !p->q_out) || (Hkv && !p->k_out) || !p->positions || (p->rot > 0 && !p->inv_freq)) return SL8_ERR_NULL;
  const int elem = p->dtype == SL8_F32 ? 4 : 2;
  RopeArgs a{};
  a.q = RopeTensor{p->q, p->q_out, p->q_stride_b, p->q_stride_h, p->q_stride_s, p->q_out_stride_b, p->q_out_stride_h, p->q_out_stride_s};
  a.k = RopeTensor{p->k, p->k_out, p->k_stride_b, p->k_stride_h, p->k_stride_s, p->k_out_stride_b, p->k_out_stride_h, p->k_out_stride_s};
  a.f = RopeFreq{p->positions, p->pos_stride_axis, p->pos_stride_b, p->pos_stride_s, p->inv_freq, p->n_axes > 1 ? p->freq_axis : nullptr,
                 p->pos_is_64 != 0, p->n_axes, p->rot / 2, p->inverse ? -1.f : 1.f};
  if ((int64_t)p->B * p->S > 0xffffffffll) return SL8_ERR_TOO_LARGE;
  a.tokens = (uint32_t)((int64_t)p->B * p->S);
  a.S = p->S; a.Hq = Hq; a.H = Hq + Hkv; a.interleaved = p->interleaved;
  const int vec = piece_size(*p, elem);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case SL8_F16: return launch_rope_vec<__half>(a, p->D, vec, s);
    case SL8_BF16: return launch_rope_vec<__nv_bfloat16>(a, p->D, vec, s);
    default: return launch_rope_vec<float>(a, p->D, vec, s);
  }
}
