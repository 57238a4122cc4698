// Rotary position arithmetic shared by the standalone rotation (rope.cu) and by the append to the
// paged cache (paged_kv.cu).
//
// Channel pair i of a row (i < rot / 2) is turned by t = pos[axis(i)] * inv_freq[i]:
//   y_a = a cos t - b sin t,  y_b = b cos t + a sin t,
// with (a, b) = (x[i], x[i + rot/2]) or, interleaved, (x[2i], x[2i + 1]).  Channels from rot on stay.
#pragma once
#include "sl8_common.cuh"

namespace sl8 {

struct RopeFreq {
  const void* positions;      // int32 or int64, indexed by the strides below
  int64_t pos_sa, pos_sb, pos_ss;
  const float* inv_freq;      // [rot / 2]
  const uint8_t* freq_axis;   // [rot / 2] or null (axis 0)
  int pos64, n_axes, half;    // half = rot / 2
  float sin_sign;             // multiplies the sines; -1: the inverse rotation (the gradient)
};

// Angles in fixed point.  A frequency is held as its turns per position modulo one, in units of 2^-64
// (formed once per block in 64-bit floating point); position * frequency modulo 2^64 is then the fraction
// of a turn for ANY 64-bit position -- the wrap-around is the reduction.  A 32-bit floating product would be
// 0.03 rad off at position 10^6; this one is off by the rounding of the frequency alone, 2^-53 of the turns.
__device__ __forceinline__ unsigned long long rope_turns(float inv_freq) {
  double t = (double)inv_freq * 0.15915494309189533577;   // 1 / (2 pi)
  t -= floor(t);
  return (unsigned long long)(t * 18446744073709551616.0);
}
// The block's table of frequencies; the caller synchronises.
__device__ __forceinline__ void rope_table(unsigned long long* table, const RopeFreq& f) {
  for (int i = threadIdx.x; i < f.half; i += blockDim.x) table[i] = rope_turns(__ldg(f.inv_freq + i));
}

__device__ __forceinline__ long long rope_position(const RopeFreq& f, int axis, int64_t b, int64_t s) {
  const int64_t at = axis * f.pos_sa + b * f.pos_sb + s * f.pos_ss;
  return f.pos64 ? __ldg(reinterpret_cast<const long long*>(f.positions) + at)
                 : (long long)__ldg(reinterpret_cast<const int*>(f.positions) + at);
}

// cos and sin of position * frequency for two frequencies: the quarter turn comes off the top bits, the rest is an
// angle in [-pi/4, pi/4] and two Taylor series (the first terms left out are 2e-9 and 2.5e-8 there), on the packed
// fp32 pipe.
__device__ __forceinline__ void rope_angle2(long long pos0, unsigned long long turns0, long long pos1, unsigned long long turns1,
                                            float2& c, float2& s) {
  const uint32_t u0 = (uint32_t)(((unsigned long long)pos0 * turns0) >> 32) + 0x20000000u;
  const uint32_t u1 = (uint32_t)(((unsigned long long)pos1 * turns1) >> 32) + 0x20000000u;
  auto all = [](float v) { return make_float2(v, v); };
  const float2 x = __fmul2_rn(make_float2((float)((int)(u0 & 0x3fffffffu) - 0x20000000), (float)((int)(u1 & 0x3fffffffu) - 0x20000000)),
                              all(1.5707963267948966f * 0x1p-30f));
  const float2 x2 = __fmul2_rn(x, x);
  float2 sn = __ffma2_rn(x2, all(2.7557319e-6f), all(-1.9841270e-4f));      // 1/9!, -1/7!
  sn = __ffma2_rn(sn, x2, all(8.3333333e-3f));                               // 1/5!
  sn = __ffma2_rn(sn, x2, all(-1.6666667e-1f));                              // -1/3!
  sn = __ffma2_rn(__fmul2_rn(sn, x2), x, x);
  float2 cs = __ffma2_rn(x2, all(2.4801587e-5f), all(-1.3888889e-3f));      // 1/8!, -1/6!
  cs = __ffma2_rn(cs, x2, all(4.1666667e-2f));                               // 1/4!
  cs = __ffma2_rn(cs, x2, all(-0.5f));
  cs = __ffma2_rn(cs, x2, all(1.f));
  // by quarters: (cos, sin) -> (-sin, cos) -> (-cos, -sin) -> (sin, -cos)
  auto turn = [](uint32_t u, float cv, float sv, float& co, float& so) {
    const bool odd = (u >> 30) & 1;
    co = __uint_as_float(__float_as_uint(odd ? sv : cv) ^ ((u + 0x40000000u) & 0x80000000u));
    so = __uint_as_float(__float_as_uint(odd ? cv : sv) ^ (u & 0x80000000u));
  };
  turn(u0, cs.x, sn.x, c.x, s.x);
  turn(u1, cs.y, sn.y, c.y, s.y);
}

// cos / sin of VEC consecutive frequencies from i0 on for the token (b, s).
template <int VEC>
__device__ __forceinline__ void rope_angles(const RopeFreq& f, const unsigned long long* table, int i0, int64_t b, int64_t s,
                                            float (&c)[VEC], float (&sn)[VEC]) {
  long long pos[VEC];
  pos[0] = f.freq_axis ? 0 : rope_position(f, 0, b, s);
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    pos[e] = f.freq_axis ? rope_position(f, min((int)__ldg(f.freq_axis + i0 + e), f.n_axes - 1), b, s) : pos[0];
#pragma unroll
  for (int e = 0; e < VEC; e += 2) {
    const int e1 = VEC == 1 ? 0 : e + 1;
    float2 cc, ss;
    rope_angle2(pos[e], table[i0 + e], pos[e1], table[i0 + e1], cc, ss);
    c[e] = cc.x;
    c[e1] = VEC == 1 ? cc.x : cc.y;
    sn[e] = ss.x * f.sin_sign;
    sn[e1] = (VEC == 1 ? ss.x : ss.y) * f.sin_sign;
  }
}

// VEC elements in one aligned piece (or 16-byte pieces where they are longer), held as packed words.
template <typename T, int VEC>
struct Piece {
  static constexpr int BYTES = sizeof(T) * VEC;
  struct alignas(BYTES > 16 ? 16 : (BYTES < 4 ? 4 : BYTES)) Bits {
    uint32_t w[BYTES >= 4 ? BYTES / 4 : 1];
  };
  Bits bits;

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (BYTES == 2) bits.w[0] = *reinterpret_cast<const uint16_t*>(p);
    else bits = *reinterpret_cast<const Bits*>(p);
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (BYTES == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)bits.w[0];
    else *reinterpret_cast<Bits*>(p) = bits;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < (BYTES >= 4 ? BYTES / 4 : 1); ++e) bits.w[e] = 0;
  }
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = __uint_as_float(bits.w[e]);
    } else if constexpr (VEC == 1) {
      x[0] = unpack2<T>(bits.w[0]).x;
    } else {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        const float2 y = unpack2<T>(bits.w[e]);
        x[2 * e] = y.x;
        x[2 * e + 1] = y.y;
      }
    }
  }
  __device__ __forceinline__ void put(const float (&x)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) bits.w[e] = __float_as_uint(x[e]);
    } else if constexpr (VEC == 1) {
      bits.w[0] = pack2<T>(x[0], 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) bits.w[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    }
  }
};

template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> piece_load(const T* p) {
  Piece<T, VEC> x;
  x.load(p);
  return x;
}

// Turns the two pieces of one item.  Half layout: a[e] pairs with b[e].  Interleaved: the pieces are
// consecutive channels and (a[0], a[1]), (a[2], a[3]) ... (b[0], b[1]) ... are the pairs.  Two elements per
// instruction on the packed fp32 pipe.
template <int VEC>
__device__ __forceinline__ void rope_turn(float (&a)[VEC], float (&b)[VEC], const float (&c)[VEC], const float (&s)[VEC],
                                          bool interleaved) {
  if constexpr (VEC == 1) {
    const float x = a[0], y = b[0];
    a[0] = x * c[0] - y * s[0];
    b[0] = y * c[0] + x * s[0];
  } else if (!interleaved) {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const float2 x = make_float2(a[e], a[e + 1]), y = make_float2(b[e], b[e + 1]);
      const float2 cc = make_float2(c[e], c[e + 1]), ss = make_float2(s[e], s[e + 1]);
      const float2 u = __ffma2_rn(x, cc, __fmul2_rn(y, make_float2(-ss.x, -ss.y))), w = __ffma2_rn(y, cc, __fmul2_rn(x, ss));
      a[e] = u.x; a[e + 1] = u.y;
      b[e] = w.x; b[e + 1] = w.y;
    }
  } else {
    auto one = [](float& x, float& y, float cv, float sv) {   // (x, y) -> (x c - y s, y c + x s)
      const float2 r = __ffma2_rn(make_float2(x, y), make_float2(cv, cv), __fmul2_rn(make_float2(y, x), make_float2(-sv, sv)));
      x = r.x;
      y = r.y;
    };
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      one(a[2 * e], a[2 * e + 1], c[e], s[e]);
      one(b[2 * e], b[2 * e + 1], c[VEC / 2 + e], s[VEC / 2 + e]);
    }
  }
}

// First channels of the two pieces of item j of a row (VEC channels each; items 0 .. D / (2 VEC) - 1).
template <int VEC>
__device__ __forceinline__ int2 rope_item(int j, int half, bool interleaved) {
  if (j * VEC < half && !interleaved) return make_int2(j * VEC, half + j * VEC);
  return make_int2(2 * j * VEC, 2 * j * VEC + VEC);
}

}  // namespace sl8
