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
  float sin_sign;             // -1: the inverse rotation (the gradient)
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

// cos and sin of position * frequency: the quarter turn comes off the top bits, the rest is an angle in
// [-pi/4, pi/4] and two Taylor series (the first terms left out are 2e-9 and 2.5e-8 there).
__device__ __forceinline__ void rope_angle(long long pos, unsigned long long turns, float& c, float& s) {
  const uint32_t u = (uint32_t)(((unsigned long long)pos * turns) >> 32) + 0x20000000u;
  const int quarter = u >> 30;
  const float x = (float)((int)(u & 0x3fffffffu) - 0x20000000) * (1.5707963267948966f * 0x1p-30f);
  const float x2 = x * x;
  float sn = fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);      // 1/9!, -1/7!
  sn = fmaf(sn, x2, 8.3333333e-3f);                         // 1/5!
  sn = fmaf(sn, x2, -1.6666667e-1f);                        // -1/3!
  sn = fmaf(sn * x2, x, x);
  float cs = fmaf(x2, 2.4801587e-5f, -1.3888889e-3f);      // 1/8!, -1/6!
  cs = fmaf(cs, x2, 4.1666667e-2f);                         // 1/4!
  cs = fmaf(cs, x2, -0.5f);
  cs = fmaf(cs, x2, 1.f);
  c = quarter & 1 ? sn : cs;
  s = quarter & 1 ? cs : sn;
  if (quarter == 1 || quarter == 2) c = -c;
  if (quarter >= 2) s = -s;
}

// cos / sin of VEC consecutive frequencies from i0 on for the token (b, s).
template <int VEC>
__device__ __forceinline__ void rope_angles(const RopeFreq& f, const unsigned long long* table, int i0, int64_t b, int64_t s,
                                            float (&c)[VEC], float (&sn)[VEC]) {
  long long pos = f.freq_axis ? 0 : rope_position(f, 0, b, s);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (f.freq_axis) pos = rope_position(f, min((int)__ldg(f.freq_axis + i0 + e), f.n_axes - 1), b, s);
    rope_angle(pos, table[i0 + e], c[e], sn[e]);
    sn[e] *= f.sin_sign;
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
// consecutive channels and (a[0], a[1]), (a[2], a[3]) ... (b[0], b[1]) ... are the pairs.
template <int VEC>
__device__ __forceinline__ void rope_turn(float (&a)[VEC], float (&b)[VEC], const float (&c)[VEC], const float (&s)[VEC],
                                          bool interleaved) {
  if (!interleaved) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x = a[e], y = b[e];
      a[e] = x * c[e] - y * s[e];
      b[e] = y * c[e] + x * s[e];
    }
    return;
  }
  if constexpr (VEC == 1) {
    const float x = a[0], y = b[0];
    a[0] = x * c[0] - y * s[0];
    b[0] = y * c[0] + x * s[0];
  } else {
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      const float x = a[2 * e], y = a[2 * e + 1], u = b[2 * e], w = b[2 * e + 1];
      a[2 * e] = x * c[e] - y * s[e];
      a[2 * e + 1] = y * c[e] + x * s[e];
      b[2 * e] = u * c[VEC / 2 + e] - w * s[VEC / 2 + e];
      b[2 * e + 1] = w * c[VEC / 2 + e] + u * s[VEC / 2 + e];
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
