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

__device__ __forceinline__ double rope_position(const RopeFreq& f, int axis, int64_t b, int64_t s) {
  const int64_t at = axis * f.pos_sa + b * f.pos_sb + s * f.pos_ss;
  return f.pos64 ? (double)__ldg(reinterpret_cast<const long long*>(f.positions) + at)
                 : (double)__ldg(reinterpret_cast<const int*>(f.positions) + at);
}

// cos and sin of position * frequency.  The number of turns is formed and reduced to [-1/2, 1/2]
// in 64 bits: at position 10^6 a 32-bit product is already 0.03 rad off.  What is left is exact
// enough for fp32 (sincospif: 2 ulp).
__device__ __forceinline__ void rope_angle(double pos, float freq, float& c, float& s) {
  double turns = pos * (double)freq * 0.15915494309189533577;
  turns -= rint(turns);
  sincospif((float)(2.0 * turns), &s, &c);
}

// cos / sin of VEC consecutive frequencies from i0 on for the token (b, s).
template <int VEC>
__device__ __forceinline__ void rope_angles(const RopeFreq& f, int i0, int64_t b, int64_t s, float (&c)[VEC], float (&sn)[VEC]) {
  double pos = f.freq_axis ? 0.0 : rope_position(f, 0, b, s);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (f.freq_axis) pos = rope_position(f, min((int)__ldg(f.freq_axis + i0 + e), f.n_axes - 1), b, s);
    rope_angle(pos, __ldg(f.inv_freq + i0 + e), c[e], sn[e]);
    sn[e] *= f.sin_sign;
  }
}

// VEC elements in one aligned piece (or 16-byte pieces where they are longer).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Piece {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> piece_load(const T* p) {
  return *reinterpret_cast<const Piece<T, VEC>*>(p);
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
