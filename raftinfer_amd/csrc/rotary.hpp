// Rotary positions: the angles of a row, and the norm and rotation of a head that
// lies across lanes in 16-byte pieces.
#pragma once

#include "common.hpp"

namespace raftinfer::amd {

// cos and sin of position * frequency, times magnitude: the product and its reduction
// to one turn in 64 bits (in 32, angles of far positions would be off by whole radians),
// then a 32-bit sincos of the reduced angle.
__device__ __forceinline__ void rotary_cos_sin(std::uint32_t position, double frequency, float magnitude, float &cs, float &sn) {
  const double theta = static_cast<double>(position) * frequency;
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  const double t = theta - kTwoPi * rint(theta / kTwoPi);
  sincosf(static_cast<float>(t), &sn, &cs);
  cs *= magnitude;
  sn *= magnitude;
}

// 16 bytes of a type as floats and back (one rounding, to nearest even).
template <typename T> struct Piece16;
template <> struct Piece16<bf16_bits> {
  static constexpr int kValues = 8;
  static __device__ __forceinline__ void unpack(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = bf16_lo(w[e]);
      x[2 * e + 1] = bf16_hi(w[e]);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[8]) {
    return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  }
};
template <> struct Piece16<_Float16> {
  static constexpr int kValues = 8;
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void unpack(u32x4 w, float (&x)[8]) {
    const vec v = __builtin_bit_cast(vec, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(v[e]);
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[8]) {
    vec v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<_Float16>(x[e]);
    return __builtin_bit_cast(u32x4, v);
  }
};
template <> struct Piece16<float> {
  static constexpr int kValues = 4;
  static __device__ __forceinline__ void unpack(u32x4 w, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(w[e]);
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[4]) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
};

// Sum over groups of LANES neighbouring lanes.
template <int LANES> __device__ __forceinline__ float lanes_sum(float x) {
  if constexpr (LANES >= 2) x += dpp<kDppXor1>(x);
  if constexpr (LANES >= 4) x += dpp<kDppXor2>(x);
  if constexpr (LANES >= 8) x += dpp<kDppHalfMirror>(x);
  if constexpr (LANES >= 16) x += dpp<kDppMirror>(x);
  if constexpr (LANES >= 32) x = sum_xor16(x);
  if constexpr (LANES >= 64) x = sum_xor32(x);
  return x;
}

// 1 / sqrt(sum * share + epsilon), off by one step of 32 bits.  (The instruction takes values below 2^-126 for 0: a
// small mean that no epsilon holds up is scaled by 2^96 first.)
__device__ __forceinline__ float inverse_rms(float sum, float share, float epsilon) {
  const float x = fmaf(sum, share, epsilon);
  if (epsilon >= 0x1p-96f) return __builtin_amdgcn_rsqf(x); // (uniform)
  const bool small = x < 0x1p-96f;
  return __builtin_amdgcn_rsqf(small ? x * 0x1p96f : x) * (small ? 0x1p48f : 1.0f);
}

// A head lies in LANES neighbouring lanes, N values in each, in order; lane c has values
// N c .. (0 behind head_dim).  rot: cos of the pairs, then sin.  Halves: pairs a multiple of
// N, the partner values are pairs / N lanes away.  Every lane of the wave must call it.
template <int N, int LANES>
__device__ __forceinline__ void norm_rotate(float (&x)[N], const float (&w)[N], bool norm, bool interleaved, int c, std::uint32_t pairs,
                                            float head_dim, const float *rot, float epsilon) {
  if (norm) { // (uniform)
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) ss = fmaf(x[e], x[e], ss);
    const float scale = inverse_rms(lanes_sum<LANES>(ss), 1.0f / head_dim, epsilon);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = x[e] * scale * w[e];
  }
  if (pairs == 0) return; // (uniform)
  const std::uint32_t d0 = N * c;
  if (interleaved) {
    if (d0 >= 2 * pairs) return;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float cs = rot[(d0 + e) / 2], sn = rot[pairs + (d0 + e) / 2];
      const float a = x[e], b = x[e + 1];
      x[e] = a * cs - b * sn;
      x[e + 1] = a * sn + b * cs;
    }
    return;
  }
  const bool first = d0 < pairs;
  const int away = static_cast<int>(pairs / N), from = (threadIdx.x & 63) + (first ? away : -away);
  float other[N];
#pragma unroll
  for (int e = 0; e < N; ++e) other[e] = __shfl(x[e], from);
  if (d0 >= 2 * pairs) return;
  const std::uint32_t p = first ? d0 : d0 - pairs;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float cs = rot[p + e], sn = rot[pairs + p + e];
    x[e] = first ? x[e] * cs - other[e] * sn : other[e] * sn + x[e] * cs;
  }
}

} // namespace raftinfer::amd
