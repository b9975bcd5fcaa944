// Device pieces and launch interfaces of the compact KV cache (8-bit blocks,
// sliding window with sinks, key weights, eviction).
#pragma once

#include "decode_scan.hpp"

namespace raftinfer::amd {

constexpr int kCompactBlock = 32;   // positions per scale, and keys per tile
constexpr int kCompactMaxGroup = 16; // query heads per KV head

// What the kernels read of one call.  Strides and planes in elements.
struct CompactArgs {
  const bf16_bits *query, *key, *value, *gate;
  bf16_bits *output;
  unsigned char *cache;
  std::size_t cache_stride;      // bytes between sequences
  const std::uint32_t *lengths;  // or null: past + tokens
  float *weights;
  std::uint32_t tokens, sequences, kv_heads, group, max_ctx, past, window, sinks, observed;
  bool head_major;
  bool store_inside; // prefill of bf16: the attention kernel stores the rows, and reads the new ones from key / value
};

// One KV head of one sequence's cache.
template <bool Fp8> struct CompactHead {
  using T = std::conditional_t<Fp8, unsigned char, bf16_bits>;
  T *k, *v;             // row 0
  float *ks, *vs;       // scales (Fp8)
  std::size_t row;      // elements between positions
  __device__ __forceinline__ CompactHead(unsigned char *cache, std::uint32_t kvh, std::uint32_t kv_heads,
                                         std::uint32_t max_ctx, bool head_major) {
    const std::size_t plane = static_cast<std::size_t>(max_ctx) * kv_heads * kHeadDim;
    row = head_major ? kHeadDim : static_cast<std::size_t>(kv_heads) * kHeadDim;
    k = reinterpret_cast<T *>(cache) + static_cast<std::size_t>(kvh) * (head_major ? max_ctx : 1u) * kHeadDim;
    v = k + plane;
    const std::size_t blocks = (max_ctx + kCompactBlock - 1) / kCompactBlock;
    ks = reinterpret_cast<float *>(cache + 2 * plane) + kvh * blocks;
    vs = ks + kv_heads * blocks;
  }
};

// The 32-key tiles that a range of query positions first .. last sees (some of
// whose keys may be masked): those of the sinks, then those from the first
// token's window to the last token.
struct SeenTiles {
  std::uint32_t sink_tiles, second, total;
  __host__ __device__ __forceinline__ SeenTiles(std::uint32_t first, std::uint32_t last, std::uint32_t window,
                                                std::uint32_t sinks) {
    const std::uint32_t all = last / kCompactBlock + 1;
    const std::uint32_t lo = window != 0 && first >= window ? first - window + 1 : 0;
    if (lo <= sinks) { // nothing lies between the sinks and the window
      sink_tiles = 0;
      second = 0;
    } else {
      sink_tiles = (sinks + kCompactBlock - 1) / kCompactBlock;
      second = lo / kCompactBlock < sink_tiles ? sink_tiles : lo / kCompactBlock;
    }
    total = sink_tiles + all - second;
  }
  __host__ __device__ __forceinline__ std::uint32_t tile(std::uint32_t i) const {
    return i < sink_tiles ? i : second + (i - sink_tiles);
  }
};

// Whether a token at position p sees key j.
__host__ __device__ __forceinline__ bool compact_sees(std::uint32_t j, std::uint32_t p, std::uint32_t window,
                                                      std::uint32_t sinks) {
  return (j <= p) & ((window == 0) | (j < sinks) | (p - j < window)); // (no branches)
}

// ------------------------------------------------------- e4m3 and scales
// The scale that values of at most amax (finite, >= 0) need: the smallest power
// of two s with amax <= 448 s = 1.75 * 2^8 s, and a normal number.
__device__ __forceinline__ float compact_scale(float amax) {
  const std::uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<std::uint32_t>(e < 1 ? 1 : e) << 23);
}
// 1 / s for such a scale (exact: the exponents are 1 .. 247).
__device__ __forceinline__ float compact_inverse(float s) {
  return __uint_as_float((254u << 23) - (__float_as_uint(s) & 0x7F800000u));
}
// Under the largest scale, 2^120, codes end at 240: the next one, 256, would stand for 2^128,
// which neither f32 nor bf16 holds.  (Finite values reach 255 / 128 2^127.)
constexpr float kCompactTopScale = 0x1p120f;
__device__ __forceinline__ float compact_below_top(float x) {
  constexpr float kMost = 240 * kCompactTopScale;
  return x > kMost ? kMost : x < -kMost ? -kMost : x; // (NaN stays)
}
// Four values, already divided by their scale, as e4m3 codes (nearest even).
__device__ __forceinline__ std::uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<std::uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}
// Eight codes times a scale as bf16 (exact: 4 significant bits; but for what lies below 2^-126).
__device__ __forceinline__ u32x4 fp8x8_to_bf16(std::uint32_t lo, std::uint32_t hi, float scale = 1.0f) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const pair b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const pair c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const pair d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return u32x4{__builtin_bit_cast(std::uint32_t, a), __builtin_bit_cast(std::uint32_t, b),
               __builtin_bit_cast(std::uint32_t, c), __builtin_bit_cast(std::uint32_t, d)};
}
// Four codes as f32.
__device__ __forceinline__ floatx4 fp8x4_to_f32(std::uint32_t w) {
  typedef float pair __attribute__((ext_vector_type(2)));
  const pair a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const pair b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return floatx4{a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ bool is_finite_f32(float x) {
  return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
}

// ------------------------------------------------- operands out of LDS
__device__ __forceinline__ bf16x8 lds_operand(unsigned addr) {
  return __builtin_bit_cast(bf16x8, *(const __attribute__((address_space(3))) u32x4 *)(std::uintptr_t)(addr));
}
// Transposed: of 16 lanes, lane r supplies 8 bytes of row r / 4 (bf16) and receives its
// element of 4 rows, or of row r / 2 (codes) and receives its code of 8 rows.
__device__ __forceinline__ u32x2 lds_tr_operand(unsigned addr) {
  typedef short quad __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) quad *)(std::uintptr_t)(addr)));
}
__device__ __forceinline__ u32x2 lds_tr8_operand(unsigned addr) {
  typedef int pair __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) pair *)(std::uintptr_t)(addr)));
}

// ---------------------------------------------------------- launches
void compact_append(const CompactArgs &a, bool fp8, hipStream_t stream);

std::size_t compact_decode_workspace(const CompactArgs &a);
void compact_decode(const CompactArgs &a, bool fp8, void *workspace, hipStream_t stream);

std::size_t compact_prefill_workspace(const CompactArgs &a);
void compact_prefill(CompactArgs a, bool fp8, void *workspace, hipStream_t stream);

struct CompactEvictArgs {
  const unsigned char *cache;
  const float *weights;
  unsigned char *out_cache;
  float *out_weights;
  std::int32_t *kept;
  std::uint32_t kv_heads, context, max_ctx, keep, out_max_ctx, sinks, recent;
  bool head_major;
};
std::size_t compact_evict_workspace(const CompactEvictArgs &a);
void compact_evict(const CompactEvictArgs &a, bool fp8, bool out_fp8, void *workspace, hipStream_t stream);

// Takes (reads and clears) the count of decode sequences with a bad length.
std::uint32_t compact_take_capacity_errors();

} // namespace raftinfer::amd
