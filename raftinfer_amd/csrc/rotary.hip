// Rotary positions of heads (include/raftinfer_amd/qwen35_paged_cache.hpp,
// qwen35_rotary and qwen35_rotary_frequencies).
#include "call_checks.hpp"
#include "rotary.hpp"
#include "raftinfer_amd/qwen35_paged_cache.hpp"

#include <algorithm>
#include <cmath>

namespace raftinfer::kernels {
namespace {

using namespace raftinfer::amd;
using Err = Qwen35PrimitiveError;

constexpr int kRotaryThreads = 256;

struct RotaryArgs {
  const void *input, *weight;
  void *output;
  const std::uint32_t *positions;
  const double *frequencies;
  std::size_t in_row, in_head, out_row, out_head;
  std::uint32_t rows, heads, head_dim, pairs;
  std::uint32_t group_rows; // rows of a workgroup
  bool interleaved;
  float magnitude, epsilon;
};

// cos and sin of the workgroup's rows: [row][cos of the pairs, sin].
__device__ __forceinline__ void fill_rotation(const RotaryArgs &a, std::uint32_t row0, std::uint32_t rows, float *rot) {
  for (std::uint32_t i = threadIdx.x; i < rows * a.pairs; i += kRotaryThreads) {
    const std::uint32_t r = i / a.pairs, p = i - r * a.pairs;
    float cs, sn;
    rotary_cos_sin(a.positions[row0 + r], a.frequencies[p], a.magnitude, cs, sn);
    rot[2 * a.pairs * r + p] = cs;
    rot[2 * a.pairs * r + a.pairs + p] = sn;
  }
}

// Heads in 16-byte pieces, LANES lanes each, four heads of a lane's group asked for before
// the first is used; the first four before the angles are formed.  Every lane's loads come
// before its stores, and a head's lanes run together: the output may be the input.  Memory bounds long calls (6001 rows of
// 16 heads of 256 in bf16 18.7 us, 5.3 TB/s), the launch and the angles' 64-bit reduction short ones (one row 4.4 us).
template <typename T, typename Wt, int LANES>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float rot[];
  constexpr int N = Piece16<T>::kValues, kGroups = kRotaryThreads / LANES, kBatch = 4;
  const std::uint32_t row0 = blockIdx.x * a.group_rows;
  const std::uint32_t rows = a.rows - row0 < a.group_rows ? a.rows - row0 : a.group_rows;
  const std::uint32_t units = rows * a.heads;
  const int c = threadIdx.x % LANES;
  const bool there = static_cast<std::uint32_t>(N * c) < a.head_dim;
  const std::uint32_t u0 = threadIdx.x / LANES;
  u32x4 raw[kBatch];
  const auto load = [&](std::uint32_t first) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t u = first + kGroups * b;
      raw[b] = u32x4{};
      if (u >= units || !there) continue;
      const std::uint32_t r = u / a.heads, h = u - r * a.heads;
      raw[b] = *reinterpret_cast<const u32x4 *>(static_cast<const T *>(a.input) + (row0 + r) * a.in_row + h * a.in_head + N * c);
    }
  };
  load(u0);
  float w[N];
#pragma unroll
  for (int e = 0; e < N; ++e) w[e] = a.weight != nullptr && there ? Elem<Wt>::load(static_cast<const Wt *>(a.weight), N * c + e) : 0.f;
  fill_rotation(a, row0, rows, rot);
  __syncthreads();
  // (every wave makes the same number of turns: the heads' sums and partners go over lanes)
  for (std::uint32_t first = u0; first - u0 < units; first += kGroups * kBatch) {
    if (first != u0) load(first);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t u = first + kGroups * b, in = u < units ? u : units - 1;
      const std::uint32_t r = in / a.heads, h = in - r * a.heads;
      float x[N];
      Piece16<T>::unpack(raw[b], x);
      norm_rotate<N, LANES>(x, w, a.weight != nullptr, a.interleaved, c, a.pairs, static_cast<float>(a.head_dim), rot + 2 * a.pairs * r, a.epsilon);
      if (u < units && there)
        *reinterpret_cast<u32x4 *>(static_cast<T *>(a.output) + (row0 + r) * a.out_row + h * a.out_head + N * c) = Piece16<T>::pack(x);
    }
  }
}

// Any head_dim, stride and alignment: a wave takes one head at a time, lane l the pairs and
// the other dims l, l + 64, ..; a pair's two values are loaded before either is stored.
template <typename T, typename Wt>
__global__ __launch_bounds__(kRotaryThreads) void rotary_any_kernel(RotaryArgs a) {
  extern __shared__ float rot[];
  const std::uint32_t row = blockIdx.x;
  fill_rotation(a, row, 1, rot);
  __syncthreads();
  const std::uint32_t lane = threadIdx.x & 63;
  const auto *weight = static_cast<const Wt *>(a.weight);
  for (std::uint32_t h = threadIdx.x >> 6; h < a.heads; h += kRotaryThreads / 64) {
    const T *src = static_cast<const T *>(a.input) + row * a.in_row + h * a.in_head;
    T *dst = static_cast<T *>(a.output) + row * a.out_row + h * a.out_head;
    float scale = 1.0f;
    if (weight != nullptr) {
      float ss = 0.f;
      for (std::uint32_t d = lane; d < a.head_dim; d += 64) {
        const float x = Elem<T>::load(src, d);
        ss = fmaf(x, x, ss);
      }
      scale = 1.0f / sqrtf(wave_sum(ss) / static_cast<float>(a.head_dim) + a.epsilon);
    }
    const auto value = [&](std::uint32_t d) {
      const float x = Elem<T>::load(src, d);
      return weight != nullptr ? x * scale * Elem<Wt>::load(weight, d) : x;
    };
    for (std::uint32_t p = lane; p < a.pairs; p += 64) {
      const std::uint32_t i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.pairs;
      const float x = value(i), y = value(j), cs = rot[p], sn = rot[a.pairs + p];
      Elem<T>::store(dst, i, x * cs - y * sn);
      Elem<T>::store(dst, j, x * sn + y * cs);
    }
    for (std::uint32_t d = 2 * a.pairs + lane; d < a.head_dim; d += 64) {
      const float x = value(d);
      Elem<T>::store(dst, d, x);
    }
  }
}

std::size_t or_dense(std::size_t stride, std::size_t dense) { return stride != 0 ? stride : dense; }

template <typename T, typename Wt> void launch(RotaryArgs a, bool wide, hipStream_t stream) {
  const std::size_t row_lds = 2 * a.pairs * sizeof(float);
  if (!wide) {
    a.group_rows = 1;
    rotary_any_kernel<T, Wt><<<a.rows, kRotaryThreads, row_lds, stream>>>(a);
    return;
  }
  constexpr int N = Piece16<T>::kValues;
  const std::uint32_t pieces = (a.head_dim + N - 1) / N;
  const auto go = [&]<int LANES>() {
    // a turn of four heads a lane for every workgroup, at most 8 rows
    const std::uint32_t turn = 4 * kRotaryThreads / LANES;
    a.group_rows = std::clamp<std::uint32_t>(turn / a.heads, 1, 8);
    rotary_kernel<T, Wt, LANES><<<(a.rows + a.group_rows - 1) / a.group_rows, kRotaryThreads, a.group_rows * row_lds, stream>>>(a);
  };
  if (pieces <= 8) go.template operator()<8>();
  else if (pieces <= 16) go.template operator()<16>();
  else if (pieces <= 32) go.template operator()<32>();
  else go.template operator()<64>();
}

} // namespace

float qwen35_rotary_frequencies(double *frequencies, std::size_t rotary_dim, double base, Qwen35RotaryScaling scaling,
                                double factor, double trained, double fast, double slow) {
  require<Err>(frequencies != nullptr, "rotary frequencies pointer is null");
  require<Err>(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= 16384, "rotary_dim must be even, 2 to 16384");
  require<Err>(std::isfinite(base) && base > 1.0, "rotary base must be finite and above 1");
  require<Err>(scaling == Qwen35RotaryScaling::none || scaling == Qwen35RotaryScaling::linear ||
                   scaling == Qwen35RotaryScaling::by_pair || scaling == Qwen35RotaryScaling::by_turns,
               "unsupported rotary scaling");
  const bool blend = scaling == Qwen35RotaryScaling::by_pair || scaling == Qwen35RotaryScaling::by_turns;
  require<Err>(scaling == Qwen35RotaryScaling::none || (std::isfinite(factor) && factor >= 1.0),
               "rotary factor must be finite and at least 1");
  require<Err>(!blend || (std::isfinite(trained) && trained > 0.0), "rotary trained_tokens must be finite and positive");
  require<Err>(!blend || (std::isfinite(fast) && std::isfinite(slow) && slow > 0.0 && fast > slow),
               "rotary turns must be finite, 0 < slow_turns < fast_turns");
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  const double dim = static_cast<double>(rotary_dim);
  const auto pair_of = [&](double turns) { return dim * std::log(trained / (kTwoPi * turns)) / (2.0 * std::log(base)); };
  double low = 0.0, high = 0.0;
  if (scaling == Qwen35RotaryScaling::by_pair) {
    low = std::max(0.0, std::floor(pair_of(fast)));
    high = std::min(dim - 1.0, std::ceil(pair_of(slow)));
  }
  for (std::size_t p = 0; p < rotary_dim / 2; ++p) {
    const double f = std::pow(base, -2.0 * static_cast<double>(p) / dim);
    double kept = 1.0;
    if (scaling == Qwen35RotaryScaling::linear) kept = 0.0;
    if (scaling == Qwen35RotaryScaling::by_pair)
      kept = 1.0 - std::clamp((static_cast<double>(p) - low) / std::max(high - low, 1e-3), 0.0, 1.0);
    if (scaling == Qwen35RotaryScaling::by_turns) kept = std::clamp((trained * f / kTwoPi - slow) / (fast - slow), 0.0, 1.0);
    frequencies[p] = scaling == Qwen35RotaryScaling::none ? f : f * kept + f / factor * (1.0 - kept);
  }
  return scaling == Qwen35RotaryScaling::by_pair ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
}

void qwen35_rotary(const void *input, const void *weight, void *output, const std::uint32_t *positions,
                   const double *frequencies, Qwen35RotaryShape s, float epsilon, RaftInferDataType dtype,
                   RaftInferDataType wdt, hipStream_t stream) {
  require<Err>(input != nullptr, "rotary input pointer is null");
  require<Err>(output != nullptr, "rotary output pointer is null");
  require<Err>(positions != nullptr, "rotary positions pointer is null");
  require<Err>(frequencies != nullptr, "rotary frequencies pointer is null");
  require<Err>(stream != nullptr, "HIP stream is null");
  require<Err>(dtype == RAFTINFER_DTYPE_F32 || dtype == RAFTINFER_DTYPE_F16 || dtype == RAFTINFER_DTYPE_BF16,
               "unsupported Qwen3.5 primitive dtype");
  require<Err>(weight == nullptr || wdt == dtype || wdt == RAFTINFER_DTYPE_F32,
               "rotary weight dtype must be the activations' or f32");
  require<Err>(s.rows > 0 && s.rows <= 0x7FFFFFu, "rotary rows must be 1 to 2^23 - 1");
  require<Err>(s.heads > 0 && s.heads <= 65535, "rotary heads must be 1 to 65535");
  require<Err>(s.head_dim > 0 && s.head_dim <= 16384, "rotary head_dim must be 1 to 16384");
  require<Err>(s.rotary_dim > 0 && s.rotary_dim % 2 == 0 && s.rotary_dim <= s.head_dim,
               "rotary_dim must be even, 2 to head_dim");
  require<Err>(std::isfinite(s.magnitude), "rotary magnitude must be finite");
  require<Err>(std::isfinite(epsilon) && epsilon >= 0.0f, "rotary epsilon must be finite and non-negative");
  const std::size_t size = dtype == RAFTINFER_DTYPE_F32 ? 4 : 2, wsize = wdt == RAFTINFER_DTYPE_F32 ? 4 : 2;
  RotaryArgs a{};
  a.in_head = or_dense(s.input_head_stride, s.head_dim);
  a.in_row = or_dense(s.input_row_stride, s.heads * s.head_dim);
  a.out_head = or_dense(s.output_head_stride, s.head_dim);
  a.out_row = or_dense(s.output_row_stride, s.heads * s.head_dim);
  const auto extent = [&](std::size_t row, std::size_t head) { // elements
    const char *overflow = "rotary shape overflow";
    return checked_add<Err>(checked_add<Err>(checked_mul<Err>(s.rows - 1, row, overflow), checked_mul<Err>(s.heads - 1, head, overflow), overflow),
                            s.head_dim, overflow);
  };
  const std::size_t in_bytes = checked_mul<Err>(extent(a.in_row, a.in_head), size, "rotary shape overflow");
  const std::size_t out_bytes = checked_mul<Err>(extent(a.out_row, a.out_head), size, "rotary shape overflow");
  require<Err>(strides_apart(s.rows, a.out_row, s.heads, a.out_head, s.head_dim), "rotary output rows or heads overlap");
  require<Err>(((reinterpret_cast<std::uintptr_t>(input) | reinterpret_cast<std::uintptr_t>(output)) & (size - 1)) == 0 &&
                   (reinterpret_cast<std::uintptr_t>(weight) & (wsize - 1)) == 0 &&
                   (reinterpret_cast<std::uintptr_t>(positions) & 3) == 0 && (reinterpret_cast<std::uintptr_t>(frequencies) & 7) == 0,
               "rotary pointers must be aligned to their elements");
  const bool in_place = input == output && a.in_row == a.out_row && a.in_head == a.out_head;
  const Bytes in{input, in_place ? 0 : in_bytes}, w{weight, weight != nullptr ? s.head_dim * wsize : 0};
  validate_apart<Err>({{output, out_bytes}}, {in, w, {positions, 4 * s.rows}, {frequencies, 4 * s.rotary_dim}},
                      "rotary output overlaps other arguments");
  a.input = input;
  a.weight = weight;
  a.output = output;
  a.positions = positions;
  a.frequencies = frequencies;
  a.rows = static_cast<std::uint32_t>(s.rows);
  a.heads = static_cast<std::uint32_t>(s.heads);
  a.head_dim = static_cast<std::uint32_t>(s.head_dim);
  a.pairs = static_cast<std::uint32_t>(s.rotary_dim / 2);
  a.interleaved = s.interleaved;
  a.magnitude = s.magnitude;
  a.epsilon = epsilon;
  // 16-byte pieces: all of a head's rows must begin at one, no pair may lie across two halves'
  // pieces, and a wave must hold a head
  const std::size_t n = 16 / size;
  const bool wide = aligned16(input) && aligned16(output) && s.head_dim % n == 0 && s.head_dim <= 64 * n &&
                    a.in_row % n == 0 && a.in_head % n == 0 && a.out_row % n == 0 && a.out_head % n == 0 &&
                    (s.interleaved ? s.rotary_dim : s.rotary_dim / 2) % n == 0;
  const StreamDevice<Err> device(stream, "rotary");
  const auto go = [&]<typename T>() {
    if (weight != nullptr && wdt == RAFTINFER_DTYPE_F32) launch<T, float>(a, wide, stream);
    else launch<T, T>(a, wide, stream);
  };
  if (dtype == RAFTINFER_DTYPE_F32) go.operator()<float>();
  else if (dtype == RAFTINFER_DTYPE_F16) go.operator()<_Float16>();
  else go.operator()<bf16_bits>();
  check_launch<Err>("qwen35_rotary");
}

} // namespace raftinfer::kernels
