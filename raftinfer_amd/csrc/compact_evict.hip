// Eviction from the compact KV cache: which entries stay, and their rows in order.
#include "compact_cache.hpp"

namespace raftinfer::amd {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;

// Weights as unsigned numbers in the same order: -0 is 0, NaN above everything.
__device__ __forceinline__ std::uint32_t rank_of(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const std::uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix sum over the workgroup's threads; total: the sum of all.
__device__ std::uint32_t block_prefix(std::uint32_t x, std::uint32_t *waves, std::uint32_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  std::uint32_t sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const std::uint32_t y = __shfl_up(sum, d);
    if (lane >= d) sum += y;
  }
  __syncthreads(); // `waves` may still be read from the last call
  if (lane == 63) waves[wave] = sum;
  __syncthreads();
  std::uint32_t before = 0, all = 0;
  for (int w = 0; w < kSelectThreads / 64; ++w) {
    if (w == wave) before = all;
    all += waves[w];
  }
  total = all;
  return before + sum - x;
}

// One workgroup per KV head.  The threshold is the k-th largest rank of the entries
// between the sinks and the recent ones, found digit by digit (8 bits, most
// significant first) from histograms; then the kept indices in ascending order.
__global__ __launch_bounds__(kSelectThreads) void compact_select_kernel(CompactEvictArgs a) {
  __shared__ std::uint32_t hist[256], waves[kSelectThreads / 64], picked[2];
  const std::uint32_t kvh = blockIdx.x;
  const float *w = a.weights + static_cast<std::size_t>(kvh) * a.max_ctx;
  const std::uint32_t lo = a.sinks, hi = a.context - a.recent;
  std::uint32_t need = a.keep - a.sinks - a.recent; // of the entries lo .. hi - 1
  std::uint32_t prefix = 0;
  if (need != 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (threadIdx.x < 256) hist[threadIdx.x] = 0;
      __syncthreads();
      for (std::uint32_t i = lo + threadIdx.x; i < hi; i += kSelectThreads) {
        const std::uint32_t r = rank_of(w[i]);
        if (shift == 24 || (r >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(r >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        std::uint32_t left = need;
        int d = 255;
        for (; d > 0 && hist[d] < left; --d) left -= hist[d];
        picked[0] = static_cast<std::uint32_t>(d);
        picked[1] = left;
      }
      __syncthreads();
      prefix |= picked[0] << shift;
      need = picked[1];
    }
  }
  // Kept: above the threshold, and the first `need` that equal it.
  const bool some = a.keep != a.sinks + a.recent;
  const std::uint32_t seg = (a.context + kSelectThreads - 1) / kSelectThreads;
  const std::uint32_t first = threadIdx.x * seg < a.context ? threadIdx.x * seg : a.context;
  const std::uint32_t last = first + seg < a.context ? first + seg : a.context;
  std::uint32_t sure = 0, equal = 0;
  for (std::uint32_t i = first; i < last; ++i) {
    const std::uint32_t r = rank_of(w[i]);
    const bool always = i < lo || i >= hi;
    sure += always || (some && r > prefix);
    equal += !always && some && r == prefix;
  }
  std::uint32_t total;
  const std::uint32_t equal_before = block_prefix(equal, waves, total);
  std::uint32_t take = equal_before < need ? need - equal_before : 0;
  take = take < equal ? take : equal;
  std::uint32_t at = block_prefix(sure + take, waves, total);
  std::int32_t *kept = a.kept + static_cast<std::size_t>(kvh) * a.keep;
  for (std::uint32_t i = first; i < last; ++i) {
    const std::uint32_t r = rank_of(w[i]);
    bool stays = i < lo || i >= hi || (some && r > prefix);
    if (!stays && some && r == prefix && take != 0) {
      stays = true;
      --take;
    }
    if (stays) kept[at++] = static_cast<std::int32_t>(i);
  }
}

// A workgroup fills one block of 32 positions of one plane and head (grid (blocks of
// the new cache, 2 kv_heads)), thread (row, piece) = (tid / 8, tid % 8) 32 dims of a
// position; the K plane's workgroups move the weights too.
template <bool Fp8, bool OutFp8>
__global__ __launch_bounds__(kMoveThreads) void compact_move_kernel(CompactEvictArgs a) {
  __shared__ float wave_max_of[kMoveThreads / kWave];
  const std::uint32_t kvh = blockIdx.y >> 1, plane = blockIdx.y & 1;
  const std::uint32_t block = blockIdx.x;
  const std::int32_t *kept = a.kept + static_cast<std::size_t>(kvh) * a.keep;
  if (plane == 0 && threadIdx.x < kCompactBlock) {
    const std::uint32_t i = block * kCompactBlock + threadIdx.x;
    if (i < a.out_max_ctx)
      a.out_weights[static_cast<std::size_t>(kvh) * a.out_max_ctx + i] =
          i < a.keep ? a.weights[static_cast<std::size_t>(kvh) * a.max_ctx + kept[i]] : 0.f;
  }
  if (block * kCompactBlock >= a.keep) return; // (uniform)
  const std::uint32_t row = block * kCompactBlock + (threadIdx.x >> 3);
  const int piece = threadIdx.x & 7;
  const bool real = row < a.keep;
  const std::uint32_t from = real ? static_cast<std::uint32_t>(kept[row]) : 0;
  const CompactHead<Fp8> src(const_cast<unsigned char *>(a.cache), kvh, a.kv_heads, a.max_ctx, a.head_major);
  const CompactHead<OutFp8> dst(a.out_cache, kvh, a.kv_heads, a.out_max_ctx, a.head_major);
  const auto *s = (plane ? src.v : src.k) + static_cast<std::size_t>(from) * src.row + 32 * piece;
  auto *d = (plane ? dst.v : dst.k) + static_cast<std::size_t>(row) * dst.row + 32 * piece;
  if constexpr (!OutFp8) {
    if (!real) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<u32x4 *>(d)[j] = reinterpret_cast<const u32x4 *>(s)[j];
  } else {
    float x[32];
    float amax = 0.f;
    if (real) {
      if constexpr (Fp8) {
        const float scale = (plane ? src.vs : src.ks)[from / kCompactBlock];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const u32x4 w = reinterpret_cast<const u32x4 *>(s)[j];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const floatx4 f = fp8x4_to_f32(w[e]);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[16 * j + 4 * e + k] = f[k] * scale;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 w = reinterpret_cast<const u32x4 *>(s)[j];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const std::uint32_t u = w[e];
            x[8 * j + 2 * e] = bf16_lo(u);
            x[8 * j + 2 * e + 1] = bf16_hi(u);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        if (is_finite_f32(x[e])) amax = fmaxf(amax, fabsf(x[e]));
        else x[e] = __builtin_nanf("");
      }
    }
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) wave_max_of[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(wave_max_of[0], wave_max_of[1]), fmaxf(wave_max_of[2], wave_max_of[3]));
    const float scale = compact_scale(amax);
    const float inv = compact_inverse(scale);
    if (threadIdx.x == 0) (plane ? dst.vs : dst.ks)[block] = scale;
    if (!real) return;
    u32x4 out[2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      out[j >> 2][j & 3] = pack_fp8x4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
    reinterpret_cast<u32x4 *>(d)[0] = out[0];
    reinterpret_cast<u32x4 *>(d)[1] = out[1];
  }
}

} // namespace

std::size_t compact_evict_workspace(const CompactEvictArgs &) { return 0; }

void compact_evict(const CompactEvictArgs &a, bool fp8, bool out_fp8, void *, hipStream_t stream) {
  compact_select_kernel<<<a.kv_heads, kSelectThreads, 0, stream>>>(a);
  const dim3 grid{(a.out_max_ctx + kCompactBlock - 1) / kCompactBlock, 2 * a.kv_heads};
  if (fp8) compact_move_kernel<true, true><<<grid, kMoveThreads, 0, stream>>>(a);
  else if (out_fp8) compact_move_kernel<false, true><<<grid, kMoveThreads, 0, stream>>>(a);
  else compact_move_kernel<false, false><<<grid, kMoveThreads, 0, stream>>>(a);
}

} // namespace raftinfer::amd
