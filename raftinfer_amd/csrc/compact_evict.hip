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
__device__ __forceinline__ std::uint32_t block_prefix(std::uint32_t x, std::uint32_t *waves, std::uint32_t &total) {
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
#pragma unroll
  for (int w = 0; w < kSelectThreads / 64; ++w) {
    before = w == wave ? all : before;
    all += waves[w];
  }
  total = all;
  return before + sum - x;
}

// Which entries stay: all sinks and recent ones, and of the others (lo .. hi - 1) those
// whose rank is above a threshold, and the first `need` that equal it.  The threshold is
// the k-th largest rank, found by histograms over its first 11, next 11 and last 10 bits,
// of which the second and third count only what shares the digits found.  Weights spread
// over many values of the first 11 bits (exponent and 3 of mantissa), so few lanes of a
// wave meet in a bin.
struct Wanted {
  std::uint32_t lo, hi, need;
  __device__ __forceinline__ explicit Wanted(const CompactEvictArgs &a)
      : lo(a.sinks), hi(a.context - a.recent), need(a.keep - a.sinks - a.recent) {}
};
__device__ __forceinline__ int digit_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__device__ __forceinline__ std::uint32_t digit_mask(int level) { return level == 2 ? 1023u : 2047u; }
__device__ __forceinline__ std::uint32_t digits_above(int level) { return level == 0 ? 0u : level == 1 ? 0xFFE00000u : 0xFFFFFC00u; }

struct SelectShared {
  std::uint32_t hist[2048], waves[kSelectThreads / 64], picked[2];
};
// From the histogram of a level (thread t: h1 and h0, the counts of bins 2047 - 2 t and
// 2046 - 2 t) the digit of the need-th largest entry, and how many entries of that digit
// are still wanted.
__device__ __forceinline__ std::uint32_t pick_digit(SelectShared &sh, std::uint32_t h1, std::uint32_t h0, std::uint32_t &need) {
  std::uint32_t total;
  const std::uint32_t before = block_prefix(h0 + h1, sh.waves, total);
  if (before < need && need <= before + h0 + h1) {
    const bool first = need <= before + h1;
    sh.picked[0] = first ? 2047 - 2 * threadIdx.x : 2046 - 2 * threadIdx.x;
    sh.picked[1] = need - before - (first ? 0 : h1);
  }
  __syncthreads();
  need = sh.picked[1];
  return sh.picked[0];
}
__device__ __forceinline__ std::uint32_t pick_digit(SelectShared &sh, std::uint32_t &need) {
  return pick_digit(sh, sh.hist[2047 - 2 * threadIdx.x], sh.hist[2046 - 2 * threadIdx.x], need);
}
__device__ __forceinline__ void clear_histogram(SelectShared &sh) {
  for (int i = threadIdx.x; i < 2048; i += kSelectThreads) sh.hist[i] = 0;
  __syncthreads();
}
// Ranks of entries first + 1024 i + thread; 0, which no weight has, for those that the
// weights do not decide (sinks, recent ones, behind the last).
template <int R>
__device__ __forceinline__ void load_weights(const CompactEvictArgs &a, std::uint32_t first, float (&x)[R]) {
  const float *w = a.weights + static_cast<std::size_t>(blockIdx.x) * a.max_ctx;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const std::uint32_t at = first + i * kSelectThreads + threadIdx.x;
    x[i] = w[at < a.context ? at : a.context - 1];
  }
}
template <int R>
__device__ __forceinline__ void ranks_of(const Wanted &wanted, std::uint32_t first, const float (&x)[R], std::uint32_t (&r)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
    r[i] = first + i * kSelectThreads + threadIdx.x - wanted.lo < wanted.hi - wanted.lo ? rank_of(x[i]) : 0u;
}
template <int R>
__device__ __forceinline__ void load_ranks(const CompactEvictArgs &a, const Wanted &wanted, std::uint32_t first, std::uint32_t (&r)[R]) {
  float x[R];
  load_weights<R>(a, first, x);
  ranks_of<R>(wanted, first, x, r);
}
// Writes the kept ones of those entries in ascending order: counts per row of 1024
// entries and wave, one prefix sum, and a lane's place from its wave's masks.
// sure_before, equal_before: kept for sure, and equal to the threshold, among the entries
// before `first`.
template <int R>
__device__ __forceinline__ void write_kept(const CompactEvictArgs &a, std::uint32_t *waves, std::uint32_t *sure_of,
                                           std::uint32_t *equal_of, const std::uint32_t (&r)[R], std::uint32_t first, bool some,
                                           std::uint32_t threshold, std::uint32_t need, std::uint32_t sure_before,
                                           std::uint32_t equal_before) {
  constexpr int kWaves = kSelectThreads / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  std::int32_t *kept = a.kept + static_cast<std::size_t>(blockIdx.x) * a.keep;
  const auto is_sure = [&](int i, std::uint32_t at) { return r[i] == 0 ? at < a.context : some && r[i] > threshold; };
  const auto is_equal = [&](int i) { return some && r[i] == threshold; };
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const std::uint64_t sure = __builtin_amdgcn_ballot_w64(is_sure(i, first + i * kSelectThreads + threadIdx.x));
    const std::uint64_t equal = __builtin_amdgcn_ballot_w64(is_equal(i));
    if (lane == 0) {
      sure_of[i * kWaves + wave] = static_cast<std::uint32_t>(__popcll(sure));
      equal_of[i * kWaves + wave] = static_cast<std::uint32_t>(__popcll(equal));
    }
  }
  __syncthreads();
  std::uint32_t total;
  const bool entry = threadIdx.x < R * kWaves;
  const std::uint32_t sure_at = block_prefix(entry ? sure_of[threadIdx.x] : 0u, waves, total);
  const std::uint32_t equal_at = block_prefix(entry ? equal_of[threadIdx.x] : 0u, waves, total);
  if (entry) {
    sure_of[threadIdx.x] = sure_before + sure_at;
    equal_of[threadIdx.x] = equal_before + equal_at;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const std::uint32_t at = first + i * kSelectThreads + threadIdx.x;
    const bool sure = is_sure(i, at), equal = is_equal(i);
    const std::uint64_t sm = __builtin_amdgcn_ballot_w64(sure), em = __builtin_amdgcn_ballot_w64(equal);
    const auto below = [](std::uint64_t m) {
      return __builtin_amdgcn_mbcnt_hi(static_cast<std::uint32_t>(m >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<std::uint32_t>(m), 0u));
    };
    const std::uint32_t eq = equal_of[i * kWaves + wave] + below(em), su = sure_of[i * kWaves + wave] + below(sm);
    if (sure || (equal && eq < need)) kept[su + (eq < need ? eq : need)] = static_cast<std::int32_t>(at);
  }
}

// One workgroup per KV head, its threads hold R weights each.  Bound by the barriers of its
// passes: 4001 entries 8.2 us.
template <int R>
__global__ __launch_bounds__(kSelectThreads) void compact_select_kernel(CompactEvictArgs a) {
  __shared__ SelectShared sh;
  __shared__ std::uint32_t sure_of[R * kSelectThreads / 64], equal_of[R * kSelectThreads / 64];
  const Wanted wanted(a);
  std::uint32_t need = wanted.need, threshold = 0;
  std::uint32_t r[R];
  load_ranks<R>(a, wanted, 0, r);
  if (need != 0) {
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      clear_histogram(sh);
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (r[i] != 0 && (r[i] & digits_above(level)) == threshold)
          atomicAdd(&sh.hist[(r[i] >> digit_shift(level)) & digit_mask(level)], 1u);
      __syncthreads();
      threshold |= pick_digit(sh, need) << digit_shift(level);
    }
  }
  write_kept<R>(a, sh.waves, sure_of, equal_of, r, 0, wanted.need != 0, threshold, need, 0, 0);
}

// Longer caches: three launches over segments of 4096 entries (grid (kv_heads,
// segments)).  The first counts each segment's first digits.  In the second every
// segment finds the threshold's first digit, and leaves how many entries have a larger
// one and the ranks of those that share it (few, unless many weights are alike).  In the
// third every segment finds the rest of the threshold from all of these, and writes its
// kept entries behind those of the segments before it.  No count depends on the order in
// which workgroups run.  60001 entries of 4 heads: 3.5 + 6.8 + 9.4 us, the latency of dependent
// loads and barriers (the weights are 1 MB).
constexpr int kSegR = 4;
constexpr std::uint32_t kSegment = kSegR * kSelectThreads;
static_assert(kSegment == 4096); // (the entry point allows 65535 of them)
struct SelectScratch {
  std::uint32_t *hist;    // [kv_head][segment][2048]
  std::uint32_t *larger;  // [kv_head][segment]: entries kept for sure after the first digit
  std::uint32_t *shared;  // [kv_head][segment]: entries that share the first digit
  std::uint32_t *ranks;   // [kv_head][segment][4096]: their ranks
};

__global__ __launch_bounds__(kSelectThreads) void compact_count_kernel(CompactEvictArgs a, SelectScratch sc) {
  __shared__ SelectShared sh;
  const Wanted wanted(a);
  std::uint32_t r[kSegR];
  load_ranks<kSegR>(a, wanted, blockIdx.y * kSegment, r);
  clear_histogram(sh);
#pragma unroll
  for (int i = 0; i < kSegR; ++i)
    if (r[i] != 0) atomicAdd(&sh.hist[r[i] >> 21], 1u);
  __syncthreads();
  std::uint32_t *out = sc.hist + (static_cast<std::size_t>(blockIdx.x) * gridDim.y + blockIdx.y) * 2048;
  for (int i = threadIdx.x; i < 2048; i += kSelectThreads) out[i] = sh.hist[i];
}

__global__ __launch_bounds__(kSelectThreads) void compact_narrow_kernel(CompactEvictArgs a, SelectScratch sc) {
  __shared__ SelectShared sh;
  const Wanted wanted(a);
  float x[kSegR];
  load_weights<kSegR>(a, blockIdx.y * kSegment, x);
  const std::size_t seg = static_cast<std::size_t>(blockIdx.x) * gridDim.y + blockIdx.y;
  std::uint32_t digit = 2048; // no entry is wanted: all of them are smaller
  if (wanted.need != 0) {
    const std::uint32_t *hist = sc.hist + static_cast<std::size_t>(blockIdx.x) * gridDim.y * 2048 + 2046 - 2 * threadIdx.x;
    std::uint32_t h0 = 0, h1 = 0, need = wanted.need;
    for (std::uint32_t s0 = 0; s0 < gridDim.y; s0 += 16) { // (sixteen loads under way: they come from other XCDs' workgroups)
      u32x2 h[16];
#pragma unroll
      for (std::uint32_t b = 0; b < 16; ++b)
        h[b] = *reinterpret_cast<const u32x2 *>(hist + static_cast<std::size_t>(s0 + b < gridDim.y ? s0 + b : s0) * 2048);
#pragma unroll
      for (std::uint32_t b = 0; b < 16; ++b) {
        h0 += s0 + b < gridDim.y ? h[b][0] : 0u;
        h1 += s0 + b < gridDim.y ? h[b][1] : 0u;
      }
    }
    digit = pick_digit(sh, h1, h0, need);
  }
  std::uint32_t r[kSegR];
  ranks_of<kSegR>(wanted, blockIdx.y * kSegment, x, r);
  std::uint32_t larger = 0, shared = 0;
#pragma unroll
  for (int i = 0; i < kSegR; ++i) {
    const std::uint32_t at = blockIdx.y * kSegment + i * kSelectThreads + threadIdx.x;
    larger += r[i] == 0 ? at < a.context : (r[i] >> 21) > digit;
    shared += r[i] != 0 && (r[i] >> 21) == digit;
  }
  std::uint32_t all_larger, all_shared;
  (void)block_prefix(larger, sh.waves, all_larger);
  std::uint32_t place = block_prefix(shared, sh.waves, all_shared);
#pragma unroll
  for (int i = 0; i < kSegR; ++i)
    if (r[i] != 0 && (r[i] >> 21) == digit) sc.ranks[seg * kSegment + place++] = r[i]; // (in no particular order)
  if (threadIdx.x == 0) {
    sc.larger[seg] = all_larger;
    sc.shared[seg] = all_shared;
  }
}

__global__ __launch_bounds__(kSelectThreads) void compact_write_kernel(CompactEvictArgs a, SelectScratch sc) {
  __shared__ SelectShared sh;
  __shared__ std::uint32_t sure_of[kSegR * kSelectThreads / 64], equal_of[kSegR * kSelectThreads / 64];
  const Wanted wanted(a);
  float x[kSegR];
  load_weights<kSegR>(a, blockIdx.y * kSegment, x);
  const std::size_t seg0 = static_cast<std::size_t>(blockIdx.x) * gridDim.y;
  // f(rank, segment) over the ranks that share the threshold's first digit, a wave those of
  // every 16th segment, four loads at a time under way.  The first four, and how many its
  // first segment has, are asked for here with all else.
  const std::uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const std::size_t first_seg = seg0 + (wave < gridDim.y ? wave : 0);
  const std::uint32_t first_n = sc.shared[first_seg];
  std::uint32_t first_ranks[4]; // (what lies behind the last of those is not used)
#pragma unroll
  for (int b = 0; b < 4; ++b) first_ranks[b] = sc.ranks[first_seg * kSegment + lane + 64 * b];
  const auto each = [&](auto f) {
    for (std::uint32_t s = wave; s < gridDim.y; s += kSelectThreads / 64) {
      const std::uint32_t n = s == wave ? first_n : sc.shared[seg0 + s];
      const std::uint32_t *ranks = sc.ranks + (seg0 + s) * kSegment;
      for (std::uint32_t i = lane; i < n; i += 4 * 64) {
        std::uint32_t r4[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) r4[b] = first_ranks[b];
        if (s != wave || i != lane) {
#pragma unroll
          for (int b = 0; b < 4; ++b) r4[b] = ranks[i + 64 * b < n ? i + 64 * b : i];
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (i + 64 * b < n) f(r4[b], s);
      }
    }
  };
  // Kept for sure after the first digit: in all segments before this one, and in all (which
  // leaves what is wanted of the digit).
  std::uint32_t mine = 0, all = 0;
  for (std::uint32_t s = threadIdx.x; s < gridDim.y; s += kSelectThreads) {
    const std::uint32_t n = sc.larger[seg0 + s];
    all += n;
    mine += s < blockIdx.y ? n : 0u;
  }
  std::uint32_t r[kSegR];
  ranks_of<kSegR>(wanted, blockIdx.y * kSegment, x, r);
  std::uint32_t larger_before, larger_all;
  (void)block_prefix(mine, sh.waves, larger_before);
  (void)block_prefix(all, sh.waves, larger_all);
  std::uint32_t need = a.keep - larger_all, threshold = 0, sure_before = larger_before, equal_before = 0;
  if (wanted.need != 0) {
    clear_histogram(sh);
    each([&](std::uint32_t rank, std::uint32_t) {
      sh.picked[0] = rank >> 21; // (the same for all; there is one, as need is not 0)
      atomicAdd(&sh.hist[(rank >> 10) & 2047u], 1u);
    });
    __syncthreads();
    threshold = sh.picked[0] << 21;
    __syncthreads();
    threshold |= pick_digit(sh, need) << 10;
    __syncthreads();
    clear_histogram(sh);
    each([&](std::uint32_t rank, std::uint32_t) {
      if ((rank & 0xFFFFFC00u) == threshold) atomicAdd(&sh.hist[rank & 1023u], 1u);
    });
    __syncthreads();
    threshold |= pick_digit(sh, need);
    std::uint32_t above = 0, equal = 0;
    each([&](std::uint32_t rank, std::uint32_t s) {
      above += s < blockIdx.y && rank > threshold;
      equal += s < blockIdx.y && rank == threshold;
    });
    std::uint32_t all_above;
    (void)block_prefix(above, sh.waves, all_above);
    (void)block_prefix(equal, sh.waves, equal_before);
    sure_before += all_above;
  }
  write_kept<kSegR>(a, sh.waves, sure_of, equal_of, r, blockIdx.y * kSegment, wanted.need != 0, threshold, need, sure_before,
                    equal_before);
}

// A workgroup fills one block of 32 positions of one plane and head (grid (blocks of
// the new cache, 2 kv_heads)), thread (row, piece) = (tid / 8, tid % 8) 32 dims of a
// position; the K plane's workgroups move the weights too.  Bound by memory: 16384 8-bit
// entries of 4 heads, 67 MB, 15.2 us.
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
    if (scale == kCompactTopScale) {
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = compact_below_top(x[e]);
    }
    u32x4 out[2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      out[j >> 2][j & 3] = pack_fp8x4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
    reinterpret_cast<u32x4 *>(d)[0] = out[0];
    reinterpret_cast<u32x4 *>(d)[1] = out[1];
  }
}

} // namespace

namespace {
// One workgroup per head up to here (60001 entries in registers spilled and took 73 us).
constexpr std::uint32_t kOneGroup = 16 * kSelectThreads;
std::size_t segments_of(const CompactEvictArgs &a) {
  return a.context <= kOneGroup ? 0 : static_cast<std::size_t>(a.kv_heads) * ((a.context + kSegment - 1) / kSegment);
}
} // namespace

std::size_t compact_evict_workspace(const CompactEvictArgs &a) {
  return segments_of(a) * (2048 + 2 + kSegment) * sizeof(std::uint32_t);
}

void compact_evict(const CompactEvictArgs &a, bool fp8, bool out_fp8, void *workspace, hipStream_t stream) {
  if (a.context <= 4 * kSelectThreads) {
    compact_select_kernel<4><<<a.kv_heads, kSelectThreads, 0, stream>>>(a);
  } else if (a.context <= kOneGroup) {
    compact_select_kernel<16><<<a.kv_heads, kSelectThreads, 0, stream>>>(a);
  } else {
    const std::size_t n = segments_of(a);
    auto *p = static_cast<std::uint32_t *>(workspace);
    const SelectScratch sc{p, p + n * (2048 + kSegment), p + n * (2048 + kSegment + 1), p + n * 2048};
    const dim3 grid{a.kv_heads, static_cast<unsigned>(n / a.kv_heads)};
    compact_count_kernel<<<grid, kSelectThreads, 0, stream>>>(a, sc);
    compact_narrow_kernel<<<grid, kSelectThreads, 0, stream>>>(a, sc);
    compact_write_kernel<<<grid, kSelectThreads, 0, stream>>>(a, sc);
  }
  const dim3 grid{(a.out_max_ctx + kCompactBlock - 1) / kCompactBlock, 2 * a.kv_heads};
  if (fp8) compact_move_kernel<true, true><<<grid, kMoveThreads, 0, stream>>>(a);
  else if (out_fp8) compact_move_kernel<false, true><<<grid, kMoveThreads, 0, stream>>>(a);
  else compact_move_kernel<false, false><<<grid, kMoveThreads, 0, stream>>>(a);
}

} // namespace raftinfer::amd
