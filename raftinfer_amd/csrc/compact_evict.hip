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

// How many lanes before this one a mask has.
__device__ __forceinline__ std::uint32_t lanes_below(std::uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<std::uint32_t>(m >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<std::uint32_t>(m), 0u));
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
// over many values of the first 11 bits (sign, exponent and 2 of mantissa), or many are alike
// (keys that no observed token saw have weight 0).
struct Wanted {
  std::uint32_t lo, hi, need;
  __device__ __forceinline__ explicit Wanted(const CompactEvictArgs &a)
      : lo(a.sinks), hi(a.context - a.recent), need(a.keep - a.sinks - a.recent) {}
};
__device__ __forceinline__ int digit_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__device__ __forceinline__ std::uint32_t digit_mask(int level) { return level == 2 ? 1023u : 2047u; }
__device__ __forceinline__ std::uint32_t digits_above(int level) { return level == 0 ? 0u : level == 1 ? 0xFFE00000u : 0xFFFFFC00u; }

struct SelectShared {
  std::uint32_t hist[2048], waves[kSelectThreads / 64], picked[2], equal;
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
// Counts a lane's digit.  Those that have the first lane's are added at once (each by itself,
// the choice took 52 us of 16384 equal weights; now 17, and 15.5 of spread ones).
__device__ __forceinline__ void count_digit(SelectShared &sh, std::uint32_t digit, bool counts) {
  const std::uint64_t all = __builtin_amdgcn_ballot_w64(counts);
  if (all == 0) return;
  const std::uint32_t first = __builtin_amdgcn_readlane(digit, __builtin_ctzll(all));
  const std::uint64_t alike = __builtin_amdgcn_ballot_w64(digit == first) & all, leader = all & -all;
  if (__builtin_amdgcn_inverse_ballot_w64((all & ~alike) | leader))
    atomicAdd(&sh.hist[digit], __builtin_amdgcn_inverse_ballot_w64(leader) ? static_cast<std::uint32_t>(__popcll(alike)) : 1u);
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
// before `first`; on return, those entries' added.
template <int R>
__device__ __forceinline__ void write_kept(const CompactEvictArgs &a, std::uint32_t *waves, std::uint32_t *sure_of,
                                           std::uint32_t *equal_of, const std::uint32_t (&r)[R], std::uint32_t first, bool some,
                                           std::uint32_t threshold, std::uint32_t need, std::uint32_t &sure_before,
                                           std::uint32_t &equal_before) {
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
  std::uint32_t all; // (both counts in one sum: neither exceeds 16384)
  const bool entry = threadIdx.x < R * kWaves;
  const std::uint32_t at = block_prefix(entry ? sure_of[threadIdx.x] << 16 | equal_of[threadIdx.x] : 0u, waves, all);
  if (entry) {
    sure_of[threadIdx.x] = sure_before + (at >> 16);
    equal_of[threadIdx.x] = equal_before + (at & 0xFFFFu);
  }
  sure_before += all >> 16;
  equal_before += all & 0xFFFFu;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const std::uint32_t at = first + i * kSelectThreads + threadIdx.x;
    const bool sure = is_sure(i, at), equal = is_equal(i);
    const std::uint64_t sm = __builtin_amdgcn_ballot_w64(sure), em = __builtin_amdgcn_ballot_w64(equal);
    const std::uint32_t eq = equal_of[i * kWaves + wave] + lanes_below(em), su = sure_of[i * kWaves + wave] + lanes_below(sm);
    if (sure || (equal && eq < need)) kept[su + (eq < need ? eq : need)] = static_cast<std::int32_t>(at);
  }
}

// One workgroup per KV head, its threads hold R weights each.  Bound by the barriers of its
// passes: 4001 entries 8.1 us.
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
        count_digit(sh, (r[i] >> digit_shift(level)) & digit_mask(level), r[i] != 0 && (r[i] & digits_above(level)) == threshold);
      __syncthreads();
      threshold |= pick_digit(sh, need) << digit_shift(level);
    }
  }
  std::uint32_t sure_before = 0, equal_before = 0;
  write_kept<R>(a, sh.waves, sure_of, equal_of, r, 0, wanted.need != 0, threshold, need, sure_before, equal_before);
}

// Longer caches: launches over segments (grid (kv_heads, segments)), at most 64 a head, so that
// the work is linear in the entries.  A launch counts each segment's digits of a level; the next
// one adds the segments up, which gives the threshold's digit, and what the segments before its
// own hold above it.  The last one writes each segment's kept entries behind those of the segments
// before it.  Segments of 4096 entries take three launches: the second one leaves the ranks that
// share the first digit (few, unless many weights are alike), and every workgroup of the third
// counts the last digits among them.  Longer segments take four: there that could be 64 times
// all ranks.  No count depends on the order in which workgroups run.
//
// 60001 entries of 4 heads: 4.0 + 7.0 + 9.7 us, the latency of dependent loads and barriers (the
// weights are 1 MB).  With the move, spread and equal weights: 60001 entries 33 and 51 us (four launches
// 38 and 38), 262144 85 and 152 (94 and 89); 1000000 of one head in four 103 and 99.
constexpr int kSegR = 4;
constexpr std::uint32_t kPiece = kSegR * kSelectThreads;
constexpr std::uint32_t kMostSegments = 64;
struct Segments {
  std::uint32_t count, pieces; // of a head, of a segment
  __host__ __device__ __forceinline__ explicit Segments(std::uint32_t context) {
    const std::uint32_t all = (context + kPiece - 1) / kPiece;
    pieces = (all + kMostSegments - 1) / kMostSegments;
    count = (all + pieces - 1) / pieces;
  }
};
struct SelectScratch {
  std::uint32_t *hist;   // [level][kv_head][segment][2048]; level 2 in place of the ranks
  std::uint32_t *ranks;  // [kv_head][segment][4096]: ranks that share the first digit (segments of 4096)
  std::uint32_t *shared; // [kv_head][segment]: how many
  std::uint32_t *above;  // [level 0, 1][kv_head][segment]: entries of the segments before with the digits found and a larger one
  std::uint32_t *found;  // [level 0, 1][kv_head][2]: the threshold's digits so far, entries of these that are still wanted
};
__device__ __forceinline__ std::size_t level_of(int level) { // of `above`
  return (static_cast<std::size_t>(level) * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y;
}

// The threshold's digit at a level, as pick_digit, from the head's histograms.  above: this
// thread's share of the entries of the segments before this one with a larger digit; behind the
// next barrier sh.equal holds those with that one.
__device__ __forceinline__ std::uint32_t find_digit(SelectShared &sh, const SelectScratch &sc, int level, std::uint32_t &need,
                                                    std::uint32_t &above) {
  const std::uint32_t *hist =
      sc.hist + (static_cast<std::size_t>(level) * gridDim.x + blockIdx.x) * gridDim.y * 2048 + 2046 - 2 * threadIdx.x;
  std::uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
  for (std::uint32_t s0 = 0; s0 < gridDim.y; s0 += 16) { // (sixteen loads under way: they come from other XCDs' workgroups)
    u32x2 h[16];
#pragma unroll
    for (std::uint32_t b = 0; b < 16; ++b)
      h[b] = *reinterpret_cast<const u32x2 *>(hist + static_cast<std::size_t>(s0 + b < gridDim.y ? s0 + b : s0) * 2048);
#pragma unroll
    for (std::uint32_t b = 0; b < 16; ++b) {
      h0 += s0 + b < gridDim.y ? h[b][0] : 0u;
      h1 += s0 + b < gridDim.y ? h[b][1] : 0u;
      b0 += s0 + b < blockIdx.y ? h[b][0] : 0u;
      b1 += s0 + b < blockIdx.y ? h[b][1] : 0u;
    }
  }
  const std::uint32_t digit = pick_digit(sh, h1, h0, need);
  const std::uint32_t mine = 2047 - 2 * threadIdx.x; // h1's
  if (mine >> 1 == digit >> 1) sh.equal = digit & 1 ? b1 : b0;
  above = (mine > digit ? b1 : 0u) + (mine - 1 > digit ? b0 : 0u);
  return digit;
}

// Level 0 to 2: the histograms of that level's digits (after the first, of the entries that
// share the threshold's digits before).  Ranks: level 1 also leaves these entries' ranks.
template <int Level, bool Ranks>
__global__ __launch_bounds__(kSelectThreads) void compact_count_kernel(CompactEvictArgs a, SelectScratch sc) {
  __shared__ SelectShared sh;
  const Wanted wanted(a);
  if (wanted.need == 0) return; // (uniform)
  const std::uint32_t pieces = Segments(a.context).pieces;
  std::uint32_t first = blockIdx.y * pieces * kPiece;
  float x[kSegR];
  load_weights<kSegR>(a, first, x);
  clear_histogram(sh);
  std::uint32_t threshold = 0, above = 0, need = wanted.need;
  if constexpr (Level > 0) {
    if constexpr (Level == 2) {
      threshold = sc.found[2 * blockIdx.x];
      need = sc.found[2 * blockIdx.x + 1];
    }
    threshold |= find_digit(sh, sc, Level - 1, need, above) << digit_shift(Level - 1);
  }
  for (std::uint32_t piece = 0;;) {
    std::uint32_t r[kSegR];
    ranks_of<kSegR>(wanted, first, x, r);
    if (++piece < pieces) load_weights<kSegR>(a, first + kPiece, x);
    const auto counts = [&](int i) { return r[i] != 0 && (r[i] & digits_above(Level)) == threshold; };
#pragma unroll
    for (int i = 0; i < kSegR; ++i) count_digit(sh, (r[i] >> digit_shift(Level)) & digit_mask(Level), counts(i));
    if constexpr (Ranks) {
      // (with `above` in one sum: 4096 and, of at most 64 segments, 2^18 entries)
      std::uint32_t n = 0, all;
#pragma unroll
      for (int i = 0; i < kSegR; ++i) n += counts(i);
      std::uint32_t place = block_prefix(above << 13 | n, sh.waves, all) & 0x1FFFu;
      above = all >> 13;
      const std::size_t seg = level_of(0);
#pragma unroll
      for (int i = 0; i < kSegR; ++i)
        if (counts(i)) sc.ranks[seg * kPiece + place++] = r[i]; // (in no particular order)
      if (threadIdx.x == 0) sc.shared[seg] = all & 0x1FFFu;
    }
    if (piece == pieces) break;
    first += kPiece;
  }
  if constexpr (Level > 0) {
    if constexpr (!Ranks) {
      const std::uint32_t share = above;
      (void)block_prefix(share, sh.waves, above);
    }
    if (threadIdx.x == 0) {
      sc.above[level_of(Level - 1)] = above;
      if (blockIdx.y == 0) {
        std::uint32_t *found = sc.found + 2 * ((Level - 1) * gridDim.x + blockIdx.x);
        found[0] = threshold;
        found[1] = need;
      }
    }
  }
  __syncthreads();
  std::uint32_t *out = sc.hist + level_of(Level) * 2048;
  for (int i = threadIdx.x; i < 2048; i += kSelectThreads) out[i] = sh.hist[i];
}

template <bool Ranks>
__global__ __launch_bounds__(kSelectThreads) void compact_write_kernel(CompactEvictArgs a, SelectScratch sc) {
  __shared__ SelectShared sh;
  __shared__ std::uint32_t sure_of[kSegR * kSelectThreads / 64], equal_of[kSegR * kSelectThreads / 64];
  const Wanted wanted(a);
  const std::uint32_t pieces = Segments(a.context).pieces;
  std::uint32_t first = blockIdx.y * pieces * kPiece;
  float x[kSegR];
  load_weights<kSegR>(a, first, x);
  // sinks and recent entries before this segment
  std::uint32_t sure_before = (first < wanted.lo ? first : wanted.lo) + (first > wanted.hi ? first - wanted.hi : 0u);
  std::uint32_t equal_before = 0, threshold = 0, need = 0;
  if (Ranks && wanted.need != 0) {
    // A wave takes the ranks of every 16th segment, four loads at a time under way.  The first four,
    // and how many its first segment has, are asked for here with all else.
    const std::uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const std::size_t seg0 = static_cast<std::size_t>(blockIdx.x) * gridDim.y, first_seg = seg0 + (wave < gridDim.y ? wave : 0);
    const std::uint32_t first_n = sc.shared[first_seg];
    std::uint32_t r4[4]; // (what lies behind the last of those is not used)
#pragma unroll
    for (int b = 0; b < 4; ++b) r4[b] = sc.ranks[first_seg * kPiece + lane + 64 * b];
    threshold = sc.found[2 * blockIdx.x];
    need = sc.found[2 * blockIdx.x + 1];
    sure_before += sc.above[level_of(0)];
    clear_histogram(sh);
    std::uint32_t above;
    threshold |= find_digit(sh, sc, 1, need, above) << digit_shift(1);
    // bins of the last digit: of all segments, and behind them of those before this one
    for (std::uint32_t s = wave; s < gridDim.y; s += kSelectThreads / 64) {
      const std::uint32_t n = s == wave ? first_n : sc.shared[seg0 + s];
      const std::uint32_t *ranks = sc.ranks + (seg0 + s) * kPiece;
      for (std::uint32_t i = 0; i < n; i += 4 * 64) {
        if (s != wave || i != 0) {
#pragma unroll
          for (int b = 0; b < 4; ++b) r4[b] = ranks[i + lane + 64 * b < n ? i + lane + 64 * b : i];
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bool counts = i + lane + 64 * b < n && (r4[b] & digits_above(2)) == threshold;
          if (__builtin_amdgcn_ballot_w64(counts) == 0) continue;
          count_digit(sh, r4[b] & digit_mask(2), counts);
          if (s < blockIdx.y) count_digit(sh, (r4[b] & digit_mask(2)) + 1024, counts);
        }
      }
    }
    __syncthreads();
    const std::uint32_t top = 1023 - 2 * threadIdx.x; // this thread's bins: top and top - 1
    const bool bins = threadIdx.x < 512;
    const std::uint32_t b1 = bins ? sh.hist[1024 + top] : 0u, b0 = bins ? sh.hist[1023 + top] : 0u;
    const std::uint32_t digit = pick_digit(sh, bins ? sh.hist[top] : 0u, bins ? sh.hist[top - 1] : 0u, need) - 1024;
    equal_before = sh.hist[1024 + digit];
    std::uint32_t all;
    (void)block_prefix(above + (bins && top > digit ? b1 : 0u) + (bins && top - 1 > digit ? b0 : 0u), sh.waves, all);
    sure_before += all;
    threshold |= digit;
  } else if (wanted.need != 0) {
    const std::uint32_t *found = sc.found + 2 * (gridDim.x + blockIdx.x);
    threshold = found[0];
    need = found[1];
    sure_before += sc.above[level_of(0)] + sc.above[level_of(1)];
    std::uint32_t above, all;
    threshold |= find_digit(sh, sc, 2, need, above);
    (void)block_prefix(above, sh.waves, all);
    sure_before += all;
    equal_before = sh.equal;
  }
  for (std::uint32_t piece = 0;;) {
    std::uint32_t r[kSegR];
    ranks_of<kSegR>(wanted, first, x, r);
    if (++piece < pieces) load_weights<kSegR>(a, first + kPiece, x);
    write_kept<kSegR>(a, sh.waves, sure_of, equal_of, r, first, wanted.need != 0, threshold, need, sure_before, equal_before);
    if (piece == pieces) break;
    first += kPiece;
    __syncthreads(); // sure_of and equal_of are read
  }
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
std::size_t segments_of(const CompactEvictArgs &a) { // of all heads
  return a.context <= kOneGroup ? 0 : static_cast<std::size_t>(a.kv_heads) * Segments(a.context).count;
}
} // namespace

std::size_t compact_evict_workspace(const CompactEvictArgs &a) {
  const std::size_t n = segments_of(a);
  return n == 0 ? 0 : (n * (2 * 2048 + kPiece + 3) + 4 * a.kv_heads) * sizeof(std::uint32_t);
}

void compact_evict(const CompactEvictArgs &a, bool fp8, bool out_fp8, void *workspace, hipStream_t stream) {
  if (a.context <= 4 * kSelectThreads) {
    compact_select_kernel<4><<<a.kv_heads, kSelectThreads, 0, stream>>>(a);
  } else if (a.context <= kOneGroup) {
    compact_select_kernel<16><<<a.kv_heads, kSelectThreads, 0, stream>>>(a);
  } else {
    const std::size_t n = segments_of(a);
    auto *p = static_cast<std::uint32_t *>(workspace);
    std::uint32_t *behind = p + n * (2 * 2048 + kPiece); // (level 2's histograms are no longer than the ranks)
    const SelectScratch sc{p, p + n * 2 * 2048, behind, behind + n, behind + 3 * n};
    const dim3 grid{a.kv_heads, static_cast<unsigned>(n / a.kv_heads)};
    compact_count_kernel<0, false><<<grid, kSelectThreads, 0, stream>>>(a, sc);
    if (Segments(a.context).pieces == 1) {
      compact_count_kernel<1, true><<<grid, kSelectThreads, 0, stream>>>(a, sc);
      compact_write_kernel<true><<<grid, kSelectThreads, 0, stream>>>(a, sc);
    } else {
      compact_count_kernel<1, false><<<grid, kSelectThreads, 0, stream>>>(a, sc);
      compact_count_kernel<2, false><<<grid, kSelectThreads, 0, stream>>>(a, sc);
      compact_write_kernel<false><<<grid, kSelectThreads, 0, stream>>>(a, sc);
    }
  }
  const dim3 grid{(a.out_max_ctx + kCompactBlock - 1) / kCompactBlock, 2 * a.kv_heads};
  if (fp8) compact_move_kernel<true, true><<<grid, kMoveThreads, 0, stream>>>(a);
  else if (out_fp8) compact_move_kernel<false, true><<<grid, kMoveThreads, 0, stream>>>(a);
  else compact_move_kernel<false, false><<<grid, kMoveThreads, 0, stream>>>(a);
}

} // namespace raftinfer::amd
