// Prompt attention over the compact KV cache, and the key weights of its last
// tokens.
#include "compact_cache.hpp"
#include "prefill_tile.hpp"

#include <algorithm>
#include <cfloat>

namespace raftinfer::amd {
namespace {

using prefill::fexp2;
using prefill::kLazyRescale;

constexpr int kPWaves = 4;
constexpr int kPThreads = kPWaves * kWave;
constexpr int kPCols = 32 * kPWaves; // columns (token, head of the group) per workgroup
constexpr int kTileElems = kCompactBlock * kHeadDim;
constexpr std::uint32_t kPrefillCus = 256;

// Partials of a split call, [split][kv_head][column], and the final max (exp2
// domain) and 1 / sum of each column for the key weights.  An output is divided by the sum
// of the probabilities as they were rounded to bf16 for the product with V (l), so that it is
// an average of the V rows; the key weights by the sum of the exact ones (lw).
struct PrefillScratch {
  float *m, *l, *lw, *o, *final;
  std::uint32_t cols;         // columns of a KV head, rounded up to whole workgroups
  std::uint32_t block;        // columns of a workgroup
  std::uint32_t tiles, most;  // of a column block's ranges: tiles of one, ranges
};

// A column block's ranges: of about equal length, and of `tiles` tiles unless those were
// more than `most`.
struct TileRanges {
  std::uint32_t count, each, more; // the first `more` have a tile above `each`
  __device__ __forceinline__ TileRanges(const PrefillScratch &sc, std::uint32_t total) {
    count = (total + sc.tiles - 1) / sc.tiles;
    count = count < sc.most ? count : sc.most;
    each = total / count;
    more = total - each * count;
  }
  __device__ __forceinline__ std::uint32_t begin(std::uint32_t i) const { return i * each + (i < more ? i : more); }
};

// 16-byte chunk c of row r of a bf16 tile lies at c ^ row_key(r): the 16 rows of a
// ds_read_b128 pass and the 4 rows x 64 bytes of a ds_read_b64_tr_b16 pass share no bank.
__device__ __forceinline__ int row_key(int r) { return 4 * (r & 3) + ((r >> 2) & 3); }
__device__ __forceinline__ int tile_at(int r, int c) { return r * kHeadDim + ((c ^ row_key(r)) << 3); } // in elements

// 64 or 80 KiB: two workgroups per CU.
template <bool Fp8> struct PrefillShared {
  bf16_bits k[2][kTileElems];
  bf16_bits v[2][kTileElems];
  // 8 bit: a tile's K codes, then V codes, rows of 256 bytes
  unsigned char raw[Fp8 ? 2 * kTileElems : 16];
};

// Sets the infinite and NaN values among eight bf16 to 0; whether there were any.
__device__ __forceinline__ bool without_odd(u32x4 &w) {
  std::uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const std::uint32_t x = w[e];
    const std::uint32_t fine = ((x & 0x7F80u) != 0x7F80u ? 0xFFFFu : 0u) | ((x & 0x7F800000u) != 0x7F800000u ? 0xFFFF0000u : 0u);
    bad |= ~fine;
    w[e] = x & fine;
  }
  return bad != 0;
}

// Whether some column of tokens p_lo .. p_hi does not see some key of the tile at j0.
__device__ __forceinline__ bool tile_masked(std::uint32_t j0, std::uint32_t p_lo, std::uint32_t p_hi, std::uint32_t window,
                                            std::uint32_t sinks) {
  return j0 + kCompactBlock - 1 > p_lo || (window != 0 && j0 + kCompactBlock > sinks && p_hi - j0 >= window);
}

// Row j (positions of a tile j .. have rows row_bytes apart) of the K or V of one KV head: in
// the cache, or of the call's own tokens, where the kernel stores them itself, in key / value
// (past is then a multiple of the tile, so no tile has rows of both).
template <bool Fp8> struct KeyRows {
  const unsigned char *at;
  std::uint32_t row_bytes;
  __device__ __forceinline__ KeyRows(const CompactArgs &a, const CompactHead<Fp8> &c, std::uint32_t kvh, std::uint32_t j, bool is_v) {
    if (!Fp8 && a.store_inside && j >= a.past) {
      row_bytes = a.kv_heads * kHeadDim * 2;
      at = reinterpret_cast<const unsigned char *>((is_v ? a.value : a.key) +
                                                   (static_cast<std::size_t>(j - a.past) * a.kv_heads + kvh) * kHeadDim);
    } else {
      row_bytes = static_cast<std::uint32_t>(c.row * sizeof(typename CompactHead<Fp8>::T));
      at = reinterpret_cast<const unsigned char *>((is_v ? c.v : c.k) + static_cast<std::size_t>(j) * c.row);
    }
  }
};
// Stores the rows of the tokens whose first column is among col0 .. col_end - 1.
__device__ __forceinline__ void store_rows(const CompactArgs &a, const CompactHead<false> &c, std::uint32_t kvh, std::uint32_t col0,
                                           std::uint32_t col_end) {
  const std::uint32_t t0 = (col0 + a.group - 1) / a.group, t1 = (col_end + a.group - 1) / a.group;
  constexpr int kBatch = 8;
  const std::size_t from = kvh * kHeadDim, row = c.row;
  const bf16_bits *key = a.key + from, *value = a.value + from;
  bf16_bits *k = c.k, *v = c.v;
  for (std::uint32_t i0 = threadIdx.x; i0 < (t1 - t0) * 64; i0 += kBatch * kPThreads) { // 16 bytes; a token's K, then V
    u32x4 x[kBatch];
    const auto at = [&](int b) { return i0 + kPThreads * b < (t1 - t0) * 64 ? i0 + kPThreads * b : i0; };
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t i = at(b);
      x[b] = *reinterpret_cast<const u32x4 *>((i & 32 ? value : key) + static_cast<std::size_t>(t0 + i / 64) * a.kv_heads * kHeadDim + 8 * (i & 31));
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t i = at(b);
      *reinterpret_cast<u32x4 *>((i & 32 ? v : k) + static_cast<std::size_t>(a.past + t0 + i / 64) * row + 8 * (i & 31)) = x[b];
    }
  }
}

// Adds the infinite and NaN values of the masked tiles among begin, begin + stride, ..
// to the accumulators of a column that sees their keys (a positive probability times
// such a value is the value).  The lane has kQuads quads of its column's dims: quad i is
// dims 4 k + 256 / kQuads * i + 0 .. 3, and add(4 i + e, x) adds to one.
template <bool Fp8, int kQuads, class Add>
__device__ __forceinline__ void add_odd_values(const CompactHead<Fp8> &c, const SeenTiles &seen, std::uint32_t begin,
                                               std::uint32_t end, std::uint32_t stride, std::uint32_t p_lo, std::uint32_t p_hi,
                                               std::uint32_t pos, const CompactArgs &a, std::uint32_t kvh, int k, Add add) {
#pragma unroll 1
  for (std::uint32_t it = begin; it < end; it += stride) {
    const std::uint32_t j0 = seen.tile(it) * kCompactBlock;
    if (!tile_masked(j0, p_lo, p_hi, a.window, a.sinks)) continue;
#pragma unroll 1
    for (std::uint32_t j = j0; j < j0 + kCompactBlock && j <= p_hi; ++j) {
      if (!compact_sees(j, pos, a.window, a.sinks)) continue;
      const auto *row = reinterpret_cast<const typename CompactHead<Fp8>::T *>(KeyRows<Fp8>(a, c, kvh, j, true).at) + 4 * k;
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        floatx4 v;
        if constexpr (Fp8) {
          v = fp8x4_to_f32(*reinterpret_cast<const std::uint32_t *>(row + kHeadDim / kQuads * i));
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2 *>(row + kHeadDim / kQuads * i);
          v = floatx4{bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) add(4 * i + e, is_finite_f32(v[e]) ? 0.f : v[e]);
      }
    }
  }
}

// A workgroup takes 128 columns (column = token * group + head) of one KV head and a
// contiguous range of the 32-key tiles that they see; a wave takes 32 columns.  The
// tiles lie in two LDS slots as bf16, shared by the waves, and are asked for by
// LDS-direct loads a tile ahead: bf16 tiles in place, 8-bit tiles as codes, which each
// wave turns into bf16 times the block's scale (exact: 4 significant bits, a power of
// two) for the rows that it loaded.  S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_32x32x16_bf16, Q and O in registers.  A tile's softmax, one barrier, then
// its product with V and the next tile's scores in turn: two workgroups share a CU, so
// that one's softmax runs beside the other's products.
//
// 500 tokens of 16 heads behind 30001, 8 bit: 285 us, 870 TFLOP/s; 6001 behind a window of
// 1024, bf16, with the store: 152 us; 2001 with key weights 67 us.  An 8-bit tile takes a wave 4300 clocks,
// 1024 of them of matrix time (two waves a SIMD, 50% busy): by time stamps softmax 450, conversion
// 1000, barrier 200, products 2300, the rest between them; no waits for loads, no bank conflicts.  At
// 128 B a clock, and 64 of transposed reads, LDS needs 4100 clocks for the eight waves of a CU: V's
// operands 2048, K's 1024, codes in and out and bf16 tiles in 1024.  So it bounds the tile: every
// operand serves 32 columns only.  (64 columns a wave spilled with the accumulators left to the
// compiler.)  One workgroup of 256 columns per CU took 174 us for the window.
template <bool Fp8, bool Split, bool Weigh>
__global__ __launch_bounds__(kPThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void compact_prefill_kernel(
    CompactArgs a, PrefillScratch sc) {
  __shared__ __attribute__((aligned(1024))) PrefillShared<Fp8> sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kh = lane >> 5;
  // Longest column blocks first; but the first ranges shortest first, since nearly all ranges
  // run at once, two on a CU, and the later ranges, the long blocks', then come to the CUs
  // of the short blocks (2000 tokens 97.6 -> 90.1 us, 2000 behind 2000 167 -> 158, 3500 174 ->
  // 165, 1200 58 -> 60).
  const std::uint32_t place = Split && blockIdx.y == 0 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const std::uint32_t kvh = place % a.kv_heads;
  const std::uint32_t all_cols = a.tokens * a.group;
  const std::uint32_t blocks = (all_cols + kPCols - 1) / kPCols;
  const std::uint32_t col0 = (blocks - 1 - place / a.kv_heads) * kPCols;
  const std::uint32_t col_end = col0 + kPCols < all_cols ? col0 + kPCols : all_cols;
  const std::uint32_t p_lo = a.past + col0 / a.group, p_hi = a.past + (col_end - 1) / a.group;
  const std::uint32_t n_keys = p_hi + 1;
  const SeenTiles seen(p_lo, p_hi, a.window, a.sinks);
  std::uint32_t begin = 0, end = seen.total;
  bool part = false; // of several
  if constexpr (Split) {
    const TileRanges ranges(sc, seen.total);
    if (blockIdx.y >= ranges.count) return; // (uniform)
    begin = ranges.begin(blockIdx.y);
    end = ranges.begin(blockIdx.y + 1);
    part = ranges.count > 1;
  }
  const CompactHead<Fp8> c(a.cache, kvh, a.kv_heads, a.max_ctx, a.head_major);

  // This lane's column; those past the last repeat it.  (Formed anew where it is used:
  // the loop over the tiles needs every register.)
  const auto late_lane = [&] {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
  };
  const auto column = [&] { return col0 + 32 * wave + (late_lane() & 31); };
  const auto token_of = [&](std::uint32_t col) { return (col < all_cols ? col : all_cols - 1) / a.group; };
  const auto io_row = [&](std::uint32_t col) {
    const std::uint32_t in = col < all_cols ? col : all_cols - 1, tok = in / a.group;
    return (static_cast<std::size_t>(tok) * a.kv_heads + kvh) * a.group + (in - tok * a.group);
  };

  bf16x8 q[16];
  {
    const bf16_bits *src = a.query + io_row(column()) * kHeadDim + 8 * kh;
#pragma unroll
    for (int s = 0; s < 16; ++s) q[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(src + 16 * s));
  }

  // Loads of tile `it`'s K or V (a wave loads rows 8 wave .. + 7): rows past the last
  // key repeat it (their scores are masked).  In a whole tile the instructions' offsets
  // are the lane's, an exclusive-or (the rows' keys differ in bits of their own) and a
  // scalar.
  const auto load_tile = [&](std::uint32_t it, bool is_v) {
    const std::uint32_t j0 = seen.tile(it) * kCompactBlock;
    const std::uint32_t last = n_keys - 1 - j0; // >= 0: the tile has a key
    const KeyRows<Fp8> rows(a, c, kvh, j0, is_v);
    const unsigned char *tile = rows.at;
    const std::uint32_t row_bytes = rows.row_bytes;
    const int l = late_lane();
    constexpr int kInst = Fp8 ? 2 : 4, kRows = 8 / kInst; // rows an instruction
    const unsigned to = Fp8 ? lds_address(sh.raw) + (is_v ? kTileElems : 0) + 2048u * wave
                            : lds_address(is_v ? sh.v[(it - begin) & 1] : sh.k[(it - begin) & 1]) + 4096u * wave;
    const std::uint32_t in = l / (64 / kRows), chunk = l % (64 / kRows); // row and 16-byte chunk of instruction 0
    if (last >= kCompactBlock - 1) {
      const std::uint32_t off = in * row_bytes + 16u * (Fp8 ? chunk : chunk ^ row_key(8 * wave + in));
#pragma unroll
      for (int i = 0; i < kInst; ++i)
        load_lds_b128<0>(tile + (8u * wave + kRows * i) * row_bytes, Fp8 ? off : off ^ (16u * (8 * (i & 1) + (i >> 1))), to + 1024u * i);
    } else {
#pragma unroll
      for (int i = 0; i < kInst; ++i) {
        const std::uint32_t r = 8 * wave + kRows * i + in;
        load_lds_b128<0>(tile, (r < last ? r : last) * row_bytes + 16u * (Fp8 ? chunk : chunk ^ row_key(r)), to + 1024u * i);
      }
    }
  };
  // This wave's rows of tile `it`'s K or V have landed (the caller waits): 8-bit codes
  // become bf16 times the block's scale.  A masked key has
  // probability 0, and 0 times an infinite or NaN value is not 0: in V tiles that some
  // column does not see whole, such values are taken out here and added behind the
  // loop, to the columns that see their keys.
  std::uint64_t odd = 0; // lanes that took values out
  const auto finish_tile = [&](std::uint32_t it, bool is_v, [[maybe_unused]] float scale) {
    const int slot = (it - begin) & 1;
    const bool clean = is_v && tile_masked(seen.tile(it) * kCompactBlock, p_lo, p_hi, a.window, a.sinks);
    bf16_bits *tile = is_v ? sh.v[slot] : sh.k[slot];
    const int l = late_lane();
    if constexpr (Fp8) {
      // lane -> 8 dims (one bf16 chunk) of rows 2 i + lane / 32
      u32x2 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        raw[i] = *reinterpret_cast<const u32x2 *>(sh.raw + (is_v ? kTileElems : 0) + (8 * wave + 2 * i) * kHeadDim + 8 * l);
      const int at = (l & 31) ^ row_key(8 * wave + (l >> 5));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 x = fp8x8_to_bf16(raw[i][0], raw[i][1], scale);
        if (clean) odd |= __builtin_amdgcn_ballot_w64(without_odd(x));
        *reinterpret_cast<u32x4 *>(tile + (8 * wave + 2 * i + (l >> 5)) * kHeadDim + 8 * (at ^ (8 * (i & 1) + (i >> 1)))) = x;
      }
    } else if (clean) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 *mine = reinterpret_cast<u32x4 *>(tile + 2048 * wave + 512 * i + 8 * l);
        u32x4 w = *mine;
        const bool bad = without_odd(w);
        if (bad) *mine = w;
        odd |= __builtin_amdgcn_ballot_w64(bad);
      }
    }
  };

  // Operand addresses: K row n32, chunk 2 s + kh; V by transposed reads, where lane r
  // of a 16-lane group supplies 4 dims of key row r / 4 and receives its dim of 4 keys.
  // (Chunk numbers differ from a lane's first by an exclusive-or, or by 16.)
  const unsigned k_lane = 2 * tile_at(n32, kh);
  const int v_row = 4 * kh + ((lane & 15) >> 2);
  const unsigned v_lane = 2 * (tile_at(v_row, 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 4 * (lane & 1));

  floatx16 o[8];
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) o[nb] = floatx16{};
  float m_run = -FLT_MAX, l_run = 0.f;
  [[maybe_unused]] float lw_run = 0.f;

  const auto scale_of = [&](const float *scales, std::uint32_t it) {
    if constexpr (Fp8) return scales[seen.tile(it)]; // (a scalar load: no LDS reads are under way then)
    return 1.0f;
  };
  const auto k_addr = [&](std::uint32_t it) { return lds_address(sh.k[(it - begin) & 1]) + k_lane; };
  const auto read_k = [&](unsigned base, int i) { return lds_operand((base ^ (32u * (i >> 1))) + 256u * (i & 1)); }; // k-step i / 2 + 8 (i % 2)
  const auto read_v = [&](unsigned base, int i) { // key step i / 8, dims block i % 8
    // rows 8 apart have keys that differ in bit 1
    const unsigned at = 256u * ((i >> 2) & 1) + 8192u * (i >> 3);
    const u32x2 lo = lds_tr_operand((base ^ (64u * (i & 3))) + at), hi = lds_tr_operand((base ^ (64u * (i & 3) + 32u)) + (at + 4096u));
    return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
  };
  const auto q_of = [&](int i) -> const bf16x8 & { return q[(i >> 1) + 8 * (i & 1)]; };

  floatx16 s = floatx16{}; // scores of tile it: register i has key 8 (i / 4) + 4 kh + i % 4
  {
    load_tile(begin, false);
    load_tile(begin, true);
    const float ks = scale_of(c.ks, begin);
    if constexpr (!Fp8) {
      if (a.store_inside && (!Split || blockIdx.y == 0)) store_rows(a, c, kvh, col0, col_end);
    }
    wait_vm<0>();
    finish_tile(begin, false, ks);
    if (begin + 1 < end) load_tile(begin + 1, false);
    __syncthreads();
    // The waits for q belong here: left to the first use in the loop, they would be made on
    // every tile, for the tiles' loads too.
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(q[i]));
    const unsigned base = k_addr(begin);
#pragma unroll
    for (int i = 0; i < 16; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_k(base, i), q_of(i), s, 0, 0, 0);
  }
  // One tile; kMore: it is not the last.
  const auto step = [&]<bool kMore>(std::uint32_t it) __attribute__((always_inline)) {
    const std::uint32_t j0 = seen.tile(it) * kCompactBlock;
    [[maybe_unused]] const float vs = scale_of(c.vs, it), ks = kMore ? scale_of(c.ks, it + 1) : 1.0f;
    constexpr float kScale = kLog2e / 16.0f;
    if (tile_masked(j0, p_lo, p_hi, a.window, a.sinks)) { // some column does not see some key
      const int late = late_lane();
      const std::uint32_t pos = a.past + token_of(col0 + 32 * wave + (late & 31));
      const std::uint32_t j_lane = j0 + 4 * (late >> 5);
      if (a.window == 0) {
        const int lim = static_cast<int>(pos) - static_cast<int>(j_lane);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) <= lim ? s[i] : -INFINITY;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[i] = compact_sees(j_lane + 8 * (i >> 2) + (i & 3), pos, a.window, a.sinks) ? s[i] : -INFINITY;
      }
    }
    float mx = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[i]), s[i + 1]);
    mx = max_xor32(mx) * kScale;
    // m_run lies 2^8 above the max that it was last set to, and the accumulators are scaled
    // only where a max grows past it: no probability exceeds 1.
    const bool grow = mx > m_run;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float m_new = mx + kLazyRescale, f = grow ? fexp2(m_run - m_new) : 1.0f;
      l_run *= f;
      if constexpr (Weigh) lw_run *= f;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) o[nb] *= f;
      m_run = grow ? m_new : m_run;
    }
    // k-slot (kb, kh, e) of V^T P^T <-> key 16 kb + 8 (e / 4) + 4 kh + e % 4, the order of s.
    bf16x8 pb[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = fexp2(fmaf(s[8 * kb + 2 * e], kScale, -m_run)), p1 = fexp2(fmaf(s[8 * kb + 2 * e + 1], kScale, -m_run));
        const std::uint32_t pair = pack_bf16x2(p0, p1);
        w[e] = pair;
        l_run = dot2_bf16(pair, 0x3F803F80u, l_run); // (1, 1)
        if constexpr (Weigh) lw_run += p0 + p1;
      }
      pb[kb] = __builtin_bit_cast(bf16x8, w);
    }
    // V(it) and K(it + 1), asked for a tile ago
    wait_vm<0>();
    finish_tile(it, true, vs);
    if constexpr (Fp8 && kMore) finish_tile(it + 1, false, ks);
    __syncthreads(); // ... of every wave; and no wave reads V(it - 1) or K(it) any more
    const unsigned v_base = lds_address(sh.v[(it - begin) & 1]) + v_lane;
    if constexpr (kMore) {
      load_tile(it + 1, true);
      if (it + 2 < end) load_tile(it + 2, false);
      // O += V(it) P(it), then S(it + 1); operands are read kRing products ahead.
      const unsigned k_base = k_addr(it + 1);
      constexpr int kRing = 6;
      bf16x8 op[kRing];
#pragma unroll
      for (int i = 0; i < kRing; ++i) op[i] = read_v(v_base, i);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[i & 7] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[i % kRing], pb[i >> 3], o[i & 7], 0, 0, 0);
        op[i % kRing] = i + kRing < 16 ? read_v(v_base, i + kRing) : read_k(k_base, i + kRing - 16);
        __builtin_amdgcn_sched_barrier(0);
      }
      s = floatx16{};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[(i + 16) % kRing], q_of(i), s, 0, 0, 0);
        if (i + kRing < 16) op[(i + 16) % kRing] = read_k(k_base, i + kRing);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        o[i & 7] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_v(v_base, i), pb[i >> 3], o[i & 7], 0, 0, 0);
    }
  };
  for (std::uint32_t it = begin; it + 1 < end; ++it) step.template operator()<true>(it);
  step.template operator()<false>(end - 1);
  __syncthreads();

  const std::uint32_t col = column();
  // (the tiles' LDS is free)
  auto *odd_of = reinterpret_cast<std::uint32_t *>(&sh);
  if (lane == 0) odd_of[wave] = odd != 0;
  __syncthreads();
  if ((odd_of[0] | odd_of[1] | odd_of[2] | odd_of[3]) != 0)
    add_odd_values<Fp8, 32>(c, seen, begin, end, 1, p_lo, p_hi, a.past + token_of(col), a, kvh, kh,
                            [&](int i, float x) __attribute__((always_inline)) { o[i >> 4][i & 15] += x; });
  const float l = sum_xor32(l_run);
  [[maybe_unused]] const float lw = Weigh ? sum_xor32(lw_run) : 0.f;
  if (Split && part) {
    const std::size_t at = (static_cast<std::size_t>(blockIdx.y) * a.kv_heads + kvh) * sc.cols + col;
    if (kh == 0) {
      sc.m[at] = m_run;
      sc.l[at] = l;
      if constexpr (Weigh) sc.lw[at] = lw;
    }
    float *dst = sc.o + at * kHeadDim + 4 * kh;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<floatx4 *>(dst + 32 * nb + 8 * x) =
            floatx4{o[nb][4 * x], o[nb][4 * x + 1], o[nb][4 * x + 2], o[nb][4 * x + 3]};
  } else {
    if (col >= all_cols) return;
    const float inv = 1.0f / l;
    if (Weigh && kh == 0) {
      const std::size_t at = static_cast<std::size_t>(kvh) * sc.cols + col;
      sc.final[2 * at] = m_run;
      sc.final[2 * at + 1] = 1.0f / lw;
    }
    const std::size_t base = io_row(col) * kHeadDim + 4 * kh;
    u32x2 g[32]; // (every load before the first store, which it might alias)
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] = *reinterpret_cast<const u32x2 *>(a.gate + base + 8 * i);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int nb = i >> 2, x = 4 * (i & 3);
      const float r0 = o[nb][x] * inv * sigmoid_gate(bf16_lo(g[i][0])), r1 = o[nb][x + 1] * inv * sigmoid_gate(bf16_hi(g[i][0]));
      const float r2 = o[nb][x + 2] * inv * sigmoid_gate(bf16_lo(g[i][1])), r3 = o[nb][x + 3] * inv * sigmoid_gate(bf16_hi(g[i][1]));
      *reinterpret_cast<u32x2 *>(a.output + base + 8 * i) = u32x2{pack_bf16x2(r0, r1), pack_bf16x2(r2, r3)};
    }
  }
}

// The same for calls with too few columns to fill the chip by 128: a workgroup takes 32
// columns of one KV head, its waves take every fourth tile of the range by themselves and
// are joined in LDS.  Products on v_mfma_f32_16x16x32_bf16 with two blocks of 16 columns.
// K and V rows lie in LDS as they are in the cache (8-bit operands become bf16 behind the
// read; the block's scales go on the scores and on V's operands), asked for by
// LDS-direct loads of the wave's own kStages tiles ahead.
//
// 500 tokens of 16 heads, 8 bit: 17.4 us for 2.1 GFLOP, of which 3.4 until q and the first
// rows are there, 1.6 a tile (at one wave per SIMD, for 128 accumulators and q: products
// with K 860 clocks, softmax and the next loads' issue 1290, products with V and loads 1180),
// 3 for the join.  K and V through registers, as decode has them: 21.5.
constexpr int kKCols = 32;
struct KeysShared {
  union {
    unsigned char rows[kPWaves][4 * kTileElems]; // [stage][K, V], 16-byte chunks as keys_at
    // (the pad puts the 16 columns of a store on banks of their own)
    float acc[kPWaves][kKCols][kHeadDim + 4];
  };
  alignas(1024) bf16_bits gate[kPWaves][kKCols / kPWaves][kHeadDim];
  float m[kPWaves][kKCols], l[kPWaves][kKCols], lw[kPWaves][kKCols];
};
// What a row's number is exclusive-ored to its 16-byte chunks' places with (linear in the
// bits of r): a pass of the K reads takes one chunk of 16 rows, of the V reads
// 16 bytes of the 16 rows 4 k + 0 .. 3, 16 + 4 k + 0 .. 3 of two k (8 bit) or 32 of 8 rows.
template <bool Fp8> __device__ __forceinline__ constexpr std::uint32_t keys_at(std::uint32_t r, bool is_v) {
  if (!is_v) return r & 15;
  return Fp8 ? (r & 3) | (r >> 4 & 1) << 2 | (r >> 2 & 1) << 3 : 2 * (r & 7);
}
template <bool Fp8, bool Split, bool Weigh>
__global__ __launch_bounds__(kPThreads, 1) void compact_prefill_keys_kernel(
    CompactArgs a, PrefillScratch sc) {
  __shared__ __attribute__((aligned(1024))) KeysShared sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col16 = lane & 15, kq = lane >> 4;
  // grid (kv_heads, column blocks, splits)
  const std::uint32_t kvh = blockIdx.x;
  const std::uint32_t all_cols = a.tokens * a.group;
  const std::uint32_t col0 = (gridDim.y - 1 - blockIdx.y) * kKCols; // longest first
  const std::uint32_t last_x = all_cols - col0 < kKCols ? all_cols - col0 - 1 : kKCols - 1;
  // Column col0 + x (x < 32; those past the last repeat it) is head in_first + x - token_in(x)
  // * group of token first + token_in(x).  The quotient of n <= 46 and group <= 16 is
  // n (1024 / group + 1) >> 10, as 16 n < 1024.
  const std::uint32_t first = col0 / a.group, in_first = col0 - first * a.group, over = 1024 / a.group + 1;
  const auto token_in = [&](std::uint32_t x) { return ((x < last_x ? x : last_x) + in_first) * over >> 10; };
  const std::uint32_t p_lo = a.past + first, p_hi = p_lo + token_in(last_x);
  // First element of the column's row of query, gate and output, from `row0`.  (The launch
  // has at most 2^14 KV heads and a workgroup 47 rows between its tokens: 32 bits hold it.)
  const std::size_t row0 = (static_cast<std::size_t>(first) * a.kv_heads + kvh) * a.group * kHeadDim;
  const auto row_at = [&](std::uint32_t x) {
    const std::uint32_t tok = token_in(x);
    return (tok * (a.kv_heads - 1) * a.group + in_first + (x < last_x ? x : last_x)) * kHeadDim;
  };
  const SeenTiles seen(p_lo, p_hi, a.window, a.sinks);
  std::uint32_t begin = 0, end = seen.total;
  bool part = false; // of several
  if constexpr (Split) {
    const TileRanges ranges(sc, seen.total);
    if (blockIdx.z >= ranges.count) return; // (uniform)
    begin = ranges.begin(blockIdx.z);
    end = ranges.begin(blockIdx.z + 1);
    part = ranges.count > 1;
  }
  const CompactHead<Fp8> c(a.cache, kvh, a.kv_heads, a.max_ctx, a.head_major);

  // Steps: the wave's tiles.  LDS-direct loads of one plane of step t: rows past the last
  // key repeat it (their scores are masked).
  const std::uint32_t steps = begin + wave < end ? (end - begin - wave + kPWaves - 1) / kPWaves : 0;
  const auto tile_of = [&](std::uint32_t t) { return seen.tile(begin + wave + kPWaves * t); };
  constexpr int kStages = Fp8 ? 2 : 1;
  constexpr int kRowBytes = Fp8 ? 256 : 512, kRows = 1024 / kRowBytes; // rows of an instruction
  constexpr int kLoads = kCompactBlock / kRows;
  const unsigned rows_at = lds_address(sh.rows[wave]);
  const auto plane_at = [&](std::uint32_t t, bool is_v) {
    return rows_at + kRowBytes * kCompactBlock * (2 * (t % kStages) + is_v);
  };
  const std::uint32_t in_row = lane / (64 / kRows), chunk = lane % (64 / kRows);
  const auto load = [&](std::uint32_t t, bool is_v) __attribute__((always_inline)) {
    const std::uint32_t j0 = tile_of(t) * kCompactBlock, last = p_hi - j0; // >= 0: the tile has a key
    const KeyRows<Fp8> rows(a, c, kvh, j0, is_v);
    const unsigned char *tile = rows.at;
    const std::uint32_t row_bytes = rows.row_bytes;
    const unsigned to = plane_at(t, is_v);
    if (last >= kCompactBlock - 1) {
      const std::uint32_t off = in_row * row_bytes + 16 * (chunk ^ keys_at<Fp8>(in_row, is_v));
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        load_lds_b128<0>(tile + kRows * i * row_bytes, off ^ (16 * keys_at<Fp8>(kRows * i, is_v)), to + 1024 * i);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const std::uint32_t r = kRows * i + in_row;
        load_lds_b128<0>(tile, (r < last ? r : last) * row_bytes + 16 * (chunk ^ keys_at<Fp8>(r, is_v)), to + 1024 * i);
      }
    }
  };
  // Lane l: scales of step t0 + l.
  float ks_of = 1.0f, vs_of = 1.0f;
  const auto load_scales = [&](std::uint32_t t0) {
    if constexpr (Fp8) {
      const std::uint32_t t = t0 + lane < steps ? t0 + lane : steps - 1;
      ks_of = c.ks[tile_of(t)];
      vs_of = c.vs[tile_of(t)];
    }
  };
  const auto lane_value = [](float x, std::uint32_t l) {
    return __uint_as_float(static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(x)), l)));
  };

  // q of the lane's two columns, in the dims that its K operands hold.
  bf16x8 qb[2][8];
  std::uint32_t pos[2];
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    pos[cb] = p_lo + token_in(16 * cb + col16);
    const bf16_bits *q = a.query + row0 + row_at(16 * cb + col16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int dim = Fp8 ? 64 * (i >> 1) + 16 * kq + 8 * (i & 1) : 32 * i + 8 * kq;
      qb[cb][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(q + dim));
    }
  }
  if (steps != 0) {
    load_scales(0);
    load(0, false);
    load(0, true);
    if (kStages == 2 && steps > 1) {
      load(1, false);
      load(1, true);
    }
  }
  // The wave writes columns 4 i + wave: their gates, two at a time.
  if (!part) {
#pragma unroll
    for (int i = 0; i < kKCols / kPWaves; i += 2)
      load_lds_b128<0>(a.gate + row0, 2 * row_at(kPWaves * (i + (lane >> 5)) + wave) + 16 * (lane & 31), lds_address(sh.gate[wave][i]));
  }
  if constexpr (!Fp8) {
    if (a.store_inside && (!Split || blockIdx.z == 0)) store_rows(a, c, kvh, col0, col0 + last_x + 1);
  }
#pragma unroll
  for (int cb = 0; cb < 2; ++cb)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(qb[cb][i]));
  asm volatile("" : "+v"(ks_of), "+v"(vs_of));

  // K operands: row 16 rb + col16, chunk 4 i + kq.  V operands by transposed reads, k-slot
  // (kq, e) of the product <-> key 16 (e / 4) + 4 kq + e % 4, the order of the scores.
  const unsigned k_lane = kRowBytes * col16 + 16 * (kq ^ keys_at<Fp8>(col16, false));
  const std::uint32_t v_row = Fp8 ? 16 * (col16 >> 3) + 4 * kq + (col16 >> 1 & 3) : 4 * kq + (col16 >> 2);
  const unsigned v_lane = kRowBytes * v_row + (16 * ((Fp8 ? 0 : col16 >> 1 & 1) ^ keys_at<Fp8>(v_row, true)) + 8 * (col16 & 1));

  floatx4 acc[2][16]; // [column block][16 dims]: dims 16 db + 4 kq + e of the lane's column
#pragma unroll
  for (int cb = 0; cb < 2; ++cb)
#pragma unroll
    for (int db = 0; db < 16; ++db) acc[cb][db] = floatx4{};
  float m_run[2] = {-FLT_MAX, -FLT_MAX}, l_run[2] = {0.f, 0.f};
  [[maybe_unused]] float lw_run[2] = {0.f, 0.f};
  std::uint64_t odd = 0; // lanes that took infinite or NaN values out of a masked tile

#pragma unroll 1
  for (std::uint32_t t = 0; t < steps; ++t) {
    if (Fp8 && t % 64 == 0 && t != 0) {
      load_scales(t);
      asm volatile("" : "+v"(ks_of), "+v"(vs_of)); // (waited for here, not on every step)
    }
    const float k_scale = (Fp8 ? lane_value(ks_of, t % 64) : 1.0f) * (kLog2e / 16.0f);
    const float v_scale = Fp8 ? lane_value(vs_of, t % 64) : 1.0f;
    const std::uint32_t j0 = tile_of(t) * kCompactBlock;
    const bool masked = tile_masked(j0, p_lo, p_hi, a.window, a.sinks);
    // K(t): what may be under way behind it is V(t), K(t + 1), V(t + 1) (and the gates)
    if (kStages == 2 && t + 1 < steps) wait_vm<3 * kLoads>(); else wait_vm<kLoads>();
    floatx4 s[2][2]; // [column block][row block]: keys j0 + 16 rb + 4 kq + i
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) s[cb][rb] = floatx4{};
    const unsigned k_base = plane_at(t, false) + k_lane;
    const auto read_k = [&](int i) { return lds_operand((k_base ^ (64u * (i >> 1))) + 16 * kRowBytes * (i & 1)); };
    // (operands are read kRing products ahead: left to the compiler, one, and each waits)
    constexpr int kRing = 8;
    // 8-bit operands are converted between the products of the one before.
    const auto pair_of = [](std::uint32_t w, bool hi, float scale) {
      typedef __bf16 pair __attribute__((ext_vector_type(2)));
      const pair x = hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
      return __builtin_bit_cast(std::uint32_t, x);
    };
    {
      bf16x8 op[kRing];
#pragma unroll
      for (int i = 0; i < kRing; ++i) op[i] = read_k(i);
      if constexpr (Fp8) {
        // operand n: half n & 1 of read n / 2
        const auto code = [&](int n, int w) { return __builtin_bit_cast(u32x4, op[n >> 1])[2 * (n & 1) + w]; };
        u32x4 now{pair_of(code(0, 0), false, 1.0f), pair_of(code(0, 0), true, 1.0f), pair_of(code(0, 1), false, 1.0f), pair_of(code(0, 1), true, 1.0f)}, next = now;
#pragma unroll
        for (int n = 0; n < kRowBytes / 16; ++n) {
          const int rb = n >> 1 & 1, qi = 2 * (n >> 2) + (n & 1);
#pragma unroll
          for (int cb = 0; cb < 2; ++cb) {
            s[cb][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, now), qb[cb][qi], s[cb][rb], 0, 0, 0);
            if (n + 1 < kRowBytes / 16) {
              next[2 * cb] = pair_of(code(n + 1, cb), false, 1.0f);
              next[2 * cb + 1] = pair_of(code(n + 1, cb), true, 1.0f);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          now = next;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kRowBytes / 32; ++i) {
#pragma unroll
          for (int cb = 0; cb < 2; ++cb) s[cb][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op[i % kRing], qb[cb][i >> 1], s[cb][i & 1], 0, 0, 0);
          if (i + kRing < kRowBytes / 32) op[i % kRing] = read_k(i + kRing);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkm0(); // the reads are done: their place is free
    if (t + kStages < steps) load(t + kStages, false);
    if (masked) {
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[cb][rb][i] = compact_sees(j0 + 16 * rb + 4 * kq + i, pos[cb], a.window, a.sinks) ? s[cb][rb][i] : -INFINITY;
    }
    // m_run lies 2^8 above the max that it was last set to, and the accumulators are scaled
    // only where a max grows past it.  (Not at the max itself, which the probabilities could exceed by
    // 2^8: times the largest values that is no f32.)
    float mx[2];
    bool grow = false;
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      float x = fmaxf(s[cb][0][0], s[cb][1][0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) x = fmaxf(fmaxf(x, s[cb][0][i]), s[cb][1][i]);
      mx[cb] = max_xor32(max_xor16(x)) * k_scale;
      grow |= mx[cb] > m_run[cb];
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        const float m_new = mx[cb] > m_run[cb] ? mx[cb] + kLazyRescale : m_run[cb], f = fexp2(m_run[cb] - m_new);
        l_run[cb] *= f;
        if constexpr (Weigh) lw_run[cb] *= f;
#pragma unroll
        for (int db = 0; db < 16; ++db) {
          // (in accumulation registers but for here: moved out and in on every tile otherwise)
          floatx4 x = acc[cb][db];
          asm volatile("" : "+v"(x));
          x *= f;
          asm volatile("" : "+v"(x));
          acc[cb][db] = x;
        }
        m_run[cb] = m_new;
      }
    }
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int db = 0; db < 16; ++db) asm volatile("" : "+a"(acc[cb][db]));
    u32x4 pw[2];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = fexp2(fmaf(s[cb][rb][i], k_scale, -m_run[cb]));
          if constexpr (Weigh) lw_run[cb] += e[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          pw[cb][2 * rb + i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
          l_run[cb] = dot2_bf16(pw[cb][2 * rb + i], 0x3F803F80u, l_run[cb]); // (1, 1)
        }
      }
    // V(t): behind it K(t + 1) and, of two stages, V(t + 1) and K(t + 2)
    if (kStages == 2 && t + 2 < steps) wait_vm<3 * kLoads>();
    else if (t + 1 < steps) wait_vm<kStages * kLoads>();
    else wait_vm<0>();
    const unsigned v_plane = plane_at(t, true);
    if (masked) {
      // A masked key has probability 0, and 0 times an infinite or NaN value is not 0: such
      // values are taken out here and added behind the loop, to the columns that see them.
      // (A value is odd if its exponent's, or its code's, bits are all set.)
      constexpr std::uint32_t kOnes = Fp8 ? 0x7F7F7F7Fu : 0x7F807F80u, kOne = Fp8 ? 0x01010101u : 0x00800080u;
      std::uint32_t carry = 0;
#pragma unroll 4
      for (int i = 0; i < kLoads; ++i) {
        const u32x4 w = __builtin_bit_cast(u32x4, lds_operand(v_plane + 1024 * i + 16 * lane));
#pragma unroll
        for (int e = 0; e < 4; ++e) carry |= (w[e] & kOnes) + kOne;
      }
      const std::uint64_t bad = __builtin_amdgcn_ballot_w64((carry & 0x80808080u & ~kOnes) != 0);
      if (bad != 0) {
        odd |= bad;
#pragma unroll 1
        for (int i = 0; i < kLoads; ++i) {
          const unsigned at = v_plane + 1024 * i + 16 * lane;
          u32x4 w = __builtin_bit_cast(u32x4, lds_operand(at));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const std::uint32_t top = ((w[e] & kOnes) + kOne) & 0x80808080u & ~kOnes;
            // all bits of the values whose top bit is set
            w[e] &= ~(Fp8 ? (top >> 7) * 0xFFu : (top >> 15) * 0xFFFFu);
          }
          *(__attribute__((address_space(3))) u32x4 *)(std::uintptr_t)(at) = w;
        }
      }
      wave_lds_order();
    }
    const unsigned v_base = v_plane + v_lane;
    const auto read_v = [&](int db) {
      if constexpr (Fp8) {
        return lds_tr8_operand(v_base ^ (16u * db));
      } else {
        const u32x2 lo = lds_tr_operand(v_base ^ (32u * db)), hi = lds_tr_operand((v_base ^ (32u * db)) + 16 * kRowBytes);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    std::conditional_t<Fp8, u32x2, u32x4> op[kRing];
#pragma unroll
    for (int db = 0; db < kRing; ++db) op[db] = read_v(db);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 now;
    if constexpr (Fp8) now = u32x4{pair_of(op[0][0], false, v_scale), pair_of(op[0][0], true, v_scale), pair_of(op[0][1], false, v_scale), pair_of(op[0][1], true, v_scale)};
#pragma unroll
    for (int db = 0; db < 16; ++db) {
      if constexpr (!Fp8) now = op[db % kRing];
      u32x4 next = now;
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        acc[cb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, now), __builtin_bit_cast(bf16x8, pw[cb]), acc[cb][db], 0, 0, 0);
        if (Fp8 && db + 1 < 16) {
          next[2 * cb] = pair_of(op[(db + 1) % kRing][cb], false, v_scale);
          next[2 * cb + 1] = pair_of(op[(db + 1) % kRing][cb], true, v_scale);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (db + kRing < 16) op[db % kRing] = read_v(db + kRing);
      now = next;
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkm0();
    if (t + kStages < steps) load(t + kStages, true);
  }
  if (odd != 0) {
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
      add_odd_values<Fp8, 16>(c, seen, begin + wave, end, kPWaves, p_lo, p_hi, pos[cb], a, kvh, kq,
                              [&](int i, float x) __attribute__((always_inline)) { acc[cb][i >> 2][i & 3] += x; });
  }

  // Join the waves: a wave takes every fourth column, a lane four dims.
  wait_vm<0>();
  __syncthreads();
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    const float l = sum_xor32(sum_xor16(l_run[cb]));
    [[maybe_unused]] const float lw = Weigh ? sum_xor32(sum_xor16(lw_run[cb])) : 0.f;
    if (kq == 0) {
      sh.m[wave][16 * cb + col16] = m_run[cb];
      sh.l[wave][16 * cb + col16] = l;
      if constexpr (Weigh) sh.lw[wave][16 * cb + col16] = lw;
    }
#pragma unroll
    for (int db = 0; db < 16; ++db) *reinterpret_cast<floatx4 *>(&sh.acc[wave][16 * cb + col16][16 * db + 4 * kq]) = acc[cb][db];
  }
  __syncthreads();
  // Lane x, and x + 32: the waves' shares of column x.
  float m = -FLT_MAX, l = 0.f, share[kPWaves];
  [[maybe_unused]] float lw = 0.f;
#pragma unroll
  for (int w = 0; w < kPWaves; ++w) m = fmaxf(m, sh.m[w][lane & 31]);
#pragma unroll
  for (int w = 0; w < kPWaves; ++w) {
    share[w] = fexp2(sh.m[w][lane & 31] - m);
    l = fmaf(sh.l[w][lane & 31], share[w], l);
    if constexpr (Weigh) lw = fmaf(sh.lw[w][lane & 31], share[w], lw);
  }
  if (Split && part) {
    const std::size_t at = (static_cast<std::size_t>(blockIdx.z) * a.kv_heads + kvh) * sc.cols + col0;
    if (threadIdx.x < kKCols) {
      sc.m[at + lane] = m;
      sc.l[at + lane] = l;
      if constexpr (Weigh) sc.lw[at + lane] = lw;
    }
#pragma unroll
    for (int i = 0; i < kKCols / kPWaves; ++i) {
      const int x = kPWaves * i + wave;
      floatx4 o{};
#pragma unroll
      for (int w = 0; w < kPWaves; ++w) o += *reinterpret_cast<const floatx4 *>(&sh.acc[w][x][4 * lane]) * lane_value(share[w], x);
      *reinterpret_cast<floatx4 *>(sc.o + (at + x) * kHeadDim + 4 * lane) = o;
    }
  } else {
    const float inv = 1.0f / l;
    if (Weigh && threadIdx.x <= last_x) {
      const std::size_t at = static_cast<std::size_t>(kvh) * sc.cols + col0 + lane;
      sc.final[2 * at] = m;
      sc.final[2 * at + 1] = 1.0f / lw;
    }
    u32x2 out[kKCols / kPWaves];
#pragma unroll
    for (int i = 0; i < kKCols / kPWaves; ++i) {
      const int x = kPWaves * i + wave;
      floatx4 o{};
#pragma unroll
      for (int w = 0; w < kPWaves; ++w) o += *reinterpret_cast<const floatx4 *>(&sh.acc[w][x][4 * lane]) * lane_value(share[w] * inv, x);
      const u32x2 g = *reinterpret_cast<const u32x2 *>(&sh.gate[wave][i][4 * lane]);
      out[i] = u32x2{pack_bf16x2(o[0] * sigmoid_gate(bf16_lo(g[0])), o[1] * sigmoid_gate(bf16_hi(g[0]))),
                     pack_bf16x2(o[2] * sigmoid_gate(bf16_lo(g[1])), o[3] * sigmoid_gate(bf16_hi(g[1])))};
    }
#pragma unroll
    for (int i = 0; i < kKCols / kPWaves; ++i)
      if (kPWaves * i + wave <= static_cast<int>(last_x))
        *reinterpret_cast<u32x2 *>(a.output + row0 + row_at(kPWaves * i + wave) + 4 * lane) = out[i];
  }
}

// Joins the ranges of the columns that have several: W waves per column take them in
// turn, eight loads of a partial row at a time in flight, a lane four dims.  Bound by
// memory where there are many (500 tokens of 16 heads in 8 ranges: 74 MB, 15.5 us), else by
// its round trips (16 tokens in 40: 4.3 us).
template <int W>
__global__ __launch_bounds__(kPThreads) void compact_prefill_merge_kernel(CompactArgs a, PrefillScratch sc) {
  __shared__ float o_of[kPWaves][kHeadDim];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::uint32_t all_cols = a.tokens * a.group;
  const std::uint32_t col_of = blockIdx.x * (kPWaves / W) + wave / W;
  const std::uint32_t col = col_of < all_cols ? col_of : all_cols - 1;
  const std::uint32_t kvh = blockIdx.y;
  const std::uint32_t first = col - col % sc.block, last = first + sc.block < all_cols ? first + sc.block - 1 : all_cols - 1;
  const std::uint32_t splits =
      TileRanges(sc, SeenTiles(a.past + first / a.group, a.past + last / a.group, a.window, a.sinks).total).count;
  if (splits == 1) return; // (for W > 1 the whole workgroup)
  const std::size_t stride = static_cast<std::size_t>(a.kv_heads) * sc.cols; // between splits
  const std::size_t at0 = static_cast<std::size_t>(kvh) * sc.cols + col;
  const std::uint32_t tok = col / a.group;
  const std::size_t out_at =
      ((static_cast<std::size_t>(tok) * a.kv_heads + kvh) * a.group + (col - tok * a.group)) * kHeadDim + 4 * lane;
  const u32x2 g = *reinterpret_cast<const u32x2 *>(a.gate + out_at);
  constexpr int kBatch = 8;
  floatx4 x[kBatch];
  const auto load = [&](std::uint32_t s0) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t s = s0 + W * b < splits ? s0 + W * b : splits - 1;
      x[b] = *reinterpret_cast<const floatx4 *>(sc.o + (at0 + s * stride) * kHeadDim + 4 * lane);
    }
  };
  const std::uint32_t s_first = W == 1 ? 0 : wave % W;
  load(s_first);
  // max and sum over the splits; those without a key that the column sees have l = 0
  float m = -FLT_MAX, l = 0.f, lw = 0.f;
  for (std::uint32_t s = lane; s < splits; s += 64) {
    const float ms = sc.m[at0 + s * stride], ls = sc.l[at0 + s * stride];
    const float lws = a.weights != nullptr ? sc.lw[at0 + s * stride] : 0.f;
    const float m_new = fmaxf(m, ms), f = fexp2(m - m_new), fs = fexp2(ms - m_new);
    l = l * f + ls * fs;
    lw = lw * f + lws * fs;
    m = m_new;
  }
  const float m_all = wave_max(m);
  const float inv = 1.0f / wave_sum(l * fexp2(m - m_all));
  floatx4 o{};
  for (std::uint32_t s0 = s_first; s0 < splits; s0 += W * kBatch) {
    if (s0 != s_first) load(s0);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t s = s0 + W * b;
      if (s >= splits) break;
      const float ms = sc.m[at0 + s * stride];
      if (ms == -FLT_MAX && sc.l[at0 + s * stride] == 0.f) continue; // nothing was summed
      o += x[b] * fexp2(ms - m_all);
    }
  }
  if constexpr (W > 1) {
    *reinterpret_cast<floatx4 *>(&o_of[wave][4 * lane]) = o;
    __syncthreads();
    if (wave % W != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) o += *reinterpret_cast<const floatx4 *>(&o_of[wave + w][4 * lane]);
  }
  if (col_of >= all_cols) return;
  if (a.weights != nullptr) {
    const float all = wave_sum(lw * fexp2(m - m_all));
    if (lane == 0) {
      sc.final[2 * at0] = m_all;
      sc.final[2 * at0 + 1] = 1.0f / all;
    }
  }
  const float r0 = o[0] * inv * sigmoid_gate(bf16_lo(g[0])), r1 = o[1] * inv * sigmoid_gate(bf16_hi(g[0]));
  const float r2 = o[2] * inv * sigmoid_gate(bf16_lo(g[1])), r3 = o[3] * inv * sigmoid_gate(bf16_hi(g[1]));
  *reinterpret_cast<u32x2 *>(a.output + out_at) = u32x2{pack_bf16x2(r0, r1), pack_bf16x2(r2, r3)};
}

// Key weights of the last `observed` tokens: a workgroup owns a 32-key tile of one KV
// head, its 8 waves take every eighth block of 32 observed columns and form the
// probabilities again from the columns' final max and sum.  The owner sums them, so
// nothing is added twice or in a changing order.  64 tokens over 2001 keys: 10.6 us, round
// trips (q and the sums, K, the weights) and a wave's chain of products; 11.7 with 4 waves.
constexpr int kWeighWaves = 8;
constexpr std::uint32_t kWeighGrid = 1u << 22; // tiles of a launch: fewer than 2^32 threads in x
template <bool Fp8>
__global__ __launch_bounds__(kWeighWaves *kWave, 1) void compact_prefill_weigh_kernel(CompactArgs a, PrefillScratch sc,
                                                                                           std::uint32_t before) {
  __shared__ float sum[kWeighWaves][kCompactBlock];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, kh = lane >> 5;
  const std::uint32_t kvh = blockIdx.y;
  const std::uint32_t last = a.past + a.tokens - 1;
  const SeenTiles seen(a.past + a.tokens - a.observed, last, a.window, a.sinks);
  const std::uint32_t tile = seen.tile(before + blockIdx.x), j0 = tile * kCompactBlock;
  const CompactHead<Fp8> c(a.cache, kvh, a.kv_heads, a.max_ctx, a.head_major);
  float k_scale = kLog2e / 16.0f;
  if constexpr (Fp8) k_scale *= c.ks[tile];
  const std::uint32_t all_cols = a.tokens * a.group;
  std::uint32_t c0 = (a.tokens - a.observed) * a.group + 32 * wave;
  bf16x8 k[16], q[16];
  float m = 0.f, inv = 0.f;
  std::uint32_t pos = 0;
  const auto load = [&] { // a block's columns: those past the last repeat it
    const std::uint32_t col = c0 + n32 < all_cols ? c0 + n32 : all_cols - 1, tok = col / a.group;
    pos = a.past + tok;
    const bf16_bits *src =
        a.query + ((static_cast<std::size_t>(tok) * a.kv_heads + kvh) * a.group + (col - tok * a.group)) * kHeadDim + 8 * kh;
#pragma unroll
    for (int b = 0; b < 16; ++b) q[b] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(src + 16 * b));
    const std::size_t at = static_cast<std::size_t>(kvh) * sc.cols + col;
    m = sc.final[2 * at];
    inv = sc.final[2 * at + 1];
  };
  if (c0 < all_cols) load();
  {
    const std::uint32_t j = j0 + n32 <= last ? j0 + n32 : last;
    const auto *row = c.k + static_cast<std::size_t>(j) * c.row + 8 * kh;
#pragma unroll
    for (int s = 0; s < 16; ++s) {
      if constexpr (Fp8) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(row + 16 * s);
        k[s] = __builtin_bit_cast(bf16x8, fp8x8_to_bf16(w[0], w[1]));
      } else {
        k[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(row + 16 * s));
      }
    }
  }
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = 0.f;
  for (; c0 < all_cols;) {
    const bool real = c0 + n32 < all_cols;
    floatx16 s = floatx16{}, s1 = floatx16{}; // (two chains)
#pragma unroll
    for (int b = 0; b < 16; b += 2) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[b], q[b], s, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[b + 1], q[b + 1], s1, 0, 0, 0);
    }
    s += s1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const std::uint32_t j = j0 + 8 * (i >> 2) + 4 * kh + (i & 3);
      w[i] += real && compact_sees(j, pos, a.window, a.sinks) ? fexp2(s[i] * k_scale - m) * inv : 0.f;
    }
    c0 += 32 * kWeighWaves;
    if (c0 < all_cols) load();
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = sum_xor16(row16_sum(w[i])); // over the 32 columns
    if (n32 == 0) sum[wave][8 * (i >> 2) + 4 * kh + (i & 3)] = w[i];
  }
  __syncthreads();
  if (threadIdx.x < kCompactBlock && j0 + threadIdx.x <= last) {
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < kWeighWaves; ++i) all += sum[i][threadIdx.x];
    a.weights[static_cast<std::size_t>(kvh) * a.max_ctx + j0 + threadIdx.x] += all;
  }
}

std::uint32_t col_blocks(const CompactArgs &a) { return (a.tokens * a.group + kPCols - 1) / kPCols; }
std::uint32_t key_col_blocks(const CompactArgs &a) { return (a.tokens * a.group + kKCols - 1) / kKCols; }

// How a call is run.  All figures: 4 KV heads of 4 query heads, 8 bit (bf16), store and
// merge included.
//
// Little work: waves that split the tiles, in ranges of at least 16 tiles until every CU has
// a workgroup.  The measure is (32 columns, tile) per CU, up to 40 of 8 bit or 32 of bf16.
// Against tiles shared by 128 columns: 500 tokens 26.9 us (27.8) for 36.9 (36.1), 128 tokens
// 19.0 (20.1) for 26.6 (26.2), 10 behind 100 18.9 (19.7) for 22.0 (21.1), 2 behind 30000 33.5
// (44.6) for 48.3 (54.5), 1000 tokens (32 per CU) 43.4 (45.6) for 54.2 (52.0), 500 behind
// 1000 (40) 41.1 (42.4) for 47.7 (45.0); 1000 behind a window of 500 (35) 47.3 (49.7) for
// 47.3 (46.3), 300 behind a window of 2048 (41) 51.8 for 48.3, 1200 tokens (45) 57.8 (60.6)
// for 59.6 (56.6), 500 behind 4000 (130) 82.1 (85.5) for 77.3 (75.2).  Ranges of 8, 16 and 32
// tiles: 2 behind 30000 34.1 / 33.5 / 36.5 us, 64 behind 4000 31.2 / 31.5 / 37.1.
//
// Else two workgroups of 128 columns per CU where each has 16 tiles in the mean, or one per
// CU, of at least four tiles.  Two overlap softmax and products but leave more partial rows
// to be joined (one against two: 500 behind 2000, 10 tiles at two, 58.1 against 61.8 us,
// behind 4000, 18 tiles, 79.1 against 77.5, 3000 tokens 164 (145) against 137 (131)).  A
// column block is cut into as many ranges as its own tiles need: a prompt's first ones into
// one, which is not joined (1400 tokens 67.3 us, all blocks cut alike 82.6).
struct PrefillSplit {
  bool by_keys;        // compact_prefill_keys_kernel
  std::uint32_t count; // ranges of the longest column block
  std::uint32_t tiles; // of a range
};
PrefillSplit split_of(const CompactArgs &a, bool fp8, std::uint32_t past) {
  const std::uint32_t last = past + a.tokens - 1;
  // about the tiles of the last block, which has the most
  const std::uint32_t span = (kPCols + a.group - 1) / a.group + 1;
  const std::uint32_t tiles = SeenTiles(a.tokens > span ? last - span + 1 : past, last, a.window, a.sinks).total;
  const std::uint32_t fewest = std::min(SeenTiles(past, past, a.window, a.sinks).total, tiles);
  // in the mean: they grow over the tokens that see the first key
  const std::uint64_t reach = static_cast<std::uint64_t>(a.window) + a.sinks;
  const std::uint64_t growing = a.window == 0 ? a.tokens : std::min<std::uint64_t>(reach > past ? reach - past : 0, a.tokens);
  const double mean = tiles - 0.5 * (tiles - fewest) * static_cast<double>(growing) / a.tokens;
  const double small = static_cast<double>(key_col_blocks(a)) * a.kv_heads * mean; // (32 columns, tile)
  const double wide = static_cast<double>(col_blocks(a)) * a.kv_heads * mean;
  const auto ranges = [&](bool by_keys, double work, double workgroups, std::uint32_t least) {
    const double wanted = std::max(1.0, workgroups * tiles / work); // of the longest block
    const std::uint32_t most = (tiles + least - 1) / least;
    const auto n = wanted < most ? static_cast<std::uint32_t>(wanted) : most;
    return PrefillSplit{by_keys, n, (tiles + n - 1) / n};
  };
  if (small <= kPrefillCus * (fp8 ? 40.0 : 32.0)) return ranges(true, small, kPrefillCus, 16);
  return ranges(false, wide, wide >= 2 * kPrefillCus * 16.0 ? 2 * kPrefillCus : kPrefillCus, 4);
}
// The ranges that the workspace holds: what a prompt's start or its end in a full cache
// takes, whichever type it has.  (A call between them that would take more takes these.)
std::uint32_t most_ranges(const CompactArgs &a) {
  std::uint32_t most = 1;
  for (const std::uint32_t past : {0u, a.max_ctx - a.tokens})
    for (const bool fp8 : {false, true}) most = std::max(most, split_of(a, fp8, past).count);
  return most;
}

PrefillScratch scratch_of(const CompactArgs &a, std::uint32_t ranges, void *workspace, std::size_t *bytes) {
  PrefillScratch sc{};
  sc.cols = col_blocks(a) * kPCols;
  auto *p = static_cast<unsigned char *>(workspace);
  std::size_t at = 0;
  const auto take = [&](std::size_t floats) {
    auto *q = reinterpret_cast<float *>(p + at);
    at += (floats * sizeof(float) + 15) / 16 * 16;
    return q;
  };
  const std::size_t cols = static_cast<std::size_t>(sc.cols) * a.kv_heads;
  if (a.observed != 0) sc.final = take(2 * cols);
  if (ranges > 1) {
    sc.m = take(ranges * cols);
    sc.l = take(ranges * cols);
    if (a.observed != 0) sc.lw = take(ranges * cols);
    sc.o = take(ranges * cols * kHeadDim);
  }
  if (bytes != nullptr) *bytes = at;
  return sc;
}

template <bool Fp8> void launch_prefill(const CompactArgs &a, void *workspace, hipStream_t stream) {
  PrefillSplit split = split_of(a, Fp8, a.past);
  split.count = std::min(split.count, most_ranges(a));
  PrefillScratch sc = scratch_of(a, split.count, workspace, nullptr);
  sc.block = split.by_keys ? kKCols : kPCols;
  sc.tiles = split.tiles;
  sc.most = split.count;
  const dim3 grid{col_blocks(a) * a.kv_heads, split.count}, keys_grid{a.kv_heads, key_col_blocks(a), split.count};
  const auto launch = [&](auto several) {
    if (split.by_keys && a.weights != nullptr)
      compact_prefill_keys_kernel<Fp8, several, true><<<keys_grid, kPThreads, 0, stream>>>(a, sc);
    else if (split.by_keys)
      compact_prefill_keys_kernel<Fp8, several, false><<<keys_grid, kPThreads, 0, stream>>>(a, sc);
    else if (a.weights != nullptr)
      compact_prefill_kernel<Fp8, several, true><<<grid, kPThreads, 0, stream>>>(a, sc);
    else
      compact_prefill_kernel<Fp8, several, false><<<grid, kPThreads, 0, stream>>>(a, sc);
  };
  if (split.count > 1) {
    launch(std::true_type{});
    const std::uint32_t cols = a.tokens * a.group;
    if (split.count > 8)
      compact_prefill_merge_kernel<kPWaves><<<dim3{cols, a.kv_heads}, kPThreads, 0, stream>>>(a, sc);
    else
      compact_prefill_merge_kernel<1><<<dim3{(cols + kPWaves - 1) / kPWaves, a.kv_heads}, kPThreads, 0, stream>>>(a, sc);
  } else {
    launch(std::false_type{});
  }
  const std::uint32_t last = a.past + a.tokens - 1;
  if (a.weights != nullptr) {
    const SeenTiles seen(last + 1 - a.observed, last, a.window, a.sinks);
    for (std::uint32_t before = 0; before < seen.total; before += kWeighGrid)
      compact_prefill_weigh_kernel<Fp8><<<dim3{std::min(seen.total - before, kWeighGrid), a.kv_heads}, kWeighWaves * kWave, 0, stream>>>(a, sc, before);
  }
}

} // namespace

std::size_t compact_prefill_workspace(const CompactArgs &a) {
  std::size_t bytes = 0;
  (void)scratch_of(a, most_ranges(a), nullptr, &bytes);
  return bytes;
}

// 8-bit rows, and bf16 rows that begin inside a tile, are stored by a launch of their own.
// (Inside, in a graph: 128 tokens 15.4 us for 19.4, 500 22.9 for 26.8, 6001 behind a window of
// 1024 156.7 for 161.)
void compact_prefill(CompactArgs a, bool fp8, void *workspace, hipStream_t stream) {
  a.store_inside = !fp8 && a.past % kCompactBlock == 0;
  if (!a.store_inside) compact_append(a, fp8, stream);
  if (fp8) launch_prefill<true>(a, workspace, stream);
  else launch_prefill<false>(a, workspace, stream);
}

} // namespace raftinfer::amd
