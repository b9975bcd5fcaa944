// Prompt attention over the compact KV cache, and the key weights of its last
// tokens.
#include "compact_cache.hpp"
#include "prefill_tile.hpp"

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
// domain) and 1 / sum of each column for the key weights.
struct PrefillScratch {
  float *m, *l, *o, *final;
  std::uint32_t splits, cols; // cols: rounded up to whole workgroups
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

// Adds the infinite and NaN values of the masked tiles to the accumulators of the
// columns that see their keys (a positive probability times such a value is the
// value).  Register 4 x + e of o[nb] is dim 32 nb + 8 x + 4 kh + e of the lane's column.
template <bool Fp8>
__device__ __forceinline__ void add_odd_values(const CompactHead<Fp8> &c, const SeenTiles &seen, std::uint32_t begin,
                                               std::uint32_t end, std::uint32_t p_lo, std::uint32_t p_hi, std::uint32_t pos,
                                               std::uint32_t window, std::uint32_t sinks, std::uint32_t n_keys, int kh,
                                               floatx16 (&o)[8]) {
#pragma unroll 1
  for (std::uint32_t it = begin; it < end; ++it) {
    const std::uint32_t j0 = seen.tile(it) * kCompactBlock;
    if (!tile_masked(j0, p_lo, p_hi, window, sinks)) continue;
#pragma unroll 1
    for (std::uint32_t j = j0; j < j0 + kCompactBlock && j < n_keys; ++j) {
      if (!compact_sees(j, pos, window, sinks)) continue;
      const auto *row = c.v + static_cast<std::size_t>(j) * c.row + 4 * kh;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          floatx4 v;
          if constexpr (Fp8) {
            v = fp8x4_to_f32(*reinterpret_cast<const std::uint32_t *>(row + 32 * nb + 8 * x));
          } else {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(row + 32 * nb + 8 * x);
            v = floatx4{bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nb][4 * x + e] += is_finite_f32(v[e]) ? 0.f : v[e];
        }
    }
  }
}
__device__ __forceinline__ u32x4 fp8x8_to_bf16_scaled(std::uint32_t lo, std::uint32_t hi, float scale) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const pair b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const pair c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const pair d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return u32x4{__builtin_bit_cast(std::uint32_t, a), __builtin_bit_cast(std::uint32_t, b),
               __builtin_bit_cast(std::uint32_t, c), __builtin_bit_cast(std::uint32_t, d)};
}
__device__ __forceinline__ bf16x8 lds_operand(unsigned addr) {
  return __builtin_bit_cast(bf16x8, *(const __attribute__((address_space(3))) u32x4 *)(std::uintptr_t)(addr));
}
__device__ __forceinline__ u32x2 lds_tr_operand(unsigned addr) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((prefill::lds_short4v *)(std::uintptr_t)(addr)));
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
template <bool Fp8, bool Split, bool Weigh>
__global__ __launch_bounds__(kPThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void compact_prefill_kernel(
    CompactArgs a, PrefillScratch sc) {
  __shared__ __attribute__((aligned(1024))) PrefillShared<Fp8> sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kh = lane >> 5;
  const std::uint32_t kvh = blockIdx.x % a.kv_heads;
  const std::uint32_t all_cols = a.tokens * a.group;
  const std::uint32_t blocks = (all_cols + kPCols - 1) / kPCols;
  const std::uint32_t col0 = (blocks - 1 - blockIdx.x / a.kv_heads) * kPCols; // longest first
  const std::uint32_t col_end = col0 + kPCols < all_cols ? col0 + kPCols : all_cols;
  const std::uint32_t p_lo = a.past + col0 / a.group, p_hi = a.past + (col_end - 1) / a.group;
  const std::uint32_t n_keys = p_hi + 1;
  const SeenTiles seen(p_lo, p_hi, a.window, a.sinks);
  const std::uint32_t begin = Split ? static_cast<std::uint32_t>(static_cast<std::uint64_t>(seen.total) * blockIdx.y / sc.splits) : 0;
  const std::uint32_t end = Split ? static_cast<std::uint32_t>(static_cast<std::uint64_t>(seen.total) * (blockIdx.y + 1) / sc.splits) : seen.total;
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
  const std::uint32_t row_bytes = static_cast<std::uint32_t>(c.row * sizeof(typename CompactHead<Fp8>::T));
  const auto load_tile = [&](std::uint32_t it, bool is_v) {
    const std::uint32_t j0 = seen.tile(it) * kCompactBlock;
    const std::uint32_t last = n_keys - 1 - j0; // >= 0: the tile has a key
    const auto *tile = reinterpret_cast<const unsigned char *>((is_v ? c.v : c.k) + static_cast<std::size_t>(j0) * c.row);
    const int l = late_lane();
    constexpr int kInst = Fp8 ? 2 : 4, kRows = 8 / kInst; // rows an instruction
    const unsigned to = Fp8 ? lds_address(sh.raw) + (is_v ? kTileElems : 0) + 2048u * wave
                            : lds_address(is_v ? sh.v[(it - begin) & 1] : sh.k[(it - begin) & 1]) + 4096u * wave;
    const std::uint32_t in = l / (64 / kRows), chunk = l % (64 / kRows); // row and 16-byte chunk of instruction 0
    if (last >= kCompactBlock - 1) {
      const std::uint32_t off = in * row_bytes + 16u * (Fp8 ? chunk : chunk ^ row_key(8 * wave + in));
#pragma unroll
      for (int i = 0; i < kInst; ++i)
        load_lds_b128(tile + (8u * wave + kRows * i) * row_bytes, Fp8 ? off : off ^ (16u * (8 * (i & 1) + (i >> 1))), to + 1024u * i);
    } else {
#pragma unroll
      for (int i = 0; i < kInst; ++i) {
        const std::uint32_t r = 8 * wave + kRows * i + in;
        load_lds_b128(tile, (r < last ? r : last) * row_bytes + 16u * (Fp8 ? chunk : chunk ^ row_key(r)), to + 1024u * i);
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
        u32x4 x = fp8x8_to_bf16_scaled(raw[i][0], raw[i][1], scale);
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
  if (begin < end) {
    load_tile(begin, false);
    load_tile(begin, true);
    const float ks = scale_of(c.ks, begin);
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
    // The accumulators are scaled only where a max grows by more than 2^8, which
    // the probabilities can exceed 1 by.
    const bool grow = mx > m_run + kLazyRescale;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float f = grow ? fexp2(m_run - mx) : 1.0f;
      l_run *= f;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) o[nb] *= f;
      m_run = grow ? mx : m_run;
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
        // The sum is that of the rounded probabilities, with which the output is a convex
        // combination of the V rows; key weights need the exact one.
        if constexpr (Weigh) l_run += p0 + p1; else l_run = dot2_bf16(pair, 0x3F803F80u, l_run);
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
  if (begin < end) {
    for (std::uint32_t it = begin; it + 1 < end; ++it) step.template operator()<true>(it);
    step.template operator()<false>(end - 1);
  }
  __syncthreads();

  const std::uint32_t col = column();
  // (the tiles' LDS is free)
  auto *odd_of = reinterpret_cast<std::uint32_t *>(&sh);
  if (lane == 0) odd_of[wave] = odd != 0;
  __syncthreads();
  if ((odd_of[0] | odd_of[1] | odd_of[2] | odd_of[3]) != 0) add_odd_values<Fp8>(c, seen, begin, end, p_lo, p_hi, a.past + token_of(col), a.window, a.sinks, n_keys, kh, o);
  const float l = sum_xor32(l_run);
  if constexpr (Split) {
    const std::size_t at = (static_cast<std::size_t>(blockIdx.y) * a.kv_heads + kvh) * sc.cols + col;
    if (kh == 0) {
      sc.m[at] = m_run;
      sc.l[at] = l;
    }
    if (begin == end) return;
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
    if (a.weights != nullptr && kh == 0) {
      const std::size_t at = static_cast<std::size_t>(kvh) * sc.cols + col;
      sc.final[2 * at] = m_run;
      sc.final[2 * at + 1] = inv;
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

// Joins a split call: W waves per column take its splits in turn, eight loads of a
// partial row at a time in flight, a lane four dims.
template <int W>
__global__ __launch_bounds__(kPThreads) void compact_prefill_merge_kernel(CompactArgs a, PrefillScratch sc) {
  __shared__ float o_of[kPWaves][kHeadDim];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::uint32_t all_cols = a.tokens * a.group;
  const std::uint32_t col_of = blockIdx.x * (kPWaves / W) + wave / W;
  const std::uint32_t col = col_of < all_cols ? col_of : all_cols - 1;
  const std::uint32_t kvh = blockIdx.y;
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
      const std::uint32_t s = s0 + W * b < sc.splits ? s0 + W * b : sc.splits - 1;
      x[b] = *reinterpret_cast<const floatx4 *>(sc.o + (at0 + s * stride) * kHeadDim + 4 * lane);
    }
  };
  const std::uint32_t first = W == 1 ? 0 : wave % W;
  load(first);
  // max and sum over the splits; those without a key that the column sees have l = 0
  float m = -FLT_MAX, l = 0.f;
  for (std::uint32_t s = lane; s < sc.splits; s += 64) {
    const float ms = sc.m[at0 + s * stride], ls = sc.l[at0 + s * stride];
    const float m_new = fmaxf(m, ms);
    l = l * fexp2(m - m_new) + ls * fexp2(ms - m_new);
    m = m_new;
  }
  const float m_all = wave_max(m);
  const float inv = 1.0f / wave_sum(l * fexp2(m - m_all));
  floatx4 o{};
  for (std::uint32_t s0 = first; s0 < sc.splits; s0 += W * kBatch) {
    if (s0 != first) load(s0);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const std::uint32_t s = s0 + W * b;
      if (s >= sc.splits) break;
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
  if (a.weights != nullptr && lane == 0) {
    sc.final[2 * at0] = m_all;
    sc.final[2 * at0 + 1] = inv;
  }
  const float r0 = o[0] * inv * sigmoid_gate(bf16_lo(g[0])), r1 = o[1] * inv * sigmoid_gate(bf16_hi(g[0]));
  const float r2 = o[2] * inv * sigmoid_gate(bf16_lo(g[1])), r3 = o[3] * inv * sigmoid_gate(bf16_hi(g[1]));
  *reinterpret_cast<u32x2 *>(a.output + out_at) = u32x2{pack_bf16x2(r0, r1), pack_bf16x2(r2, r3)};
}

// Key weights of the last `observed` tokens: a workgroup owns a 32-key tile of one KV
// head, its waves take every fourth block of 32 observed columns and form the
// probabilities again from the columns' final max and sum.  The owner sums them, so
// nothing is added twice or in a changing order.
template <bool Fp8>
__global__ __launch_bounds__(kPThreads, 2) void compact_prefill_weigh_kernel(CompactArgs a, PrefillScratch sc) {
  __shared__ float sum[kPWaves][kCompactBlock];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, kh = lane >> 5;
  const std::uint32_t kvh = blockIdx.y;
  const std::uint32_t last = a.past + a.tokens - 1;
  const SeenTiles seen(a.past + a.tokens - a.observed, last, a.window, a.sinks);
  const std::uint32_t tile = seen.tile(blockIdx.x), j0 = tile * kCompactBlock;
  const CompactHead<Fp8> c(a.cache, kvh, a.kv_heads, a.max_ctx, a.head_major);
  float k_scale = kLog2e / 16.0f;
  if constexpr (Fp8) k_scale *= c.ks[tile];
  bf16x8 k[16];
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
  const std::uint32_t all_cols = a.tokens * a.group;
  for (std::uint32_t c0 = (a.tokens - a.observed) * a.group + 32 * wave; c0 < all_cols; c0 += 32 * kPWaves) {
    const bool real = c0 + n32 < all_cols;
    const std::uint32_t col = real ? c0 + n32 : all_cols - 1;
    const std::uint32_t tok = col / a.group, pos = a.past + tok;
    const bf16_bits *q =
        a.query + ((static_cast<std::size_t>(tok) * a.kv_heads + kvh) * a.group + (col - tok * a.group)) * kHeadDim + 8 * kh;
    floatx16 s = floatx16{};
#pragma unroll
    for (int b = 0; b < 16; ++b)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[b], __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(q + 16 * b)), s, 0, 0, 0);
    const std::size_t at = static_cast<std::size_t>(kvh) * sc.cols + col;
    const float m = sc.final[2 * at], inv = sc.final[2 * at + 1];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const std::uint32_t j = j0 + 8 * (i >> 2) + 4 * kh + (i & 3);
      w[i] += real && compact_sees(j, pos, a.window, a.sinks) ? fexp2(s[i] * k_scale - m) * inv : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = sum_xor16(row16_sum(w[i])); // over the 32 columns
    if (n32 == 0) sum[wave][8 * (i >> 2) + 4 * kh + (i & 3)] = w[i];
  }
  __syncthreads();
  if (threadIdx.x < kCompactBlock && j0 + threadIdx.x <= last)
    a.weights[static_cast<std::size_t>(kvh) * a.max_ctx + j0 + threadIdx.x] +=
        (sum[0][threadIdx.x] + sum[1][threadIdx.x]) + (sum[2][threadIdx.x] + sum[3][threadIdx.x]);
}

std::uint32_t col_blocks(const CompactArgs &a) { return (a.tokens * a.group + kPCols - 1) / kPCols; }

// Key splits of a call whose widest column block sees `tiles` tiles: two workgroups per
// CU where each still has 16 tiles, else one per CU, of at least four tiles.  Two per CU
// overlap softmax and products but leave twice the partial rows to be joined.  Measured
// (2 KV heads, 8 query heads each; one against two per CU): 500 tokens behind 2000
// (10 tiles at two) 58.1 against 61.8 us, behind 4000 (18) 79.1 against 77.5, behind
// 16000 (64) 208 against 174; 1000 tokens (8) 48.8 against 55.6, 1500 (23) 77.2 against
// 71.3.  Four tiles against eight: 2 tokens behind 2000 26.5 against 31.5 us, 500 tokens
// 36.0 against 38.5.  (Grows with `tiles`: the workspace is sized at the largest.)
std::uint32_t split_count(const CompactArgs &a, std::uint32_t tiles) {
  const std::uint64_t groups = static_cast<std::uint64_t>(col_blocks(a)) * a.kv_heads;
  const std::uint64_t wanted = groups * tiles >= 2 * kPrefillCus * 16 ? 2 * kPrefillCus : kPrefillCus;
  const std::uint64_t splits = groups >= wanted ? 1 : wanted / groups;
  const std::uint64_t most = (static_cast<std::uint64_t>(tiles) + 3) / 4;
  return static_cast<std::uint32_t>(splits < most ? splits : most);
}

PrefillScratch scratch_of(const CompactArgs &a, std::uint32_t splits, void *workspace, std::size_t *bytes) {
  PrefillScratch sc{};
  sc.splits = splits;
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
  if (splits > 1) {
    sc.m = take(splits * cols);
    sc.l = take(splits * cols);
    sc.o = take(splits * cols * kHeadDim);
  }
  if (bytes != nullptr) *bytes = at;
  return sc;
}

template <bool Fp8> void launch_prefill(const CompactArgs &a, void *workspace, hipStream_t stream) {
  const std::uint32_t last = a.past + a.tokens - 1;
  // a column block's tiles: at most those of the last block's span ending at the last key
  const std::uint32_t span = (kPCols + a.group - 1) / a.group + 1;
  const std::uint32_t first = a.tokens > span ? last - span + 1 : a.past;
  const std::uint32_t splits = split_count(a, SeenTiles(first, last, a.window, a.sinks).total);
  const PrefillScratch sc = scratch_of(a, splits, workspace, nullptr);
  const dim3 grid{col_blocks(a) * a.kv_heads, splits};
  const auto launch = [&](auto split) {
    if (a.weights != nullptr)
      compact_prefill_kernel<Fp8, split, true><<<grid, kPThreads, 0, stream>>>(a, sc);
    else
      compact_prefill_kernel<Fp8, split, false><<<grid, kPThreads, 0, stream>>>(a, sc);
  };
  if (splits > 1) {
    launch(std::true_type{});
    const std::uint32_t cols = a.tokens * a.group;
    if (splits > 8)
      compact_prefill_merge_kernel<kPWaves><<<dim3{cols, a.kv_heads}, kPThreads, 0, stream>>>(a, sc);
    else
      compact_prefill_merge_kernel<1><<<dim3{(cols + kPWaves - 1) / kPWaves, a.kv_heads}, kPThreads, 0, stream>>>(a, sc);
  } else {
    launch(std::false_type{});
  }
  if (a.weights != nullptr) {
    const SeenTiles seen(last + 1 - a.observed, last, a.window, a.sinks);
    compact_prefill_weigh_kernel<Fp8><<<dim3{seen.total, a.kv_heads}, kPThreads, 0, stream>>>(a, sc);
  }
}

} // namespace

std::size_t compact_prefill_workspace(const CompactArgs &a) {
  std::size_t bytes = 0;
  (void)scratch_of(a, split_count(a, (a.max_ctx + kCompactBlock - 1) / kCompactBlock), nullptr, &bytes);
  return bytes;
}

void compact_prefill(const CompactArgs &a, bool fp8, void *workspace, hipStream_t stream) {
  compact_append(a, fp8, stream);
  if (fp8) launch_prefill<true>(a, workspace, stream);
  else launch_prefill<false>(a, workspace, stream);
}

} // namespace raftinfer::amd
