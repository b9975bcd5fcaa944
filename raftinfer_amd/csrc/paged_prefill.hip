// Attention of chunks over the paged KV cache where there is much work: K and V tiles
// streamed through LDS, 64 columns a wave.
#include "paged_cache.hpp"
#include "prefill_stream.hpp"

#include <algorithm>

namespace raftinfer::amd {
namespace {

using namespace prefill;

__device__ unsigned int g_stream_capacity_errors = 0;

// out = sigmoid(gate) / l sum_j p_j v_j over tiles of 32 keys in one pass, p_j = 2^(q k_j log2(e) / 16 - m), l = sum_j p_j:
// S^T = K q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_bf16, the probabilities of a tile formed among the matrix instructions of
// the step before their product.  64 columns of a wave are what lets an operand read from LDS (16 clocks of the unit's 32 for
// each product of 32 columns) feed two products; their 256 accumulators fill the accumulation registers, one wave a SIMD.
// Measured (16 query and 4 KV heads): 2048 tokens of 32768 1094 to 1150 TFLOP/s (a product of 8192^3 in the BLAS library 1300),
// 500 of 30501 910 to 960, 8001 910 to 940.  By the counters the matrix units are busy for 56%, 48% and 42% of the waves' time in
// these; at that share 1094 and 1150 TFLOP/s are clocks of 1.87 and 1.97 GHz (1.75, 2.0 and 1.86 under the profiler).  A step of 64
// keys has 2048 clocks of matrix time and takes about 3,600 in the first: exponentials and packing among them, LDS reads, one
// barrier.  Start and end of a workgroup take 35,000 to 40,000 clocks: 4,000 to find its work, 12,000 until the first tiles and
// queries are there, 20,000 to join the key groups, for gates and stores: 2% of the first's, 8% of the
// second's, a seventh of the third's.
//
// Two key groups of two waves; the waves of a group share its tiles, each has 64 columns of its
// own.  A ring slot holds a tile's K or V: 32 rows of 512 bytes.  (One group of four waves, which
// halves the bytes that go into LDS for a column and has no groups to join, was no faster over long contexts, 1159
// against 1151 TFLOP/s for 2048 tokens of 32768, and keeps Q operands in scratch; on whole prompts, where the
// join is a larger share, it was not measured.)
constexpr int kGroups = 2, kShare = kWaves / kGroups;
constexpr int kStreamCols = 64 * kShare;
constexpr unsigned kSlot = 32 * kRowBytes;
constexpr unsigned kArea = 5 * kSlot;       // a key group's ring
constexpr int kLoads = 16 / kShare;         // of a wave, of an item: two rows each
constexpr unsigned kPart = kSlot / kShare;  // a wave's share of a slot: one granule

constexpr float kSlack = 16.0f; // log2 units

template <bool HeadMajor>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1, 1))) void paged_stream_kernel(
    PagedArgs a, PagedScratch sc, PagedSplit sp) {
  constexpr int L = kLoads;
  __shared__ __attribute__((aligned(16384))) unsigned char sh[kGroups * kArea];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave % kGroups, cg = wave / kGroups; // key group, column group
  // The hardware deals workgroups to the 8 dies in turn and of a die's to its 4 engines in turn, whatever has
  // become free: every other row of 32 takes the engines the other way round, so that of items that lie
  // longest first each engine gets about as much.  (16 sequences of up to 8192 behind a window of 4096, ten of
  // them single tokens, 268 workgroups for 256 places, in a graph: 208 -> 185 us.)
  const std::uint32_t turned = (blockIdx.x & 32) != 0 ? blockIdx.x ^ 24 : blockIdx.x;
  const std::uint32_t index = scalar(turned / a.kv_heads), kvh = turned - index * a.kv_heads;
  PagedItem it;
  if (!paged_find<kStreamCols, kKTile, true>(a, sp, sc, index, blockIdx.x == 0 && wave == 0, &g_stream_capacity_errors, it)) return;
  const std::uint32_t range = scalar(it.local / it.blocks), block = it.blocks - 1 - (it.local - range * it.blocks); // longest first
  if (!it.seq.valid) {
    paged_fill_nan<kThreads>(a, it, block * kStreamCols, kStreamCols, kvh);
    return;
  }
  const PagedBlock b = paged_block<kStreamCols, kKTile>(a, it, block);
  if (range >= b.count) return;
  const std::uint32_t begin = b.begin(range), end = b.begin(range + 1);
  const bool part = b.count > 1;
  const std::uint32_t slot = it.first_part + block * it.ranges + range;
  if (part && slot >= sp.parts) return; // (only where sequences share rows)
  // (the lane's index anew: what is derived from it is not kept over the loop)
  const auto late_lane = [&]() __attribute__((always_inline)) {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
  };
  // Token (of the block's, from tok0) and head of the group of column x: those past the last repeat it.
  // (x + 15 < 2^8 columns from a token's first: the quotient is x (2^16 / group + 1) >> 16.)
  const std::uint32_t in_first = b.col0 - b.tok0 * a.group, last_x = b.col_end - 1 - b.col0;
  const auto place = [&](std::uint32_t x, std::uint32_t &tok, std::uint32_t &head) __attribute__((always_inline)) {
    const std::uint32_t c = in_first + (x < last_x ? x : last_x);
    tok = c * a.group_inverse >> 16;
    head = c - tok * a.group;
  };
  const bf16_bits *q0 = a.query + static_cast<std::size_t>(it.seq.row0 + b.tok0) * a.q_row + kvh * a.group * a.q_head;
  const float scale = kLog2e / 16.0f;

  // Q^T operands: block bq, k-step kk holds dims 16 kk + 8 half .. + 7 of its column.
  const int col = lane & 31, half = lane >> 5;
  bf16x8 qa[2][16];
  const auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int bq = 0; bq < 2; ++bq) {
      std::uint32_t tok, head;
      place(64 * cg + 32 * bq + col, tok, head);
      const bf16_bits *q = q0 + tok * a.q_row + head * a.q_head + 8 * half;
#pragma unroll
      for (int kk = 0; kk < 16; ++kk) qa[bq][kk] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(q + 16 * kk));
    }
  };

  // ---- loads.  Tile t of the group is tile begin + 2 t + kg; this wave loads granule cg of it.  A granule in front of the first key or behind
  // the last repeats theirs; a granule's rows are all read, keys or not (their scores are masked, and
  // their values cleaned).
  const std::uint32_t m = (end - begin + kGroups - 1) / kGroups; // of every group (the barriers); the last can lie behind the range
  const auto tile_of = [&](std::uint32_t t) { return begin + kGroups * t + kg; };
  const std::uint32_t first_granule = b.first_key / kPageGranule, last_granule = b.p_hi / kPageGranule;
  std::uint64_t bad = 0; // lanes that met a bad page
  // Lane l: first K row of this wave's granule of tile t0 + l.
  std::uint32_t row_of = 0, t0 = 0;
  const auto load_table = [&](std::uint32_t from) __attribute__((always_inline)) {
    t0 = from;
    std::uint32_t g = 2 * tile_of(from + late_lane()) + cg;
    g = g < first_granule ? first_granule : g < last_granule ? g : last_granule;
    bool wrong = false;
    row_of = paged_row(a, it.id, kvh, g * kPageGranule, wrong);
    bad |= __builtin_amdgcn_ballot_w64(wrong);
  };
  const std::uint32_t row_bytes = HeadMajor ? kRowBytes : a.row_step * kRowBytes;
  // K: chunk c (0 .. 31) of row r at c ^ f, f = r / 2 % 8 + 8 (r % 2); V: f = 4 (r / 2 % 2) + 8 (r % 2):
  // the 16 rows of a ds_read_b128 pass over K share no bank, nor do the 4 rows x 64 bytes of a
  // ds_read_b64_tr_b16 pass over V.
  const std::uint32_t off0 = half * row_bytes + 16u * (col ^ (8 * half));
  const unsigned lds0 = lds_address(sh), ring = lds0 + kg * kArea;
  const auto base_of = [&](std::uint32_t t, bool is_v) __attribute__((always_inline)) {
    const std::uint32_t row = lane_u32(row_of, t - t0) + (is_v ? a.plane_rows : 0);
    return a.pages + static_cast<std::size_t>(row) * kRowBytes;
  };
  // Load i of an item (rows 2 i, 2 i + 1 of the share), whole.  The instruction's offset counts for both
  // addresses: the lane's is less by as much (rows are at least 512 bytes apart).
  const std::uint32_t skip = 2 * (row_bytes - kRowBytes);
  const auto load_whole = [&](const unsigned char *base, bool is_v, unsigned to, auto ic) __attribute__((always_inline)) {
    constexpr int i = ic;
    std::uint32_t off = is_v ? load_offset<64u * (i & 1), 0>(off0) : load_offset<16u * i, 0>(off0);
    if constexpr (!HeadMajor && (i & 3) != 0) off += (i & 3) * skip;
    load_lds_b128_at<1024 * (i & 3)>(base + (i >> 2) * 8 * (HeadMajor ? kRowBytes : row_bytes), off, to + 4096u * (i >> 2));
  };
  const unsigned share_at = kPart * cg;
  const auto load_item = [&](std::uint32_t t, bool is_v, unsigned to) __attribute__((always_inline)) {
    const unsigned char *base = base_of(t, is_v);
    static_for<L>([&](auto i) __attribute__((always_inline)) { load_whole(base, is_v, to + share_at, i); });
  };
  // Ring items K(0) K(1) V(0) K(2) V(1) K(3) V(2) ..; item n uses slot n % 5.  While item n is
  // read, item n + 3 is loaded into the slot of n - 2, which every wave has left when it passes
  // the barrier in front of item n.  Items behind the last tile are loaded too (the last granule
  // again), so that every step waits for the same number of loads.
  load_table(0);
  load_item(0, false, ring);
  load_q();
  acc_fence();
  static_for<256>([](auto r) __attribute__((always_inline)) { acc_set<r>(0.f); });
  acc_fence();
  float m_run[2], top[2] = {-FLT_MAX, -FLT_MAX}, l_run[2] = {0.f, 0.f};

  // Slot addresses of ring items n - 1 .. n + 3 (n: the next to be read).
  unsigned p0 = ring + 4 * kSlot, p1 = ring, p2 = ring + kSlot, p3 = ring + 2 * kSlot, p4 = ring + 3 * kSlot;
  const auto advance = [&](int items) __attribute__((always_inline)) {
    for (int i = 0; i < items; ++i) {
      const unsigned x = p0;
      p0 = p1; p1 = p2; p2 = p3; p3 = p4; p4 = x;
    }
  };
  // K operand of k-step kk: chunk 2 kk + half of row col.  V^T operand (transposed read) of dims
  // block nb and key step kb: rows 16 kb + 4 half + r / 4 and 8 below, dims 32 nb + 16 (g & 1) + 4 (r & 3).
  const unsigned k_lane = col * 512u + 16u * (half ^ (((col >> 1) & 7) + 8 * (col & 1)));
  const int vg = (lane >> 4) & 1, vr = lane & 15, vrow = 4 * half + (vr >> 2);
  const unsigned v_lane = vrow * 512u + 16u * ((2 * vg + ((vr & 3) >> 1)) ^ (4 * ((vrow >> 1) & 1) + 8 * (vrow & 1))) + 8u * (vr & 1);
  bf16x8 op[4];      // operands of the next four MFMA groups, across phases
  unsigned at = 0;   // lane address of the tile being read
  unsigned at_x = 0; // ... of the exclusive-or group being read
  // Order within a phase, s = 0 .. 15: k-steps s / 2 and s / 2 + 8 in turn; for V, key step
  // s / 8 and dims blocks s / 2 % 4 and s / 2 % 4 + 4 in turn.  Such pairs share their exclusive-or.
  const auto k_operand = [&](auto sc) __attribute__((always_inline)) {
    constexpr int s = sc;
    if constexpr (s % 2 == 0) at_x = at ^ (32u * (s >> 1));
    return lds_read_b128(at_x + 256u * (s & 1));
  };
  const auto v_operand = [&](auto sc) __attribute__((always_inline)) {
    constexpr int s = sc;
    constexpr unsigned off = 256u * (s & 1) + 8192u * (s >> 3);
    if constexpr (s % 2 == 0) at_x = at ^ (64u * ((s >> 1) & 3));
    const u32x2 lo = lds_read_tr16(at_x + off), hi = lds_read_tr16(at_x + off + 4096u);
    return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
  };

  floatx16 s0[2], s1[2];
  std::uint32_t pk[2][8]; // P^T, bf16 pairs in accumulator order
  float mx[2];            // max of the next S over this lane's keys
  // Pair u of the probabilities (blocks in turn): registers 2i, 2i + 1 of an S.  Rounded to bf16, as the
  // product with V takes them (in two parts it would be twice as long, half of a step's matrix time more); the
  // sum takes the same rounded probabilities, so that a row of equal values is theirs.  The empty asm keeps the pair where it is
  // written, among the MFMAs.
  const auto soft_pair = [&](const floatx16(&s)[2], auto uc) __attribute__((always_inline)) {
    constexpr int bq = uc % 2, i = uc / 2;
    const float x0 = fexp2(fmaf(s[bq][2 * i], scale, -m_run[bq]));
    const float x1 = fexp2(fmaf(s[bq][2 * i + 1], scale, -m_run[bq]));
    pk[bq][i] = pack_bf16x2(x0, x1);
    l_run[bq] = dot2_bf16(pk[bq][i], 0x3F803F80u, l_run[bq]);
    asm volatile("" : "+v"(pk[bq][i]), "+v"(l_run[bq]));
  };
  // Pairs [from, from + count) spread over the steps of a part of `steps` steps.
  const auto soft_step = [&](const floatx16(&s)[2], auto sc, auto from, auto count, auto steps) __attribute__((always_inline)) {
    constexpr int u0 = sc * count / steps, u1 = (sc + 1) * count / steps;
    static_for<u1 - u0>([&](auto k) __attribute__((always_inline)) { soft_pair(s, std::integral_constant<int, from + u0 + k>{}); });
  };
  constexpr std::integral_constant<int, 0> c0{};
  constexpr std::integral_constant<int, 12> kQkPairs{}; // of 16; all of key step 0 among them
  constexpr std::integral_constant<int, 4> kPvPairs{};
  constexpr std::integral_constant<int, 16> c16{};
  constexpr std::integral_constant<int, 8> c8{};
  const auto lane_max = [&](const floatx16(&s)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int bq = 0; bq < 2; ++bq) {
      mx[bq] = max3(s[bq][0], s[bq][1], s[bq][2]);
#pragma unroll
      for (int i = 3; i < 15; i += 2) mx[bq] = max3(mx[bq], s[bq][i], s[bq][i + 1]);
      mx[bq] = max3(mx[bq], s[bq][15], s[bq][15]);
    }
  };
  // m_run lies up to 2^kSlack above the largest score so far (top): no probability exceeds 1, and the
  // accumulators are scaled only where a score passes it, then to the whole distance for all columns of the block.
  // (A step without costs nothing; with it, 128 registers each read, multiplied and written.)
  const auto new_max = [&](bool first) __attribute__((always_inline)) {
    static_for<2>([&](auto bq) __attribute__((always_inline)) {
      top[bq] = fmaxf(top[bq], max_xor32(mx[bq]) * scale);
      if (first) { // nothing is accumulated yet
        m_run[bq] = top[bq] + kSlack;
      } else if (__builtin_amdgcn_ballot_w64(top[bq] > m_run[bq]) != 0) {
        mfma_drain();
        const float m_new = top[bq] + kSlack, f = fexp2(m_run[bq] - m_new);
        l_run[bq] *= f;
        m_run[bq] = m_new;
        static_for<128>([&](auto r) __attribute__((always_inline)) { acc_set<128 * bq + r>(acc_get<128 * bq + r>() * f); });
      }
    });
  };
  // Keys that a column does not see, and those behind the range, score -inf (register i: key 8 (i / 4) +
  // 4 half + i % 4 of the tile).
  const auto mask = [&](floatx16(&s)[2], std::uint32_t tile) __attribute__((always_inline)) {
    const int le = late_lane(), j0 = static_cast<int>(tile * kKTile) + 4 * (le >> 5);
#pragma unroll
    for (int bq = 0; bq < 2; ++bq) {
      std::uint32_t tok, head;
      place(64 * cg + 32 * bq + (le & 31), tok, head);
      const int p = static_cast<int>(b.p_lo + tok);
      const int to = tile < end ? p - j0 : -1; // the last key seen, from the lane's first
      const int from = a.window != 0 ? p - static_cast<int>(a.window) - j0 : -1; // the last in front of the window
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i >> 2) + (i & 3);
        s[bq][i] = ((key > to) | (key <= from)) ? -INFINITY : s[bq][i];
      }
      asm volatile("" : "+v"(s[bq])); // (one block after the other)
    }
    lane_max(s);
  };
  // A masked key has probability 0, and 0 times an infinite or NaN value is not 0: in V tiles that
  // some column does not see whole, such values are taken out of this wave's share of the slot and
  // added behind the loop, to the columns that see their keys.
  std::uint64_t odd = 0; // lanes that took values out
  const auto clean = [&](unsigned from) __attribute__((always_inline)) {
    const unsigned mine = from + share_at + 16u * late_lane();
#pragma unroll 1
    for (unsigned i = 0; i < L; ++i) {
      u32x4 w = *lds_ptr<u32x4>(mine + 1024u * i);
      std::uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const std::uint32_t ones = ((w[e] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
        any |= ones;
        w[e] &= ~((ones >> 15) * 0xFFFFu);
      }
      if (any != 0) *lds_ptr<u32x4>(mine + 1024u * i) = w;
      odd |= __builtin_amdgcn_ballot_w64(any != 0);
    }
    wait_lgkm0();
  };
  // Tiles that every column sees whole: from clear_from on, clear_count of them.
  const std::uint32_t clear_from = a.window != 0 && b.p_hi >= a.window ? (b.p_hi - a.window) / kKTile + 1 : 0;
  const std::uint32_t causal = (b.p_lo + 1) / kKTile < end ? (b.p_lo + 1) / kKTile : end;
  const std::uint32_t clear_count = causal > clear_from ? causal - clear_from : 0;
  const auto masked = [&](std::uint32_t t) __attribute__((always_inline)) { return tile_of(t) - clear_from >= clear_count; };
  const auto barrier = []() __attribute__((always_inline)) { __builtin_amdgcn_s_barrier(); };

  // out = K Q^T of the tile at `at`, on the matrix unit, while (soft) the vector unit turns s into
  // probabilities.  load(step) issues the wave's loads of this phase, ready() waits for V.
  const auto qk = [&](auto soft, const floatx16(&s)[2], floatx16(&out)[2], auto load, auto ready, unsigned v_slot)
      __attribute__((always_inline)) {
    static_for<16>([&](auto st) __attribute__((always_inline)) {
      constexpr int q = st & 3, kk = (st >> 1) + 8 * (st & 1);
      if constexpr (st == 0) s_mfma_zero(out[0], op[q], qa[0][kk]); else s_mfma(out[0], op[q], qa[0][kk]);
      if constexpr (soft) soft_step(s, st, c0, kQkPairs, c16);
      if constexpr (st == 0) s_mfma_zero(out[1], op[q], qa[1][kk]); else s_mfma(out[1], op[q], qa[1][kk]);
      if constexpr (soft && st == 12) {
        ready();
        at = v_slot + v_lane;
      }
      if constexpr (st < 12) op[q] = k_operand(std::integral_constant<int, st + 4>{});
      else if constexpr (soft) op[q] = v_operand(std::integral_constant<int, st - 12>{});
      load(st);
      if constexpr (st % 2 == 1) acc_fence();
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // O += V^T P^T, the remaining probabilities of s formed on the way; with kMax the max of `next` over
  // this lane's keys is taken and the next K tile begun.
  const auto pv = [&](auto kMax, const floatx16(&s)[2], const floatx16(&next)[2], auto load, auto ready, unsigned k_slot)
      __attribute__((always_inline)) {
    acc_fence();
    const auto p_operand = [&](int bq, int kb) __attribute__((always_inline)) {
      return __builtin_bit_cast(bf16x8, u32x4{pk[bq][4 * kb], pk[bq][4 * kb + 1], pk[bq][4 * kb + 2], pk[bq][4 * kb + 3]});
    };
    static_for<16>([&](auto st) __attribute__((always_inline)) {
      constexpr int q = st & 3, kb = st >> 3, nb = ((st >> 1) & 3) + 4 * (st & 1);
      acc_mfma<nb>(op[q], p_operand(0, kb));
      if constexpr (st < 8) soft_step(s, st, kQkPairs, kPvPairs, c8);
      acc_mfma<8 + nb>(op[q], p_operand(1, kb));
      if constexpr (kMax && st == 12) {
        ready();
        at = k_slot + k_lane;
      }
      if constexpr (st < 12) op[q] = v_operand(std::integral_constant<int, st + 4>{});
      else if constexpr (kMax) op[q] = k_operand(std::integral_constant<int, st - 12>{});
      if constexpr (kMax && st >= 8) { // two values of each block per step
        constexpr int i = 2 * (st - 8);
#pragma unroll
        for (int bq = 0; bq < 2; ++bq) mx[bq] = max3(st == 8 ? next[bq][0] : mx[bq], next[bq][i], next[bq][i + 1]);
      }
      load(st);
      if constexpr (st % 4 == 3) acc_fence();
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  // Step n: tile n (its S in s, mx its max) -> O, with S(n + 1) formed on the way.  The two S buffers
  // alternate by name: a copy placed right behind the MFMA that writes it would read it too early.
  std::uint32_t n = 0;
  constexpr int kEvery = 16 / L; // a load every so many steps of a phase
  constexpr int kBefore = (12 + kEvery - 1) / kEvery; // loads of a phase issued in front of step 12
  const auto step = [&](auto kClear, floatx16(&s)[2], floatx16(&next)[2]) __attribute__((always_inline)) {
    if (!kClear && masked(n)) {
      mask(s, tile_of(n));
      wait_vm<L>(); // V(n); K(n + 2) is behind it
      clean(p2);
    }
    new_max(n == 0);
    // QK reads K(n + 1) and loads V(n + 1), PV reads V(n) and loads K(n + 3).
    const unsigned char *vb = base_of(n + 1, true), *kb = base_of(n + 3, false);
    const unsigned v_to = p4 + share_at, k_to = p0 + share_at;
    qk(std::true_type{}, s, next,
       [&](auto st) __attribute__((always_inline)) {
         if constexpr (st % kEvery == 0) load_whole(vb, true, v_to, std::integral_constant<int, st / kEvery>{});
       },
       [&]() __attribute__((always_inline)) {
         wait_vm<L + kBefore>();
         barrier();
       },
       p2);
    pv(std::true_type{}, s, next,
       [&](auto st) __attribute__((always_inline)) {
         if constexpr (st % kEvery == 0) load_whole(kb, false, k_to, std::integral_constant<int, st / kEvery>{});
       },
       [&]() __attribute__((always_inline)) {
         wait_vm<L + kBefore>();
         barrier();
       },
       p3);
    advance(2);
    ++n;
  };
  // The wait for q is one for every load in front of it: K(0), but for no other.
#pragma unroll
  for (int bq = 0; bq < 2; ++bq)
#pragma unroll
    for (int kk = 0; kk < 16; ++kk) asm volatile("" : "+v"(qa[bq][kk]));
  wait_vm<0>();
  load_item(1, false, ring + kSlot);
  load_item(0, true, ring + 2 * kSlot);
  barrier();
  // S of the first tile, K(2) loaded.
  at = p1 + k_lane;
  static_for<4>([&](auto i) __attribute__((always_inline)) { op[i] = k_operand(i); });
  {
    const unsigned char *kb = base_of(2, false);
    qk(std::false_type{}, s0, s0,
       [&](auto st) __attribute__((always_inline)) {
         if constexpr (st % kEvery == 0) load_whole(kb, false, p4 + share_at, std::integral_constant<int, st / kEvery>{});
       },
       [] {}, 0);
  }
  advance(1);
  s_drain(s0);
  lane_max(s0);
  if (m > 1) { // K(1); V(0) and K(2) are behind it
    wait_vm<2 * L>();
    barrier();
    at = p1 + k_lane;
    static_for<4>([&](auto i) __attribute__((always_inline)) { op[i] = k_operand(i); });
  }
  // (Loops of their own for tiles that some column does not see whole: where the mask is formed, Q
  // operands are spilled, and the wait for a reload waits for the loads in front of it too.)
  while (n + 1 < m) {
    if (n + 4 - t0 >= 64) load_table(n + 1);
    // clear pairs whose loads the table has: n + 1 is clear, n + 2 < m, n + 4 in the table
    while (n + 2 < m && !masked(n) && !masked(n + 1) && n + 4 - t0 < 64) {
      step(std::true_type{}, s0, s1);
      step(std::true_type{}, s1, s0);
    }
    if (n + 1 >= m) break;
    if (n + 4 - t0 >= 64) continue;
    step(std::false_type{}, s0, s1);
    if (n + 1 >= m) {
      s_drain(s1);
#pragma unroll
      for (int bq = 0; bq < 2; ++bq) s0[bq] = s1[bq];
      break;
    }
    step(std::false_type{}, s1, s0);
  }
  wait_vm<0>();
  if (masked(n)) {
    mask(s0, tile_of(n));
    clean(p2);
  }
  new_max(n == 0);
  static_for<kQkPairs>([&](auto u) __attribute__((always_inline)) { soft_pair(s0, u); });
  barrier();
  at = p2 + v_lane;
  static_for<4>([&](auto i) __attribute__((always_inline)) { op[i] = v_operand(i); });
  pv(std::false_type{}, s0, s0, [](auto) __attribute__((always_inline)) {}, [] {}, 0);
  mfma_drain();
  wait_lgkm0();
  __syncthreads(); // every wave has left the ring

  // ---- epilogue.  Of the two key groups, group kg finishes block kg of its columns: a wave hands the
  // other block's sums over in LDS, [quad][lane], half of them at a time; the gates of its block's 32
  // columns are on the way meanwhile, a row of 512 bytes a column, 16-byte chunk c of row r at c ^ swz(r).
  constexpr unsigned kGatesAt = 65536, kMaxAt = 131072, kFlagsAt = kMaxAt + 8192;
  const int le = late_lane(), col_e = le & 31, half_e = le >> 5;
  const unsigned rows = lds0 + kGatesAt + 16384u * wave;
  std::uint32_t tok_e, head_e; // of column col_e of the block
  place(64 * cg + 32 * kg + col_e, tok_e, head_e);
  // ... of rows 2 i + half_e, for whole rows by 32 lanes
  const std::uint32_t both = tok_e << 8 | head_e;
  const auto row_of_column = [&](int i, std::size_t row, std::size_t head) __attribute__((always_inline)) {
    std::uint32_t from = both;
    asm volatile("" : "+v"(from)); // (formed anew where it is used)
    const auto x = static_cast<std::uint32_t>(__builtin_amdgcn_ds_bpermute(4 * (2 * i + half_e), static_cast<int>(from)));
    return (x >> 8) * row + (x & 255) * head + 8 * (col_e ^ swz(2 * i + half_e));
  };
  const std::size_t first_row = it.seq.row0 + b.tok0, first_head = kvh * a.group;
  if (a.gate != nullptr && !part) {
    const bf16_bits *gate = a.gate + first_row * a.g_row + first_head * a.g_head;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      load_lds_b128_lane(gate + row_of_column(i, a.g_row, a.g_head), rows + 1024u * i);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
  auto *max_of = lds_ptr<float>(lds0 + kMaxAt); // [wave][max, sum][lane] of the block handed over
  max_of[128 * wave + le] = kg == 0 ? m_run[1] : m_run[0];
  max_of[128 * wave + kWave + le] = kg == 0 ? l_run[1] : l_run[0];
  auto *flag_of = lds_ptr<std::uint32_t>(lds0 + kFlagsAt);
  if (le == 0) flag_of[wave] = (odd != 0 ? 1u : 0u) | (bad != 0 ? 2u : 0u);
  if ((bad != 0) & (le == 0)) atomicAdd(&g_stream_capacity_errors, 1u);
  float mm = kg == 0 ? m_run[0] : m_run[1], ll = kg == 0 ? l_run[0] : l_run[1]; // of column col_e
  floatx4 f[32]; // quad i: dims 8 i + 4 half_e .. + 3
  auto *to = lds_ptr<floatx4>(lds0 + 16384u * wave) + le;
  const auto *from = lds_ptr<floatx4>(lds0 + 16384u * (wave ^ 1)) + le;
  float own = 1.0f, other = 1.0f;
  const auto hand = [&](auto bc, auto h) __attribute__((always_inline)) { // block bc is the wave's own
    static_for<16>([&](auto i) __attribute__((always_inline)) {
      constexpr int r = 128 * (1 - bc) + 64 * h + 4 * i;
      to[kWave * i] = floatx4{acc_get<r>(), acc_get<r + 1>(), acc_get<r + 2>(), acc_get<r + 3>()};
    });
    static_for<16>([&](auto i) __attribute__((always_inline)) {
      constexpr int r = 128 * bc + 64 * h + 4 * i;
      f[16 * h + i] = floatx4{acc_get<r>(), acc_get<r + 1>(), acc_get<r + 2>(), acc_get<r + 3>()};
    });
  };
  static_for<2>([&](auto h) __attribute__((always_inline)) {
    if constexpr (h == 1) __syncthreads(); // what was handed over first has been read
    if (kg == 0) hand(c0, h); else hand(std::integral_constant<int, 1>{}, h);
    __syncthreads();
    if constexpr (h == 0) {
      const float m_other = max_of[128 * (wave ^ 1) + le], l_other = max_of[128 * (wave ^ 1) + kWave + le];
      const float m_all = fmaxf(mm, m_other);
      own = fexp2(mm - m_all);
      other = fexp2(m_other - m_all);
      mm = m_all;
      ll = sum_xor32(ll * own + l_other * other);
    }
    // (a few at a time: all the loads at once would take more vector registers than there are, and the
    // accumulation registers are not the compiler's)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      f[16 * h + i] = f[16 * h + i] * own + from[kWave * i] * other;
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    acc_fence();
  });
  const std::uint32_t flags = flag_of[0] | flag_of[1] | flag_of[2] | flag_of[3];
  if ((flags & 2u) != 0) ll = __builtin_nanf("");
  if ((flags & 1u) != 0) {
#pragma unroll 1
    for (std::uint32_t tile = begin; tile < end; ++tile) {
      if (tile - clear_from < clear_count) continue;
#pragma unroll 1
      for (std::uint32_t j = tile * kKTile; j < (tile + 1) * kKTile && j <= b.p_hi; ++j) {
        if (!paged_sees(j, b.p_lo + tok_e, a.window)) continue;
        bool ignored = false;
        const std::uint32_t row = paged_row(a, it.id, kvh, j, ignored) + a.plane_rows;
        const unsigned char *v = a.pages + static_cast<std::size_t>(row) * kRowBytes + 8 * half_e;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const u32x2 w = *reinterpret_cast<const u32x2 *>(v + 16 * i);
          const float v4[4] = {bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
#pragma unroll
          for (int e = 0; e < 4; ++e) f[i][e] += (__float_as_uint(v4[e]) & 0x7F800000u) != 0x7F800000u ? 0.f : v4[e];
        }
      }
    }
  }
  const std::uint32_t x0 = 64 * cg + 32 * kg; // of the block in the workgroup's columns
  if (part) { // (paged_stream_merge_kernel reads the sums as they lie in the lanes)
    const std::size_t at0 = (static_cast<std::size_t>(slot) * a.kv_heads + kvh) * kStreamCols + x0;
    if (half_e == 0) {
      sc.m[at0 + col_e] = mm;
      sc.l[at0 + col_e] = ll;
    }
    auto *o = reinterpret_cast<floatx4 *>(sc.o + at0 * kHeadDim) + le;
#pragma unroll
    for (int i = 0; i < 32; ++i) o[kWave * i] = f[i];
    return;
  }
  const float inv = 1.0f / ll;
  const unsigned mine = rows + 512u * col_e + 8u * half_e;
  const bool gated = a.gate != nullptr;
  wait_vm<0>();
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    auto *piece = lds_ptr<u32x2>(mine + 16u * (i ^ swz(col_e)));
    const u32x2 g = *piece; // (without a gate: anything)
    const auto out = [&](int e, float x) { return f[i][e] * inv * (gated ? sigmoid_gate(x) : 1.0f); };
    *piece = u32x2{pack_bf16x2(out(0, bf16_lo(g[0])), out(1, bf16_hi(g[0]))), pack_bf16x2(out(2, bf16_lo(g[1])), out(3, bf16_hi(g[1])))};
    if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
  }
  wave_lds_order(); // the rows' pieces are read back by other lanes of this wave
  bf16_bits *out = a.output + first_row * a.o_row + first_head * a.o_head;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const u32x4 row = *lds_ptr<u32x4>(rows + 1024u * i + 16u * le);
    const std::size_t at_row = row_of_column(i, a.o_row, a.o_head);
    if (x0 + 2 * i + half_e <= last_x) *reinterpret_cast<u32x4 *>(out + at_row) = row;
    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
  }
}

// Joins the ranges of split column blocks, 32 columns of a KV head at a time: by as many workgroups as work
// side by side, since only the device knows how many blocks there are (one for each that could be: 9.6 us where none
// is split, 16 sequences).  A wave takes four quads of every lane's column, eight ranges' at a time on the way.
constexpr int kJoinWaves = 8, kJoinGrid = 1024;
__global__ __launch_bounds__(kJoinWaves *kWave) void paged_stream_merge_kernel(PagedArgs a, PagedScratch sc, PagedSplit sp) {
  constexpr std::uint32_t kSlices = kStreamCols / 32;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::uint32_t all = sc.plan[1] * a.kv_heads * kSlices;
  for (std::uint32_t at = blockIdx.x; at < all; at += gridDim.x) {
    const std::uint32_t of_heads = at / kSlices, index = scalar(of_heads / a.kv_heads), kvh = of_heads - index * a.kv_heads;
    PagedItem it;
    if (!paged_find_split<kStreamCols, kKTile, true>(a, sc, index, it)) return;
    const PagedBlock b = paged_block<kStreamCols, kKTile>(a, it, it.local);
    const std::uint32_t x0 = 32 * (at % kSlices), part0 = it.first_part + it.local * it.ranges;
    if (b.count == 1 || b.col0 + x0 >= b.col_end) continue;
    if (part0 + b.count > sp.parts) return; // (only where sequences share rows)
    const std::size_t stride = static_cast<std::size_t>(a.kv_heads) * kStreamCols; // between parts
    const std::size_t at0 = part0 * stride + static_cast<std::size_t>(kvh) * kStreamCols + x0;
    const std::uint32_t last_x = b.col_end - 1 - b.col0, x = x0 + col < last_x ? x0 + col : last_x;
    const std::uint32_t c = b.col0 - b.tok0 * a.group + x, tok = c * a.group_inverse >> 16, head = c - tok * a.group;
    const std::size_t row = it.seq.row0 + b.tok0 + tok, h = kvh * a.group + head;
    const int dim = 32 * wave + 4 * half; // quad 4 wave + i: dims 32 wave + 8 i + 4 half
    u32x2 g[4];
    if (a.gate != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = *reinterpret_cast<const u32x2 *>(a.gate + row * a.g_row + h * a.g_head + dim + 8 * i);
    }
    const auto *o = reinterpret_cast<const floatx4 *>(sc.o + at0 * kHeadDim) + 4 * kWave * wave + lane;
    float m_run = -FLT_MAX, l = 0.f;
    floatx4 sum[4]{};
    constexpr int kBatch = 8;
    for (std::uint32_t s0 = 0; s0 < b.count; s0 += kBatch) {
      floatx4 in[kBatch][4];
      float m[kBatch], ls[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const std::uint32_t s = s0 + k < b.count ? s0 + k : b.count - 1;
        m[k] = sc.m[at0 + s * stride + col];
        ls[k] = s0 + k < b.count ? sc.l[at0 + s * stride + col] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) in[k][i] = o[s * stride * (kHeadDim / 4) + kWave * i];
      }
      float m_new = m_run;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) m_new = fmaxf(m_new, m[k]);
      const float f = fexp2(m_run - m_new);
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] *= f;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (s0 + k >= b.count) break;
        const float fk = fexp2(m[k] - m_new);
        l += ls[k] * fk;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += in[k][i] * fk;
      }
      m_run = m_new;
    }
    if (x0 + col > last_x) continue;
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      floatx4 y = sum[i] * inv;
      if (a.gate != nullptr) {
        y[0] *= sigmoid_gate(bf16_lo(g[i][0])); y[1] *= sigmoid_gate(bf16_hi(g[i][0]));
        y[2] *= sigmoid_gate(bf16_lo(g[i][1])); y[3] *= sigmoid_gate(bf16_hi(g[i][1]));
      }
      *reinterpret_cast<u32x2 *>(a.output + row * a.o_row + h * a.o_head + dim + 8 * i) =
          u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    }
  }
}

} // namespace

void launch_paged_stream(const PagedArgs &a, const PagedScratch &sc, const PagedSplit &sp, std::uint32_t items,
                         std::uint32_t split_blocks, hipStream_t stream) {
  const auto go = [&](auto kernel) { kernel<<<(items * a.kv_heads + 31) / 32 * 32, kThreads, 0, stream>>>(a, sc, sp); };
  go(a.row_step == 1 ? paged_stream_kernel<true> : paged_stream_kernel<false>);
  if (split_blocks != 0)
    paged_stream_merge_kernel<<<std::min<std::uint32_t>(split_blocks * a.kv_heads * (kStreamCols / 32), kJoinGrid), kJoinWaves * kWave, 0, stream>>>(a, sc, sp);
}

std::uint32_t paged_take_stream_errors() {
  unsigned int value = 0;
  const unsigned int zero = 0;
  if (hipMemcpyFromSymbol(&value, HIP_SYMBOL(g_stream_capacity_errors), sizeof value) != hipSuccess ||
      hipMemcpyToSymbol(HIP_SYMBOL(g_stream_capacity_errors), &zero, sizeof zero) != hipSuccess)
    throw std::runtime_error("reading the capacity error counter failed");
  return value;
}

} // namespace raftinfer::amd
