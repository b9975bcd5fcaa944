// Device pieces of the paged KV cache: the pool's rows, a ragged batch's sequences,
// and how a batch's work is dealt to workgroups.
#pragma once

#include "decode_scan.hpp"

#include <cfloat>

namespace raftinfer::amd {

constexpr int kPageGranule = 16;      // positions that always lie in one page, next to each other
constexpr int kPagedMaxGroup = 16;    // query heads per KV head
constexpr int kRowBytes = kHeadDim * 2;

// What the kernels read of one call.  Strides in elements; row_step, head_step and
// plane_rows in rows of 512 bytes: between positions, KV heads, and K and V.
struct PagedArgs {
  const bf16_bits *query, *gate; // gate: or null
  bf16_bits *output;
  const unsigned char *pages;
  const std::int32_t *table;
  const std::uint32_t *starts; // or null: one row for each sequence
  const std::uint32_t *lengths;
  std::size_t q_row, q_head, g_row, g_head, o_row, o_head;
  std::uint32_t rows, sequences, kv_heads, group, page_count, page_tokens, table_pages, max_ctx, window;
  std::uint32_t row_step, head_step, plane_rows;
  std::uint32_t group_inverse, group_inverse30; // 2^16 / group + 1, 2^30 / group + 1
  int page_shift; // log2 of page_tokens, or -1
};

// One sequence's share of a batch.  Not valid: its rows, as far as they are the call's,
// become NaN.
struct PagedSeq {
  std::uint32_t row0, n, ctx;
  bool valid;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &a, std::uint32_t s) {
  const std::uint32_t c = a.lengths[s];
  if (a.starts == nullptr) return {s, c != 0 ? 1u : 0u, c, c <= a.max_ctx};
  const std::uint32_t b = a.starts[s], e = a.starts[s + 1];
  PagedSeq q{b, 0, c, true};
  if (b == e) return q;
  if (b > e || b >= a.rows) {
    q.valid = false;
  } else {
    q.valid = e <= a.rows && c >= e - b && c <= a.max_ctx;
    q.n = (e < a.rows ? e : a.rows) - b;
  }
  return q;
}

// The page-table entry's place and the position in the page of position j.
__device__ __forceinline__ void paged_place(const PagedArgs &a, std::uint32_t j, std::uint32_t &entry, std::uint32_t &in) {
  std::uint32_t page = a.page_tokens;
  asm volatile("" : "+s"(page)); // (no reciprocal of it is kept in registers)
  if (a.page_shift >= 0) entry = j >> a.page_shift; else entry = j / page;
  in = j - entry * page;
}
// The K row (512 bytes each, from the pool's first) of position j of a KV head; a bad page: `bad` is
// set and page 0 taken.  (The host sees to it that the pool has fewer than 2^32 rows.)
__device__ __forceinline__ std::uint32_t paged_row(const PagedArgs &a, std::uint32_t seq, std::uint32_t kvh, std::uint32_t j,
                                                   bool &bad) {
  std::uint32_t entry, in;
  paged_place(a, j, entry, in);
  auto page = static_cast<std::uint32_t>(a.table[static_cast<std::size_t>(seq) * a.table_pages + entry]);
  if (page >= a.page_count) {
    bad = true;
    page = 0;
  }
  return page * 2 * a.plane_rows + kvh * a.head_step + in * a.row_step;
}

// -------------------------------------------------------- dealing out the work
// A column is a (token, head of the group) of one KV head; a workgroup takes kCols columns
// of a sequence and KV head, and of the tiles (of kUnit keys) that they see a range.  All of a batch's
// workgroups deal the work out alike, each by itself, from the sequences' lengths: no launch in front.  The
// whole batch has W (column block, tile) pairs; ranges have at most T = max(least, W / slots) tiles of
// a sequence's longest block, so that about `slots` = 2^slot_bits workgroups per KV head run; 2^many_bits
// times as many for `many` sequences and more, whose blocks are of different lengths.  (Chunks of much
// work weigh T against others, see paged_rounds.)  The kernel that joins the ranges reads T from the workspace.
struct PagedSplit {
  std::uint32_t least, slot_bits, many, many_bits;
  std::uint32_t parts; // partial results that the workspace holds, each of a block and KV head
};
struct PagedScratch {
  float *m, *l, *o; // [part][kv_head][column of the block]; o: 256 floats of each
  std::uint32_t *plan; // where there are parts: tiles of a range, and split column blocks of a KV head
};

struct PagedItem {
  PagedSeq seq;
  std::uint32_t id, blocks, ranges, range_tiles; // of its sequence
  std::uint32_t local;      // index in the sequence's items, or split blocks
  std::uint32_t first_part; // of its sequence
};

template <int Ctrl, int RowMask> __device__ __forceinline__ std::uint32_t dpp_zero(std::uint32_t x) {
  return static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), Ctrl, RowMask, 0xF, false));
}
// Sum over this lane and those below it.
__device__ __forceinline__ std::uint32_t wave_prefix(std::uint32_t x) {
  x += dpp_zero<0x111, 0xF>(x); // row_shr 1, 2, 4, 8
  x += dpp_zero<0x112, 0xF>(x);
  x += dpp_zero<0x114, 0xF>(x);
  x += dpp_zero<0x118, 0xF>(x);
  x += dpp_zero<0x142, 0xA>(x); // lane 15 of the row below, into rows 1 and 3
  x += dpp_zero<0x143, 0xC>(x); // lane 31, into rows 2 and 3
  return x;
}
__device__ __forceinline__ std::uint32_t lane_u32(std::uint32_t x, int lane) {
  return static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// A value that is the same in every lane, in a scalar register (a quotient comes out of the
// vector unit and would stay in a vector register).
__device__ __forceinline__ std::uint32_t scalar(std::uint32_t x) {
  return static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}

// Tiles that a sequence's longest column block sees (at least 1), and its blocks.
template <int kCols, int kUnit>
__device__ __forceinline__ void paged_extent(const PagedArgs &a, const PagedSeq &q, std::uint32_t &blocks, std::uint32_t &tiles) {
  blocks = (q.n * a.group + kCols - 1) / kCols;
  if (!q.valid) {
    tiles = 1;
    return;
  }
  tiles = (q.ctx + kUnit - 1) / kUnit;
  if (a.window != 0) { // the window and the tokens of a block, both ends inside tiles
    const std::uint32_t span = (kCols + a.group - 2) * a.group_inverse / 65536 + 1;
    const std::uint32_t some = (a.window + (span < q.n ? span : q.n) + kUnit - 3) / kUnit + 1;
    tiles = some < tiles ? some : tiles;
  }
}

template <int Ctrl, int RowMask> __device__ __forceinline__ std::uint32_t dpp_most(std::uint32_t x) {
  const std::uint32_t y = dpp_zero<Ctrl, RowMask>(x);
  return x > y ? x : y;
}
__device__ __forceinline__ std::uint32_t wave_most(std::uint32_t x) {
  x = dpp_most<0x118, 0xF>(dpp_most<0x114, 0xF>(dpp_most<0x112, 0xF>(dpp_most<0x111, 0xF>(x))));
  return lane_u32(dpp_most<0x143, 0xC>(dpp_most<0x142, 0xA>(x)), 63);
}
// Item `index` (of_blocks: split column block `index`) of sequences with ranges of t tiles: q, id, blocks and
// tiles are those of up to 64 sequences, or of the batch's first, which are then read again.
template <int kCols, int kUnit>
__device__ __forceinline__ bool paged_pick(const PagedArgs &a, std::uint32_t index, bool of_blocks, std::uint32_t t, PagedSeq q, std::uint32_t id,
                                           std::uint32_t blocks, std::uint32_t tiles, PagedItem &item) {
  const std::uint32_t lane = threadIdx.x & 63;
  std::uint32_t before = 0, parts_before = 0;
  for (std::uint32_t s0 = 0; s0 < a.sequences; s0 += 64) {
    if (a.sequences > 64) {
      blocks = 0;
      id = s0 + lane;
      if (id < a.sequences) {
        q = paged_seq(a, id);
        paged_extent<kCols, kUnit>(a, q, blocks, tiles);
      }
    }
    const std::uint32_t ranges = (tiles + t - 1) / t;
    const std::uint32_t parts = ranges > 1 ? blocks * ranges : 0;
    const std::uint32_t mine = of_blocks ? (ranges > 1 ? blocks : 0) : blocks * ranges;
    const std::uint32_t upto = before + wave_prefix(mine), parts_upto = parts_before + wave_prefix(parts);
    const std::uint64_t hit = __builtin_amdgcn_ballot_w64(index < upto);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      item.seq.row0 = lane_u32(q.row0, at);
      item.seq.n = lane_u32(q.n, at);
      item.seq.ctx = lane_u32(q.ctx, at);
      item.seq.valid = lane_u32(q.valid, at) != 0;
      item.id = lane_u32(id, at);
      item.blocks = lane_u32(blocks, at);
      item.ranges = lane_u32(ranges, at);
      item.range_tiles = t;
      item.local = index - lane_u32(upto - mine, at);
      item.first_part = lane_u32(parts_upto - parts, at);
      return true;
    }
    before = lane_u32(upto, 63);
    parts_before = lane_u32(parts_upto, 63);
  }
  return false;
}

// Workgroups that fill a compute unit, `slots` of a KV head at once: the range length whose last workgroup
// should end first, one candidate a lane, from half of the share to twice of it.  A candidate's cost is the
// larger of the mean load, and over the sequences, which lie longest first, of ceil(N / slots) x: N items so far,
// of x tiles and more (a workgroup's start and end among them), of which some place takes as many.  Not for a
// sequence whose unsplit blocks grow from little to much, which fill places up by themselves.  (Measured beside
// paged_find.)
constexpr float kEnds = 20; // tiles that a workgroup's start and end take as long as
constexpr float kJoin = 12; // the same for the joining of ranges
__device__ __forceinline__ std::uint32_t paged_rounds(std::uint32_t blocks, std::uint32_t lo, std::uint32_t tiles, std::uint32_t share,
                                                      std::uint32_t bits, std::uint32_t sequences, std::uint32_t least) {
  if (share >> 16 != 0) return share;
  const std::uint32_t lane = threadIdx.x & 63;
  if (sequences > 16) { // neighbours as one, so that 16 remain at most (400 clocks each: 64 took 28,800)
    const std::uint32_t width = scalar((sequences + 15) / 16);
    std::uint32_t all = 0;
    float l = 0, f = 0;
    for (std::uint32_t i = 0; i < width; ++i) {
      const std::uint32_t at = lane * width + i;
      const auto of = [&](std::uint32_t x) {
        return static_cast<std::uint32_t>(__builtin_amdgcn_ds_bpermute(static_cast<int>(4 * (at & 63)), static_cast<int>(x)));
      };
      const std::uint32_t b = of(blocks), last = of(tiles), first = of(lo);
      if (at >= sequences) continue;
      all += b;
      l = fmaf(static_cast<float>(b), static_cast<float>(last), l);
      f = fmaf(static_cast<float>(b), static_cast<float>(first), f);
    }
    const float each = __builtin_amdgcn_rcpf(static_cast<float>(all != 0 ? all : 1));
    blocks = all;
    tiles = static_cast<std::uint32_t>(fmaf(l, each, 0.5f));
    lo = static_cast<std::uint32_t>(fmaf(f, each, 0.5f));
    sequences = (sequences + width - 1) / width;
  }
  std::uint32_t t = (share * (64 + 3 * lane) + 127) / 128; // (at least half of the share: items stay within blocks + 2 slots)
  t = t > least ? t : least;
  const float length = static_cast<float>(t), inverse = __builtin_amdgcn_rcpf(length);
  // the sum of ceil(x) from 0 to u, by parts: (n + 1) (u - n / 2), n whole
  const auto area = [](float u, float &n) {
    n = floorf(u);
    return fmaf(-0.5f, n, u);
  };
  float load = 0, longest = 0, shortest = FLT_MAX;
  std::uint32_t ahead = 0;
  for (std::uint32_t j = 0; j < sequences; ++j) {
    const std::uint32_t b = lane_u32(blocks, j), last = lane_u32(tiles, j), first = lane_u32(lo, j);
    if (b == 0) break;
    const float l = static_cast<float>(last), f = static_cast<float>(first), mid = 0.5f * (f + l);
    // the mean of a block's items: ceil(tiles / t), over tiles that grow from first to last
    const float u1 = l * inverse;
    float each = ceilf(u1);
    if (last - first >= 2) { // (uniform)
      float n0, n1;
      const float u0 = f * inverse, a0 = area(u0, n0), a1 = area(u1, n1);
      each = fmaf(n1, a1, a1 - fmaf(n0, a0, a0)) * __builtin_amdgcn_rcpf(fmaxf(u1 - u0, 1e-6f));
    }
    each = t >= last ? 1.0f : each;
    const float x = fmaf(mid, __builtin_amdgcn_rcpf(each), kEnds);
    const std::uint32_t items = static_cast<std::uint32_t>(fmaf(static_cast<float>(b), each, 0.999f));
    ahead += items;
    shortest = fminf(shortest, x);
    const float some = static_cast<float>((ahead + (1u << bits) - 1) >> bits) * shortest;
    longest = fmaxf(longest, b > 1 && 2 * first < last && t >= last ? l + kEnds : some);
    load = fmaf(static_cast<float>(items), x, load);
  }
  float cost = fmaxf(longest, load * (1.0f / static_cast<float>(1u << bits)));
  if (t < lane_u32(tiles, 0)) cost += kJoin;
  const std::uint32_t best = ~wave_most(~((__float_as_uint(cost) & ~63u) | lane)); // (costs are not negative)
  return lane_u32(t, best & 63);
}
// Lays the sequences of a wave so that the longest come first.
template <int kUnit>
__device__ __forceinline__ void paged_sort(PagedSeq &q, std::uint32_t &id, std::uint32_t &blocks, std::uint32_t &lo, std::uint32_t &tiles,
                                           std::uint32_t sequences) {
  const std::uint32_t lane = threadIdx.x & 63, front = (q.ctx - q.n) / kUnit + 1;
  lo = q.valid && front < tiles ? front : tiles; // of the first block; the last has `tiles`
  if (sequences == 1) return;
  const std::uint32_t key = (blocks != 0 ? lo + tiles : 0) << 6 | (63 - lane); // (tiles are fewer than 2^24)
  std::uint32_t rank = lane;
  if (lane < sequences) {
    rank = 0;
    for (std::uint32_t j = 0; j < sequences; ++j) rank += static_cast<std::uint32_t>(lane_u32(key, j) > key);
  }
  const auto sorted = [&](std::uint32_t x) {
    return static_cast<std::uint32_t>(__builtin_amdgcn_ds_permute(static_cast<int>(4 * rank), static_cast<int>(x)));
  };
  q.row0 = sorted(q.row0);
  q.n = sorted(q.n);
  q.ctx = sorted(q.ctx);
  q.valid = sorted(q.valid) != 0;
  id = sorted(id);
  blocks = sorted(blocks);
  lo = sorted(lo);
  tiles = sorted(tiles);
}

// Finds item `index` of the batch; false: there are fewer.  By a whole wave, 64 sequences at a
// time.  `first`: the caller is the one wave that counts bad sequences, in `count`, and writes the
// plan for the kernel that joins the ranges.  With kRounds the items of up to 64 sequences are
// the longest first and their ranges' length is chosen (16 query and 4 KV heads, against an even
// share in the batch's order, in a graph, us: 300 tokens of 30000 291 -> 189, 200 of 60000 374 -> 255, 16 sequences of
// up to 8192 behind a window of 4096, ten of them single tokens, 260 -> 185; it takes a workgroup 1.6 to 6 us, of 1 to 64
// sequences).
template <int kCols, int kUnit, bool kRounds = false>
__device__ __forceinline__ bool paged_find(const PagedArgs &a, const PagedSplit &sp, const PagedScratch &sc, std::uint32_t index, bool first,
                                           unsigned int *count, PagedItem &item) {
  const std::uint32_t lane = threadIdx.x & 63;
  std::uint64_t work = 0;
  std::uint32_t live = 0;
  PagedSeq q{};
  std::uint32_t blocks = 0, lo = 1, tiles = 1, bad = 0, id = lane;
  for (std::uint32_t s0 = 0; s0 < a.sequences; s0 += 64) {
    blocks = 0;
    if (s0 + lane < a.sequences) {
      q = paged_seq(a, s0 + lane);
      paged_extent<kCols, kUnit>(a, q, blocks, tiles);
      bad += !q.valid;
    }
    const std::uint64_t w = static_cast<std::uint64_t>(blocks) * tiles;
    live += __builtin_popcountll(__builtin_amdgcn_ballot_w64(blocks != 0));
    work += lane_u32(wave_prefix(static_cast<std::uint32_t>(w) & 0xFFFFFFu), 63);
    if (__builtin_amdgcn_ballot_w64(w >> 24 != 0) != 0)
      work += static_cast<std::uint64_t>(lane_u32(wave_prefix(static_cast<std::uint32_t>(w >> 24)), 63)) << 24;
  }
  if (first && bad != 0) atomicAdd(count, bad);
  const std::uint32_t bits = sp.slot_bits + (live >= sp.many ? sp.many_bits : 0);
  const std::uint64_t share = (work + (std::uint64_t{1} << bits) - 1) >> bits;
  std::uint32_t t = share >> 28 != 0 ? 1u << 28 : share > sp.least ? static_cast<std::uint32_t>(share) : sp.least;
  if (kRounds && a.sequences <= 64) {
    paged_sort<kUnit>(q, id, blocks, lo, tiles, a.sequences);
    t = paged_rounds(blocks, lo, tiles, t, bits, a.sequences, sp.least);
  }
  if (first && sp.parts != 0) {
    std::uint32_t split = 0;
    for (std::uint32_t s0 = 0; s0 < a.sequences; s0 += 64) {
      if (a.sequences > 64) {
        blocks = 0;
        if (s0 + lane < a.sequences) paged_extent<kCols, kUnit>(a, paged_seq(a, s0 + lane), blocks, tiles);
      }
      split += lane_u32(wave_prefix(tiles > t ? blocks : 0), 63);
    }
    if (lane == 0) {
      sc.plan[0] = t;
      sc.plan[1] = split;
    }
  }
  return paged_pick<kCols, kUnit>(a, index, false, t, q, id, blocks, tiles, item);
}
// Finds split column block `index` for the kernel that joins its ranges.
template <int kCols, int kUnit, bool kRounds = false>
__device__ __forceinline__ bool paged_find_split(const PagedArgs &a, const PagedScratch &sc, std::uint32_t index, PagedItem &item) {
  const std::uint32_t lane = threadIdx.x & 63;
  const std::uint32_t t = sc.plan[0];
  PagedSeq q{};
  std::uint32_t blocks = 0, lo = 1, tiles = 1, id = lane;
  if (lane < a.sequences) {
    q = paged_seq(a, lane);
    paged_extent<kCols, kUnit>(a, q, blocks, tiles);
  }
  if (kRounds && a.sequences <= 64) paged_sort<kUnit>(q, id, blocks, lo, tiles, a.sequences);
  return paged_pick<kCols, kUnit>(a, index, true, t, q, id, blocks, tiles, item);
}

// A column block's tokens and keys, and its ranges of about equal length.
struct PagedBlock {
  std::uint32_t col0, col_end;    // of its sequence's columns
  std::uint32_t tok0;             // first token
  std::uint32_t p_lo, p_hi;       // its tokens' positions
  std::uint32_t first_key;        // that any of them sees
  std::uint32_t first, total;     // tiles
  std::uint32_t count, each, more; // ranges; the first `more` have a tile above `each`
  __device__ __forceinline__ std::uint32_t begin(std::uint32_t i) const { return first + i * each + (i < more ? i : more); }
};

template <int kCols, int kUnit>
__device__ __forceinline__ PagedBlock paged_block(const PagedArgs &a, const PagedItem &it, std::uint32_t block) {
  // (columns are fewer than 2^22: the quotient is column * (2^30 / group + 1) >> 30)
  const auto token = [&](std::uint32_t col) {
    return static_cast<std::uint32_t>(static_cast<std::uint64_t>(col) * a.group_inverse30 >> 30);
  };
  const std::uint32_t cols = it.seq.n * a.group, past = it.seq.ctx - it.seq.n;
  PagedBlock b;
  b.col0 = block * kCols;
  b.col_end = cols - b.col0 < kCols ? cols : b.col0 + kCols;
  b.tok0 = token(b.col0);
  b.p_lo = past + b.tok0;
  b.p_hi = past + token(b.col_end - 1);
  b.first_key = a.window != 0 && b.p_lo >= a.window ? b.p_lo - a.window + 1 : 0;
  b.first = b.first_key / kUnit;
  b.total = b.p_hi / kUnit + 1 - b.first;
  b.count = 1;
  b.each = b.total;
  b.more = 0;
  if (it.ranges > 1) {
    b.count = scalar((b.total + it.range_tiles - 1) / it.range_tiles);
    b.count = b.count < it.ranges ? b.count : it.ranges;
    b.each = scalar(b.total / b.count);
    b.more = b.total - b.each * b.count;
  }
  return b;
}

// Whether a token at position p sees key j.  (no branches)
__device__ __forceinline__ bool paged_sees(std::uint32_t j, std::uint32_t p, std::uint32_t window) {
  return (j <= p) & ((window == 0) | (p - j < window));
}

// NaN to the rows of a block's columns.
template <int kThreads>
__device__ __forceinline__ void paged_fill_nan(const PagedArgs &a, const PagedItem &it, std::uint32_t col0, std::uint32_t cols,
                                               std::uint32_t kvh) {
  const std::uint32_t all = it.seq.n * a.group;
  for (std::uint32_t i = threadIdx.x; i < cols * (kHeadDim / 2); i += kThreads) {
    const std::uint32_t col = col0 + i / (kHeadDim / 2), d = i % (kHeadDim / 2);
    if (col >= all) break;
    const std::uint32_t tok = col / a.group, h = col - tok * a.group;
    *reinterpret_cast<std::uint32_t *>(a.output + (it.seq.row0 + tok) * a.o_row + (kvh * a.group + h) * a.o_head + 2 * d) = 0x7FC07FC0u;
  }
}

// ------------------------------------------------------------- launches
// Chunks with much work (paged_prefill.hip).
constexpr std::uint32_t kStreamBlockCols = 128, kStreamUnit = 32;
void launch_paged_stream(const PagedArgs &a, const PagedScratch &sc, const PagedSplit &sp, std::uint32_t items,
                         std::uint32_t split_blocks, hipStream_t stream);
std::uint32_t paged_take_stream_errors();
std::size_t paged_decode_workspace(const PagedArgs &a);
void paged_decode(const PagedArgs &a, void *workspace, hipStream_t stream);
std::size_t paged_prefill_workspace(const PagedArgs &a);
void paged_prefill(const PagedArgs &a, void *workspace, hipStream_t stream);

struct PagedAppendArgs {
  PagedArgs paged; // query, output and their strides; no gate
  const bf16_bits *key, *value;
  unsigned char *pages;
  const double *frequencies;
  const void *q_weight, *k_weight;
  bool weight_f32, interleaved;
  std::size_t k_row, k_head, v_row, v_head;
  std::uint32_t rotary_dim, units_inverse; // 2^32 / heads of a row + 1 (set by paged_append)
  float magnitude, epsilon;
};
void paged_append(const PagedAppendArgs &a, hipStream_t stream);

// Take (read and clear) the counts of bad sequences and pages, of attention calls and of appends.
std::uint32_t paged_take_capacity_errors();
std::uint32_t paged_take_append_errors();

} // namespace raftinfer::amd
