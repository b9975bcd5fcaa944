// Attention over the paged KV cache by waves that split the keys: single tokens, and
// chunks with little work.
#include "paged_cache.hpp"
#include "compact_cache.hpp"
#include "prefill_tile.hpp"

#include <algorithm>

namespace raftinfer::amd {
namespace {

using prefill::fexp2;
using prefill::kLazyRescale;

__device__ unsigned int g_paged_capacity_errors = 0;

// A slot holds one step's K or V: 16 rows of 512 bytes, 16-byte chunk c of row r at
// c ^ rows_key(r): a pass of the K reads takes one chunk of 16 rows, of the transposed V
// reads 32 bytes of 8 rows.  (Linear in the bits of r.)
constexpr int kSlotBytes = kPageGranule * kRowBytes;
__device__ __forceinline__ constexpr std::uint32_t rows_key(std::uint32_t r, bool is_v) { return is_v ? 2 * (r & 7) : r & 15; }

template <int WAVES> struct RowsShared {
  union {
    alignas(1024) unsigned char rows[WAVES][2][kSlotBytes]; // K, V
    // (the pad puts the 16 columns of a store on banks of their own)
    float acc[WAVES][16][kHeadDim + 4];
  };
  float m[WAVES][32], l[WAVES][32];
};

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float(static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(x)), lane)));
}
// Two values cut to bf16.
__device__ __forceinline__ std::uint32_t cut_bf16x2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// A workgroup takes 16 CB columns of one sequence and KV head and a range of their keys; wave
// w takes the range's steps (16 keys) w, w + WAVES, ..  S = K q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32_bf16, operands out of LDS, where LDS-direct loads put the rows as
// they lie in the pages; K(t + 1) is asked for when K(t) has been read, V(t + 1) when V(t)
// has.  A product with V takes 16 keys in its 32 places: the probabilities in two bf16
// parts, 16 bits together.
template <int CB, int WAVES, bool Stream>
__global__ __launch_bounds__(WAVES *kWave, 8 / WAVES) void paged_rows_kernel(PagedArgs a, PagedScratch sc, PagedSplit sp) {
  __shared__ RowsShared<WAVES> sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col16 = lane & 15, kq = lane >> 4;
  const std::uint32_t index = scalar(blockIdx.x / a.kv_heads), kvh = blockIdx.x - index * a.kv_heads;
  PagedItem it;
  if (!paged_find<16 * CB, kPageGranule>(a, sp, index, false, blockIdx.x == 0 && wave == 0 ? &g_paged_capacity_errors : nullptr, it)) return;
  const std::uint32_t range = scalar(it.local / it.blocks), block = it.blocks - 1 - (it.local - range * it.blocks); // longest first
  if (!it.seq.valid) {
    paged_fill_nan<WAVES * kWave>(a, it, block * 16 * CB, 16 * CB, kvh);
    return;
  }
  const PagedBlock b = paged_block<16 * CB, kPageGranule>(a, it, block);
  if (range >= b.count) return;
  const std::uint32_t begin = b.begin(range), end = b.begin(range + 1);
  const bool part = b.count > 1;
  const std::uint32_t slot = it.first_part + block * it.ranges + range;
  if (part && slot >= sp.parts) return; // (only where sequences share rows)

  // Column x of the block (those past the last repeat it): its row of query, gate, output.  (The
  // quotient of fewer than 2^8 columns from a token's first.)
  const std::uint32_t in_first = b.col0 - b.tok0 * a.group, last_x = b.col_end - 1 - b.col0;
  const auto place = [&](std::uint32_t x, std::uint32_t &tok, std::uint32_t &head) {
    const std::uint32_t c = in_first + (x < last_x ? x : last_x), t = c * a.group_inverse >> 16;
    tok = b.tok0 + t;
    head = kvh * a.group + (c - t * a.group);
  };
  bf16x8 qb[CB][8];
  std::uint32_t pos[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    std::uint32_t tok, head;
    place(16 * cb + col16, tok, head);
    pos[cb] = it.seq.ctx - it.seq.n + tok;
    const bf16_bits *q = a.query + (it.seq.row0 + tok) * a.q_row + head * a.q_head + 8 * kq;
#pragma unroll
    for (int i = 0; i < 8; ++i) qb[cb][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(q + 32 * i));
  }

  const std::uint32_t steps = begin + wave < end ? (end - begin - wave + WAVES - 1) / WAVES : 0;
  const auto granule = [&](std::uint32_t t) { return begin + wave + WAVES * t; };
  // Lane l: the first row of step t0 + l.
  bool bad = false;
  std::uint32_t row_of = 0;
  const auto load_table = [&](std::uint32_t t0) {
    row_of = t0 + lane < steps ? paged_row(a, it.id, kvh, granule(t0 + lane) * kPageGranule, bad) : 0;
  };
  const unsigned slots = lds_address(sh.rows[wave][0]);
  const std::uint32_t in_row = lane >> 5, chunk = lane & 31, row_bytes = a.row_step * kRowBytes;
  const auto load = [&](std::uint32_t t, bool is_v) __attribute__((always_inline)) {
    const std::uint32_t row = lane_u32(row_of, t & 63) + (is_v ? a.plane_rows : 0);
    const unsigned char *base = a.pages + static_cast<std::size_t>(row) * kRowBytes;
    const unsigned to = slots + (is_v ? kSlotBytes : 0);
    const std::uint32_t last = b.p_hi - granule(t) * kPageGranule; // rows past it repeat it
    const std::uint32_t off = 16 * (chunk ^ rows_key(in_row, is_v));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const std::uint32_t r = 2 * i + in_row;
      load_lds_b128(base, (r < last ? r : last) * row_bytes + (off ^ (16 * rows_key(2 * i, is_v))), to + 1024 * i);
    }
  };
  if (steps != 0) load_table(0);
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(qb[cb][i]));
  if (steps != 0) {
    load(0, false);
    load(0, true);
  }

  const unsigned k_lane = slots + kRowBytes * col16 + 16 * (kq ^ rows_key(col16, false));
  const std::uint32_t v_row = 4 * kq + (col16 >> 2);
  const unsigned v_lane = slots + kSlotBytes + kRowBytes * v_row + (16 * ((col16 >> 1 & 1) ^ rows_key(v_row, true)) + 8 * (col16 & 1));

  floatx4 acc[CB][16]; // dims 16 db + 4 kq + e of the lane's column
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int db = 0; db < 16; ++db) acc[cb][db] = floatx4{};
  float m_run[CB], l_run[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m_run[cb] = -FLT_MAX;
    l_run[cb] = 0.f;
  }
  std::uint64_t odd = 0; // lanes that took infinite or NaN values out of a masked step

#pragma unroll 1
  for (std::uint32_t t = 0; t < steps; ++t) {
    const std::uint32_t j0 = granule(t) * kPageGranule;
    // some column does not see some key
    const bool masked = j0 + kPageGranule - 1 > b.p_lo || (a.window != 0 && b.p_hi - j0 >= a.window);
    if ((t + 1) % 64 == 0 && t + 1 < steps) load_table(t + 1);
    wait_vm<8>(); // K(t)
    floatx4 s[CB];
    {
      floatx4 s1[CB];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) s[cb] = s1[cb] = floatx4{};
      bf16x8 op[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) op[i] = lds_operand(k_lane ^ (64u * i));
#pragma unroll
      for (int i = 0; i < 8; i += 2)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          s[cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op[i], qb[cb][i], s[cb], 0, 0, 0);
          s1[cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op[i + 1], qb[cb][i + 1], s1[cb], 0, 0, 0);
        }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) s[cb] += s1[cb];
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkm0(); // the reads are done: their place is free
    const bool more = t + 1 < steps;
    if (more) load(t + 1, false);
    constexpr float kScale = kLog2e / 16.0f;
    bool grow = false;
    float mx[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[cb][i] *= kScale;
        if (masked) s[cb][i] = paged_sees(j0 + 4 * kq + i, pos[cb], a.window) ? s[cb][i] : -INFINITY;
      }
      mx[cb] = max_xor32(max_xor16(fmaxf(fmaxf(s[cb][0], s[cb][1]), fmaxf(s[cb][2], s[cb][3]))));
      grow |= mx[cb] > m_run[cb];
    }
    // m_run lies 2^8 above the max that it was last set to: no probability exceeds 1, and the
    // accumulators are seldom scaled.
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        const float m_new = mx[cb] > m_run[cb] ? mx[cb] + kLazyRescale : m_run[cb], f = fexp2(m_run[cb] - m_new);
        l_run[cb] *= f;
#pragma unroll
        for (int db = 0; db < 16; ++db) acc[cb][db] *= f;
        m_run[cb] = m_new;
      }
    }
    // In two parts: the first, cut to bf16 below p (1 - 2^-9), and what it leaves.  Neither is 0 or
    // negative where p is not, so that an infinite value gives that and no NaN.
    u32x4 pw[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = fexp2(s[cb][i] - m_run[cb]);
        l_run[cb] += e[i];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = e[2 * i], y = e[2 * i + 1];
        const std::uint32_t w = cut_bf16x2(fmaf(x, -0x1p-9f, x), fmaf(y, -0x1p-9f, y));
        pw[cb][i] = w;
        pw[cb][2 + i] = pack_bf16x2(x - bf16_lo(w), y - bf16_hi(w));
      }
    }
    if (more) wait_vm<8>(); else wait_vm<0>(); // V(t)
    if (masked) {
      // A masked key has probability 0, and 0 times an infinite or NaN value is not 0: such
      // values are taken out here and added behind the loop, to the columns that see them.
      // (A value is odd if its exponent's bits are all set.)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned at = slots + kSlotBytes + 1024 * i + 16 * lane;
        u32x4 w = __builtin_bit_cast(u32x4, lds_operand(at));
        std::uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const std::uint32_t top = ((w[e] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
          any |= top;
          w[e] &= ~((top >> 15) * 0xFFFFu);
        }
        if (any != 0) *(__attribute__((address_space(3))) u32x4 *)(std::uintptr_t)(at) = w;
        odd |= __builtin_amdgcn_ballot_w64(any != 0);
      }
      wave_lds_order();
    }
    // k-slot (kq, e) of the product <-> key 4 kq + e % 4.  Operands are read kRing products ahead.
    constexpr int kRing = 8;
    u32x2 op[kRing];
#pragma unroll
    for (int db = 0; db < kRing; ++db) op[db] = lds_tr_operand(v_lane ^ (32u * db));
#pragma unroll
    for (int db = 0; db < 16; ++db) {
      const u32x2 w = op[db % kRing];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
        acc[cb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[0], w[1]}),
                                                              __builtin_bit_cast(bf16x8, pw[cb]), acc[cb][db], 0, 0, 0);
      if (db + kRing < 16) op[db % kRing] = lds_tr_operand(v_lane ^ (32u * (db + kRing)));
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_lgkm0();
    if (more) load(t + 1, true);
  }
  if (odd != 0) {
#pragma unroll 1
    for (std::uint32_t t = 0; t < steps; ++t) {
      const std::uint32_t j0 = granule(t) * kPageGranule;
      if (j0 + kPageGranule - 1 <= b.p_lo && (a.window == 0 || b.p_hi - j0 < a.window)) continue;
      bool ignored = false;
      const std::uint32_t row0 = paged_row(a, it.id, kvh, j0, ignored) + a.plane_rows;
#pragma unroll 1
      for (std::uint32_t j = j0; j < j0 + kPageGranule && j <= b.p_hi; ++j) {
        const auto *row = reinterpret_cast<const bf16_bits *>(a.pages + static_cast<std::size_t>(row0 + (j - j0) * a.row_step) * kRowBytes) + 4 * kq;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          if (!paged_sees(j, pos[cb], a.window)) continue;
#pragma unroll
          for (int db = 0; db < 16; ++db) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(row + 16 * db);
            const float v[4] = {bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[cb][db][e] += is_finite_f32(v[e]) ? 0.f : v[e];
          }
        }
      }
    }
  }
  if (__builtin_amdgcn_ballot_w64(bad) != 0) {
    if (lane == 0) atomicAdd(&g_paged_capacity_errors, 1u);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) l_run[cb] = __builtin_nanf("");
  }

  // Join the waves, 16 columns at a time: a wave takes every WAVES-th column, a lane four dims.
  wait_vm<0>();
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    __syncthreads();
    const float l_all = sum_xor32(sum_xor16(l_run[cb]));
    if (kq == 0) {
      sh.m[wave][col16] = m_run[cb];
      sh.l[wave][col16] = l_all;
    }
#pragma unroll
    for (int db = 0; db < 16; ++db) *reinterpret_cast<floatx4 *>(&sh.acc[wave][col16][16 * db + 4 * kq]) = acc[cb][db];
    __syncthreads();
    float m = -FLT_MAX, l = 0.f, share[WAVES]; // of column `col16`
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, sh.m[w][col16]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      share[w] = fexp2(sh.m[w][col16] - m);
      l = fmaf(sh.l[w][col16], share[w], l);
    }
    const std::size_t at = (static_cast<std::size_t>(slot) * a.kv_heads + kvh) * (16 * CB) + 16 * cb;
    if (part && threadIdx.x < 16) {
      sc.m[at + lane] = m;
      sc.l[at + lane] = l;
    }
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < 16 / WAVES; ++i) {
      const int x = WAVES * i + wave;
      if (b.col0 + 16 * cb + x >= b.col_end) continue;
      floatx4 o{};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) o += *reinterpret_cast<const floatx4 *>(&sh.acc[w][x][4 * lane]) * lane_value(share[w], x);
      if (part) {
        *reinterpret_cast<floatx4 *>(sc.o + (at + x) * kHeadDim + 4 * lane) = o;
        continue;
      }
      o *= lane_value(inv, x);
      std::uint32_t tok, head;
      place(16 * cb + x, tok, head);
      if (a.gate != nullptr) {
        const u32x2 g = *reinterpret_cast<const u32x2 *>(a.gate + (it.seq.row0 + tok) * a.g_row + head * a.g_head + 4 * lane);
        o[0] *= sigmoid_gate(bf16_lo(g[0])); o[1] *= sigmoid_gate(bf16_hi(g[0]));
        o[2] *= sigmoid_gate(bf16_lo(g[1])); o[3] *= sigmoid_gate(bf16_hi(g[1]));
      }
      *reinterpret_cast<u32x2 *>(a.output + (it.seq.row0 + tok) * a.o_row + head * a.o_head + 4 * lane) =
          u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
    }
  }
}

// Joins the ranges of the split column blocks: grid (columns of a block / (4 / W), split blocks times
// KV heads); W waves per column take its ranges in turn, a lane four dims.
constexpr int kMergeWaves = 4;
template <int CB, int W>
__global__ __launch_bounds__(kMergeWaves *kWave) void paged_merge_kernel(PagedArgs a, PagedScratch sc, PagedSplit sp) {
  __shared__ float o_of[kMergeWaves][kHeadDim];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr std::uint32_t kCols = 16 * CB;
  const std::uint32_t index = scalar(blockIdx.y / a.kv_heads), kvh = blockIdx.y - index * a.kv_heads;
  PagedItem it;
  if (!paged_find<kCols, kPageGranule>(a, sp, index, true, nullptr, it)) return;
  const PagedBlock b = paged_block<kCols, kPageGranule>(a, it, it.local);
  if (b.count == 1) return;
  const std::uint32_t x = blockIdx.x * (kMergeWaves / W) + wave / W, col = b.col0 + x;
  const bool mine = col < b.col_end;
  if (W == 1 && !mine) return;
  const std::uint32_t part0 = it.first_part + it.local * it.ranges;
  if (part0 + b.count > sp.parts) return; // (only where sequences share rows)
  if (W > 1 && b.col0 + blockIdx.x * (kMergeWaves / W) >= b.col_end) return; // (uniform)
  const std::size_t stride = static_cast<std::size_t>(a.kv_heads) * kCols; // between parts
  const std::size_t at0 = part0 * stride + static_cast<std::size_t>(kvh) * kCols + (mine ? x : b.col_end - 1 - b.col0);
  const std::uint32_t tok = (mine ? col : b.col_end - 1) / a.group, head = kvh * a.group + ((mine ? col : b.col_end - 1) - tok * a.group);
  u32x2 g{};
  if (a.gate != nullptr) g = *reinterpret_cast<const u32x2 *>(a.gate + (it.seq.row0 + tok) * a.g_row + head * a.g_head + 4 * lane);
  constexpr int kBatch = 8;
  floatx4 o_in[kBatch];
  const auto load = [&](std::uint32_t s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const std::uint32_t s = s0 + W * i < b.count ? s0 + W * i : b.count - 1;
      o_in[i] = *reinterpret_cast<const floatx4 *>(sc.o + (at0 + s * stride) * kHeadDim + 4 * lane);
    }
  };
  const std::uint32_t s_first = W == 1 ? 0 : wave % W;
  load(s_first);
  // max and sum over the ranges; those without a key that the column sees have l = 0
  float m = -FLT_MAX, l = 0.f;
  for (std::uint32_t s = lane; s < b.count; s += 64) {
    const float ms = sc.m[at0 + s * stride], ls = sc.l[at0 + s * stride];
    const float m_new = fmaxf(m, ms);
    l = l * fexp2(m - m_new) + ls * fexp2(ms - m_new);
    m = m_new;
  }
  const float m_all = wave_max(m);
  const float inv = 1.0f / wave_sum(l * fexp2(m - m_all));
  floatx4 o{};
  for (std::uint32_t s0 = s_first; s0 < b.count; s0 += W * kBatch) {
    if (s0 != s_first) load(s0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const std::uint32_t s = s0 + W * i;
      if (s >= b.count) break;
      o += o_in[i] * fexp2(sc.m[at0 + s * stride] - m_all);
    }
  }
  if constexpr (W > 1) {
    *reinterpret_cast<floatx4 *>(&o_of[wave][4 * lane]) = o;
    __syncthreads();
    if (wave % W != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) o += *reinterpret_cast<const floatx4 *>(&o_of[wave + w][4 * lane]);
  }
  if (!mine) return;
  o *= inv;
  if (a.gate != nullptr) {
    o[0] *= sigmoid_gate(bf16_lo(g[0])); o[1] *= sigmoid_gate(bf16_hi(g[0]));
    o[2] *= sigmoid_gate(bf16_lo(g[1])); o[3] *= sigmoid_gate(bf16_hi(g[1]));
  }
  *reinterpret_cast<u32x2 *>(a.output + (it.seq.row0 + tok) * a.o_row + head * a.o_head + 4 * lane) =
      u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

// What any batch of a shape takes, per KV head.
struct Bounds {
  PagedSplit split;
  std::uint32_t items, split_blocks;
};
std::uint32_t floor_log2(std::uint32_t x) {
  std::uint32_t n = 0;
  while (x >> (n + 1) != 0) ++n;
  return n;
}
Bounds bounds_of(const PagedArgs &a, std::uint32_t block_cols, std::uint32_t unit, std::uint32_t least, std::uint32_t workgroups) {
  Bounds r{};
  const std::uint32_t slot_bits = workgroups > a.kv_heads ? floor_log2(workgroups / a.kv_heads) : 0;
  r.split = {least, slot_bits, 0};
  const std::uint64_t seqs = std::min(a.sequences, a.rows);
  const std::uint64_t blocks = (static_cast<std::uint64_t>(a.rows) * a.group + seqs * (block_cols - 1)) / block_cols;
  std::uint64_t tiles = (static_cast<std::uint64_t>(a.max_ctx) + unit - 1) / unit;
  if (a.window != 0) tiles = std::min<std::uint64_t>(tiles, (static_cast<std::uint64_t>(a.window) + block_cols + unit) / unit + 2);
  const std::uint64_t ranges = (tiles + least - 1) / least, slots = std::uint64_t{1} << slot_bits;
  r.items = static_cast<std::uint32_t>(std::min(blocks * ranges, blocks + slots));
  r.split_blocks = ranges == 1 ? 0 : static_cast<std::uint32_t>(std::min(blocks, slots));
  r.split.parts = ranges == 1 ? 0 : static_cast<std::uint32_t>(std::min(blocks * ranges, 2 * slots));
  return r;
}
PagedScratch scratch_of(const PagedArgs &a, const PagedSplit &sp, std::uint32_t block_cols, void *workspace, std::size_t *bytes) {
  const std::size_t cols = static_cast<std::size_t>(sp.parts) * a.kv_heads * block_cols;
  auto *p = static_cast<float *>(workspace);
  if (bytes != nullptr) *bytes = cols * (kHeadDim + 2) * sizeof(float);
  return {p, p + cols, p + 2 * cols};
}

Bounds decode_bounds(const PagedArgs &a) { return bounds_of(a, 16, kPageGranule, 32, 512); }
Bounds few_bounds(const PagedArgs &a) { return bounds_of(a, 32, kPageGranule, 32, 512); }
Bounds stream_bounds(const PagedArgs &a) { return bounds_of(a, kStreamBlockCols, kStreamUnit, 8, 256); }
bool streams(const PagedArgs &a) { return a.rows * a.group >= 1024; }

template <int CB, int W> void launch_merge(const PagedArgs &a, const PagedScratch &sc, const Bounds &bd, hipStream_t stream) {
  if (bd.split_blocks == 0) return;
  const dim3 grid{16 * CB / (kMergeWaves / W), bd.split_blocks * a.kv_heads};
  paged_merge_kernel<CB, W><<<grid, kMergeWaves * kWave, 0, stream>>>(a, sc, bd.split);
}

} // namespace

std::size_t paged_decode_workspace(const PagedArgs &a) {
  std::size_t bytes = 0;
  (void)scratch_of(a, decode_bounds(a).split, 16, nullptr, &bytes);
  return bytes;
}
void paged_decode(const PagedArgs &a, void *workspace, hipStream_t stream) {
  const Bounds bd = decode_bounds(a);
  const PagedScratch sc = scratch_of(a, bd.split, 16, workspace, nullptr);
  paged_rows_kernel<1, 4, true><<<bd.items * a.kv_heads, 4 * kWave, 0, stream>>>(a, sc, bd.split);
  launch_merge<1, 4>(a, sc, bd, stream);
}

std::size_t paged_prefill_workspace(const PagedArgs &a) {
  std::size_t few = 0, much = 0;
  (void)scratch_of(a, few_bounds(a).split, 32, nullptr, &few);
  (void)scratch_of(a, stream_bounds(a).split, kStreamBlockCols, nullptr, &much);
  return std::max(few, much);
}
void paged_prefill(const PagedArgs &a, void *workspace, hipStream_t stream) {
  if (streams(a)) {
    const Bounds bd = stream_bounds(a);
    const PagedScratch sc = scratch_of(a, bd.split, kStreamBlockCols, workspace, nullptr);
    void *count = nullptr;
    if (hipGetSymbolAddress(&count, HIP_SYMBOL(g_paged_capacity_errors)) != hipSuccess) return;
    launch_paged_stream(a, sc, bd.split, bd.items, bd.split_blocks, static_cast<unsigned int *>(count), stream);
    return;
  }
  const Bounds bd = few_bounds(a);
  const PagedScratch sc = scratch_of(a, bd.split, 32, workspace, nullptr);
  paged_rows_kernel<2, 4, false><<<bd.items * a.kv_heads, 4 * kWave, 0, stream>>>(a, sc, bd.split);
  launch_merge<2, 1>(a, sc, bd, stream);
}

std::uint32_t paged_take_capacity_errors() {
  unsigned int value = 0;
  const unsigned int zero = 0;
  if (hipMemcpyFromSymbol(&value, HIP_SYMBOL(g_paged_capacity_errors), sizeof value) != hipSuccess ||
      hipMemcpyToSymbol(HIP_SYMBOL(g_paged_capacity_errors), &zero, sizeof zero) != hipSuccess)
    throw std::runtime_error("reading the capacity error counter failed");
  return value;
}

} // namespace raftinfer::amd
