// Attention over the paged KV cache by waves that split the keys: single tokens, and
// chunks with little work.
#include "paged_cache.hpp"
#include "compact_cache.hpp"
#include "prefill_stream.hpp"

#include <algorithm>

namespace raftinfer::amd {
namespace {

using prefill::fexp2;
using prefill::kLazyRescale;

__device__ unsigned int g_paged_capacity_errors = 0;

// A form of the kernel: 16 CB columns a workgroup, WAVES waves, steps of 16 G keys.
template <int CB_, int WAVES_, int G_> struct Form {
  static constexpr int CB = CB_, WAVES = WAVES_, G = G_;
  static constexpr int kCols = 16 * CB, kKeys = kPageGranule * G, kThreads = WAVES * kWave;
  static constexpr int kLoads = 8 * G;                 // of a plane of a step, 1 KiB each
  static constexpr unsigned kPlane = kLoads * 1024;    // bytes
};
using DecodeForm = Form<1, 4, 1>;
using FewForm = Form<2, 4, 2>;

// 16-byte chunk c of row r of a granule lies at c ^ rows_key(r): a pass of the K reads takes one
// chunk of 16 rows, of the transposed V reads 32 bytes of 8 rows.  (Linear in the bits of r.)
__device__ __forceinline__ constexpr std::uint32_t rows_key(std::uint32_t r, bool is_v) { return is_v ? 2 * (r & 7) : r & 15; }

template <class F> struct RowsShared {
  union {
    alignas(1024) unsigned char rows[F::WAVES][2][F::kPlane]; // K, V
    // (the pad puts the 16 columns of a store on banks of their own)
    float acc[F::WAVES][16][kHeadDim + 4];
  };
  float m[F::WAVES][16], l[F::WAVES][16];
};

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float(static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(x)), lane)));
}
// Two values cut to bf16.
__device__ __forceinline__ std::uint32_t cut_bf16x2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// load_lds_b128_at; Once: the memory is not read again.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int kOffset, bool Once> __device__ __forceinline__ void load_rows(const void *base, std::uint32_t voff, unsigned lds) {
  if constexpr (Once)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3 nt" : : "s"(lds), "v"(voff), "s"(base), "n"(kOffset) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" : : "s"(lds), "v"(voff), "s"(base), "n"(kOffset) : "memory", "m0");
}
#pragma clang diagnostic pop

// A workgroup takes the columns of one block of one KV head and a range of their keys; wave w takes the
// range's steps w, w + WAVES, ..  S = K q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16, operands
// out of LDS, where LDS-direct loads put the rows as they lie in the pages: whole granules, whose rows
// behind the last key are masked, and cleaned, like other keys that a column does not see.  A product
// with V has 32 places: of 16 keys (G = 1) the probabilities in two bf16 parts, which cost nothing there (off by
// 2^-15 + 2^-17 of themselves at most), of 32 keys one part, 8 bits: two would double those products.  What bounds it: long caches the memory (32 sequences of up to 32768 tokens 6.05 TB/s, one of 60001 6.3 in
// the kernel; non-temporal loads where more than 16 MiB are read once: 6.05 against 5.3 TB/s plain, but warm small caches
// are slower with them), short calls the round trips: of 15 us for 16 tokens of 217, 1.4 to find the work, 2 for the table
// and the first keys, 2.5 for the queries, 4 for two steps, 4 to join the waves.
template <class F, bool HeadMajor, bool Once>
__global__ __launch_bounds__(F::kThreads, 1) void paged_rows_kernel(PagedArgs a, PagedScratch sc, PagedSplit sp) {
  constexpr int CB = F::CB, WAVES = F::WAVES, G = F::G, L = F::kLoads;
  __shared__ RowsShared<F> sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col16 = lane & 15, kq = lane >> 4;
  const std::uint32_t index = scalar(blockIdx.x / a.kv_heads), kvh = blockIdx.x - index * a.kv_heads;
  PagedItem it;
  if (!paged_find<F::kCols, F::kKeys>(a, sp, sc, index, blockIdx.x == 0 && wave == 0, &g_paged_capacity_errors, it)) return;
  const std::uint32_t range = scalar(it.local / it.blocks), block = it.blocks - 1 - (it.local - range * it.blocks); // longest first
  if (!it.seq.valid) {
    paged_fill_nan<F::kThreads>(a, it, block * F::kCols, F::kCols, kvh);
    return;
  }
  const PagedBlock b = paged_block<F::kCols, F::kKeys>(a, it, block);
  if (range >= b.count) return;
  const std::uint32_t begin = b.begin(range), end = b.begin(range + 1);
  const bool part = b.count > 1;
  const std::uint32_t slot = it.first_part + block * it.ranges + range;
  if (part && slot >= sp.parts) return; // (only where sequences share rows)

  const std::uint32_t steps = begin + wave < end ? (end - begin - wave + WAVES - 1) / WAVES : 0;
  const auto tile_of = [&](std::uint32_t t) { return begin + wave + WAVES * t; };
  // Lane l: first K row of granule l % G of step t0 + l / G.  A granule in front of the first key or
  // behind the last repeats theirs.
  std::uint64_t bad = 0; // lanes that met a bad page
  std::uint32_t row_of = 0, t0 = 0;
  const auto load_table = [&](std::uint32_t from) __attribute__((always_inline)) {
    t0 = from;
    const std::uint32_t first = b.first_key / kPageGranule, last = b.p_hi / kPageGranule;
    std::uint32_t g = tile_of(from + lane / G) * G + lane % G;
    g = g < first ? first : g < last ? g : last;
    bool wrong = false;
    row_of = paged_row(a, it.id, kvh, g * kPageGranule, wrong);
    bad |= __builtin_amdgcn_ballot_w64(wrong);
  };
  // Of a granule's rows 2 i, 2 i + 1 for load i.  (The instruction's offset counts for both addresses: the
  // lane's is less by as much; rows are at least 512 bytes apart.)
  const std::uint32_t row_bytes = HeadMajor ? kRowBytes : a.row_step * kRowBytes, skip = 2 * (row_bytes - kRowBytes);
  const std::uint32_t off_row = (lane >> 5) * row_bytes;
  const std::uint32_t off_k = off_row + 16 * ((lane & 31) ^ rows_key(lane >> 5, false)), off_v = off_row + 16 * ((lane & 31) ^ rows_key(lane >> 5, true));
  const unsigned k_plane = lds_address(sh.rows[wave][0]), v_plane = k_plane + F::kPlane;
  const auto load = [&](std::uint32_t t, auto is_v) __attribute__((always_inline)) {
    prefill::static_for<L>([&](auto ic) __attribute__((always_inline)) {
      constexpr int g = ic / 8, i = ic % 8;
      const std::uint32_t row = lane_u32(row_of, (t - t0) * G + g) + (is_v ? a.plane_rows : 0);
      const unsigned char *base = a.pages + static_cast<std::size_t>(row) * kRowBytes + (i >> 2) * 8 * (HeadMajor ? kRowBytes : row_bytes);
      std::uint32_t off = (is_v ? off_v : off_k) ^ (16 * rows_key(2 * i, is_v));
      if constexpr (!HeadMajor && (i & 3) != 0) off += (i & 3) * skip;
      load_rows<1024 * (i & 3), Once>(base, off, (is_v ? v_plane : k_plane) + 8192 * g + 4096 * (i >> 2));
    });
  };
  constexpr std::false_type kIsK{};
  constexpr std::true_type kIsV{};

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
  if (steps != 0) {
    load_table(0);
    load(0, kIsK);
  }
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    std::uint32_t tok, head;
    place(16 * cb + col16, tok, head);
    pos[cb] = it.seq.ctx - it.seq.n + tok;
    const bf16_bits *q = a.query + (it.seq.row0 + tok) * a.q_row + head * a.q_head + 8 * kq;
#pragma unroll
    for (int i = 0; i < 8; ++i) qb[cb][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(q + 32 * i));
  }
  // (the wait for q is one for every load in front of it: K(0), but for no other)
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(qb[cb][i]));
  if (steps != 0) load(0, kIsV);
  // The gates of the columns that this wave writes: every WAVES-th of 16, four dims a lane.
  constexpr int kMine = 16 / WAVES;
  [[maybe_unused]] u32x2 gate[CB][kMine];
  const bool gated = a.gate != nullptr && !part;
  if (gated) {
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        std::uint32_t tok, head;
        place(16 * cb + WAVES * i + wave, tok, head);
        gate[cb][i] = *reinterpret_cast<const u32x2 *>(a.gate + (it.seq.row0 + tok) * a.g_row + head * a.g_head + 4 * lane);
      }
  }

  const unsigned k_lane = kRowBytes * col16 + 16 * (kq ^ rows_key(col16, false));
  const std::uint32_t v_row = 4 * kq + (col16 >> 2);
  const unsigned v_lane = kRowBytes * v_row + (16 * ((col16 >> 1 & 1) ^ rows_key(v_row, true)) + 8 * (col16 & 1));

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
  const auto masked = [&](std::uint32_t j0) { // some column does not see some key
    return j0 + F::kKeys - 1 > b.p_lo || (a.window != 0 && b.p_hi - j0 >= a.window);
  };

#pragma unroll 1
  for (std::uint32_t t = 0; t < steps; ++t) {
    const std::uint32_t j0 = tile_of(t) * F::kKeys;
    const bool hide = masked(j0), more = t + 1 < steps;
    if ((t + 1 - t0) * G >= 64 && more) load_table(t + 1);
    wait_vm<L>(); // K(t): V(t) is behind it
    floatx4 s[CB][G]; // keys j0 + 16 g + 4 kq + e
    {
      const unsigned k_base = k_plane + k_lane;
      const auto read_k = [&](int i) { return lds_operand((k_base ^ (64u * (i / G))) + 8192u * (i % G)); };
      constexpr int kRing = 8;
      bf16x8 op[kRing];
#pragma unroll
      for (int i = 0; i < kRing; ++i) op[i] = read_k(i);
      floatx4 two[CB][2]{}; // two chains: even and odd k-steps (G = 1), or a granule each
#pragma unroll
      for (int i = 0; i < 8 * G; ++i) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
          two[cb][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op[i % kRing], qb[cb][i / G], two[cb][i & 1], 0, 0, 0);
        if (i + kRing < 8 * G) op[i % kRing] = read_k(i + kRing);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        if constexpr (G == 1) s[cb][0] = two[cb][0] + two[cb][1];
        else { s[cb][0] = two[cb][0]; s[cb][G - 1] = two[cb][1]; }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkm0(); // the reads are done: their place is free
    if (more) load(t + 1, kIsK);
    constexpr float kScale = kLog2e / 16.0f;
    bool grow = false;
    float mx[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      if (hide) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[cb][g][i] = paged_sees(j0 + 16 * g + 4 * kq + i, pos[cb], a.window) ? s[cb][g][i] : -INFINITY;
      }
      float x = fmaxf(fmaxf(s[cb][0][0], s[cb][0][1]), fmaxf(s[cb][0][2], s[cb][0][3]));
      if constexpr (G == 2) x = fmaxf(x, fmaxf(fmaxf(s[cb][1][0], s[cb][1][1]), fmaxf(s[cb][1][2], s[cb][1][3])));
      mx[cb] = max_xor32(max_xor16(x)) * kScale;
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
    u32x4 pw[CB]; // the product's k-slots (kq, e): key 4 kq + e % 4, of granule e / 4 where there are two
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = fexp2(fmaf(s[cb][g][i], kScale, -m_run[cb]));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = e[2 * i], y = e[2 * i + 1];
          if constexpr (G == 1) {
            // In two parts: the first, cut to bf16 below p (1 - 2^-9), and what it leaves.  Neither is 0
            // or negative where p is not, so that an infinite value gives that and no NaN.
            const std::uint32_t w = cut_bf16x2(fmaf(x, -0x1p-9f, x), fmaf(y, -0x1p-9f, y));
            pw[cb][i] = w;
            pw[cb][2 + i] = pack_bf16x2(x - bf16_lo(w), y - bf16_hi(w));
            l_run[cb] += x + y;
          } else { // the sum takes the same rounded probabilities as the product
            pw[cb][2 * g + i] = pack_bf16x2(x, y);
            l_run[cb] = dot2_bf16(pw[cb][2 * g + i], 0x3F803F80u, l_run[cb]);
          }
        }
      }
    }
    if (more) wait_vm<L>(); else wait_vm<0>(); // V(t): K(t + 1) is behind it
    if (hide) {
      // A masked key has probability 0, and 0 times an infinite or NaN value is not 0: such
      // values are taken out here and added behind the loop, to the columns that see them.
      // (A value is odd if its exponent's bits are all set.)
#pragma unroll 4
      for (int i = 0; i < L; ++i) {
        const unsigned at = v_plane + 1024 * i + 16 * lane;
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
    // Operands are read kRing products ahead.
    constexpr int kRing = 8;
    const unsigned v_base = v_plane + v_lane;
    const auto read_v = [&](int db) {
      const u32x2 lo = lds_tr_operand(v_base ^ (32u * db));
      if constexpr (G == 1) return lo;
      else {
        const u32x2 hi = lds_tr_operand((v_base ^ (32u * db)) + 8192u);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    std::conditional_t<G == 1, u32x2, u32x4> op[kRing];
#pragma unroll
    for (int db = 0; db < kRing; ++db) op[db] = read_v(db);
#pragma unroll
    for (int db = 0; db < 16; ++db) {
      const auto w = op[db % kRing];
      u32x4 v;
      if constexpr (G == 1) v = u32x4{w[0], w[1], w[0], w[1]}; else v = w;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
        acc[cb][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, pw[cb]), acc[cb][db], 0, 0, 0);
      if (db + kRing < 16) op[db % kRing] = read_v(db + kRing);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_lgkm0();
    if (more) load(t + 1, kIsV);
  }
  if (odd != 0) {
#pragma unroll 1
    for (std::uint32_t t = 0; t < steps; ++t) {
      const std::uint32_t j0 = tile_of(t) * F::kKeys;
      if (!masked(j0)) continue;
#pragma unroll 1
      for (std::uint32_t j = j0 > b.first_key ? j0 : b.first_key; j < j0 + F::kKeys && j <= b.p_hi; ++j) {
        bool ignored = false;
        const std::uint32_t row = paged_row(a, it.id, kvh, j, ignored) + a.plane_rows;
        const auto *v_at = reinterpret_cast<const bf16_bits *>(a.pages + static_cast<std::size_t>(row) * kRowBytes) + 4 * kq;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          if (!paged_sees(j, pos[cb], a.window)) continue;
#pragma unroll
          for (int db = 0; db < 16; ++db) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(v_at + 16 * db);
            const float v[4] = {bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[cb][db][e] += is_finite_f32(v[e]) ? 0.f : v[e];
          }
        }
      }
    }
  }
  if (bad != 0) {
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
    const std::size_t at = (static_cast<std::size_t>(slot) * a.kv_heads + kvh) * F::kCols + 16 * cb;
    if (part && threadIdx.x < 16) {
      sc.m[at + lane] = m;
      sc.l[at + lane] = l;
    }
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
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
      if (gated) {
        const u32x2 g = gate[cb][i];
        o[0] *= sigmoid_gate(bf16_lo(g[0])); o[1] *= sigmoid_gate(bf16_hi(g[0]));
        o[2] *= sigmoid_gate(bf16_lo(g[1])); o[3] *= sigmoid_gate(bf16_hi(g[1]));
      }
      *reinterpret_cast<u32x2 *>(a.output + (it.seq.row0 + tok) * a.o_row + head * a.o_head + 4 * lane) =
          u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
    }
  }
}

// Joins the ranges of the split column blocks: grid (columns of a block / WAVES, split blocks times KV
// heads); a wave takes a column, a lane four dims, eight ranges' rows at a time on the way.
template <class F, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void paged_merge_kernel(PagedArgs a, PagedScratch sc, PagedSplit sp) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr std::uint32_t kCols = F::kCols;
  const std::uint32_t index = scalar(blockIdx.y / a.kv_heads), kvh = blockIdx.y - index * a.kv_heads;
  PagedItem it;
  if (!paged_find_split<kCols, F::kKeys>(a, sc, index, it)) return;
  const PagedBlock b = paged_block<kCols, F::kKeys>(a, it, it.local);
  if (b.count == 1) return;
  const std::uint32_t x = blockIdx.x * WAVES + wave, col = b.col0 + x;
  if (col >= b.col_end) return;
  const std::uint32_t part0 = it.first_part + it.local * it.ranges;
  if (part0 + b.count > sp.parts) return; // (only where sequences share rows)
  const std::size_t stride = static_cast<std::size_t>(a.kv_heads) * kCols; // between parts
  const std::size_t at0 = part0 * stride + static_cast<std::size_t>(kvh) * kCols + x;
  const std::uint32_t c = b.col0 - b.tok0 * a.group + x, t = c * a.group_inverse >> 16;
  const std::uint32_t tok = b.tok0 + t, head = kvh * a.group + (c - t * a.group);
  u32x2 g{};
  if (a.gate != nullptr) g = *reinterpret_cast<const u32x2 *>(a.gate + (it.seq.row0 + tok) * a.g_row + head * a.g_head + 4 * lane);
  constexpr int kBatch = 8;
  floatx4 o_in[kBatch];
  const auto load = [&](std::uint32_t s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const std::uint32_t s = s0 + i < b.count ? s0 + i : b.count - 1;
      o_in[i] = *reinterpret_cast<const floatx4 *>(sc.o + (at0 + s * stride) * kHeadDim + 4 * lane);
    }
  };
  load(0);
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
  for (std::uint32_t s0 = 0; s0 < b.count; s0 += kBatch) {
    if (s0 != 0) load(s0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const std::uint32_t s = s0 + i;
      if (s >= b.count) break;
      o += o_in[i] * fexp2(sc.m[at0 + s * stride] - m_all);
    }
  }
  o *= inv;
  if (a.gate != nullptr) {
    o[0] *= sigmoid_gate(bf16_lo(g[0])); o[1] *= sigmoid_gate(bf16_hi(g[0]));
    o[2] *= sigmoid_gate(bf16_lo(g[1])); o[3] *= sigmoid_gate(bf16_hi(g[1]));
  }
  *reinterpret_cast<u32x2 *>(a.output + (it.seq.row0 + tok) * a.o_row + head * a.o_head + 4 * lane) =
      u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

// The same for single tokens, whose ranges can be many and columns few: grid (4 quarters of the dims times
// heads of the group, split blocks times KV heads).  A wave loads 64 dims of four ranges' rows at a time.
constexpr int kDecodeJoin = 4; // waves
__global__ __launch_bounds__(kDecodeJoin *kWave) void paged_decode_merge_kernel(PagedArgs a, PagedScratch sc, PagedSplit sp) {
  __shared__ floatx4 o_of[kDecodeJoin][16];
  const int lane = threadIdx.x & 63, quad = lane & 15, sub = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  using F = DecodeForm;
  const std::uint32_t index = scalar(blockIdx.y / a.kv_heads), kvh = blockIdx.y - index * a.kv_heads;
  const std::uint32_t x = blockIdx.x >> 2; // head of the group
  const int dim = 64 * (blockIdx.x & 3) + 4 * quad;
  PagedItem it;
  if (!paged_find_split<F::kCols, F::kKeys>(a, sc, index, it)) return;
  const PagedBlock b = paged_block<F::kCols, F::kKeys>(a, it, it.local);
  if (b.count == 1) return;
  const std::uint32_t part0 = it.first_part + it.local * it.ranges;
  if (part0 + b.count > sp.parts) return; // (only where sequences share rows)
  const std::size_t stride = static_cast<std::size_t>(a.kv_heads) * F::kCols; // between parts
  const std::size_t at0 = part0 * stride + static_cast<std::size_t>(kvh) * F::kCols + x;
  const std::size_t head = kvh * a.group + x;
  u32x2 g{};
  if (a.gate != nullptr) g = *reinterpret_cast<const u32x2 *>(a.gate + it.seq.row0 * a.g_row + head * a.g_head + dim);
  constexpr int kBatch = 4, kEvery = 4 * kDecodeJoin;
  float m_run = -FLT_MAX, l = 0.f; // of the lane's ranges (the 16 lanes of a row alike)
  floatx4 o{};
  for (std::uint32_t s0 = 4 * wave + sub; s0 - sub < b.count; s0 += kBatch * kEvery) {
    floatx4 in[kBatch];
    float m[kBatch], ls[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const bool there = s0 + k * kEvery < b.count;
      const std::size_t at = at0 + (there ? s0 + k * kEvery : b.count - 1) * stride;
      m[k] = sc.m[at];
      ls[k] = sc.l[at];
      in[k] = *reinterpret_cast<const floatx4 *>(sc.o + at * kHeadDim + dim);
      if (!there) { // (counted once, by its own lane)
        m[k] = -FLT_MAX;
        ls[k] = 0.f;
        in[k] = floatx4{};
      }
    }
    float m_new = m_run;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) m_new = fmaxf(m_new, m[k]);
    const float f = fexp2(m_run - m_new);
    l *= f;
    o *= f;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float fk = fexp2(m[k] - m_new);
      l += ls[k] * fk;
      o += in[k] * fk;
    }
    m_run = m_new;
  }
  // over the four rows of a wave, then over the waves
  const float m_wave = max_xor32(max_xor16(m_run)), f = fexp2(m_run - m_wave);
  l = sum_xor32(sum_xor16(l * f));
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = sum_xor32(sum_xor16(o[e] * f));
  __shared__ float m_of[kDecodeJoin], l_of[kDecodeJoin];
  if (lane < 16) o_of[wave][lane] = o;
  if (lane == 0) {
    m_of[wave] = m_wave;
    l_of[wave] = l;
  }
  __syncthreads();
  if (threadIdx.x >= 16) return;
  float m_all = -FLT_MAX, l_all = 0.f;
  floatx4 y{};
#pragma unroll
  for (int w = 0; w < kDecodeJoin; ++w) m_all = fmaxf(m_all, m_of[w]);
#pragma unroll
  for (int w = 0; w < kDecodeJoin; ++w) {
    const float fw = fexp2(m_of[w] - m_all);
    l_all += l_of[w] * fw;
    y += o_of[w][lane] * fw;
  }
  y *= 1.0f / l_all;
  if (a.gate != nullptr) {
    y[0] *= sigmoid_gate(bf16_lo(g[0])); y[1] *= sigmoid_gate(bf16_hi(g[0]));
    y[2] *= sigmoid_gate(bf16_lo(g[1])); y[3] *= sigmoid_gate(bf16_hi(g[1]));
  }
  *reinterpret_cast<u32x2 *>(a.output + it.seq.row0 * a.o_row + head * a.o_head + dim) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
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
Bounds bounds_of(const PagedArgs &a, std::uint32_t block_cols, std::uint32_t unit, std::uint32_t least, std::uint32_t workgroups,
                 std::uint32_t many, std::uint32_t many_bits, bool rounds = false) {
  Bounds r{};
  const std::uint32_t slot_bits = workgroups > a.kv_heads ? floor_log2(workgroups / a.kv_heads) : 0;
  r.split = {least, slot_bits, many, many_bits, 0};
  const std::uint64_t seqs = std::min(a.sequences, a.rows);
  const std::uint64_t blocks = (static_cast<std::uint64_t>(a.rows) * a.group + seqs * (block_cols - 1)) / block_cols;
  std::uint64_t tiles = (static_cast<std::uint64_t>(a.max_ctx) + unit - 1) / unit;
  if (a.window != 0) tiles = std::min<std::uint64_t>(tiles, (static_cast<std::uint64_t>(a.window) + block_cols + unit) / unit + 2);
  const std::uint64_t ranges = (tiles + least - 1) / least, slots = std::uint64_t{1} << (slot_bits + (seqs >= many || rounds ? many_bits : 0));
  r.items = static_cast<std::uint32_t>(std::min(blocks * ranges, blocks + slots));
  r.split_blocks = ranges == 1 ? 0 : static_cast<std::uint32_t>(std::min(blocks, slots));
  r.split.parts = ranges == 1 ? 0 : static_cast<std::uint32_t>(std::min({blocks * ranges, blocks + slots, 2 * slots}));
  return r;
}
PagedScratch scratch_of(const PagedArgs &a, const PagedSplit &sp, std::uint32_t block_cols, void *workspace, std::size_t *bytes) {
  const std::size_t cols = static_cast<std::size_t>(sp.parts) * a.kv_heads * block_cols;
  auto *p = static_cast<float *>(workspace);
  if (bytes != nullptr) *bytes = sp.parts == 0 ? 0 : cols * (kHeadDim + 2) * sizeof(float) + 16;
  return {p, p + cols, p + 2 * cols, reinterpret_cast<std::uint32_t *>(p + cols * (kHeadDim + 2))};
}

Bounds decode_bounds(const PagedArgs &a) { return bounds_of(a, DecodeForm::kCols, DecodeForm::kKeys, 32, 256, 2, 2); }
// Whether the caches are read past the last-level cache: where they could hold more than 16 MiB.
bool reads_once(const PagedArgs &a) {
  return static_cast<std::uint64_t>(a.sequences) * a.max_ctx * a.kv_heads * 2 * kRowBytes > (16u << 20);
}
Bounds few_bounds(const PagedArgs &a) { return bounds_of(a, FewForm::kCols, FewForm::kKeys, 16, 256, 8, 1); }
Bounds stream_bounds(const PagedArgs &a) { return bounds_of(a, kStreamBlockCols, kStreamUnit, 8, 256, 1u << 31, 1, true); }
// Which kernel a chunk takes, by the (column, key) pairs of all heads that the sequences can have: the
// stream kernel fetches a key once for 128 columns and keeps the matrix units busy, but its start and end cost
// about 15 us of every workgroup (ring, 256 accumulator registers, the joining of its key groups).  Up to 40
// squares of 32 x 32 pairs for each of 256 workgroups the rows kernel is the faster (16 query and 4 KV heads, us, rows
// kernel first: 512 tokens 20.5 / 38.6, 1000 43.7 / 57.4, 500 of 1500 37.5 / 44.2, 64 of 4000 25.3 / 37.6, 16 of
// 30000 56.7 / 69.6), above it the stream kernel (100 of 8000 68.3 / 51.5, 300 of 4000 78.4 / 56.4, 500 of 30501 and
// 8001: twice as fast and more).  Several sequences: 4 of up to 500 tokens 41.5 / 42.6, 8 with 7 single tokens up to 8000
// 105 / 80, 16 with up to 8192 behind a window of 4096, in a graph, 289 / 185.  Where the rows kernel would take a third round of
// workgroups, few keys or not, the stream kernel is the faster too (windows of 32 and 200: 900 tokens 26.7 / 26.6 and 31.4 / 35.3,
// 1200 38.1 / 22.3 and 46.1 / 36.3), unless its blocks would be half empty (600 sequences of 2 tokens 136 / 195).
bool streams(const PagedArgs &a) {
  const std::uint64_t seqs = std::min(a.sequences, a.rows);
  const std::uint64_t each = std::min<std::uint64_t>((a.rows + seqs - 1) / seqs, a.max_ctx);
  std::uint64_t keys = a.max_ctx - each / 2; // in the mean
  if (a.window != 0) keys = std::min<std::uint64_t>(keys, std::uint64_t{a.window} + 32);
  const std::uint64_t columns = static_cast<std::uint64_t>(a.rows) * a.group * a.kv_heads;
  return columns * keys > 40u * 256 * 32 * 32 || (columns > 2u * 256 * 32 && each * a.group >= 2 * 32);
}

template <class F, bool Once> void launch_rows(const PagedArgs &a, const PagedScratch &sc, const Bounds &bd, hipStream_t stream) {
  const auto go = [&](auto kernel) { kernel<<<bd.items * a.kv_heads, F::kThreads, 0, stream>>>(a, sc, bd.split); };
  go(a.row_step == 1 ? paged_rows_kernel<F, true, Once> : paged_rows_kernel<F, false, Once>);
}

} // namespace

std::size_t paged_decode_workspace(const PagedArgs &a) {
  std::size_t bytes = 0;
  (void)scratch_of(a, decode_bounds(a).split, DecodeForm::kCols, nullptr, &bytes);
  return bytes;
}
void paged_decode(const PagedArgs &a, void *workspace, hipStream_t stream) {
  const Bounds bd = decode_bounds(a);
  const PagedScratch sc = scratch_of(a, bd.split, DecodeForm::kCols, workspace, nullptr);
  if (reads_once(a)) launch_rows<DecodeForm, true>(a, sc, bd, stream);
  else launch_rows<DecodeForm, false>(a, sc, bd, stream);
  if (bd.split_blocks != 0)
    paged_decode_merge_kernel<<<dim3{4 * a.group, bd.split_blocks * a.kv_heads}, kDecodeJoin * kWave, 0, stream>>>(a, sc, bd.split);
}

std::size_t paged_prefill_workspace(const PagedArgs &a) {
  std::size_t few = 0, much = 0;
  (void)scratch_of(a, few_bounds(a).split, FewForm::kCols, nullptr, &few);
  (void)scratch_of(a, stream_bounds(a).split, kStreamBlockCols, nullptr, &much);
  return std::max(few, much);
}
void paged_prefill(const PagedArgs &a, void *workspace, hipStream_t stream) {
  if (streams(a)) {
    const Bounds bd = stream_bounds(a);
    const PagedScratch sc = scratch_of(a, bd.split, kStreamBlockCols, workspace, nullptr);
    launch_paged_stream(a, sc, bd.split, bd.items, bd.split_blocks, stream);
    return;
  }
  const Bounds bd = few_bounds(a);
  const PagedScratch sc = scratch_of(a, bd.split, FewForm::kCols, workspace, nullptr);
  launch_rows<FewForm, false>(a, sc, bd, stream);
  if (bd.split_blocks != 0)
    paged_merge_kernel<FewForm, 4><<<dim3{FewForm::kCols / 4, bd.split_blocks * a.kv_heads}, 4 * kWave, 0, stream>>>(a, sc, bd.split);
}

std::uint32_t paged_take_capacity_errors() {
  unsigned int value = 0;
  const unsigned int zero = 0;
  if (hipMemcpyFromSymbol(&value, HIP_SYMBOL(g_paged_capacity_errors), sizeof value) != hipSuccess ||
      hipMemcpyToSymbol(HIP_SYMBOL(g_paged_capacity_errors), &zero, sizeof zero) != hipSuccess)
    throw std::runtime_error("reading the capacity error counter failed");
  return value + paged_take_stream_errors();
}

} // namespace raftinfer::amd
