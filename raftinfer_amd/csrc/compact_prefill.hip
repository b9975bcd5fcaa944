// Prompt attention over the compact KV cache, and the key weights of its last
// tokens.
#include "compact_cache.hpp"
#include "prefill_tile.hpp"

#include <cfloat>

namespace raftinfer::amd {
namespace {

using prefill::fexp2;
using prefill::kLazyRescale;
using prefill::lds_b128;
using prefill::lds_tr16;

constexpr int kPWaves = 4;
constexpr int kPThreads = kPWaves * kWave;
constexpr int kPCols = 32 * kPWaves; // columns (token, head of the group) per workgroup
constexpr int kTileElems = kCompactBlock * kHeadDim;
constexpr std::uint32_t kPrefillTarget = 512; // workgroups that a call aims at: two per CU

// Partials of a split call, [split][kv_head][column], and the final max (exp2
// domain) and 1 / sum of each column for the key weights.
struct PrefillScratch {
  float *m, *l, *o, *final;
  std::uint32_t splits, cols; // cols: rounded up to whole workgroups
};

struct PrefillShared {
  bf16_bits k[2][kTileElems]; // 16-byte chunk c of row r at c ^ (r & 7)
  bf16_bits v[2][kTileElems];
  std::uint32_t odd[2]; // the tile in slot i has infinite or NaN values
};

__device__ __forceinline__ int tile_at(int r, int c) { return r * kHeadDim + ((c ^ (r & 7)) << 3); }

__device__ __forceinline__ std::uint32_t odd_bits(std::uint32_t w) {
  return ((w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u) ? 1u : 0u;
}

// A workgroup takes 128 columns (column = token * group + head) of one KV head and a
// contiguous range of the 32-key tiles that they see; a wave takes 32 columns.  The
// tiles pass through two LDS slots, as bf16, shared by the waves.  S^T = K Q^T and
// O^T = V^T P^T on v_mfma_f32_32x32x16_bf16, Q and O in registers.
template <bool Fp8, bool Split>
__global__ __launch_bounds__(kPThreads, 2) void compact_prefill_kernel(CompactArgs a, PrefillScratch sc) {
  __shared__ PrefillShared sh;
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

  const std::uint32_t col = col0 + 32 * wave + n32;
  const std::uint32_t col_in = col < all_cols ? col : all_cols - 1; // columns past the last repeat it
  const std::uint32_t tok = col_in / a.group;
  const std::uint32_t pos = a.past + tok;
  const std::size_t io_row =
      (static_cast<std::size_t>(tok) * a.kv_heads + kvh) * a.group + (col_in - tok * a.group);

  bf16x8 q[16];
  {
    const bf16_bits *src = a.query + io_row * kHeadDim + 8 * kh;
#pragma unroll
    for (int s = 0; s < 16; ++s) q[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(src + 16 * s));
  }
  if (tid < 2) sh.odd[tid] = 0;

  // Staging: rows past the last key repeat it (their scores are masked).
  constexpr int kStage = Fp8 ? 4 : 1;
  [[maybe_unused]] u32x4 st[kStage];
  const auto load_tile = [&](std::uint32_t it, int slot) {
    const std::uint32_t j0 = seen.tile(it) * kCompactBlock;
    const std::uint32_t last = n_keys - 1 - j0; // >= 0: the tile has a key
    if constexpr (Fp8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        std::uint32_t r = 16 * i + (tid >> 4);
        r = r < last ? r : last;
        const std::size_t off = static_cast<std::size_t>(j0 + r) * c.row + 16 * (tid & 15);
        st[2 * i] = *reinterpret_cast<const u32x4 *>(c.k + off);
        st[2 * i + 1] = *reinterpret_cast<const u32x4 *>(c.v + off);
      }
    } else {
      const unsigned lk = lds_address(sh.k[slot]), lv = lds_address(sh.v[slot]);
      const bf16_bits *kb = c.k + static_cast<std::size_t>(j0) * c.row, *vb = c.v + static_cast<std::size_t>(j0) * c.row;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int inst = 4 * wave + i;
        const int r = 2 * inst + kh;
        const std::uint32_t rr = static_cast<std::uint32_t>(r) < last ? r : last;
        const std::uint32_t voff = rr * static_cast<std::uint32_t>(c.row * 2) + 16u * (n32 ^ (r & 7));
        load_lds_b128(kb, voff, lk + 1024u * inst);
        load_lds_b128(vb, voff, lv + 1024u * inst);
      }
    }
  };
  const auto store_tile = [&](int slot) {
    if constexpr (Fp8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 16 * i + (tid >> 4), piece = tid & 15;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          *reinterpret_cast<u32x4 *>(sh.k[slot] + tile_at(r, 2 * piece + h)) = fp8x8_to_bf16(st[2 * i][2 * h], st[2 * i][2 * h + 1]);
          *reinterpret_cast<u32x4 *>(sh.v[slot] + tile_at(r, 2 * piece + h)) = fp8x8_to_bf16(st[2 * i + 1][2 * h], st[2 * i + 1][2 * h + 1]);
        }
      }
    } else {
      wait_vm<0>();
    }
  };

  // Operand addresses: K row n32, chunk 2 s + kh; V by transposed reads, where lane r
  // of a 16-lane group supplies 4 dims of key row r / 4 and receives its dim of 4 keys.
  int k_at[4], v_at[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) k_at[j] = tile_at(n32, 2 * j + kh);
  {
    const int g = lane >> 4, r = lane & 15;
    const int row = 4 * kh + (r >> 2);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int d = 32 * j + 16 * (g & 1) + 4 * (r & 3);
      v_at[j] = tile_at(row, d >> 3) + (d & 7);
    }
  }

  floatx16 o[8];
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) o[nb] = floatx16{};
  float m_run = -FLT_MAX, l_run = 0.f;

  if (begin < end) {
    load_tile(begin, 0);
    store_tile(0);
  }
  __syncthreads();
  for (std::uint32_t it = begin; it < end; ++it) {
    const int slot = (it - begin) & 1;
    const std::uint32_t tile = seen.tile(it);
    const std::uint32_t j0 = tile * kCompactBlock;
    const bool more = it + 1 < end;
    if (more) load_tile(it + 1, slot ^ 1);
    float k_scale = kLog2e / 16.0f;
    [[maybe_unused]] float v_scale = 1.0f;
    if constexpr (Fp8) {
      k_scale *= c.ks[tile];
      v_scale = c.vs[tile];
    }
    const bf16_bits *kt = sh.k[slot], *vt = sh.v[slot];
    // Some column does not see some key of the tile (the same for every wave).
    const bool masked = j0 + kCompactBlock - 1 > p_lo ||
                        (a.window != 0 && j0 + kCompactBlock > a.sinks && p_hi - j0 >= a.window);
    bool odd = false;
    if (masked) {
      // A masked key has probability 0, and 0 times an infinite or NaN value is not
      // 0: such a tile takes another path, key by key.
      std::uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(vt + 8 * (tid + kPThreads * i));
        bad |= odd_bits(w[0]) | odd_bits(w[1]) | odd_bits(w[2]) | odd_bits(w[3]);
      }
      if (__builtin_amdgcn_ballot_w64(bad != 0) != 0 && lane == 0) sh.odd[slot] = tile + 1;
      __syncthreads();
      odd = sh.odd[slot] == tile + 1;
    }

    floatx16 s = floatx16{};
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      bf16x8 ka[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) ka[j] = lds_b128(kt + k_at[j] + 64 * b);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[j], q[4 * b + j], s, 0, 0, 0);
    }
    // Register i holds key j0 + 8 (i / 4) + 4 kh + i % 4 of this lane's column.
    float mx = -INFINITY;
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const std::uint32_t j = j0 + 8 * (i >> 2) + 4 * kh + (i & 3);
        s[i] = compact_sees(j, pos, a.window, a.sinks) ? s[i] * k_scale : -INFINITY;
        mx = fmaxf(mx, s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] *= k_scale;
        mx = fmaxf(mx, s[i]);
      }
    }
    mx = max_xor32(mx);
    // The accumulators are scaled only where a max grows by more than 2^8, which
    // the probabilities can exceed 1 by.
    const bool grow = mx > m_run + kLazyRescale;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float m_new = grow ? mx : m_run;
      const float f = grow ? fexp2(m_run - mx) : 1.0f;
      l_run *= f;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) o[nb] *= f;
      m_run = m_new;
    }
    float p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = fexp2(s[i] - m_run);
      l_run += p[i];
      if constexpr (Fp8) p[i] *= v_scale;
    }
    if (!odd) {
      // k-slot (kb, kh, e) <-> key 16 kb + 8 (e / 4) + 4 kh + e % 4, the order of p.
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const u32x4 w{pack_bf16x2(p[8 * kb], p[8 * kb + 1]), pack_bf16x2(p[8 * kb + 2], p[8 * kb + 3]),
                      pack_bf16x2(p[8 * kb + 4], p[8 * kb + 5]), pack_bf16x2(p[8 * kb + 6], p[8 * kb + 7])};
        const bf16x8 pb = __builtin_bit_cast(bf16x8, w);
#pragma unroll
        for (int nb = 0; nb < 8; ++nb) {
          const bf16_bits *v0 = vt + v_at[nb & 1] + 64 * (nb >> 1) + 16 * kb * kHeadDim;
          const u32x2 lo = lds_tr16(v0), hi = lds_tr16(v0 + 8 * kHeadDim);
          o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]}),
                                                          pb, o[nb], 0, 0, 0);
        }
      }
    } else {
#pragma unroll 1
      for (int r = 0; r < kCompactBlock; ++r) {
        // p of key r: register 4 (r / 8) + r % 4 of the column's lane with kh = r / 4 % 2
        float pr = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) pr = i == 4 * (r >> 3) + (r & 3) ? p[i] : pr;
        pr = __shfl(pr, n32 + 32 * ((r >> 2) & 1));
        const bool sees = compact_sees(j0 + r, pos, a.window, a.sinks);
#pragma unroll
        for (int nb = 0; nb < 8; ++nb) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int d = 32 * nb + 8 * x + 4 * kh;
            const u32x2 w = *reinterpret_cast<const u32x2 *>(vt + tile_at(r, d >> 3) + (d & 7));
            const float v0 = bf16_lo(w[0]), v1 = bf16_hi(w[0]), v2 = bf16_lo(w[1]), v3 = bf16_hi(w[1]);
            o[nb][4 * x] += sees ? pr * v0 : 0.f;
            o[nb][4 * x + 1] += sees ? pr * v1 : 0.f;
            o[nb][4 * x + 2] += sees ? pr * v2 : 0.f;
            o[nb][4 * x + 3] += sees ? pr * v3 : 0.f;
          }
        }
      }
    }
    if (more) store_tile(slot ^ 1);
    __syncthreads();
  }

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
    const std::size_t base = io_row * kHeadDim + 4 * kh;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const std::size_t at = base + 32 * nb + 8 * x;
        const u32x2 g = *reinterpret_cast<const u32x2 *>(a.gate + at);
        const float r0 = o[nb][4 * x] * inv * sigmoid_gate(bf16_lo(g[0]));
        const float r1 = o[nb][4 * x + 1] * inv * sigmoid_gate(bf16_hi(g[0]));
        const float r2 = o[nb][4 * x + 2] * inv * sigmoid_gate(bf16_lo(g[1]));
        const float r3 = o[nb][4 * x + 3] * inv * sigmoid_gate(bf16_hi(g[1]));
        *reinterpret_cast<u32x2 *>(a.output + at) = u32x2{pack_bf16x2(r0, r1), pack_bf16x2(r2, r3)};
      }
  }
}

// Joins a split call: a wave per column, a lane four dims.
__global__ __launch_bounds__(kPThreads) void compact_prefill_merge_kernel(CompactArgs a, PrefillScratch sc) {
  const std::uint32_t col = blockIdx.x * kPWaves + (threadIdx.x >> 6);
  const std::uint32_t kvh = blockIdx.y;
  const int lane = threadIdx.x & 63;
  if (col >= a.tokens * a.group) return;
  float m = -FLT_MAX;
  for (std::uint32_t s = 0; s < sc.splits; ++s)
    m = fmaxf(m, sc.m[(static_cast<std::size_t>(s) * a.kv_heads + kvh) * sc.cols + col]);
  float l = 0.f;
  floatx4 o{};
  for (std::uint32_t s = 0; s < sc.splits; ++s) {
    const std::size_t at = (static_cast<std::size_t>(s) * a.kv_heads + kvh) * sc.cols + col;
    const float ls = sc.l[at], ms = sc.m[at];
    if (ls == 0.f && ms == -FLT_MAX) continue; // the split holds no key that the column sees
    const float f = fexp2(ms - m);
    l = fmaf(ls, f, l);
    o += *reinterpret_cast<const floatx4 *>(sc.o + at * kHeadDim + 4 * lane) * f;
  }
  const float inv = 1.0f / l;
  if (a.weights != nullptr && lane == 0) {
    const std::size_t at = static_cast<std::size_t>(kvh) * sc.cols + col;
    sc.final[2 * at] = m;
    sc.final[2 * at + 1] = inv;
  }
  const std::uint32_t tok = col / a.group;
  const std::size_t at =
      ((static_cast<std::size_t>(tok) * a.kv_heads + kvh) * a.group + (col - tok * a.group)) * kHeadDim + 4 * lane;
  const u32x2 g = *reinterpret_cast<const u32x2 *>(a.gate + at);
  const float r0 = o[0] * inv * sigmoid_gate(bf16_lo(g[0])), r1 = o[1] * inv * sigmoid_gate(bf16_hi(g[0]));
  const float r2 = o[2] * inv * sigmoid_gate(bf16_lo(g[1])), r3 = o[3] * inv * sigmoid_gate(bf16_hi(g[1]));
  *reinterpret_cast<u32x2 *>(a.output + at) = u32x2{pack_bf16x2(r0, r1), pack_bf16x2(r2, r3)};
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

// Key splits of a call whose widest column block sees `tiles` tiles.
std::uint32_t split_count(const CompactArgs &a, std::uint32_t tiles) {
  const std::uint64_t groups = static_cast<std::uint64_t>(col_blocks(a)) * a.kv_heads;
  std::uint64_t splits = groups >= kPrefillTarget ? 1 : kPrefillTarget / groups;
  if (splits > (tiles + 3) / 4) splits = (tiles + 3) / 4; // at least four tiles each
  return static_cast<std::uint32_t>(splits);
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
  if (splits > 1) {
    compact_prefill_kernel<Fp8, true><<<grid, kPThreads, 0, stream>>>(a, sc);
    compact_prefill_merge_kernel<<<dim3{(a.tokens * a.group + kPWaves - 1) / kPWaves, a.kv_heads}, kPThreads, 0, stream>>>(a, sc);
  } else {
    compact_prefill_kernel<Fp8, false><<<grid, kPThreads, 0, stream>>>(a, sc);
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
