// Decode attention over the compact KV cache: one new token per sequence.
#include "compact_cache.hpp"
#include "prefill_tile.hpp"

#include <cfloat>

namespace raftinfer::amd {
namespace {

using prefill::fexp2;
using prefill::lds_tr16;

constexpr int kDecodeWaves = 4;
constexpr int kDecodeThreads = kDecodeWaves * kWave;
// Workgroups that a call aims at: two per CU, twice.
constexpr std::uint32_t kDecodeTarget = 1024;

__device__ unsigned int g_compact_capacity_errors = 0;

// Partials of a call, one per (query head, partition): max and sum (exp2 domain),
// and the unnormalised output; with key weights also every score and each
// head's final max and 1 / sum.
struct DecodeScratch {
  float *m, *l, *o, *scores, *final;
  std::uint32_t tiles, parts, score_stride;
};

__device__ __forceinline__ std::uint32_t context_of(const CompactArgs &a, std::uint32_t seq) {
  return a.lengths == nullptr ? a.past + 1 : a.lengths[seq];
}

struct DecodeShared {
  union {
    bf16_bits v[kDecodeWaves][kCompactBlock * kHeadDim]; // 16-byte chunk c of row r at c ^ (r & 7)
    float acc[kDecodeWaves][kCompactMaxGroup][kHeadDim];
  };
  float m[kDecodeWaves][kCompactMaxGroup];
  float l[kDecodeWaves][kCompactMaxGroup];
};

// A workgroup takes one partition (sc.tiles 32-key tiles) of one KV head and
// sequence; its waves take every fourth tile.  Both products run on
// v_mfma_f32_16x16x32_bf16 with the query heads of the group as the 16 columns
// (those past the group are zero): S = K q^T with K rows as loaded, O^T = V^T P^T
// with V transposed by the LDS read.  Codes become bf16 without loss; the block's
// K scale multiplies the scores, its V scale the probabilities.
template <bool Fp8, bool Weigh>
__global__ __launch_bounds__(kDecodeThreads, 2) void compact_decode_kernel(CompactArgs a, DecodeScratch sc) {
  __shared__ DecodeShared sh;
  const std::uint32_t part = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const std::uint32_t n = context_of(a, seq);
  if (n == 0 || n > a.max_ctx) return;
  const std::uint32_t p = n - 1;
  const SeenTiles seen(p, p, a.window, a.sinks);
  const std::uint32_t begin = part * sc.tiles;
  if (begin >= seen.total) return;
  const std::uint32_t end = begin + sc.tiles < seen.total ? begin + sc.tiles : seen.total;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15; // MFMA column (query head) and A row
  const int kq = lane >> 4;  // k-quarter
  const CompactHead<Fp8> c(a.cache + seq * a.cache_stride, kvh, a.kv_heads, a.max_ctx, a.head_major);
  constexpr int kPieces = Fp8 ? 4 : 8; // 16-byte pieces of a K row that a lane loads

  // q of column `col`, in the dims that this lane's K pieces hold.
  bf16x8 qb[8];
  {
    const bf16_bits *q = a.query + ((static_cast<std::size_t>(seq) * a.kv_heads + kvh) * a.group + col) * kHeadDim;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int dim = Fp8 ? 64 * (i >> 1) + 16 * kq + 8 * (i & 1) : 32 * i + 8 * kq;
      u32x4 w{0u, 0u, 0u, 0u};
      if (col < static_cast<int>(a.group)) w = *reinterpret_cast<const u32x4 *>(q + dim);
      qb[i] = __builtin_bit_cast(bf16x8, w);
    }
  }
  // Transposed V reads: lane r of a 16-lane group supplies 4 dims of key row r / 4
  // and receives its dim of 4 keys.
  const bf16_bits *vt[4];
  {
    const int row = 4 * kq + (col >> 2);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      vt[j] = &sh.v[wave][row * kHeadDim + (((2 * j + ((col >> 1) & 1)) ^ (row & 7)) << 3) + 4 * (col & 1)];
  }

  floatx4 acc[16];
#pragma unroll
  for (int db = 0; db < 16; ++db) acc[db] = floatx4{};
  float m_run = -FLT_MAX, l_run = 0.f;

  for (std::uint32_t it = begin + wave; it < end; it += kDecodeWaves) {
    const std::uint32_t tile = seen.tile(it);
    const std::uint32_t j0 = tile * kCompactBlock;
    const bool whole = j0 + kCompactBlock <= n &&
                       (a.window == 0 || p - j0 < a.window || j0 + kCompactBlock <= a.sinks); // every key is seen
    u32x4 kr[2][kPieces];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      std::uint32_t j = j0 + 16 * rb + col;
      j = j < n ? j : n - 1;
      const auto *row = c.k + static_cast<std::size_t>(j) * c.row;
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        kr[rb][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(
            reinterpret_cast<const unsigned char *>(row) + 64 * i + 16 * kq));
    }
    // V: 16 lanes (Fp8) or 32 take one row.
    constexpr int kVLoads = Fp8 ? 8 : 16;
    constexpr int kRowLanes = Fp8 ? 16 : 32;
    u32x4 vr[kVLoads];
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const std::uint32_t j = j0 + (64 / kRowLanes) * i + lane / kRowLanes;
      const auto *row = c.v + static_cast<std::size_t>(j < n ? j : n - 1) * c.row;
      vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(
          reinterpret_cast<const unsigned char *>(row) + 16 * (lane % kRowLanes)));
    }
    float k_scale = kLog2e / 16.0f, v_scale = 1.0f;
    if constexpr (Fp8) {
      k_scale *= c.ks[tile];
      v_scale = c.vs[tile];
    }

    // Scores of keys j0 + 16 rb + 4 kq + i for head `col`.
    float s[2][4];
    float mx = -INFINITY;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      floatx4 d{};
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const u32x4 w = kr[rb][i];
        if constexpr (Fp8) {
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fp8x8_to_bf16(w[0], w[1])),
                                                      qb[2 * i], d, 0, 0, 0);
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fp8x8_to_bf16(w[2], w[3])),
                                                      qb[2 * i + 1], d, 0, 0, 0);
        } else {
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), qb[i], d, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[rb][i] = d[i] * k_scale;
        if (!whole && !compact_sees(j0 + 16 * rb + 4 * kq + i, p, a.window, a.sinks)) s[rb][i] = -INFINITY;
        mx = fmaxf(mx, s[rb][i]);
      }
    }
    if constexpr (Weigh) {
      if (col < static_cast<int>(a.group)) {
        float *row = sc.scores + ((static_cast<std::size_t>(seq) * a.kv_heads + kvh) * a.group + col) * sc.score_stride;
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
          *reinterpret_cast<floatx4 *>(row + j0 + 16 * rb + 4 * kq) = floatx4{s[rb][0], s[rb][1], s[rb][2], s[rb][3]};
      }
    }
    mx = max_xor32(max_xor16(mx));
    if (__builtin_amdgcn_ballot_w64(mx > m_run) != 0) {
      const float m_new = fmaxf(m_run, mx);
      const float f = fexp2(m_run - m_new);
      l_run *= f;
#pragma unroll
      for (int db = 0; db < 16; ++db) acc[db] *= f;
      m_run = m_new;
    }
    u32x4 pw;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = fexp2(s[rb][i] - m_run);
        l_run += e[i];
        e[i] *= v_scale;
      }
      pw[2 * rb] = pack_bf16x2(e[0], e[1]);
      pw[2 * rb + 1] = pack_bf16x2(e[2], e[3]);
    }
    const bf16x8 pb = __builtin_bit_cast(bf16x8, pw);

    // V rows into LDS as bf16; a key that is not seen gives a row of zeros (its
    // probability is 0, and 0 times what an unused row holds may be NaN).
    wave_lds_order();
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int r = (64 / kRowLanes) * i + lane / kRowLanes;
      const int piece = lane % kRowLanes;
      u32x4 w = vr[i];
      if (!whole && !compact_sees(j0 + r, p, a.window, a.sinks)) w = u32x4{0u, 0u, 0u, 0u};
      bf16_bits *row = sh.v[wave] + r * kHeadDim;
      if constexpr (Fp8) {
        *reinterpret_cast<u32x4 *>(row + (((2 * piece) ^ (r & 7)) << 3)) = fp8x8_to_bf16(w[0], w[1]);
        *reinterpret_cast<u32x4 *>(row + (((2 * piece + 1) ^ (r & 7)) << 3)) = fp8x8_to_bf16(w[2], w[3]);
      } else {
        *reinterpret_cast<u32x4 *>(row + ((piece ^ (r & 7)) << 3)) = w;
      }
    }
    wave_lds_order();
    // k-slot (kq, e) of the product <-> key 16 (e / 4) + 4 kq + e % 4, the order
    // in which the scores lie.
#pragma unroll
    for (int db = 0; db < 16; ++db) {
      const bf16_bits *v0 = vt[db & 3] + 64 * (db >> 2);
      const u32x2 lo = lds_tr16(v0), hi = lds_tr16(v0 + 16 * kHeadDim);
      acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]}), pb, acc[db], 0, 0, 0);
    }
  }

  // Join the waves.  l: the four lanes of a column hold partial sums.
  const float l_tot = sum_xor32(sum_xor16(l_run));
  __syncthreads();
  if (lane < kCompactMaxGroup) {
    sh.m[wave][lane] = m_run;
    sh.l[wave][lane] = l_tot;
  }
#pragma unroll
  for (int db = 0; db < 16; ++db) *reinterpret_cast<floatx4 *>(&sh.acc[wave][col][16 * db + 4 * kq]) = acc[db];
  __syncthreads();
  const int d = threadIdx.x;
  for (std::uint32_t h = 0; h < a.group; ++h) {
    float m = -FLT_MAX, l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; ++w) m = fmaxf(m, sh.m[w][h]);
#pragma unroll
    for (int w = 0; w < kDecodeWaves; ++w) {
      const float f = fexp2(sh.m[w][h] - m);
      l = fmaf(sh.l[w][h], f, l);
      o = fmaf(sh.acc[w][h][d], f, o);
    }
    const std::size_t at = ((static_cast<std::size_t>(seq) * a.kv_heads + kvh) * a.group + h) * sc.parts + part;
    sc.o[at * kHeadDim + d] = o;
    if (d == 0) {
      sc.m[at] = m;
      sc.l[at] = l;
    }
  }
}

// One workgroup per (query head, sequence): wave w takes partials w, w + 4, ..,
// a lane four dims.
__global__ __launch_bounds__(kDecodeThreads) void compact_merge_kernel(CompactArgs a, DecodeScratch sc) {
  __shared__ float o_of[kDecodeWaves][kHeadDim], m_of[kDecodeWaves], l_of[kDecodeWaves];
  const std::uint32_t head = blockIdx.x, seq = blockIdx.y;
  const std::uint32_t heads = a.kv_heads * a.group;
  const std::uint32_t n = context_of(a, seq);
  const std::size_t row = static_cast<std::size_t>(seq) * heads + head;
  if (n == 0 || n > a.max_ctx) {
    if (head == 0 && threadIdx.x == 0) atomicAdd(&g_compact_capacity_errors, 1u);
    a.output[row * kHeadDim + threadIdx.x] = f32_to_bf16(__builtin_nanf(""));
    return;
  }
  const std::uint32_t active = (SeenTiles(n - 1, n - 1, a.window, a.sinks).total + sc.tiles - 1) / sc.tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -FLT_MAX, l = 0.f;
  floatx4 o{};
  for (std::uint32_t i = wave; i < active; i += kDecodeWaves) {
    const std::size_t at = row * sc.parts + i;
    const float mi = sc.m[at];
    const float m_new = fmaxf(m, mi);
    const float f = fexp2(m - m_new), g = fexp2(mi - m_new);
    o = o * f + *reinterpret_cast<const floatx4 *>(sc.o + at * kHeadDim + 4 * lane) * g;
    l = l * f + sc.l[at] * g;
    m = m_new;
  }
  *reinterpret_cast<floatx4 *>(&o_of[wave][4 * lane]) = o;
  if (lane == 0) {
    m_of[wave] = m;
    l_of[wave] = l;
  }
  __syncthreads();
  m = fmaxf(fmaxf(m_of[0], m_of[1]), fmaxf(m_of[2], m_of[3]));
  float sum = 0.f, out = 0.f;
#pragma unroll
  for (int w = 0; w < kDecodeWaves; ++w) {
    const float f = fexp2(m_of[w] - m);
    sum = fmaf(l_of[w], f, sum);
    out = fmaf(o_of[w][threadIdx.x], f, out);
  }
  const std::size_t at = row * kHeadDim + threadIdx.x;
  a.output[at] = f32_to_bf16(out / sum * sigmoid_gate(bf16_to_f32(a.gate[at])));
  if (a.weights != nullptr && threadIdx.x == 0) {
    sc.final[2 * row] = m;
    sc.final[2 * row + 1] = 1.0f / sum;
  }
}

// weights[kvh][j] += the group's probabilities of key j; a thread per seen key.
__global__ __launch_bounds__(kDecodeThreads) void compact_weigh_kernel(CompactArgs a, DecodeScratch sc) {
  const std::uint32_t kvh = blockIdx.y, seq = blockIdx.z;
  const std::uint32_t n = context_of(a, seq);
  if (n == 0 || n > a.max_ctx) return;
  const SeenTiles seen(n - 1, n - 1, a.window, a.sinks);
  const std::uint32_t it = (blockIdx.x * kDecodeThreads + threadIdx.x) / kCompactBlock;
  if (it >= seen.total) return;
  const std::uint32_t j = seen.tile(it) * kCompactBlock + threadIdx.x % kCompactBlock;
  if (!compact_sees(j, n - 1, a.window, a.sinks)) return;
  const std::size_t row = (static_cast<std::size_t>(seq) * a.kv_heads + kvh) * a.group;
  float w = 0.f;
  for (std::uint32_t h = 0; h < a.group; ++h)
    w += fexp2(sc.scores[(row + h) * sc.score_stride + j] - sc.final[2 * (row + h)]) * sc.final[2 * (row + h) + 1];
  a.weights[(static_cast<std::size_t>(seq) * a.kv_heads + kvh) * a.max_ctx + j] += w;
}

std::uint32_t most_tiles(const CompactArgs &a, std::uint32_t n) {
  // over all contexts up to n: the tiles of n itself, or of a full window with both ends inside tiles
  const std::uint32_t all = (n + kCompactBlock - 1) / kCompactBlock;
  if (a.window == 0) return all;
  const std::size_t some = static_cast<std::size_t>((a.sinks + kCompactBlock - 1) / kCompactBlock) +
                           (a.window + kCompactBlock - 1) / kCompactBlock + 1;
  return some < all ? static_cast<std::uint32_t>(some) : all;
}

// At most this many partitions for any context up to max_ctx.
std::uint32_t most_parts(const CompactArgs &a) {
  const std::uint32_t units = a.sequences * a.kv_heads;
  const std::uint32_t target = units >= kDecodeTarget ? 1 : kDecodeTarget / units;
  const std::uint32_t few = (most_tiles(a, a.max_ctx) + kDecodeWaves - 1) / kDecodeWaves;
  return few < target ? few : target;
}

std::size_t round16(std::size_t bytes) { return (bytes + 15) / 16 * 16; }

DecodeScratch scratch_of(const CompactArgs &a, void *workspace, std::size_t *bytes) {
  const std::size_t heads = static_cast<std::size_t>(a.sequences) * a.kv_heads * a.group;
  const std::size_t parts = most_parts(a);
  DecodeScratch sc{};
  sc.parts = static_cast<std::uint32_t>(parts);
  sc.score_stride = (a.max_ctx + kCompactBlock - 1) / kCompactBlock * kCompactBlock;
  auto *p = static_cast<unsigned char *>(workspace);
  std::size_t at = 0;
  const auto take = [&](std::size_t floats) {
    auto *q = reinterpret_cast<float *>(p + at);
    at += round16(floats * sizeof(float));
    return q;
  };
  sc.o = take(heads * parts * kHeadDim);
  sc.m = take(heads * parts);
  sc.l = take(heads * parts);
  if (a.observed != 0) {
    sc.scores = take(heads * sc.score_stride);
    sc.final = take(heads * 2);
  }
  if (bytes != nullptr) *bytes = at;
  return sc;
}

template <bool Fp8> void launch_decode(const CompactArgs &a, const DecodeScratch &sc, std::uint32_t parts, hipStream_t stream) {
  const dim3 grid{parts, a.kv_heads, a.sequences};
  if (a.weights != nullptr)
    compact_decode_kernel<Fp8, true><<<grid, kDecodeThreads, 0, stream>>>(a, sc);
  else
    compact_decode_kernel<Fp8, false><<<grid, kDecodeThreads, 0, stream>>>(a, sc);
}

} // namespace

std::size_t compact_decode_workspace(const CompactArgs &a) {
  std::size_t bytes = 0;
  (void)scratch_of(a, nullptr, &bytes);
  return bytes;
}

void compact_decode(const CompactArgs &a, bool fp8, void *workspace, hipStream_t stream) {
  compact_append(a, fp8, stream);
  DecodeScratch sc = scratch_of(a, workspace, nullptr);
  const std::uint32_t longest = a.lengths == nullptr ? a.past + 1 : a.max_ctx;
  const std::uint32_t total = a.lengths == nullptr ? SeenTiles(a.past, a.past, a.window, a.sinks).total
                                                   : most_tiles(a, longest);
  sc.tiles = (total + sc.parts - 1) / sc.parts;
  if (sc.tiles < kDecodeWaves) sc.tiles = kDecodeWaves;
  const std::uint32_t parts = (total + sc.tiles - 1) / sc.tiles;
  if (fp8) launch_decode<true>(a, sc, parts, stream);
  else launch_decode<false>(a, sc, parts, stream);
  compact_merge_kernel<<<dim3{a.kv_heads * a.group, a.sequences}, kDecodeThreads, 0, stream>>>(a, sc);
  if (a.weights != nullptr)
    compact_weigh_kernel<<<dim3{(total * kCompactBlock + kDecodeThreads - 1) / kDecodeThreads, a.kv_heads, a.sequences},
                           kDecodeThreads, 0, stream>>>(a, sc);
}

std::uint32_t compact_take_capacity_errors() {
  unsigned int value = 0;
  const unsigned int zero = 0;
  if (hipMemcpyFromSymbol(&value, HIP_SYMBOL(g_compact_capacity_errors), sizeof value) != hipSuccess ||
      hipMemcpyToSymbol(HIP_SYMBOL(g_compact_capacity_errors), &zero, sizeof zero) != hipSuccess)
    throw std::runtime_error("reading the capacity error counter failed");
  return value;
}

} // namespace raftinfer::amd
