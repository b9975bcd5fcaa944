// Decode attention over the compact KV cache: one new token per sequence.
#include "compact_cache.hpp"
#include "prefill_tile.hpp"

#include <cfloat>

namespace raftinfer::amd {
namespace {

using prefill::fexp2;

constexpr int kMergeThreads = 512;
constexpr int kMergeWaves = kMergeThreads / kWave;

__device__ unsigned int g_compact_capacity_errors = 0;

// Partials of a call, one per (query head, partition): max and sum (exp2 domain),
// and the unnormalised output; with key weights also every score.
struct DecodeScratch {
  float *m, *l, *o, *scores;
  std::uint32_t tiles, parts, score_stride; // parts: rows of m, l, o per head
};

__device__ __forceinline__ std::uint32_t context_of(const CompactArgs &a, std::uint32_t seq) {
  return a.lengths == nullptr ? a.past + 1 : a.lengths[seq];
}

template <int WAVES> struct DecodeShared {
  union {
    // V rows as cached (a step of 8-bit or bf16 rows takes 8 KiB), 16-byte chunk c of row r at
    // c ^ v_key(r)
    alignas(1024) unsigned char v[WAVES][8192];
    // (the pad puts the 16 heads of a store on banks of their own)
    float acc[WAVES][kCompactMaxGroup][kHeadDim + 4];
  };
  float m[WAVES][kCompactMaxGroup];
  float l[WAVES][kCompactMaxGroup];
  alignas(16) unsigned char fresh[2][2 * kHeadDim]; // the new token's K and V rows, as stored
};

// (a pass of the transposed reads takes 16 bytes of the 16 rows 4 k + 0 .. 3, 16 + 4 k + 0 .. 3
// of two k, or of bf16 32 bytes of 8 rows: no two on one bank)
template <bool Fp8> __device__ __forceinline__ std::uint32_t v_key(std::uint32_t r) {
  return Fp8 ? (r & 3) | (r >> 4 & 1) << 2 | (r >> 2 & 1) << 3 : 2 * (r & 7);
}
__device__ __forceinline__ float max_finite_bf16x8(u32x4 w, float m) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const std::uint32_t u = w[e];
    const float a = fabsf(bf16_lo(u)), b = fabsf(bf16_hi(u));
    m = fmaxf(m, is_finite_f32(a) ? a : 0.f);
    m = fmaxf(m, is_finite_f32(b) ? b : 0.f);
  }
  return m;
}
__device__ __forceinline__ float finite_or_nan(float x) { return is_finite_f32(x) ? x : __builtin_nanf(""); }
// Sixteen bf16 values as codes of scale 1 / inv (Top: which may be the largest).
template <bool Top> __device__ __forceinline__ u32x4 bf16x16_to_fp8(u32x4 lo, u32x4 hi, float inv) {
  const auto part = [&](float x) {
    const float f = finite_or_nan(x);
    return (Top && inv == 1.0f / kCompactTopScale ? compact_below_top(f) : f) * inv;
  };
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const std::uint32_t x = e < 2 ? lo[2 * e] : hi[2 * e - 4], y = e < 2 ? lo[2 * e + 1] : hi[2 * e - 3];
    r[e] = pack_fp8x4(part(bf16_lo(x)), part(bf16_hi(x)), part(bf16_lo(y)), part(bf16_hi(y)));
  }
  return r;
}
// Two values cut to bf16.
__device__ __forceinline__ std::uint32_t cut_bf16x2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float(static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(x)), lane)));
}
__device__ __forceinline__ u32x4 rescale_fp8x16(u32x4 w, float ratio) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const floatx4 f = fp8x4_to_f32(w[e]);
    r[e] = pack_fp8x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
  }
  return r;
}

// A workgroup takes one partition (sc.tiles 32-key tiles) of one KV head and
// sequence; wave w takes its steps w, w + WAVES, ..  Both products run on
// v_mfma_f32_16x16x32_bf16 with the query heads of the group as the 16 columns
// (those past the group repeat the last): S = K q^T with K rows as loaded, O^T = V^T P^T
// with V transposed by the LDS read.  Codes become bf16 behind the reads, without loss; the block's
// K scale multiplies the scores, its V scale V's operands (a probability times the least scales is no
// normal number).  Probabilities go into the product in two bf16 parts, 16 bits together (one part:
// an average of equal values was up to a step of bf16 off).
//
// The kernel is bound by its cache reads, so a wave (32 8-bit or 16 bf16 rows a
// step) asks for rows a step ahead: K(t + 1) goes out when S(t) is formed, V(t + 1)
// when V(t) is in LDS.  32 ragged sequences of up to 32768, 8 bit, 4 KV heads: 202 us,
// 5.3 TB/s; one of 60001 23.0 us, 5.3 TB/s; 16 behind a window of 4096, bf16, 43.5 us,
// 5.8 TB/s.  201 tokens, 8.9 us, are round trips: lengths, then rows and scales, gate, output.
//
// The step that holds the new token's position covers its scale block, so its wave also
// stores the row: it raises the block's scale where the row needs that, rounds the
// block's other codes again in its registers, and attends over what it writes.
template <bool Fp8, bool Weigh, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, 8 / WAVES) void compact_decode_kernel(CompactArgs a, DecodeScratch sc) {
  __shared__ DecodeShared<WAVES> sh;
  // Workgroups go to the 8 XCDs in turn.  All units' first partitions lie first (short
  // contexts have no others), and a partition's units are rotated by its number, so
  // that a unit's partitions and the partitions of one number are spread over the XCDs.
  const std::uint32_t units = a.kv_heads * a.sequences;
  const std::uint32_t part = blockIdx.x / units;
  const std::uint32_t unit_id = (blockIdx.x % units + part) % units;
  const std::uint32_t kvh = unit_id % a.kv_heads, seq = unit_id / a.kv_heads;
  const bool last = gridDim.x == units; // one partition each: no merge follows
  const std::uint32_t n = context_of(a, seq);
  if (n == 0 || n > a.max_ctx) {
    // no valid context: NaN rows, counted once (here only if no merge follows)
    if (last) {
      if (kvh == 0 && threadIdx.x == 0) atomicAdd(&g_compact_capacity_errors, 1u);
      bf16_bits *out = a.output + (static_cast<std::size_t>(seq) * a.kv_heads + kvh) * a.group * kHeadDim;
      for (std::uint32_t i = threadIdx.x; i < a.group * kHeadDim; i += WAVES * kWave) out[i] = 0x7FC0;
    }
    return;
  }
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
  const std::size_t unit = static_cast<std::size_t>(seq) * a.kv_heads + kvh;
  constexpr int kStep = Fp8 ? 32 : 16;     // keys per step (8 KiB of K and of V)
  constexpr int kSteps = kCompactBlock / kStep;
  constexpr int kRB = kStep / 16;          // blocks of 16 K rows
  constexpr int kPieces = Fp8 ? 4 : 8;     // 16-byte pieces of a K row that a lane loads
  constexpr int kRowLanes = Fp8 ? 16 : 32; // V: lanes that take one row
  constexpr int kVRows = 64 / kRowLanes;
  constexpr int kVLoads = kStep / kVRows;
  const auto first_key = [&](std::uint32_t it) {
    return seen.tile(it / kSteps) * kCompactBlock + kStep * (it % kSteps);
  };

  // Scales come by vector loads: a scalar load counts with the LDS reads, whose next
  // wait would wait for it.
  int lane0;
  asm volatile("v_mov_b32 %0, 0" : "=v"(lane0));
  u32x4 kr[kRB][kPieces];
  u32x4 vr[kVLoads];
  float ks = 1.0f, vs = 1.0f; // scales of the rows in kr, vr
  const auto load_k = [&](std::uint32_t j0) {
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      std::uint32_t j = j0 + 16 * rb + col;
      j = j < n ? j : n - 1;
      const auto *row = reinterpret_cast<const unsigned char *>(c.k + static_cast<std::size_t>(j) * c.row) + 16 * kq;
      // (Not non-temporal, as V: a load takes half of each line, and the other half came from
      // memory again.  Batch of 32 218 -> 203 us, 60001 tokens 33.4 -> 30.2 in a graph; V so
      // too 216 and 34.4.)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) kr[rb][i] = *reinterpret_cast<const u32x4 *>(row + 64 * i);
    }
    if constexpr (Fp8) ks = c.ks[j0 / kCompactBlock + lane0];
  };
  const auto load_v = [&](std::uint32_t j0) {
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      std::uint32_t j = j0 + kVRows * i + lane / kRowLanes;
      j = j < n ? j : n - 1;
      const auto *row = reinterpret_cast<const unsigned char *>(c.v + static_cast<std::size_t>(j) * c.row);
      vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + 16 * (lane % kRowLanes)));
    }
    if constexpr (Fp8) vs = c.vs[j0 / kCompactBlock + lane0];
  };
  std::uint32_t it = begin * kSteps + wave;
  // The last step with a key is the one that holds the new token's row.
  const std::uint32_t newest_step = (seen.total - 1) * kSteps + p % kCompactBlock / kStep;
  const std::uint32_t it_end = end * kSteps <= newest_step ? end * kSteps : newest_step + 1;
  // The new token's rows, for the wave whose step holds them: lanes 0 .. 15 have K, 16 ..
  // 31 V, 16 dims each.
  const bool owner = newest_step + 1 == it_end && (newest_step - begin * kSteps) % WAVES == static_cast<std::uint32_t>(wave);
  const int plane = (lane >> 4) & 1, piece = lane & 15;
  u32x4 row_new[2];
  [[maybe_unused]] float scale_old = 0.f;
  if (owner) {
    const u32x4 *x = reinterpret_cast<const u32x4 *>((plane ? a.value : a.key) + unit * kHeadDim + 16 * piece);
    row_new[0] = x[0];
    row_new[1] = x[1];
    if constexpr (Fp8) scale_old = ((plane ? c.vs : c.ks) + p / kCompactBlock)[0];
  }
  // q of column `col`, in the dims that this lane's K pieces hold.  (Loaded before the
  // cache rows: a wait for it is then one for nothing younger.)
  bf16x8 qb[8];
  {
    const bf16_bits *q = a.query + (unit * a.group + (col < static_cast<int>(a.group) ? col : a.group - 1)) * kHeadDim;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int dim = Fp8 ? 64 * (i >> 1) + 16 * kq + 8 * (i & 1) : 32 * i + 8 * kq;
      qb[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(q + dim));
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  // (a wave without a step loads the first one's rows: the same reason)
  load_k(first_key(it < it_end ? it : begin * kSteps));
  load_v(first_key(it < it_end ? it : begin * kSteps));

  // The new token's rows into the cache, and into LDS for the step.  grow: what the block's other codes are multiplied by, 0 where
  // its scale stays.
  [[maybe_unused]] float grow_k = 0.f, grow_v = 0.f, new_ks = 1.0f, new_vs = 1.0f;
  if (owner) {
    const u32x4 lo = row_new[0], hi = row_new[1];
    unsigned char *dst = reinterpret_cast<unsigned char *>((plane ? c.v : c.k) + static_cast<std::size_t>(p) * c.row);
    if constexpr (Fp8) {
      float *scale = (plane ? c.vs : c.ks) + p / kCompactBlock;
      const float before = p % kCompactBlock != 0 ? scale_old : 0.f;
      const float amax = row16_max(max_finite_bf16x8(hi, max_finite_bf16x8(lo, 0.f)));
      const float after = fmaxf(before, compact_scale(amax));
      const float inv = compact_inverse(after);
      u32x4 codes = bf16x16_to_fp8<false>(lo, hi, inv);
      if (__builtin_amdgcn_ballot_w64(after == kCompactTopScale) != 0) codes = bf16x16_to_fp8<true>(lo, hi, inv);
      const float grow = before != 0.f && after != before ? before * inv : 0.f;
      if (lane < 32) {
        *reinterpret_cast<u32x4 *>(dst + 16 * piece) = codes;
        *reinterpret_cast<u32x4 *>(&sh.fresh[plane][16 * piece]) = codes;
        if (piece == 0) *scale = after;
      }
      new_ks = lane_value(after, 0);
      new_vs = lane_value(after, 16);
      grow_k = lane_value(grow, 0);
      grow_v = lane_value(grow, 16);
    } else if (lane < 32) {
      reinterpret_cast<u32x4 *>(dst + 32 * piece)[0] = lo;
      reinterpret_cast<u32x4 *>(dst + 32 * piece)[1] = hi;
      *reinterpret_cast<u32x4 *>(&sh.fresh[plane][32 * piece]) = lo;
      *reinterpret_cast<u32x4 *>(&sh.fresh[plane][32 * piece + 16]) = hi;
    }
    wave_lds_order();
  }

  // Transposed V reads: of 16 lanes, lane r supplies 8 bytes (8 or 4 dims) of key row r / 2 or
  // r / 4 of the group's and receives its dim of all of them.
  constexpr int kVBytes = Fp8 ? 256 : 512;
  const std::uint32_t v_row = Fp8 ? 16 * (col >> 3) + 4 * kq + (col >> 1 & 3) : 4 * kq + (col >> 2);
  const unsigned v_read = lds_address(sh.v[wave]) + kVBytes * v_row +
                          (16 * ((Fp8 ? 0 : col >> 1 & 1) ^ v_key<Fp8>(v_row)) + 8 * (col & 1));
  const std::uint32_t v_put_row = lane / kRowLanes; // of the first load: row kVRows i + v_put_row for load i
  const unsigned v_put = kVBytes * v_put_row + 16 * ((lane % kRowLanes) ^ v_key<Fp8>(v_put_row));

  floatx4 acc[16];
#pragma unroll
  for (int db = 0; db < 16; ++db) acc[db] = floatx4{};
  float m_run = -FLT_MAX, l_run = 0.f;

  // One step; kMore: it is not the wave's last.  (Two copies, and no condition on the
  // loads: with one, the waits for K and V would allow for the other's absence.)
  const auto step = [&]<bool kMore>() __attribute__((always_inline)) {
    const std::uint32_t j0 = first_key(it);
    const bool newest = !kMore && owner;
    const std::uint32_t r_new = p % kStep;
    const bool whole = j0 + kStep <= n &&
                       (a.window == 0 || p - j0 < a.window || j0 + kStep <= a.sinks); // every key is seen
    if (newest) {
      if constexpr (Fp8) {
        if (grow_k != 0.f) {
#pragma unroll
          for (int rb = 0; rb < kRB; ++rb) {
            if (16 * rb + col >= static_cast<int>(r_new)) continue;
            unsigned char *dst = c.k + static_cast<std::size_t>(j0 + 16 * rb + col) * c.row + 16 * kq;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
              kr[rb][i] = rescale_fp8x16(kr[rb][i], grow_k);
              *reinterpret_cast<u32x4 *>(dst + 64 * i) = kr[rb][i];
            }
          }
        }
        ks = new_ks;
      }
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb)
        if (16 * rb + col == static_cast<int>(r_new)) {
#pragma unroll
          for (int i = 0; i < kPieces; ++i) kr[rb][i] = *reinterpret_cast<const u32x4 *>(&sh.fresh[0][64 * i + 16 * kq]);
        }
    }

    // Scores of keys j0 + 16 rb + 4 kq + i for head `col`.
    const float k_scale = ks * (kLog2e / 16.0f);
    float s[kRB][4];
    float mx = -INFINITY;
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
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
      for (int i = 0; i < 4; ++i) s[rb][i] = d[i] * k_scale;
    }
    if (!whole) {
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[rb][i] = compact_sees(j0 + 16 * rb + 4 * kq + i, p, a.window, a.sinks) ? s[rb][i] : -INFINITY;
    }
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rb][i]);
    if constexpr (kMore) load_k(first_key(it + WAVES));
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (Weigh) {
      if (col < static_cast<int>(a.group)) {
        float *row = sc.scores + (unit * a.group + col) * sc.score_stride;
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb)
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
    if (newest) {
      if constexpr (Fp8) {
        if (grow_v != 0.f) {
#pragma unroll
          for (int i = 0; i < kVLoads; ++i) {
            const std::uint32_t row = kVRows * i + lane / kRowLanes;
            if (row >= r_new) continue;
            vr[i] = rescale_fp8x16(vr[i], grow_v);
            *reinterpret_cast<u32x4 *>(c.v + static_cast<std::size_t>(j0 + row) * c.row + 16 * (lane % kRowLanes)) = vr[i];
          }
        }
        vs = new_vs;
      }
      const u32x4 fresh = *reinterpret_cast<const u32x4 *>(&sh.fresh[1][16 * (lane % kRowLanes)]);
#pragma unroll
      for (int i = 0; i < kVLoads; ++i)
        if (kVRows * i + lane / kRowLanes == static_cast<int>(r_new)) vr[i] = fresh;
    }
    // In two parts: pw, cut to bf16 below p (1 - 2^-9), and pl, what it leaves.  Neither is 0 or
    // negative where p is not, so that an infinite value gives that and no NaN.
    std::uint32_t pw[2 * kRB], pl[2 * kRB];
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = fexp2(s[rb][i] - m_run);
        l_run += e[i];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = e[2 * i], y = e[2 * i + 1];
        const std::uint32_t w = cut_bf16x2(fmaf(x, -0x1p-9f, x), fmaf(y, -0x1p-9f, y));
        pw[2 * rb + i] = w;
        pl[2 * rb + i] = pack_bf16x2(x - bf16_lo(w), y - bf16_hi(w));
      }
    }
    // V rows into LDS as cached; a key that is not seen gives a row of zeros (its
    // probability is 0, and 0 times what an unused row holds may be NaN).
    if (!whole) {
#pragma unroll
      for (int i = 0; i < kVLoads; ++i) {
        const std::uint32_t keep = compact_sees(j0 + kVRows * i + lane / kRowLanes, p, a.window, a.sinks) ? ~0u : 0u;
        vr[i] &= u32x4{keep, keep, keep, keep};
      }
    }
    if constexpr (Fp8) asm volatile("" : "+v"(vs)); // (one wait for all of V: 60001 tokens 25.6 -> 25.2 us)
    wave_lds_order();
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) // (v_key is linear in the bits of the row)
      *reinterpret_cast<u32x4 *>(&sh.v[wave][(v_put ^ (16 * v_key<Fp8>(kVRows * i))) + kVBytes * kVRows * i]) = vr[i];
    [[maybe_unused]] const float v_scale = lane_value(vs, 0);
    if constexpr (kMore) load_v(first_key(it + WAVES));
    __builtin_amdgcn_sched_barrier(0);
    wave_lds_order();
    // k-slot (kq, e) of the product <-> key 16 (e / 4) + 4 kq + e % 4, the order
    // in which the scores lie.  Operands are read kRing products ahead.
    constexpr int kRing = 8;
    const auto read_v = [&](int db) {
      if constexpr (Fp8) return lds_tr8_operand(v_read ^ (16u * db));
      else return lds_tr_operand(v_read ^ (32u * db));
    };
    u32x2 op[kRing];
#pragma unroll
    for (int db = 0; db < kRing; ++db) op[db] = read_v(db);
    [[maybe_unused]] bf16x8 before; // 8 bit: the operand of product db - 1, whose second one follows product db
    const auto second = [&](int db) {
      if constexpr (Fp8)
        acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(before, __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]}), acc[db], 0, 0, 0);
    };
#pragma unroll
    for (int db = 0; db < 16; ++db) {
      const u32x2 w = op[db % kRing];
      if constexpr (Fp8) {
        const bf16x8 v = __builtin_bit_cast(bf16x8, fp8x8_to_bf16(w[0], w[1], v_scale));
        acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, u32x4{pw[0], pw[1], pw[2], pw[3]}), acc[db], 0, 0, 0);
        if (db > 0) second(db - 1);
        before = v;
      } else { // 16 keys: both parts in one product
        acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[0], w[1]}),
                                                          __builtin_bit_cast(bf16x8, u32x4{pw[0], pw[1], pl[0], pl[1]}), acc[db], 0, 0, 0);
      }
      if (db + kRing < 16) op[db % kRing] = read_v(db + kRing);
      __builtin_amdgcn_sched_barrier(0);
    }
    second(15);
  };
  for (; it + WAVES < it_end; it += WAVES) step.template operator()<true>();
  if (it < it_end) step.template operator()<false>();

  // Join the waves.  l: the four lanes of a column hold partial sums.
  const float l_tot = sum_xor32(sum_xor16(l_run));
  __syncthreads();
  if (lane < kCompactMaxGroup) {
    sh.m[wave][lane] = m_run;
    sh.l[wave][lane] = l_tot;
  }
  if (col < static_cast<int>(a.group)) {
#pragma unroll
    for (int db = 0; db < 16; ++db) *reinterpret_cast<floatx4 *>(&sh.acc[wave][col][16 * db + 4 * kq]) = acc[db];
  }
  __syncthreads();
  for (std::uint32_t i = threadIdx.x; i < a.group * kHeadDim; i += WAVES * kWave) {
    const std::uint32_t h = i / kHeadDim, d = i % kHeadDim;
    float m = -FLT_MAX, l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, sh.m[w][h]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = fexp2(sh.m[w][h] - m);
      l = fmaf(sh.l[w][h], f, l);
      o = fmaf(sh.acc[w][h][d], f, o);
    }
    if (last) {
      const std::size_t at = unit * a.group * kHeadDim + i;
      a.output[at] = f32_to_bf16(o / l * sigmoid_gate(bf16_to_f32(a.gate[at])));
      continue;
    }
    const std::size_t at = (unit * a.group + h) * sc.parts + part;
    sc.o[at * kHeadDim + d] = o;
    if (d == 0) {
      sc.m[at] = m;
      sc.l[at] = l;
    }
  }
  if constexpr (Weigh) {
    if (!last) return;
    for (std::uint32_t i = threadIdx.x; i < seen.total * kCompactBlock; i += WAVES * kWave) {
      const std::uint32_t j = seen.tile(i / kCompactBlock) * kCompactBlock + i % kCompactBlock;
      if (!compact_sees(j, p, a.window, a.sinks)) continue;
      float w = 0.f;
      for (std::uint32_t h = 0; h < a.group; ++h) {
        float m = -FLT_MAX, l = 0.f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) m = fmaxf(m, sh.m[x][h]);
#pragma unroll
        for (int x = 0; x < WAVES; ++x) l = fmaf(sh.l[x][h], fexp2(sh.m[x][h] - m), l);
        w += fexp2(sc.scores[(unit * a.group + h) * sc.score_stride + j] - m) * (1.0f / l);
      }
      a.weights[unit * a.max_ctx + j] += w;
    }
  }
}

// Max and 1 / sum over a head's partials, by one wave.
__device__ __forceinline__ void final_of(const DecodeScratch &sc, std::size_t row, std::uint32_t active, float &m, float &inv) {
  const int lane = threadIdx.x & 63;
  float l = 0.f;
  m = -FLT_MAX;
  for (std::uint32_t i = lane; i < active; i += 64) {
    const float mi = sc.m[row * sc.parts + i], li = sc.l[row * sc.parts + i];
    const float m_new = fmaxf(m, mi);
    l = l * fexp2(m - m_new) + li * fexp2(mi - m_new);
    m = m_new;
  }
  const float m_all = wave_max(m);
  inv = 1.0f / wave_sum(l * fexp2(m - m_all));
  m = m_all;
}

// Blocks x < query heads join a head's partials: wave w takes partials w, w + 8, ..
// in batches of 8, whose loads go out before the partials' maxima are known; a lane
// has four dims.  The blocks behind them (key weights) add the group's probabilities
// to 512 seen keys of one KV head each.  Two round trips to memory: 4 us with 64 partials.
__global__ __launch_bounds__(kMergeThreads) void compact_merge_kernel(CompactArgs a, DecodeScratch sc) {
  __shared__ float o_of[kMergeWaves][kHeadDim], m_of[kCompactMaxGroup], l_of[kCompactMaxGroup];
  const std::uint32_t seq = blockIdx.y;
  const std::uint32_t heads = a.kv_heads * a.group;
  const std::uint32_t n = context_of(a, seq);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool valid = n != 0 && n <= a.max_ctx;
  if (blockIdx.x < heads) {
    const std::uint32_t head = blockIdx.x;
    const std::size_t row = static_cast<std::size_t>(seq) * heads + head;
    if (!valid) {
      if (head == 0 && threadIdx.x == 0) atomicAdd(&g_compact_capacity_errors, 1u);
      if (threadIdx.x < kHeadDim) a.output[row * kHeadDim + threadIdx.x] = 0x7FC0;
      return;
    }
    const float gate = threadIdx.x < kHeadDim ? bf16_to_f32(a.gate[row * kHeadDim + threadIdx.x]) : 0.f;
    const std::uint32_t active = (SeenTiles(n - 1, n - 1, a.window, a.sinks).total + sc.tiles - 1) / sc.tiles;
    constexpr int kBatch = 8;
    floatx4 x[kBatch];
    float mx[kBatch];
    const auto load = [&](std::uint32_t i0) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const std::uint32_t i = i0 + kMergeWaves * b < active ? i0 + kMergeWaves * b : active - 1;
        x[b] = *reinterpret_cast<const floatx4 *>(sc.o + (row * sc.parts + i) * kHeadDim + 4 * lane);
        mx[b] = sc.m[row * sc.parts + i];
      }
    };
    load(wave);
    float m, inv;
    final_of(sc, row, active, m, inv);
    floatx4 o{};
    for (std::uint32_t i0 = wave; i0 < active; i0 += kMergeWaves * kBatch) {
      if (i0 != static_cast<std::uint32_t>(wave)) load(i0);
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (i0 + kMergeWaves * b < active) o += x[b] * fexp2(mx[b] - m);
    }
    *reinterpret_cast<floatx4 *>(&o_of[wave][4 * lane]) = o;
    __syncthreads();
    if (threadIdx.x >= kHeadDim) return;
    float out = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w) out += o_of[w][threadIdx.x];
    a.output[row * kHeadDim + threadIdx.x] = f32_to_bf16(out * inv * sigmoid_gate(gate));
    return;
  }
  if (!valid) return;
  const SeenTiles seen(n - 1, n - 1, a.window, a.sinks);
  const std::uint32_t chunk = (blockIdx.x - heads) / a.kv_heads, kvh = (blockIdx.x - heads) % a.kv_heads;
  if (chunk * kMergeThreads >= seen.total * kCompactBlock) return; // (uniform)
  const std::uint32_t active = (seen.total + sc.tiles - 1) / sc.tiles;
  const std::size_t unit = static_cast<std::size_t>(seq) * a.kv_heads + kvh;
  for (std::uint32_t h = wave; h < a.group; h += kMergeWaves) {
    float m, inv;
    final_of(sc, unit * a.group + h, active, m, inv);
    if (lane == 0) {
      m_of[h] = m;
      l_of[h] = inv;
    }
  }
  __syncthreads();
  const std::uint32_t i = chunk * kMergeThreads + threadIdx.x;
  if (i >= seen.total * kCompactBlock) return;
  const std::uint32_t j = seen.tile(i / kCompactBlock) * kCompactBlock + i % kCompactBlock;
  if (!compact_sees(j, n - 1, a.window, a.sinks)) return;
  float w = 0.f;
  for (std::uint32_t h = 0; h < a.group; ++h)
    w += fexp2(sc.scores[(unit * a.group + h) * sc.score_stride + j] - m_of[h]) * l_of[h];
  a.weights[unit * a.max_ctx + j] += w;
}

std::uint32_t most_tiles(const CompactArgs &a, std::uint32_t n) {
  // over all contexts up to n: the tiles of n itself, or of a full window with both ends inside tiles
  const std::uint32_t all = (n + kCompactBlock - 1) / kCompactBlock;
  if (a.window == 0) return all;
  const std::size_t some = static_cast<std::size_t>((a.sinks + kCompactBlock - 1) / kCompactBlock) +
                           (a.window + kCompactBlock - 1) / kCompactBlock + 1;
  return some < all ? static_cast<std::uint32_t>(some) : all;
}

// How a call is split whose contexts have up to `total` tiles.  Short contexts: one
// workgroup of 8 waves per unit and no merge (201 tokens: 8.9 us; cut in two with a
// merge 14.5 against 14.4 in a graph, and a launch more).  Else partitions of 4 to 32
// tiles such that about 256 workgroups of 4 waves run, one or two per CU (in a graph: 16
// sequences behind a window of 4096 in 32 / 24 / 16 tiles 52.2 / 57.2 / 53.9 us, 4 of 8192
// with key weights 27.7 / 32.7 / 28.4); no longer where there are more (32 ragged sequences,
// 32 / 64 tiles: 203 / 210 us), and at most 64 partitions, which the merge takes in one
// batch (60001 tokens, 64 / 128: 30.3 / 31.0 us, 16000 tokens 17.1 / 18.8).  Where that leaves
// at most one workgroup per CU, it gets 8 waves from 32 tiles on (60001 tokens: 33.5 against 35.0
// us with 4); of fewer tiles 4 are faster (4 / 8 waves: 16000 tokens, 8 tiles, 12.9 / 13.1 us; 4 of
// 8192 in bf16, 16 tiles, 28.9 / 30.3, with key weights 32.0 / 32.9; 45000 tokens, 24 tiles, 22.1 / 22.7).
constexpr std::uint32_t kAlone = 16;
constexpr std::uint32_t kMostParts = 64;
struct DecodeSplit {
  int waves;
  std::uint32_t tiles, parts;
};
DecodeSplit split_of(const CompactArgs &a, std::uint32_t total) {
  if (total <= kAlone) return {8, kAlone, 1};
  const std::uint64_t units = static_cast<std::uint64_t>(a.sequences) * a.kv_heads;
  const std::uint64_t even = (total * units / 256 + 2) / 4 * 4;
  std::uint32_t tiles = even < 4 ? 4 : even > 32 ? 32 : static_cast<std::uint32_t>(even);
  const std::uint32_t least = ((total + kMostParts - 1) / kMostParts + 3) / 4 * 4;
  if (tiles < least) tiles = least;
  const std::uint32_t parts = (total + tiles - 1) / tiles;
  if (parts * units > 256 || tiles < 32) return {4, tiles, parts};
  return {8, (tiles + 7) / 8 * 8, (total + (tiles + 7) / 8 * 8 - 1) / ((tiles + 7) / 8 * 8)};
}
// The most partitions that any context of at most `total` tiles is cut into.
std::uint32_t most_parts(std::uint32_t total) {
  if (total <= kAlone) return 1;
  return (total + 3) / 4 < kMostParts ? (total + 3) / 4 : kMostParts;
}

std::size_t round16(std::size_t bytes) { return (bytes + 15) / 16 * 16; }

DecodeScratch scratch_of(const CompactArgs &a, std::size_t parts, void *workspace, std::size_t *bytes) {
  const std::size_t heads = static_cast<std::size_t>(a.sequences) * a.kv_heads * a.group;
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
  if (a.observed != 0) sc.scores = take(heads * sc.score_stride);
  if (parts > 1) {
    sc.o = take(heads * parts * kHeadDim);
    sc.m = take(heads * parts);
    sc.l = take(heads * parts);
  }
  if (bytes != nullptr) *bytes = at;
  return sc;
}

template <bool Fp8, bool Weigh>
void launch_decode(const CompactArgs &a, const DecodeScratch &sc, const DecodeSplit &split, hipStream_t stream) {
  const unsigned grid = split.parts * a.kv_heads * a.sequences;
  if (split.waves == 8)
    compact_decode_kernel<Fp8, Weigh, 8><<<grid, 8 * kWave, 0, stream>>>(a, sc);
  else
    compact_decode_kernel<Fp8, Weigh, 4><<<grid, 4 * kWave, 0, stream>>>(a, sc);
}

} // namespace

std::size_t compact_decode_workspace(const CompactArgs &a) {
  std::size_t bytes = 0;
  (void)scratch_of(a, most_parts(most_tiles(a, a.max_ctx)), nullptr, &bytes);
  return bytes;
}

void compact_decode(const CompactArgs &a, bool fp8, void *workspace, hipStream_t stream) {
  const std::uint32_t total = a.lengths == nullptr ? SeenTiles(a.past, a.past, a.window, a.sinks).total
                                                   : most_tiles(a, a.max_ctx);
  const DecodeSplit split = split_of(a, total);
  DecodeScratch sc = scratch_of(a, split.parts, workspace, nullptr);
  sc.tiles = split.tiles;
  const bool weigh = a.weights != nullptr;
  if (fp8 && weigh) launch_decode<true, true>(a, sc, split, stream);
  else if (fp8) launch_decode<true, false>(a, sc, split, stream);
  else if (weigh) launch_decode<false, true>(a, sc, split, stream);
  else launch_decode<false, false>(a, sc, split, stream);
  if (split.parts == 1) return;
  const std::uint32_t chunks = weigh ? (total * kCompactBlock + kMergeThreads - 1) / kMergeThreads : 0;
  compact_merge_kernel<<<dim3{a.kv_heads * (a.group + chunks), a.sequences}, kMergeThreads, 0, stream>>>(a, sc);
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
