// Entry points and sizing of the paged KV cache, and the store of new rows with their
// norm and rotation (include/raftinfer_amd/qwen35_paged_cache.hpp).
#include "call_checks.hpp"
#include "paged_cache.hpp"
#include "rotary.hpp"
#include "raftinfer_amd/qwen35_paged_cache.hpp"

#include <algorithm>
#include <cmath>

namespace raftinfer::amd {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendLanes = kHeadDim / 8; // of a head, 16 bytes each

__device__ unsigned int g_append_capacity_errors = 0;

// The sequence that row r belongs to, if query_starts do not fall: the first s with
// starts[s + 1] > r, by 64 probes at a time.  `sequences` if there is none.
__device__ __forceinline__ std::uint32_t sequence_of(const PagedArgs &a, std::uint32_t r) {
  const std::uint32_t lane = threadIdx.x & 63;
  std::uint32_t lo = 0, end = a.sequences;
  while (lo < end) {
    const std::uint32_t step = (end - lo + 63) / 64, at = lo + step * (lane + 1) - 1;
    const std::uint32_t below = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < end && a.starts[at < end ? at + 1 : 0] <= r));
    lo += below * step;
    if (step == 1) return lo;
    end = lo + step - 1 < end ? lo + step - 1 : end; // the probe there is behind r
  }
  return lo;
}

// A workgroup takes kRows rows: its waves look up the rows' sequences, positions and pages, one wave a row, while the
// first heads (query, key, value; 32 lanes each, 16 bytes a lane) are on their way, and four heads of a lane's
// group are asked for at a time, the next four before these are used.  What bounds a workgroup is the chain of loads in front of a store
// (starts, lengths, table: 10 us of a workgroup with five of them on a compute unit); one row each keeps short calls
// short (32 rows 7.0 us), four share the chain in long ones.
template <int kRows> __global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(PagedAppendArgs x) {
  __shared__ float rot[kRows][kHeadDim]; // cos of the pairs, then sin
  __shared__ std::uint32_t place[kRows][2]; // the K row of head 0, and whether: 0 the row is not stored, 1 its query only, 2 all
  const PagedArgs &a = x.paged;
  const std::uint32_t row0 = blockIdx.x * kRows, rows = a.rows - row0 < kRows ? a.rows - row0 : kRows, lane = threadIdx.x & 63;
  const std::uint32_t q_heads = a.query != nullptr ? a.kv_heads * a.group : 0;
  const std::uint32_t units = q_heads + 2 * a.kv_heads, all = units * rows;
  const int c = threadIdx.x % kAppendLanes;
  constexpr std::uint32_t kGroups = kAppendThreads / kAppendLanes;
  constexpr int kBatch = 4;
  const std::uint32_t u0 = threadIdx.x / kAppendLanes;
  const auto row_of = [&](std::uint32_t u) { return kRows == 1 ? 0u : __umulhi(u, x.units_inverse); };
  const auto load = [&](std::uint32_t first, u32x4 (&raw)[kBatch]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const std::uint32_t n = first + kGroups * i < all ? first + kGroups * i : all - 1;
      const std::uint32_t r = row_of(n), u = n - r * units;
      const std::size_t row = row0 + r;
      const bf16_bits *src = u < q_heads ? a.query + row * a.q_row + u * a.q_head
                             : u < q_heads + a.kv_heads ? x.key + row * x.k_row + (u - q_heads) * x.k_head
                                                        : x.value + row * x.v_row + (u - q_heads - a.kv_heads) * x.v_head;
      raw[i] = *reinterpret_cast<const u32x4 *>(src + 8 * c);
    }
  };
  u32x4 raw[kBatch];
  load(u0, raw);
  float qw[8], kw[8];
  const auto weights = [&](const void *weight, float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e] = weight == nullptr ? 0.f : x.weight_f32 ? static_cast<const float *>(weight)[8 * c + e]
                                                    : bf16_to_f32(static_cast<const bf16_bits *>(weight)[8 * c + e]);
  };
  weights(x.q_weight, qw);
  weights(x.k_weight, kw);
  if (row0 == 0 && threadIdx.x < 64) { // bad sequences are counted here
    std::uint32_t bad = 0;
    for (std::uint32_t s = lane; s < a.sequences; s += 64) bad += !paged_seq(a, s).valid;
    if (bad != 0) atomicAdd(&g_append_capacity_errors, bad);
  }
  const std::uint32_t pairs = x.rotary_dim / 2, wave = scalar(threadIdx.x >> 6);
  // (of one row every wave, and its angles by the first pairs / 64 of them; else wave w the rows w, w + 4, ..)
  for (std::uint32_t r = kRows == 1 ? 0 : wave; r < rows; r += kRows == 1 ? 1 : kAppendThreads / 64) {
    const std::uint32_t row = row0 + r, seq = scalar(sequence_of(a, row));
    std::uint32_t to = 0, what = 0;
    if (seq < a.sequences) { // (else behind the last sequence's rows)
      const PagedSeq q = paged_seq(a, seq);
      if (q.valid && row >= q.row0 && row - q.row0 < q.n) {
        const std::uint32_t position = q.ctx - q.n + (row - q.row0);
        bool bad = false;
        to = paged_row(a, seq, 0, position, bad);
        what = bad ? 1 : 2;
        for (std::uint32_t p = kRows == 1 ? threadIdx.x : lane; p < pairs; p += kRows == 1 ? kAppendThreads : 64) {
          float cs, sn;
          rotary_cos_sin(position, x.frequencies[p], x.magnitude, cs, sn);
          rot[r][p] = cs;
          rot[r][pairs + p] = sn;
        }
        if (bad && (kRows == 1 ? threadIdx.x : lane) == 0) atomicAdd(&g_append_capacity_errors, 1u);
      }
    }
    if (kRows == 1 && what == 0) return; // (uniform)
    if (lane == 0) {
      place[r][0] = to;
      place[r][1] = what;
    }
  }
  __syncthreads();
  for (std::uint32_t first = u0; first - u0 < all; first += kGroups * kBatch) {
    u32x4 next[kBatch];
    const bool more = first - u0 + kGroups * kBatch < all; // (uniform)
    if (more) load(first + kGroups * kBatch, next);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const std::uint32_t n = first + kGroups * i < all ? first + kGroups * i : all - 1;
      const std::uint32_t r = row_of(n), u = n - r * units;
      const bool is_q = u < q_heads, is_v = u >= q_heads + a.kv_heads;
      float v[8], w[8];
      Piece16<bf16_bits>::unpack(raw[i], v);
      // (two heads of a wave can be of two kinds: the norm is taken of both)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = is_q ? qw[e] : kw[e];
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v[e];
      if (__builtin_amdgcn_ballot_w64(!is_v) != 0) { // (a wave of values only: as they are)
        if (x.q_weight != nullptr || x.k_weight != nullptr) {
          norm_rotate<8, kAppendLanes>(y, w, true, false, c, 0, kHeadDim, rot[r], x.epsilon);
          const bool norm = (is_q ? x.q_weight : x.k_weight) != nullptr;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = norm ? y[e] : v[e];
        }
        norm_rotate<8, kAppendLanes>(y, w, false, x.interleaved, c, pairs, kHeadDim, rot[r], x.epsilon);
      }
      const u32x4 out = is_v ? raw[i] : Piece16<bf16_bits>::pack(y);
      const std::uint32_t what = place[r][1];
      if (first + kGroups * i >= all || what == 0) continue;
      const std::size_t row = row0 + r;
      if (is_q) {
        *reinterpret_cast<u32x4 *>(a.output + row * a.o_row + u * a.o_head + 8 * c) = out;
      } else if (what == 2) {
        const std::uint32_t kvh = is_v ? u - q_heads - a.kv_heads : u - q_heads;
        const std::size_t at = place[r][0] + kvh * a.head_step + (is_v ? a.plane_rows : 0);
        *reinterpret_cast<u32x4 *>(x.pages + at * kRowBytes + 16 * c) = out;
      }
    }
    if (more) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) raw[i] = next[i];
    }
  }
}

} // namespace

void paged_append(const PagedAppendArgs &args, hipStream_t stream) {
  PagedAppendArgs a = args;
  const std::uint32_t units = (a.paged.query != nullptr ? a.paged.kv_heads * a.paged.group : 0) + 2 * a.paged.kv_heads;
  a.units_inverse = 0xFFFFFFFFu / units + 1; // (of products below 2^32: units and four rows of them)
  if (a.paged.rows >= 1024) paged_append_kernel<4><<<(a.paged.rows + 3) / 4, kAppendThreads, 0, stream>>>(a);
  else paged_append_kernel<1><<<a.paged.rows, kAppendThreads, 0, stream>>>(a);
}

std::uint32_t paged_take_append_errors() {
  unsigned int value = 0;
  const unsigned int zero = 0;
  if (hipMemcpyFromSymbol(&value, HIP_SYMBOL(g_append_capacity_errors), sizeof value) != hipSuccess ||
      hipMemcpyToSymbol(HIP_SYMBOL(g_append_capacity_errors), &zero, sizeof zero) != hipSuccess)
    throw std::runtime_error("reading the capacity error counter failed");
  return value;
}

} // namespace raftinfer::amd

namespace raftinfer::kernels {
namespace {

using namespace raftinfer::amd;
using Err = Qwen35PrimitiveError;

// Positions, rows of 512 bytes, columns and workgroups are 32-bit in the kernels.
constexpr std::size_t kMaxPositions = std::size_t{1} << 28;
constexpr std::size_t kMaxPoolRows = std::size_t{1} << 31; // K and V rows of all KV heads
constexpr std::size_t kMaxQueryRows = std::size_t{1} << 22; // rows times query heads
constexpr std::size_t kMaxSequences = 65535;
constexpr std::size_t kMaxKvHeads = 1024;

void validate_shape(const Qwen35PagedShape &s) {
  require<Err>(s.rows > 0, "paged cache rows must be positive");
  require<Err>(s.sequences > 0 && s.sequences <= kMaxSequences, "paged cache sequences must be 1 to 65535");
  require<Err>(s.kv_heads > 0 && s.kv_heads <= kMaxKvHeads, "paged cache kv_heads must be 1 to 1024");
  require<Err>(s.query_heads > 0 && s.query_heads % s.kv_heads == 0 && s.query_heads / s.kv_heads <= kPagedMaxGroup,
               "paged cache query_heads must be 1 to 16 per KV head");
  require<Err>(s.head_dim == kHeadDim, "paged cache head_dim must be 256");
  require<Err>(s.rows <= kMaxQueryRows / s.query_heads, "paged cache has more than 2^22 query rows");
  require<Err>(s.page_tokens > 0 && s.page_tokens % kPageGranule == 0 && s.page_tokens <= kMaxPositions,
               "paged cache page_tokens must be a multiple of 16");
  require<Err>(s.pages > 0 && s.pages <= kMaxPoolRows / 2 / s.kv_heads / s.page_tokens,
               "paged cache pages must be 1 to 2^31 rows of all KV heads");
  require<Err>(s.table_pages > 0 && s.table_pages <= kMaxPositions, "paged cache table_pages must be 1 to 2^28");
  require<Err>(s.max_context_tokens > 0 && s.max_context_tokens <= kMaxPositions,
               "paged cache max_context_tokens must be 1 to 2^28");
}

std::size_t pool_bytes(const Qwen35PagedShape &s) { return s.pages * 2 * s.kv_heads * s.page_tokens * kRowBytes; }

PagedArgs to_args(const Qwen35PagedShape &s, Qwen35KvCacheLayout layout) {
  require<Err>(layout == Qwen35KvCacheLayout::token_major || layout == Qwen35KvCacheLayout::head_major,
               "unsupported paged cache layout");
  const bool head_major = layout == Qwen35KvCacheLayout::head_major;
  const auto u32 = [](std::size_t x) { return static_cast<std::uint32_t>(x); };
  PagedArgs a{};
  a.rows = u32(s.rows);
  a.sequences = u32(s.sequences);
  a.kv_heads = u32(s.kv_heads);
  a.group = u32(s.query_heads / s.kv_heads);
  a.group_inverse = 65536 / a.group + 1;
  a.group_inverse30 = (1u << 30) / a.group + 1;
  a.page_count = u32(s.pages);
  a.page_tokens = u32(s.page_tokens);
  a.table_pages = u32(s.table_pages);
  a.max_ctx = u32(std::min(s.max_context_tokens, s.table_pages * s.page_tokens)); // (the table names no page for more)
  a.window = s.window_tokens < a.max_ctx ? u32(s.window_tokens) : 0; // one that holds every position is none
  a.row_step = head_major ? 1 : a.kv_heads;
  a.head_step = head_major ? a.page_tokens : 1;
  a.plane_rows = a.kv_heads * a.page_tokens;
  a.page_shift = -1;
  if ((a.page_tokens & (a.page_tokens - 1)) == 0)
    for (a.page_shift = 0; (1u << a.page_shift) < a.page_tokens;) ++a.page_shift;
  return a;
}

bool aligned4(const void *p) { return (reinterpret_cast<std::uintptr_t>(p) & 3u) == 0; }

// A tensor [rows][heads][256] with strides (0: dense): strides as used, and its bytes.
struct Tensor {
  std::size_t row, head, bytes;
  Tensor(std::size_t rows, std::size_t heads, std::size_t row_stride, std::size_t head_stride)
      : row(row_stride != 0 ? row_stride : heads * kHeadDim), head(head_stride != 0 ? head_stride : kHeadDim), bytes(0) {
    const char *overflow = "paged cache strides overflow";
    require<Err>(row % 8 == 0 && head % 8 == 0, "paged cache strides must be multiples of 8");
    const std::size_t elems = checked_add<Err>(checked_add<Err>(checked_mul<Err>(rows - 1, row, overflow),
                                                                checked_mul<Err>(heads - 1, head, overflow), overflow),
                                               kHeadDim, overflow);
    bytes = checked_mul<Err>(elems, 2, overflow);
  }
};

void validate_pool(const Qwen35PagedShape &s, const void *pages, std::size_t pages_bytes, const std::int32_t *table,
                   const std::uint32_t *starts, bool with_starts, const std::uint32_t *lengths, RaftInferDataType act,
                   hipStream_t stream) {
  require<Err>(pages != nullptr, "paged cache pages pointer is null");
  require<Err>(table != nullptr, "paged cache page_table pointer is null");
  require<Err>(!with_starts || starts != nullptr, "paged cache query_starts pointer is null");
  require<Err>(lengths != nullptr, "paged cache context_lengths pointer is null");
  require<Err>(stream != nullptr, "paged cache HIP stream is null");
  require<Err>(act == RAFTINFER_DTYPE_BF16, "paged cache activations must be bf16");
  require<Err>(aligned16(pages), "paged cache pages must be 16-byte aligned");
  require<Err>(aligned4(table) && aligned4(starts) && aligned4(lengths),
               "paged cache page_table, query_starts and context_lengths must be 4-byte aligned");
  require<Err>(pages_bytes >= pool_bytes(s), "paged cache is too small");
}

std::size_t table_bytes(const Qwen35PagedShape &s) { return s.sequences * s.table_pages * sizeof(std::int32_t); }

void attention(const char *name, bool decode, const void *query, const void *gate, void *output, const void *pages,
               std::size_t pages_bytes, const std::int32_t *table, const std::uint32_t *starts,
               const std::uint32_t *lengths, void *workspace, std::size_t workspace_bytes, const Qwen35PagedShape &s,
               const Qwen35PagedStrides &st, RaftInferDataType act, Qwen35KvCacheLayout layout, hipStream_t stream) {
  validate_shape(s);
  require<Err>(!decode || s.rows == s.sequences, "paged decode takes one row per sequence");
  PagedArgs a = to_args(s, layout);
  require<Err>(query != nullptr, "paged attention query pointer is null");
  require<Err>(output != nullptr, "paged attention output pointer is null");
  validate_pool(s, pages, pages_bytes, table, starts, !decode, lengths, act, stream);
  const Tensor q(s.rows, s.query_heads, st.query_row, st.query_head), g(s.rows, s.query_heads, st.gate_row, st.gate_head),
      o(s.rows, s.query_heads, st.output_row, st.output_head);
  require<Err>(aligned16(query) && aligned16(gate) && aligned16(output),
               "paged attention query, gate and output must be 16-byte aligned");
  require<Err>(strides_apart(s.rows, o.row, s.query_heads, o.head, kHeadDim), "paged attention output rows or heads overlap");
  const std::size_t need = decode ? paged_decode_workspace(a) : paged_prefill_workspace(a);
  require<Err>(need == 0 || workspace != nullptr, "paged attention workspace is null");
  require<Err>(workspace_bytes >= need, "paged attention workspace is too small");
  require<Err>(aligned16(workspace), "paged attention workspace must be 16-byte aligned");
  validate_apart<Err>({{output, o.bytes}, {workspace, need}},
                      {{query, q.bytes}, {gate, gate != nullptr ? g.bytes : 0}, {pages, pool_bytes(s)}, {table, table_bytes(s)},
                       {starts, starts != nullptr ? 4 * (s.sequences + 1) : 0}, {lengths, 4 * s.sequences}},
                      "paged attention outputs overlap other arguments");
  a.query = static_cast<const bf16_bits *>(query);
  a.gate = static_cast<const bf16_bits *>(gate);
  a.output = static_cast<bf16_bits *>(output);
  a.pages = static_cast<const unsigned char *>(pages);
  a.table = table;
  a.starts = starts;
  a.lengths = lengths;
  a.q_row = q.row; a.q_head = q.head;
  a.g_row = g.row; a.g_head = g.head;
  a.o_row = o.row; a.o_head = o.head;
  const StreamDevice<Err> device(stream, "paged attention");
  if (decode) paged_decode(a, workspace, stream);
  else paged_prefill(a, workspace, stream);
  check_launch<Err>(name);
}

} // namespace

std::size_t qwen35_paged_cache_bytes(Qwen35PagedShape shape) {
  validate_shape(shape);
  return pool_bytes(shape);
}

std::size_t qwen35_paged_decode_workspace_bytes(Qwen35PagedShape shape) {
  validate_shape(shape);
  require<Err>(shape.rows == shape.sequences, "paged decode takes one row per sequence");
  return paged_decode_workspace(to_args(shape, Qwen35KvCacheLayout::head_major));
}

std::size_t qwen35_paged_prefill_workspace_bytes(Qwen35PagedShape shape) {
  validate_shape(shape);
  return paged_prefill_workspace(to_args(shape, Qwen35KvCacheLayout::head_major));
}

void qwen35_paged_cache_append(const void *query, const void *key, const void *value, void *query_output, void *pages,
                               std::size_t pages_bytes, const std::int32_t *table, const std::uint32_t *starts,
                               const std::uint32_t *lengths, const double *frequencies, const void *query_weight,
                               const void *key_weight, Qwen35PagedShape s, Qwen35PagedRotary r, RaftInferDataType act,
                               RaftInferDataType weight_dtype, Qwen35KvCacheLayout layout, hipStream_t stream) {
  validate_shape(s);
  PagedAppendArgs x{};
  x.paged = to_args(s, layout);
  require<Err>((query != nullptr) == (query_output != nullptr), "paged append query and query_output go together");
  require<Err>(key != nullptr, "paged append key pointer is null");
  require<Err>(value != nullptr, "paged append value pointer is null");
  validate_pool(s, pages, pages_bytes, table, starts, true, lengths, act, stream);
  require<Err>(r.rotary_dim <= kHeadDim && r.rotary_dim % (r.interleaved ? 8 : 16) == 0,
               "paged append rotary_dim must be 0 to 256, a multiple of 16, or 8 interleaved");
  require<Err>((r.rotary_dim != 0) == (frequencies != nullptr), "paged append frequencies go with rotary_dim");
  require<Err>(std::isfinite(r.magnitude), "rotary magnitude must be finite");
  require<Err>(std::isfinite(r.epsilon) && r.epsilon >= 0.0f, "rotary epsilon must be finite and non-negative");
  const bool weighted = query_weight != nullptr || key_weight != nullptr;
  require<Err>(!weighted || weight_dtype == RAFTINFER_DTYPE_BF16 || weight_dtype == RAFTINFER_DTYPE_F32,
               "paged append weights must be bf16 or f32");
  const Tensor q(s.rows, s.query_heads, r.query_row_stride, r.query_head_stride), k(s.rows, s.kv_heads, r.key_row_stride, r.key_head_stride),
      v(s.rows, s.kv_heads, r.value_row_stride, r.value_head_stride), o(s.rows, s.query_heads, r.output_row_stride, r.output_head_stride);
  require<Err>(aligned16(query) && aligned16(key) && aligned16(value) && aligned16(query_output),
               "paged append inputs and query_output must be 16-byte aligned");
  const std::size_t weight_size = weight_dtype == RAFTINFER_DTYPE_F32 ? 4 : 2;
  require<Err>(((reinterpret_cast<std::uintptr_t>(query_weight) | reinterpret_cast<std::uintptr_t>(key_weight)) & (weight_size - 1)) == 0 &&
                   (reinterpret_cast<std::uintptr_t>(frequencies) & 7) == 0,
               "paged append weights and frequencies must be aligned to their elements");
  require<Err>(strides_apart(s.rows, o.row, s.query_heads, o.head, kHeadDim), "paged append query_output rows or heads overlap");
  validate_apart<Err>({{query_output, query_output != nullptr ? o.bytes : 0}, {pages, pool_bytes(s)}},
                      {{query, query != nullptr ? q.bytes : 0}, {key, k.bytes}, {value, v.bytes}, {table, table_bytes(s)},
                       {starts, 4 * (s.sequences + 1)}, {lengths, 4 * s.sequences}, {frequencies, 4 * r.rotary_dim},
                       {query_weight, query_weight != nullptr ? kHeadDim * weight_size : 0},
                       {key_weight, key_weight != nullptr ? kHeadDim * weight_size : 0}},
                      "paged append outputs overlap other arguments");
  PagedArgs &a = x.paged;
  a.query = static_cast<const bf16_bits *>(query);
  a.output = static_cast<bf16_bits *>(query_output);
  a.table = table;
  a.starts = starts;
  a.lengths = lengths;
  a.q_row = q.row; a.q_head = q.head;
  a.o_row = o.row; a.o_head = o.head;
  x.key = static_cast<const bf16_bits *>(key);
  x.value = static_cast<const bf16_bits *>(value);
  x.pages = static_cast<unsigned char *>(pages);
  x.frequencies = frequencies;
  x.q_weight = query_weight;
  x.k_weight = key_weight;
  x.weight_f32 = weight_dtype == RAFTINFER_DTYPE_F32;
  x.interleaved = r.interleaved;
  x.k_row = k.row; x.k_head = k.head;
  x.v_row = v.row; x.v_head = v.head;
  x.rotary_dim = static_cast<std::uint32_t>(r.rotary_dim);
  x.magnitude = r.magnitude;
  x.epsilon = r.epsilon;
  const StreamDevice<Err> device(stream, "paged append");
  paged_append(x, stream);
  check_launch<Err>("qwen35_paged_cache_append");
}

void qwen35_paged_attention_prefill(const void *query, const void *gate, void *output, const void *pages,
                                    std::size_t pages_bytes, const std::int32_t *page_table,
                                    const std::uint32_t *query_starts, const std::uint32_t *context_lengths, void *workspace,
                                    std::size_t workspace_bytes, Qwen35PagedShape shape, Qwen35PagedStrides strides,
                                    RaftInferDataType act, Qwen35KvCacheLayout layout, hipStream_t stream) {
  attention("qwen35_paged_attention_prefill", false, query, gate, output, pages, pages_bytes, page_table, query_starts,
            context_lengths, workspace, workspace_bytes, shape, strides, act, layout, stream);
}

void qwen35_paged_attention_decode(const void *query, const void *gate, void *output, const void *pages,
                                   std::size_t pages_bytes, const std::int32_t *page_table,
                                   const std::uint32_t *context_lengths, void *workspace, std::size_t workspace_bytes,
                                   Qwen35PagedShape shape, Qwen35PagedStrides strides, RaftInferDataType act,
                                   Qwen35KvCacheLayout layout, hipStream_t stream) {
  attention("qwen35_paged_attention_decode", true, query, gate, output, pages, pages_bytes, page_table, nullptr,
            context_lengths, workspace, workspace_bytes, shape, strides, act, layout, stream);
}

} // namespace raftinfer::kernels
