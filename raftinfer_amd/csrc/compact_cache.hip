// Entry points, sizing and the row store of the compact KV cache
// (include/raftinfer_amd/qwen35_compact_cache.hpp).
#include "compact_cache.hpp"
#include "raftinfer_amd/qwen35_compact_cache.hpp"

#include <initializer_list>

namespace raftinfer::amd {
namespace {

constexpr int kStoreThreads = 256;

// Positions stored before this call, or false where the length is out of range.
__device__ __forceinline__ bool stored_before(const CompactArgs &a, std::uint32_t seq, std::uint32_t &past) {
  past = a.past;
  if (a.lengths == nullptr) return true;
  const std::uint32_t n = a.lengths[seq];
  past = n - 1;
  return n != 0 && n <= a.max_ctx;
}

// bf16 rows, 16 bytes a thread: grid (pieces of tokens * kv_heads rows, 2 planes, sequences).
// A copy, at the rate of one (6001 tokens of 4 KV heads 10.0 us, 4.9 TB/s read and written).
__global__ __launch_bounds__(kStoreThreads) void compact_store_bf16_kernel(CompactArgs a) {
  const std::size_t i = static_cast<std::size_t>(blockIdx.x) * kStoreThreads + threadIdx.x;
  const std::size_t rows = static_cast<std::size_t>(a.tokens) * a.kv_heads;
  const std::size_t r = i >> 5;
  std::uint32_t past;
  if (r >= rows || !stored_before(a, blockIdx.z, past)) return;
  const auto t = static_cast<std::uint32_t>(r / a.kv_heads), kvh = static_cast<std::uint32_t>(r % a.kv_heads);
  CompactHead<false> c(a.cache + blockIdx.z * a.cache_stride, kvh, a.kv_heads, a.max_ctx, a.head_major);
  const bf16_bits *src = (blockIdx.y ? a.value : a.key) + (blockIdx.z * rows + r) * kHeadDim + 8 * (i & 31);
  bf16_bits *dst = (blockIdx.y ? c.v : c.k) + static_cast<std::size_t>(past + t) * c.row + 8 * (i & 31);
  *reinterpret_cast<u32x4 *>(dst) = *reinterpret_cast<const u32x4 *>(src);
}

// 8-bit rows: a workgroup owns one block of one plane and head (grid (blocks that
// the call reaches, 2 kv_heads, sequences)), thread (row, piece) = (tid / 8,
// tid % 8) 32 dims of one of its positions.  Rows that the call stores are read
// from key / value; rows from before keep their codes, rounded again where the
// block's scale grew (a division by a power of two, exact for normal codes).  Two round
// trips to memory and a barrier bound it: 500 tokens of 4 KV heads 3.9 us.
__global__ __launch_bounds__(kStoreThreads) void compact_store_fp8_kernel(CompactArgs a) {
  __shared__ float wave_max_of[kStoreThreads / kWave];
  std::uint32_t past;
  const std::uint32_t seq = blockIdx.z;
  if (!stored_before(a, seq, past)) return; // (uniform)
  const std::uint32_t kvh = blockIdx.y >> 1, plane = blockIdx.y & 1;
  const std::uint32_t block = past / kCompactBlock + blockIdx.x;
  const std::uint32_t end = past + a.tokens;
  if (block * kCompactBlock >= end) return; // (uniform)
  const std::uint32_t pos = block * kCompactBlock + (threadIdx.x >> 3);
  const int piece = threadIdx.x & 7;
  CompactHead<true> c(a.cache + seq * a.cache_stride, kvh, a.kv_heads, a.max_ctx, a.head_major);
  unsigned char *codes = (plane ? c.v : c.k) + static_cast<std::size_t>(pos) * c.row + 32 * piece;
  float *scale = (plane ? c.vs : c.ks) + block;
  const bool fresh = pos >= past && pos < end;
  const bool old = pos < past;
  float x[32];
  float amax = 0.f;
  if (fresh) {
    const std::size_t row = (static_cast<std::size_t>(seq) * a.tokens + (pos - past)) * a.kv_heads + kvh;
    const bf16_bits *src = (plane ? a.value : a.key) + row * kHeadDim + 32 * piece;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32x4 w = reinterpret_cast<const u32x4 *>(src)[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const std::uint32_t u = w[e];
        x[8 * j + 2 * e] = bf16_lo(u);
        x[8 * j + 2 * e + 1] = bf16_hi(u);
      }
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      if (is_finite_f32(x[e])) amax = fmaxf(amax, fabsf(x[e]));
      else x[e] = __builtin_nanf("");
    }
  }
  amax = wave_max(amax);
  if ((threadIdx.x & 63) == 0) wave_max_of[threadIdx.x >> 6] = amax;
  const bool has_old = block * kCompactBlock < past;
  const float before = has_old ? *scale : 0.f;
  __syncthreads(); // every thread has read the old scale
  amax = fmaxf(fmaxf(wave_max_of[0], wave_max_of[1]), fmaxf(wave_max_of[2], wave_max_of[3]));
  const float after = fmaxf(before, compact_scale(amax));
  const float inv = compact_inverse(after);
  if (threadIdx.x == 0) *scale = after;
  u32x4 out[2];
  if (fresh) {
    if (after == kCompactTopScale) {
#pragma unroll
      for (int e = 0; e < 32; ++e) x[e] = compact_below_top(x[e]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      out[j >> 2][j & 3] = pack_fp8x4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
  } else if (old && after != before) {
    const float ratio = before * inv;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 w = reinterpret_cast<const u32x4 *>(codes)[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const floatx4 f = fp8x4_to_f32(w[e]);
        out[j][e] = pack_fp8x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
      }
    }
  } else {
    return;
  }
  reinterpret_cast<u32x4 *>(codes)[0] = out[0];
  reinterpret_cast<u32x4 *>(codes)[1] = out[1];
}

} // namespace

void compact_append(const CompactArgs &a, bool fp8, hipStream_t stream) {
  if (fp8) {
    const std::uint32_t blocks =
        a.tokens == 1 ? 1u : (a.past % kCompactBlock + a.tokens + kCompactBlock - 1) / kCompactBlock;
    compact_store_fp8_kernel<<<dim3{blocks, 2 * a.kv_heads, a.sequences}, kStoreThreads, 0, stream>>>(a);
  } else {
    const std::size_t pieces = static_cast<std::size_t>(a.tokens) * a.kv_heads * 32;
    const auto blocks = static_cast<unsigned>(ceil_div_unchecked(pieces, kStoreThreads));
    compact_store_bf16_kernel<<<dim3{blocks, 2, a.sequences}, kStoreThreads, 0, stream>>>(a);
  }
}

} // namespace raftinfer::amd

namespace raftinfer::kernels {
namespace {

using namespace raftinfer::amd;
using Err = Qwen35PrimitiveError;

// Positions, rows and columns are 32-bit in the kernels, and a grid holds fewer than
// 2^32 threads in x and 2^16 workgroups in y and z.  At these limits the threads in x are:
// stores 2^26 rows * 32, or 2^26 / 32 blocks * 256; decode 2^17 units * 64 partitions * 256; its merge (2^31 /
// 512 + 2^15 pieces of weights + 2^19 heads) * 512; prefill 2^26 / 128 + 2^15 column blocks * 256 (few
// enough are cut that the merge of their columns, a wave or a workgroup each, is below 2^24); key weights 2^22 tiles * 512
// (kWeighGrid; a launch more for others); eviction 2^15 heads * 1024 and 2^28 / 32 blocks * 256.
constexpr std::size_t kMaxPositions = std::size_t{1} << 28;
constexpr std::size_t kMaxHeadPositions = std::size_t{1} << 31; // over all KV heads
constexpr std::size_t kMaxQueryRows = std::size_t{1} << 26;
constexpr std::size_t kMaxUnits = std::size_t{1} << 17; // sequences times KV heads
constexpr std::size_t kMaxGrid = 65535;
constexpr std::size_t kMaxEvictContext = kMaxGrid * 4096; // (the documented limit)

std::size_t cache_bytes_of(std::size_t positions, std::size_t kv_heads, Qwen35CompactCacheDType dtype) {
  const char *overflow = "compact cache byte size overflow";
  require<Err>(dtype == Qwen35CompactCacheDType::bf16 || dtype == Qwen35CompactCacheDType::fp8_e4m3,
               "unsupported compact cache dtype");
  const std::size_t values =
      checked_mul<Err>(checked_mul<Err>(positions, 2 * kHeadDim, overflow), kv_heads, overflow);
  if (dtype == Qwen35CompactCacheDType::bf16) return checked_mul<Err>(values, 2, overflow);
  // 4-byte scales of 2 planes, rounded up so that caches can lie one behind the other
  const std::size_t scales =
      checked_mul<Err>(checked_mul<Err>(ceil_div_unchecked(positions, kQwen35CompactBlockTokens), 8, overflow),
                       kv_heads, overflow);
  return checked_add<Err>(values, (scales + 31) / 32 * 32, overflow);
}

void validate_heads(std::size_t kv_heads, std::size_t head_dim) {
  require<Err>(kv_heads > 0 && kv_heads <= kMaxGrid / 2, "compact cache kv_heads must be 1 to 32767");
  require<Err>(head_dim == kHeadDim, "compact cache head_dim must be 256");
}

void validate_positions(std::size_t positions, std::size_t kv_heads) {
  require<Err>(positions > 0 && positions <= kMaxPositions && positions <= kMaxHeadPositions / kv_heads,
               "compact attention max_context_tokens must be 1 to 2^28, 2^31 over all KV heads");
}

void validate_layout(Qwen35KvCacheLayout layout) {
  require<Err>(layout == Qwen35KvCacheLayout::token_major || layout == Qwen35KvCacheLayout::head_major,
               "unsupported compact cache layout");
}

// The stream's device for the launches of a call, where another one is current.
class StreamDevice {
public:
  explicit StreamDevice(hipStream_t stream) {
    int device = 0;
    require<Err>(hipGetDevice(&current_) == hipSuccess && hipStreamGetDevice(stream, &device) == hipSuccess,
                 "compact attention HIP stream has no device");
    if (device == current_) return;
    require<Err>(hipSetDevice(device) == hipSuccess, "compact attention cannot select the stream's device");
    changed_ = true;
  }
  ~StreamDevice() {
    if (changed_) (void)hipSetDevice(current_);
  }
  StreamDevice(const StreamDevice &) = delete;
  StreamDevice &operator=(const StreamDevice &) = delete;

private:
  int current_ = 0;
  bool changed_ = false;
};

bool aligned16(const void *p) { return (reinterpret_cast<std::uintptr_t>(p) & 15u) == 0; }

// lengths_given: past_tokens is not read.
void validate_shape(const Qwen35CompactShape &s, bool lengths_given) {
  validate_heads(s.kv_heads, s.head_dim);
  require<Err>(s.tokens > 0, "compact attention tokens must be positive");
  require<Err>(s.sequences > 0 && s.sequences <= kMaxGrid, "compact attention sequences must be 1 to 65535");
  validate_positions(s.max_context_tokens, s.kv_heads);
  require<Err>(s.sequences <= kMaxUnits / s.kv_heads, "compact attention has too many sequences and KV heads");
  require<Err>(s.query_heads > 0 && s.query_heads % s.kv_heads == 0 &&
                   s.query_heads / s.kv_heads <= kCompactMaxGroup,
               "compact attention query_heads must be 1 to 16 per KV head");
  require<Err>(s.tokens <= kMaxQueryRows / s.query_heads, "compact attention has too many query rows");
  if (!lengths_given)
    require<Err>(s.tokens <= s.max_context_tokens && s.past_tokens <= s.max_context_tokens - s.tokens,
                 "compact attention context exceeds cache capacity");
  require<Err>(s.observed_tokens <= s.tokens, "compact attention observes more tokens than the call has");
}

struct Bytes {
  const void *at;
  std::size_t count;
};
// What a call writes overlaps neither what it reads nor what else it writes.
void validate_apart(std::initializer_list<Bytes> written, std::initializer_list<Bytes> read, const char *message) {
  const auto apart = [](const Bytes &a, const Bytes &b) {
    const auto x = reinterpret_cast<std::uintptr_t>(a.at), y = reinterpret_cast<std::uintptr_t>(b.at);
    return x <= y ? a.count <= y - x : b.count <= x - y;
  };
  for (auto w = written.begin(); w != written.end(); ++w) {
    for (auto other = w + 1; other != written.end(); ++other) require<Err>(apart(*w, *other), message);
    for (const Bytes &r : read) require<Err>(apart(*w, r), message);
  }
}
Bytes lengths_of(const Qwen35CompactShape &s, const std::uint32_t *lengths) {
  return {lengths, lengths != nullptr ? s.sequences * sizeof(std::uint32_t) : 0};
}
void validate_lengths(const std::uint32_t *lengths) {
  require<Err>((reinterpret_cast<std::uintptr_t>(lengths) & 3u) == 0, "compact attention context_lengths must be 4-byte aligned");
}
// Checked last: everything else about the call is valid.
void validate_overlap(const Qwen35CompactShape &s, const void *q, const void *k, const void *v, const void *g,
                      const void *output, const void *cache, std::size_t cache_bytes, const std::uint32_t *lengths,
                      const float *weights, const void *workspace, std::size_t workspace_bytes) {
  const std::size_t tokens = s.sequences * s.tokens;
  const std::size_t heads = tokens * s.query_heads * kHeadDim * 2, rows = tokens * s.kv_heads * kHeadDim * 2;
  const std::size_t weight_bytes = weights != nullptr ? s.sequences * s.kv_heads * s.max_context_tokens * sizeof(float) : 0;
  validate_apart({{output, heads}, {cache, cache_bytes}, {weights, weight_bytes}, {workspace, workspace_bytes}},
                 {{q, heads}, {k, rows}, {v, rows}, {g, heads}, lengths_of(s, lengths)},
                 "compact attention outputs overlap other arguments");
}

std::size_t validate_cache(const Qwen35CompactShape &s, Qwen35CompactCacheDType dtype, const void *cache,
                    std::size_t bytes) {
  const std::size_t one = cache_bytes_of(s.max_context_tokens, s.kv_heads, dtype);
  require<Err>(cache != nullptr, "compact cache pointer is null");
  require<Err>(aligned16(cache), "compact cache must be 16-byte aligned");
  std::size_t need = one;
  if (s.sequences > 1) {
    require<Err>(s.cache_stride_bytes >= one && s.cache_stride_bytes % 16 == 0,
                 "compact cache stride is too small or no multiple of 16");
    need = checked_add<Err>(checked_mul<Err>(s.sequences - 1, s.cache_stride_bytes, "compact cache byte size overflow"),
                            one, "compact cache byte size overflow");
  }
  require<Err>(bytes >= need, "compact cache is too small");
  return need;
}

CompactArgs to_args(const Qwen35CompactShape &s) {
  CompactArgs a{};
  a.cache_stride = s.sequences > 1 ? s.cache_stride_bytes : 0;
  a.tokens = static_cast<std::uint32_t>(s.tokens);
  a.sequences = static_cast<std::uint32_t>(s.sequences);
  a.kv_heads = static_cast<std::uint32_t>(s.kv_heads);
  a.group = static_cast<std::uint32_t>(s.query_heads / s.kv_heads);
  a.max_ctx = static_cast<std::uint32_t>(s.max_context_tokens);
  a.past = static_cast<std::uint32_t>(s.past_tokens < kMaxPositions ? s.past_tokens : 0);
  // a window that holds every position is none
  a.window = s.window_tokens < s.max_context_tokens ? static_cast<std::uint32_t>(s.window_tokens) : 0;
  a.sinks = static_cast<std::uint32_t>(s.sink_tokens < s.max_context_tokens ? s.sink_tokens : s.max_context_tokens);
  a.observed = static_cast<std::uint32_t>(s.observed_tokens);
  return a;
}

void fill_pointers(CompactArgs &a, const void *q, const void *k, const void *v, const void *g, void *o, void *cache,
                   Qwen35KvCacheLayout layout) {
  a.query = static_cast<const bf16_bits *>(q);
  a.key = static_cast<const bf16_bits *>(k);
  a.value = static_cast<const bf16_bits *>(v);
  a.gate = static_cast<const bf16_bits *>(g);
  a.output = static_cast<bf16_bits *>(o);
  a.cache = static_cast<unsigned char *>(cache);
  a.head_major = layout == Qwen35KvCacheLayout::head_major;
}

void validate_call(const void *q, const void *k, const void *v, const void *g, const void *o, const float *weights,
                   const void *workspace, std::size_t workspace_bytes, std::size_t need,
                   const Qwen35CompactShape &s, RaftInferDataType act, Qwen35KvCacheLayout layout,
                   hipStream_t stream) {
  require<Err>(q != nullptr, "compact attention query pointer is null");
  require<Err>(k != nullptr, "compact attention key pointer is null");
  require<Err>(v != nullptr, "compact attention value pointer is null");
  require<Err>(g != nullptr, "compact attention gate pointer is null");
  require<Err>(o != nullptr, "compact attention output pointer is null");
  require<Err>(stream != nullptr, "compact attention HIP stream is null");
  require<Err>(act == RAFTINFER_DTYPE_BF16, "compact attention activations must be bf16");
  validate_layout(layout);
  require<Err>(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(g) && aligned16(o),
               "compact attention inputs and output must be 16-byte aligned");
  require<Err>((weights != nullptr) == (s.observed_tokens > 0),
               "compact attention key_weights go with observed_tokens");
  require<Err>((reinterpret_cast<std::uintptr_t>(weights) & 3u) == 0,
               "compact attention key_weights must be 4-byte aligned");
  require<Err>(need == 0 || workspace != nullptr, "compact attention workspace is null");
  require<Err>(workspace_bytes >= need, "compact attention workspace is too small");
  require<Err>(aligned16(workspace), "compact attention workspace must be 16-byte aligned");
}

} // namespace

std::size_t qwen35_compact_cache_bytes(Qwen35CompactShape shape, Qwen35CompactCacheDType dtype) {
  validate_heads(shape.kv_heads, shape.head_dim);
  validate_positions(shape.max_context_tokens, shape.kv_heads);
  return cache_bytes_of(shape.max_context_tokens, shape.kv_heads, dtype);
}

std::size_t qwen35_compact_decode_workspace_bytes(Qwen35CompactShape shape) {
  validate_shape(shape, true);
  require<Err>(shape.tokens == 1, "compact decode takes one token per sequence");
  return compact_decode_workspace(to_args(shape));
}

std::size_t qwen35_compact_prefill_workspace_bytes(Qwen35CompactShape shape) {
  validate_shape(shape, true);
  require<Err>(shape.sequences == 1, "compact prefill takes one sequence");
  require<Err>(shape.tokens <= shape.max_context_tokens, "compact attention context exceeds cache capacity");
  return compact_prefill_workspace(to_args(shape));
}

void qwen35_compact_cache_append(const void *key, const void *value, void *kv_cache,
                                 std::size_t kv_cache_bytes, const std::uint32_t *context_lengths,
                                 Qwen35CompactShape shape, RaftInferDataType act,
                                 Qwen35CompactCacheDType cache_dtype, Qwen35KvCacheLayout layout,
                                 hipStream_t stream) {
  require<Err>(key != nullptr, "compact attention key pointer is null");
  require<Err>(value != nullptr, "compact attention value pointer is null");
  require<Err>(stream != nullptr, "compact attention HIP stream is null");
  require<Err>(act == RAFTINFER_DTYPE_BF16, "compact attention activations must be bf16");
  validate_shape(shape, context_lengths != nullptr);
  require<Err>(context_lengths == nullptr || shape.tokens == 1, "compact append with lengths stores one token per sequence");
  validate_layout(layout);
  const std::size_t used = validate_cache(shape, cache_dtype, kv_cache, kv_cache_bytes);
  require<Err>(aligned16(key) && aligned16(value), "compact attention inputs and output must be 16-byte aligned");
  const std::size_t rows = shape.sequences * shape.tokens * shape.kv_heads * kHeadDim * 2;
  validate_lengths(context_lengths);
  validate_apart({{kv_cache, used}}, {{key, rows}, {value, rows}, lengths_of(shape, context_lengths)},
                 "compact cache overlaps the rows to be stored or their lengths");
  CompactArgs a = to_args(shape);
  fill_pointers(a, nullptr, key, value, nullptr, nullptr, kv_cache, layout);
  a.lengths = context_lengths;
  const StreamDevice device(stream);
  compact_append(a, cache_dtype == Qwen35CompactCacheDType::fp8_e4m3, stream);
  check_launch<Err>("qwen35_compact_cache_append");
}

void qwen35_compact_attention_prefill(const void *query, const void *key, const void *value,
                                      const void *gate, void *output, void *kv_cache,
                                      std::size_t kv_cache_bytes, float *key_weights, void *workspace,
                                      std::size_t workspace_bytes, Qwen35CompactShape shape,
                                      RaftInferDataType act, Qwen35CompactCacheDType cache_dtype,
                                      Qwen35KvCacheLayout layout, hipStream_t stream) {
  validate_shape(shape, false);
  const std::size_t need = qwen35_compact_prefill_workspace_bytes(shape);
  validate_call(query, key, value, gate, output, key_weights, workspace, workspace_bytes, need, shape, act, layout,
                stream);
  const std::size_t used = validate_cache(shape, cache_dtype, kv_cache, kv_cache_bytes);
  validate_overlap(shape, query, key, value, gate, output, kv_cache, used, nullptr, key_weights, workspace, need);
  CompactArgs a = to_args(shape);
  fill_pointers(a, query, key, value, gate, output, kv_cache, layout);
  a.weights = key_weights;
  const StreamDevice device(stream);
  compact_prefill(a, cache_dtype == Qwen35CompactCacheDType::fp8_e4m3, workspace, stream);
  check_launch<Err>("qwen35_compact_attention_prefill");
}

void qwen35_compact_attention_decode(const void *query, const void *key, const void *value,
                                     const void *gate, void *output, void *kv_cache,
                                     std::size_t kv_cache_bytes, const std::uint32_t *context_lengths,
                                     float *key_weights, void *workspace, std::size_t workspace_bytes,
                                     Qwen35CompactShape shape, RaftInferDataType act,
                                     Qwen35CompactCacheDType cache_dtype, Qwen35KvCacheLayout layout,
                                     hipStream_t stream) {
  validate_shape(shape, context_lengths != nullptr);
  const std::size_t need = qwen35_compact_decode_workspace_bytes(shape);
  validate_call(query, key, value, gate, output, key_weights, workspace, workspace_bytes, need, shape, act, layout,
                stream);
  const std::size_t used = validate_cache(shape, cache_dtype, kv_cache, kv_cache_bytes);
  validate_lengths(context_lengths);
  validate_overlap(shape, query, key, value, gate, output, kv_cache, used, context_lengths, key_weights, workspace, need);
  CompactArgs a = to_args(shape);
  fill_pointers(a, query, key, value, gate, output, kv_cache, layout);
  a.weights = key_weights;
  a.lengths = context_lengths;
  const StreamDevice device(stream);
  compact_decode(a, cache_dtype == Qwen35CompactCacheDType::fp8_e4m3, workspace, stream);
  check_launch<Err>("qwen35_compact_attention_decode");
}

namespace {

CompactEvictArgs evict_args(const Qwen35EvictShape &s) {
  validate_heads(s.kv_heads, s.head_dim);
  require<Err>(s.context_tokens > 0, "compact eviction context_tokens must be positive");
  validate_positions(s.max_context_tokens, s.kv_heads);
  validate_positions(s.out_max_context_tokens, s.kv_heads);
  require<Err>(s.context_tokens <= s.max_context_tokens, "compact eviction context exceeds cache capacity");
  require<Err>(s.context_tokens <= kMaxEvictContext, "compact eviction context_tokens must be at most 65535 * 4096");
  require<Err>(s.keep_tokens > 0 && s.keep_tokens <= s.context_tokens,
               "compact eviction keep_tokens must be 1 to context_tokens");
  require<Err>(s.keep_tokens <= s.out_max_context_tokens, "compact eviction keeps more than the new cache holds");
  require<Err>(s.sink_tokens <= s.keep_tokens && s.recent_tokens <= s.keep_tokens - s.sink_tokens,
               "compact eviction keep_tokens are fewer than the sinks and the recent tokens");
  CompactEvictArgs a{};
  a.kv_heads = static_cast<std::uint32_t>(s.kv_heads);
  a.context = static_cast<std::uint32_t>(s.context_tokens);
  a.max_ctx = static_cast<std::uint32_t>(s.max_context_tokens);
  a.keep = static_cast<std::uint32_t>(s.keep_tokens);
  a.out_max_ctx = static_cast<std::uint32_t>(s.out_max_context_tokens);
  a.sinks = static_cast<std::uint32_t>(s.sink_tokens);
  a.recent = static_cast<std::uint32_t>(s.recent_tokens);
  return a;
}

} // namespace

std::size_t qwen35_compact_evict_workspace_bytes(Qwen35EvictShape shape) {
  return compact_evict_workspace(evict_args(shape));
}

void qwen35_compact_cache_evict(const void *kv_cache, std::size_t kv_cache_bytes, const float *key_weights,
                                void *out_cache, std::size_t out_cache_bytes, float *out_weights,
                                std::int32_t *kept_indices, void *workspace, std::size_t workspace_bytes,
                                Qwen35EvictShape shape, Qwen35CompactCacheDType cache_dtype,
                                Qwen35CompactCacheDType out_cache_dtype, Qwen35KvCacheLayout layout,
                                hipStream_t stream) {
  CompactEvictArgs a = evict_args(shape);
  require<Err>(kv_cache != nullptr && out_cache != nullptr, "compact cache pointer is null");
  require<Err>(key_weights != nullptr && out_weights != nullptr, "compact eviction key weights pointer is null");
  require<Err>(kept_indices != nullptr, "compact eviction kept_indices pointer is null");
  require<Err>(stream != nullptr, "compact attention HIP stream is null");
  validate_layout(layout);
  require<Err>(kv_cache_bytes >= cache_bytes_of(shape.max_context_tokens, shape.kv_heads, cache_dtype) &&
                   out_cache_bytes >= cache_bytes_of(shape.out_max_context_tokens, shape.kv_heads, out_cache_dtype),
               "compact cache is too small");
  require<Err>(cache_dtype == out_cache_dtype || cache_dtype == Qwen35CompactCacheDType::bf16,
               "compact eviction does not widen an 8-bit cache");
  require<Err>(aligned16(kv_cache) && aligned16(out_cache), "compact cache must be 16-byte aligned");
  const auto bits = reinterpret_cast<std::uintptr_t>(key_weights) | reinterpret_cast<std::uintptr_t>(out_weights) |
                    reinterpret_cast<std::uintptr_t>(kept_indices);
  require<Err>((bits & 3u) == 0, "compact eviction weights and indices must be 4-byte aligned");
  const std::size_t need = compact_evict_workspace(a);
  require<Err>(need == 0 || workspace != nullptr, "compact attention workspace is null");
  require<Err>(workspace_bytes >= need, "compact attention workspace is too small");
  require<Err>(aligned16(workspace), "compact attention workspace must be 16-byte aligned");
  const std::size_t in_bytes = cache_bytes_of(shape.max_context_tokens, shape.kv_heads, cache_dtype);
  const std::size_t out_bytes = cache_bytes_of(shape.out_max_context_tokens, shape.kv_heads, out_cache_dtype);
  validate_apart({{out_cache, out_bytes},
                  {out_weights, shape.kv_heads * shape.out_max_context_tokens * sizeof(float)},
                  {kept_indices, shape.kv_heads * shape.keep_tokens * sizeof(std::int32_t)},
                  {workspace, need}},
                 {{kv_cache, in_bytes}, {key_weights, shape.kv_heads * shape.max_context_tokens * sizeof(float)}},
                 "compact eviction outputs overlap other arguments");
  a.cache = static_cast<const unsigned char *>(kv_cache);
  a.weights = key_weights;
  a.out_cache = static_cast<unsigned char *>(out_cache);
  a.out_weights = out_weights;
  a.kept = kept_indices;
  a.head_major = layout == Qwen35KvCacheLayout::head_major;
  const StreamDevice device(stream);
  compact_evict(a, cache_dtype == Qwen35CompactCacheDType::fp8_e4m3,
                out_cache_dtype == Qwen35CompactCacheDType::fp8_e4m3, workspace, stream);
  check_launch<Err>("qwen35_compact_cache_evict");
}

} // namespace raftinfer::kernels
