// The compact KV cache for long contexts (additive; no counterpart in the
// reference): gated attention over a cache held in 8 bits, attention that sees a
// sliding window and a few first tokens, and eviction of the entries that drew
// least attention.  The three share one cache, so a program stores a prompt in 8
// bits, decodes behind a window, and cuts the cache to a budget with the weights
// that the attention calls added up.
//
// Validation failures throw Qwen35PrimitiveError before any launch.  Nothing
// allocates, creates streams or synchronizes; every call may be captured into a
// graph.  Calls that run at the same time need a workspace each.  What a call
// writes (outputs, cache, key weights, workspace) overlaps none of its other
// arguments.
//
// Cache of one sequence: bf16, the layout of the online attention's bf16 cache
// ([K plane | V plane], [kv_head][max_context_tokens][256] head-major or
// [max_context_tokens][kv_head][256] token-major); or 8 bits, the same two planes
// of e4m3 codes, then the scales, float [2][kv_heads][ceil(max_context_tokens /
// 32)] in either layout.  A scale belongs to the 32 positions 32 b .. 32 b + 31 of
// one plane and head.  It is the smallest power of two s with which every finite
// value that was stored is at most 448 s, and a code stands for code * s; under the
// largest scale, 2^120, codes end at 240, since 256 would stand for 2^128, which is
// no f32.  A row that needs a larger scale than its block has raises it, and the
// block's earlier rows are rounded to the new one (exact but for codes that become
// subnormal).  Infinite and NaN values are stored as NaN.  A block's scale starts
// anew with its first position, so a buffer needs no clearing between sequences.
#pragma once

#include "qwen35_attention.hpp"

#include <cstddef>
#include <cstdint>

namespace raftinfer::kernels {

enum class Qwen35CompactCacheDType : std::uint8_t { bf16 = 1, fp8_e4m3 = 2 };

// Positions that share a scale in an 8-bit cache.
inline constexpr std::size_t kQwen35CompactBlockTokens = 32;

struct Qwen35CompactShape {
  std::size_t tokens;      // of each sequence in this call; decode: 1
  std::size_t sequences;   // prefill: 1
  std::size_t query_heads; // a multiple of kv_heads, at most 16 per KV head
  std::size_t kv_heads;
  std::size_t head_dim;    // 256
  std::size_t max_context_tokens;
  std::size_t past_tokens; // positions stored before this call (decode with context_lengths: not read)
  std::size_t cache_stride_bytes; // between sequences' caches (one sequence: not read)
  // A token at position p sees the keys j <= p with j < sink_tokens or
  // j > p - window_tokens; window_tokens 0: all j <= p.
  std::size_t window_tokens;
  std::size_t sink_tokens;
  // The call's last observed_tokens tokens add what attention they pay to each
  // key to key_weights (0: none do, key_weights is null).
  std::size_t observed_tokens;
};

// Eviction of one sequence's cache: of the first context_tokens entries of every
// head, keep_tokens are kept, namely the first sink_tokens, the last
// recent_tokens, and of the others those with the largest weight (equal weights:
// the lower index; NaN counts as the largest).
struct Qwen35EvictShape {
  std::size_t kv_heads;
  std::size_t head_dim; // 256
  std::size_t context_tokens; // at most 65535 * 4096
  std::size_t max_context_tokens;
  std::size_t keep_tokens;
  std::size_t out_max_context_tokens;
  std::size_t sink_tokens;
  std::size_t recent_tokens;
};

// Bytes of one sequence's cache (a multiple of 32).
std::size_t qwen35_compact_cache_bytes(Qwen35CompactShape shape, Qwen35CompactCacheDType cache_dtype);

// Workspace of the calls below, for every past_tokens of the shape.
std::size_t qwen35_compact_decode_workspace_bytes(Qwen35CompactShape shape);
std::size_t qwen35_compact_prefill_workspace_bytes(Qwen35CompactShape shape);
std::size_t qwen35_compact_evict_workspace_bytes(Qwen35EvictShape shape);

// Stores `tokens` rows of every sequence at past_tokens (context_lengths given:
// tokens is 1 and the row goes to length - 1).  key, value: [sequences][tokens]
// [kv_heads][256] bf16.  The attention calls do this themselves.
void qwen35_compact_cache_append(const void *key, const void *value, void *kv_cache,
                                 std::size_t kv_cache_bytes, const std::uint32_t *context_lengths,
                                 Qwen35CompactShape shape, RaftInferDataType activation_dtype,
                                 Qwen35CompactCacheDType cache_dtype, Qwen35KvCacheLayout cache_layout,
                                 hipStream_t stream);

// Stores the rows, then out[t][h] = sigmoid(gate[t][h]) * attention of query[t][h]
// over the cache: softmax(q k / 16) over the keys that the token sees.  query,
// gate, output: [tokens][query_heads][256] bf16.  key_weights: float
// [kv_heads][max_context_tokens], to which each seen key's probabilities are
// added, over the observed tokens and the head's group of query heads.  Before
// the division by the softmax's sum the values are summed in f32 with
// probabilities of at most 1: finite where |probability * value| over a token's
// keys sums to less than 2^128.
void qwen35_compact_attention_prefill(const void *query, const void *key, const void *value,
                                      const void *gate, void *output, void *kv_cache,
                                      std::size_t kv_cache_bytes, float *key_weights, void *workspace,
                                      std::size_t workspace_bytes, Qwen35CompactShape shape,
                                      RaftInferDataType activation_dtype,
                                      Qwen35CompactCacheDType cache_dtype,
                                      Qwen35KvCacheLayout cache_layout, hipStream_t stream);

// The same for one new token of each of `sequences` sequences, [sequences] in place
// of [tokens], caches cache_stride_bytes apart, key_weights
// [sequences][kv_heads][max_context_tokens].  context_lengths (device,
// uint32[sequences]): each sequence's context, the new token included, which is
// stored at length - 1; null: past_tokens + 1 for all.  A length of 0 or above
// max_context_tokens makes that sequence's output NaN, stores nothing and is
// counted (qwen35_online_attention_consume_capacity_errors).
void qwen35_compact_attention_decode(const void *query, const void *key, const void *value,
                                     const void *gate, void *output, void *kv_cache,
                                     std::size_t kv_cache_bytes, const std::uint32_t *context_lengths,
                                     float *key_weights, void *workspace, std::size_t workspace_bytes,
                                     Qwen35CompactShape shape, RaftInferDataType activation_dtype,
                                     Qwen35CompactCacheDType cache_dtype,
                                     Qwen35KvCacheLayout cache_layout, hipStream_t stream);

// Copies the kept entries of every head, in their order, to positions 0 ..
// keep_tokens - 1 of out_cache, their weights to out_weights (float
// [kv_heads][out_max_context_tokens], 0 behind them), and their indices to
// kept_indices (int32 [kv_heads][keep_tokens]).  key_weights: float
// [kv_heads][max_context_tokens].  A bf16 cache may go to an 8-bit one; 8-bit
// blocks get the scales that their new rows need.
void qwen35_compact_cache_evict(const void *kv_cache, std::size_t kv_cache_bytes,
                                const float *key_weights, void *out_cache, std::size_t out_cache_bytes,
                                float *out_weights, std::int32_t *kept_indices, void *workspace,
                                std::size_t workspace_bytes, Qwen35EvictShape shape,
                                Qwen35CompactCacheDType cache_dtype,
                                Qwen35CompactCacheDType out_cache_dtype,
                                Qwen35KvCacheLayout cache_layout, hipStream_t stream);

} // namespace raftinfer::kernels
