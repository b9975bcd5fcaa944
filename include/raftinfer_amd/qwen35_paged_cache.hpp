// Rotary positions of heads row by row, and the paged KV cache (additive; no
// counterpart in the reference): keys and values of many sequences in the pages of
// one pool, gated attention of a ragged batch's new tokens over them.  A serving
// step is qwen35_paged_cache_append (norm and rotation of the new queries and keys,
// store of the new rows), then qwen35_paged_attention_prefill, or _decode where every
// sequence has one new token.
//
// Validation failures throw Qwen35PrimitiveError before any launch.  Nothing
// allocates, creates streams or synchronizes; every call may be captured into a
// graph.  Calls that run at the same time need a workspace each.  What a call writes
// overlaps none of its other arguments, but for the rows that qwen35_rotary turns in
// place.
//
// Pool: bf16 [pages][K, V][kv_heads][page_tokens][256] (head-major) or
// [pages][K, V][page_tokens][kv_heads][256] (token-major).  Page table, device int32
// [sequences][table_pages]: entry i of a sequence is the page of its positions
// i page_tokens .. (i + 1) page_tokens - 1.  Only entries of positions that a call
// stores or that its new tokens see are used; the others may hold anything.
//
// Ragged batch: query_starts, device uint32 [sequences + 1], not falling: sequence s
// has the call's rows query_starts[s] .. query_starts[s + 1] - 1 (none: it takes no
// part); context_lengths, device uint32 [sequences]: its context c, the n new tokens
// included, which are positions c - n .. c - 1.  Rows in front of the first and behind
// the last sequence's are left as they were.
//
// What the host cannot check is checked on the device, before any access: a sequence
// whose rows fall or end behind the call's, whose context is below its new tokens or
// above max_context_tokens or the table's positions, or that needs a page number that is not below `pages`.  The
// attention calls make such a sequence's rows NaN (a bad page: at least the rows that
// see it; rows behind the call's are not written), the append stores none of it (a bad
// page: none of the rows that belong there).  Each is counted at least once
// (qwen35_online_attention_consume_capacity_errors).  Where query_starts fall, sequences
// can share rows: such rows, and any row of that batch, may hold NaN, what another of the
// sequences gives them, or what they held; nothing else is written.
#pragma once

#include "qwen35_attention.hpp"

#include <cstddef>
#include <cstdint>

namespace raftinfer::kernels {

// How the frequencies of a rotation are scaled for positions beyond the trained ones.
// f_p = base^(-2 p / rotary_dim) is pair p's angle per position, its turns over the
// trained context t_p = f_p trained_tokens / 2 pi.  by_pair and by_turns keep the
// frequencies that turn often and divide those that do not turn: f_p (k + (1 - k) /
// factor).  by_turns: k = (t_p - slow_turns) / (fast_turns - slow_turns), held to 0 .. 1.
// by_pair: k falls from 1 to 0 between the pair (rounded down) that turns fast_turns
// times and the one (rounded up) that turns slow_turns times, held to 0 .. rotary_dim - 1.
// (Models with by_pair have 32 and 1 for fast_turns and slow_turns, models with by_turns 4 and 1.)
enum class Qwen35RotaryScaling : std::uint8_t { none = 0, linear = 1, by_pair = 2, by_turns = 3 };

// Writes rotary_dim / 2 frequencies (host) for the calls below, which take them in
// device memory.  linear: f_p / factor.  trained_tokens, fast_turns and slow_turns are
// read by by_pair and by_turns.  Returns the magnitude that goes with them: by_pair
// 0.1 ln(factor) + 1, else 1.
float qwen35_rotary_frequencies(double *frequencies, std::size_t rotary_dim, double base,
                                Qwen35RotaryScaling scaling, double factor, double trained_tokens,
                                double fast_turns, double slow_turns);

// Strides in elements between rows and heads; 0: as [rows][heads][head_dim] without gaps.
struct Qwen35RotaryShape {
  std::size_t rows;
  std::size_t heads;
  std::size_t head_dim;   // at most 16384
  std::size_t rotary_dim; // the first dims of a head, an even number of them
  bool interleaved;       // pair p is dims 2 p, 2 p + 1; else p, p + rotary_dim / 2
  float magnitude;        // cos and sin are multiplied by it
  std::size_t input_row_stride, input_head_stride, output_row_stride, output_head_stride;
};

// output = RoPE(input / rms(input) * weight) of every head, by the rows' positions
// (device uint32 [rows]); weight null: RoPE(input).  frequencies: device double
// [rotary_dim / 2].  An angle is position * frequency in 64 bits, reduced to one turn.
// The mean of a head's squares is held in 32 bits: right for sums of squares below 2^128, and
// with epsilon 0 for a mean of at least 2^-126 (smaller ones lose bits, below 2^-149 it is 0).
// output may be input, with the same strides.
void qwen35_rotary(const void *input, const void *weight, void *output, const std::uint32_t *positions,
                   const double *frequencies, Qwen35RotaryShape shape, float epsilon,
                   RaftInferDataType dtype, RaftInferDataType weight_dtype, hipStream_t stream);

struct Qwen35PagedShape {
  std::size_t rows;        // of the call's tensors: at least the new tokens of all sequences
  std::size_t sequences;
  std::size_t query_heads; // a multiple of kv_heads, at most 16 per KV head
  std::size_t kv_heads;
  std::size_t head_dim;    // 256
  std::size_t pages;       // of the pool
  std::size_t page_tokens; // a multiple of 16
  std::size_t table_pages;
  std::size_t max_context_tokens; // of the call's sequences, at most 2^28; above table_pages * page_tokens: that many
  std::size_t window_tokens; // a token at position p sees j <= p with j > p - window_tokens; 0: all j <= p
};

// Norm, rotation and strides of an append.  Strides as above; multiples of 8.
struct Qwen35PagedRotary {
  std::size_t rotary_dim; // 0: no rotation, frequencies is null
  bool interleaved;
  float magnitude;
  float epsilon;
  std::size_t query_row_stride, query_head_stride, key_row_stride, key_head_stride;
  std::size_t value_row_stride, value_head_stride, output_row_stride, output_head_stride;
};

// Strides of an attention call's query, gate and output; multiples of 8.
struct Qwen35PagedStrides {
  std::size_t query_row, query_head, gate_row, gate_head, output_row, output_head;
};

// Bytes of a pool.
std::size_t qwen35_paged_cache_bytes(Qwen35PagedShape shape);

// Workspace of the attention calls, for every batch of the shape.
std::size_t qwen35_paged_decode_workspace_bytes(Qwen35PagedShape shape);
std::size_t qwen35_paged_prefill_workspace_bytes(Qwen35PagedShape shape);

// Of every row that belongs to a sequence: query_output = RoPE(norm(query)),
// RoPE(norm(key)) and value to the row's position in the pages.  query [rows]
// [query_heads][256] (null, with query_output: only keys and values), key and value
// [rows][kv_heads][256], bf16.  query_weight, key_weight [256], bf16 or f32; null: that
// one is not normalised.  One rounding to bf16, of the turned value.
void qwen35_paged_cache_append(const void *query, const void *key, const void *value, void *query_output,
                               void *pages, std::size_t pages_bytes, const std::int32_t *page_table,
                               const std::uint32_t *query_starts, const std::uint32_t *context_lengths,
                               const double *frequencies, const void *query_weight, const void *key_weight,
                               Qwen35PagedShape shape, Qwen35PagedRotary rotary,
                               RaftInferDataType activation_dtype, RaftInferDataType weight_dtype,
                               Qwen35KvCacheLayout cache_layout, hipStream_t stream);

// output = sigmoid(gate) * softmax(query k / 16) v over the keys that each row's token
// sees, which the pages hold; gate null: without the sigmoid.  query, gate, output: bf16
// [rows][query_heads][256].  Before the division by the softmax's sum the values are
// summed in f32 with probabilities of at most 1: finite where |probability * value|
// over a token's keys sums to less than 2^128.  (The sums are held scaled down by up to
// 2^16, so products below 2^-110 lose bits.)
// Probabilities enter the product with the values in bf16, 8 bits, and are divided by the
// sum of what they were rounded to: besides its own rounding an output is off by up to
// 2^-8 of the probabilities' mean of |value - output|.
void qwen35_paged_attention_prefill(const void *query, const void *gate, void *output, const void *pages,
                                    std::size_t pages_bytes, const std::int32_t *page_table,
                                    const std::uint32_t *query_starts, const std::uint32_t *context_lengths,
                                    void *workspace, std::size_t workspace_bytes, Qwen35PagedShape shape,
                                    Qwen35PagedStrides strides, RaftInferDataType activation_dtype,
                                    Qwen35KvCacheLayout cache_layout, hipStream_t stream);

// The same with one new token of each sequence: row s belongs to sequence s, rows equals
// sequences.  A context length of 0 marks an unused row, which is left as it was.
// Probabilities are held in two bf16 parts, off by 2^-15 + 2^-17 of themselves at most, so
// that a token's output can differ from the other call's by that call's rounding of them.
void qwen35_paged_attention_decode(const void *query, const void *gate, void *output, const void *pages,
                                   std::size_t pages_bytes, const std::int32_t *page_table,
                                   const std::uint32_t *context_lengths, void *workspace,
                                   std::size_t workspace_bytes, Qwen35PagedShape shape,
                                   Qwen35PagedStrides strides, RaftInferDataType activation_dtype,
                                   Qwen35KvCacheLayout cache_layout, hipStream_t stream);

} // namespace raftinfer::kernels
