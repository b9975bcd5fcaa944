"""Host-side mirror of the reference kernel interface for the attention /
gated-delta hot path, over torch device tensors.

Names, argument meaning and error behaviour follow the reference's
cpp/kernels/qwen35_attention.cuh, qwen35_online_attention.cuh and
qwen35_delta.cuh: validation failures raise Qwen35PrimitiveError (attention)
or Qwen35DeltaError (delta) before anything is enqueued.  Every call goes
through libraftinfer_amd.so; nothing here computes on the CPU.  Tensors are
caller-owned device buffers; byte sizes passed to the library are the tensors'
own sizes.  ``stream`` is a torch.cuda.Stream (or raw hipStream_t int); the
default is the current stream, which must not be the null stream.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _lib
from ._lib import (AttentionPolicy, AttentionShape, BatchedDecodeShape, CompactShape, DecodeLayout,
                   DecodePlan, DeltaCoreShape, DeltaPolicy, DeltaShape, EvictShape, PagedRotary,
                   PagedShape, PagedStrides, RaftInferError, RotaryShape)

# cpp/execution/qwen35_execution_policy.hpp:7-27 and cpp/include/raftinfer/tensor.h:10-15
MATERIALIZED, ONLINE_TILED = 0, 1
AUTO, SINGLE_BLOCK, SPLIT_K_256, SPLIT_K_512 = 0, 1, 2, 3
CACHE_F32, CACHE_BF16 = 0, 1
TOKEN_MAJOR, HEAD_MAJOR = 0, 1
DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 1, 2, 3
SCHEDULE_CURRENT, SCHEDULE_PREFILL_CANDIDATE, SCHEDULE_DECODE_CANDIDATE = 0, 1, 2


class Qwen35PrimitiveError(RaftInferError):
    """Attention validation / launch failure (cpp/kernels/qwen35_primitives.cuh:15-19)."""


class Qwen35DeltaError(RaftInferError):
    """Gated-delta validation / launch failure (cpp/kernels/qwen35_delta.cuh:14-18)."""


def _call(err_type, status: int) -> None:
    try:
        _lib.check(status)
    except RaftInferError as e:
        raise err_type(e.status, str(e)) from None


@dataclass(frozen=True)
class Qwen35AttentionShape:
    tokens: int
    query_heads: int
    kv_heads: int
    head_dim: int
    max_context_tokens: int
    past_tokens: int

    def c(self) -> AttentionShape:
        return AttentionShape(self.tokens, self.query_heads, self.kv_heads, self.head_dim,
                              self.max_context_tokens, self.past_tokens)


@dataclass(frozen=True)
class Qwen35AttentionLaunchPolicy:
    implementation: int = ONLINE_TILED
    kv_cache_dtype: int = CACHE_BF16
    kv_cache_layout: int = HEAD_MAJOR

    def c(self) -> AttentionPolicy:
        return AttentionPolicy(self.implementation, self.kv_cache_dtype, self.kv_cache_layout)


@dataclass(frozen=True)
class GatedDeltaShape:
    tokens: int
    hidden_size: int
    key_heads: int
    value_heads: int
    key_dim: int
    value_dim: int
    conv_width: int
    epsilon: float

    def c(self) -> DeltaShape:
        return DeltaShape(self.tokens, self.hidden_size, self.key_heads, self.value_heads,
                          self.key_dim, self.value_dim, self.conv_width, self.epsilon)


@dataclass(frozen=True)
class GatedDeltaLaunchPolicy:
    schedule: int = SCHEDULE_CURRENT
    warps_per_block: int = 4
    transposed_boundary_state: bool = False

    def c(self) -> DeltaPolicy:
        return DeltaPolicy(self.schedule, self.warps_per_block, int(self.transposed_boundary_state))


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _fptr(t):
    return None if t is None else ctypes.cast(t.data_ptr(), ctypes.POINTER(ctypes.c_float))


def _nbytes(t) -> int:
    if t is None:
        return 0
    try:
        return t.nbytes
    except AttributeError:  # not a tensor
        return t.numel() * t.element_size()


def _stream(stream) -> ctypes.c_void_p:
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    handle = stream if isinstance(stream, int) else stream.cuda_stream
    return ctypes.c_void_p(handle)


_DTYPE_CODES: dict = {}


def _dtype_code(t) -> int:
    if not _DTYPE_CODES:
        import torch
        _DTYPE_CODES.update({torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16})
    return _DTYPE_CODES.get(t.dtype, 0)


# ------------------------------------------------------------- sizing API

def qwen35_attention_workspace_floats(shape: Qwen35AttentionShape) -> int:
    out = ctypes.c_size_t()
    _call(Qwen35PrimitiveError,
          _lib.load().raftinfer_amd_attention_workspace_floats(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_attention_cache_bytes(shape, policy: Qwen35AttentionLaunchPolicy) -> int:
    out = ctypes.c_size_t()
    _call(Qwen35PrimitiveError,
          _lib.load().raftinfer_amd_attention_cache_bytes(shape.c(), policy.c(), ctypes.byref(out)))
    return out.value


def qwen35_attention_workspace_bytes(shape, policy: Qwen35AttentionLaunchPolicy) -> int:
    out = ctypes.c_size_t()
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_attention_workspace_bytes(
        shape.c(), policy.c(), ctypes.byref(out)))
    return out.value


def qwen35_online_decode_plan(shape, requested: int, context_tokens: int) -> tuple:
    """(resolved_mode, partition_tokens, split_k_threshold_tokens, context_bucket_tokens,
    active_partition_capacity) -- cpp/kernels/qwen35_online_attention.cu:1071-1109."""
    out = DecodePlan()
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_decode_plan(
        shape.c(), requested, context_tokens, ctypes.byref(out)))
    return out.as_tuple()


def qwen35_online_decode_workspace_layout(shape, resolved_mode: int) -> tuple:
    """(partial_count, max_offset, sum_offset, value_offset, bytes) -- :1111-1143."""
    out = DecodeLayout()
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_decode_workspace_layout(
        shape.c(), resolved_mode, ctypes.byref(out)))
    return out.as_tuple()


def qwen35_online_attention_prefill_supported(shape, activation_dtype: int,
                                              policy: Qwen35AttentionLaunchPolicy) -> bool:
    return bool(_lib.load().raftinfer_amd_online_attention_prefill_supported(
        shape.c(), activation_dtype, policy.c()))


def qwen35_gated_delta_workspace_bytes(shape: GatedDeltaShape) -> int:
    out = ctypes.c_size_t()
    _call(Qwen35DeltaError,
          _lib.load().raftinfer_amd_gated_delta_workspace_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_gated_delta_core_workspace_bytes(tokens, key_heads, value_heads, key_dim,
                                            value_dim) -> int:
    out = ctypes.c_size_t()
    _call(Qwen35DeltaError, _lib.load().raftinfer_amd_gated_delta_core_workspace_bytes(
        DeltaCoreShape(tokens, key_heads, value_heads, key_dim, value_dim), ctypes.byref(out)))
    return out.value


def qwen35_batched_decode_workspace_bytes(sequences, max_context_tokens, cache_stride_bytes,
                                          single_block_max_tokens=512) -> int:
    out = ctypes.c_size_t()
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_batched_decode_workspace_bytes(
        BatchedDecodeShape(sequences, max_context_tokens, cache_stride_bytes,
                           single_block_max_tokens), ctypes.byref(out)))
    return out.value


# ------------------------------------------------------------ enqueue API

def qwen35_causal_attention(query, key, value, gate, output, kv_cache, workspace, shape,
                            activation_dtype: int, policy: Qwen35AttentionLaunchPolicy,
                            stream=None, kv_cache_bytes=None, workspace_bytes=None) -> None:
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_causal_attention(
        _ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output), _ptr(kv_cache),
        _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes, _ptr(workspace),
        _nbytes(workspace) if workspace_bytes is None else workspace_bytes, shape.c(),
        activation_dtype, policy.c(), _stream(stream)))


def qwen35_online_attention_prefill(query, key, value, gate, output, kv_cache, shape,
                                    activation_dtype, cache_dtype, cache_layout, stream=None,
                                    kv_cache_bytes=None) -> None:
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_attention_prefill(
        _ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output), _ptr(kv_cache),
        _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes, shape.c(),
        activation_dtype, cache_dtype, cache_layout, _stream(stream)))


def qwen35_online_attention_decode(query, key, value, gate, output, kv_cache, workspace, shape,
                                   activation_dtype, cache_dtype, cache_layout, plan=None,
                                   device_position=None, stream=None, kv_cache_bytes=None,
                                   workspace_bytes=None) -> None:
    """plan=None selects the plan-less single-block overload
    (cpp/kernels/qwen35_online_attention.cu:1316-1328)."""
    lib = _lib.load()
    pos = None if device_position is None else ctypes.cast(device_position.data_ptr(),
                                                           ctypes.POINTER(ctypes.c_uint32))
    cache_bytes = _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes
    if plan is None:
        _call(Qwen35PrimitiveError, lib.raftinfer_amd_online_attention_decode_single(
            _ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output), _ptr(kv_cache),
            cache_bytes, shape.c(), activation_dtype, cache_dtype, cache_layout, pos,
            _stream(stream)))
        return
    _call(Qwen35PrimitiveError, lib.raftinfer_amd_online_attention_decode(
        _ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output), _ptr(kv_cache), cache_bytes,
        _ptr(workspace), _nbytes(workspace) if workspace_bytes is None else workspace_bytes,
        shape.c(), activation_dtype, cache_dtype, cache_layout, DecodePlan(*plan), pos,
        _stream(stream)))


@dataclass
class Qwen35FusedNormRope:
    """The producer parameters of the fused attention entry points."""
    query_norm_weight: object  # device tensor [head_dim]
    key_norm_weight: object
    rotary_dim: int
    rope_base: float
    epsilon: float

    def c(self):
        wd = _dtype_code(self.query_norm_weight)
        return _lib.FusedNormRope(_ptr(self.query_norm_weight), _ptr(self.key_norm_weight), wd,
                                  self.rotary_dim, self.rope_base, self.epsilon)


def qwen35_online_attention_decode_fused(query_gate, key, value, output, kv_cache, workspace, shape,
                                         norm: Qwen35FusedNormRope, cache_dtype, cache_layout, plan,
                                         device_position=None, stream=None) -> None:
    """The q split + RMSNorm + RoPE of q and k fused into the decode attention."""
    pos = None if device_position is None else ctypes.cast(device_position.data_ptr(),
                                                           ctypes.POINTER(ctypes.c_uint32))
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_attention_decode_fused(
        _ptr(query_gate), _ptr(key), _ptr(value), _ptr(output), _ptr(kv_cache), _nbytes(kv_cache),
        _ptr(workspace), _nbytes(workspace), shape.c(), norm.c(), cache_dtype, cache_layout,
        DecodePlan(*plan), pos, _stream(stream)))


def qwen35_online_attention_prefill_fused(query_gate, key, value, output, kv_cache, shape,
                                          norm: Qwen35FusedNormRope, cache_dtype=CACHE_BF16,
                                          cache_layout=HEAD_MAJOR, stream=None) -> None:
    """The q split + RMSNorm + RoPE of q and k fused into the causal gated prefill."""
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_attention_prefill_fused(
        _ptr(query_gate), _ptr(key), _ptr(value), _ptr(output), _ptr(kv_cache), _nbytes(kv_cache),
        shape.c(), norm.c(), cache_dtype, cache_layout, _stream(stream)))


def qwen35_online_attention_static_workspace_bytes() -> int:
    return int(_lib.load().raftinfer_amd_online_attention_static_workspace_bytes())


def qwen35_online_attention_decode_static_workspace(query, key, value, gate, output, kv_cache, shape,
                                                    activation_dtype, cache_dtype, cache_layout,
                                                    plan, device_position=None, stream=None) -> None:
    """The allocation-free decode: as qwen35_online_attention_decode with a
    plan, with the split-K workspace in the library's static device array."""
    pos = None if device_position is None else ctypes.cast(device_position.data_ptr(),
                                                           ctypes.POINTER(ctypes.c_uint32))
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_attention_decode_static_workspace(
        _ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output), _ptr(kv_cache),
        _nbytes(kv_cache), shape.c(), activation_dtype, cache_dtype, cache_layout, DecodePlan(*plan),
        pos, _stream(stream)))


def qwen35_online_attention_decode_batched(query, key, value, gate, output, kv_cache,
                                           context_lengths, workspace, max_context_tokens,
                                           cache_stride_bytes, single_block_max_tokens=512,
                                           activation_dtype=DTYPE_BF16, stream=None) -> None:
    shape = BatchedDecodeShape(query.shape[0], max_context_tokens, cache_stride_bytes,
                               single_block_max_tokens)
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_online_attention_decode_batched(
        _ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output), _ptr(kv_cache),
        _nbytes(kv_cache), ctypes.cast(context_lengths.data_ptr(), ctypes.POINTER(ctypes.c_uint32)),
        _ptr(workspace), _nbytes(workspace), shape, activation_dtype, _stream(stream)))


class Qwen35DecodeAttentionGraphs:
    """Per-context-bucket captured decode steps (include/raftinfer_amd/hip_graph_decode.hpp),
    the variant table of cpp/execution/qwen35_executor.cu:2191-2226 on hipGraph.  The
    tensors must outlive the object; ``device_position`` (int32/uint32, 1 element) is read
    by the kernels at replay time."""

    def __init__(self, shape, mode, activation_dtype, cache_dtype, cache_layout, query, key, value,
                 gate, output, kv_cache, workspace, device_position, stream=None, device_id=0):
        self._lib = _lib.load()
        self._keep = (query, key, value, gate, output, kv_cache, workspace, device_position)
        pos = ctypes.cast(device_position.data_ptr(), ctypes.POINTER(ctypes.c_uint32))
        buf = _lib.DecodeBuffers(_ptr(query), _ptr(key), _ptr(value), _ptr(gate), _ptr(output),
                                 _ptr(kv_cache), _nbytes(kv_cache), _ptr(workspace),
                                 _nbytes(workspace), pos)
        handle = ctypes.c_void_p()
        _call(Qwen35PrimitiveError, self._lib.raftinfer_amd_decode_graphs_create(
            device_id, _stream(stream), shape.c(), mode, activation_dtype, cache_dtype, cache_layout,
            buf, ctypes.byref(handle)))
        self._handle = handle

    def variant_count(self) -> int:
        out = ctypes.c_size_t()
        _call(Qwen35PrimitiveError, self._lib.raftinfer_amd_decode_graphs_variant_count(
            self._handle, ctypes.byref(out)))
        return out.value

    def variant_for(self, position: int) -> int:
        out = ctypes.c_size_t()
        _call(Qwen35PrimitiveError, self._lib.raftinfer_amd_decode_graphs_variant_for(
            self._handle, position, ctypes.byref(out)))
        return out.value

    def replay(self, position: int) -> None:
        _call(Qwen35PrimitiveError, self._lib.raftinfer_amd_decode_graphs_replay(self._handle, position))

    def close(self) -> None:
        if self._handle:
            self._lib.raftinfer_amd_decode_graphs_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def consume_capacity_errors() -> int:
    out = ctypes.c_uint32()
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_consume_capacity_errors(ctypes.byref(out)))
    return out.value


# ------------------------------------------------------ compact KV cache
# include/raftinfer_amd/qwen35_compact_cache.hpp
CACHE_FP8_E4M3 = 2  # compact caches only (or CACHE_BF16)


@dataclass(frozen=True)
class Qwen35CompactShape:
    tokens: int
    sequences: int
    query_heads: int
    kv_heads: int
    head_dim: int
    max_context_tokens: int
    past_tokens: int
    cache_stride_bytes: int = 0
    window_tokens: int = 0
    sink_tokens: int = 0
    observed_tokens: int = 0

    def c(self) -> CompactShape:
        return CompactShape(self.tokens, self.sequences, self.query_heads, self.kv_heads, self.head_dim,
                            self.max_context_tokens, self.past_tokens, self.cache_stride_bytes,
                            self.window_tokens, self.sink_tokens, self.observed_tokens)


@dataclass(frozen=True)
class Qwen35EvictShape:
    kv_heads: int
    head_dim: int
    context_tokens: int
    max_context_tokens: int
    keep_tokens: int
    out_max_context_tokens: int
    sink_tokens: int = 0
    recent_tokens: int = 0

    def c(self) -> EvictShape:
        return EvictShape(self.kv_heads, self.head_dim, self.context_tokens, self.max_context_tokens,
                          self.keep_tokens, self.out_max_context_tokens, self.sink_tokens,
                          self.recent_tokens)


def _raw(t):
    return None if t is None else t.data_ptr()


_raw_stream = None  # of a device, by its index (0.1 us; a Stream object takes 1.8 us to make)


def _stream_of(stream, tensor) -> int:
    """The stream's handle; None: the current stream of the tensor's device."""
    if stream is None:
        global _raw_stream
        if _raw_stream is None:
            import torch
            _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
        if tensor.is_cuda:
            return _raw_stream(tensor.get_device())
        import torch
        return torch.cuda.current_stream(tensor.device).cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


def _checked(status: int) -> None:
    if status != 0:
        _call(Qwen35PrimitiveError, status)


def qwen35_compact_cache_bytes(shape: Qwen35CompactShape, cache_dtype: int) -> int:
    """Bytes of one sequence's cache."""
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_compact_cache_bytes(shape.c(), cache_dtype, ctypes.byref(out)))
    return out.value


def qwen35_compact_decode_workspace_bytes(shape: Qwen35CompactShape) -> int:
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_compact_decode_workspace_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_compact_prefill_workspace_bytes(shape: Qwen35CompactShape) -> int:
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_compact_prefill_workspace_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_compact_evict_workspace_bytes(shape: Qwen35EvictShape) -> int:
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_compact_evict_workspace_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_compact_cache_append(key, value, kv_cache, shape: Qwen35CompactShape, activation_dtype: int,
                                cache_dtype: int, cache_layout: int, context_lengths=None, stream=None,
                                kv_cache_bytes=None) -> None:
    """Stores shape.tokens rows of every sequence (8-bit caches: codes and scales)."""
    _checked(_lib.load().raftinfer_amd_compact_cache_append(
        _raw(key), _raw(value), _raw(kv_cache),
        _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes, _raw(context_lengths),
        shape.c(), activation_dtype, cache_dtype, cache_layout, _stream_of(stream, key)))


def qwen35_compact_attention_prefill(query, key, value, gate, output, kv_cache,
                                     shape: Qwen35CompactShape, activation_dtype: int,
                                     cache_dtype: int, cache_layout: int, workspace=None,
                                     key_weights=None, stream=None, kv_cache_bytes=None,
                                     workspace_bytes=None) -> None:
    """Stores the prompt's rows and attends over the cache, within the shape's window."""
    _checked(_lib.load().raftinfer_amd_compact_attention_prefill(
        _raw(query), _raw(key), _raw(value), _raw(gate), _raw(output), _raw(kv_cache),
        _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes, _raw(key_weights),
        _raw(workspace), _nbytes(workspace) if workspace_bytes is None else workspace_bytes, shape.c(),
        activation_dtype, cache_dtype, cache_layout, _stream_of(stream, query)))


def qwen35_compact_attention_decode(query, key, value, gate, output, kv_cache,
                                    shape: Qwen35CompactShape, activation_dtype: int, cache_dtype: int,
                                    cache_layout: int, workspace, context_lengths=None,
                                    key_weights=None, stream=None, kv_cache_bytes=None,
                                    workspace_bytes=None) -> None:
    """One new token of each sequence; context_lengths (int32/uint32, on the device) include it."""
    _checked(_lib.load().raftinfer_amd_compact_attention_decode(
        _raw(query), _raw(key), _raw(value), _raw(gate), _raw(output), _raw(kv_cache),
        _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes, _raw(context_lengths),
        _raw(key_weights), _raw(workspace),
        _nbytes(workspace) if workspace_bytes is None else workspace_bytes, shape.c(),
        activation_dtype, cache_dtype, cache_layout, _stream_of(stream, query)))


def qwen35_compact_cache_evict(kv_cache, key_weights, out_cache, out_weights, kept_indices,
                               shape: Qwen35EvictShape, cache_dtype: int, out_cache_dtype: int,
                               cache_layout: int, workspace=None, stream=None, kv_cache_bytes=None,
                               out_cache_bytes=None, workspace_bytes=None) -> None:
    """The sinks, the recent entries and those with the largest weights, to out_cache."""
    _checked(_lib.load().raftinfer_amd_compact_cache_evict(
        _raw(kv_cache), _nbytes(kv_cache) if kv_cache_bytes is None else kv_cache_bytes,
        _raw(key_weights), _raw(out_cache),
        _nbytes(out_cache) if out_cache_bytes is None else out_cache_bytes, _raw(out_weights),
        _raw(kept_indices), _raw(workspace),
        _nbytes(workspace) if workspace_bytes is None else workspace_bytes, shape.c(), cache_dtype,
        out_cache_dtype, cache_layout, _stream_of(stream, kv_cache)))


# ------------------------------------------- rotary positions, paged KV cache
# include/raftinfer_amd/qwen35_paged_cache.hpp.  Tensors [rows, heads, dim] may have any strides
# that the header allows; they are read off the tensors.
SCALING_NONE, SCALING_LINEAR, SCALING_BY_PAIR, SCALING_BY_TURNS = 0, 1, 2, 3


@dataclass(frozen=True)
class Qwen35RotaryShape:
    rows: int
    heads: int
    head_dim: int
    rotary_dim: int
    interleaved: bool = False
    magnitude: float = 1.0

    # (all fields at once: set one by one, as a frozen dataclass does, a call's shape takes twice as long to make)
    def __init__(self, rows, heads, head_dim, rotary_dim, interleaved=False, magnitude=1.0):
        self.__dict__.update(rows=rows, heads=heads, head_dim=head_dim, rotary_dim=rotary_dim,
                             interleaved=interleaved, magnitude=magnitude)


@dataclass(frozen=True)
class Qwen35PagedShape:
    rows: int
    sequences: int
    query_heads: int
    kv_heads: int
    head_dim: int
    pages: int
    page_tokens: int
    table_pages: int
    max_context_tokens: int
    window_tokens: int = 0

    def __init__(self, rows, sequences, query_heads, kv_heads, head_dim, pages, page_tokens, table_pages,
                 max_context_tokens, window_tokens=0):
        self.__dict__.update(rows=rows, sequences=sequences, query_heads=query_heads, kv_heads=kv_heads,
                             head_dim=head_dim, pages=pages, page_tokens=page_tokens, table_pages=table_pages,
                             max_context_tokens=max_context_tokens, window_tokens=window_tokens)

    def c(self) -> PagedShape:
        return PagedShape(*self.__dict__.values())


@dataclass(frozen=True)
class Qwen35PagedRotary:
    rotary_dim: int
    interleaved: bool = False
    magnitude: float = 1.0
    epsilon: float = 1e-6

    def __init__(self, rotary_dim, interleaved=False, magnitude=1.0, epsilon=1e-6):
        self.__dict__.update(rotary_dim=rotary_dim, interleaved=interleaved, magnitude=magnitude, epsilon=epsilon)


_TYPES = None


def _types():
    """(types of indices, of frequencies, of pages, of activations by their code, of weights)."""
    global _TYPES
    if _TYPES is None:
        import torch
        _TYPES = ((torch.int32, torch.uint32), (torch.float64,), (torch.bfloat16, torch.uint8, torch.int8),
                  {DTYPE_F32: torch.float32, DTYPE_F16: torch.float16, DTYPE_BF16: torch.bfloat16},
                  (torch.float32, torch.float16, torch.bfloat16))
    return _TYPES


def _strides(t) -> tuple:
    """(row, head) strides of a tensor [rows, heads, dim] whose dims are neighbours; anything else must be dense."""
    try:
        row, head, dim = t.stride()
    except (AttributeError, ValueError):  # not three dimensions
        _dense(t)
        return 0, 0
    rows, heads, dims = t.shape
    if dim != 1 and dims != 1:
        raise Qwen35PrimitiveError(1, "the last dimension of a tensor of heads must be contiguous")
    if (row == 0 and rows > 1) or (head == 0 and heads > 1):
        raise Qwen35PrimitiveError(1, "rows and heads must not be broadcast")
    # (the stride of a dimension of one element says nothing)
    return (row if rows > 1 else 0), (head if heads > 1 else 0)


def _dense(t):
    """The address of an argument without strides of its own."""
    if t is None:
        return None
    try:
        if not t.is_contiguous():
            raise Qwen35PrimitiveError(1, "indices, pages, weights and workspaces must be contiguous")
    except AttributeError:  # not a tensor: it has an address only
        pass
    return t.data_ptr()


def _heads(t, dtype, size) -> tuple:
    """(address, row stride, head stride) of an activation of `size` [rows, heads, dim]; strides of 0: dense."""
    if t is None:
        return None, 0, 0
    try:
        if t.dtype is not dtype:
            raise Qwen35PrimitiveError(1, f"activations must be of one type, {dtype}: got {t.dtype}")
        if t.shape != size:
            return _other_heads(t, size)
        row, head, one = t.stride()
        if one == 1 and row > 0 and head > 0:
            return t.data_ptr(), (row if size[0] > 1 else 0), (head if size[1] > 1 else 0)
    except (AttributeError, ValueError):  # an address, with strides or without; not three dimensions
        pass
    return (t.data_ptr(), *_strides(t))


def _other_heads(t, size) -> tuple:
    """The same of a tensor of another size: part of a larger one, or the same values without gaps in other dimensions."""
    strides = _strides(t)
    rows, heads, dim = size
    shape = tuple(t.shape)
    if len(shape) == 3 and shape[0] >= rows and shape[1] >= heads and shape[2] >= dim:
        return (t.data_ptr(), *strides)
    if not t.is_contiguous() or t.numel() < rows * heads * dim or shape == (heads, rows, dim):
        raise Qwen35PrimitiveError(1, f"an activation must be [{rows}, {heads}, {dim}]: got {list(shape)}")
    return t.data_ptr(), 0, 0


def _listed(t, dtypes, least, what):
    """The address of an argument of at least `least` elements of one of the types that follow each other."""
    if t is None:
        return None
    try:
        if t.dtype in dtypes and t.numel() >= least and t.is_contiguous():
            return t.data_ptr()
        if not t.is_contiguous():
            raise Qwen35PrimitiveError(1, "indices, pages, weights and workspaces must be contiguous")
        if t.dtype not in dtypes:
            raise Qwen35PrimitiveError(1, f"{what} must be of type {' or '.join(map(str, dtypes))}: got {t.dtype}")
        raise Qwen35PrimitiveError(1, f"{what} must have {least} elements: got {t.numel()}")
    except AttributeError:  # not a tensor: it has an address only
        pass
    return t.data_ptr()


def _table(t, dtypes, shape) -> tuple:
    """(address of a page table [sequences, table_pages], the call's shape).  The shape's max_context_tokens may be
    above the positions of a table that is a tensor; of a bare address nothing but the shape tells the size."""
    try:
        if t.dtype in dtypes and t.shape == (shape.sequences, shape.table_pages) and t.is_contiguous():
            return t.data_ptr(), shape.c()
        at = _listed(t, dtypes, shape.sequences * shape.table_pages, "page_table")
        if shape.sequences > 1 and len(t.shape) == 2 and t.shape[1] != shape.table_pages:
            raise Qwen35PrimitiveError(1, f"page_table must have rows of {shape.table_pages} entries: got {t.shape[1]}")
        return at, shape.c()
    except AttributeError:  # a bare address, or none
        _within_table(shape)
        return (None if t is None else t.data_ptr()), shape.c()


def qwen35_rotary_frequencies(rotary_dim: int, base: float, scaling: int = SCALING_NONE,
                              factor: float = 1.0, trained_tokens: float = 0.0,
                              fast_turns: float | None = None, slow_turns: float = 1.0) -> tuple:
    """(the rotary_dim / 2 angles per position, their magnitude), on the host.  fast_turns None: 32 by pair, 4 by
    turns, as models with these scalings have them."""
    if fast_turns is None:
        fast_turns = 4.0 if scaling == SCALING_BY_TURNS else 32.0
    out = (ctypes.c_double * max(1, rotary_dim // 2))()
    magnitude = ctypes.c_float()
    _checked(_lib.load().raftinfer_amd_rotary_frequencies(
        out, rotary_dim, base, scaling, factor, trained_tokens, fast_turns, slow_turns,
        ctypes.byref(magnitude)))
    return list(out), magnitude.value


def qwen35_rotary(input, weight, output, positions, frequencies, shape: Qwen35RotaryShape,
                  epsilon: float, stream=None) -> None:
    """RoPE(input / rms(input) * weight) of every head by the rows' positions (int32/uint32); weight
    None: no norm.  frequencies: float64 [rotary_dim / 2].  output may be input."""
    index, wide, _, _, floats = _TYPES or _types()
    rows, heads, dim, kind = shape.rows, shape.heads, shape.head_dim, input.dtype
    dtype = _dtype_code(input)
    src, in_row, in_head = _heads(input, kind, (rows, heads, dim))
    dst, out_row, out_head = _heads(output, kind, (rows, heads, dim))
    _checked((_lib._lib or _lib.load()).raftinfer_amd_rotary(
        src, _listed(weight, floats, dim, "weight"), dst, _listed(positions, index, rows, "positions"),
        _listed(frequencies, wide, shape.rotary_dim // 2, "frequencies"),
        RotaryShape(rows, heads, dim, shape.rotary_dim, shape.interleaved, shape.magnitude, in_row, in_head, out_row, out_head),
        epsilon, dtype, dtype if weight is None or weight.dtype is kind else _dtype_code(weight), _stream_of(stream, input)))


def _within_table(shape: Qwen35PagedShape) -> None:
    """Where no page table is at hand whose size the call could go by, the shape's own numbers have to agree."""
    positions = shape.table_pages * shape.page_tokens
    if 0 < positions < shape.max_context_tokens:
        raise Qwen35PrimitiveError(1, "paged cache max_context_tokens must be within the page table")


def qwen35_paged_cache_bytes(shape: Qwen35PagedShape) -> int:
    _within_table(shape)
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_paged_cache_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_paged_decode_workspace_bytes(shape: Qwen35PagedShape) -> int:
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_paged_decode_workspace_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_paged_prefill_workspace_bytes(shape: Qwen35PagedShape) -> int:
    out = ctypes.c_size_t()
    _checked(_lib.load().raftinfer_amd_paged_prefill_workspace_bytes(shape.c(), ctypes.byref(out)))
    return out.value


def qwen35_paged_cache_append(query, key, value, query_output, pages, page_table, query_starts,
                              context_lengths, frequencies, query_weight, key_weight,
                              shape: Qwen35PagedShape, rotary: Qwen35PagedRotary, cache_layout: int,
                              activation_dtype: int = DTYPE_BF16, weight_dtype=None, stream=None,
                              pages_bytes=None) -> None:
    """The batch's queries normalised and turned to query_output, its keys (likewise) and values to
    their positions in the pages."""
    if weight_dtype is None:
        weight = query_weight if query_weight is not None else key_weight
        weight_dtype = DTYPE_BF16 if weight is None else _dtype_code(weight)
        if key_weight is not None and key_weight is not weight and key_weight.dtype is not weight.dtype:
            raise Qwen35PrimitiveError(1, "query_weight and key_weight must be of one type")
    index, wide, raw, kinds, _ = _TYPES or _types()
    act, dim = kinds.get(activation_dtype), shape.head_dim
    heads, kv_heads = (shape.rows, shape.query_heads, dim), (shape.rows, shape.kv_heads, dim)
    weights = (kinds.get(weight_dtype),)
    q, q_row, q_head = _heads(query, act, heads)
    k, k_row, k_head = _heads(key, act, kv_heads)
    v, v_row, v_head = _heads(value, act, kv_heads)
    out, out_row, out_head = _heads(query_output, act, heads)
    table, call = _table(page_table, index, shape)
    _checked((_lib._lib or _lib.load()).raftinfer_amd_paged_cache_append(
        q, k, v, out, _listed(pages, raw, 0, "pages"),
        _nbytes(pages) if pages_bytes is None else pages_bytes, table,
        _listed(query_starts, index, shape.sequences + 1, "query_starts"),
        _listed(context_lengths, index, shape.sequences, "context_lengths"),
        _listed(frequencies, wide, rotary.rotary_dim // 2, "frequencies"),
        _listed(query_weight, weights, dim, "query_weight"), _listed(key_weight, weights, dim, "key_weight"),
        call,
        PagedRotary(rotary.rotary_dim, rotary.interleaved, rotary.magnitude, rotary.epsilon,
                    q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head),
        activation_dtype, weight_dtype, cache_layout, _stream_of(stream, key)))


def qwen35_paged_attention_prefill(query, gate, output, pages, page_table, query_starts,
                                   context_lengths, workspace, shape: Qwen35PagedShape,
                                   cache_layout: int, activation_dtype: int = DTYPE_BF16, stream=None,
                                   pages_bytes=None, workspace_bytes=None) -> None:
    """Attention of every sequence's new tokens over its pages; gate None: no gate."""
    index, _, raw, kinds, _ = _TYPES or _types()
    act, heads = kinds.get(activation_dtype), (shape.rows, shape.query_heads, shape.head_dim)
    q, q_row, q_head = _heads(query, act, heads)
    g, g_row, g_head = _heads(gate, act, heads)
    out, out_row, out_head = _heads(output, act, heads)
    table, call = _table(page_table, index, shape)
    _checked((_lib._lib or _lib.load()).raftinfer_amd_paged_attention_prefill(
        q, g, out, _listed(pages, raw, 0, "pages"),
        _nbytes(pages) if pages_bytes is None else pages_bytes, table,
        _listed(query_starts, index, shape.sequences + 1, "query_starts"),
        _listed(context_lengths, index, shape.sequences, "context_lengths"), _dense(workspace),
        _nbytes(workspace) if workspace_bytes is None else workspace_bytes, call,
        PagedStrides(q_row, q_head, g_row, g_head, out_row, out_head), activation_dtype, cache_layout, _stream_of(stream, query)))


def qwen35_paged_attention_decode(query, gate, output, pages, page_table, context_lengths, workspace,
                                  shape: Qwen35PagedShape, cache_layout: int,
                                  activation_dtype: int = DTYPE_BF16, stream=None, pages_bytes=None,
                                  workspace_bytes=None) -> None:
    """The same for one new token of every sequence; a context length of 0: an unused row."""
    index, _, raw, kinds, _ = _TYPES or _types()
    act, heads = kinds.get(activation_dtype), (shape.rows, shape.query_heads, shape.head_dim)
    q, q_row, q_head = _heads(query, act, heads)
    g, g_row, g_head = _heads(gate, act, heads)
    out, out_row, out_head = _heads(output, act, heads)
    table, call = _table(page_table, index, shape)
    _checked((_lib._lib or _lib.load()).raftinfer_amd_paged_attention_decode(
        q, g, out, _listed(pages, raw, 0, "pages"),
        _nbytes(pages) if pages_bytes is None else pages_bytes, table,
        _listed(context_lengths, index, shape.sequences, "context_lengths"), _dense(workspace),
        _nbytes(workspace) if workspace_bytes is None else workspace_bytes, call,
        PagedStrides(q_row, q_head, g_row, g_head, out_row, out_head), activation_dtype, cache_layout, _stream_of(stream, query)))


def qwen35_gated_delta(input, conv_weight, recurrent_a, dt_bias, output_norm_weight, output,
                       convolution_state, recurrent_state, workspace, shape: GatedDeltaShape,
                       dtype: int, weight_dtype: int, policy: GatedDeltaLaunchPolicy | None = None,
                       stream=None, workspace_bytes=None) -> None:
    lib = _lib.load()
    ws_bytes = _nbytes(workspace) if workspace_bytes is None else workspace_bytes
    common = (_ptr(input), _ptr(conv_weight), _ptr(recurrent_a), _ptr(dt_bias),
              _ptr(output_norm_weight), _ptr(output), _fptr(convolution_state),
              _fptr(recurrent_state), _ptr(workspace), ws_bytes, shape.c())
    if policy is None:
        _call(Qwen35DeltaError, lib.raftinfer_amd_gated_delta_auto(
            *common, dtype, weight_dtype, _stream(stream)))
    else:
        _call(Qwen35DeltaError, lib.raftinfer_amd_gated_delta(
            *common, policy.c(), dtype, weight_dtype, _stream(stream)))


def qwen35_gated_delta_unpacked(qkv, beta, alpha, gate, conv_weight, recurrent_a, dt_bias,
                                output_norm_weight, output, convolution_state, recurrent_state,
                                workspace, shape: GatedDeltaShape, dtype: int, weight_dtype: int,
                                policy: GatedDeltaLaunchPolicy | None = None, stream=None) -> None:
    """qwen35_pack_linear_delta_input + qwen35_gated_delta in one call, reading the four
    projection outputs in place (no packed copy)."""
    policy = policy or GatedDeltaLaunchPolicy()
    _call(Qwen35DeltaError, _lib.load().raftinfer_amd_gated_delta_unpacked(
        _ptr(qkv), _ptr(beta), _ptr(alpha), _ptr(gate), _ptr(conv_weight), _ptr(recurrent_a),
        _ptr(dt_bias), _ptr(output_norm_weight), _ptr(output), _fptr(convolution_state),
        _fptr(recurrent_state), _ptr(workspace), _nbytes(workspace), shape.c(), policy.c(), dtype,
        weight_dtype, _stream(stream)))


def qwen35_gated_delta_core(q, k, v, beta, log_decay, q_scale, state, output, workspace=None,
                            chunked=True, stream=None) -> None:
    T, hk, dk = q.shape
    hv, dv = v.shape[1], v.shape[2]
    _call(Qwen35DeltaError, _lib.load().raftinfer_amd_gated_delta_core(
        _ptr(q), _ptr(k), _ptr(v), _fptr(beta), _fptr(log_decay), ctypes.c_float(q_scale),
        _fptr(state), _ptr(output), _ptr(workspace), _nbytes(workspace),
        DeltaCoreShape(T, hk, hv, dk, dv), int(chunked), _stream(stream)))


# ------------------------------------------------------ attention producers
# cpp/kernels/qwen35_primitives.cuh:34-41, :63-67, :93-96.
@dataclass
class QkNormRopeShape:
    tokens: int
    heads: int
    head_dim: int
    rotary_dim: int
    position_offset: int
    rope_base: float

    def c(self):
        return _lib.QkNormRopeShape(self.tokens, self.heads, self.head_dim, self.rotary_dim,
                                    self.position_offset, self.rope_base)


def qwen35_qk_norm_rope(input, weight, output, shape: QkNormRopeShape, epsilon, dtype,
                        weight_dtype, stream=None, device_position=None) -> None:
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_qk_norm_rope(
        _ptr(input), _ptr(weight), _ptr(output), shape.c(), ctypes.c_float(epsilon), dtype,
        weight_dtype, _stream(stream), _ptr(device_position)))


def qwen35_split_full_query_gate(query_gate, query, gate, tokens, heads, head_dim, dtype,
                                 stream=None) -> None:
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_split_full_query_gate(
        _ptr(query_gate), _ptr(query), _ptr(gate), tokens, heads, head_dim, dtype,
        _stream(stream)))


def qwen35_split_query_gate_norm_rope(query_gate, weight, query, gate, shape: QkNormRopeShape,
                                      epsilon, dtype, weight_dtype, stream=None,
                                      device_position=None) -> None:
    """Additive: qwen35_split_full_query_gate then qwen35_qk_norm_rope on the query, fused."""
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_split_query_gate_norm_rope(
        _ptr(query_gate), _ptr(weight), _ptr(query), _ptr(gate), shape.c(),
        ctypes.c_float(epsilon), dtype, weight_dtype, _stream(stream), _ptr(device_position)))


def qwen35_pack_linear_delta_input(qkv, beta, alpha, gate, packed, tokens, qkv_width, beta_width,
                                   alpha_width, gate_width, dtype, stream=None) -> None:
    """cpp/kernels/qwen35_primitives.cuh:98-102."""
    _call(Qwen35PrimitiveError, _lib.load().raftinfer_amd_pack_linear_delta_input(
        _ptr(qkv), _ptr(beta), _ptr(alpha), _ptr(gate), _ptr(packed), tokens, qkv_width,
        beta_width, alpha_width, gate_width, dtype, _stream(stream)))
