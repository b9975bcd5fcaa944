"""CPU tests of the compact KV cache: sizes, refusals before any launch, and the 64-bit reference itself."""
import dataclasses

import numpy as np
import pytest
import torch

import compact_reference as ref
from raftinfer_amd import ops
from test_boundary import FakeTensor

S, E = ops.Qwen35CompactShape, ops.Qwen35EvictShape
BF16, FP8 = ops.CACHE_BF16, ops.CACHE_FP8_E4M3
MODEL = S(1, 1, 16, 4, 256, 4096, 100)
BIG = FakeTensor(nbytes=1 << 50)


def test_reference_codes_are_e4m3():
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), ref.E4M3, equal_nan=True)
    x = torch.cat([torch.randn(4000, generator=torch.Generator().manual_seed(1)).double() * 50,
                   torch.tensor(ref.E4M3[:126] + ref.E4M3[1:127]) / 2, torch.zeros(2), -torch.zeros(2)]).float()
    x = x[x.abs() <= 448]
    assert np.array_equal(x.to(torch.float8_e4m3fn).view(torch.uint8).numpy(), ref.to_codes(x.numpy()))


@pytest.mark.parametrize("amax,scale", [(0, 2.0 ** -126), (448, 1), (448.0001, 2), (1, 2.0 ** -8), (1.75, 2.0 ** -8),
                                        (1.76, 2.0 ** -7), (3.3e38, 2.0 ** 120), (2.0 ** -130, 2.0 ** -126)])
def test_reference_scale(amax, scale):
    assert ref.scale_for(amax) == scale


def test_sizes():
    assert ops.qwen35_compact_cache_bytes(MODEL, BF16) == 2 * 4096 * 4 * 256 * 2
    assert ops.qwen35_compact_cache_bytes(MODEL, FP8) == 2 * 4096 * 4 * 256 + 2 * 4 * 128 * 4
    # one position, three heads: 24 bytes of scales, rounded up to 32
    assert ops.qwen35_compact_cache_bytes(S(1, 1, 3, 3, 256, 1, 0), FP8) == 2 * 3 * 256 + 32
    a = ops.qwen35_compact_decode_workspace_bytes(MODEL)
    assert a > 0 and a == ops.qwen35_compact_decode_workspace_bytes(dataclasses.replace(MODEL, past_tokens=0))
    assert ops.qwen35_compact_decode_workspace_bytes(dataclasses.replace(MODEL, observed_tokens=1)) > a
    assert ops.qwen35_compact_evict_workspace_bytes(E(4, 256, 4096, 4096, 100, 100)) >= 0


@pytest.mark.parametrize("change,message", [
    ({"head_dim": 128}, "head_dim must be 256"), ({"kv_heads": 0}, "kv_heads"), ({"query_heads": 0}, "query_heads"),
    ({"query_heads": 6}, "query_heads"), ({"query_heads": 68}, "query_heads"), ({"tokens": 0}, "tokens must be positive"),
    ({"sequences": 0}, "sequences"), ({"sequences": 65536}, "sequences"), ({"max_context_tokens": 0}, "max_context_tokens"),
    ({"max_context_tokens": 2 ** 28 + 1}, "max_context_tokens"), ({"kv_heads": 4096, "query_heads": 4096, "max_context_tokens": 2 ** 20}, "max_context_tokens"),
    ({"kv_heads": 1024, "query_heads": 1024, "sequences": 129}, "too many sequences"), ({"past_tokens": 4096}, "exceeds cache capacity"),
    ({"past_tokens": 2 ** 64 - 1}, "exceeds cache capacity"), ({"observed_tokens": 2}, "observes more"),
    ({"tokens": 2}, "one token"), ({"observed_tokens": 1}, "key_weights go with")])
def test_decode_refuses_shapes(change, message):
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_compact_attention_decode(BIG, BIG, BIG, BIG, BIG, BIG, dataclasses.replace(MODEL, **change), ops.DTYPE_BF16,
                                            FP8, 1, BIG, stream=0x1234)


@pytest.mark.parametrize("change,message", [
    ({"sequences": 2}, "one sequence"), ({"tokens": 4000}, "exceeds cache capacity"), ({"tokens": 2 ** 40}, "too many query rows"),
    ({"observed_tokens": 11}, "observes more"), ({"observed_tokens": 4}, "key_weights go with")])
def test_prefill_refuses_shapes(change, message):
    shape = dataclasses.replace(MODEL, tokens=10, **{k: v for k, v in change.items()}) if "tokens" not in change else \
        dataclasses.replace(MODEL, **change)
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_compact_attention_prefill(BIG, BIG, BIG, BIG, BIG, BIG, shape, ops.DTYPE_BF16, FP8, 1, BIG, stream=0x1234)


@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_attention_refuses_pointers_and_types(call):
    fn = getattr(ops, f"qwen35_compact_attention_{call}")
    need = getattr(ops, f"qwen35_compact_{call}_workspace_bytes")(MODEL)

    def go(i=None, bad=None, shape=MODEL, act=ops.DTYPE_BF16, dtype=FP8, layout=1, ws=BIG, stream=0x1234, **kw):
        args = [BIG] * 6
        if i is not None:
            args[i] = bad
        fn(*args, shape, act, dtype, layout, ws, stream=stream, **kw)

    for i, name in enumerate(["query", "key", "value", "gate", "output", "cache"]):
        with pytest.raises(ops.Qwen35PrimitiveError, match=f"{name} pointer is null"):
            go(i, None, kv_cache_bytes=1 << 40)
        with pytest.raises(ops.Qwen35PrimitiveError, match="16-byte aligned"):
            go(i, FakeTensor(1 << 50, 0x100008))
    for kw, message in [({"act": ops.DTYPE_F32}, "must be bf16"), ({"act": ops.DTYPE_F16}, "must be bf16"),
                        ({"dtype": 0}, "unsupported compact cache dtype"), ({"dtype": 3}, "unsupported compact cache dtype"),
                        ({"layout": 2}, "unsupported compact cache layout"), ({"stream": 0}, "stream is null"),
                        ({"ws": FakeTensor(1 << 50, 0x100004)}, "workspace must be 16-byte aligned"),
                        ({"key_weights": BIG}, "key_weights go with"),
                        ({"kv_cache_bytes": ops.qwen35_compact_cache_bytes(MODEL, FP8) - 1}, "cache is too small"),
                        ({"dtype": BF16, "kv_cache_bytes": ops.qwen35_compact_cache_bytes(MODEL, BF16) - 1}, "cache is too small")]:
        with pytest.raises(ops.Qwen35PrimitiveError, match=message):
            go(**kw)
    if need:
        with pytest.raises(ops.Qwen35PrimitiveError, match="workspace is null"):
            go(ws=None)
        with pytest.raises(ops.Qwen35PrimitiveError, match="workspace is too small"):
            go(workspace_bytes=need - 1)
    weighed = dataclasses.replace(MODEL, observed_tokens=1)
    with pytest.raises(ops.Qwen35PrimitiveError, match="key_weights must be 4-byte aligned"):
        go(shape=weighed, key_weights=FakeTensor(1 << 50, 0x100002))


def test_batch_stride():
    one = ops.qwen35_compact_cache_bytes(MODEL, FP8)
    for stride, size, message in [(one - 16, 1 << 50, "stride"), (one + 8, 1 << 50, "stride"), (one, 3 * one - 1, "too small"),
                                  (2 ** 63, 1 << 50, "overflow")]:
        shape = dataclasses.replace(MODEL, sequences=3, cache_stride_bytes=stride)
        with pytest.raises(ops.Qwen35PrimitiveError, match=message):
            ops.qwen35_compact_attention_decode(BIG, BIG, BIG, BIG, BIG, BIG, shape, ops.DTYPE_BF16, FP8, 1, BIG,
                                                stream=0x1234, kv_cache_bytes=size)


def test_append_refusals():
    for kw, message in [({"shape": dataclasses.replace(MODEL, tokens=3997)}, "exceeds cache capacity"),
                        ({"shape": dataclasses.replace(MODEL, tokens=2), "context_lengths": BIG}, "one token per sequence"),
                        ({"act": ops.DTYPE_F32}, "must be bf16"), ({"layout": 9}, "layout"), ({"dtype": 0}, "dtype")]:
        with pytest.raises(ops.Qwen35PrimitiveError, match=message):
            ops.qwen35_compact_cache_append(BIG, BIG, BIG, kw.get("shape", MODEL), kw.get("act", ops.DTYPE_BF16),
                                            kw.get("dtype", FP8), kw.get("layout", 1),
                                            context_lengths=kw.get("context_lengths"), stream=0x1234)


@pytest.mark.parametrize("change,message", [
    ({"context_tokens": 0}, "context_tokens must be positive"), ({"context_tokens": 4097}, "exceeds cache capacity"),
    ({"keep_tokens": 0}, "keep_tokens"), ({"keep_tokens": 3001}, "keep_tokens"), ({"out_max_context_tokens": 999}, "more than the new cache"),
    ({"sink_tokens": 1001}, "fewer than the sinks"), ({"sink_tokens": 500, "recent_tokens": 501}, "fewer than the sinks"),
    ({"recent_tokens": 2 ** 64 - 1}, "fewer than the sinks"), ({"head_dim": 64}, "head_dim"), ({"kv_heads": 0}, "kv_heads"),
    ({"max_context_tokens": 2 ** 31}, "max_context_tokens")])
def test_evict_refuses_shapes(change, message):
    shape = dataclasses.replace(E(4, 256, 3000, 4096, 1000, 1000), **change)
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_compact_cache_evict(BIG, BIG, BIG, BIG, BIG, shape, FP8, FP8, 1, BIG, stream=0x1234)


def test_evict_refuses_pointers_and_types():
    shape = E(4, 256, 3000, 4096, 1000, 1000)

    def go(i=None, bad=None, dtype=BF16, out=BF16, layout=1, ws=BIG, stream=0x1234, **kw):
        args = [BIG] * 5
        if i is not None:
            args[i] = bad
        ops.qwen35_compact_cache_evict(*args, shape, dtype, out, layout, ws, stream=stream, **kw)

    for i, message in enumerate(["cache pointer", "weights pointer", "cache pointer", "weights pointer", "kept_indices pointer"]):
        with pytest.raises(ops.Qwen35PrimitiveError, match=message):
            go(i, None, kv_cache_bytes=1 << 40, out_cache_bytes=1 << 40)
        with pytest.raises(ops.Qwen35PrimitiveError, match="aligned"):
            go(i, FakeTensor(1 << 50, 0x100002))
    for kw, message in [({"dtype": FP8}, "does not widen"), ({"dtype": 0}, "dtype"), ({"out": 7}, "dtype"), ({"layout": 3}, "layout"),
                        ({"stream": 0}, "stream is null"), ({"kv_cache_bytes": 10}, "too small"), ({"out_cache_bytes": 10}, "too small")]:
        with pytest.raises(ops.Qwen35PrimitiveError, match=message):
            go(**kw)


def places(sizes, overlap=None):
    """Stand-ins for the arguments, one behind the other; overlap (i, j, by): i starts `by` bytes before the end of j."""
    at, t = 1 << 32, []
    for n in sizes:
        t.append(FakeTensor(n, at))
        at += (n + 255) // 256 * 256
    if overlap:
        i, j, by = overlap
        t[i] = FakeTensor(sizes[i], t[j].data_ptr() + sizes[j] - by)
    return t


@pytest.mark.parametrize("call", ["decode", "prefill"])
@pytest.mark.parametrize("written", [4, 5, 6, 7])   # output, cache, workspace, key weights
def test_attention_refuses_overlap(call, written):
    shape = dataclasses.replace(MODEL, observed_tokens=1)
    need = getattr(ops, f"qwen35_compact_{call}_workspace_bytes")(shape)
    assert need > 0
    head, row = 16 * 512, 4 * 512
    sizes = [head, row, row, head, head, ops.qwen35_compact_cache_bytes(shape, FP8), need, 4 * 4096 * 4]
    for other in set(range(8)) - {written}:
        t = places(sizes, (written, other, 16))
        with pytest.raises(ops.Qwen35PrimitiveError, match="outputs overlap other arguments"):
            getattr(ops, f"qwen35_compact_attention_{call}")(*t[:6], shape, ops.DTYPE_BF16, FP8, 1, t[6], key_weights=t[7],
                                                             stream=0x1234)


def test_append_refuses_overlap():
    row, cache = 4 * 512, ops.qwen35_compact_cache_bytes(MODEL, FP8)
    for other in (0, 1):
        t = places([row, row, cache], (2, other, 16))
        with pytest.raises(ops.Qwen35PrimitiveError, match="overlaps the rows"):
            ops.qwen35_compact_cache_append(*t, MODEL, ops.DTYPE_BF16, FP8, 1, stream=0x1234)


@pytest.mark.parametrize("written", [2, 3, 4, 5])   # cache, weights, indices, workspace
def test_evict_refuses_overlap(written):
    shape = E(4, 256, 30000, 40000, 1000, 1200)
    need = ops.qwen35_compact_evict_workspace_bytes(shape)
    assert need > 0
    big, small = (S(1, 1, 4, 4, 256, n, 0) for n in (40000, 1200))
    sizes = [ops.qwen35_compact_cache_bytes(big, BF16), 4 * 40000 * 4, ops.qwen35_compact_cache_bytes(small, FP8), 4 * 1200 * 4,
             4 * 1000 * 4, need]
    for other in set(range(6)) - {written}:
        t = places(sizes, (written, other, 16))
        with pytest.raises(ops.Qwen35PrimitiveError, match="outputs overlap other arguments"):
            ops.qwen35_compact_cache_evict(*t[:5], shape, BF16, FP8, 1, t[5], stream=0x1234)


def test_evict_refuses_too_many_segments():
    shape = E(1, 256, 65535 * 4096 + 1, 2 ** 28, 10, 10)
    with pytest.raises(ops.Qwen35PrimitiveError, match="at most 65535"):
        ops.qwen35_compact_evict_workspace_bytes(shape)
    assert ops.qwen35_compact_evict_workspace_bytes(dataclasses.replace(shape, context_tokens=65535 * 4096)) > 0


@pytest.mark.parametrize("written", [4, 5, 6, 7])   # output, cache, workspace, key weights
def test_decode_refuses_lengths_that_it_would_write(written):
    """The lengths are read again after the cache, the workspace and the outputs are written."""
    shape = dataclasses.replace(MODEL, observed_tokens=1, sequences=3, cache_stride_bytes=ops.qwen35_compact_cache_bytes(MODEL, FP8))
    need = ops.qwen35_compact_decode_workspace_bytes(shape)
    head, row = 3 * 16 * 512, 3 * 4 * 512
    sizes = [head, row, row, head, head, 3 * shape.cache_stride_bytes, need, 3 * 4 * 4096 * 4, 3 * 4]
    for by in (12, 4):   # the whole of the lengths, and the first of them
        t = places(sizes, (8, written, by))
        with pytest.raises(ops.Qwen35PrimitiveError, match="outputs overlap other arguments"):
            ops.qwen35_compact_attention_decode(*t[:6], shape, ops.DTYPE_BF16, FP8, 1, t[6], key_weights=t[7], context_lengths=t[8],
                                                stream=0x1234)


def test_append_refuses_lengths_that_it_would_write():
    row, cache = 4 * 512, ops.qwen35_compact_cache_bytes(MODEL, FP8)
    for by in (4, cache):   # the cache's last bytes, and its first
        t = places([row, row, cache, 4], (3, 2, by))
        with pytest.raises(ops.Qwen35PrimitiveError, match="overlaps the rows"):
            ops.qwen35_compact_cache_append(*t[:3], MODEL, ops.DTYPE_BF16, FP8, 1, context_lengths=t[3], stream=0x1234)


def test_refuses_lengths_that_are_not_aligned():
    bad = FakeTensor(4, (1 << 60) + 2)
    t = places([16 * 512, 4 * 512, 4 * 512, 16 * 512, 16 * 512, ops.qwen35_compact_cache_bytes(MODEL, FP8),
                ops.qwen35_compact_decode_workspace_bytes(MODEL)])
    with pytest.raises(ops.Qwen35PrimitiveError, match="context_lengths must be 4-byte aligned"):
        ops.qwen35_compact_attention_decode(*t[:6], MODEL, ops.DTYPE_BF16, FP8, 1, t[6], context_lengths=bad, stream=0x1234)
    with pytest.raises(ops.Qwen35PrimitiveError, match="context_lengths must be 4-byte aligned"):
        ops.qwen35_compact_cache_append(*t[1:3], t[5], MODEL, ops.DTYPE_BF16, FP8, 1, context_lengths=bad, stream=0x1234)
