"""CPU tests of rotary positions and the paged KV cache: frequencies, sizes, refusals before any launch."""
import dataclasses

import numpy as np
import pytest
import torch

import paged_reference as ref
from raftinfer_amd import ops
from test_boundary import FakeTensor

P, R, Q = ops.Qwen35PagedShape, ops.Qwen35PagedRotary, ops.Qwen35RotaryShape
MODEL = P(rows=40, sequences=3, query_heads=16, kv_heads=4, head_dim=256, pages=100, page_tokens=16, table_pages=20,
          max_context_tokens=320)
STEP = dataclasses.replace(MODEL, rows=3)
SCALINGS = {"none": ops.SCALING_NONE, "linear": ops.SCALING_LINEAR, "pair": ops.SCALING_BY_PAIR, "turns": ops.SCALING_BY_TURNS}


def spaced(count):
    """Arguments 1 TiB apart, so that none overlaps another."""
    return [FakeTensor(addr=(i + 1) << 40, nbytes=1 << 39) for i in range(count)]


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("rotary,base,factor,trained", [(64, 1e7, 8.0, 32768.0), (2, 1e4, 2.0, 100.0), (256, 5e5, 32.0, 8192.0),
                                                       (128, 1e4, 1.0, 4096.0)])
def test_frequencies(scaling, rotary, base, factor, trained):
    got, magnitude = ops.qwen35_rotary_frequencies(rotary, base, SCALINGS[scaling], factor, trained, 32.0, 1.0)
    want, m = ref.frequencies(rotary, base, scaling, factor, trained)
    assert np.allclose(got, want, rtol=1e-13, atol=0) and abs(magnitude - m) <= 2.0 ** -24 * m
    assert len(got) == rotary // 2


@pytest.mark.parametrize("change,message", [
    ({"rotary_dim": 0}, "rotary_dim must be even"), ({"rotary_dim": 3}, "rotary_dim must be even"), ({"rotary_dim": 16386}, "rotary_dim"),
    ({"base": 1.0}, "base"), ({"base": float("nan")}, "base"), ({"scaling": 4}, "unsupported rotary scaling"),
    ({"factor": 0.5}, "factor"), ({"factor": float("inf")}, "factor"), ({"trained_tokens": 0.0}, "trained_tokens"),
    ({"slow_turns": 32.0}, "turns"), ({"slow_turns": 0.0}, "turns")])
def test_frequencies_refusals(change, message):
    args = {"rotary_dim": 64, "base": 1e7, "scaling": ops.SCALING_BY_PAIR, "factor": 2.0, "trained_tokens": 100.0, **change}
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_rotary_frequencies(**args)


def test_sizes():
    assert ops.qwen35_paged_cache_bytes(MODEL) == 100 * 2 * 4 * 16 * 256 * 2
    # contexts that no call splits need nothing
    assert ops.qwen35_paged_decode_workspace_bytes(dataclasses.replace(STEP, max_context_tokens=16)) == 0
    long = dataclasses.replace(STEP, table_pages=5000, max_context_tokens=80000)
    assert 0 < ops.qwen35_paged_decode_workspace_bytes(long) < 64 << 20
    # a window bounds what is split
    assert ops.qwen35_paged_decode_workspace_bytes(dataclasses.replace(long, window_tokens=10)) == 0
    more = dataclasses.replace(MODEL, rows=4000, table_pages=5000, max_context_tokens=80000)
    assert 0 < ops.qwen35_paged_prefill_workspace_bytes(more) < 512 << 20


@pytest.mark.parametrize("change,message", [
    ({"rows": 0}, "rows must be positive"), ({"sequences": 0}, "sequences"), ({"sequences": 65536, "rows": 65536}, "sequences"),
    ({"kv_heads": 0}, "kv_heads"), ({"kv_heads": 1025, "query_heads": 1025}, "kv_heads"), ({"query_heads": 0}, "query_heads"),
    ({"query_heads": 6}, "query_heads"), ({"query_heads": 68}, "query_heads"), ({"head_dim": 128}, "head_dim must be 256"),
    ({"rows": 2 ** 18 + 1}, "query rows"), ({"page_tokens": 0}, "page_tokens"), ({"page_tokens": 24}, "page_tokens"),
    ({"pages": 0}, "pages must be"), ({"pages": 2 ** 24 + 1}, "pages must be"), ({"table_pages": 0}, "table_pages"),
    ({"max_context_tokens": 0}, "max_context_tokens"), ({"max_context_tokens": 321}, "max_context_tokens"),
    ({"max_context_tokens": 2 ** 28 + 1, "table_pages": 2 ** 27}, "max_context_tokens")])
def test_shape_refusals(change, message):
    shape = dataclasses.replace(MODEL, **change)
    a = spaced(9)
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_paged_attention_prefill(*a[:7], a[7], shape, 1, stream=0x1234)
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_paged_cache_append(*a, None, None, shape, R(64), 1, stream=0x1234)
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_paged_cache_bytes(shape)


@pytest.mark.parametrize("call", ["prefill", "decode"])
def test_attention_refusals(call):
    prefill = call == "prefill"
    shape = MODEL if prefill else STEP
    shape = dataclasses.replace(shape, pages=10000, table_pages=5000, max_context_tokens=80000)
    names = ["query", "gate", "output", "pages", "page_table"] + ["query_starts"] * prefill + ["context_lengths", "workspace"]
    fn = getattr(ops, f"qwen35_paged_attention_{call}")

    def go(layout=1, act=ops.DTYPE_BF16, stream=0x1234, shape=shape, sizes={}, **put):
        a = dict(zip(names, spaced(len(names))))
        a.update(put)
        fn(*a.values(), shape, layout, act, stream=stream, **sizes)

    refused = lambda message: pytest.raises(ops.Qwen35PrimitiveError, match=message)  # noqa: E731
    for name in names:
        if name != "gate":
            with refused(f"{name} .*is null|{name} is null"):
                go(**{name: None})
        align = 16 if name in ("query", "gate", "output", "pages", "workspace") else 4
        with refused("aligned"):
            go(**{name: FakeTensor(addr=(77 << 40) + align // 2, nbytes=1 << 39)})
    with refused("stream is null"):
        go(stream=0)
    with refused("layout"):
        go(layout=2)
    with refused("must be bf16"):
        go(act=ops.DTYPE_F16)
    with refused("cache is too small"):
        go(sizes={"pages_bytes": 10000 * 2 * 4 * 16 * 512 - 1})
    need = getattr(ops, f"qwen35_paged_{call}_workspace_bytes")(shape)
    with refused("workspace is too small"):
        go(sizes={"workspace_bytes": need - 1})
    for written in ("output", "workspace"):
        for other in names:
            if other != written:
                with refused("overlap"):
                    a = dict(zip(names, spaced(len(names))))
                    go(**{written: a[other]})
    if not prefill:
        with refused("one row per sequence"):
            go(shape=dataclasses.replace(shape, rows=4))
        with refused("one row per sequence"):
            ops.qwen35_paged_decode_workspace_bytes(dataclasses.replace(shape, rows=4))


def test_strides_are_checked():
    a = spaced(9)
    rows, heads = STEP.rows, STEP.query_heads
    for strides, message in [((heads * 256, 252, 1), "multiples of 8"), ((256, 256, 1), "output rows or heads overlap"),
                             ((heads * 256, 128, 1), "output rows or heads overlap"), ((2 ** 62, 256, 1), "overflow")]:
        out = FakeTensor(addr=50 << 40, nbytes=1 << 30)
        out.ndim, out.shape, out.stride = 3, (rows, heads, 256), lambda s=strides: s
        with pytest.raises(ops.Qwen35PrimitiveError, match=message):
            ops.qwen35_paged_attention_decode(a[0], a[1], out, *a[3:6], a[6], STEP, 1, stream=0x1234)
    x = torch.empty(4, 16, 256, dtype=torch.bfloat16).transpose(1, 2)
    with pytest.raises(ops.Qwen35PrimitiveError, match="contiguous"):
        ops.qwen35_paged_attention_decode(x, *a[1:6], a[6], STEP, 1, stream=0x1234)


@pytest.mark.parametrize("change,message", [
    ({"rotary_dim": 258}, "rotary_dim"), ({"rotary_dim": 24}, "rotary_dim"), ({"rotary_dim": 12, "interleaved": True}, "rotary_dim"),
    ({"rotary_dim": 0}, "frequencies go with"), ({"magnitude": float("nan")}, "magnitude"), ({"epsilon": -1.0}, "epsilon"),
    ({"epsilon": float("inf")}, "epsilon")])
def test_append_refuses_rotary(change, message):
    a = spaced(9)
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_paged_cache_append(*a, None, None, MODEL, dataclasses.replace(R(64), **change), 1, stream=0x1234)


def test_append_refusals():
    names = ["query", "key", "value", "query_output", "pages", "page_table", "query_starts", "context_lengths", "frequencies",
             "query_weight", "key_weight"]

    def go(layout=1, act=ops.DTYPE_BF16, weight_dtype=ops.DTYPE_BF16, stream=0x1234, sizes={}, **put):
        a = dict(zip(names, spaced(len(names))))
        a.update(put)
        ops.qwen35_paged_cache_append(*a.values(), MODEL, R(64), layout, act, weight_dtype, stream=stream, **sizes)

    refused = lambda message: pytest.raises(ops.Qwen35PrimitiveError, match=message)  # noqa: E731
    for name in ("key", "value", "pages", "page_table", "query_starts", "context_lengths"):
        with refused(f"{name} pointer is null"):
            go(**{name: None})
    for name in ("query", "query_output"):
        with refused("go together"):
            go(**{name: None})
    with refused("frequencies go with"):
        go(frequencies=None)
    for i, name in enumerate(names):
        with refused("aligned"):
            go(**{name: FakeTensor(addr=(77 << 40) + 1, nbytes=1 << 39)})
    with refused("stream is null"):
        go(stream=0)
    with refused("layout"):
        go(layout=9)
    with refused("must be bf16"):
        go(act=ops.DTYPE_F32)
    with refused("weights must be"):
        go(weight_dtype=ops.DTYPE_F16)
    with refused("cache is too small"):
        go(sizes={"pages_bytes": 100 * 2 * 4 * 16 * 512 - 1})
    for written in ("query_output", "pages"):
        for other in names:
            if other != written:
                with refused("overlap"):
                    go(**{written: dict(zip(names, spaced(len(names))))[other]})


@pytest.mark.parametrize("change,message", [
    ({"rows": 0}, "rows"), ({"rows": 2 ** 23}, "rows"), ({"heads": 0}, "heads"), ({"heads": 65536}, "heads"), ({"head_dim": 0}, "head_dim"),
    ({"head_dim": 16385}, "head_dim"), ({"rotary_dim": 0}, "rotary_dim"), ({"rotary_dim": 63}, "rotary_dim"),
    ({"rotary_dim": 258}, "rotary_dim"), ({"magnitude": float("inf")}, "magnitude")])
def test_rotary_refuses_shapes(change, message):
    x = torch.empty(8, dtype=torch.bfloat16)
    a = spaced(5)
    for t in a:
        t.dtype = torch.bfloat16
    with pytest.raises(ops.Qwen35PrimitiveError, match=message):
        ops.qwen35_rotary(*a, dataclasses.replace(Q(10, 4, 256, 64), **change), 1e-6, stream=0x1234)


def test_rotary_refusals():
    def go(stream=0x1234, epsilon=1e-6, dtype=torch.bfloat16, wdt=torch.bfloat16, **put):
        names = ["input", "weight", "output", "positions", "frequencies"]
        a = dict(zip(names, spaced(5)))
        a.update(put)
        for k, t in a.items():
            if t is not None:
                t.dtype = wdt if k == "weight" else dtype
        ops.qwen35_rotary(*a.values(), Q(10, 4, 256, 64), epsilon, stream=stream)

    refused = lambda message: pytest.raises(ops.Qwen35PrimitiveError, match=message)  # noqa: E731
    with refused("stream is null"):
        go(stream=0)
    with refused("epsilon"):
        go(epsilon=float("nan"))
    with refused("unsupported"):
        go(dtype=torch.float64)
    with refused("weight dtype"):
        go(wdt=torch.float16)
    for name in ("input", "weight", "output", "positions", "frequencies"):
        with refused("aligned to their elements"):
            go(**{name: FakeTensor(addr=(77 << 40) + 1, nbytes=1 << 39)})
        if name != "output":  # one row of it lies in the output's
            with refused("overlaps"):
                go(**{name: FakeTensor(addr=(3 << 40) + 1024, nbytes=1 << 39)})


def test_views_that_have_no_strides_to_pass():
    """Broadcast rows or heads, and index tensors with gaps, are refused before any address is taken."""
    q = torch.zeros(3, 16, 256, dtype=torch.bfloat16)
    rest = [FakeTensor(addr=(i + 1) << 40, nbytes=1 << 39) for i in range(5)]
    out = torch.zeros(3, 16, 256, dtype=torch.bfloat16)
    table = torch.zeros(3, 40, dtype=torch.int32)
    refused = lambda message: pytest.raises(ops.Qwen35PrimitiveError, match=message)  # noqa: E731
    decode = lambda q, table: ops.qwen35_paged_attention_decode(q, None, out, rest[0], table, rest[1], rest[2], STEP, 1, stream=0x1234,  # noqa: E731
                                                                workspace_bytes=1 << 39)
    for bad in (q[:1].expand(3, 16, 256), q[:, :1].expand(3, 16, 256)):
        with refused("broadcast"):
            decode(bad, rest[3])
    with refused("last dimension"):
        decode(q.transpose(1, 2), rest[3])
    with refused("contiguous"):
        decode(q, table[:, ::2])
    with refused("contiguous"):
        decode(q, table[:, :20])
    with refused("contiguous"):
        decode(q.reshape(3, 4096)[:, ::2], rest[3])
    with refused("contiguous"):
        ops.qwen35_rotary(q, None, out, torch.zeros(6, dtype=torch.int32)[::2], rest[0], Q(3, 16, 256, 64), 1e-6, stream=0x1234)
    with refused("one type"):
        ops.qwen35_paged_cache_append(rest[0], rest[1], rest[2], rest[3], rest[4], rest[0], rest[1], rest[2], rest[3],
                                      torch.ones(256), torch.ones(256, dtype=torch.bfloat16), STEP, R(64), 1, stream=0x1234)


def test_a_bound_above_the_table_is_the_tables():
    """A program's largest context can be above what a call's page table holds: the sizes are those of the table's positions, and
    calls refuse what comes behind the shape's checks."""
    for shape, call in ((MODEL, "prefill"), (STEP, "decode")):
        table_pages = 600  # 9600 positions
        tight = dataclasses.replace(shape, pages=10000, table_pages=table_pages, max_context_tokens=table_pages * 16)
        size = getattr(ops, f"qwen35_paged_{call}_workspace_bytes")
        assert size(tight) > 0
        for bound in (table_pages * 16 + 1, 262144, 2 ** 28):
            for window in (0, 100, table_pages * 16 + 5):
                loose = dataclasses.replace(tight, max_context_tokens=bound, window_tokens=window)
                assert size(loose) == size(dataclasses.replace(tight, window_tokens=window))
            a = spaced(7)
            table = torch.zeros(3, table_pages, dtype=torch.int32)
            starts = [a[4]] if call == "prefill" else []
            with pytest.raises(ops.Qwen35PrimitiveError, match="workspace is too small"):
                getattr(ops, f"qwen35_paged_attention_{call}")(*a[:4], table, *starts, a[5], a[6], dataclasses.replace(tight, max_context_tokens=bound), 1,
                                                               stream=0x1234, workspace_bytes=0)
    a = spaced(9)
    with pytest.raises(ops.Qwen35PrimitiveError, match="overlap"):
        ops.qwen35_paged_cache_append(a[0], a[1], a[2], a[0], a[4], torch.zeros(3, 20, dtype=torch.int32), *a[6:9], None, None,
                                      dataclasses.replace(MODEL, max_context_tokens=6001), R(64), 1, stream=0x1234)


def real(shape, decode=False):
    """Arguments of an attention call that are tensors, on the host: a call that is not refused for them is for its null stream."""
    bf, i32 = torch.bfloat16, torch.int32
    x = {"query": torch.zeros(shape.rows, 16, 256, dtype=bf), "gate": torch.zeros(shape.rows, 16, 256, dtype=bf),
         "output": torch.zeros(shape.rows, 16, 256, dtype=bf), "pages": torch.zeros(shape.pages, 2, 4, 16, 256, dtype=bf),
         "page_table": torch.zeros(shape.sequences, shape.table_pages, dtype=i32), "query_starts": torch.zeros(shape.sequences + 1, dtype=i32),
         "context_lengths": torch.zeros(shape.sequences, dtype=i32), "workspace": torch.zeros(1 << 20, dtype=torch.uint8)}
    if decode:
        del x["query_starts"]
    return x


def append_arguments(shape):
    x = real(shape)
    q = {k: x[k] for k in ("pages", "page_table", "query_starts", "context_lengths")}
    key = torch.zeros(shape.rows, 4, 256, dtype=torch.bfloat16)
    return {"query": x["query"], "key": key, "value": key.clone(), "query_output": x["output"], **q, "frequencies": torch.zeros(32, dtype=torch.float64),
            "query_weight": torch.ones(256), "key_weight": torch.ones(256)}


CALLS = {"prefill": lambda a, **kw: ops.qwen35_paged_attention_prefill(*a.values(), MODEL, 1, stream=0, **kw),
         "decode": lambda a, **kw: ops.qwen35_paged_attention_decode(*a.values(), STEP, 1, stream=0, **kw),
         "append": lambda a, **kw: ops.qwen35_paged_cache_append(*a.values(), MODEL, R(64), 1, stream=0, **kw),
         "rotary": lambda a, **kw: ops.qwen35_rotary(*a.values(), Q(40, 16, 256, 64), 1e-6, stream=0, **kw)}


def arguments(call):
    if call == "append":
        return append_arguments(MODEL)
    if call == "rotary":
        x = append_arguments(MODEL)
        return {"input": x["query"], "weight": x["query_weight"], "output": x["query_output"], "positions": torch.zeros(40, dtype=torch.int32),
                "frequencies": x["frequencies"]}
    return real(MODEL if call == "prefill" else STEP, call == "decode")


def right(call, change={}, **kw):
    """The call with these arguments is refused for its stream alone."""
    with pytest.raises(ops.Qwen35PrimitiveError, match="stream is null"):
        CALLS[call]({**arguments(call), **change}, **kw)


@pytest.mark.parametrize("call", list(CALLS))
def test_element_types(call):
    """A tensor of another element type than the call reads is refused: its bytes would be taken for that type's."""
    right(call)
    a = arguments(call)
    indices = [k for k in a if k in ("positions", "page_table", "query_starts", "context_lengths")]
    for name in indices:
        right(call, {name: a[name].view(torch.uint32)})
        for other in (torch.int64, torch.float32, torch.int16):
            with pytest.raises(ops.Qwen35PrimitiveError, match=f"{name} must be of type"):
                CALLS[call]({**a, name: a[name].to(other)})
    if "frequencies" in a:
        with pytest.raises(ops.Qwen35PrimitiveError, match="frequencies must be of type"):
            CALLS[call]({**a, "frequencies": a["frequencies"].float()})
    for name in ("query", "key", "value", "query_output", "gate", "output"):
        if name in a:
            for other in (torch.float16, torch.float32, torch.int16):
                with pytest.raises(ops.Qwen35PrimitiveError, match="activations must be of one type"):
                    CALLS[call]({**a, name: a[name].to(other)})
    if "pages" in a:
        right(call, {"pages": a["pages"].view(torch.uint8)})
        for other in (torch.float16, torch.float32):
            with pytest.raises(ops.Qwen35PrimitiveError, match="pages must be of type"):
                CALLS[call]({**a, "pages": a["pages"].to(other)})
    if call == "append":
        right(call, {"query_weight": torch.ones(256, dtype=torch.bfloat16), "key_weight": torch.ones(256, dtype=torch.bfloat16)})
        with pytest.raises(ops.Qwen35PrimitiveError, match="query_weight must be of type"):
            CALLS[call](a, weight_dtype=ops.DTYPE_BF16)
    if call == "rotary":
        right(call, {"weight": None})
        with pytest.raises(ops.Qwen35PrimitiveError, match="weight must be of type"):
            CALLS[call]({**a, "weight": torch.ones(256, dtype=torch.float64)})


@pytest.mark.parametrize("call", list(CALLS))
def test_tensors_too_small(call):
    """A tensor of fewer elements than the shape says would be read, or written, past its end."""
    a = arguments(call)
    for name in [k for k in a if k in ("positions", "page_table", "query_starts", "context_lengths", "frequencies", "weight", "query_weight", "key_weight")]:
        with pytest.raises(ops.Qwen35PrimitiveError, match=f"{name} must have"):
            CALLS[call]({**a, name: a[name][:-1].contiguous()})
    if call != "rotary":
        more = {k: v for k, v in a.items()}
        wider = torch.zeros(3, 21, dtype=torch.int32)
        with pytest.raises(ops.Qwen35PrimitiveError, match="rows of 20 entries"):
            CALLS[call]({**more, "page_table": wider})
        right(call, {"page_table": torch.zeros(60, dtype=torch.int32)})
        right(call, {"page_table": torch.zeros(5, 20, dtype=torch.int32), "context_lengths": torch.zeros(9, dtype=torch.int32)})
    for name in ("input", "query", "key", "value", "query_output", "gate", "output"):
        if name in a:
            with pytest.raises(ops.Qwen35PrimitiveError, match="activation must be"):
                CALLS[call]({**a, name: a[name][:-1]})
            with pytest.raises(ops.Qwen35PrimitiveError, match="activation must be"):
                CALLS[call]({**a, name: a[name][:, :-1]})
            with pytest.raises(ops.Qwen35PrimitiveError, match="activation must be"):
                CALLS[call]({**a, name: a[name][..., :-8]})


@pytest.mark.parametrize("call", list(CALLS))
def test_activations_in_other_dimensions(call):
    """Strides are those of rows and heads only where the dimensions are rows, heads and dim: a tensor [1, rows, heads * dim] had
    its rows' stride taken for the heads', and was read past its end."""
    a = arguments(call)
    for name in ("input", "query", "key", "value", "query_output", "gate", "output"):
        if name not in a:
            continue
        x = a[name]
        rows, heads, dim = x.shape
        for same in (x.view(1, rows, heads * dim), x.view(rows, 1, heads * dim), x.view(rows, heads * dim), x.view(rows * heads, dim),
                     x.view(1, rows * heads, dim), x.view(rows, heads, 2, dim // 2), x.view(-1)):
            assert ops._heads(same, x.dtype, (rows, heads, dim))[1:] in ((0, 0), (heads * dim, 0)), same.shape
            right(call, {name: same})
        # part of a larger tensor, given whole
        more = torch.zeros(rows + 2, heads + 3, dim + 8, dtype=x.dtype)
        assert ops._heads(more, x.dtype, (rows, heads, dim))[1:] == ((heads + 3) * (dim + 8), dim + 8)
        right(call, {name: more})
        for other in (x.transpose(0, 1).contiguous(), x.view(1, rows, heads * dim).expand(2, rows, heads * dim)):
            with pytest.raises(ops.Qwen35PrimitiveError):
                CALLS[call]({**a, name: other})


def test_frequencies_left_at_their_defaults():
    """By turns from 4 to 1 of them over the trained context, by pair from 32 to 1: what models with these scalings publish."""
    for scaling, name, fast in ((ops.SCALING_BY_TURNS, "turns", 4.0), (ops.SCALING_BY_PAIR, "pair", 32.0)):
        got, magnitude = ops.qwen35_rotary_frequencies(128, 5e5, scaling, 8.0, 8192.0)
        want, m = ref.frequencies(128, 5e5, name, 8.0, 8192.0, fast, 1.0)
        assert np.allclose(got, want, rtol=1e-13, atol=0) and abs(magnitude - m) <= 2.0 ** -24 * m
        other, _ = ref.frequencies(128, 5e5, name, 8.0, 8192.0, 36.0 - fast, 1.0)
        assert not np.allclose(got, other, rtol=1e-3, atol=0)


def test_the_library_takes_a_bound_above_the_table_everywhere():
    """Through the C interface, where nothing but the shape is at hand, the pool's bytes too."""
    import ctypes
    from raftinfer_amd import _lib
    for bound, ok in ((321, True), (2 ** 28, True), (2 ** 28 + 1, False), (0, False)):
        size = ctypes.c_size_t()
        shape = dataclasses.replace(MODEL, max_context_tokens=bound).c()
        status = _lib.load().raftinfer_amd_paged_cache_bytes(shape, ctypes.byref(size))
        assert (status == 0) == ok, bound
        assert not ok or size.value == ops.qwen35_paged_cache_bytes(MODEL)
