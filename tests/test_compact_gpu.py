"""The compact KV cache (8-bit blocks, sliding window with sinks, key weights, eviction) against its definition in
64 bits (compact_reference.py)."""
import numpy as np
import pytest
import torch

import compact_reference as ref
from helpers import bf16, normal, rng
from raftinfer_amd import ops

pytestmark = pytest.mark.gpu

D = 256
BF16, FP8 = ops.CACHE_BF16, ops.CACHE_FP8_E4M3


def dev(a, dtype=torch.bfloat16):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to("cuda", dtype)


def host(t):
    return t.float().cpu().numpy()


class Cache:
    """One sequence's cache on the device beside its reference.  Unused places hold other values (in an 8-bit
    cache NaN codes among them; bf16: NaN)."""

    def __init__(self, r, dtype, layout, hkv, cap):
        self.dtype, self.layout, self.hkv, self.cap = dtype, layout, hkv, cap
        if dtype == FP8:
            self.ref = ref.Fp8Cache(hkv, cap, r)
            self.buf = torch.from_numpy(self.ref.buffer(layout)).cuda()
        else:
            self.ref = np.full((2, hkv, cap, D), np.nan, np.float32)
            self.buf = torch.full((2 * hkv * cap * D,), float("nan"), device="cuda", dtype=torch.bfloat16).view(torch.uint8)

    def shape(self, t, heads, past, **kw):
        return ops.Qwen35CompactShape(t, 1, heads, self.hkv, D, self.cap, past, **kw)

    def want_store(self, past, k, v):
        if self.dtype == FP8:
            self.ref.store(past, k, v)
        else:
            self.ref[0, :, past:past + len(k)] = k.transpose(1, 0, 2)
            self.ref[1, :, past:past + len(k)] = v.transpose(1, 0, 2)

    def store(self, past, k, v):
        self.want_store(past, k, v)
        ops.qwen35_compact_cache_append(dev(k), dev(v), self.buf, self.shape(len(k), self.hkv, past), ops.DTYPE_BF16,
                                        self.dtype, self.layout)

    def held(self, n):
        return self.ref.held(n) if self.dtype == FP8 else self.ref[:, :, :n].astype(np.float64)

    def check(self, what=""):
        """Every byte that the definition fixes: codes (NaN codes as NaN), scales, and places that nothing wrote."""
        raw = self.buf.cpu().numpy()
        if self.dtype == FP8:
            got = ref.Fp8Cache(self.hkv, self.cap).load(raw, self.layout)
            assert np.array_equal(got.scales, self.ref.scales), what
            assert np.array_equal(ref.E4M3[got.codes], ref.E4M3[self.ref.codes], equal_nan=True), what
        else:
            got = torch.from_numpy(raw).view(torch.bfloat16).float().numpy()
            got = got.reshape((2, self.hkv, self.cap, D) if self.layout == 1 else (2, self.cap, self.hkv, D))
            got = got if self.layout == 1 else got.transpose(0, 2, 1, 3)
            assert np.array_equal(got, self.ref, equal_nan=True), what


def rows(r, t, hkv, heavy=True):
    x = normal(r, t, hkv, D)
    if heavy:
        x[r.random((t, hkv)) < 0.05] *= 8
    return bf16(x)


def filled(r, dtype, layout, hkv, cap, n):
    c = Cache(r, dtype, layout, hkv, cap)
    if n:
        c.store(0, rows(r, n, hkv), rows(r, n, hkv))
    return c


def near(got, want, bound, what=""):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(err / np.maximum(bound, 1e-300)):.2f} bounds"


def near_weights(got, before, want, rel, what=""):
    near(got, before + want, want * rel + 2.0 ** -23 * (np.abs(before) + want) + 1e-38, what)


def run_decode(c, r, heads, past, window=0, sinks=0, weights=False, nan_value_at=None):
    k, v = rows(r, 1, c.hkv), rows(r, 1, c.hkv)
    q, g = bf16(normal(r, 1, heads, D)), bf16(normal(r, 1, heads, D))
    shape = c.shape(1, heads, past, window_tokens=window, sink_tokens=sinks, observed_tokens=int(weights))
    ws = torch.full((ops.qwen35_compact_decode_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    out = torch.empty(heads * D, device="cuda", dtype=torch.bfloat16)
    before = r.random((c.hkv, c.cap)).astype(np.float32) if weights else None
    w = dev(before, torch.float32) if weights else None
    ops.qwen35_compact_attention_decode(dev(q), dev(k), dev(v), dev(g), out, c.buf, shape, ops.DTYPE_BF16, c.dtype,
                                        c.layout, ws, key_weights=w)
    c.want_store(past, k, v)
    want, bound, ww, rel = ref.attention(q, g, c.held(past + 1), past, window, sinks, int(weights))
    torch.cuda.synchronize()
    near(host(out).reshape(1, heads, D), want, bound, "out")
    c.check("cache")
    if weights:
        n = past + 1
        near_weights(host(w)[:, :n], before[:, :n], ww, rel, "weights")
        assert np.array_equal(host(w)[:, n:], before[:, n:])


def run_prefill(c, r, heads, t, past, window=0, sinks=0, observed=0):
    k, v = rows(r, t, c.hkv), rows(r, t, c.hkv)
    q, g = bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    shape = c.shape(t, heads, past, window_tokens=window, sink_tokens=sinks, observed_tokens=observed)
    ws = torch.full((ops.qwen35_compact_prefill_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    out = torch.empty(t * heads * D, device="cuda", dtype=torch.bfloat16)
    before = r.random((c.hkv, c.cap)).astype(np.float32) if observed else None
    w = dev(before, torch.float32) if observed else None
    ops.qwen35_compact_attention_prefill(dev(q), dev(k), dev(v), dev(g), out, c.buf, shape, ops.DTYPE_BF16, c.dtype,
                                         c.layout, ws, key_weights=w)
    c.want_store(past, k, v)
    n = past + t
    want, bound, ww, rel = ref.attention(q, g, c.held(n), past, window, sinks, observed)
    torch.cuda.synchronize()
    near(host(out).reshape(t, heads, D), want, bound, "out")
    c.check("cache")
    if observed:
        near_weights(host(w)[:, :n], before[:, :n], ww, rel, "weights")
        assert np.array_equal(host(w)[:, n:], before[:, n:])


# ------------------------------------------------------------------ store

@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hkv,cap,steps", [(4, 70, [1] * 70), (1, 100, [5, 27, 1, 40, 27]), (3, 33, [33]),
                                           (4, 64, [31, 2, 31]), (2, 129, [1, 96, 32])])
def test_store_in_steps(gpu, layout, dtype, hkv, cap, steps):
    r = rng(1)
    c = Cache(r, dtype, layout, hkv, cap)
    past = 0
    for i, t in enumerate(steps):
        # rows of growing size: a block's scale grows with its later rows
        c.store(past, bf16(rows(r, t, hkv) * 1.5 ** (i % 40)), bf16(rows(r, t, hkv) / 1.5 ** (i % 40)))
        past += t
        if i in (0, len(steps) // 2, len(steps) - 1):
            c.check(f"step {i}")


def test_store_extremes(gpu):
    r = rng(2)
    c = Cache(r, FP8, 1, 2, 96)
    x = rows(r, 40, 2)
    x[3, 0, :] = 0                                   # a zero row
    x[5, 0, 7], x[6, 1, 9], x[7, 1, 1] = np.inf, -np.inf, np.nan
    x[9, 1, :] = 448.0 * 4
    x[10, 1, 0] = 464.0 * 4                          # above 448 s for s = 4: scale 8
    x[33, 0, 5] = 3e38                               # block 1, head 0: every other code becomes 0
    y = np.zeros((40, 2, D), np.float32)             # V: all zero, the smallest scale
    y[34, 1, :4] = [2.0 ** -126, 2.0 ** -130, -2.0 ** -133, 2.0 ** -120]
    c.store(0, bf16(x), bf16(y))
    c.check("first")
    c.store(40, bf16(rows(r, 3, 2)), bf16(rows(r, 3, 2)))  # raises V's smallest scales
    c.check("grown")
    c.store(20, bf16(rows(r, 2, 2)), bf16(rows(r, 2, 2)))  # back inside block 0: rows behind stay as they are
    c.check("rolled back")


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_store_with_lengths(gpu, dtype):
    r = rng(3)
    cap, hkv = 50, 4
    caches = [filled(r, dtype, 1, hkv, cap, n) for n in (0, 31, 32, 49, 7, 9)]
    lengths = [1, 32, 33, 50, 0, 51]  # the last two store nothing
    buf = torch.stack([c.buf for c in caches])
    k, v = rows(r, 6, hkv), rows(r, 6, hkv)
    shape = ops.Qwen35CompactShape(1, 6, 16, hkv, D, cap, 0, buf.shape[1])
    ops.qwen35_compact_cache_append(dev(k), dev(v), buf, shape, ops.DTYPE_BF16, dtype, 1,
                                    context_lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32))
    for i, c in enumerate(caches):
        if 1 <= lengths[i] <= cap:
            c.want_store(lengths[i] - 1, k[i:i + 1], v[i:i + 1])
        c.buf = buf[i]
        c.check(f"sequence {i}")


# ------------------------------------------------------------------ decode

@pytest.mark.parametrize("dtype,layout", [(BF16, 1), (FP8, 1), (FP8, 0)])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 129, 500, 1301])
def test_decode_contexts(gpu, dtype, layout, n):
    r = rng(10 + n)
    run_decode(filled(r, dtype, layout, 4, n + (n % 3) * 50, n - 1), r, 16, n - 1, weights=n % 2 == 1)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hkv,group", [(1, 1), (1, 16), (2, 3), (4, 8), (5, 2)])
def test_decode_heads(gpu, dtype, hkv, group):
    r = rng(20 + group)
    run_decode(filled(r, dtype, group % 2, hkv, 300, 210), r, hkv * group, 210, weights=True)


@pytest.mark.parametrize("dtype,layout", [(BF16, 0), (BF16, 1), (FP8, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 4), (32, 0), (33, 64), (100, 33), (100, 500), (899, 0),
                                          (900, 1), (5000, 3)])
def test_decode_window(gpu, dtype, layout, window, sinks):
    r = rng(30 + window)
    run_decode(filled(r, dtype, layout, 4, 1000, 900), r, 16, 900, window, sinks, weights=sinks % 2 == 1)


def test_decode_long(gpu):
    r = rng(40)
    run_decode(filled(r, FP8, 1, 1, 20000, 19000), r, 4, 19000, weights=True)
    run_decode(filled(r, BF16, 1, 1, 9000, 8999), r, 4, 8999)


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_decode_batch(gpu, dtype):
    r = rng(50)
    cap, hkv, heads = 700, 4, 16
    lengths = [1, 700, 33, 0, 256, 701, 64]
    caches = [filled(r, dtype, 1, hkv, cap, max(0, min(n, cap) - 1)) for n in lengths]
    buf = torch.stack([c.buf for c in caches])
    b = len(lengths)
    k, v, q, g = rows(r, b, hkv), rows(r, b, hkv), bf16(normal(r, b, heads, D)), bf16(normal(r, b, heads, D))
    shape = ops.Qwen35CompactShape(1, b, heads, hkv, D, cap, 0, buf.shape[1], 128, 5, 1)
    ws = torch.full((ops.qwen35_compact_decode_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    w = torch.zeros(b, hkv, cap, device="cuda")
    out = torch.empty(b, heads, D, device="cuda", dtype=torch.bfloat16)
    ops.consume_capacity_errors()
    ops.qwen35_compact_attention_decode(dev(q), dev(k), dev(v), dev(g), out, buf, shape, ops.DTYPE_BF16, dtype, 1, ws,
                                        context_lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32),
                                        key_weights=w)
    assert ops.consume_capacity_errors() == 2
    for i, c in enumerate(caches):
        c.buf, n = buf[i], lengths[i]
        if n == 0 or n > cap:
            assert torch.isnan(out[i]).all() and not w[i].any()
        else:
            c.want_store(n - 1, k[i:i + 1], v[i:i + 1])
            want, bound, ww, rel = ref.attention(q[i:i + 1], g[i:i + 1], c.held(n), n - 1, 128, 5, 1)
            near(host(out[i])[None], want, bound, f"sequence {i}")
            near_weights(host(w[i])[:, :n], 0.0, ww, rel, f"weights {i}")
            assert not w[i, :, n:].any()
        c.check(f"cache {i}")


# ------------------------------------------------------------------ prefill

@pytest.mark.parametrize("dtype,layout", [(BF16, 1), (BF16, 0), (FP8, 1), (FP8, 0)])
@pytest.mark.parametrize("t,past", [(1, 0), (1, 40), (2, 31), (31, 0), (33, 0), (64, 64), (70, 301), (129, 5)])
def test_prefill_lengths(gpu, dtype, layout, t, past):
    r = rng(60 + t)
    c = filled(r, dtype, layout, 4, past + t + t % 40, past)
    run_prefill(c, r, 16, t, past, observed=t // 2)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hkv,group", [(1, 1), (1, 16), (2, 3), (3, 5), (2, 8)])
def test_prefill_heads(gpu, dtype, hkv, group):
    r = rng(70 + group)
    run_prefill(filled(r, dtype, 1, hkv, 200, 37), r, hkv * group, 50, 37, observed=50)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("t,past", [(100, 0), (40, 333)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (7, 0), (32, 32), (50, 3), (64, 70), (90, 0), (300, 1)])
def test_prefill_window(gpu, dtype, t, past, window, sinks):
    r = rng(80 + window)
    run_prefill(filled(r, dtype, 1, 4, past + t, past), r, 16, t, past, window, sinks, observed=min(t, window))


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_prefill_long_past(gpu, dtype):
    # few query rows behind many keys: the keys are split over workgroups
    r = rng(90)
    run_prefill(filled(r, dtype, 1, 1, 5000, 4801), r, 4, 5, 4801, observed=5)


def test_prefill_many_tokens(gpu):
    # enough columns that the keys are not split
    r = rng(91)
    t, hkv, heads = 4200, 4, 16
    c = Cache(r, BF16, 1, hkv, t)
    k, v, q, g = rows(r, t, hkv), rows(r, t, hkv), bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    shape = c.shape(t, heads, 0, window_tokens=100, sink_tokens=4, observed_tokens=3)
    ws = torch.empty(ops.qwen35_compact_prefill_workspace_bytes(shape), device="cuda", dtype=torch.uint8)
    w = torch.zeros(hkv, t, device="cuda")
    out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
    ops.qwen35_compact_attention_prefill(dev(q), dev(k), dev(v), dev(g), out, c.buf, shape, ops.DTYPE_BF16, BF16, 1, ws,
                                         key_weights=w)
    c.want_store(0, k, v)
    got = host(out)
    for i in (0, 1, 31, 99, 100, 103, 104, 105, 2049, 4100, 4199):
        want, bound, ww, rel = ref.attention(q[i:i + 1], g[i:i + 1], c.held(i + 1), i, 100, 4, 1)
        near(got[i:i + 1], want, bound, f"token {i}")
    want = np.zeros((hkv, t))
    for i in (4197, 4198, 4199):
        _, _, ww, rel = ref.attention(q[i:i + 1], g[i:i + 1], c.held(i + 1), i, 100, 4, 1)
        want[:, :i + 1] += ww
    near_weights(host(w), 0.0, want, rel.max() + 2.0 ** -20, "weights")


def some_tokens(t):
    return sorted({0, 1, 7, 8, 9, 15, 16, 31, 32, 33, t // 2, t - 3, t - 2, t - 1} & set(range(t)))


# Enough columns and keys that workgroups of 128 columns share the tiles, whole and split over the keys; the last
# three of them, of 128 and of 32 columns, split the later tokens' keys only.
WIDE = [(16, 16, 130, 600, 0, 0), (16, 16, 131, 700, 333, 40), (7, 13, 501, 300, 0, 0), (7, 13, 503, 800, 400, 3),
        (2, 16, 130, 3001, 0, 0), (2, 16, 131, 4000, 3000, 70), (1, 16, 300, 5000, 4999, 1), (1, 3, 900, 4000, 0, 0),
        (2, 5, 700, 640, 0, 0), (4, 4, 1400, 0, 0, 0), (1, 1, 1200, 0, 0, 0), (1, 2, 700, 5, 600, 3)]


@pytest.mark.parametrize("dtype,layout", [(BF16, 1), (FP8, 1), (BF16, 0), (FP8, 0)])
@pytest.mark.parametrize("hkv,group,t,past,window,sinks", WIDE)
def test_prefill_wide(gpu, dtype, layout, hkv, group, t, past, window, sinks):
    r = rng(92 + t)
    heads, n, observed = hkv * group, past + t, 3
    c = filled(r, dtype, layout, hkv, n + 5, past)
    k, v, q, g = rows(r, t, hkv), rows(r, t, hkv), bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    shape = c.shape(t, heads, past, window_tokens=window, sink_tokens=sinks, observed_tokens=observed)
    ws = torch.full((ops.qwen35_compact_prefill_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    w = torch.zeros(hkv, n + 5, device="cuda")
    out, again = (torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    args = dev(q), dev(k), dev(v), dev(g)
    ops.qwen35_compact_attention_prefill(*args, out, c.buf, shape, ops.DTYPE_BF16, dtype, layout, ws, key_weights=w)
    c.want_store(past, k, v)
    got = host(out)
    assert np.isfinite(got).all()
    for i in some_tokens(t):
        m = past + i + 1
        want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], c.held(m), past + i, window, sinks)
        near(got[i:i + 1], want, bound, f"token {i}")
    want, rel = np.zeros((hkv, n)), 0.0
    for i in range(t - observed, t):
        _, _, ww, e = ref.attention(q[i:i + 1], g[i:i + 1], c.held(past + i + 1), past + i, window, sinks, 1)
        want[:, :past + i + 1] += ww
        rel = max(rel, e.max())
    near_weights(host(w)[:, :n], 0.0, want, rel + 2.0 ** -20, "weights")
    # without the weights, and over the same rows once more: the same bits
    plain = c.shape(t, heads, past, window_tokens=window, sink_tokens=sinks)
    small = torch.full((ops.qwen35_compact_prefill_workspace_bytes(plain),), 0xFF, device="cuda", dtype=torch.uint8)
    for o in (out, again):
        ops.qwen35_compact_attention_prefill(*args, o, c.buf, plain, ops.DTYPE_BF16, dtype, layout, small)
    assert torch.equal(out, again)
    for i in some_tokens(t):
        m = past + i + 1
        want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], c.held(m), past + i, window, sinks)
        near(host(out)[i:i + 1], want, bound, f"token {i} without weights")


@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("hkv,group,t,past,window,sinks", [(16, 16, 130, 600, 0, 0), (16, 16, 131, 700, 333, 40),
                                                           (2, 16, 131, 4000, 3000, 70), (16, 16, 130, 608, 0, 0)])
def test_bad_values_among_wide_columns(gpu, what, hkv, group, t, past, window, sinks):
    r = rng(93)
    heads, n = hkv * group, past + t
    k, v = rows(r, n, hkv), rows(r, n, hkv)
    q, g = bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    bad = [n - 20, past + t // 2] + ([past - window + 10] if window else [])   # seen by some tokens each
    v[bad] = what
    c = Cache(r, BF16, 1, hkv, n)
    c.store(0, k[:past], v[:past])
    shape = c.shape(t, heads, past, window_tokens=window, sink_tokens=sinks)
    out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(ops.qwen35_compact_prefill_workspace_bytes(shape), device="cuda", dtype=torch.uint8)
    ops.qwen35_compact_attention_prefill(dev(q), dev(k[past:]), dev(v[past:]), dev(g), out, c.buf, shape, ops.DTYPE_BF16,
                                         BF16, 1, ws)
    held, got = np.stack([k.transpose(1, 0, 2), v.transpose(1, 0, 2)]).astype(np.float64), host(out)
    for i in sorted(set(some_tokens(t)) | {t - 21, t - 20, t - 19, t // 2 - 1, t // 2 + 1}):
        ok = ref.sees(past + i, window, sinks, n)
        if ok[bad].any():
            assert not np.isfinite(got[i]).any(), i
        else:
            held_i = np.where(ok[None, None, :, None], held, 0)
            want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], held_i, past + i, window, sinks)
            near(got[i:i + 1], want, bound, f"token {i}")


@pytest.mark.parametrize("dtype,layout", [(BF16, 0), (FP8, 1), (FP8, 0)])
def test_many_heads(gpu, dtype, layout):
    r = rng(94)
    c = filled(r, dtype, layout, 1000, 80, 33)
    run_prefill(c, r, 2000, 5, 33, observed=2)
    run_decode(c, r, 2000, 38, weights=True)
    run_decode(c, r, 3000, 39, window=20, sinks=3)


@pytest.mark.parametrize("dtype,layout,past", [(FP8, 1, 200), (FP8, 0, 200), (BF16, 1, 200), (BF16, 0, 500)])
def test_rows_behind_4_gib(gpu, dtype, layout, past):
    """The last positions of a cache whose planes pass 2^32 bytes, against a small cache: a window hides the rest."""
    r = rng(95)
    hkv, heads, cap, small = 4, 16, 1 << 22, 1024
    base = cap - small
    c = Cache(r, dtype, layout, hkv, small)
    shape = lambda t, p, **kw: ops.Qwen35CompactShape(t, 1, heads, hkv, D, cap, base + p, window_tokens=64, **kw)
    big = torch.empty(ops.qwen35_compact_cache_bytes(shape(1, 0), dtype), device="cuda", dtype=torch.uint8)
    assert big.numel() > 1 << 32
    k, v = rows(r, past, hkv), rows(r, past, hkv)
    ops.qwen35_compact_cache_append(dev(k), dev(v), big, shape(past, 0), ops.DTYPE_BF16, dtype, layout)
    c.want_store(0, k, v)

    def check(t, p, call, size):
        k, v, q, g = rows(r, t, hkv), rows(r, t, hkv), bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
        sh = shape(t, p)
        ws = torch.empty(size(sh), device="cuda", dtype=torch.uint8)
        out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
        call(dev(q), dev(k), dev(v), dev(g), out, big, sh, ops.DTYPE_BF16, dtype, layout, ws)
        c.want_store(p, k, v)
        want, bound, _, _ = ref.attention(q, g, c.held(p + t), p, 64)
        near(host(out), want, bound, f"{t} behind {p}")

    check(70, past, ops.qwen35_compact_attention_prefill, ops.qwen35_compact_prefill_workspace_bytes)
    check(1, past + 70, ops.qwen35_compact_attention_decode, ops.qwen35_compact_decode_workspace_bytes)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("t,past,hkv,group", [(130, 3001, 2, 16), (20, 3001, 2, 8), (300, 0, 4, 4)])
def test_prefill_in_a_graph(gpu, dtype, t, past, hkv, group):
    """Captured once and replayed with eager calls of other inputs between, on the same workspace in turn."""
    r = rng(96)
    heads = hkv * group
    c = filled(r, dtype, 1, hkv, past + t, past)
    shape = c.shape(t, heads, past, observed_tokens=2)
    ws = torch.empty(ops.qwen35_compact_prefill_workspace_bytes(shape), device="cuda", dtype=torch.uint8)
    weights = torch.zeros(hkv, past + t, device="cuda")
    inputs = [[dev(normal(r, t, m, D)) for m in (heads, hkv, hkv, heads)] for _ in range(3)]
    held = [x.clone() for x in inputs[0]]
    start = c.buf.clone()

    def go(x, out, stream=None):
        ops.qwen35_compact_attention_prefill(*x, out, c.buf, shape, ops.DTYPE_BF16, dtype, 1, ws, key_weights=weights,
                                             stream=stream)

    want = []
    for x in inputs:
        c.buf.copy_(start)
        weights.zero_()
        out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
        go(x, out)
        want.append((out, c.buf.clone(), weights.clone()))
    out = torch.empty_like(want[0][0])
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        go(held, out, stream)
    for i in (0, 2, 1, 2):
        go(inputs[(i + 1) % 3], torch.empty_like(out))
        for dst, src in zip(held, inputs[i]):
            dst.copy_(src)
        c.buf.copy_(start)
        weights.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((out, c.buf, weights), want[i]):
            assert torch.equal(got, w), i


# ------------------------------------------------------------------ values that reach no one

@pytest.mark.parametrize("t,past,window,sinks", [(40, 100, 0, 0), (40, 100, 30, 0), (40, 100, 30, 40), (1, 100, 30, 40),
                                                 (40, 96, 0, 0), (40, 96, 30, 40)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_bad_values_reach_only_the_tokens_that_see_them(gpu, t, past, window, sinks, what):
    # rows of infinite or NaN values in K (100 + 20) and V (one in the window's edge, one in the new tokens)
    r = rng(100)
    hkv, heads, n = 2, 8, past + t
    k, v = rows(r, n, hkv), rows(r, n, hkv)
    q, g = bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    bad_k, bad_v = [45], [90, past + t // 2]
    k[bad_k] = what
    v[bad_v] = what
    c = Cache(r, BF16, 1, hkv, n)
    c.store(0, k[:past], v[:past])
    shape = c.shape(t, heads, past, window_tokens=window, sink_tokens=sinks)
    out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
    call, size = ((ops.qwen35_compact_attention_prefill, ops.qwen35_compact_prefill_workspace_bytes) if t > 1 else
                  (ops.qwen35_compact_attention_decode, ops.qwen35_compact_decode_workspace_bytes))
    ws = torch.empty(size(shape), device="cuda", dtype=torch.uint8)
    call(dev(q), dev(k[past:]), dev(v[past:]), dev(g), out, c.buf, shape, ops.DTYPE_BF16, BF16, 1, ws)
    held = np.stack([k.transpose(1, 0, 2), v.transpose(1, 0, 2)]).astype(np.float64)
    got = host(out)
    for i in range(t):
        ok = ref.sees(past + i, window, sinks, n)
        if ok[bad_k].any():
            continue  # a score of infinity or NaN: what the row gives is not defined beyond being the softmax's
        if ok[bad_v].any():
            assert not np.isfinite(got[i]).any(), i
        else:
            held_i = np.where(ok[None, None, :, None], held, 0)
            want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], held_i, past + i, window, sinks)
            near(got[i:i + 1], want[:, :, :], bound, f"token {i}")


# ------------------------------------------------------------------ eviction

def weights_of(r, hkv, n):
    w = np.exp(2 * r.standard_normal((hkv, n))).astype(np.float32)
    w[r.random((hkv, n)) < 0.3] = 0          # many equal weights
    return w


@pytest.mark.parametrize("dtype,out_dtype,layout", [(BF16, BF16, 1), (BF16, FP8, 1), (FP8, FP8, 1), (FP8, FP8, 0), (BF16, BF16, 0)])
@pytest.mark.parametrize("n,keep,sinks,recent,spare", [(1, 1, 0, 0, 0), (64, 64, 3, 5, 0), (100, 33, 0, 0, 40), (100, 1, 1, 0, 3),
                                                       (333, 100, 4, 96, 0), (333, 101, 4, 96, 1), (1500, 700, 4, 64, 5), (4096, 1000, 0, 1, 0),
                                                       (4097, 4000, 5, 0, 0), (17000, 33, 1, 1, 0)])
def test_evict(gpu, dtype, out_dtype, layout, n, keep, sinks, recent, spare):
    r = rng(110 + n)
    hkv = 3
    c = filled(r, dtype, layout, hkv, n + spare, n)
    out = Cache(r, out_dtype, layout, hkv, keep + spare)
    w = np.concatenate([weights_of(r, hkv, n), np.full((hkv, spare), 9e9, np.float32)], 1)
    out_w = torch.full((hkv, keep + spare), 7.0, device="cuda")
    kept = torch.full((hkv, keep), -1, device="cuda", dtype=torch.int32)
    shape = ops.Qwen35EvictShape(hkv, D, n, n + spare, keep, keep + spare, sinks, recent)
    ws = torch.full((max(16, ops.qwen35_compact_evict_workspace_bytes(shape)),), 0xFF, device="cuda", dtype=torch.uint8)
    ops.qwen35_compact_cache_evict(c.buf, dev(w, torch.float32), out.buf, out_w, kept, shape, dtype, out_dtype, layout, ws)
    held = c.held(n)
    for h in range(hkv):
        idx = ref.keep_indices(w[h], n, keep, sinks, recent)
        assert np.array_equal(kept[h].cpu().numpy(), idx), h
        assert np.array_equal(host(out_w[h]), np.concatenate([w[h][idx], np.zeros(spare, np.float32)]))
        if out_dtype == FP8:
            one = ref.Fp8Cache(1, keep + spare)
            one.store(0, held[0, h, idx][:, None], held[1, h, idx][:, None])
            out.ref.codes[:, h, :keep] = one.codes[:, 0, :keep]
            blocks = -(-keep // 32)
            out.ref.scales[:, h, :blocks] = one.scales[:, 0, :blocks]
        else:
            out.ref[:, h, :keep] = held[:, h, idx]
    out.check("new cache")
    c.check("old cache")


@pytest.mark.parametrize("n,keep", [(16384, 200), (16385, 107), (65536, 9000), (65537, 65000), (150001, 40000)])
@pytest.mark.parametrize("few", [False, True])
def test_evict_selection_of_long_caches(gpu, n, keep, few):
    # the choice alone (rows of one head): spread weights, or a handful of different ones
    r = rng(125)
    w = weights_of(r, 2, n) if not few else r.integers(0, 4, (2, n)).astype(np.float32)
    buf = torch.zeros(ops.qwen35_compact_cache_bytes(ops.Qwen35CompactShape(1, 1, 2, 2, D, n, 0), FP8), device="cuda", dtype=torch.uint8)
    out = torch.zeros(ops.qwen35_compact_cache_bytes(ops.Qwen35CompactShape(1, 1, 2, 2, D, keep, 0), FP8), device="cuda", dtype=torch.uint8)
    out_w, kept = torch.empty(2, keep, device="cuda"), torch.empty(2, keep, device="cuda", dtype=torch.int32)
    shape = ops.Qwen35EvictShape(2, D, n, n, keep, keep, 7, 100)
    ws = torch.full((ops.qwen35_compact_evict_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    ops.qwen35_compact_cache_evict(buf, dev(w, torch.float32), out, out_w, kept, shape, FP8, FP8, 1, ws)
    for h in range(2):
        rank = w[h].astype(np.float64)
        rank[:7] = rank[n - 100:] = np.inf
        want = np.sort(np.argsort(-rank, kind="stable")[:keep])
        assert np.array_equal(kept[h].cpu().numpy(), want)
        assert np.array_equal(host(out_w[h]), w[h][want])


def test_evict_order_of_odd_weights(gpu):
    r = rng(120)
    n, keep = 12, 6
    w = np.array([[0.0, -0.0, np.nan, 1.0, np.inf, 1.0, -1.0, -np.inf, 1.0, 1e-40, 0.0, 2e-40]], np.float32)
    c, out = filled(r, BF16, 1, 1, n, n), Cache(r, BF16, 1, 1, keep)
    out_w, kept = torch.empty(1, keep, device="cuda"), torch.empty(1, keep, device="cuda", dtype=torch.int32)
    ops.qwen35_compact_cache_evict(c.buf, dev(w, torch.float32), out.buf, out_w, kept,
                                   ops.Qwen35EvictShape(1, D, n, n, keep, keep), BF16, BF16, 1)
    assert kept[0].tolist() == [2, 3, 4, 5, 8, 11]
    shape = ops.Qwen35EvictShape(1, D, n, n, 9, 9)
    out9, w9 = Cache(r, BF16, 1, 1, 9), torch.empty(1, 9, device="cuda")
    kept = torch.empty(1, 9, device="cuda", dtype=torch.int32)
    ops.qwen35_compact_cache_evict(c.buf, dev(w, torch.float32), out9.buf, w9, kept, shape, BF16, BF16, 1)
    assert kept[0].tolist() == [0, 1, 2, 3, 4, 5, 8, 9, 11]  # 0 and -0 are equal: the lower index stays


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, FP8), (FP8, FP8)])
def test_prompt_evict_decode(gpu, dtype, out_dtype):
    """A prompt with observed tokens, its cache cut to a budget, then decode steps behind a window."""
    r = rng(130)
    hkv, heads, t, keep = 4, 16, 300, 90
    c = Cache(r, dtype, 1, hkv, t)
    k, v, q, g = rows(r, t, hkv), rows(r, t, hkv), bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    w = torch.zeros(hkv, t, device="cuda")
    shape = c.shape(t, heads, 0, observed_tokens=16)
    ws = torch.empty(ops.qwen35_compact_prefill_workspace_bytes(shape), device="cuda", dtype=torch.uint8)
    out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
    ops.qwen35_compact_attention_prefill(dev(q), dev(k), dev(v), dev(g), out, c.buf, shape, ops.DTYPE_BF16, dtype, 1, ws,
                                         key_weights=w)
    c.want_store(0, k, v)
    _, _, ww, rel = ref.attention(q[-16:], g[-16:], c.held(t), t - 16, observed=16)
    near_weights(host(w), 0.0, ww, rel)
    cap = keep + 40
    small = Cache(r, out_dtype, 1, hkv, cap)
    small_w = torch.empty(hkv, cap, device="cuda")
    kept = torch.empty(hkv, keep, device="cuda", dtype=torch.int32)
    ops.qwen35_compact_cache_evict(c.buf, w, small.buf, small_w, kept,
                                   ops.Qwen35EvictShape(hkv, D, t, t, keep, cap, 4, 16), dtype, out_dtype, 1)
    held = c.held(t)
    for h in range(hkv):
        idx = ref.keep_indices(host(w)[h], t, keep, 4, 16)
        assert np.array_equal(kept[h].cpu().numpy(), idx)
        if out_dtype == FP8:
            one = ref.Fp8Cache(1, keep)
            one.store(0, held[0, h, idx][:, None], held[1, h, idx][:, None])
            small.ref.codes[:, h, :keep], small.ref.scales[:, h, :3] = one.codes[:, 0], one.scales[:, 0]
        else:
            small.ref[:, h, :keep] = held[:, h, idx]
    small.check("cut")
    for past in range(keep, keep + 12):
        run_decode(small, r, heads, past, window=60, sinks=4, weights=True)


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_decode_in_a_graph(gpu, dtype):
    """Steps captured once and replayed over growing lengths, with eager work between the replays."""
    r = rng(140)
    hkv, heads, cap, b = 4, 16, 400, 3
    caches = [filled(r, dtype, 1, hkv, cap, n) for n in (31, 250, 1)]
    lengths = torch.tensor([32, 251, 2], device="cuda", dtype=torch.int32)
    buf = torch.stack([c.buf for c in caches])
    shape = ops.Qwen35CompactShape(1, b, heads, hkv, D, cap, 0, buf.shape[1], 200, 3, 1)
    ws = torch.empty(ops.qwen35_compact_decode_workspace_bytes(shape), device="cuda", dtype=torch.uint8)
    x = [torch.zeros(b, n, D, device="cuda", dtype=torch.bfloat16) for n in (heads, hkv, hkv, heads)]
    out = torch.empty(b, heads, D, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(b, hkv, cap, device="cuda")
    eager = (buf.clone(), w.clone(), torch.empty_like(out), torch.empty_like(ws))

    def step(buf, w, out, ws, stream=None):
        ops.qwen35_compact_attention_decode(*x, out, buf, shape, ops.DTYPE_BF16, dtype, 1, ws, context_lengths=lengths,
                                            key_weights=w, stream=stream)

    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step(buf, w, out, ws, side)
    for i in range(5):
        for t, n in zip(x, (heads, hkv, hkv, heads)):
            t.copy_(dev(rows(r, b, n)))
        step(*eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[2]) and torch.equal(buf, eager[0]) and torch.equal(w, eager[1]), i
        lengths += 1


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_prompt_and_eviction_in_a_graph(gpu, dtype):
    r = rng(150)
    hkv, heads, t, keep = 4, 16, 130, 50
    c = Cache(r, dtype, 1, hkv, t)
    shape = c.shape(t, heads, 0, window_tokens=90, sink_tokens=2, observed_tokens=20)
    eshape = ops.Qwen35EvictShape(hkv, D, t, t, keep, keep, 2, 10)
    x = [torch.zeros(t, n, D, device="cuda", dtype=torch.bfloat16) for n in (heads, hkv, hkv, heads)]

    def state():
        return dict(buf=torch.zeros_like(c.buf), out=torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16),
                    w=torch.zeros(hkv, t, device="cuda"), ow=torch.empty(hkv, keep, device="cuda"),
                    kept=torch.empty(hkv, keep, device="cuda", dtype=torch.int32),
                    small=torch.zeros(ops.qwen35_compact_cache_bytes(
                        ops.Qwen35CompactShape(1, 1, heads, hkv, D, keep, 0), dtype), device="cuda", dtype=torch.uint8),
                    ws=torch.empty(max(ops.qwen35_compact_prefill_workspace_bytes(shape),
                                       ops.qwen35_compact_evict_workspace_bytes(eshape)), device="cuda", dtype=torch.uint8))

    def step(s, stream=None):
        ops.qwen35_compact_attention_prefill(*x, s["out"], s["buf"], shape, ops.DTYPE_BF16, dtype, 1, s["ws"],
                                             key_weights=s["w"], stream=stream)
        ops.qwen35_compact_cache_evict(s["buf"], s["w"], s["small"], s["ow"], s["kept"], eshape, dtype, dtype, 1, s["ws"],
                                       stream=stream)

    a, b = state(), state()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step(a, side)
    for i in range(4):
        for tns, n in zip(x, (heads, hkv, hkv, heads)):
            tns.copy_(dev(rows(r, t, n)))
        step(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for key in ("out", "w", "ow", "kept", "small", "buf"):
            assert torch.equal(a[key], b[key]), (i, key)


def test_two_streams(gpu):
    """Calls on two streams with a workspace each give what they give one after the other."""
    r = rng(160)
    hkv, heads, n = 4, 16, 2000
    sets = []
    for dtype in (BF16, FP8):
        c = filled(r, dtype, 1, hkv, n, n - 1)
        shape = c.shape(1, heads, n - 1, window_tokens=1500)
        x = [dev(rows(r, 1, m)) for m in (heads, hkv, hkv, heads)]
        ws = torch.empty(ops.qwen35_compact_decode_workspace_bytes(shape), device="cuda", dtype=torch.uint8)
        sets.append((c, shape, x, ws, torch.empty(heads * D, device="cuda", dtype=torch.bfloat16)))
    alone = []
    for c, shape, x, ws, out in sets:
        ops.qwen35_compact_attention_decode(*x, out, c.buf, shape, ops.DTYPE_BF16, c.dtype, 1, ws)
        torch.cuda.synchronize()
        alone.append(out.clone())
        out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, (c, shape, x, ws, out) in zip(streams, sets):
            ops.qwen35_compact_attention_decode(*x, out, c.buf, shape, ops.DTYPE_BF16, c.dtype, 1, ws, stream=s)
    torch.cuda.synchronize()
    for (_, _, _, _, out), want in zip(sets, alone):
        assert torch.equal(out, want)
