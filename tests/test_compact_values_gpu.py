"""The compact KV cache at values where roundings show and at the ends of their range: what the values are averaged with
sums to what the average is divided by, key weights change no output, the largest and the smallest values, infinities and NaN."""
import numpy as np
import pytest
import torch

import compact_reference as ref
from helpers import bf16, normal, rng
from raftinfer_amd import ops
from test_compact_gpu import BF16, D, FP8, WIDE, Cache, dev, filled, host, near, rows

pytestmark = pytest.mark.gpu

# (KV heads, group, tokens, past, window, sinks): few columns and many, keys whole and in ranges
SHAPES = [(2, 4, 2, 0, 0, 0), (2, 4, 40, 100, 0, 0), (1, 4, 5, 3001, 0, 0), (4, 4, 70, 333, 100, 40)] + \
    [WIDE[i] for i in (0, 1, 4, 7, 8)]


def prefill(c, x, t, heads, past, window=0, sinks=0, observed=0):
    shape = c.shape(t, heads, past, window_tokens=window, sink_tokens=sinks, observed_tokens=observed)
    ws = torch.full((ops.qwen35_compact_prefill_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    out = torch.empty(t, heads, D, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(c.hkv, c.cap, device="cuda") if observed else None
    ops.qwen35_compact_attention_prefill(*x, out, c.buf, shape, ops.DTYPE_BF16, c.dtype, c.layout, ws, key_weights=w)
    return out, w


def decode(c, x, heads, past, window=0, sinks=0, weigh=False):
    shape = c.shape(1, heads, past, window_tokens=window, sink_tokens=sinks, observed_tokens=int(weigh))
    ws = torch.full((ops.qwen35_compact_decode_workspace_bytes(shape),), 0xFF, device="cuda", dtype=torch.uint8)
    out = torch.empty(1, heads, D, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(c.hkv, c.cap, device="cuda") if weigh else None
    ops.qwen35_compact_attention_decode(*x, out, c.buf, shape, ops.DTYPE_BF16, c.dtype, c.layout, ws, key_weights=w)
    return out, w


# ------------------------------------------------------------------ an average of equal values is that value

ALIKE = 1.875  # a bf16 and an e4m3 number; its neighbours in bf16 are 2^-7 away


def alike(hkv, n):
    """Keys of score 0 and, 15 of 16, of a score whose probability is 0.9 of half a bf16 step above 1/2 of that (so
    bf16 rounds it down by 2^-8.2 of itself), and the same value at every key.  The score is the sum of the key's first four dims
    / 16, e4m3 numbers of a block's scale 2^-5."""
    rest = -16 * np.log(0.5 * (1 + 0.9 * 2.0 ** -8))
    k = np.zeros((n, hkv, D), np.float32)
    at = np.arange(n) % 16 != 0
    for i in range(4):
        digit = 0.0 if rest == 0 else 2.0 ** (max(np.floor(np.log2(abs(rest))), -11) - 3)
        part = np.round(rest / digit) * digit
        k[at, :, i] = -part
        rest -= part
    assert abs(rest) < 2.0 ** -12
    return k, np.full((n, hkv, D), ALIKE, np.float32)


def queries(t, heads):
    q = np.zeros((t, heads, D), np.float32)
    q[..., :4] = 1
    return dev(q), dev(np.full((t, heads, D), 200, np.float32))  # a gate that is 1 in f32


# The sums take n steps of 2^-24 each and the quotient two more: 2^-11.6 of the value at 5000 keys, where 2^-8.9 of
# it is half a step of the result.  So every output is the value itself.
@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("observed", [0, 1])
@pytest.mark.parametrize("hkv,group,t,past,window,sinks", SHAPES)
def test_prefill_of_equal_values(gpu, dtype, observed, hkv, group, t, past, window, sinks):
    k, v = alike(hkv, past + t)
    c = Cache(rng(1), dtype, 1, hkv, past + t)
    if past:
        c.store(0, k[:past], v[:past])
    q, g = queries(t, hkv * group)
    out, w = prefill(c, (q, dev(k[past:]), dev(v[past:]), g), t, hkv * group, past, window, sinks, observed)
    assert (host(out) == ALIKE).all()
    if observed:  # probabilities that sum to 1 a head
        total = host(w).astype(np.float64).sum(1)
        assert np.abs(total / group - 1).max() < (past + t + 64) * 2.0 ** -23


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("n,window", [(1, 0), (17, 0), (300, 0), (301, 100), (700, 0), (4001, 0), (4001, 2100)])
def test_decode_of_equal_values(gpu, dtype, weigh, n, window):
    hkv, group = 2, 8
    k, v = alike(hkv, n)
    c = Cache(rng(2), dtype, 1, hkv, n)
    if n > 1:
        c.store(0, k[:-1], v[:-1])
    q, g = queries(1, hkv * group)
    out, w = decode(c, (q, dev(k[-1:]), dev(v[-1:]), g), hkv * group, n - 1, window, 0, weigh)
    assert (host(out) == ALIKE).all()
    if weigh:
        total = host(w).astype(np.float64).sum(1)
        assert np.abs(total / group - 1).max() < (n + 64) * 2.0 ** -23


# ------------------------------------------------------------------ key weights change no output

@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hkv,group,t,past,window,sinks", SHAPES)
def test_prefill_with_weights_gives_the_same_output(gpu, dtype, hkv, group, t, past, window, sinks):
    r = rng(3)
    heads = hkv * group
    c = filled(r, dtype, 1, hkv, past + t, past)
    x = dev(normal(r, t, heads, D)), dev(rows(r, t, hkv)), dev(rows(r, t, hkv)), dev(normal(r, t, heads, D))
    start = c.buf.clone()
    plain, _ = prefill(c, x, t, heads, past, window, sinks)
    c.buf.copy_(start)
    weighed, _ = prefill(c, x, t, heads, past, window, sinks, observed=min(t, 3))
    assert torch.equal(plain, weighed)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("n,window", [(1, 0), (300, 0), (4001, 0), (4001, 2100)])
def test_decode_with_weights_gives_the_same_output(gpu, dtype, n, window):
    r = rng(4)
    hkv, heads = 2, 16
    c = filled(r, dtype, 1, hkv, n, n - 1)
    x = dev(normal(r, 1, heads, D)), dev(rows(r, 1, hkv)), dev(rows(r, 1, hkv)), dev(normal(r, 1, heads, D))
    start = c.buf.clone()
    plain, _ = decode(c, x, heads, n - 1, window)
    c.buf.copy_(start)
    weighed, _ = decode(c, x, heads, n - 1, window, weigh=True)
    assert torch.equal(plain, weighed)


@pytest.mark.parametrize("what", [np.inf, -np.inf])
@pytest.mark.parametrize("n,at,k_size", [(1, 0, 1), (40, 3, 0), (40, 39, 1), (700, 500, 1), (4001, 17, 0)])
def test_decode_of_infinite_values(gpu, what, n, at, k_size):
    """A seen value of infinity gives infinity, also to keys whose probability is the largest (equal keys: all are)."""
    r = rng(5)
    hkv, heads = 2, 16
    k, v = bf16(normal(r, n, hkv, D) * k_size), rows(r, n, hkv)
    v[at, :, 5] = what
    c = Cache(r, BF16, 1, hkv, n)
    if n > 1:
        c.store(0, k[:-1], v[:-1])
    out, _ = decode(c, (dev(normal(r, 1, heads, D)), dev(k[-1:]), dev(v[-1:]), dev(normal(r, 1, heads, D))), heads, n - 1)
    got = host(out)
    assert (got[..., 5] == what).all() and np.isfinite(np.delete(got, 5, -1)).all()


# ------------------------------------------------------------------ values up to the largest

MOST = 255 * 2.0 ** 120  # of bf16
TOP = 240 * 2.0 ** 120   # of an 8-bit cache: the next code would stand for 2^128


def below_top(x, dtype):
    return np.where(np.isfinite(x), np.clip(x, -TOP, TOP), x) if dtype == FP8 else x


def append(c, past, k, v):
    ops.qwen35_compact_cache_append(dev(k), dev(v), c.buf, c.shape(len(k), c.hkv, past), ops.DTYPE_BF16, c.dtype, c.layout)
    c.want_store(past, below_top(k, c.dtype), below_top(v, c.dtype))


@pytest.mark.parametrize("layout", [0, 1])
def test_store_of_the_largest_values(gpu, layout):
    r = rng(6)
    c = Cache(r, FP8, layout, 2, 100)
    k, v = rows(r, 70, 2), rows(r, 70, 2)
    k[3, 0, :4] = [MOST, -MOST, TOP, 248 * 2.0 ** 120]
    k[4, 0, :2] = [np.inf, np.nan]
    k[5, 1, 7] = 224 * 2.0 ** 120       # under the same scale, and no code above 224
    v[40, 1, 9] = -249 * 2.0 ** 120
    v[41, 0, 3] = 2.0 ** 126            # a scale below the largest
    append(c, 0, k[:35], v[:35])
    c.check("first")
    append(c, 35, k[35:], v[35:])
    c.check("second")
    held = c.held(70)
    assert np.nanmax(np.abs(held)) == TOP


def largest(r, t, past, hkv, heads, v_at, k_at):
    """A value of the largest size at the keys v_at, whose scores lie 2^7 above those of the keys before; a largest number
    at the keys k_at, in a dim that no query looks at."""
    n = past + t
    k, v = bf16(normal(r, n, hkv, D) / 64), rows(r, n, hkv)
    q = np.zeros((t, heads, D), np.float32)
    q[..., 0] = 4
    k[v_at, :, 0] = 19.5   # 19.5 * 4 / 16 / ln 2 = 7.03
    v[v_at, :, 5], v[v_at, :, 6] = MOST, -MOST
    k[k_at, :, 9] = MOST
    return q, k, v, bf16(normal(r, t, heads, D))


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hkv,group,t,past,window,sinks", SHAPES[1:])
def test_prefill_of_the_largest_values(gpu, dtype, hkv, group, t, past, window, sinks):
    r = rng(7)
    heads, n = hkv * group, past + t
    q, k, v, g = largest(r, t, past, hkv, heads, [past + t // 2], [n // 7])
    c = Cache(r, dtype, 1, hkv, n)
    if past:
        append(c, 0, k[:past], v[:past])
    out, _ = prefill(c, (dev(q), dev(k[past:]), dev(v[past:]), dev(g)), t, heads, past, window, sinks)
    c.want_store(past, below_top(k[past:], dtype), below_top(v[past:], dtype))
    c.check()
    got = host(out)
    assert np.isfinite(got).all()
    for i in sorted({0, t // 2 - 1, t // 2, t // 2 + 1, t - 2, t - 1} & set(range(t))):
        want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], c.held(past + i + 1), past + i, window, sinks)
        near(got[i:i + 1], want, bound, f"token {i}")


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("n,at", [(1, 0), (40, 39), (40, 7), (700, 500), (4001, 4000), (4001, 300)])
def test_decode_of_the_largest_values(gpu, dtype, n, at):
    r = rng(8)
    hkv, heads = 2, 16
    q, k, v, g = largest(r, 1, n - 1, hkv, heads, [at], [n // 7])
    c = Cache(r, dtype, 1, hkv, n)
    if n > 1:
        append(c, 0, k[:-1], v[:-1])
    out, _ = decode(c, (dev(q), dev(k[-1:]), dev(v[-1:]), dev(g)), heads, n - 1)
    c.want_store(n - 1, below_top(k[-1:], dtype), below_top(v[-1:], dtype))
    c.check()
    want, bound, _, _ = ref.attention(q, g, c.held(n), n - 1)
    near(host(out), want, bound)


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_evict_of_the_largest_values(gpu, dtype):
    r = rng(9)
    hkv, n, keep = 2, 200, 90
    k, v = rows(r, n, hkv), rows(r, n, hkv)
    k[50, 0, 3], v[51, 1, 4] = MOST, -MOST
    c, out = Cache(r, dtype, 1, hkv, n), Cache(r, FP8, 1, hkv, keep)
    append(c, 0, k, v)
    w = np.zeros((hkv, n), np.float32)
    w[:, 30:120] = 1
    out_w, kept = torch.empty(hkv, keep, device="cuda"), torch.empty(hkv, keep, device="cuda", dtype=torch.int32)
    ops.qwen35_compact_cache_evict(c.buf, dev(w, torch.float32), out.buf, out_w, kept,
                                   ops.Qwen35EvictShape(hkv, D, n, n, keep, keep), dtype, FP8, 1)
    assert (kept.cpu().numpy() == np.arange(30, 120)).all()
    held = below_top(c.held(n)[:, :, 30:120], FP8)
    out.ref.store(0, held[0].transpose(1, 0, 2), held[1].transpose(1, 0, 2))
    out.check()
    assert np.nanmax(np.abs(out.held(keep))) == TOP


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("call,n", [("decode", 40), ("decode", 700), ("decode", 4001), ("few", 200), ("many", 700)])
def test_small_values(gpu, dtype, call, n):
    """Values of 1e-36, under the least scale of an 8-bit cache."""
    r = rng(10)
    hkv, heads, t = (16, 256, 130) if call == "many" else (2, 16, 1 if call == "decode" else 30)
    k, v = rows(r, n, hkv), bf16(rows(r, n, hkv, heavy=False) * 1e-36)
    q, g = bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    c = Cache(r, dtype, 1, hkv, n)
    c.store(0, k[:n - t], v[:n - t])
    x = dev(q), dev(k[n - t:]), dev(v[n - t:]), dev(g)
    out, _ = decode(c, x, heads, n - 1) if call == "decode" else prefill(c, x, t, heads, n - t)
    c.want_store(n - t, k[n - t:], v[n - t:])
    for i in sorted({0, t // 2, t - 1}):
        want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], c.held(n - t + i + 1), n - t + i)
        # (a code below 2^-6 and a product or result below 2^-126 may be rounded to a multiple of 2^-133)
        near(host(out)[i:i + 1], want, bound + 2.0 ** -132, f"token {i}")


# ------------------------------------------------------------------ the largest cache

def test_the_largest_cache(gpu):
    """2^28 positions of equal keys and values, full: every weight is 2^-28 and the output the value.  (Sums of equal powers
    of two are exact.)"""
    cap = 1 << 28
    torch.cuda.empty_cache()
    shape = ops.Qwen35CompactShape(1, 1, 1, 1, D, cap, cap - 1, observed_tokens=1)
    size = ops.qwen35_compact_cache_bytes(shape, FP8)
    if torch.cuda.mem_get_info()[0] < size + (8 << 30):
        pytest.skip(f"needs {size >> 30} GiB of GPU memory")
    buf = torch.full((size,), 0x38, device="cuda", dtype=torch.uint8)   # the code of 1
    buf[2 * cap * D:].view(torch.float32).fill_(1)
    q, one = (torch.full((1, 1, D), x, device="cuda", dtype=torch.bfloat16) for x in (0, 1))
    gate = torch.full((1, 1, D), 200, device="cuda", dtype=torch.bfloat16)
    for call, need in ((ops.qwen35_compact_attention_prefill, ops.qwen35_compact_prefill_workspace_bytes),
                       (ops.qwen35_compact_attention_decode, ops.qwen35_compact_decode_workspace_bytes)):
        ws = torch.empty(need(shape), device="cuda", dtype=torch.uint8)
        out, w = torch.zeros(1, 1, D, device="cuda", dtype=torch.bfloat16), torch.zeros(cap, device="cuda")
        call(q, one, one, gate, out, buf, shape, ops.DTYPE_BF16, FP8, 1, ws, key_weights=w)
        torch.cuda.synchronize()
        assert (out == 1).all(), call
        assert (w == 2.0 ** -28).all(), call
        del ws, w
    del buf
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ NaN codes reach only the tokens that see them

@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hkv,group,t,past,window,sinks", [
    (2, 4, 40, 100, 0, 0), (2, 4, 40, 100, 30, 0), (2, 4, 40, 100, 30, 40), (2, 4, 40, 96, 0, 0), (2, 4, 1, 100, 30, 40),
    (2, 8, 20, 3001, 2900, 0), (16, 16, 130, 600, 0, 0), (16, 16, 131, 700, 333, 40), (2, 16, 131, 4000, 3000, 70)])
def test_bad_values_in_8_bit(gpu, layout, what, hkv, group, t, past, window, sinks):
    """Rows of infinite or NaN values are stored as NaN: in K at 45, in V among the new tokens, at a window's edge and
    where no window reaches."""
    r = rng(11)
    heads, n = hkv * group, past + t
    k, v = rows(r, n, hkv), rows(r, n, hkv)
    q, g = bf16(normal(r, t, heads, D)), bf16(normal(r, t, heads, D))
    bad_k = [45] if window and sinks < 45 else []
    bad_v = sorted({past + t // 2, n - 1} | ({past - window + t // 2, past - window - 3} if window else set()))
    k[bad_k] = what
    v[bad_v, 0] = what     # all of a row, and of another head one value
    v[bad_v, 1, 77] = what
    c = Cache(r, FP8, layout, hkv, n)
    c.store(0, k[:past], v[:past])
    x = dev(q), dev(k[past:]), dev(v[past:]), dev(g)
    out, _ = prefill(c, x, t, heads, past, window, sinks) if t > 1 else decode(c, x, heads, past, window, sinks)
    c.want_store(past, k[past:], v[past:])
    c.check()
    got = host(out)
    for i in sorted({0, 1, t // 2 - 1, t // 2, t // 2 + 1, t - 2, t - 1} & set(range(t))):
        ok = ref.sees(past + i, window, sinks, n)
        seen_k, seen_v = ok[bad_k].any(), ok[bad_v].any()
        held = np.where(ok[None, None, :, None], c.held(n), 0)
        clean = np.nan_to_num(held, nan=0.0)
        want, bound, _, _ = ref.attention(q[i:i + 1], g[i:i + 1], clean, past + i, window, sinks)
        bad = np.zeros((heads, D), bool)
        if seen_k:
            bad[:] = True
        if seen_v:
            bad[:group] = True
            bad[group:2 * group, 77] = True
        assert np.isnan(got[i][bad]).all(), i
        near(got[i][~bad], want[0][~bad], bound[0][~bad], f"token {i}")


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("n,at,window", [(1, 0, 0), (40, 39, 0), (40, 7, 0), (40, 7, 20), (700, 650, 0), (4001, 3990, 0), (4001, 300, 2000)])
def test_decode_of_bad_values_in_8_bit(gpu, layout, n, at, window):
    r = rng(12)
    hkv, heads = 2, 16
    k, v = rows(r, n, hkv), rows(r, n, hkv)
    v[at, 1, 200] = np.nan
    c = Cache(r, FP8, layout, hkv, n)
    if n > 1:
        c.store(0, k[:-1], v[:-1])
    q, g = bf16(normal(r, 1, heads, D)), bf16(normal(r, 1, heads, D))
    out, w = decode(c, (dev(q), dev(k[-1:]), dev(v[-1:]), dev(g)), heads, n - 1, window, weigh=True)
    c.want_store(n - 1, k[-1:], v[-1:])
    c.check()
    seen = ref.sees(n - 1, window, 0, n)
    want, bound, ww, rel = ref.attention(q, g, np.nan_to_num(c.held(n)), n - 1, window, 0, 1)
    got, bad = host(out), np.zeros((1, heads, D), bool)
    bad[0, heads // 2:, 200] = seen[at]
    assert np.isnan(got[bad]).all()
    near(got[~bad], want[~bad], bound[~bad])
    near(host(w), ww, ww * rel + 2.0 ** -23 * ww + 1e-38, "weights")
