"""Rotary positions and the paged KV cache on the GPU, against the 64-bit reference."""
import dataclasses

import numpy as np
import pytest
import torch

import paged_reference as ref
from raftinfer_amd import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
P = ops.Qwen35PagedShape


def wide(t):
    return t.detach().cpu().double().numpy()


class Batch:
    """A ragged batch over a shuffled pool.  each: (new tokens, context) of every sequence; places that no token may read
    hold NaN, table entries that no call may use hold garbage."""

    def __init__(self, each, kv_heads=4, group=4, page=16, head_major=True, window=0, gate=True, seed=0, lead=0, tail=0, spare=2,
                 decode=False, scale=1.0):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.each, self.page, self.head_major, self.window = each, page, head_major, window
        self.kv_heads, self.group, self.decode = kv_heads, group, decode
        heads = kv_heads * group
        self.rows = lead + sum(n for n, _ in each) + tail
        need = [-(-c // page) for _, c in each]
        pool = sum(need) + spare
        starts = np.concatenate([[0], np.cumsum([n for n, _ in each])]) + lead
        self.starts_host = starts
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor([c for _, c in each], dtype=torch.int32, device="cuda")
        where = torch.randperm(pool, generator=g, device="cuda", dtype=torch.int32).cpu().numpy()
        width = max(max(need), 1) + 1
        table = np.random.default_rng(seed).integers(-2 ** 31, 2 ** 31, (len(each), width)).astype(np.int32)
        shape = (pool, 2, kv_heads, page, 256) if head_major else (pool, 2, page, kv_heads, 256)
        pages = torch.full(shape, float("nan"), device="cuda", dtype=BF)
        taken = 0
        for i, ((n, c), k) in enumerate(zip(each, need)):
            lo = max(0, c - n + 1 - window) if window else 0
            for p in range(k):
                if (p + 1) * page <= lo:
                    taken += 1
                    continue  # in front of the window: the entry names no page, the page holds NaN
                table[i, p] = where[taken]
                a, e = max(lo - p * page, 0), min(c - p * page, page)
                x = torch.randn(2, kv_heads, e - a, 256, generator=g, device="cuda") * scale
                x *= 1 + 7 * (torch.rand(2, kv_heads, e - a, 1, generator=g, device="cuda") < 0.02)
                at = pages[int(where[taken])]
                if head_major:
                    at[:, :, a:e] = x.to(BF)
                else:
                    at[:, a:e] = x.transpose(1, 2).to(BF)
                taken += 1
        self.pages, self.table = pages, torch.tensor(table, device="cuda")
        self.q = torch.randn(self.rows, heads, 256, generator=g, device="cuda").to(BF)
        self.gate = torch.randn(self.rows, heads, 256, generator=g, device="cuda").to(BF) if gate else None
        self.out = torch.full((self.rows, heads, 256), 7.0, device="cuda", dtype=BF)
        self.shape = P(self.rows, len(each), heads, kv_heads, 256, pool, page, width, max(max(c for _, c in each), 1), window)

    def workspace(self):
        size = ops.qwen35_paged_decode_workspace_bytes if self.decode else ops.qwen35_paged_prefill_workspace_bytes
        return torch.full((max(size(self.shape), 16),), 0xFF, device="cuda", dtype=torch.uint8)

    def call(self, workspace=None, **kw):
        ws = self.workspace() if workspace is None else workspace
        layout = ops.HEAD_MAJOR if self.head_major else ops.TOKEN_MAJOR
        shape = kw.pop("shape", self.shape)
        if self.decode:
            ops.qwen35_paged_attention_decode(self.q, self.gate, self.out, self.pages, self.table, self.lengths, ws, shape, layout, **kw)
        else:
            ops.qwen35_paged_attention_prefill(self.q, self.gate, self.out, self.pages, self.table, self.starts, self.lengths, ws, shape,
                                               layout, **kw)
        return self.out

    def want(self, i):
        """(rows, output, tolerance) of sequence i."""
        n, c = self.each[i]
        a = int(self.starts_host[i])
        lo = max(0, c - n + 1 - self.window) if self.window else 0
        table = self.table[i].cpu().numpy().copy()
        table[:lo // self.page] = 0
        kv = ref.rows_of(wide(self.pages), table, c, self.page, self.head_major)
        gate = None if self.gate is None else wide(self.gate[a:a + n])
        out, spread, reach = ref.attention(wide(self.q[a:a + n]), gate, kv, c, self.window)
        return slice(a, a + n), out, ref.tolerance(out, spread, reach)

    def check(self, only=None):
        torch.cuda.synchronize()
        got = wide(self.out)
        touched = np.zeros(self.rows, bool)
        for i, (n, _) in enumerate(self.each):
            if n == 0 or (only is not None and i not in only):
                continue
            rows, want, tol = self.want(i)
            touched[rows] = True
            assert np.array_equal(np.isnan(got[rows]), np.isnan(want)), i
            fine = np.isfinite(want)
            assert np.array_equal(got[rows][~fine], want[~fine], equal_nan=True), i
            off = np.abs(got[rows] - want)[fine] - tol[fine]
            assert (off <= 0).all(), (i, self.each[i], off.max())
        if only is None:
            assert (got[~touched] == 7).all(), "rows of no sequence were written"


def errors():
    return ops.consume_capacity_errors()


# ------------------------------------------------------------------- rotary

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, BF])
@pytest.mark.parametrize("rows,heads,dim,rotary", [(1, 16, 256, 64), (37, 3, 256, 256), (5, 1, 128, 32), (9, 5, 80, 20), (3, 2, 96, 96),
                                                   (2, 7, 64, 16), (1, 1, 2, 2), (4, 70, 256, 128), (2, 3, 1000, 400), (11, 2, 33, 30),
                                                   (3, 4, 512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [None, "own", "f32"])
def test_rotary(gpu, dtype, rows, heads, dim, rotary, interleaved, norm):
    g = torch.Generator(device="cuda").manual_seed(rows * dim)
    x = torch.randn(rows, heads, 2, dim, generator=g, device="cuda").to(dtype)[:, :, 1]  # strided
    w = None if norm is None else (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(dtype if norm == "own" else torch.float32)
    positions = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
    positions[0] = -1  # 2^32 - 1 as uint32
    freq, magnitude = ops.qwen35_rotary_frequencies(rotary, 1e7, ops.SCALING_BY_PAIR, 4.0, 32768.0)
    out = torch.full((heads, rows, dim), 9.0, device="cuda", dtype=dtype).transpose(0, 1)
    shape = ops.Qwen35RotaryShape(rows, heads, dim, rotary, interleaved, magnitude)
    f = torch.tensor(freq, dtype=torch.float64, device="cuda")
    ops.qwen35_rotary(x, w, out, positions, f, shape, 1e-6)
    torch.cuda.synchronize()
    want = ref.rotate(wide(x), None if w is None else wide(w), positions.cpu().numpy().view(np.uint32), freq, magnitude, interleaved, 1e-6)
    # sizes of a pair bound its two results; 32 bits: a norm's sum of dim squares, the reduced angle (up to pi, half a step of
    # which is pi 2^-24) and its sine and cosine (2 steps), the products and the sum; the result is rounded once
    pair = np.abs(ref.rotate(np.abs(wide(x)), None if w is None else np.abs(wide(w)), [0] * rows, freq, 1.0, interleaved, 1e-6))
    n = rotary // 2
    i, j = (np.arange(0, rotary, 2), np.arange(1, rotary, 2)) if interleaved else (np.arange(n), np.arange(n, rotary))
    size = pair.copy()
    size[..., i] = size[..., j] = (pair[..., i] + pair[..., j]) * magnitude
    half = torch.finfo(dtype).eps / 2
    tol = half * np.abs(want) + size * 2.0 ** -24 * (12 + (0 if w is None else dim / 2 + 4)) + torch.finfo(dtype).smallest_normal * half
    assert (np.abs(wide(out) - want) <= tol).all()
    # in place
    same = x.clone() if dtype != BF else x
    ops.qwen35_rotary(same, w, same, positions, f, shape, 1e-6)
    torch.cuda.synchronize()
    assert torch.equal(same, out)


def test_rotary_at_zero_is_the_norm(gpu):
    x = torch.randn(3, 4, 256, device="cuda").to(BF)
    out = torch.empty_like(x)
    f = torch.tensor(ops.qwen35_rotary_frequencies(64, 1e7)[0], dtype=torch.float64, device="cuda")
    ops.qwen35_rotary(x, None, out, torch.zeros(3, dtype=torch.int32, device="cuda"), f, ops.Qwen35RotaryShape(3, 4, 256, 64), 1e-6)
    torch.cuda.synchronize()
    assert torch.equal(x, out)


def test_rotary_matches_the_producer(gpu):
    """The half layout without scaling is qwen35_qk_norm_rope at consecutive positions (both round once from 32 bits)."""
    x, w = torch.randn(50, 4, 256, device="cuda").to(BF), (1 + 0.1 * torch.randn(256, device="cuda")).to(BF)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.qwen35_qk_norm_rope(x, w, a, ops.QkNormRopeShape(50, 4, 256, 64, 1000, 1e7), 1e-6, 3, 3)
    f = torch.tensor(ops.qwen35_rotary_frequencies(64, 1e7)[0], dtype=torch.float64, device="cuda")
    ops.qwen35_rotary(x, w, b, torch.arange(1000, 1050, dtype=torch.int32, device="cuda"), f, ops.Qwen35RotaryShape(50, 4, 256, 64), 1e-6)
    torch.cuda.synchronize()
    # one step of bf16 where the 32-bit values straddle a border
    assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * a.float().abs() + 1e-6).all() and (a == b).float().mean() > 0.999


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("each,page,kv_heads,group,rotary,interleaved,norm", [
    ([(1, 1)], 16, 4, 4, 64, False, "bf16"), ([(5, 5), (1, 300), (0, 40), (33, 50)], 16, 4, 4, 64, False, "bf16"),
    ([(17, 100), (1, 49)], 48, 3, 5, 256, True, "f32"), ([(64, 64)], 64, 1, 16, 32, False, None), ([(3, 10), (2, 2)], 32, 5, 1, 0, False, "q"),
    ([(1, i + 1) for i in range(70)], 16, 2, 2, 128, True, "k")])
def test_append(gpu, each, page, kv_heads, group, rotary, interleaved, norm, head_major):
    b = Batch(each, kv_heads, group, page, head_major, seed=3, lead=2, tail=3)
    before = b.pages.clone()
    g, heads = b.g, kv_heads * group
    proj = torch.randn(b.rows, heads, 2, 256, generator=g, device="cuda").to(BF)
    k = torch.randn(kv_heads, b.rows, 256, generator=g, device="cuda").to(BF).transpose(0, 1)
    v = torch.randn(b.rows, kv_heads + 1, 256, generator=g, device="cuda").to(BF)[:, 1:]
    wq, wk = ((1 + 0.1 * torch.randn(256, generator=g, device="cuda")).to(torch.float32 if norm == "f32" else BF) for _ in (0, 1))
    if norm in (None, "k"):
        wq = None
    if norm in (None, "q"):
        wk = None
    freq, magnitude = ops.qwen35_rotary_frequencies(rotary, 1e7, ops.SCALING_BY_TURNS, 8.0, 100.0) if rotary else ([], 1.0)
    f = torch.tensor(freq, dtype=torch.float64, device="cuda") if rotary else None
    out = torch.full((b.rows, heads, 256), 7.0, device="cuda", dtype=BF)
    layout = ops.HEAD_MAJOR if head_major else ops.TOKEN_MAJOR
    r = ops.Qwen35PagedRotary(rotary, interleaved, magnitude, 1e-6)
    errors()
    ops.qwen35_paged_cache_append(proj[:, :, 0], k, v, out, b.pages, b.table, b.starts, b.lengths, f, wq, wk, b.shape, r, layout)
    torch.cuda.synchronize()
    assert errors() == 0
    expect, seen = wide(before), np.zeros(b.rows, bool)
    got_q, got_pages = wide(out), wide(b.pages)
    close = lambda x, y, ref_x: (np.abs(x - y) <= ref.HALF_BF16 * np.abs(y) + 2e-4 * np.abs(ref_x).max()).all()  # noqa: E731
    table = b.table.cpu().numpy()
    for i, (n, c) in enumerate(each):
        a = int(b.starts_host[i])
        seen[a:a + n] = True
        at = np.arange(c - n, c)
        turn = lambda x, w: ref.rotate(wide(x[a:a + n]), None if w is None else wide(w), at, freq, magnitude, interleaved, 1e-6)  # noqa: E731
        if n:
            y = turn(proj[:, :, 0], wq)
            # (32 bits: 256 squares and a few roundings, 2e-5 of the largest value; 2e-4 leaves the angle's)
            assert close(got_q[a:a + n], y, y)
            y = turn(k, wk)
            for t in range(n):
                page_at, in_page = table[i, at[t] // page], at[t] % page
                where = (page_at, slice(None), slice(None), in_page) if head_major else (page_at, slice(None), in_page)
                assert close(got_pages[where][0], y[t], y) and np.array_equal(got_pages[where][1], wide(v[a + t]))
                expect[where] = got_pages[where]
    assert (got_q[~seen] == 7).all()
    assert np.array_equal(got_pages, expect, equal_nan=True), "other places were written"
    # without queries: the same pages
    again = before.clone()
    ops.qwen35_paged_cache_append(None, k, v, None, again, b.table, b.starts, b.lengths, f, None, wk, b.shape, r, layout)
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), b.pages.view(torch.int16))


def test_append_refuses_bad_sequences_on_the_device(gpu):
    b = Batch([(3, 20), (3, 20), (3, 20), (3, 20), (3, 20)], seed=1)
    b.lengths[0] = 2                              # below its new tokens
    b.lengths[1] = b.shape.max_context_tokens + 1
    b.table[2, 1] = b.shape.pages                 # the page of its positions 17 .. 19
    b.table[3, 0] = -1                            # not needed: nothing is stored there
    b.starts[5] = 99                              # behind the call's rows
    k, v = (torch.randn(b.rows, 4, 256, device="cuda").to(BF) for _ in (0, 1))
    before, out = b.pages.clone(), torch.full_like(b.q, 7.0)
    errors()
    ops.qwen35_paged_cache_append(b.q, k, v, out, b.pages, b.table, b.starts, b.lengths, None, None, None, b.shape,
                                  ops.Qwen35PagedRotary(0), ops.HEAD_MAJOR)
    torch.cuda.synchronize()
    assert errors() >= 4
    page = int(b.table[3, 1])
    assert torch.equal(b.pages[page, 0, :, 1:4].transpose(0, 1), k[9:12]) and torch.equal(b.pages[page, 1, :, 1:4].transpose(0, 1), v[9:12])
    b.pages[page] = before[page]
    assert torch.equal(b.pages.view(torch.int16), before.view(torch.int16))
    assert torch.equal(out[9:12], b.q[9:12]) and (out[:6] == 7).all() and (out[12:] == 7).all()


# ---------------------------------------------------------------- attention

RAGGED = [(1, 1), (2, 2), (0, 5), (16, 16), (17, 33), (1, 300), (40, 41), (5, 64)]


@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("window", [0, 1, 20])
def test_prefill_ragged(gpu, page, head_major, window):
    b = Batch(RAGGED, page=page, head_major=head_major, window=window, lead=1, tail=2, seed=page)
    b.call()
    b.check()
    assert errors() == 0


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 16), (2, 3), (5, 7), (8, 2), (3, 12)])
def test_prefill_heads(gpu, kv_heads, group):
    b = Batch([(9, 40), (33, 70)], kv_heads, group, seed=group, gate=group != 3)
    b.call()
    b.check()


@pytest.mark.parametrize("n,c", [(1, 1), (15, 15), (31, 32), (32, 32), (33, 33), (64, 1000), (130, 700), (300, 300), (3, 1600), (200, 201)])
@pytest.mark.parametrize("window", [0, 97])
def test_prefill_lengths(gpu, n, c, window):
    b = Batch([(n, c)], window=window, seed=n)
    b.call()
    b.check()


@pytest.mark.parametrize("each", [[(1, 1)], [(1, 15)], [(1, 16)], [(1, 17)], [(1, 3000)], [(1, c) for c in (1, 2, 700, 33, 64, 65, 1500)],
                                  [(1, 7 * i + 1) for i in range(80)]])
@pytest.mark.parametrize("page,head_major,window", [(16, True, 0), (80, False, 0), (32, True, 50)])
def test_decode(gpu, each, page, head_major, window):
    b = Batch(each, page=page, head_major=head_major, window=window, decode=True, seed=len(each), gate=window == 0)
    b.call()
    b.check()
    assert errors() == 0


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 16), (2, 3), (5, 7), (32, 1)])
def test_decode_heads(gpu, kv_heads, group):
    b = Batch([(1, 100), (1, 9)], kv_heads, group, decode=True, seed=group)
    b.call()
    b.check()


def test_decode_leaves_unused_rows(gpu):
    b = Batch([(1, 50), (1, 40), (1, 30)], decode=True, seed=5)
    b.lengths[1] = 0
    b.call()
    b.check(only=(0, 2))
    assert (b.out[1] == 7).all() and errors() == 0


@pytest.mark.parametrize("decode", [True, False])
def test_bad_sequences_are_nan_and_counted(gpu, decode):
    n = 1 if decode else 3
    b = Batch([(n, 60), (n, 70), (n, 80), (n, 90), (n, 100)], decode=decode, seed=8)
    top = b.shape.max_context_tokens
    b.lengths[1] = top + 1
    b.table[3, 2] = b.shape.pages
    if not decode:
        b.lengths[0] = 2          # below its new tokens
        b.starts[5] = 1000        # behind the call's rows
    errors()
    b.call()
    b.check(only=(2,) if not decode else (0, 2, 4))
    assert errors() >= (2 if decode else 4)
    bad = [1, 3] if decode else [0, 1, 3, 4]
    for i in bad:
        assert torch.isnan(b.out[n * i:n * i + n]).all(), i


def test_falling_starts_write_nothing_else(gpu):
    b = Batch([(4, 30), (4, 30), (4, 30)], seed=2, tail=4)
    b.starts[1] = 9  # sequence 0 takes rows 0 .. 8, 1 falls from 9 to 8
    b.lengths[0] = 30
    errors()
    b.call()
    torch.cuda.synchronize()
    rows, want, tol = b.want(2)
    assert (np.abs(wide(b.out[9:12]) - want[1:]) <= tol[1:]).all()
    assert errors() >= 1 and (b.out[12:] == 7).all()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_odd_values_reach_only_who_sees_them(gpu, decode, value):
    """An infinite or NaN V value of a seen key goes to the tokens that see it, and to no other; so do NaN keys."""
    b = Batch([(1, 40), (1, 70)] if decode else [(20, 40), (45, 70), (3, 16)], decode=decode, seed=4, scale=0.2)
    for i, j in ((0, 39), (1, 60), (1, 3)):
        page, at = int(b.table[i, j // 16]), j % 16
        b.pages[page, 1, i, at, 17 + i] = value
    b.call()
    b.check()
    b.pages[int(b.table[0, 2]), 0, 1, 35 - 32] = float("nan")
    b.out.fill_(7)
    b.call()
    b.check()


def test_strided_tensors(gpu):
    """Query and gate as the projection leaves them, [rows][heads][query, gate][256]; heads-first output."""
    b = Batch([(20, 50), (3, 9)], seed=6)
    proj = torch.stack((b.q, b.gate), 2).contiguous()
    b.q, b.gate = proj[:, :, 0], proj[:, :, 1]
    b.out = torch.full((16, b.rows, 256), 7.0, device="cuda", dtype=BF).transpose(0, 1)
    b.call()
    b.check()


def test_another_stream_and_two_at_once(gpu):
    a, b = Batch([(30, 400)], seed=1), Batch([(1, 500), (1, 2000)], seed=2, decode=True)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    wa, wb = a.workspace(), b.workspace()
    torch.cuda.synchronize()
    for _ in range(5):
        a.call(wa, stream=s)
        b.call(wb, stream=t)
    torch.cuda.synchronize()
    a.check()
    b.check()


def test_shared_pages(gpu):
    """Two sequences whose first pages are the same."""
    b = Batch([(2, 64), (3, 60)], seed=9)
    b.table[1, :3] = b.table[0, :3]
    b.call()
    b.check()


def test_largest_scores_and_values(gpu):
    """Probabilities stay at most 1 while the maximum grows along the keys: 400 values of 2^119 sum to less than 2^128."""
    b = Batch([(1, 400)], decode=True, seed=3)
    top = 2.0 ** 119
    table = b.table.cpu().numpy()
    for j in range(400):
        b.pages[int(table[0, j // 16]), 0, :, j % 16] = b.q[0, ::4].float().mul(j / 400).to(BF)
        b.pages[int(table[0, j // 16]), 1, :, j % 16] = top
    b.gate.fill_(100.0)
    b.call()
    torch.cuda.synchronize()
    assert (b.out == top).all()


@pytest.mark.parametrize("decode", [True, False])
def test_graph_replays(gpu, decode):
    """One captured graph follows the device's lengths, tables and starts, also between eager calls on another workspace."""
    each = [(1, 900), (1, 33)] if decode else [(40, 900), (7, 33)]
    b = Batch(each, decode=decode, seed=11)
    b.shape = dataclasses.replace(b.shape, max_context_tokens=b.shape.table_pages * b.page)
    ws, eager_ws = b.workspace(), b.workspace()
    b.call(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu):
        b.call(ws, stream=torch.cuda.current_stream())
    for step in range(4):
        b.out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        b.check()
        got = b.out.clone()
        b.out.fill_(7)
        b.call(eager_ws)
        torch.cuda.synchronize()
        assert torch.equal(got, b.out)
        # the longer sequence ends earlier
        n, c = b.each[0]
        c = c // 3 + n
        b.each = [(n, c)] + b.each[1:]
        b.lengths[0] = c


def test_step_of_a_server(gpu):
    """Append and attention over three steps (prompts, chunks with single tokens, single tokens) equal attention over the
    whole sequences at once."""
    g = torch.Generator(device="cuda").manual_seed(5)
    total, page, hkv, hq = [75, 40, 130], 16, 4, 16
    x = [[torch.randn(t, h, 256, generator=g, device="cuda").to(BF) for h in (hq, hkv, hkv, hq)] for t in total]
    freq, m = ops.qwen35_rotary_frequencies(64, 1e7, ops.SCALING_BY_PAIR, 2.0, 64.0)
    f = torch.tensor(freq, dtype=torch.float64, device="cuda")
    wq, wk = ((1 + 0.1 * torch.randn(256, generator=g, device="cuda")).to(BF) for _ in (0, 1))
    table = torch.randperm(30, generator=g, device="cuda", dtype=torch.int32).view(3, 10)
    pages = torch.full((30, 2, hkv, page, 256), float("nan"), device="cuda", dtype=BF)
    done, outs = [0, 0, 0], [[], [], []]
    for new in ([30, 40, 1], [44, 0, 128], [1, 0, 1]):
        rows, live = sum(new), [i for i in range(3) if new[i]]
        parts = [torch.cat([x[i][k][done[i]:done[i] + new[i]] for i in range(3)]) for k in range(4)]
        done = [d + n for d, n in zip(done, new)]
        starts = torch.tensor([0, new[0], new[0] + new[1], rows], dtype=torch.int32, device="cuda")
        lengths = torch.tensor(done, dtype=torch.int32, device="cuda")
        q, out = torch.empty_like(parts[0]), torch.empty_like(parts[0])
        shape = P(rows, 3, hq, hkv, 256, 30, page, 10, 160)
        ops.qwen35_paged_cache_append(parts[0], parts[1], parts[2], q, pages, table, starts, lengths, f, wq, wk, shape,
                                      ops.Qwen35PagedRotary(64, False, m), ops.HEAD_MAJOR)
        if max(new) == 1:
            only = torch.tensor(live, device="cuda")
            shape = P(rows, rows, hq, hkv, 256, 30, page, 10, 160)
            ws = torch.empty(max(16, ops.qwen35_paged_decode_workspace_bytes(shape)), device="cuda", dtype=torch.uint8)
            ops.qwen35_paged_attention_decode(q, parts[3], out, pages, table[only].contiguous(), lengths[only].contiguous(), ws, shape, ops.HEAD_MAJOR)
        else:
            ws = torch.empty(max(16, ops.qwen35_paged_prefill_workspace_bytes(shape)), device="cuda", dtype=torch.uint8)
            ops.qwen35_paged_attention_prefill(q, parts[3], out, pages, table, starts, lengths, ws, shape, ops.HEAD_MAJOR)
        torch.cuda.synchronize()
        for i in range(3):
            a = sum(new[:i])
            outs[i].append(out[a:a + new[i]])
    for i in range(3):
        at = np.arange(total[i])
        turn = lambda y, w: torch.tensor(ref.rotate(wide(y), wide(w), at, freq, m, False, 1e-6)).to(BF).double().numpy()  # noqa: E731
        k = turn(x[i][1], wk)
        kv = np.stack([k, wide(x[i][2])]).transpose(0, 2, 1, 3)
        want, spread, reach = ref.attention(turn(x[i][0], wq), wide(x[i][3]), kv, total[i])
        # queries and keys can be rounded to a neighbour of the reference's: 2^-8 of each product, of which some are off
        loose = 2.0 ** -7 * 16 * np.abs(want).max()
        assert (np.abs(wide(torch.cat(outs[i])) - want) <= ref.tolerance(want, spread, reach) + loose * 0.05).all()


def test_offsets_beyond_4_gib(gpu):
    """Rows behind 2^32 bytes of the pool, and a query tensor's rows far apart."""
    page, hkv = 256, 4
    pages = torch.zeros(5000, 2, hkv, page, 256, device="cuda", dtype=BF)  # 5.2 GB
    b = Batch([(2, 300)], page=page, seed=12, spare=0)
    pages[4998:5000] = b.pages
    b.table[0, :2] += 4998
    b.pages = pages
    b.shape = dataclasses.replace(b.shape, pages=5000)
    b.call()
    torch.cuda.synchronize()
    got = b.out.clone()
    b.pages, b.table = pages[4998:].clone(), b.table - 4998
    b.check()
    b.shape = dataclasses.replace(b.shape, pages=2)
    b.call()
    torch.cuda.synchronize()
    assert torch.equal(got, b.out)
    k = torch.randn(2, hkv, 256, device="cuda").to(BF)
    table = torch.tensor([[4999, 4998]], dtype=torch.int32, device="cuda")
    ops.qwen35_paged_cache_append(None, k, k, None, pages, table, b.starts, b.lengths, None, None, None,
                                  dataclasses.replace(b.shape, pages=5000, table_pages=2), ops.Qwen35PagedRotary(0), ops.HEAD_MAJOR)
    torch.cuda.synchronize()
    assert torch.equal(pages[4998, 0, :, 42:44].transpose(0, 1), k) and torch.equal(pages[4998, 1, :, 42:44].transpose(0, 1), k)


# ------------------------------------- chunks of much work, as far as the host can tell

def roomy(b):
    """The batch with a page table of a million positions, which makes a call take the kernel for chunks of much work."""
    extra = (1 << 20) // b.page - b.table.shape[1]
    garbage = torch.randint(-2 ** 31, 2 ** 31 - 1, (b.table.shape[0], extra), generator=b.g, device="cuda", dtype=torch.int64).to(torch.int32)
    b.table = torch.cat([b.table, garbage], 1).contiguous()
    b.shape = dataclasses.replace(b.shape, table_pages=b.table.shape[1], max_context_tokens=b.table.shape[1] * b.page)
    return b


@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("page", [16, 48, 64])
def test_roomy_ragged(gpu, page, head_major):
    errors()
    b = Batch(RAGGED, page=page, head_major=head_major, lead=1, tail=2, seed=page)
    roomy(b).call()
    b.check()
    assert errors() == 0


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 16), (2, 3), (5, 7), (8, 2), (3, 12)])
@pytest.mark.parametrize("head_major", [True, False])
def test_roomy_heads(gpu, kv_heads, group, head_major):
    b = Batch([(9, 40), (33, 70), (150, 400)], kv_heads, group, seed=group, gate=group != 3, head_major=head_major)
    roomy(b).call()
    b.check()


@pytest.mark.parametrize("n,c", [(31, 32), (32, 32), (33, 33), (64, 1000), (130, 700), (300, 300), (40, 3000), (65, 2049), (257, 1025)])
def test_roomy_lengths(gpu, n, c):
    b = roomy(Batch([(n, c)], seed=n))
    b.call()
    b.check()


@pytest.mark.parametrize("kv_heads,each,window,page,head_major", [
    (8, [(600, 620), (33, 400), (80, 80), (1, 300)], 97, 16, True), (8, [(400, 900), (500, 501)], 66, 48, False),
    (4, [(300, 1000), (1, 800), (260, 260), (40, 340)], 300, 32, True)])
def test_roomy_window(gpu, kv_heads, each, window, page, head_major):
    b = Batch(each, kv_heads, 16, page, head_major, window, seed=window, lead=2, tail=1)
    rows = sum(n for n, _ in each)
    assert rows * 16 * kv_heads * window > 40 * 2 ** 18 * 0.7
    roomy(b).call()
    b.check()


def test_roomy_bad_sequences(gpu):
    b = Batch([(9, 60), (9, 70), (9, 80), (9, 90), (9, 100)], seed=8)
    b.table[3, 2] = b.shape.pages
    roomy(b)
    b.lengths[0] = 2              # below its new tokens
    b.lengths[1] = b.shape.max_context_tokens + 1
    b.starts[5] = 1000            # behind the call's rows
    errors()
    b.call()
    b.check(only=(2,))
    assert errors() >= 4
    for i in [0, 1, 3, 4]:
        assert torch.isnan(b.out[9 * i:9 * i + 9]).all(), i


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_roomy_odd_values(gpu, value):
    b = Batch([(20, 40), (45, 70), (30, 36), (200, 400)], seed=4, scale=0.2)
    for i, j in ((0, 39), (1, 60), (1, 3), (3, 130), (3, 350), (3, 399)):
        b.pages[int(b.table[i, j // 16]), 1, i, j % 16, 17 + i] = value
    roomy(b).call()
    b.check()
    b.pages[int(b.table[0, 2]), 0, 1, 35 - 32] = float("nan")
    b.out.fill_(7)
    b.call()
    b.check()


def test_roomy_strided_and_shared(gpu):
    b = Batch([(64, 64), (33, 90), (60, 64)], seed=9)
    b.table[2, :4] = b.table[0, :4]
    proj = torch.stack((b.q, b.gate), 2).contiguous()
    b.q, b.gate = proj[:, :, 0], proj[:, :, 1]
    b.out = torch.full((16, b.rows, 256), 7.0, device="cuda", dtype=BF).transpose(0, 1)
    roomy(b).call()
    b.check()


@pytest.mark.parametrize("chunk", [True, False])
def test_values_of_every_size(gpu, chunk):
    """Scores grow along the keys, so that the kept maximum moves; values near the smallest that keep their bits and near the largest."""
    for size in (2.0 ** -96, 2.0 ** 118):
        b = Batch([(40, 500)], seed=3)
        if chunk:
            roomy(b)
        table = b.table.cpu().numpy()
        mean = b.q[:, ::4].float().mean(0)
        for j in range(500):
            b.pages[int(table[0, j // 16]), 0, :, j % 16] = (mean * (j / 25)).to(BF)
            b.pages[int(table[0, j // 16]), 1, :, j % 16] = b.pages[int(table[0, j // 16]), 1, :, j % 16].float().clamp(-1, 1).mul(size).to(BF)
        b.call()
        b.check()


def test_roomy_two_at_once_on_streams(gpu):
    a, b = roomy(Batch([(30, 400), (1, 90)], seed=1)), roomy(Batch([(77, 500), (90, 2000)], seed=2))
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    wa, wb = a.workspace(), b.workspace()
    torch.cuda.synchronize()
    for _ in range(5):
        a.call(wa, stream=s)
        b.call(wb, stream=t)
    torch.cuda.synchronize()
    a.check()
    b.check()


def test_roomy_graph_replays(gpu):
    b = roomy(Batch([(40, 900), (200, 333)], seed=11))
    ws, eager_ws = b.workspace(), b.workspace()
    b.call(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu):
        b.call(ws, stream=torch.cuda.current_stream())
    for step in range(4):
        b.out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        b.check()
        got = b.out.clone()
        b.out.fill_(7)
        b.call(eager_ws)
        torch.cuda.synchronize()
        assert torch.equal(got, b.out)
        n, c = b.each[0]
        c = c // 3 + n
        b.each = [(n, c)] + b.each[1:]
        b.lengths[0] = c


def test_same_sequence_in_every_kernel(gpu):
    """A sequence's rows do not depend on what else is in the batch by more than the tolerance; the same call twice gives the same bits."""
    b = Batch([(40, 900)], seed=13)
    first = b.call().clone()
    b.out.fill_(7)
    assert torch.equal(b.call(), first)
    roomy(b)
    b.out.fill_(7)
    second = b.call().clone()
    b.check()
    b.out.fill_(7)
    assert torch.equal(b.call(), second)


@pytest.mark.parametrize("sequences", [2, 13, 64, 65, 130])
@pytest.mark.parametrize("chunk", [False, True])
def test_many_sequences(gpu, sequences, chunk):
    """Up to and beyond what one wave holds, some without rows, in no order of length."""
    rng = np.random.default_rng(sequences)
    each = [(0, int(rng.integers(0, 50))) if i % 7 == 3 else (int(rng.integers(1, 9 if i % 5 else 60)), int(rng.integers(60, 500 if i % 11 else 2500)))
            for i in range(sequences)]
    b = Batch(each, 2, 3, seed=sequences, lead=1)
    (roomy(b) if chunk else b).call()
    b.check()
    assert errors() == 0


@pytest.mark.parametrize("window", [1, 7, 40])
def test_small_windows_of_long_chunks(gpu, window):
    """Rows enough for the kernel for chunks of much work, with next to no keys each."""
    b = Batch([(1100, 1100), (40, 300)], window=window, seed=window, head_major=window != 7)
    b.call()
    b.check()


def test_graphs_that_share_a_workspace(gpu):
    """Two captured graphs, of a chunk and of single tokens, use one workspace in turn."""
    a, b = roomy(Batch([(60, 900), (30, 500)], seed=21)), Batch([(1, 3000), (1, 700)], seed=22, decode=True)
    shared = torch.full((max(a.workspace().numel(), b.workspace().numel()),), 0xFF, device="cuda", dtype=torch.uint8)
    graphs = []
    for x in (a, b):
        x.call(shared)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=gpu):
            x.call(shared, stream=torch.cuda.current_stream())
        graphs.append(graph)
    for _ in range(3):
        for x in (a, b):
            x.out.fill_(7)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        a.check()
        b.check()


@pytest.mark.parametrize("sequences,decode", [(700, True), (700, False), (4300, True)])
def test_sequences_beyond_waves(gpu, sequences, decode):
    """Several sequences a lane, and beyond 64 of them; some unused, one long."""
    rng = np.random.default_rng(sequences)
    each = [(1 if decode else int(rng.integers(0, 4)), int(rng.integers(4, 40))) for i in range(sequences)]
    each[sequences // 3] = (1, 3000)
    b = Batch(each, 1, 2, seed=sequences, decode=decode)
    idle = [i for i in range(sequences) if decode and i % 9 == 4]
    if idle:
        b.lengths[torch.tensor(idle, device="cuda")] = 0
    b.call()
    torch.cuda.synchronize()
    b.pages = b.pages.cpu().double()  # (once, not for every sequence)
    b.check(only=set(range(sequences)) - set(idle))
    assert all((b.out[i] == 7).all() for i in idle[:50]) and errors() == 0


@pytest.mark.parametrize("head_major,rotary,interleaved,norm,kv_heads,group", [(True, 64, False, "bf16", 4, 4), (False, 256, True, "f32", 3, 5),
                                                                               (True, 0, False, "q", 1, 1), (False, 32, False, "k", 1, 16)])
def test_append_of_long_chunks(gpu, head_major, rotary, interleaved, norm, kv_heads, group):
    """Rows enough for several a workgroup, sequences that begin and end inside one."""
    each = [(701, 800), (0, 9), (330, 330), (1, 50), (2, 2), (1, 17), (6, 100)]
    test_append(gpu, each, 48, kv_heads, group, rotary, interleaved, norm, head_major)


def test_append_of_long_chunks_refuses_bad_sequences(gpu):
    b = Batch([(501, 600), (3, 20), (402, 500), (203, 300), (2, 7)], seed=7)
    before, out = b.pages.clone(), torch.full_like(b.q, 7.0)
    b.lengths[1] = 2                              # below its new tokens
    b.table[2, 499 // 16] = -1                    # the page of the positions 496 .. 499
    b.starts[5] = b.rows + 9                      # behind the call's rows
    k, v = (torch.randn(b.rows, 4, 256, generator=b.g, device="cuda").to(BF) for _ in (0, 1))
    errors()
    ops.qwen35_paged_cache_append(b.q, k, v, out, b.pages, b.table, b.starts, b.lengths, None, None, None, b.shape,
                                  ops.Qwen35PagedRotary(0), ops.HEAD_MAJOR)
    torch.cuda.synchronize()
    assert errors() >= 3
    expect = before.clone()
    for i, skip in ((0, 600), (2, 496), (3, 300)):
        n, c = b.each[i]
        for p in range(c - n, min(c, skip)):
            page, row = int(b.table[i, p // 16]), int(b.starts_host[i]) + p - (c - n)
            expect[page, 0, :, p % 16], expect[page, 1, :, p % 16] = k[row], v[row]
    assert torch.equal(b.pages.view(torch.int16), expect.view(torch.int16))
    assert torch.equal(out[:501], b.q[:501]) and torch.equal(out[504:1109], b.q[504:1109])
    assert (out[501:504] == 7).all() and (out[1109:] == 7).all()


@pytest.mark.parametrize("kind", ["decode", "few", "much"])
def test_more_heads_than_places(gpu, kind):
    """KV heads beyond the workgroups that are dealt out for each."""
    b = Batch([(1 if kind == "decode" else 12, 600)], 260, 1, seed=2, decode=kind == "decode")
    if kind == "much":
        roomy(b)
    b.call()
    torch.cuda.synchronize()
    b.pages = b.pages.cpu().double()
    b.check()
    assert errors() == 0


@pytest.mark.parametrize("kind", ["decode", "few", "much"])
def test_infinite_keys(gpu, kind):
    """A score of +inf makes its row NaN, one of -inf leaves its key out; rows that do not see the key are as ever."""
    b = Batch([(1, 600), (1, 70)] if kind == "decode" else [(40, 600), (30, 70)], seed=17, decode=kind == "decode")
    if kind == "much":
        roomy(b)
    for i, j in ((0, 590), (0, 3), (1, 60)):
        b.pages[int(b.table[i, j // 16]), 0, i, j % 16, 5] = float("inf")
    b.call()
    torch.cuda.synchronize()
    got = wide(b.out)
    some = False
    for i, (n, c) in enumerate(b.each):
        rows, want, tol = b.want(i)
        assert np.array_equal(np.isnan(got[rows]), np.isnan(want)), i
        some |= np.isnan(want).any() and not np.isnan(want).all()
    assert some
    # finite rows of the KV heads that the keys do not belong to, and of the others without the keys
    b.check()


# ------------------------------------------------ bounds above the page table

@pytest.mark.parametrize("kind,window", [("decode", 0), ("decode", 30), ("few", 0), ("few", 30), ("much", 0), ("much", 66)])
def test_a_bound_above_the_table(gpu, kind, window):
    """It gives the same bits as the table's positions for a bound; a sequence above them is NaN and counted."""
    n = 1 if kind == "decode" else 20
    each = [(n, 700), (n, 333), (n, 64), (n, 450)]
    if kind == "much" and window:
        each = [(700, 900), (33, 64), (300, 450)]  # (many rows take the kernel for much work, few keys or not)
    b = Batch(each, window=window, decode=kind == "decode", seed=31)
    if kind == "much":
        roomy(b)
    positions = b.shape.table_pages * b.page
    b.shape = dataclasses.replace(b.shape, max_context_tokens=positions)
    tight = b.call().clone()
    for bound in (positions + 1, 1 << 28):
        loose = dataclasses.replace(b.shape, max_context_tokens=bound)
        size = ops.qwen35_paged_decode_workspace_bytes if b.decode else ops.qwen35_paged_prefill_workspace_bytes
        assert size(loose) == size(b.shape)
        b.out.fill_(7)
        assert torch.equal(b.call(shape=loose), tight)
    b.check()
    bad = len(each) - 1
    b.lengths[bad] = positions + 1
    b.out.fill_(7)
    errors()
    b.call(shape=loose)
    b.check(only=set(range(bad)))
    assert errors() >= 1 and torch.isnan(b.out[int(b.starts_host[bad]):]).all()


@pytest.mark.parametrize("rows", [3, 400])
def test_append_with_a_bound_above_the_table(gpu, rows):
    b = Batch([(rows, 500), (rows, 430), (rows, 420)], seed=32)
    k, v = (torch.randn(b.rows, 4, 256, generator=b.g, device="cuda").to(BF) for _ in (0, 1))
    positions = b.shape.table_pages * b.page
    b.lengths[1] = positions + 1
    before, got = b.pages.clone(), []
    for bound in (positions, positions + 1, 1 << 28):
        b.pages, out = before.clone(), torch.full_like(b.q, 7.0)
        errors()
        ops.qwen35_paged_cache_append(b.q, k, v, out, b.pages, b.table, b.starts, b.lengths, None, None, None,
                                      dataclasses.replace(b.shape, max_context_tokens=bound), ops.Qwen35PagedRotary(0), ops.HEAD_MAJOR)
        torch.cuda.synchronize()
        assert errors() >= 1
        got.append((b.pages.view(torch.int16), out))
    for pages, out in got[1:]:
        assert torch.equal(pages, got[0][0]) and torch.equal(out, got[0][1])
    expect = before.clone()
    for i in (0, 2):
        for t in range(rows):
            p, row = b.each[i][1] - rows + t, i * rows + t
            page = int(b.table[i, p // 16])
            expect[page, 0, :, p % 16], expect[page, 1, :, p % 16] = k[row], v[row]
    assert torch.equal(got[0][0], expect.view(torch.int16)) and (got[0][1][rows:2 * rows] == 7).all()


# --------------------------------------------------------- norms of small heads

@pytest.mark.parametrize("dtype,dim", [(BF, 256), (torch.float32, 128), (torch.float32, 33)])
@pytest.mark.parametrize("size", [2.0 ** -66, 2.0 ** -64, 2.0 ** -48])
def test_norm_of_small_values(gpu, dtype, dim, size):
    """Without an epsilon a head's size goes out of its norm, also where the mean of the squares is below the smallest normal number."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = (torch.randn(7, 3, dim, generator=g, device="cuda").clamp(-2, 2) * size).to(dtype)
    w = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
    out, positions = torch.empty_like(x), torch.arange(7, dtype=torch.int32, device="cuda")
    freq, _ = ops.qwen35_rotary_frequencies(32, 1e4)
    ops.qwen35_rotary(x, w, out, positions, torch.tensor(freq, dtype=torch.float64, device="cuda"), ops.Qwen35RotaryShape(7, 3, dim, 32), 0.0)
    torch.cuda.synchronize()
    want = ref.rotate(wide(x), wide(w), np.arange(7), freq, 1.0, False, 0.0)
    # 32 bits: `dim` squares, each off by 2^-150 or half a step, and their mean (a mean of at least 2^-134 is off by 2^-16 of itself,
    # its root by half of that); two dozen roundings of values up to 1.5 times the pair's; the result is rounded once
    mean = (wide(x) ** 2).mean(-1, keepdims=True)
    off = (2 * 2.0 ** -150 / mean) / 2 + 2.0 ** -24 * (dim / 2 + 24)
    assert (np.abs(wide(out) - want) <= torch.finfo(dtype).eps / 2 * np.abs(want) + 2 * off * np.abs(want).max()).all()
    if dim == 256:
        b = Batch([(7, 20)], 3, 1, seed=1)
        q, one = torch.empty_like(x), torch.ones(256, device="cuda")
        ops.qwen35_paged_cache_append(x, x, x, q, b.pages, b.table, b.starts, b.lengths, None, one, one, b.shape, ops.Qwen35PagedRotary(0, epsilon=0.0),
                                      ops.HEAD_MAJOR)
        torch.cuda.synchronize()
        y = wide(x) / np.sqrt(mean)
        assert (np.abs(wide(q) - y) <= ref.HALF_BF16 * np.abs(y) + 2 * off * np.abs(y).max()).all()
        at = torch.stack([b.pages[int(b.table[0, p // 16]), 0, :, p % 16] for p in range(13, 20)])
        assert torch.equal(at, q)


# ------------------------------------------------------ bits of the probabilities

def cancelling(each, decode, much=False):
    """Values of neighbouring keys cancel as the probabilities weigh them, so that an output shows their roundings and not its own; scores
    are small.  One query head per KV head."""
    b = Batch(each, 4, 1, decode=decode, gate=False, seed=41)
    if much:
        roomy(b)
    b.q = (b.q.float() / 8).to(BF)
    for i, (n, c) in enumerate(each):
        where = [(int(b.table[i, j // 16]), j % 16) for j in range(c)]
        k = torch.stack([b.pages[p, 0, :, at] for p, at in where]).double()              # [c, heads, 256]
        last = b.q[int(b.starts_host[i]) + n - 1].double()                               # the last token cancels
        w = torch.softmax(torch.einsum("jhd,hd->hj", k.cpu(), last.cpu()) / 16, -1)
        v = torch.randn(c, 4, 256, generator=b.g, device="cuda").cpu().double()
        for j in range(0, c - 1, 2):
            v[j] = v[j].to(BF).double()
            v[j + 1] = -v[j] * (w[:, j] / w[:, j + 1])[:, None]
        if c % 2:
            v[c - 1] = 0
        for j, (p, at) in enumerate(where):
            b.pages[p, 1, :, at] = v[j].to(BF).cuda()
    return b


def last_tokens(b):
    """Of every sequence: its last row's output, the exact one, one of probabilities in 8 bits, the sum of |probability * value|, and how far
    scores in 32 bits move a probability, relative to it."""
    for i, (n, c) in enumerate(b.each):
        row = int(b.starts_host[i]) + n - 1
        kv = ref.rows_of(wide(b.pages), b.table[i].cpu().numpy(), c, b.page, True)
        q = wide(b.q[row])
        for h in range(4):
            k, v = kv[0, h], kv[1, h]
            e = np.exp(k @ q[h] / 16 - (k @ q[h] / 16).max())
            cut = torch.tensor(e).to(BF).double().numpy()
            off = 2 * 256 * 2.0 ** -24 * (np.abs(k) @ np.abs(q[h])).max() / 16
            yield wide(b.out[row, h]), e / e.sum() @ v, cut / cut.sum() @ v, e / e.sum() @ np.abs(v), off


def test_decode_holds_probabilities_in_two_parts(gpu):
    """The first part is at most 2^-9 and a truncation (2^-7) below the probability, the rest is rounded (2^-8): off by 2^-15 + 2^-17."""
    b = cancelling([(1, 2), (1, 8), (1, 33), (1, 64)], True)
    b.call()
    torch.cuda.synchronize()
    shown = []
    for got, want, cut, size, off in last_tokens(b):
        # (sums of up to 64 products in 32 bits, exponentials, the division: 100 roundings at most)
        tol = ref.HALF_BF16 * np.abs(want) + (2.0 ** -15 + 2.0 ** -17 + off + 100 * 2.0 ** -24) * size
        assert (np.abs(got - want) <= tol).all()
        shown.append((np.abs(cut - want) > tol).mean())
    assert np.median(shown) > 0.3  # probabilities in 8 bits would not pass


@pytest.mark.parametrize("much", [False, True])
def test_chunks_hold_probabilities_in_8_bits(gpu, much):
    """Each is off by 2^-8 of itself at most, and they are divided by the sum of what they were rounded to."""
    b = cancelling([(5, 8), (3, 33), (40, 64)], False, much)
    b.call()
    torch.cuda.synchronize()
    for got, want, _, size, off in last_tokens(b):
        assert (np.abs(got - want) <= ref.HALF_BF16 * np.abs(want) + (2.0 ** -8 * 1.01 + off + 100 * 2.0 ** -24) * (size + np.abs(want))).all()


# -------------------------------- ranges longer than the page entries that a wave holds

def check_on_device(b, i):
    """Batch.check for one sequence with 64-bit sums on the GPU: pools that are too large for the host's reference."""
    n, c = b.each[i]
    a, j = int(b.starts_host[i]), torch.arange(c, device="cuda")
    page, at = b.table[i].long()[j // b.page], j % b.page
    token = c - n + torch.arange(n, device="cuda")
    hidden = j > token[:, None]
    if b.window:
        hidden |= j <= token[:, None] - b.window
    for h in range(b.kv_heads):
        k, v = ((b.pages[page, x, h, at] if b.head_major else b.pages[page, x, at, h]).double().masked_fill(hidden.all(0)[:, None], 0)
                for x in (0, 1))
        for g in range(h * b.group, (h + 1) * b.group):
            q = b.q[a:a + n, g].double()
            p = torch.softmax((q @ k.T / 16).masked_fill(hidden, -torch.inf), -1)
            want = p @ v
            seen, size = ~hidden.all(0), torch.where(hidden.all(0)[:, None], 0, v.abs())
            spread = p @ size + want.abs()                                      # (at least the mean of |value - output|)
            off = 256 * 2.0 ** -24 * (q.abs() @ k[seen].abs().T).max() / 16
            gate = 1 if b.gate is None else torch.sigmoid(b.gate[a:a + n, g].double())
            tol = ref.HALF_BF16 * (want * gate).abs() + gate * (2.0 ** -8 * 1.01 * spread * (not b.decode) + (2.0 ** -14 + 2 * off) * (p @ size))
            assert ((b.out[a:a + n, g].double() - want * gate).abs() <= tol).all(), (h, g)


@pytest.mark.parametrize("kind,n,c,kv_heads,page,head_major,window", [
    # a workgroup of the single-token kernel holds the entries of 256 tiles of 16 keys, of short chunks 128 of 32
    ("decode", 1, 20000, 64, 16, True, 0), ("decode", 1, 10007, 128, 48, False, 0), ("decode", 1, 12001, 128, 32, True, 9000),
    ("few", 2, 20000, 64, 48, True, 0), ("few", 3, 9999, 128, 16, False, 0),
    # of long chunks about 120 of 32: met where every column sees all of a tile, and in the last, masked, tiles
    ("much", 40, 6001, 260, 48, False, 0), ("much", 128, 3968, 260, 16, True, 0), ("much", 120, 3950, 260, 64, False, 0),
    ("much", 60, 6500, 260, 16, True, 4500)])
def test_long_ranges(gpu, kind, n, c, kv_heads, page, head_major, window):
    b = Batch([(n, c)], kv_heads, 1, page, head_major, window, seed=c, decode=kind == "decode", gate=kind != "few")
    columns, keys = n * kv_heads, min(c, window or c)
    assert (columns * keys > 40 * 256 * 32 * 32) == (kind == "much") or kind == "decode"
    errors()
    b.call()
    torch.cuda.synchronize()
    assert errors() == 0
    b.table[0, :max(0, c - n + 1 - window) // page if window else 0] = 0
    check_on_device(b, 0)
    # every entry counts: with any of some neighbours of the refill gone, the sequence is NaN
    table = b.table.clone()
    lo = (c - n + 1 - window) // page + 1 if window else 0
    for entry in sorted({lo, (lo + c // page) // 2, min(c // page - 1, lo + 4096 // page), (c - 1) // page}):
        b.table = table.clone()
        b.table[0, entry] = b.shape.pages
        b.call()
        torch.cuda.synchronize()
        assert errors() >= 1 and torch.isnan(b.out).all(-1).any(), entry
        assert torch.isnan(b.out[-1]).all(), entry  # (the last token sees every one of them)


def test_a_sequence_alone_and_among_others(gpu):
    """In each kernel a sequence's rows meet the reference alone and in a batch; the last token also as a single one; twice the same bits."""
    n, c = 9, 700
    others = [(3, 40), (n, c), (70, 300), (1, 900)]
    alone, among = Batch([(n, c)], seed=51), Batch(others, seed=52)
    where = [(int(alone.table[0, j]), int(among.table[1, j])) for j in range(-(-c // 16))]
    for one, other in where:
        among.pages[other] = alone.pages[one]
    at = int(among.starts_host[1])
    among.q[at:at + n], among.gate[at:at + n] = alone.q, alone.gate
    rows, want, tol = alone.want(0)
    for kind in ("few", "much"):
        if kind == "much":
            roomy(alone)
            roomy(among)
        first = [alone.call().clone(), among.call().clone()]
        for got in (first[0], first[1][at:at + n]):
            assert (np.abs(wide(got) - want) <= tol).all()
        assert torch.equal(alone.call(), first[0]) and torch.equal(among.call(), first[1])
    single = P(1, 1, 16, 4, 256, alone.shape.pages, 16, alone.shape.table_pages, c)
    out = torch.empty(1, 16, 256, device="cuda", dtype=BF)
    ws = torch.empty(max(16, ops.qwen35_paged_decode_workspace_bytes(single)), device="cuda", dtype=torch.uint8)
    ops.qwen35_paged_attention_decode(alone.q[n - 1:], alone.gate[n - 1:], out, alone.pages, alone.table, alone.lengths, ws, single, ops.HEAD_MAJOR)
    torch.cuda.synchronize()
    assert (np.abs(wide(out) - want[n - 1:]) <= tol[n - 1:]).all()


def test_append_to_its_last_bit(gpu):
    """Keys and queries of append are off by their rounding and a few dozen steps of 32 bits."""
    b = Batch([(33, 50), (1, 300)], seed=61)
    k = torch.randn(b.rows, 4, 256, generator=b.g, device="cuda").to(BF)
    w = 1 + 0.1 * torch.randn(256, generator=b.g, device="cuda")
    freq, m = ops.qwen35_rotary_frequencies(64, 1e7)
    out = torch.empty_like(b.q)
    ops.qwen35_paged_cache_append(b.q, k, k, out, b.pages, b.table, b.starts, b.lengths, torch.tensor(freq, dtype=torch.float64, device="cuda"), w, w,
                                  b.shape, ops.Qwen35PagedRotary(64, False, m, 1e-6), ops.HEAD_MAJOR)
    torch.cuda.synchronize()
    at = np.concatenate([np.arange(c - n, c) for n, c in b.each])
    stored = torch.stack([b.pages[int(b.table[i, p // 16]), 0, :, p % 16] for i, (n, c) in enumerate(b.each) for p in range(c - n, c)])
    for got, x in ((out, b.q), (stored, k)):
        want = ref.rotate(wide(x), wide(w), at, freq, m, False, 1e-6)
        # a pair's sizes bound its two results: the norm's sum of 256 squares and its root, the angle (reduced, up to pi: half a step is
        # pi 2^-24), sine and cosine (2 steps), products and sum
        pair = np.abs(ref.rotate(np.abs(wide(x)), np.abs(wide(w)), np.zeros(len(at), int), freq, 1.0, False, 1e-6))
        pair[..., :32] = pair[..., 32:64] = pair[..., :32] + pair[..., 32:64]
        assert (np.abs(wide(got) - want) <= ref.HALF_BF16 * np.abs(want) + pair * 2.0 ** -24 * (128 + 16)).all()


@pytest.mark.parametrize("dtype,dim", [(BF, 16384), (torch.float32, 16384), (torch.float16, 16382)])
def test_rotary_of_the_largest_heads(gpu, dtype, dim):
    """The angles of a row fill 64 KiB of LDS."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(2, 3, dim, generator=g, device="cuda").to(dtype)
    out, positions = torch.empty_like(x), torch.tensor([5, 100000], dtype=torch.int32, device="cuda")
    freq, _ = ops.qwen35_rotary_frequencies(dim, 1e7)
    ops.qwen35_rotary(x, None, out, positions, torch.tensor(freq, dtype=torch.float64, device="cuda"), ops.Qwen35RotaryShape(2, 3, dim, dim), 0.0)
    torch.cuda.synchronize()
    y, half = wide(x), dim // 2
    turn = np.array([[np.longdouble(p) * np.longdouble(f) % (2 * np.longdouble(np.pi)) for f in freq] for p in (5, 100000)]).astype(np.float64)[:, None]
    a, c = y[..., :half], y[..., half:]
    want = np.concatenate([a * np.cos(turn) - c * np.sin(turn), a * np.sin(turn) + c * np.cos(turn)], -1)
    size = np.tile(np.abs(a) + np.abs(c), 2)
    tol = torch.finfo(dtype).eps / 2 * np.abs(want) + size * 2.0 ** -24 * 12 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert (np.abs(wide(out) - want) <= tol).all()
