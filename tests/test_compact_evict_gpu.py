"""Which entries an eviction keeps, over long caches and weights that are alike or odd."""
import numpy as np
import pytest
import torch

from helpers import rng
from raftinfer_amd import ops
from test_compact_gpu import D, FP8, dev, host

pytestmark = pytest.mark.gpu


def setup(hkv, n, keep, sinks, recent):
    size = lambda m: ops.qwen35_compact_cache_bytes(ops.Qwen35CompactShape(1, 1, hkv, hkv, D, m, 0), FP8)
    buf, out = (torch.zeros(size(m), device="cuda", dtype=torch.uint8) for m in (n, keep))
    out_w = torch.empty(hkv, keep, device="cuda")
    kept = torch.full((hkv, keep), -1, device="cuda", dtype=torch.int32)
    shape = ops.Qwen35EvictShape(hkv, D, n, n, keep, keep, sinks, recent)
    ws = torch.full((max(16, ops.qwen35_compact_evict_workspace_bytes(shape)),), 0xFF, device="cuda", dtype=torch.uint8)
    return lambda w: (ops.qwen35_compact_cache_evict(buf, w, out, out_w, kept, shape, FP8, FP8, 1, ws), (kept, out_w))[1]


def check(w, keep, sinks, recent):
    hkv, n = w.shape
    kept, out_w = setup(hkv, n, keep, sinks, recent)(dev(w, torch.float32))
    for h in range(hkv):
        rank = np.where(np.isnan(w[h]), np.inf, w[h].astype(np.float64)) + 0.0
        # NaN above infinity, the sinks and the recent ones above all; equal ones in their order
        order = np.lexsort((np.arange(n), -rank, ~np.isnan(w[h])))
        free = order[(order >= sinks) & (order < n - recent)]
        want = np.sort(np.concatenate([np.arange(sinks), free[:keep - sinks - recent], np.arange(n - recent, n)]))
        assert np.array_equal(kept[h].cpu().numpy(), want), h
        assert np.array_equal(host(out_w[h]), w[h][want], equal_nan=True), h


def spread(r, hkv, n):
    return np.exp(2 * r.standard_normal((hkv, n))).astype(np.float32)


# one workgroup a head; segments of one piece, of two and of more, the last ones not full
LENGTHS = [3000, 16384, 16385, 40001, 262144, 262145, 300001, 1000003]


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("what", ["spread", "mostly zero", "zero", "equal", "two", "near", "odd"])
def test_evict_selection(gpu, n, what):
    r = rng(1)
    hkv = 2 if n < 500000 else 1
    w = spread(r, hkv, n)
    if what == "mostly zero":      # as behind a window; the budget exceeds what drew any attention
        w[r.random((hkv, n)) < 0.9] = 0
    elif what == "zero":
        w[:] = 0
    elif what == "equal":
        w[:] = 0.25
    elif what == "two":
        w = np.where(r.random((hkv, n)) < 0.1, 0.5, 0.25).astype(np.float32)
    elif what == "near":           # one first digit, and the same second one for most
        w = (0.75 + r.integers(0, 3000, (hkv, n)) * 2.0 ** -23).astype(np.float32)
    elif what == "odd":
        for x in (np.nan, np.inf, -np.inf, -0.0, 0.0, -1.5, 1e-40):
            w[r.random((hkv, n)) < 0.04] = x
    check(w, n // 4, 4, 32)


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("keep,sinks,recent", [("some", 5000, 2000), ("all", 3, 2), ("all but one", 0, 0), ("one", 0, 0), ("one", 0, 1),
                                               ("sinks and recent", 1000, 77), ("sinks", 2500, 0), ("recent", 0, 2999)])
def test_evict_budgets(gpu, n, keep, sinks, recent):
    sinks, recent = min(sinks, n // 3), min(recent, n // 3)
    count = {"some": n // 2 + sinks, "all": n, "all but one": n - 1, "one": 1}.get(keep, sinks + recent)
    count = min(n, max(count, sinks + recent))
    r = rng(2)
    w = spread(r, 1, n)
    w[r.random((1, n)) < 0.5] = 0
    check(w, count, sinks, recent)


@pytest.mark.parametrize("n", [16000, 60001, 400000])
def test_alike_weights_take_no_longer(gpu, n):
    """Ranks that share a histogram's bin, in a wave and over the segments, cost little more than spread ones (at
    most 1.8 times as much, at 60001; 3 to 13 times where each is counted by itself and every segment looks at all of them)."""
    r = rng(3)
    go = setup(1, n, n // 4, 4, 32)
    took = {}
    some = spread(r, 1, n)
    for name, w in (("spread", some), ("mostly zero", np.where(r.random((1, n)) < 0.9, 0, some)), ("equal", np.full((1, n), 0.25))):
        w = dev(w, torch.float32)
        for _ in range(3):
            go(w)
        times = []
        for _ in range(20):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(10):
                go(w)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        took[name] = min(times)
    assert max(took["mostly zero"], took["equal"]) < 2.5 * took["spread"], took


def test_evict_selection_in_a_graph(gpu):
    """Captured once and replayed over other weights, with eager calls on the same buffers between."""
    r = rng(4)
    n, keep = 70001, 20000
    go = setup(2, n, keep, 4, 32)
    inputs = [dev(spread(r, 2, n), torch.float32) for _ in range(3)] + [torch.zeros(2, n, device="cuda")]
    want = [go(w)[0].clone() for w in inputs]
    held = inputs[0].clone()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        kept, _ = go(held)
    for i in (0, 3, 1, 2, 3, 0):
        go(inputs[(i + 1) % 4])
        held.copy_(inputs[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want[i]), i
