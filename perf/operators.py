"""The compact KV cache of a serving program, as measurable cases.

Three operators that share one cache: gated attention over keys and values held in 8 bits with a scale for each
block of 32 tokens and head; gated attention that sees a sliding window and a few first tokens; and eviction of
the entries that drew least attention, with the attention calls that add the weights up.  Heads are the model's:
16 query / 4 KV heads of 256 dims.

An 8-bit cache holds e4m3 codes and, for each plane (K, V), KV head and block of 32 positions, a power-of-two
scale: the smallest with which no finite value of the block leaves the codes' range.  A row that needs a larger
scale than its block has raises it, and the block's earlier rows are rounded again to the new one.  Attention
reads the cache, the rows that the same call stored included.

    import perf.operators as c
    state = c.prepare(c.listed()[0], seed=1)
    outputs = c.run(state)
"""
from __future__ import annotations

import math

import torch

own = False

HQ, HKV, D = 16, 4, 256
G = HQ // HKV
BLOCK = 32               # positions that share a scale
TOP = 448.0              # largest e4m3 value
F32, F64 = torch.float32, torch.float64

_stream = None


def stream():
    """The one stream that the program enqueues everything on (the library takes no null stream)."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
        torch.cuda.set_stream(_stream)
    return _stream


# ------------------------------------------------------------------ cases

def listed():
    return [
        # One token of a short chat on an 8-bit cache: latency and launches.
        {"name": "decode_fp8_short", "kind": "decode", "fp8": True, "sequences": 1, "context": 201, "max_context": 4096, "window": 0, "sinks": 0, "weights": False},
        # One token of a long document on an 8-bit cache, ragged end.
        {"name": "decode_fp8_long", "kind": "decode", "fp8": True, "sequences": 1, "context": 60001, "max_context": 65536, "window": 0, "sinks": 0, "weights": False},
        # A serving batch of 32 sequences of very different lengths on 8-bit caches.
        {"name": "decode_fp8_batch", "kind": "decode", "fp8": True, "sequences": 32, "context": 32768, "max_context": 32768, "window": 0, "sinks": 0, "weights": False},
        # The prompt bucket of 512 tokens, start of a prompt, stored in 8 bits.
        {"name": "prefill_fp8_512", "kind": "prefill", "fp8": True, "tokens": 512, "past": 0, "max_context": 4096, "window": 0, "sinks": 0, "observed": 0},
        # A later chunk of a long document on an 8-bit cache, behind a past that ends inside a block.
        {"name": "prefill_fp8_chunk", "kind": "prefill", "fp8": True, "tokens": 500, "past": 30001, "max_context": 32768, "window": 0, "sinks": 0, "observed": 0},
        # A batch of endless streams: the last 4096 tokens and 4 sinks of a bf16 cache.
        {"name": "decode_window_batch", "kind": "decode", "fp8": False, "sequences": 16, "context": 32768, "max_context": 32768, "window": 4096, "sinks": 4, "weights": False},
        # A long prompt through a windowed layer, ragged end.
        {"name": "prefill_window_long", "kind": "prefill", "fp8": False, "tokens": 6001, "past": 0, "max_context": 8192, "window": 1024, "sinks": 4, "observed": 0},
        # A chunk of a stream on a windowed layer with an 8-bit cache; the sinks end inside a block.
        {"name": "prefill_window_chunk", "kind": "prefill", "fp8": True, "tokens": 300, "past": 9001, "max_context": 16384, "window": 2048, "sinks": 70, "observed": 0},
        # Single tokens that also add up what attention each cached key draws.
        {"name": "decode_weights", "kind": "decode", "fp8": False, "sequences": 4, "context": 8192, "max_context": 8192, "window": 0, "sinks": 0, "weights": True},
        # A prompt whose last 64 tokens say which keys draw attention, as before an eviction.
        {"name": "prefill_weights", "kind": "prefill", "fp8": False, "tokens": 2001, "past": 0, "max_context": 4096, "window": 0, "sinks": 0, "observed": 64},
        # A prompt's bf16 cache cut to a quarter.
        {"name": "evict_prompt", "kind": "evict", "fp8": False, "out_fp8": False, "context": 4001, "keep": 1024, "sinks": 4, "recent": 64},
        # A long document's 8-bit cache cut to a quarter.
        {"name": "evict_long_fp8", "kind": "evict", "fp8": True, "out_fp8": True, "context": 60001, "keep": 16384, "sinks": 4, "recent": 512},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _capacity(rng, n):
    """A cache capacity for n positions: a power of two, or one that is no multiple of anything."""
    return (1 << max(9, (n - 1).bit_length())) if rng.random() < 0.7 else n + rng.randint(1, 77)


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "evict"])
    fp8 = rng.random() < 0.6
    if kind == "evict":
        context = _log_int(rng, 2, 60001)
        keep = _log_int(rng, 1, context)
        sinks = rng.randint(0, min(8, keep))
        return {"kind": kind, "fp8": fp8, "out_fp8": fp8 or rng.random() < 0.3, "context": context, "keep": keep,
                "sinks": sinks, "recent": rng.randint(0, min(512, keep - sinks))}
    windowed = rng.random() < 0.5
    window = _log_int(rng, 1, 8192) if windowed else 0
    sinks = rng.choice([0, 1, 4, rng.randint(5, 100)]) if windowed else 0
    if kind == "decode":
        sequences = rng.choice([1, 1, _log_int(rng, 2, 32)])
        context = _log_int(rng, 1, 60001) if sequences == 1 else _log_int(rng, 300, 16384)
        return {"kind": kind, "fp8": fp8, "sequences": sequences, "context": context, "max_context": _capacity(rng, context),
                "window": window, "sinks": sinks, "weights": rng.random() < 0.3}
    if rng.random() < 0.5:  # a chunk behind a past
        tokens, past = _log_int(rng, 2, 512), _log_int(rng, 1, 30000)
    else:                   # a whole prompt
        tokens, past = _log_int(rng, 2, 4001), 0
    observed = rng.choice([0, 0, rng.randint(1, min(tokens, 128))])
    return {"kind": kind, "fp8": fp8, "tokens": tokens, "past": past, "max_context": _capacity(rng, tokens + past),
            "window": window, "sinks": sinks, "observed": observed}


# ------------------------------------------------------------------ inputs

def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def cache_bytes(positions, fp8):
    codes = 2 * positions * HKV * D
    return codes + 8 * HKV * _blocks(positions) if fp8 else 2 * codes


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def _pow2_scale(amax):
    """The smallest power of two s with amax <= 448 s (a normal number)."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=-126))


def _rows(g, *shape):
    """K or V rows of a layer: about 1% of them eight times as large, so that the softmax has maxima to find."""
    x = _randn(g, *shape)
    x *= 1 + 7 * (torch.rand(shape[:-1] + (1,), generator=g, device="cuda") < 0.01)
    return x


def _views(cache, positions, fp8):
    """(values or codes [sequences, 2, HKV, positions, D], scales [sequences, 2, HKV, blocks]) of cache buffers [sequences, bytes]."""
    n, codes = cache.shape[0], 2 * HKV * positions * D
    if not fp8:
        return cache.view(torch.bfloat16).view(n, 2, HKV, positions, D), None
    return (cache[:, :codes].view(n, 2, HKV, positions, D),
            cache[:, codes:].view(F32).view(n, 2, HKV, _blocks(positions)))


def _filled_cache(g, sequences, positions, fp8):
    """Caches whose every position holds a row, as one that sequences before have filled."""
    cache = torch.empty(sequences, cache_bytes(positions, fp8), device="cuda", dtype=torch.uint8)
    rows, scales = _views(cache, positions, fp8)
    for s in range(sequences):
        x = _rows(g, 2, HKV, positions, D)
        if not fp8:
            rows[s] = x
            continue
        pad = _blocks(positions) * BLOCK - positions
        x = torch.nn.functional.pad(x, (0, 0, 0, pad)).view(2, HKV, -1, BLOCK, D)
        scale = _pow2_scale(x.abs().amax((-1, -2)).float())
        scales[s] = scale
        x = (x.float() / scale[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        rows[s] = x.view(2, HKV, -1, D)[:, :, :positions]
    return cache


def prepare(case, seed):
    stream()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["kind"] == "evict":
        n, keep = case["context"], case["keep"]
        s["cache"] = _filled_cache(g, 1, n, case["fp8"])
        # weights as attention leaves them: far apart, and a tenth of the keys seen by no one
        w = torch.exp(3 * torch.randn(HKV, n, generator=g, device="cuda")) * 1e-3
        s["weights"] = w * (torch.rand(HKV, n, generator=g, device="cuda") >= 0.1)
        s["out_cache"] = torch.zeros(1, cache_bytes(keep, case["out_fp8"]), device="cuda", dtype=torch.uint8)
        s["out_weights"] = torch.empty(HKV, keep, device="cuda")
        s["kept"] = torch.empty(HKV, keep, device="cuda", dtype=torch.int32)
        s["workspace"] = torch.empty(64 << 20, device="cuda", dtype=torch.uint8)
        return s
    b, cap = case.get("sequences", 1), case["max_context"]
    t = case.get("tokens", 1)
    s["cache"] = _filled_cache(g, b, cap, case["fp8"])
    s["q"], s["gate"] = _randn(g, b, t, HQ, D), _randn(g, b, t, HQ, D)
    s["k"], s["v"] = _rows(g, b, t, HKV, D), _rows(g, b, t, HKV, D)
    s["out"] = torch.empty(b, t, HQ, D, device="cuda", dtype=torch.bfloat16)
    if b > 1:  # ragged: every length from 1 to the longest
        lengths = torch.randint(1, case["context"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = case["context"]
        s["lengths"] = lengths
    if case.get("weights") or case.get("observed"):
        s["weights"] = torch.rand(b, HKV, cap, generator=g, device="cuda") * 1e-2
    s["workspace"] = torch.empty(1 << 30, device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------------ plain form

def _positions(s):
    """Positions stored before the call, [sequences, 1]."""
    c = s["case"]
    if "lengths" in s:
        return s["lengths"].long()[:, None] - 1
    return torch.full((1, 1), c["past"] if c["kind"] == "prefill" else c["context"] - 1, device="cuda")


def _held(codes, scales, positions):
    """What codes [.., positions, D] and scales [.., blocks] stand for."""
    per_row = scales.repeat_interleave(BLOCK, -1)[..., :positions]
    return codes.view(torch.float8_e4m3fn).to(F32) * per_row[..., None]


def _codes(x, scale):
    return (x / scale).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_store(s):
    c = s["case"]
    cap = c["max_context"]
    rows, scales = _views(s["cache"], cap, c["fp8"])
    past = _positions(s)                                                # [b, 1]
    new = torch.stack((s["k"], s["v"]), 1).transpose(2, 3)              # [b, 2, HKV, t, D]
    b, t = new.shape[0], new.shape[3]
    every = torch.arange(b, device="cuda")[:, None, None, None]
    plane = torch.arange(2, device="cuda")[None, :, None, None]
    head = torch.arange(HKV, device="cuda")[None, None, :, None]
    at = (past + torch.arange(t, device="cuda"))[:, None, None, :]
    if not c["fp8"]:
        rows[every, plane, head, at] = new
        return
    first = past // BLOCK                                               # [b, 1]
    count = 1 if t == 1 else _blocks(c["past"] % BLOCK + t)
    pos = first * BLOCK + torch.arange(count * BLOCK, device="cuda")    # [b, count * 32]
    old = (pos < past)[:, None, None, :, None]
    fresh = ((pos >= past) & (pos < past + t))[:, None, None, :, None]
    inside = pos.clamp(max=cap - 1)[:, None, None, :]
    blocks = (first + torch.arange(count, device="cuda"))[:, None, None, :]
    before = scales[every, plane, head, blocks]                         # [b, 2, HKV, count]
    x = rows[every, plane, head, inside].view(torch.float8_e4m3fn).to(F32) * before.repeat_interleave(BLOCK, -1)[..., None]
    taken = (pos - past).clamp(0, t - 1)[:, None, None, :, None].expand(b, 2, HKV, -1, D)
    x = torch.where(fresh, torch.gather(new, 3, taken).to(F32), torch.where(old, x, 0.0))
    size = torch.where(fresh, x.abs(), 0.0).view(b, 2, HKV, count, -1).amax(-1)
    has_old = (blocks * BLOCK) < past[:, :, None, None]
    after = torch.maximum(_pow2_scale(size), torch.where(has_old, before, 0.0))
    scales[every, plane, head, blocks] = after
    codes = _codes(x, after.repeat_interleave(BLOCK, -1)[..., None])
    # places after the last stored row take the first stored row's place and value: no row there changes
    mine = past - first * BLOCK                                         # [b, 1]
    source = torch.where(pos < past + t, torch.arange(count * BLOCK, device="cuda"), mine)
    codes = torch.gather(codes, 3, source[:, None, None, :, None].expand(b, 2, HKV, -1, D))
    rows[every, plane, head, (first * BLOCK + source)[:, None, None, :]] = codes


def _plain_attention(s):
    c = s["case"]
    cap, t = c["max_context"], s["q"].shape[1]
    _plain_store(s)
    rows, scales = _views(s["cache"], cap, c["fp8"])
    n = c["past"] + t if c["kind"] == "prefill" else c["context"]
    x = _held(rows[:, :, :, :n], scales[..., :_blocks(n)], n) if c["fp8"] else rows[:, :, :, :n].to(F32)
    b = x.shape[0]
    q = s["q"].to(F32).view(b, t, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(b * HKV, t * G, D)
    score = torch.bmm(q, x[:, 0].reshape(b * HKV, n, D).transpose(1, 2)).view(b, HKV, t, G, n) / math.sqrt(D)
    where = (_positions(s) + torch.arange(t, device="cuda"))[..., None]  # [b, t, 1]
    key = torch.arange(n, device="cuda")
    seen = key <= where
    if c["window"]:
        seen &= (key < c["sinks"]) | (key > where - c["window"])
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(b * HKV, t * G, n), x[:, 1].reshape(b * HKV, n, D))
    o = o.view(b, HKV, t, G, D).permute(0, 2, 1, 3, 4).reshape(b, t, HQ, D)
    s["out"].copy_(o / (1 + torch.exp(-s["gate"].to(F32))))
    if "weights" in s:
        s["weights"][:, :, :n] += p[:, :, t - c.get("observed", 1):].sum((2, 3))
    return _answer(s)


def _plain_evict(s):
    c = s["case"]
    n, keep, sinks, recent = c["context"], c["keep"], c["sinks"], c["recent"]
    place = torch.arange(n, device="cuda")
    always = (place < sinks) | (place >= n - recent)
    rank = torch.where(always, math.inf, s["weights"])
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :keep].sort(-1).values
    s["kept"].copy_(kept)
    s["out_weights"].copy_(torch.gather(s["weights"], 1, kept))
    rows, scales = _views(s["cache"], n, c["fp8"])
    to, to_scales = _views(s["out_cache"], keep, c["out_fp8"])
    taken = kept[None, :, :, None].expand(2, HKV, keep, D)
    if not c["out_fp8"]:
        to[0] = torch.gather(rows[0], 2, taken)
    else:
        x = torch.gather(rows[0], 2, taken)
        x = x.view(torch.float8_e4m3fn).to(F32) * torch.gather(scales[0], 2, (kept // BLOCK).expand(2, HKV, keep))[..., None] if c["fp8"] else x.to(F32)
        padded = torch.nn.functional.pad(x, (0, 0, 0, _blocks(keep) * BLOCK - keep)).view(2, HKV, -1, BLOCK * D)
        to_scales[0] = _pow2_scale(padded.abs().amax(-1))
        to[0] = _codes(x, to_scales[0].repeat_interleave(BLOCK, -1)[..., :keep, None])
    return _answer(s)


def _answer(s):
    """The call's outputs and the state that it updated, without copies."""
    c = s["case"]
    if c["kind"] == "evict":
        rows, scales = _views(s["out_cache"], c["keep"], c["out_fp8"])
        r = {"kept": s["kept"], "weights": s["out_weights"]}
    else:
        rows, scales = _views(s["cache"], c["max_context"], c["fp8"])
        r = {"out": s["out"]}
        if "weights" in s:
            r["weights"] = s["weights"]
    if scales is None:
        return {**r, "cache": rows}
    return {**r, "cache": rows.view(torch.float8_e4m3fn), "scales": scales}


# ------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    if not own:
        return _plain_evict(state) if c["kind"] == "evict" else _plain_attention(state)
    from raftinfer_amd import ops
    dtype = ops.CACHE_FP8_E4M3 if c["fp8"] else ops.CACHE_BF16
    if c["kind"] == "evict":
        shape = ops.Qwen35EvictShape(HKV, D, c["context"], c["context"], c["keep"], c["keep"], c["sinks"], c["recent"])
        ops.qwen35_compact_cache_evict(state["cache"], state["weights"], state["out_cache"], state["out_weights"], state["kept"],
                                       shape, dtype, ops.CACHE_FP8_E4M3 if c["out_fp8"] else ops.CACHE_BF16, ops.HEAD_MAJOR,
                                       state["workspace"])
        return _answer(state)
    if c["kind"] == "decode":
        shape = ops.Qwen35CompactShape(1, c["sequences"], HQ, HKV, D, c["max_context"], c["context"] - 1, state["cache"].shape[1],
                                       c["window"], c["sinks"], 1 if c["weights"] else 0)
        ops.qwen35_compact_attention_decode(state["q"], state["k"], state["v"], state["gate"], state["out"], state["cache"], shape,
                                            ops.DTYPE_BF16, dtype, ops.HEAD_MAJOR, state["workspace"],
                                            context_lengths=state.get("lengths"), key_weights=state.get("weights"))
        return _answer(state)
    shape = ops.Qwen35CompactShape(c["tokens"], 1, HQ, HKV, D, c["max_context"], c["past"], state["cache"].shape[1], c["window"],
                                   c["sinks"], c["observed"])
    ops.qwen35_compact_attention_prefill(state["q"], state["k"], state["v"], state["gate"], state["out"], state["cache"], shape,
                                         ops.DTYPE_BF16, dtype, ops.HEAD_MAJOR, state["workspace"], key_weights=state.get("weights"))
    return _answer(state)


# ------------------------------------------------------------------ floors

def _seen(position, window, sinks):
    """How many keys a token at `position` sees."""
    n = position + 1
    return n if not window else min(n, window + min(sinks, max(0, n - window)))


def work(case):
    row = 2 * HKV * D * (1 if case["fp8"] else 2)  # one position's K and V
    if case["kind"] == "evict":
        n, keep = case["context"], case["keep"]
        out_row = 2 * HKV * D * (1 if case["out_fp8"] else 2)
        return {"bytes": HKV * (4 * n + 8 * keep) + keep * (row + out_row), "flops": 0}
    w, k = case["window"], case["sinks"]
    if case["kind"] == "decode":
        b, c = case["sequences"], case["context"]
        # the lengths of a batch are uniform in 1 .. context
        keys = _seen(c - 1, w, k) if b == 1 else b * sum(_seen(p, w, k) for p in range(0, c, max(1, c // 997))) / len(range(0, c, max(1, c // 997)))
        return {"bytes": keys * row + b * (HQ * D * 6 + HKV * D * 4 + row) + (8 * HKV * keys if case["weights"] else 0),
                "flops": 4 * D * HQ * keys}
    t, past = case["tokens"], case["past"]
    pairs = sum(_seen(past + i, w, k) for i in range(t))
    read = past if not w else min(past, max(0, min(past, w - 1) + min(k, max(0, past - w + 1))))
    return {"bytes": (read + t) * row + t * (HQ * D * 6 + HKV * D * 4) + (8 * HKV * (past + t) if case["observed"] else 0),
            "flops": 4 * D * HQ * pairs}


# ------------------------------------------------------------------ the definition in 64 bits

def _nearest_code(x):
    """The e4m3 value nearest to x (64 bits, |x| <= 448), halves to the even one."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _smallest_scale(size):
    e = torch.ceil(torch.log2(size.clamp(min=1e-300) / TOP))
    e = e - (torch.exp2(e - 1) * TOP >= size).double()  # the logarithm's rounding, either way
    return torch.exp2((e + (torch.exp2(e) * TOP < size).double()).clamp(min=-126))


def _exact_attention(case, seed):
    s = prepare(case, seed)
    b, t, cap, fp8 = case.get("sequences", 1), case.get("tokens", 1), case["max_context"], case["fp8"]
    rows, scales = _views(s["cache"], cap, fp8)
    held, marks = [], []
    out = torch.zeros(b, t, HQ, D, device="cuda", dtype=F64)
    weights = s["weights"].double() if "weights" in s else None
    codes = torch.empty(rows.shape, device="cuda", dtype=F32 if fp8 else torch.bfloat16)
    for i in range(b):
        past = int(s["lengths"][i]) - 1 if "lengths" in s else case.get("past", case.get("context", 1) - 1)
        n = past + t
        for plane, new in ((0, s["k"]), (1, s["v"])):
            c = rows[i, plane].view(torch.float8_e4m3fn).float() if fp8 else rows[i, plane].clone()
            if not fp8:
                c[:, past:n] = new[i].transpose(0, 1)
            else:
                for blk in range(past // BLOCK, _blocks(n)):
                    lo, hi = blk * BLOCK, min(n, blk * BLOCK + BLOCK)
                    mid = max(lo, past)
                    x = new[i, mid - past:hi - past].transpose(0, 1).double()
                    scale = _smallest_scale(x.abs().amax((1, 2)))
                    if mid > lo:
                        was = scales[i, plane, :, blk].double()
                        scale = torch.maximum(scale, was)
                        c[:, lo:mid] = _nearest_code(c[:, lo:mid].double() * (was / scale)[:, None, None]).float()
                    scales[i, plane, :, blk] = scale.float()
                    c[:, mid:hi] = _nearest_code(x / scale[:, None, None]).float()
            codes[i, plane] = c
        for h in range(HKV):
            kv = codes[i, :, h, :n].double()
            if fp8:
                kv = kv * scales[i, :, h, torch.arange(n, device="cuda") // BLOCK].double()[..., None]
            key = torch.arange(n, device="cuda")
            for a in range(0, t, 512):
                e = min(t, a + 512)
                q = s["q"][i, a:e, h * G:(h + 1) * G].double().reshape(-1, D)
                here = torch.arange(past + a, past + e, device="cuda").repeat_interleave(G)[:, None]
                hidden = key > here
                if case["window"]:
                    hidden = hidden | ((key <= here - case["window"]) & (key >= case["sinks"]))
                p = torch.softmax((q @ kv[0].T / 16.0).masked_fill(hidden, -math.inf), -1)
                out[i, a:e, h * G:(h + 1) * G] = (p @ kv[1]).view(e - a, G, D)
                if weights is not None:
                    first = t - case.get("observed", 1)
                    if e > first:
                        weights[i, h, :n] += p[max(0, first - a) * G:].sum(0)
    out *= torch.sigmoid(s["gate"].double())
    r = {"out": out, "cache": codes}
    if fp8:
        r["scales"] = scales
    if weights is not None:
        r["weights"] = weights
    return r


def _exact_evict(case, seed):
    s = prepare(case, seed)
    n, keep = case["context"], case["keep"]
    rows, scales = _views(s["cache"], n, case["fp8"])
    w = s["weights"]
    kept = torch.empty(HKV, keep, device="cuda", dtype=torch.long)
    cache = torch.empty(1, 2, HKV, keep, D, device="cuda", dtype=F32 if case["out_fp8"] else torch.bfloat16)
    out_scales = torch.empty(1, 2, HKV, _blocks(keep), device="cuda")
    end = n - case["recent"]
    for h in range(HKV):
        middle = w[h, case["sinks"]:max(end, case["sinks"])].double().cpu().tolist()
        order = sorted(range(len(middle)), key=lambda i: (-middle[i], i))[:keep - (n - len(middle))]
        rest = [i for i in range(n) if i < case["sinks"] or i >= end]
        kept[h] = torch.tensor(sorted(rest + [case["sinks"] + i for i in order])[:keep], device="cuda")
        x = rows[0, :, h].view(torch.float8_e4m3fn).float() if case["fp8"] else rows[0, :, h]
        x = x[:, kept[h]]
        if not case["out_fp8"]:
            cache[0, :, h] = x
            continue
        x = x.double()
        if case["fp8"]:
            x = x * scales[0, :, h, kept[h] // BLOCK].double()[..., None]
        for blk in range(_blocks(keep)):
            part = x[:, blk * BLOCK:(blk + 1) * BLOCK]
            scale = _smallest_scale(part.abs().amax((1, 2)))
            out_scales[0, :, h, blk] = scale.float()
            cache[0, :, h, blk * BLOCK:(blk + 1) * BLOCK] = _nearest_code(part / scale[:, None, None]).float()
    r = {"kept": None, "weights": torch.gather(w, 1, kept).double(), "cache": cache}
    if case["out_fp8"]:
        r["scales"] = out_scales
    return r


def exact(case, seed):
    return _exact_evict(case, seed) if case["kind"] == "evict" else _exact_attention(case, seed)
