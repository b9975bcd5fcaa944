"""The paged KV cache of a serving program, as measurable cases.

Four operators that belong together: rotary positions of query and key heads (the two halves of the rotated part
paired, or neighbours; part of the head; frequencies scaled for long contexts; with or without the heads' RMSNorm);
the same with the store of a ragged batch's new keys and values in cache pages; gated attention of the batch's new
tokens, a chunk of every sequence, over the pages; and its form for one new token of every sequence.  Heads are the
model's: 16 query / 4 KV heads of 256 dims, of which 64 are rotated with base 1e7.

A pool holds pages of `page_tokens` positions, [page][K, V][kv_head][position][256] (head-major) or
[page][K, V][position][kv_head][256]; row s of the page table names the pages of sequence s in the order of its
positions.  A sequence of context length c with n new tokens has them at positions c - n .. c - 1, in the call's rows
starts[s] .. starts[s + 1] - 1.

    import perf.more_operators as c
    state = c.prepare(c.listed()[0], seed=1)
    outputs = c.run(state)
"""
from __future__ import annotations

import math

import torch

own = False

HQ, HKV, D = 16, 4, 256
G = HQ // HKV
BASE = 1e7
EPS = 1e-6
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

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
        # The query heads of one token out of the query / gate projection: latency.
        {"name": "rotary_step", "kind": "rotary", "rows": 1, "heads": 16, "dim": 256, "rotary": 64, "interleaved": False, "scaling": "none",
         "factor": 1.0, "positions": 4096, "dtype": "bf16", "norm": True, "strided": True},
        # A long prompt's query heads at far positions, neighbours paired, half of the head rotated, frequencies scaled by eight.
        {"name": "rotary_prompt", "kind": "rotary", "rows": 6001, "heads": 16, "dim": 256, "rotary": 128, "interleaved": True, "scaling": "turns",
         "factor": 8.0, "positions": 1048576, "dtype": "bf16", "norm": False, "strided": False},
        # One new token of each of 32 sequences: norm, rotation and store, pages of 16.
        {"name": "append_batch", "kind": "append", "sequences": 32, "singles": 31, "tokens": 1, "context": 2048, "page_tokens": 16,
         "head_major": True, "rotary": 64, "interleaved": False, "scaling": "none", "factor": 1.0},
        # Three long chunks, token-major pages of 64, frequencies scaled by four; pages begin and end inside the chunks.
        {"name": "append_prompt", "kind": "append", "sequences": 3, "singles": 0, "tokens": 2501, "context": 6001, "page_tokens": 64,
         "head_major": False, "rotary": 64, "interleaved": False, "scaling": "pairs", "factor": 4.0},
        # A short question behind a short past: latency and launches.
        {"name": "prefill_few", "kind": "prefill", "sequences": 1, "singles": 0, "tokens": 16, "context": 217, "page_tokens": 16,
         "head_major": True, "window": 0, "gate": True},
        # The prompt bucket of 512 tokens, start of a prompt.
        {"name": "prefill_512", "kind": "prefill", "sequences": 1, "singles": 0, "tokens": 512, "context": 512, "page_tokens": 16,
         "head_major": True, "window": 0, "gate": True},
        # A serving step: 10 sequences decode one token, 6 take chunks of up to 500, contexts of up to 8192 behind a window.
        {"name": "prefill_batch", "kind": "prefill", "sequences": 16, "singles": 10, "tokens": 500, "context": 8192, "page_tokens": 16,
         "head_major": True, "window": 4096, "gate": True},
        # A later chunk of a long document, behind a past that ends inside a page.
        {"name": "prefill_chunk", "kind": "prefill", "sequences": 1, "singles": 0, "tokens": 500, "context": 30501, "page_tokens": 64,
         "head_major": True, "window": 0, "gate": True},
        # A long prompt, token-major pages, ragged end.
        {"name": "prefill_long", "kind": "prefill", "sequences": 1, "singles": 0, "tokens": 8001, "context": 8001, "page_tokens": 128,
         "head_major": False, "window": 0, "gate": True},
        # One token of a short chat: latency and launches.
        {"name": "decode_short", "kind": "decode", "sequences": 1, "singles": 1, "tokens": 1, "context": 201, "page_tokens": 16,
         "head_major": True, "window": 0, "gate": True},
        # One token of a long document, ragged end.
        {"name": "decode_long", "kind": "decode", "sequences": 1, "singles": 1, "tokens": 1, "context": 60001, "page_tokens": 64,
         "head_major": True, "window": 0, "gate": True},
        # A serving batch of 32 sequences of very different lengths.
        {"name": "decode_batch", "kind": "decode", "sequences": 32, "singles": 32, "tokens": 1, "context": 32768, "page_tokens": 16,
         "head_major": True, "window": 0, "gate": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "prefill", "prefill", "decode", "decode"])
    scaling = rng.choice(["none", "linear", "pairs", "turns"])
    factor = 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256, 256])
        return {"kind": kind, "rows": _log_int(rng, 1, 6001), "heads": rng.choice([1, 4, 5, 16]), "dim": dim,
                "rotary": rng.choice([d for d in (dim // 4 // 2 * 2, dim // 2, dim)]), "interleaved": rng.random() < 0.5,
                "scaling": scaling, "factor": factor, "positions": _log_int(rng, 512, 1048576),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "norm": rng.random() < 0.5, "strided": rng.random() < 0.5}
    page_tokens = rng.choice([16, 16, 32, 48, 64, 128, 256])
    head_major = rng.random() < 0.7
    sequences = rng.choice([1, 1, _log_int(rng, 2, 32)])
    if kind == "decode":
        context = _log_int(rng, 1, 60001) if sequences == 1 else _log_int(rng, 100, 24000)
        return {"kind": kind, "sequences": sequences, "singles": sequences, "tokens": 1, "context": context, "page_tokens": page_tokens,
                "head_major": head_major, "window": _log_int(rng, 1, 8192) if rng.random() < 0.3 else 0, "gate": rng.random() < 0.8}
    singles = rng.randint(0, sequences - 1)
    if sequences > 1:
        tokens = _log_int(rng, 2, 500)
        context = tokens + _log_int(rng, 1, 8192 - tokens) if rng.random() < 0.7 else tokens
    elif rng.random() < 0.5:  # a chunk behind a past
        tokens = _log_int(rng, 2, 500)
        context = tokens + _log_int(rng, 1, 30001)
    else:                     # a whole prompt
        tokens = context = _log_int(rng, 2, 8001)
    if kind == "append":
        return {"kind": kind, "sequences": sequences, "singles": singles, "tokens": tokens, "context": min(context, 8192 + tokens), "page_tokens": page_tokens,
                "head_major": head_major, "rotary": rng.choice([64, 64, 32, 128, 256]), "interleaved": rng.random() < 0.5,
                "scaling": scaling, "factor": factor}
    if sequences > 16:
        context = min(context, 4096)
    return {"kind": kind, "sequences": sequences, "singles": singles, "tokens": tokens, "context": context, "page_tokens": page_tokens,
            "head_major": head_major, "window": _log_int(rng, 1, 8192) if rng.random() < 0.3 else 0, "gate": rng.random() < 0.8}


def lengths(case):
    """(new tokens, context) of each sequence: `singles` of them have one new token, the others up to `tokens`, and
    contexts reach from short to the case's."""
    some = case["sequences"] - case["singles"]
    got = []
    for s in range(case["sequences"]):
        n = 1 if s < case["singles"] else max(1, case["tokens"] * (s - case["singles"] + 1) // max(1, some))
        k = s if s < case["singles"] else case["sequences"] - 1 - (s - case["singles"])
        got.append((n, n + (case["context"] - case["tokens"]) * (k + 1) // case["sequences"]))
    return got


# ------------------------------------------------------------------ inputs

def frequencies(rotary, scaling, factor, trained=32768, fast=32.0, slow=1.0):
    """(radians per position of every pair, what cos and sin are multiplied by).  Of positions further than a model was
    trained on: all frequencies divided by the factor (linear); or the slow ones, those of the fast ones left, with a
    passage between `slow` and `fast` turns over the trained context that is linear in the pair (pairs) or in the
    turns (turns)."""
    f = [BASE ** (-2 * p / rotary) for p in range(rotary // 2)]
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if scaling == "turns":
        kept = [min(1.0, max(0.0, (trained * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
        return [x * k + x / factor * (1 - k) for x, k in zip(f, kept)], 1.0
    at = lambda turns: rotary * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(BASE))  # noqa: E731
    low, high = max(0, math.floor(at(fast))), min(rotary - 1, math.ceil(at(slow)))
    kept = [1 - min(1.0, max(0.0, (p - low) / max(high - low, 1e-3))) for p in range(rotary // 2)]
    return [x * k + x / factor * (1 - k) for x, k in zip(f, kept)], 0.1 * math.log(factor) + 1


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _rows(g, *shape):
    """K or V rows of a layer: about 1% of them eight times as large, so that the softmax has maxima to find."""
    x = _randn(g, *shape)
    x *= 1 + 7 * (torch.rand(shape[:-1] + (1,), generator=g, device="cuda") < 0.01)
    return x


def prepare(case, seed):
    stream()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["kind"] in ("rotary", "append"):
        f, s["magnitude"] = frequencies(case["rotary"], case["scaling"], case["factor"])
        s["frequencies"] = torch.tensor(f, dtype=F64, device="cuda")
    if case["kind"] == "rotary":
        dtype, rows, heads, dim = TYPES[case["dtype"]], case["rows"], case["heads"], case["dim"]
        # strided: the query half of a projection [rows][heads][query, gate][dim]
        s["x"] = _randn(g, rows, heads, 2, dim, dtype=dtype)[:, :, 0] if case["strided"] else _randn(g, rows, heads, dim, dtype=dtype)
        s["weight"] = (1 + 0.1 * _randn(g, dim, dtype=F32)).to(dtype) if case["norm"] else None
        s["positions"] = torch.randint(0, case["positions"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["out"] = torch.empty(rows, heads, dim, device="cuda", dtype=dtype)
        return s
    each, page = lengths(case), case["page_tokens"]
    order = torch.randperm(len(each), generator=g, device="cuda").tolist()
    each = [each[i] for i in order]
    rows = sum(n for n, _ in each)
    need = [-(-c // page) for _, c in each]
    pool = sum(need) + 3
    s["starts"] = torch.tensor([sum(n for n, _ in each[:i]) for i in range(len(each) + 1)], dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor([c for _, c in each], dtype=torch.int32, device="cuda")
    # the pool's pages in no order; entries behind a sequence's last page name none
    where = torch.randperm(pool, generator=g, device="cuda", dtype=torch.int32)
    s["table"] = torch.full((len(each), max(need)), -1, dtype=torch.int32, device="cuda")
    for i, k in enumerate(need):
        s["table"][i, :k] = where[sum(need[:i]):sum(need[:i + 1])]
    s["pages"] = _rows(g, *((pool, 2, HKV, page, D) if case["head_major"] else (pool, 2, page, HKV, D)))
    s["rows"] = rows
    s["max_context"] = case["context"]
    s["projection"] = _randn(g, rows, HQ, 2, D)  # query and gate of every head, as the projection leaves them
    s["gate"] = s["projection"][:, :, 1] if case.get("gate") else None
    if case["kind"] == "append":
        s["k"], s["v"] = _rows(g, rows, HKV, D), _rows(g, rows, HKV, D)
        s["q_weight"], s["k_weight"] = 1 + 0.1 * _randn(g, D), 1 + 0.1 * _randn(g, D)
        s["q"] = torch.empty(rows, HQ, D, device="cuda", dtype=torch.bfloat16)
    else:
        s["q"] = _randn(g, rows, HQ, D)
        s["out"] = torch.empty(rows, HQ, D, device="cuda", dtype=torch.bfloat16)
        s["workspace"] = torch.empty(512 << 20, device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------------ plain form

def _plain_rotated(x, weight, positions, s):
    """x [rows, heads, dim]: RMSNorm, then the rotation of the first dims by the rows' positions, in 32 bits."""
    c = s["case"]
    x = x.to(F32)
    if weight is not None:
        x = x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * weight.to(F32)
    theta = positions.to(F64)[:, None, None] * s["frequencies"]
    cos, sin = (torch.cos(theta) * s["magnitude"]).to(F32), (torch.sin(theta) * s["magnitude"]).to(F32)
    part, rest = x[..., :c["rotary"]], x[..., c["rotary"]:]
    if c["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = part[..., :c["rotary"] // 2], part[..., c["rotary"] // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1)


def _plain_rotary(s):
    s["out"].copy_(_plain_rotated(s["x"], s["weight"], s["positions"], s))
    return {"out": s["out"]}


def _places(s):
    """(sequence, token, position) of every row."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    token = row - s["starts"].long()[seq]
    return seq, token, (s["lengths"].long() - s["starts"].long().diff())[seq] + token


def _plain_append(s):
    page = s["case"]["page_tokens"]
    seq, _, position = _places(s)
    s["q"].copy_(_plain_rotated(s["projection"][:, :, 0], s["q_weight"], position, s))
    k = _plain_rotated(s["k"], s["k_weight"], position, s).to(torch.bfloat16)
    to, at = s["table"][seq, position // page].long(), position % page
    if s["case"]["head_major"]:
        s["pages"][to, 0, :, at], s["pages"][to, 1, :, at] = k, s["v"]
    else:
        s["pages"][to, 0, at], s["pages"][to, 1, at] = k, s["v"]
    return {"q": s["q"], "pages": s["pages"]}


def _plain_attention(s):
    c = s["case"]
    n, page, b = c["tokens"], c["page_tokens"], c["sequences"]
    most = min(c["context"], page * s["table"].shape[1])
    seq, token, position = _places(s)
    key = torch.arange(most, device="cuda")
    to = s["table"].long()[:, key // page].clamp(min=0)                                  # [b, most]
    held = [(s["pages"][to, i, :, key % page] if c["head_major"] else s["pages"][to, i, key % page]) for i in (0, 1)]
    k, v = (x.to(F32).permute(0, 2, 1, 3).reshape(b * HKV, most, D) for x in held)
    q = torch.zeros(b, n, HQ, D, device="cuda")
    q[seq, token] = s["q"].to(F32)
    q = q.view(b, n, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(b * HKV, n * G, D)
    score = torch.bmm(q, k.transpose(1, 2)).view(b, HKV, n, G, most) / math.sqrt(D)
    first = s["lengths"].long() - s["starts"].long().diff()
    where = (first[:, None] + torch.arange(n, device="cuda"))[..., None]                 # [b, n, 1]
    seen = key <= where
    if c["window"]:
        seen &= key > where - c["window"]
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(b * HKV, n * G, most), v).view(b, HKV, n, G, D).permute(0, 2, 1, 3, 4).reshape(b, n, HQ, D)[seq, token]
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].to(F32)))
    s["out"].copy_(o)
    return {"out": s["out"]}


# ------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append}.get(c["kind"], _plain_attention)(state)
    from raftinfer_amd import ops
    if c["kind"] == "rotary":
        shape = ops.Qwen35RotaryShape(c["rows"], c["heads"], c["dim"], c["rotary"], interleaved=c["interleaved"], magnitude=state["magnitude"])
        ops.qwen35_rotary(state["x"], state["weight"], state["out"], state["positions"], state["frequencies"], shape, EPS)
        return {"out": state["out"]}
    layout = ops.HEAD_MAJOR if c["head_major"] else ops.TOKEN_MAJOR
    shape = ops.Qwen35PagedShape(state["rows"], c["sequences"], HQ, HKV, D, state["pages"].shape[0], c["page_tokens"], state["table"].shape[1],
                                 state["max_context"], c.get("window", 0))
    if c["kind"] == "append":
        rotary = ops.Qwen35PagedRotary(c["rotary"], interleaved=c["interleaved"], magnitude=state["magnitude"], epsilon=EPS)
        ops.qwen35_paged_cache_append(state["projection"][:, :, 0], state["k"], state["v"], state["q"], state["pages"], state["table"], state["starts"],
                                      state["lengths"], state["frequencies"], state["q_weight"], state["k_weight"], shape, rotary, layout)
        return {"q": state["q"], "pages": state["pages"]}
    if c["kind"] == "decode":
        ops.qwen35_paged_attention_decode(state["q"], state["gate"], state["out"], state["pages"], state["table"], state["lengths"], state["workspace"],
                                          shape, layout)
    else:
        ops.qwen35_paged_attention_prefill(state["q"], state["gate"], state["out"], state["pages"], state["table"], state["starts"], state["lengths"],
                                           state["workspace"], shape, layout)
    return {"out": state["out"]}


# ------------------------------------------------------------------ floors

def work(case):
    if case["kind"] == "rotary":
        size, values = (4 if case["dtype"] == "f32" else 2), case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * size + 4 * case["rows"] + 4 * case["rotary"], "flops": values * (4 if case["norm"] else 0) + 3 * values * case["rotary"] // case["dim"]}
    each = lengths(case)
    rows = sum(n for n, _ in each)
    table = 4 * sum(-(-c // case["page_tokens"]) for _, c in each) + 8 * len(each)
    if case["kind"] == "append":
        return {"bytes": rows * 2 * (HQ + 2 * HKV) * D * 2 + 8 * len(each) + 4 * rows // case["page_tokens"], "flops": rows * (HQ + HKV) * (4 * D + 3 * case["rotary"])}
    seen = read = 0
    for n, c in each:
        past, window = c - n, case["window"] or c
        read += c - max(0, past + 1 - window)
        # tokens at positions past .. c - 1 see position + 1 keys, window at most
        grow = max(0, min(c, window) - past)
        seen += grow * past + grow * (grow + 1) // 2 + (n - grow) * window
    return {"bytes": read * 2 * HKV * D * 2 + rows * (3 if case["gate"] else 2) * HQ * D * 2 + table, "flops": 4 * HQ * D * seen}


# ------------------------------------------------------------------ 64 bits

def _exact_turned(x, weight, positions, case, f, magnitude):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    y = x.clone()
    for p, w in enumerate(f):
        i, j = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + len(f))
        angle = positions.double()[:, None] * w
        y[..., i] = magnitude * (x[..., i] * torch.cos(angle) - x[..., j] * torch.sin(angle))
        y[..., j] = magnitude * (x[..., j] * torch.cos(angle) + x[..., i] * torch.sin(angle))
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return {"out": _exact_turned(s["x"], s["weight"], s["positions"], case, s["frequencies"].tolist(), s["magnitude"])}
    starts, ends, table, page = s["starts"].tolist(), s["lengths"].tolist(), s["table"].long(), case["page_tokens"]
    if case["kind"] == "append":
        f, pages, q = s["frequencies"].tolist(), s["pages"].double(), torch.empty(s["rows"], HQ, D, device="cuda", dtype=F64)
        for i, c in enumerate(ends):
            a, e = starts[i], starts[i + 1]
            at = torch.arange(c - (e - a), c, device="cuda")
            q[a:e] = _exact_turned(s["projection"][a:e, :, 0], s["q_weight"], at, case, f, s["magnitude"])
            k = _exact_turned(s["k"][a:e], s["k_weight"], at, case, f, s["magnitude"])
            for h in range(HKV):
                for plane, x in ((0, k), (1, s["v"].double()[a:e])):
                    where = (table[i, at // page], plane, h, at % page) if case["head_major"] else (table[i, at // page], plane, at % page, h)
                    pages[where] = x[:, h]
        return {"q": q, "pages": pages}
    out = torch.empty(s["rows"], HQ, D, device="cuda", dtype=F64)
    for i, c in enumerate(ends):
        a, e = (starts[i], starts[i + 1]) if case["kind"] == "prefill" else (i, i + 1)
        key = torch.arange(c, device="cuda")
        for h in range(HKV):
            k, v = (s["pages"][(table[i, key // page], plane, h, key % page) if case["head_major"] else (table[i, key // page], plane, key % page, h)].double()
                    for plane in (0, 1))
            for t in range(a, e, 512):
                u = min(e, t + 512)
                x = s["q"][t:u, h * G:(h + 1) * G].double().reshape(-1, D)
                at = torch.arange(c - (e - a) + t - a, c - (e - a) + u - a, device="cuda").repeat_interleave(G)[:, None]
                hidden = key > at
                if case["window"]:
                    hidden = hidden | (at - key >= case["window"])
                p = torch.softmax((x @ k.T / 16.0).masked_fill(hidden, -math.inf), -1)
                out[t:u, h * G:(h + 1) * G] = (p @ v).view(u - t, G, D)
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return {"out": out}
