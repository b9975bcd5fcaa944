"""64-bit reference of rotary positions and the paged KV cache, from the formulas (numpy, loops over sequences)."""
import math

import numpy as np

HALF_BF16 = 2.0 ** -8  # a rounding to bf16 is off by at most this, relative to the value


def frequencies(rotary_dim, base, scaling="none", factor=1.0, trained=0.0, fast=32.0, slow=1.0):
    """(angles per position, magnitude), scaling: none, linear, pair or turns."""
    out = []
    for p in range(rotary_dim // 2):
        f = base ** (-2.0 * p / rotary_dim)
        keep = 1.0
        if scaling == "linear":
            keep = 0.0
        elif scaling == "turns":
            keep = (trained * f / (2 * math.pi) - slow) / (fast - slow)
        elif scaling == "pair":
            # the pair that turns t times over the trained context: trained base^(-2 p / d) / 2 pi = t
            pair = lambda t: rotary_dim / 2 * math.log(trained / (2 * math.pi * t), base)  # noqa: E731
            first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary_dim - 1)
            keep = 1 - (p - first) / max(last - first, 1e-3)
        keep = min(max(keep, 0.0), 1.0)
        out.append(f if scaling == "none" else keep * f + (1 - keep) * f / factor)
    return out, 0.1 * math.log(factor) + 1 if scaling == "pair" else 1.0


def rotate(x, weight, positions, freq, magnitude, interleaved, epsilon):
    """x [rows, heads, dim] in 64 bits."""
    y = np.array(x, np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + epsilon) * weight
    z = y.copy()
    for p, f in enumerate(freq):
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + len(freq))
        turn = np.array([np.longdouble(int(t)) * np.longdouble(f) % (2 * np.longdouble(np.pi)) for t in positions])
        c, s = np.cos(turn).astype(np.float64)[:, None] * magnitude, np.sin(turn).astype(np.float64)[:, None] * magnitude
        z[..., i], z[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
    return z


def rows_of(pages, table_row, count, page_tokens, head_major):
    """K and V [2, kv_heads, count, 256] of a sequence's first `count` positions; pages as numpy."""
    j = np.arange(count)
    page, at = table_row[j // page_tokens], j % page_tokens
    if head_major:
        return np.stack([pages[page, p, :, at] for p in (0, 1)]).transpose(0, 2, 1, 3)
    return np.stack([pages[page, p, at] for p in (0, 1)]).transpose(0, 2, 1, 3)


def attention(q, gate, kv, context, window=0):
    """One sequence: q [n, heads, 256], gate alike or None, kv [2, kv_heads, context, 256], the n tokens the last of the
    context.  (output, what multiplies a relative error of the probabilities, of the scores) of every value."""
    n, heads, dim = q.shape
    group = heads // kv.shape[1]
    out, spread, reach = np.empty_like(q), np.empty_like(q), np.empty_like(q)
    with np.errstate(all="ignore"):
        for t in range(n):
            p = context - n + t
            lo = max(0, p + 1 - window) if window else 0
            for h in range(heads):
                k, v = kv[0, h // group, lo:p + 1], kv[1, h // group, lo:p + 1]
                s = k @ q[t, h] / 16.0
                e = np.exp(s - s.max())
                w = e / e.sum()
                seen = w != 0  # (NaN among them)
                o = w[seen] @ v[seen] if np.isfinite(v[seen]).all() else (w[seen, None] * v[seen]).sum(0)
                g = 1.0 if gate is None else 1 / (1 + np.exp(-gate[t, h]))
                out[t, h] = o * g
                spread[t, h] = w[seen] @ np.abs(v[seen] - o) * g
                # a sum of 256 products in 32 bits, one after the other, is off by 256 half steps of the sum of their sizes
                off = 256 * 2.0 ** -24 * (np.abs(k) @ np.abs(q[t, h])).max() / 16.0
                reach[t, h] = w[seen] @ np.abs(v[seen]) * g * (2 * off + 2.0 ** -14)
    return out, spread, reach


def tolerance(out, spread, reach, probability_bits=8):
    """An output is rounded to bf16; probabilities are rounded to `probability_bits` bits, and divided by the sum of what
    they were rounded to; scores, sums and the gate are held in 32 bits."""
    return HALF_BF16 * np.abs(out) + 2.0 ** -probability_bits * 1.01 * spread + reach
