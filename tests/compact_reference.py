"""The compact KV cache in 64 bits: e4m3 blocks with power-of-two scales, gated attention behind a sliding
window with sinks, key weights, eviction.  Plain numpy, one step of the definition at a time."""
from __future__ import annotations

import numpy as np

D, BLOCK = 256, 32

# e4m3 values by code: 1 sign, 4 exponent (bias 7) and 3 mantissa bits; 0x7F and 0xFF are NaN.
_e, _m = (np.arange(128) >> 3), (np.arange(128) & 7)
_positive = np.where(_e == 0, _m * 2.0 ** -9, (1 + _m / 8) * 2.0 ** (_e - 7.0))
E4M3 = np.concatenate([_positive, -_positive])
E4M3[[0x7F, 0xFF]] = np.nan


def to_codes(x):
    """Nearest e4m3 code of each |x| <= 448, ties to the even code; NaN -> 0x7F."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isnan(x), 0, x))
    values = _positive[:127]
    hi = np.clip(np.searchsorted(values, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = values[hi] - a, a - values[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(values[hi] == a, hi, code)
    code = np.where(np.signbit(x), code + 128, code)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def scale_for(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    s = 2.0 ** -126
    if amax > 0:
        s = max(s, 2.0 ** np.floor(np.log2(amax / 448)) / 2)
    while amax > 448 * s:
        s *= 2
    return s


class Fp8Cache:
    def __init__(self, kv_heads, positions, rng=None):
        """rng: what the buffer holds before anything is stored."""
        blocks = -(-positions // BLOCK)
        self.codes = np.zeros((2, kv_heads, positions, D), np.uint8)
        self.scales = np.zeros((2, kv_heads, blocks))
        if rng is not None:
            self.codes[:] = rng.integers(0, 256, self.codes.shape)  # NaN codes among them
            self.scales[:] = 2.0 ** rng.integers(-20, 20, self.scales.shape)

    def store(self, past, key, value):
        """key, value [t][kv_heads][D]."""
        t = key.shape[0]
        for plane, rows in ((0, key), (1, value)):
            for h in range(rows.shape[1]):
                for b in range(past // BLOCK, (past + t - 1) // BLOCK + 1):
                    lo, hi = max(past, b * BLOCK), min(past + t, (b + 1) * BLOCK)
                    x = rows[lo - past:hi - past, h].astype(np.float64)
                    x = np.where(np.isfinite(x), x, np.nan)
                    need = scale_for(np.nanmax(np.abs(x), initial=0))
                    scale = need
                    if b * BLOCK < past:
                        was = self.scales[plane, h, b]
                        scale = max(need, was)
                        old = self.codes[plane, h, b * BLOCK:past]
                        if scale != was:
                            self.codes[plane, h, b * BLOCK:past] = to_codes(E4M3[old] * (was / scale))
                    self.scales[plane, h, b] = scale
                    self.codes[plane, h, lo:hi] = to_codes(x / scale)

    def held(self, n):
        per_row = np.repeat(self.scales, BLOCK, -1)[:, :, :n]
        return E4M3[self.codes[:, :, :n]] * per_row[..., None]

    def buffer(self, layout):
        """The library's bytes of one sequence's cache (layout 1 head-major, 0 token-major)."""
        c = self.codes if layout == 1 else self.codes.transpose(0, 2, 1, 3)
        scales = self.scales.astype(np.float32).tobytes()
        return np.frombuffer(np.ascontiguousarray(c).tobytes() + scales + bytes(-len(scales) % 32), np.uint8).copy()

    def load(self, raw, layout):
        n = self.codes.size
        _, h, p, _ = self.codes.shape
        c = raw[:n].reshape((2, h, p, D) if layout == 1 else (2, p, h, D))
        self.codes = (c if layout == 1 else c.transpose(0, 2, 1, 3)).copy()
        self.scales = raw[n:n + 4 * self.scales.size].view(np.float32).astype(np.float64).reshape(self.scales.shape)
        return self


def sees(p, window, sinks, n):
    j = np.arange(n)
    ok = j <= p
    if window:
        ok &= (j < sinks) | (j > p - window)
    return ok


def attention(q, gate, held, past, window=0, sinks=0, observed=0):
    """q, gate [t][heads][D], held [2][kv_heads][past + t][D] -> (out [t][heads][D], bound on the bf16 result's
    distance from out, weights [kv_heads][past + t], their relative bound).

    The bound counts what a kernel may round: q k / 16 in f32 (a sum of 256 products, each partial sum off by at
    most 2^-24 of the sum of magnitudes), the difference from the max and exp2 (2^-20 together), each probability
    to bf16 before the product with V (2^-8), the f32 sums over the keys (2^-24 a step), the result to bf16 (2^-8)."""
    t, heads, _ = q.shape
    kvh, n = held.shape[1], held.shape[2]
    g = heads // kvh
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    weights = np.zeros((kvh, n))
    rel = np.zeros((kvh, n))
    for i in range(t):
        ok = sees(past + i, window, sinks, n)
        for h in range(heads):
            k, v = held[0, h // g][ok], held[1, h // g][ok]
            with np.errstate(invalid="ignore", over="ignore"):
                s = k @ q[i, h].astype(np.float64) / 16
                p = np.exp(s - s.max())
                p /= p.sum()
                size = (np.abs(k) @ np.abs(q[i, h]).astype(np.float64) / 16).max()
                e = 2 * (257 * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(s).max()) + 2.0 ** -20 + len(s) * 2.0 ** -24
                sig = 1 / (1 + np.exp(-gate[i, h].astype(np.float64)))
                out[i, h] = sig * (p @ v)
                bound[i, h] = sig * (2.0 ** -8 + e) * (p @ np.abs(v)) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(out[i, h])
            if i >= t - observed:
                weights[h // g, ok] += p
                rel[h // g] = np.maximum(rel[h // g], e)
    return out, bound, weights, rel + observed * g * 2.0 ** -24


def keep_indices(weights, n, keep, sinks, recent):
    """weights [n] of one head -> kept indices, ascending."""
    w = np.where(np.isnan(weights[:n]), np.inf, weights[:n].astype(np.float64) + 0.0)
    nan = np.isnan(weights[:n])
    middle = list(range(sinks, n - recent))
    middle.sort(key=lambda i: (not nan[i], -w[i], i))
    chosen = middle[:keep - sinks - recent]
    return np.array(sorted(list(range(sinks)) + chosen + list(range(n - recent, n))), np.int64)
