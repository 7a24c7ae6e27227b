"""CPU oracle (numpy, float64) of the quantised key / value cache: what a cache holds for rows, and attention over it.  TEST
INFRASTRUCTURE ONLY.  The reference has no such cache (simple-llm/src/gpu/gpu_kv_cache.py:66-78 is fp32); this is the definition."""
from __future__ import annotations

import numpy as np

GROUP = 32


def to_bf16(x: np.ndarray) -> np.ndarray:
    """float64 rounded once to the nearest bfloat16 (ties to even), as float64."""
    x = np.asarray(x, dtype=np.float64)
    out = x.copy()
    some = np.isfinite(x) & (x != 0)
    m, e = np.frexp(x[some])                       # x = m * 2^e, 0.5 <= |m| < 1
    step = np.ldexp(1.0, np.maximum(e - 8, -133))  # 8 bits, subnormals down to 2^-133
    out[some] = np.rint(x[some] / step) * step
    return np.where(np.abs(out) >= 2.0 ** 128, np.copysign(np.inf, out), out)


def quantise(x: np.ndarray, bits: int):
    """(codes, scales) of rows [..., D]: codes [..., D] whole numbers, scales [..., D / 32]."""
    top = 7 if bits == 4 else 127
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, GROUP)
    most = np.abs(g).max(-1)
    scales = np.where(np.isfinite(most), to_bf16(np.where(np.isfinite(most), most, 0) / top), np.nan)
    s = scales[..., None]
    with np.errstate(all="ignore"):
        codes = np.where(s > 0, np.clip(np.rint(g / s), -top, top), 0)
    return codes.reshape(x.shape), scales


def held(x: np.ndarray, bits: int) -> np.ndarray:
    codes, scales = quantise(x, bits)
    return codes * np.repeat(scales, GROUP, axis=-1)


def attention(q, k, v, scale, softcap=0.0, window=0, slopes=None):
    """One sequence.  q [m, H, D], k and v [n, G, D] (what the cache holds), query i at place n - m + i -> (out [m, H, D], the mean magnitude
    sum_t w_t |v_t| of what was averaged, and per query and head scale * sum_d |q_d| max |k| over d's group, which bounds what a score was made of)."""
    m, H, D = q.shape
    n, G = k.shape[:2]
    out, mean, size = np.zeros((m, H, D)), np.zeros((m, H, D)), np.zeros((m, H, 1))
    for i in range(m):
        p = n - m + i
        first = max(0, p + 1 - window) if window else 0
        if p < 0:
            continue
        t = np.arange(first, p + 1)
        for h in range(H):
            kk, vv = k[t, h // (H // G)], v[t, h // (H // G)]
            s = kk @ q[i, h] * scale
            most = np.nan_to_num(np.abs(kk)).max(0).reshape(-1, min(GROUP, D)).max(-1)  # of a group: its codes are steps of that
            size[i, h] = np.repeat(most, min(GROUP, D)) @ np.abs(q[i, h]) * abs(scale)
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes[h] * (p - t)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], mean[i, h] = w @ vv, w @ np.abs(vv)
    return out, mean, size


def tolerance(out, mean, size, n, dtype: str, extra: float = 0.0, largest: float = 0.0):
    """How far an output element may be off, from the formulas' roundings:
    - the output's own rounding: half a step, 2^-8 (bfloat16) or 2^-24 of the value;
    - a probability is rounded to 11 bits, and so is its product with a value scale: 2^-10 of the mean magnitude (fp32: 22 bits once, 2^-21);
    - a score is sums over groups of products with codes.  The tensor core adds 16 products and what it had, each cut off 24 bits below the
      largest, twice per group: 34 * 2^-24 of it.  bfloat16: codes as stored, up to 15 where the value's is 7, with 4 bits less: 34 * 2^-20 * 15 / 7.
      The largest product is at most `size`.  It scales probabilities above and below the line;
    - sums over n tokens, 16 at a time: 2^-23 of the mean magnitude each, and as much for their reunion;
    `extra` is an absolute error of scores beyond that (bias, cap).
    - fp16 numbers below 2^-14 lie 2^-24 apart.  A probability is held as a multiple w of 2^-10 of a score that was seen, so their sum is at least
      2^10, a value scale s as s / 2^E < 2: beyond the relative error w is off by up to 2^-25, times that scale, and the product by 2^-25, times a code up
      to L, over that sum: 3 * 2^-35 * 2^E * L.  2^E is at most 4 times the largest scale: 2^-31 * `largest`, the largest magnitude held, per token.
      (It shows where one token has nearly all the weight and a code of zero, and what is left is below 2^-31 of the values.)"""
    bf16 = dtype == "bf16"
    half, held_in = (2.0 ** -8, 2.0 ** -10) if bf16 else (2.0 ** -24, 2.0 ** -21)
    score = 34 * (2.0 ** -20 * 15 / 7 if bf16 else 2.0 ** -24) * size + extra
    summed = 2.0 ** -23 * (n / 16 + 32) * mean
    return half * np.abs(out) + (held_in + 2 * score) * mean + summed + n * 2.0 ** -31 * largest


def largest_seen(v, m, H, window=0):
    """Per query and head, of each element's group: the largest magnitude held among the tokens that the query sees.  v [n, G, D] -> [m, H, D]."""
    n, G, D = v.shape
    most = np.repeat(np.abs(np.nan_to_num(v)).reshape(n, G, D // GROUP, GROUP).max(-1), GROUP, axis=-1)
    out = np.zeros((m, H, D))
    for i in range(m):
        p = n - m + i
        if p >= 0:
            out[i] = np.repeat(most[max(0, p + 1 - window) if window else 0:p + 1].max(0), H // G, axis=0)
    return out


def tolerance_seen(out, mean, size, n, dtype: str, largest, extra: float = 0.0):
    """`tolerance` with nothing allowed for groups and tokens that an element has nothing to do with: `largest` is what `largest_seen` gives.
    Where fp16 numbers are used for a token, its value scale lies within 2^9 of its group's reference 2^E, and its weight is relative to a sum of
    2^10 at least.  Below 2^-14 weight and product are each off by up to 2^-25, the weight's times a scale below 2: 3 * 2^-25 * 2^-10 * 2^E * L,
    and a token that is seen makes L 2^E at most 2^8 * largest: 3 * 2^-27 = 48 * 2^-31 of it per token.  Other tokens' products are sums of 16 bits
    (fp32: 24), which the relative terms cover."""
    return tolerance(out, mean, size, n, dtype, extra, 48.0 * largest)
