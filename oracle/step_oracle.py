"""Plain float64 statements of the decode step's other operators (include/w4a8_step.h):
rope and the cache append, paged attention, the residual norms, the sampler's draw. NumPy only."""

from __future__ import annotations

import math
from fractions import Fraction

import numpy as np


def _arctan_of_inverse(n: int, one: int) -> int:
    """arctan(1 / n) one, by its series in integers."""
    total, power, i = 0, one // n, 1
    while power:
        total += power // i if i % 4 == 1 else -(power // i)
        power //= n * n
        i += 2
    return total


# 2 pi to 300 bits (Machin's formula).
_TURN = Fraction(2 * (16 * _arctan_of_inverse(5, 1 << 320) - 4 * _arctan_of_inverse(239, 1 << 320)), 1 << 320)


def angles(pos: np.ndarray, freq: float) -> np.ndarray:
    """pos * freq radians: the float64 product where it is exact (24 bits of freq times 29 of pos), else what is left of
    the exact product by the nearest multiple of 2 pi."""
    out = pos.astype(np.float64) * float(freq)
    for i in np.nonzero(pos >= 2 ** 29)[0]:
        a = Fraction(int(pos[i])) * Fraction(float(freq))
        out[i] = float(a - round(a / _TURN) * _TURN)
    return out


def rope(x: np.ndarray, pos: np.ndarray, inv_freq: np.ndarray, interleaved: bool) -> np.ndarray:
    """x [m, heads, d] with its first 2 * len(inv_freq) dimensions turned by pos * inv_freq."""
    x = x.astype(np.float64)
    y = x.copy()
    half = inv_freq.size
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = angles(pos, inv_freq[i])
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        y[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
        y[:, :, b] = x[:, :, b] * c + x[:, :, a] * s
    return y


def cached(cache: np.ndarray, row: np.ndarray, pos: int):
    """The positions 0 .. pos of one row of a page table that the cache holds, in order: [n, kv_heads, d]."""
    page_size = cache.shape[2]
    out = []
    for j in range(min(pos + 1, row.size * page_size)):
        p = int(row[j // page_size])
        if 0 <= p < cache.shape[0]:
            out.append(cache[p, :, j % page_size])
    return np.stack(out).astype(np.float64) if out else np.zeros((0, cache.shape[1], cache.shape[3]))


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, table: np.ndarray, pos: np.ndarray, scale: float):
    """(out [m, heads, d], bound [m, heads]): the attention, and the largest |error| a float32 evaluation may have
    from it. q [m, heads, d] float32; k, v [pages, kv_heads, page_size, d] holding the cached 16-bit values.

    The bound, u = 2^-24. A score is a sum of d products of q's 22 bits or more with the cache's values: off by
    scale * sum|q k| * (2^-21 + (d + 2) u) at most (the split, the products' sum in any order, scale and log2 e
    folded into q). The exponential turns an error e of the score into a relative one of 2 e (e small), plus 4 u of
    its own and 2^-21 where it is split. The sums of p v and p over n keys run in chains of at most n / 32 + 128
    terms (32 keys to a step, partial sums joined after); both, the quotient and the joining factors add that many
    u each."""
    m, heads, d = q.shape
    group = heads // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros((m, heads))
    u = 2.0 ** -24
    for i in range(m):
        keys, vals = cached(k, table[i], int(pos[i])), cached(v, table[i], int(pos[i]))
        if not len(keys):
            continue
        for h in range(heads):
            qk = keys[:, h // group] * q[i, h].astype(np.float64)
            s = scale * qk.sum(-1)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vals[:, h // group]
            e = np.max(abs(scale) * np.abs(qk).sum(-1)) * (2.0 ** -21 + (d + 2) * u) + np.max(np.abs(s)) * 4 * u
            bound[i, h] = np.max(np.abs(vals[:, h // group])) * (4 * e + 2.0 ** -20 + 2 * (len(keys) / 32 + 128) * u)
    return out, bound


def residual(x, y, scale, gate=None, post=None):
    """x + scale * gate * t in float32, one operation at a time, t = y or post (rmsnorm(y) * post_w, given)."""
    t = y if post is None else post
    if gate is not None:
        t = gate * t
    return x + np.float32(scale) * t


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> int:
    """One row's token, with masses as integers of 2^-44 (Python's, so exact)."""
    one = 1 << 44
    f = lambda v: float(np.float32(v))  # noqa: E731  (the settings are float32)
    temperature, top_p, min_p, u = f(temperature), f(top_p), f(min_p), f(u)
    live = [(-float(l), i) for i, l in enumerate(logits) if l > -math.inf]
    if not live:
        return -1
    live.sort()
    top = -live[0][0]
    kept = []
    for neg, i in live:
        l = -neg
        if l == top:
            w = one
        elif top == math.inf:
            w = 0
        else:
            w = int(math.exp((l - top) * (1.0 / temperature)) * one + 0.5) if temperature > 0 else 0
        if w:
            kept.append((i, w))
    if not temperature > 0:
        return kept[0][0]
    if top_k > 0:
        kept = kept[:top_k]
    if top_p < 1:
        total, mass, n = sum(w for _, w in kept), 0, 0
        need = math.ceil(top_p * float(total))
        while n < len(kept) and (n == 0 or mass < need):
            mass += kept[n][1]
            n += 1
        kept = kept[:n]
    if min_p > 0:
        kept = [t for n, t in enumerate(kept) if n == 0 or t[1] >= min_p * one]
    total = sum(w for _, w in kept)
    target = total - 1 if u >= 1 else min(int(u * float(total)), total - 1) if u > 0 else 0
    for i, w in kept:
        if target < w:
            return i
        target -= w
    return kept[-1][0]
