"""Paged attention at the ends of its types' ranges (include/w4a8_step.h) against float64."""

from __future__ import annotations

import math

import numpy as np
import pytest

import step_oracle as S
from gpu_helpers import dev, host
from test_gpu_step import Cached, check_attention

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- the largest finite V


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,heads,kv_heads", [(64, 4, 2), (96, 3, 3), (128, 8, 1), (256, 4, 2)])
@pytest.mark.parametrize("signs", ["plus", "minus", "both"])
def test_attention_largest_finite_values(gpu, dtype, d, heads, kv_heads, signs):
    """V at the ends of its type: a mean of them is no larger than they are, whatever the number of keys and however
    the row is split."""
    import torch
    c = Cached([1, 2, 40, 700, 0, 20011], kv_heads, d, 64, dtype)
    most = torch.finfo(c.dtype).max
    live = ~torch.isnan(c.v)
    c.v[live] = {"plus": torch.full_like(c.v, most), "minus": torch.full_like(c.v, -most),
                 "both": torch.where(c.v > 0, most, -most).to(c.dtype)}[signs][live]
    got = check_attention(gpu, c, heads)
    assert np.isfinite(got).all()
    c = Cached([300], kv_heads, d, 16, dtype)                   # rows of one table
    c.v[~torch.isnan(c.v)] = most
    c.pos = np.array([0, 31, 32, 150, 299], np.int32)
    got = check_attention(gpu, c, heads, table=dev(c.table).expand(5, -1))
    assert np.isfinite(got).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rise", [5.0, 5.5, 9.0])
def test_attention_largest_finite_values_behind_a_rise(gpu, dtype, rise):
    """The first 32 keys score 0, all others `rise` nats: a running maximum that moves late has weights over one."""
    import torch
    n, d = 3000, 64
    c = Cached([n], 1, d, 64, dtype)
    live = ~torch.isnan(c.v)
    c.v[live] = torch.finfo(c.dtype).max
    c.k[live] = 1.0
    c.k[int(c.table[0, 0]), 0, :32] = 0.0
    q = np.full((1, 2 * d), rise / 8, np.float32)               # 64 of them, scale 1 / 8
    got = host(gpu.paged_attention(dev(q), c.k, c.v, dev(c.table), dev(c.pos)))
    k, v = c.arrays()
    want, bound = S.attention(q.reshape(1, 2, d), k, v, c.table, c.pos, d ** -0.5)
    assert (np.abs(got.reshape(1, 2, d) - want).max(-1) <= bound).all(), got[0, :2]

@pytest.mark.parametrize("dtype,exponents", [("float16", (0, -14, -24)), ("bfloat16", (0, -60, -100, -115, -126))])
@pytest.mark.parametrize("n", [1, 300, 5000])
def test_attention_smallest_values(gpu, dtype, exponents, n):
    """Equal scores and one power of two in V: the output is that, exactly (every product p v is a power of two over
    2^-149, every sum of them and of p a count of them)."""
    c = Cached([n], 1, 64, 64, dtype)
    live = ~np.isnan(host(c.v.float()))
    for e in exponents:
        for t, value in ((c.k, 0.0), (c.v, 2.0 ** e)):
            t[dev(live)] = value
        got = host(gpu.paged_attention(dev(np.ones((1, 128), np.float32)), c.k, c.v, dev(c.table), dev(c.pos)))
        assert (got == 2.0 ** e).all(), (e, got[0, :2])


# ------------------------------------------ V that is no number, rows of one table


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,heads,kv_heads", [(64, 8, 2), (96, 3, 1), (128, 4, 2), (256, 2, 1)])
def test_attention_rows_of_one_table_nonfinite_values(gpu, dtype, d, heads, kv_heads):
    """NaN and infinities in V, several of a tile: each reaches its own dimension of the rows that attend it, and the
    bits of everything else stay. Rows out of order, empty ones and one past the table among them; a page is absent."""
    c = Cached([150], kv_heads, d, 16, dtype)
    c.table[0, 2] = -1                                           # positions 32 .. 47
    pos = np.array([70, 3, -1, 149, 64, 65, 66, 2 ** 31 - 1, 31, 100, 0, 40, 71, 72], np.int32)
    q = dev(np.random.default_rng(d).standard_normal((len(pos), heads * d)).astype(np.float32))
    args = (dev(c.table).expand(len(pos), -1), dev(pos))
    c.table[0, 10:] = -1
    clean = host(gpu.paged_attention(q, c.k, c.v, *args)).reshape(len(pos), heads, d)
    bad = np.zeros(clean.shape, bool)
    places = [(65, 0, 0, np.nan), (66, 0, 0, np.inf), (66, kv_heads - 1, d - 1, -np.inf), (3, 0, 5, np.inf), (71, 0, 17, np.nan)]
    for at, h, dim, value in places:
        c.v[int(c.table[0, at // 16]), h, at % 16, dim] = value
        per = heads // kv_heads
        bad[pos >= at, h * per:(h + 1) * per, dim] = True
    got = host(gpu.paged_attention(q, c.k, c.v, *args)).reshape(len(pos), heads, d)
    attended = pos < 150                                         # the one past the table meets slots never filled
    assert np.array_equal(np.isfinite(got[attended]), ~bad[attended])
    assert np.array_equal(got[attended][~bad[attended]], clean[attended][~bad[attended]])


# ---------------------------------------------- weights far below the largest


def _one_channel(c, scores, vals):
    """Keys of one row whose score against q = 8 e_0 at scale 1 / 8 is `scores` exactly, with `vals` [n, d]."""
    import torch
    page = c.k.shape[2]
    at = torch.from_numpy(c.table[0, np.arange(len(scores)) // page].astype(np.int64)).cuda()
    slot = torch.arange(len(scores), device="cuda") % page
    c.k[at, :, slot] = 0.0
    c.k[at, :, slot, 0] = dev(scores)[:, None].to(c.dtype)
    c.v[at, :, slot] = dev(vals)[:, None].to(c.dtype)


def _check_relative(gpu, c, scores, rows, heads=2):
    """Every output within its own relative bound: V is nowhere negative, so nothing cancels.

    A score of at most `far` nats: the factor scale log2 e and its product with q are rounded (2^-24 each), q is held to
    22 bits or more, the products' sum and the distance from the reference are rounded (2^-24 each): far 2^-21 nats
    in all at most, a relative error as large in p. p is an exponential within 2^-22 and held to 2^-22: 2^-21. The sums
    of p v and of p: n / 32 + 128 roundings each, as step_oracle's bound has them. Weights are held to 2^-88 of the largest
    at least, each times a V of at most max |V|."""
    d, n = c.k.shape[-1], len(scores)
    q = np.zeros((rows, heads, d), np.float32)
    q[:, :, 0] = 8.0
    c.pos = np.full(rows, n - 1, np.int32)
    got = host(gpu.paged_attention(dev(q.reshape(rows, -1)), c.k, c.v, dev(c.table).expand(rows, -1), dev(c.pos),
                                   scale=0.125)).reshape(rows, heads, d)
    k, v = c.arrays()
    want, _ = S.attention(q, k, v, c.table.repeat(rows, 0), c.pos, 0.125)
    far = float(np.max(np.abs(scores)))
    tol = 1.01 * far * 2.0 ** -21 + 2.0 ** -20 + 2 * (n / 32 + 128) * 2.0 ** -24
    rel = (np.abs(got - want) - n * 2.0 ** -88 * np.nanmax(v)) / want
    assert (want > 0).all() and rel.max() <= tol, (rel.max(), tol)


@pytest.mark.parametrize("dtype,nats", [("float16", (14, 18, 20, 25, 33, 45, 60, 80)), ("bfloat16", (14, 20, 33, 45))])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("n,at", [(20, 0), (20, 11), (4003, 0), (4003, 4002), (4003, 1777)])
def test_attention_sink(gpu, dtype, nats, d, n, at):
    """One key that takes nearly all the weight, its V zero: the output is the rest's, however small their weights."""
    rng = np.random.default_rng(n + at)
    c = Cached([n], 1, d, 64, dtype)
    vals = (0.5 + rng.random((n, d))).astype(np.float32)
    vals[at] = 0.0
    for far in nats:
        scores = np.zeros(n, np.float32)
        scores[at] = far
        _one_channel(c, scores, vals)
        for rows in (1, 3):                                     # alone, and rows of one table
            _check_relative(gpu, c, scores, rows)


@pytest.mark.parametrize("dtype,far", [("float16", 26), ("bfloat16", 44)])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("n", [33, 1500])
def test_attention_weights_of_every_size(gpu, dtype, far, d, n):
    """Scores spread over `far` nats, V a power of two that makes up for the weight: every key counts alike."""
    rng = np.random.default_rng(n)
    scores = (rng.integers(0, 4 * far + 1, n) / 4).astype(np.float32)
    scores[rng.integers(n)] = far
    span = round(far * math.log2(math.e))
    low = -24 if dtype == "float16" else -20
    vals = np.exp2(low + np.round((far - scores) * math.log2(math.e)))[:, None] * (1 + rng.integers(0, 2, (n, d)))
    assert vals.max() <= 65504 or dtype == "bfloat16" and span < 100
    c = Cached([n], 1, d, 32, dtype)
    _one_channel(c, scores, vals.astype(np.float32))
    for rows in (1, 3):
        _check_relative(gpu, c, scores, rows)


# ------------------------------------------------------------------ infinite K


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_attention_infinite_keys(gpu, dtype, d, value):
    """An infinite K at a position attended gives NaN in its row and KV head, whatever q's sign and bits there, and
    leaves the others' bits alone."""
    import torch
    c = Cached([100, 100, 1500], 2, d, 32, dtype)
    heads, per = 16, 8
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn((3, heads, d), generator=g, device="cuda")
    q[:, 8, 7], q[:, 9, 7], q[:, 10, 7], q[:, 11, 7] = 0.0, 1.0, -1.0, 2.0 ** -12
    q = q.view(3, -1)
    args = (dev(c.table), dev(c.pos))
    clean = host(gpu.paged_attention(q, c.k, c.v, *args)).reshape(3, heads, d)
    c.k[int(c.table[0, 1]), 1, 9, 7] = value
    c.k[int(c.table[2, 40]), 1, 3, 7] = value
    got = host(gpu.paged_attention(q, c.k, c.v, *args)).reshape(3, heads, d)
    assert np.isnan(got[[0, 2], per:]).all()
    assert np.array_equal(got[1], clean[1]) and np.array_equal(got[:, :per], clean[:, :per])
    # Rows of one table: those that attend the position, and no row before it.
    pos = torch.arange(30, 60, dtype=torch.int32, device="cuda")         # the key's is 41
    q = torch.randn((30, heads * d), generator=g, device="cuda")
    got = host(gpu.paged_attention(q, c.k, c.v, args[0][:1].expand(30, -1), pos)).reshape(30, heads, d)
    assert np.isnan(got[11:, per:]).all() and np.isfinite(got[:11]).all() and np.isfinite(got[:, :per]).all()
