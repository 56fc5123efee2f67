"""Paged attention at the ends of its types' ranges (include/w4a8_step.h) against float64."""

from __future__ import annotations

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
