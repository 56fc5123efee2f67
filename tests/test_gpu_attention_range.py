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
