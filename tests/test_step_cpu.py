"""The decode step's other entry points without a GPU: what the host refuses,
before any HIP call (include/w4a8_step.h), and the oracle on cases with known
answers."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv260gemv as kv
import step_oracle as S

A = [0x1000000 * (i + 1) for i in range(12)]      # addresses far apart; never dereferenced: every call fails its checks


def _cache(**more):
    f = dict(k=A[0], v=A[1], pages=10, page_size=16, kv_heads=2, head_dim=64, dtype=0)
    return kv.KVCache(**{**f, **more})


def _rows(**more):
    f = dict(table=A[2], table_stride=4, table_pages=4, pos=A[3], m=3)
    return kv.KVRows(**{**f, **more})


BAD_KV = [
    (dict(k=None), {}, -1), (dict(v=None), {}, -1), ({}, dict(table=None), -1), ({}, dict(pos=None), -1),
    (dict(dtype=2), {}, -2), (dict(dtype=-1), {}, -2), (dict(head_dim=80), {}, -2), (dict(head_dim=512), {}, -2),
    (dict(head_dim=0), {}, -2), (dict(page_size=8), {}, -2), (dict(page_size=48), {}, -2), (dict(page_size=512), {}, -2),
    (dict(page_size=-16), {}, -2), (dict(pages=0), {}, -2), (dict(kv_heads=0), {}, -2), (dict(kv_heads=3), {}, -2),
    ({}, dict(m=0), -2), ({}, dict(m=65537), -2), ({}, dict(table_pages=0), -2), ({}, dict(table_stride=3), -2),
    ({}, dict(table_stride=-4), -2), ({}, dict(table_pages=(1 << 26) + 1, table_stride=1 << 27), -2),
    (dict(k=A[0] + 8), {}, -3), ({}, dict(table=A[2] + 2), -3), ({}, dict(pos=A[3] + 1), -3),
]


@pytest.mark.parametrize("cache,rows,status", BAD_KV)
def test_cache_and_rows_are_checked(cache, rows, status):
    L = kv.lib()
    c, r = _cache(**cache), _rows(**rows)
    assert L.w4a8_rope_append(A[4], 4, ctypes.byref(c), ctypes.byref(r), A[5], 64, 0, A[6], None) == status
    assert L.w4a8_paged_attention(A[4], 4, ctypes.byref(c), ctypes.byref(r), 0.1, A[6], A[7], 1 << 30, None) == status


def test_append_arguments():
    L = kv.lib()
    c, r = _cache(), _rows()

    def call(qkv=A[4], heads=4, inv=A[5], rope=64, out=A[6], cache=c):
        return L.w4a8_rope_append(qkv, heads, ctypes.byref(cache), ctypes.byref(r), inv, rope, 0, out, None)

    assert call(qkv=None) == call(inv=None) == call(out=None) == -1
    assert L.w4a8_rope_append(A[4], 4, None, ctypes.byref(r), A[5], 64, 0, A[6], None) == -1
    assert call(heads=0) == call(heads=3) == call(heads=-2) == call(heads=1 << 21) == -2
    assert call(rope=0) == call(rope=3) == call(rope=66) == call(rope=-2) == -2
    assert call(qkv=A[4] + 4) == call(out=A[6] + 8) == call(inv=A[5] + 2) == -3
    assert call(out=A[4]) == call(out=A[4] + 16) == -2                    # q over q|k|v
    assert call(out=A[0] + 64) == call(qkv=A[1] + 64) == -2               # either over the cache
    assert call(cache=_cache(v=A[0] + 64)) == -2                          # K over V


def test_attention_arguments():
    L = kv.lib()
    c, r = _cache(), _rows(table_pages=4096, table_stride=4096)
    need = L.w4a8_paged_attention_workspace_bytes(4, ctypes.byref(c), ctypes.byref(r))

    def call(q=A[4], heads=4, out=A[6], ws=A[7], n=need):
        return L.w4a8_paged_attention(q, heads, ctypes.byref(c), ctypes.byref(r), 0.1, out, ws, n, None)

    assert call(q=None) == call(out=None) == -1
    assert call(heads=3) == call(heads=0) == -2
    assert call(q=A[4] + 4) == call(out=A[6] + 4) == call(ws=A[7] + 4) == -3
    assert call(out=A[4] + 16) == call(out=A[0]) == -2
    if need:
        assert call(ws=None) == -1
        assert call(n=need - 1) == call(ws=A[4]) == call(ws=A[6]) == call(ws=A[0]) == -2
    for heads, cache, rows in ((3, c, r), (0, c, r), (4, _cache(kv_heads=0), r), (4, c, _rows(m=0)), (4, c, _rows(table_pages=0))):
        assert L.w4a8_paged_attention_workspace_bytes(heads, ctypes.byref(cache), ctypes.byref(rows)) == 0
    assert L.w4a8_paged_attention_workspace_bytes(4, None, ctypes.byref(r)) == 0


def test_norm_arguments():
    L = kv.lib()

    def call(x=A[0], y=A[1], post=A[2], gate=A[3], stride=0, norm=A[4], xo=A[5], h=A[6], q8=0, k=256, m=3):
        return L.w4a8_residual_rmsnorm(x, y, post, gate, stride, 1.0, norm, 1e-5, xo, h, q8, k, m, None)

    assert call(x=None) == call(y=None) == call(xo=None) == call(h=None) == -1
    assert call(k=200) == call(k=128) == call(k=16640) == call(m=0) == call(m=(1 << 23) + 1) == -2
    assert call(stride=255) == call(stride=258) == call(stride=-256) == -2
    for name in ("x", "y", "post", "gate", "norm", "xo", "h"):
        assert call(**{name: A[7] + 4}) == -3
    assert call(xo=A[0] + 1024) == call(xo=A[1]) == call(xo=A[2]) == call(xo=A[3]) == call(xo=A[4]) == -2
    assert call(h=A[0]) == call(h=A[1]) == call(h=A[2]) == call(h=A[3]) == call(h=A[4]) == call(h=A[5]) == -2
    assert call(xo=A[0] - 1024) == -2                                     # other rows of x


def test_sample_arguments():
    L = kv.lib()
    s = kv.Sampling(None, None, None, None, 1.0, 0, 1.0, 0.0)

    def call(logits=A[0], stride=5000, m=3, n=5000, u=A[1], tokens=A[2], ws=A[3], size=1 << 40, settings=s):
        return L.w4a8_sample(logits, stride, m, n, u, ctypes.byref(settings), tokens, ws, size, None)

    assert call(logits=None) == call(u=None) == call(tokens=None) == -1
    assert L.w4a8_sample(A[0], 5000, 3, 5000, A[1], None, A[2], A[3], 1 << 40, None) == -1
    assert call(m=0) == call(m=65537) == call(n=0) == call(n=524289, stride=524289) == call(stride=4999) == -2
    assert call(logits=A[0] + 2) == call(u=A[1] + 1) == call(tokens=A[2] + 2) == call(ws=A[3] + 8) == -3
    assert call(settings=kv.Sampling(A[4] + 2, None, None, None, 1.0, 0, 1.0, 0.0)) == -3
    need = L.w4a8_sample_workspace_bytes(3, 5000)
    if need:
        assert call(ws=None) == -1
        assert call(size=need - 1) == -2
    assert L.w4a8_sample_workspace_bytes(0, 10) == L.w4a8_sample_workspace_bytes(3, 524289) == 0


@pytest.mark.parametrize("n", [5000, 20000])
def test_sample_overlaps(n):
    L = kv.lib()
    need, stride = L.w4a8_sample_workspace_bytes(3, n), n + 1000
    s = kv.Sampling(A[4], A[5], A[6], A[7], 0.0, 0, 0.0, 0.0)

    def call(tokens=A[2], ws=A[3]):
        return L.w4a8_sample(A[0], stride, 3, n, A[1], ctypes.byref(s), tokens, ws, need, None)

    for at in (A[0], A[0] + 4 * (2 * stride + n - 1), A[1], A[1] + 8, A[1] - 8, A[4], A[5], A[6], A[7]):
        assert call(tokens=at) == -2
    if need:                                             # rows in slices: the only ones with a workspace
        for at in (A[0], A[1], A[2], A[4], A[5], A[6], A[7], A[2] - (need - 4) // 16 * 16):
            assert call(ws=at) == -2


def test_rows_overlaps():
    """Outputs and workspaces over the table, the positions or the angles; rows further apart than any table."""
    L = kv.lib()
    c, r = _cache(), _rows(table_pages=4096, table_stride=4096)
    table, pos = r.table, r.pos
    need = L.w4a8_paged_attention_workspace_bytes(4, ctypes.byref(c), ctypes.byref(r))

    def attend(out=A[6], ws=A[7], rows=r):
        return L.w4a8_paged_attention(A[4], 4, ctypes.byref(c), ctypes.byref(rows), 0.1, out, ws, need, None)

    last = table + 4 * (4096 * (r.m - 1) + 4095) & -16
    assert attend(out=table) == attend(out=last) == attend(out=pos) == -2
    assert not need or attend(ws=table) == attend(ws=last) == attend(ws=pos) == -2
    assert attend(rows=_rows(table_pages=4096, table_stride=(1 << 30) + 4)) == -2

    def append(out=A[6], inv=A[7], cache=c, rows=r):
        return L.w4a8_rope_append(A[4], 4, ctypes.byref(cache), ctypes.byref(rows), inv, 64, 0, out, None)

    assert append(out=table) == append(out=last) == append(out=pos) == append(out=A[7]) == -2
    assert append(inv=A[0]) == append(inv=A[1]) == append(cache=_cache(v=table)) == append(cache=_cache(k=pos)) == -2


def test_wrappers_refuse_host_tensors():
    import torch
    kc = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    table, pos, x = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 256)
    for f in (lambda: kv.paged_attention(x, kc, kc, table, pos), lambda: kv.rope_append(x, kc, kc, table, pos, x[0, :32]),
              lambda: kv.residual_rmsnorm(x, x), lambda: kv.sample(x, x[0, :1])):
        with pytest.raises(ValueError, match="GPU"):
            f()


# ------------------------------------------------------------------ oracle


def test_oracle_rope_turns_by_the_angle():
    x = np.array([[[1.0, 0.0, 0.0, 2.0]]], np.float32)
    inv = np.array([np.pi / 2, np.pi], np.float32)
    y = S.rope(x, np.array([1]), inv, False)          # pairs (0, 2), (1, 3)
    assert np.allclose(y, [[[0, 0, 1, -2]]], atol=1e-6)
    y = S.rope(x, np.array([1]), inv, True)           # pairs (0, 1), (2, 3)
    assert np.allclose(y, [[[0, 1, 0, -2]]], atol=1e-6)


def test_oracle_attention_known_answers():
    k = np.zeros((3, 1, 16, 64))
    v = np.arange(3 * 16, dtype=np.float64).reshape(3, 1, 16, 1).repeat(64, 3)
    q = np.ones((3, 2, 64), np.float32)
    table = np.array([[2, 0], [9, 1], [-1, 7]], np.int32)
    out, _ = S.attention(q, k, v, table, np.array([17, 31, 31]), 1.0)
    assert np.allclose(out[0], (sum(range(32, 48)) + 0 + 1) / 18)   # uniform over page 2 and two tokens of page 0
    assert np.allclose(out[1], sum(range(16, 32)) / 16)             # its first page is absent
    assert not out[2].any()


def test_oracle_sample_known_answers():
    l = np.log(np.array([0.1, 0.4, 0.4, 0.1]))
    assert [S.sample(l, u) for u in (0.0, 0.39, 0.41, 0.79, 0.81, 0.89, 0.91, 1.0)] == [1, 1, 2, 2, 0, 0, 3, 3]
    assert [S.sample(l, u, top_k=2) for u in (0.49, 0.51)] == [1, 2]
    assert [S.sample(l, u, top_p=0.45) for u in (0.49, 0.51)] == [1, 2]
    assert S.sample(l, 0.99, top_p=0.39) == 1 and S.sample(l, 0.99, min_p=0.5) == 2 and S.sample(l, 0.99, temperature=0) == 1
    assert S.sample([-np.inf, np.nan], 0.5) == -1


def test_oracle_angles_of_far_positions():
    """Against the math library's own reduction: of an integer, and of an integer and a small angle apart."""
    pos = np.array([0, 5, 2 ** 29 - 1, 2 ** 29 + 1, 10 ** 9 + 7, 2 ** 31 - 1])
    got = S.angles(pos, np.float32(1.0))
    assert np.allclose(np.sin(got), np.sin(pos.astype(np.float64)), rtol=0, atol=1e-14)
    assert np.abs(got[3:]).max() <= np.pi + 1e-12
    small = pos * 2.0 ** -23
    want = np.sin(pos.astype(np.float64)) * np.cos(small) + np.cos(pos.astype(np.float64)) * np.sin(small)
    assert np.allclose(np.sin(S.angles(pos, np.float32(1 + 2.0 ** -23))), want, rtol=0, atol=1e-13)


def test_sample_workspace_is_checked():
    """Of rows in slices, the only ones with a workspace."""
    L = kv.lib()
    s = kv.Sampling(None, None, None, None, 1.0, 0, 1.0, 0.0)
    need = L.w4a8_sample_workspace_bytes(3, 20000)
    assert need > 0 and L.w4a8_sample_workspace_bytes(3, 5000) == 0

    def call(ws=A[3], size=need):
        return L.w4a8_sample(A[0], 20000, 3, 20000, A[1], ctypes.byref(s), A[2], ws, size, None)

    assert call(ws=None) == -1
    assert call(size=need - 1) == call(size=0) == -2
    assert call(ws=A[3] + 8) == -3
    assert call(ws=A[0]) == call(ws=A[1]) == call(ws=A[2]) == -2
