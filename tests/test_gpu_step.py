"""The decode step's other operators on the GPU (include/w4a8_step.h) against
float64: rope and the cache append, paged attention, the residual norms, the
sampler's draw. Unused cache slots hold NaN and unused table entries numbers
that lead nowhere, so a read of either shows."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import c_oracle as C
import step_oracle as S
from gpu_helpers import assert_bytes_equal, dev, host

pytestmark = pytest.mark.gpu

NOWHERE = (-1, 2 ** 31 - 1, -2 ** 31)     # table entries outside any cache


class Cached:
    """A cache whose rows hold lens[i] tokens at random pages; everything else NaN, or nowhere."""

    def __init__(self, lens, kv_heads, d, page, dtype, seed=0, width=None, amp=1.0, spare=3):
        import torch
        rng = np.random.default_rng(seed)
        self.dtype = getattr(torch, dtype)
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        width = width or max(1, max(need, default=1)) + 1
        order = rng.permutation(self.pages)
        table = np.array([NOWHERE[i % 3] for i in range(len(lens) * width)], np.int64).reshape(len(lens), width)
        table[table == -1] = self.pages       # one past the last page too
        shape = (self.pages, kv_heads, page, d)
        k, v = np.full(shape, np.nan, np.float32), np.full(shape, np.nan, np.float32)
        at = 0
        for i, n in enumerate(lens):
            for j in range(need[i]):
                p = table[i, j] = order[at]
                at += 1
                fill = min(page, n - j * page)
                k[p, :, :fill] = amp * rng.standard_normal((kv_heads, fill, d))
                v[p, :, :fill] = rng.standard_normal((kv_heads, fill, d))
        self.table = table.astype(np.int32)
        self.pos = np.array(lens, np.int32) - 1
        self.k, self.v = torch.from_numpy(k).to(self.dtype).cuda(), torch.from_numpy(v).to(self.dtype).cuda()

    def arrays(self):
        return host(self.k.float()), host(self.v.float())


def check_attention(gpu, c, heads, seed=1, qamp=1.0, table=None, scale=None, **more):
    m, d = len(c.pos), c.k.shape[-1]
    q = (qamp * np.random.default_rng(seed).standard_normal((m, heads, d))).astype(np.float32)
    table_t = dev(c.table) if table is None else table
    got = host(gpu.paged_attention(dev(q.reshape(m, -1)), c.k, c.v, table_t, dev(c.pos), scale=scale, **more))
    k, v = c.arrays()
    want, bound = S.attention(q, k, v, host(table_t), c.pos, d ** -0.5 if scale is None else scale)
    err = np.abs(got.reshape(m, heads, d) - want).max(-1)
    # A row that attends slots never filled (NaN) is NaN there and in the oracle.
    ok = (err <= bound) | (np.isnan(want).all(-1) & np.isnan(got.reshape(m, heads, d)).all(-1))
    assert ok.all(), (np.argwhere(~ok)[:5], np.max(err - bound), err.max())
    return got


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attention_lengths(gpu, dtype, d, page):
    check_attention(gpu, Cached(EDGES, 2, d, page, dtype), 8)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (2, 1), (6, 2), (7, 1), (16, 1), (17, 1), (40, 2), (32, 8),
                                            (128, 4)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attention_head_layouts(gpu, heads, kv_heads, dtype):
    check_attention(gpu, Cached([45, 200, 1], kv_heads, 64, 32, dtype), heads)


@pytest.mark.parametrize("dtype,d,page", [("float16", 64, 16), ("bfloat16", 128, 128), ("bfloat16", 96, 32),
                                          ("float16", 256, 64)])
def test_attention_long_rows_beside_short_ones(gpu, dtype, d, page):
    check_attention(gpu, Cached([5000, 3, 0, 1291, 20011 if d == 64 else 4097], 2, d, page, dtype), 6)


@pytest.mark.parametrize("dtype,d,lens", [("float16", 64, (2, 1009)), ("bfloat16", 128, (500, 1000))])
def test_attention_many_rows_of_some_rounds(gpu, dtype, d, lens):
    """Enough rows and heads to leave rows of several rounds whole; one row empty."""
    rows = np.random.default_rng(3).integers(*lens, 24)
    rows[5], rows[6], rows[7] = 0, 1, lens[1] - 1
    check_attention(gpu, Cached(rows, 8, d, 16, dtype), 8)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attention_large_scores(gpu, dtype):
    """One key takes nearly all the weight, scores to several hundreds, in early and late tiles."""
    check_attention(gpu, Cached([1500, 700], 1, 64, 16, dtype, amp=8.0), 4, qamp=30.0)
    check_attention(gpu, Cached([300], 1, 128, 16, dtype, amp=100.0), 2, qamp=1e-3)


def test_attention_rising_scores(gpu):
    """Every key's score above all before it: the running maximum moves at each step."""
    import torch
    n, d = 2000, 64
    c = Cached([n], 1, d, 64, "float16")
    ramp = torch.arange(n, device="cuda") / n
    flat = c.table[0, : -(-n // 64)]
    for j in range(n):
        c.k[int(flat[j // 64]), 0, j % 64] = (0.05 * ramp[j]).item()
    check_attention(gpu, c, 4, qamp=0.0)
    q = torch.full((1, 2 * d), 40.0, device="cuda")
    got = host(gpu.paged_attention(q, c.k, c.v, dev(c.table), dev(c.pos)))
    k, v = c.arrays()
    want, bound = S.attention(host(q).reshape(1, 2, d), k, v, c.table, c.pos, d ** -0.5)
    assert (np.abs(got.reshape(1, 2, d) - want).max(-1) <= bound).all()


def test_attention_extreme_queries(gpu):
    """Queries at the ends of float32's range, against keys of the smallest fp16: nothing overflows on the way."""
    c = Cached([90], 1, 64, 32, "float16", amp=2.0 ** -24)
    check_attention(gpu, c, 2, qamp=1e8)
    c = Cached([90], 1, 64, 32, "bfloat16", amp=1e-30)
    check_attention(gpu, c, 2, qamp=1e30)
    check_attention(gpu, c, 2, qamp=1e-38)


def test_attention_absent_pages(gpu):
    """Pages left behind a window, one in the middle, the row's last one, and all of them."""
    c = Cached([400, 400, 400, 400, 30], 2, 64, 32, "bfloat16")
    c.table[0, :7] = -1
    c.table[1, 5] = c.pages
    c.table[2, 12] = -2 ** 31
    c.table[3, :] = 2 ** 31 - 1
    c.table[4, :] = -1
    got = check_attention(gpu, c, 4)
    assert not got[3].any() and not got[4].any()


def test_attention_position_past_the_table(gpu):
    """A position that the table does not reach: the ones that it does are attended."""
    c = Cached([64, 64], 1, 64, 16, "float16", width=4)
    c.pos[:] = [2 ** 31 - 1, 64]
    check_attention(gpu, c, 4)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 2, 64, 16), (3, 1, 64, 32), (8, 1, 128, 16), (2, 2, 96, 64),
                                                   (4, 1, 256, 128), (9, 1, 64, 16), (20, 1, 64, 16), (16, 4, 128, 256)])
def test_attention_rows_of_one_sequence(gpu, dtype, heads, kv_heads, d, page):
    """A prompt's rows over one table (expanded): in order, and out of it with empty rows and a row past the table;
    one length to many rounds of splits; each row as it is alone, within the bound."""
    n = 700
    c = Cached([n], kv_heads, d, page, dtype)
    most = c.table.shape[1] * page
    for pos in (np.arange(45), np.arange(n - 19, n), np.array([5]), np.array([n - 1, -1, 3, 400, -7, 2 ** 31 - 1, 399, 0]),
                np.full(6, -1)):
        c.pos = np.asarray(pos, np.int32)
        c.table[0, -(-n // page):] = -1       # positions past the tokens are absent
        assert most > n
        check_attention(gpu, c, heads, table=dev(c.table).expand(len(c.pos), -1))
    c.table[0, 1] = -1
    c.pos = np.arange(0, n, 37, dtype=np.int32)
    check_attention(gpu, c, heads, table=dev(c.table).expand(len(c.pos), -1))


def test_attention_long_prompt_rows(gpu):
    """Rows of one table with splits of several rounds, far apart in length."""
    c = Cached([9000], 1, 64, 64, "float16")
    c.pos = np.array([8999, 17, 4500, 8998, 0, 8191], np.int32)
    check_attention(gpu, c, 4, table=dev(c.table).expand(len(c.pos), -1))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_rows_of_one_sequence_nonfinite(gpu, dtype, d):
    """A token with NaN or infinity in K or V reaches the rows that attend it and no row before it."""
    import torch
    c = Cached([100], 2, d, 16, dtype)
    q = torch.randn(40, 4 * d, device="cuda")
    pos = torch.arange(50, 90, dtype=torch.int32, device="cuda")
    table = dev(c.table).expand(40, -1)
    clean = host(gpu.paged_attention(q, c.k, c.v, table, pos)).reshape(40, 4, d)
    for at, half, value in ((61, c.v, math.nan), (75, c.v, math.inf), (77, c.k, math.nan), (89, c.v, -math.inf)):
        half[int(c.table[0, at // 16]), 1, at % 16, 9] = value
    got = host(gpu.paged_attention(q, c.k, c.v, table, pos)).reshape(40, 4, d)
    ok = np.isfinite(got)
    assert ok[:, :2].all() and np.array_equal(got[:, :2], clean[:, :2])
    assert ok[:11].all() and np.array_equal(got[:11], clean[:11])              # positions 50 .. 60
    assert not ok[11:, 2:, 9].any() and ok[11:27, 2:, :9].all() and ok[11:27, 2:, 10:].all()
    assert not ok[27:, 2:].any()


def test_attention_table_rows_apart(gpu):
    """Table rows that lie apart in a wider one."""
    import torch
    c = Cached([150, 90, 20], 2, 64, 16, "float16")
    wide = torch.full((3, 40), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + c.table.shape[1]] = dev(c.table)
    check_attention(gpu, c, 4, table=wide[:, 5:5 + c.table.shape[1]])


def test_attention_nonfinite(gpu):
    """NaN in q, or in K or V of a token attended, stays in its row and heads."""
    import torch
    c = Cached([100, 100, 100, 100], 2, 64, 32, "float16")
    q = torch.randn(4, 4 * 64, device="cuda")
    clean = host(gpu.paged_attention(q, c.k, c.v, dev(c.table), dev(c.pos))).reshape(4, 4, 64)
    q[0, 3] = math.nan
    c.k[int(c.table[1, 1]), 1, 5, 7] = math.nan
    c.v[int(c.table[2, 0]), 0, 31, 9] = math.nan
    got = host(gpu.paged_attention(q, c.k, c.v, dev(c.table), dev(c.pos))).reshape(4, 4, 64)
    bad = np.isnan(got)
    assert bad[0, 0].all() and not bad[0, 1:].any()
    assert bad[1, 2:].all() and not bad[1, :2].any()
    assert bad[2, :2, 9].all() and bad[2].sum() == 2
    assert not bad[3].any() and np.array_equal(got[~bad], clean[~bad])


def test_attention_deterministic_and_workspace(gpu):
    """The same bits again, into the caller's tensor and workspace, whatever that held; nothing behind either."""
    import torch
    c = Cached([3000, 40, 0, 999], 2, 128, 16, "bfloat16")
    q = torch.randn(4, 8 * 128, device="cuda")
    args = (q, c.k, c.v, dev(c.table), dev(c.pos))
    want = host(gpu.paged_attention(*args))
    cache, rows = gpu._kv_args(*args[1:])
    need = gpu.lib().w4a8_paged_attention_workspace_bytes(8, ctypes.byref(cache), ctypes.byref(rows))
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((4 * 8 * 128 + 16,), 7.0, device="cuda")
    for _ in range(2):
        assert gpu.paged_attention(*args, out=out, workspace=ws[:need] if need else None) is out
        assert_bytes_equal(host(out[:-16]), want.reshape(-1))
        assert (host(out[-16:]) == 7.0).all() and (host(ws[need:]) == 255).all()
        ws[:need].fill_(0)
    if need:
        with pytest.raises(ValueError, match="the call needs"):
            gpu.paged_attention(*args, workspace=ws[: need - 1])


def _free_bytes():
    import torch
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_cache_past_2_31_elements(gpu, dtype):
    """Append to, and attention over, the last pages of a cache of 2.2e9 elements a half."""
    import torch
    pages, kv_heads, page, d = 33600, 8, 64, 128
    assert pages * kv_heads * page * d > 2 ** 31 and _free_bytes() > 20 << 30
    k = torch.empty((pages, kv_heads, page, d), dtype=getattr(torch, dtype), device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 1, pages - 3], [pages - 2, -1]], dtype=torch.int32, device="cuda")
    inv = torch.ones(d // 2, device="cuda")
    n, heads = 70, 8
    rng = np.random.default_rng(5)
    qkv = rng.standard_normal((n, (heads + 2 * kv_heads) * d)).astype(np.float32)
    q = gpu.rope_append(dev(qkv), k, v, table[:1].expand(n, -1), torch.arange(n, dtype=torch.int32, device="cuda"), inv)
    q1 = gpu.rope_append(dev(qkv[:1]), k, v, table[1:], torch.zeros(1, dtype=torch.int32, device="cuda"), inv)
    pos = np.array([n - 1, 0], np.int32)
    got = host(gpu.paged_attention(torch.cat([q[-1:], q1]), k, v, table, dev(pos)))
    small_k, small_v = (host(t[-3:].float()) for t in (k, v))
    small = np.array([[2, 0], [1, -1]], np.int32)
    want, bound = S.attention(np.stack([host(q)[-1], host(q1)[0]]).reshape(2, heads, d), small_k, small_v, small, pos, d ** -0.5)
    assert (np.abs(got.reshape(2, heads, d) - want).max(-1) <= bound).all()


# ------------------------------------------------------------------ append


def check_append(gpu, qkv, c, inv, interleaved, heads, table=None, pos=None):
    """The whole of q and of both cache halves. The rotation: sine and cosine within 2^-23 (an ulp or so of
    them, and the angle's reduction), two products and a sum of a half-ulp each: (|a| + |b|) 2^-22 at most;
    K's rounding a half-step of its type more. V is rounded once: exact."""
    import torch
    m, kvh, d, page = qkv.shape[0], c.k.shape[1], c.k.shape[3], c.k.shape[2]
    k0, v0 = c.k.clone(), c.v.clone()
    table_h, pos_h = (c.table, c.pos) if table is None else (host(table), host(pos))
    q = host(gpu.rope_append(dev(qkv), c.k, c.v, dev(c.table) if table is None else table,
                             dev(c.pos) if pos is None else pos, dev(inv), interleaved=interleaved))
    x = qkv.reshape(m, heads + 2 * kvh, d)
    y = S.rope(x[:, : heads + kvh], pos_h, inv, interleaved)
    half = inv.size
    a = np.abs(x[:, : heads + kvh]).astype(np.float64)
    size = np.zeros_like(a)
    for i in range(half):
        p, r = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        size[..., p] = size[..., r] = a[..., p] + a[..., r]
    live = pos_h >= 0
    assert not q[~live].any()
    err = np.abs(q.reshape(m, heads, d) - y[:, :heads])[live]
    assert (err <= size[live][:, :heads] * 2.0 ** -22).all(), err.max()
    k_new, v_new, k_old, v_old = (host(t.float()) for t in (c.k, c.v, k0, v0))
    v_cast = host(torch.from_numpy(x[:, heads + kvh:].copy()).to(c.dtype).float())
    info = torch.finfo(c.dtype)
    seen = np.zeros(k_new.shape[:3], bool)
    for i in range(m):
        j = int(pos_h[i]) // page
        page_i = int(table_h[i, j]) if live[i] and j < table_h.shape[1] else -1
        if not 0 <= page_i < c.pages:
            continue
        slot = int(pos_h[i]) % page
        seen[page_i, :, slot] = True
        want = y[i, heads:]
        tol = size[i, heads:] * 2.0 ** -22 * (1 + info.eps) + np.abs(want) * info.eps / 2 + info.smallest_normal * info.eps
        assert (np.abs(k_new[page_i, :, slot] - want) <= tol).all()
        assert np.array_equal(v_new[page_i, :, slot], v_cast[i])
    for new, old in ((k_new, k_old), (v_new, v_old)):      # nothing else, NaN included
        assert np.array_equal(new[~seen], old[~seen], equal_nan=True)
    assert not np.isnan(k_new[seen]).any()


def _inv_freq(r):
    return (500000.0 ** (-np.arange(0, r, 2, dtype=np.float64) / r)).astype(np.float32)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r,heads,kvh,page", [(64, 64, 8, 2, 16), (96, 48, 3, 3, 32), (128, 128, 5, 1, 256),
                                                (256, 2, 4, 2, 64), (128, 126, 32, 8, 16)])
def test_append_decode(gpu, dtype, interleaved, d, r, heads, kvh, page):
    """A batch of rows at their own positions, empty rows and rows whose page is absent among them."""
    lens = [1, 16, 17, 0, 300, 513, 40, 41]
    c = Cached(lens, kvh, d, page, dtype, seed=d + r)
    c.table[6, 39 // page] = -5                       # its page is absent
    c.pos[7] = c.table.shape[1] * page + 3            # past its table
    qkv = np.random.default_rng(r).standard_normal((len(lens), (heads + 2 * kvh) * d)).astype(np.float32)
    check_append(gpu, qkv, c, _inv_freq(r), interleaved, heads)


@pytest.mark.parametrize("dtype,interleaved", [("float16", True), ("bfloat16", False)])
def test_append_prompt(gpu, dtype, interleaved):
    """A prompt of odd length from the middle of a page on, one table for all rows."""
    import torch
    c = Cached([200], 2, 64, 16, dtype, width=14)
    n = 187
    qkv = np.random.default_rng(3).standard_normal((n, (4 + 4) * 64)).astype(np.float32)
    pos = torch.arange(9, 9 + n, dtype=torch.int32, device="cuda")
    check_append(gpu, qkv, c, _inv_freq(64), interleaved, 4, table=dev(c.table).expand(n, -1), pos=pos)


def test_append_far_positions(gpu):
    """Angles of positions to 2^30 - 1 (float32 alone would lose them whole)."""
    import torch
    c = Cached([16, 16, 16], 1, 64, 256, "float16")
    far = torch.tensor([2 ** 30 - 1, 131071, 10 ** 6 + 1], dtype=torch.int32, device="cuda")
    width = 2 ** 30 // 256
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    qkv = np.random.default_rng(4).standard_normal((3, 3 * 64)).astype(np.float32)
    check_append(gpu, qkv, c, _inv_freq(64), False, 1, table=table.expand(3, -1), pos=far)


def test_append_overflow_and_nan(gpu):
    """What the cache's type cannot hold becomes infinity, NaN stays NaN, as torch's casts have it."""
    import torch
    c = Cached([1], 1, 64, 16, "float16")
    qkv = np.zeros((1, 3 * 64), np.float32)
    qkv[0, 128:136] = [65504, 65519.9, 65520, 1e30, -1e30, np.inf, np.nan, 2.0 ** -25]
    gpu.rope_append(dev(qkv), c.k, c.v, dev(c.table), dev(c.pos), dev(_inv_freq(2)))
    got = host(c.v[int(c.table[0, 0]), 0, 0])
    assert np.array_equal(got, torch.from_numpy(qkv[0, 128:]).half().numpy(), equal_nan=True)


# ------------------------------------------------------------------- norms


def _norm_inputs(m, k, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((m, k)) * 2).astype(np.float32)
    return (x, rng.standard_normal((m, k)).astype(np.float32), *(rng.standard_normal(k).astype(np.float32) for _ in range(3)),
            rng.standard_normal((m, k)).astype(np.float32))


@pytest.mark.parametrize("k,m", [(256, 1), (768, 5), (2048, 1), (2304, 333), (4096, 2), (8192, 3), (16384, 2), (16128, 1)])
@pytest.mark.parametrize("post,gate", [(False, None), (True, None), (True, "k"), (False, "mk"), (True, "mk")])
def test_residual_rmsnorm(gpu, k, m, post, gate):
    """Byte for byte: float32 operations one at a time, the norms the oracle's."""
    x, y, w, pw, gk, gm = _norm_inputs(m, k, k + m)
    g = {None: None, "k": gk, "mk": gm}[gate]
    scale = 0.3
    t = np.stack([C.rmsnorm(r, pw, 1e-5) for r in y]) if post else None
    want_x = S.residual(x, y, scale, g, t)
    want_h = np.stack([C.rmsnorm(r, w, 1e-5) for r in want_x])
    more = dict(post_w=dev(pw) if post else None, gate=None if g is None else dev(g), scale=scale)
    dx, dy, dw = dev(x), dev(y), dev(w)
    got_x, got_h = gpu.residual_rmsnorm(dx, dy, dw, 1e-5, **more)
    assert_bytes_equal(host(got_x), want_x, "x")
    assert_bytes_equal(host(got_h), want_h, "h")
    got_x, got_q = gpu.residual_rmsnorm(dx, dy, dw, 1e-5, q8=True, **more)
    assert_bytes_equal(host(got_x), want_x, "x beside q8")
    assert_bytes_equal(host(got_q), host(gpu.rmsnorm_q8_0_engine(got_x, dw, 1e-5)), "q8")
    got_x, none = gpu.residual_rmsnorm(dx, dy, **more)
    assert none is None
    assert_bytes_equal(host(got_x), want_x, "x without h")
    assert_bytes_equal(host(dx), x, "x as it was")
    got_x, got_h = gpu.residual_rmsnorm(dx, dy, dw, 1e-5, out=dx, **more)
    assert got_x is dx
    assert_bytes_equal(host(dx), want_x, "x in place")
    assert_bytes_equal(host(got_h), want_h, "h beside x in place")


def test_residual_rmsnorm_one_row(gpu):
    x, y, w, pw, gk, _ = _norm_inputs(1, 2048, 9)
    got_x, got_h = gpu.residual_rmsnorm(dev(x[0]), dev(y[0]), dev(w), 1e-6)
    assert got_x.shape == got_h.shape == (2048,)
    assert_bytes_equal(host(got_x), x[0] + y[0])
    assert_bytes_equal(host(got_h), C.rmsnorm(x[0] + y[0], w, 1e-6))


def test_residual_rmsnorm_open_roundings(gpu):
    """Sums of squares on a float32 rounding's border, where the order of the float64 sum decides, and rows of NaN,
    infinity and zeros: x' in place, so the order's chains read what this call stored."""
    from test_oracle_producers import _order_case
    k = 2048
    rows = np.stack([_order_case(lanes) for lanes in ({1: 512, 2: 512, 3: 512}, {0: 511}, {1: 2, 3: 2})] +
                    [np.full(k, v, np.float32) for v in (np.nan, np.inf, 0.0, 1e25)])
    w = np.random.default_rng(2).standard_normal(k).astype(np.float32)
    zero = np.zeros_like(rows)
    x = dev(rows)
    got_x, got_h = gpu.residual_rmsnorm(x, dev(zero), dev(w), 0.0, out=x)
    want_h = np.stack([C.rmsnorm(r, w, 0.0) for r in rows])
    got = host(got_h)
    assert np.array_equal(np.isnan(got), np.isnan(want_h))
    assert np.array_equal(got[~np.isnan(want_h)], want_h[~np.isnan(want_h)])
    y, zero = dev(rows), dev(zero)                       # and through the norm of y
    got = host(gpu.residual_rmsnorm(zero, y, eps=0.0, post_w=dev(w))[0])
    assert np.array_equal(np.isnan(got), np.isnan(want_h))
    assert np.array_equal(got[~np.isnan(want_h)], want_h[~np.isnan(want_h)])


# ------------------------------------------------------------------ sampler


def check_sample(gpu, logits, u, **settings):
    """The rows' tokens, each against the oracle; settings: numbers or arrays of a row's own."""
    logits, u = np.asarray(logits, np.float32), np.asarray(u, np.float32)
    given = {n: dev(np.asarray(v, np.int32 if n == "top_k" else np.float32)) if np.ndim(v) else v
             for n, v in settings.items()}
    got = host(gpu.sample(dev(logits), dev(u), **given))
    want = [S.sample(logits[i], u[i], **{n: (v[i] if np.ndim(v) else v) for n, v in settings.items()})
            for i in range(len(u))]
    assert got.tolist() == want, [(i, g, w) for i, (g, w) in enumerate(zip(got.tolist(), want)) if g != w][:5]
    return want


SETTINGS = [dict(), dict(temperature=0), dict(top_k=1), dict(top_k=40), dict(top_k=64, top_p=0.9), dict(top_k=500),
            dict(top_p=0.5), dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0),
            dict(temperature=0.2), dict(temperature=1.7, top_p=0.95), dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.05),
            dict(temperature=100.0), dict(temperature=1e-30), dict(top_k=2 ** 31 - 1, top_p=1.0)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("n", [1, 2, 63, 1000, 4097, 32003])
def test_sample(gpu, settings, n):
    rng = np.random.default_rng(n)
    m = 6
    check_sample(gpu, rng.standard_normal((m, n)) * 3, rng.random(m), **settings)


@pytest.mark.parametrize("settings", [SETTINGS[i] for i in (0, 3, 6, 7, 13)], ids=str)
@pytest.mark.parametrize("n", [128256, 524288])
def test_sample_vocabularies(gpu, settings, n):
    rng = np.random.default_rng(7)
    check_sample(gpu, rng.standard_normal((2, n)) * 2.5, [0.37, 0.93], **settings)


@pytest.mark.parametrize("temperature", [0.05, 1.0, 4.0, 50.0])
@pytest.mark.parametrize("more", [dict(top_k=5000), dict(top_k=5000, top_p=0.6), dict(top_p=0.99), dict(top_p=0.7, min_p=0.001)], ids=str)
def test_sample_wide_bins(gpu, temperature, more):
    """Bins of some tokens to most of the row: compared, spread over finer steps, or read from the row."""
    rng = np.random.default_rng(21)
    check_sample(gpu, rng.standard_normal((3, 50000)) * 2, [0.02, 0.5, 0.98], temperature=temperature, **more)


@pytest.mark.parametrize("levels", [1, 3, 40, 1000])
def test_sample_long_ties(gpu, levels):
    """Rows of a few distinct logits, more of each than any list holds."""
    rng = np.random.default_rng(levels)
    logits = rng.integers(0, levels, (4, 40000)) * (3.0 / levels)
    for more in (dict(), dict(top_k=20001), dict(top_p=0.5), dict(top_k=30000, top_p=0.9, min_p=0.2)):
        check_sample(gpu, logits, rng.random(4), **more)


@pytest.mark.parametrize("m,n", [(1, 3001), (3, 3001), (40, 3001), (300, 3001), (40, 20011), (171, 20011)])
def test_sample_rows_of_their_own_settings(gpu, m, n):
    rng = np.random.default_rng(m)
    check_sample(gpu, rng.standard_normal((m, n)) * 2, rng.random(m),
                 temperature=rng.choice([0.0, 0.5, 1.0, 2.0, -1.0, np.nan, np.inf], m), top_k=rng.choice([0, -3, 1, 7, 50, 64, 65, 2000, 5000], m),
                 top_p=rng.choice([1.0, 0.3, 0.9, 2.0, -1.0, np.nan], m), min_p=rng.choice([0.0, 0.01, 0.2, 1.0, 3.0, -1.0, np.nan], m))


@pytest.mark.parametrize("n", [64, 4096, 65536])
def test_sample_equal_logits(gpu, n):
    """All weights one: token floor(u n), whatever the value the logits share; top-k and top-p cut by index."""
    m = 64
    u = np.arange(m) / m
    for value in (0.0, -3.5, -np.finfo(np.float32).max, np.finfo(np.float32).max, np.inf):
        assert check_sample(gpu, np.full((m, n), value), u) == [i * n // m for i in range(m)]
    assert check_sample(gpu, np.zeros((m, n)), u, top_k=n // 2) == [i * n // m // 2 for i in range(m)]
    assert check_sample(gpu, np.zeros((m, n)), u, top_p=0.25) == [i * n // m // 4 for i in range(m)]
    check_sample(gpu, np.zeros((m, n)), u, top_k=n // 2 + 1, top_p=0.77, min_p=0.5)


def test_sample_ties_and_zeros(gpu):
    """Logits of few distinct values (16-bit weights make such), -0 equal to +0."""
    rng = np.random.default_rng(11)
    logits = np.round(rng.standard_normal((50, 5000)) * 2) / 2
    logits[:, ::7] *= -1.0
    u = rng.random(50)
    check_sample(gpu, logits, u)
    check_sample(gpu, logits, u, top_k=33)
    check_sample(gpu, logits, u, top_k=1234, top_p=0.8)
    zeros = np.where(np.arange(100) % 2, 0.0, -0.0)[None].repeat(4, 0)
    assert check_sample(gpu, zeros, [0.0, 0.011, 0.5, 0.999]) == [0, 1, 50, 99]


def test_sample_masked_rows(gpu):
    """-inf and NaN are never drawn; rows of nothing else give -1; a row with one token gives it."""
    n = 700
    rng = np.random.default_rng(12)
    logits = rng.standard_normal((9, n))
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2] = -np.inf
    logits[2, 650] = -1e30
    logits[3, rng.permutation(n)[:600]] = -np.inf
    logits[4, rng.permutation(n)[:600]] = np.nan
    logits[5, 100:] = -np.finfo(np.float32).max       # masked by the type's lowest value instead
    logits[6] = np.where(np.arange(n) % 3 == 0, np.inf, logits[6])
    logits[7] = np.finfo(np.float32).max * np.where(np.arange(n) % 2, 1, -1)
    logits[8, 1:] = np.nan
    for settings in (dict(), dict(temperature=0), dict(top_k=20), dict(top_p=0.7), dict(min_p=0.3),
                     dict(temperature=50.0)):
        for u in (0.0, 0.4, 0.99999):
            want = check_sample(gpu, logits, np.full(9, u), **settings)
            assert want[0] == want[1] == -1 and want[2] == 650 and want[5] < 100 and want[6] % 3 == 0 and want[7] % 2 == 1


def test_sample_extreme_temperatures(gpu):
    """Temperatures that make every weight one, or every difference infinite, over logits across float32's range."""
    rng = np.random.default_rng(15)
    big = np.finfo(np.float32).max
    logits = np.stack([rng.standard_normal(900) * 3, rng.standard_normal(900) * 1e37, rng.choice([-big, big, 0.0, 1.0], 900),
                       np.where(rng.random(900) < 0.5, -np.inf, np.clip(rng.standard_normal(900), -3, 3) * 1e38)])
    u = np.full(4, 0.61)
    for t in (np.inf, big, 1e38, 1e30, 1e-45, 1e-38):
        check_sample(gpu, logits, u, temperature=np.full(4, t))
        check_sample(gpu, logits, u, temperature=np.full(4, t), top_k=100, top_p=0.7)


@pytest.mark.parametrize("n", [5000, 12007, 20011, 128256])
def test_sample_alone_or_in_a_batch(gpu, n):
    """A row's token in batches of every slicing (and of one slice a row) is the one it gets alone."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n)
    m = 300
    logits = 3 * torch.randn((m, n), generator=g, device="cuda")
    u = torch.rand(m, generator=g, device="cuda")
    for more in (dict(), dict(top_p=0.9), dict(top_k=70, min_p=0.01)):
        whole = host(gpu.sample(logits, u, **more))
        for k in (1, 2, 5, 17, 100):
            at = [host(gpu.sample(logits[i:i + k], u[i:i + k], **more)) for i in range(0, 3 * k, k)]
            assert np.array_equal(np.concatenate(at), whole[: 3 * k]), (k, more)


def test_sample_random_numbers_out_of_range(gpu):
    logits = np.random.default_rng(13).standard_normal((7, 257))
    check_sample(gpu, logits, [-0.5, -0.0, np.nan, 1.0, 2.0, np.inf, 1 - 2.0 ** -24])


def test_sample_strided_rows_and_single_row(gpu):
    """Rows of a padded vocabulary, whose padding is above every logit; one row as a vector; a row at an odd offset."""
    import torch
    rng = np.random.default_rng(14)
    wide = np.full((5, 1009), 1e9, np.float32)
    wide[:, 3:1003] = rng.standard_normal((5, 1000))
    u = rng.random(5).astype(np.float32)
    d = dev(wide)
    want = [S.sample(wide[i, 3:1003], u[i], top_p=0.9) for i in range(5)]
    assert host(gpu.sample(d[:, 3:1003], dev(u), top_p=0.9)).tolist() == want
    for i in range(5):
        assert host(gpu.sample(d[i, 3:1003], dev(u[i:i + 1]), top_p=0.9)).tolist() == want[i:i + 1]
    out = torch.full((7,), 9, dtype=torch.int32, device="cuda")
    gpu.sample(d[:, 3:1003], dev(u), top_p=0.9, out=out)
    assert host(out).tolist() == want + [9, 9]


def test_sample_agrees_with_topk_and_argmax(gpu):
    """Greedy is topk's first; over top_k = 64, u's grid meets topk's candidates in topk's order."""
    import torch
    y = torch.randn(128256, device="cuda")
    vals, idx = gpu.topk(y, 64)
    u = torch.arange(256, device="cuda", dtype=torch.float32) / 256
    tokens = host(gpu.sample(y.expand(256, -1).contiguous(), u, top_k=64))
    ranks = [host(idx).tolist().index(t) for t in tokens.tolist()]
    assert ranks == sorted(ranks) and ranks[0] == 0 and len(set(ranks)) > 40
    assert host(gpu.sample(y, u[:1], temperature=0)).item() == host(idx)[0]


# ------------------------------------------------- streams, graphs, refusals


def test_other_stream(gpu):
    """On a side stream, behind work that is still running there."""
    import torch
    c = Cached([700, 90], 2, 64, 16, "float16")
    q, table, pos = torch.randn(2, 512, device="cuda"), dev(c.table), dev(c.pos)
    logits, u = torch.randn(3, 5000, device="cuda"), torch.rand(3, device="cuda")
    x, w = torch.randn(2, 512, device="cuda"), torch.randn(512, device="cuda")
    want = [host(gpu.paged_attention(2 * q, c.k, c.v, table, pos)), host(gpu.sample(2 * logits, u, top_p=0.9)),
            host(gpu.residual_rmsnorm(x, 2 * x, w)[1])]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-2
        lead = big[0, 0] * 0 + 2
        lead = torch.where(torch.isfinite(lead), lead, torch.full_like(lead, 2.0))
        got = [gpu.paged_attention(lead * q, c.k, c.v, table, pos), gpu.sample(lead * logits, u, top_p=0.9),
               gpu.residual_rmsnorm(x, lead * x, w)[1]]
    for g, v in zip(got, want):
        assert np.array_equal(host(g), v)


def test_step_in_a_graph(gpu):
    """append, attention, norm and draw captured once (two graphs of their own workspaces alive together) and
    replayed on new inputs, eager work between; every replay against the eager calls."""
    import torch
    heads, kvh, d, m, page = 8, 2, 64, 5, 16
    inv = dev(_inv_freq(d))

    def step(t):
        q = gpu.rope_append(t["qkv"], t["c"].k, t["c"].v, t["table"], t["pos"], inv)
        o = gpu.paged_attention(q, t["c"].k, t["c"].v, t["table"], t["pos"])
        x, h = gpu.residual_rmsnorm(t["x"], o, t["w"])
        return q, o, x, h, gpu.sample(h, t["u"], top_p=0.9), gpu.sample(h, t["u"], top_k=10)

    def state(seed):
        c = Cached([900, 40, 0, 333, 16], kvh, d, page, "bfloat16", seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = dict(c=c, table=dev(c.table), pos=dev(c.pos))
        for name, shape in (("qkv", (m, (heads + 2 * kvh) * d)), ("x", (m, heads * d)), ("w", (heads * d,))):
            t[name] = torch.randn(shape, generator=g, device="cuda")
        t["u"] = torch.rand(m, generator=g, device="cuda")
        return t

    runs = []
    for seed in (1, 2):
        t = state(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(t)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(t)
        runs.append((t, graph, out))
    for i in range(4):
        for t, _, _ in runs:
            t["qkv"].normal_()
            t["x"].normal_()
            t["u"].uniform_()
            t["pos"].add_(i % 2)
        torch.cuda.synchronize()
        for _, graph, _ in runs:
            graph.replay()
        torch.cuda.synchronize()
        for t, _, out in runs:
            got = [host(o) for o in out]
            for g, w in zip(got, step(t)):
                assert np.array_equal(g, host(w), equal_nan=True)


def test_refusals(gpu):
    """Arguments that the host can see to be wrong, before anything is launched."""
    import torch
    c = Cached([20, 20], 2, 64, 16, "float16")
    table, pos = dev(c.table), dev(c.pos)
    q, qkv, inv = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 512, device="cuda"), torch.ones(32, device="cuda")
    att, app, smp, nrm = gpu.paged_attention, gpu.rope_append, gpu.sample, gpu.residual_rmsnorm
    wide = torch.zeros(2, 16, 16, 64, device="cuda", dtype=torch.float16)
    x, y = torch.zeros(3, 256, device="cuda"), torch.zeros(100, 3, device="cuda")
    u = torch.zeros(3, device="cuda")
    bad_type = [
        lambda: att(q.half(), c.k, c.v, table, pos), lambda: att(q, c.k.float(), c.v.float(), table, pos),
        lambda: att(q, c.k, c.v, table.long(), pos), lambda: att(q, c.k, c.v, table, pos.long()),
        lambda: att(q, None, c.v, table, pos), lambda: app(qkv.double(), c.k, c.v, table, pos, inv),
        lambda: app(qkv, c.k, c.v, table, pos, inv.double()), lambda: smp(x.half(), u), lambda: smp(x, u.double()),
        lambda: smp(x, u, top_k=u), lambda: smp(x, u, top_p=u.int()), lambda: nrm(x.half(), x),
        lambda: nrm(x, x, out=x.half()), lambda: att(q, c.k, c.v, table, pos, out=q.half()),
    ]
    bad_value = [
        lambda: att(q, c.k, c.v.bfloat16(), table, pos), lambda: att(q, c.k, c.v[1:], table, pos),
        lambda: att(q, c.k[..., :32].contiguous(), c.v[..., :32].contiguous(), table, pos),
        lambda: att(q, wide[:, :, :8].contiguous(), wide[:, :, :8].contiguous(), table, pos),
        lambda: att(q, wide[:, :, :12].contiguous(), wide[:, :, :12].contiguous(), table, pos),
        lambda: att(q, wide[:, ::2], wide[:, ::2], table, pos), lambda: att(q[:, :64], c.k, c.v, table, pos),
        lambda: att(q[:, :200].contiguous(), c.k, c.v, table, pos), lambda: att(q[:1], c.k, c.v, table, pos),
        lambda: att(q[:, :192].contiguous(), c.k, c.v, table, pos), lambda: att(q, c.k, c.v, table[:1], pos),
        lambda: att(q, c.k, c.v, table.t().contiguous().t(), pos), lambda: att(q, c.k, c.v, table, pos[:1]),
        lambda: att(q, c.k.cpu(), c.v.cpu(), table, pos), lambda: att(q, c.k, c.v, table.cpu(), pos),
        lambda: att(q, c.k, c.v, table, pos, out=q[:1]), lambda: att(q.cpu(), c.k, c.v, table, pos),
        lambda: app(qkv[:, :256].contiguous(), c.k, c.v, table, pos, inv), lambda: app(qkv, c.k, c.v, table, pos, inv[:0]),
        lambda: app(qkv, c.k, c.v, table, pos, torch.ones(33, device="cuda")),
        lambda: smp(x, u[:2]), lambda: smp(y.t(), u), lambda: smp(x[:1].expand(3, -1), u), lambda: smp(x[:, :0], u),
        lambda: smp(x, u, temperature=-1.0), lambda: smp(x, u, top_k=-1), lambda: smp(x, u, top_p=math.nan),
        lambda: smp(torch.empty(1, 524289, device="cuda"), u[:1]),
        lambda: smp(torch.empty(65537, 1, device="cuda"), torch.zeros(65537, device="cuda")),
        # A count that would be 5 in 32 bits.
        lambda: smp(torch.empty(1, 2 ** 32 + 5, device="cuda"), u[:1]), lambda: smp(x, u, min_p=1.5),
        lambda: smp(x, u, top_p=u[:2]), lambda: smp(x.cpu(), u),
        lambda: nrm(x, x[:2]), lambda: nrm(x[:, :200].contiguous(), x[:, :200].contiguous()), lambda: nrm(x, x, x[0, :128]),
        lambda: nrm(x, x, gate=x[:2]), lambda: nrm(x, x, x[0].clone(), q8=True, h_out=torch.zeros(10, dtype=torch.uint8, device="cuda")),
    ]
    for i, f in enumerate(bad_type):
        with pytest.raises(TypeError):
            f()
            pytest.fail(f"TypeError {i}")
    for i, f in enumerate(bad_value):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"ValueError {i}")
    # Overlaps are the C ABI's to refuse.
    for f in (lambda: att(q, c.k, c.v, table, pos, out=q), lambda: app(qkv, c.k, c.v, table, pos, inv, out=qkv),
              lambda: nrm(x, x, out=x), lambda: nrm(x, x.clone(), x[0].clone(), h_out=x),
              lambda: att(q, c.k, c.v, table, pos, out=c.k.view(torch.float32).view(-1, 256)[:2]),
              lambda: smp(x, u, out=u.view(torch.int32)), lambda: smp(x, u, top_p=u, out=u.view(torch.int32))):
        with pytest.raises(gpu.W4A8Error) as e:
            f()
        assert e.value.status == -2
    # No rows: no launch.
    none = torch.zeros((0, 256), device="cuda")
    assert att(none, c.k, c.v, table[:0], pos[:0]).shape == (0, 256)
    assert app(torch.zeros((0, 512), device="cuda"), c.k, c.v, table[:0], pos[:0], inv).shape == (0, 256)
    assert nrm(none, none, torch.ones(256, device="cuda"))[1].shape == (0, 256)
    assert smp(none, u[:0]).shape == (0,)


# -------------------------------------------------- a decode, from end to end


def test_decode_steps(gpu):
    """Three tokens of a two-layer model through the framework alone: the fused rmsnorm GEMVs, append, attention, o,
    the residual norms, the MLP, the LM head and the draw; each of the new operators against the oracle on the
    inputs that it was given there."""
    import torch
    hidden, heads, kvh, d, ffn, vocab, page, layers = 2048, 32, 8, 64, 2048, 4000, 16, 2
    g = torch.Generator(device="cuda").manual_seed(0)

    def weight(rows, k):
        return gpu.quantize_q4_0(0.02 * torch.randn((rows, k), generator=g, device="cuda"))

    qkv_rows = (heads + 2 * kvh) * d
    L = [dict(qkv=weight(qkv_rows, hidden), o=weight(hidden, heads * d), gu=weight(2 * ffn, hidden),
              down=weight(hidden, ffn)) for _ in range(layers)]
    lm, emb = weight(vocab, hidden), torch.randn((vocab, hidden), generator=g, device="cuda")
    one = torch.ones(hidden, device="cuda")
    cache = [[torch.zeros((4, kvh, page, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(layers)]
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    inv, token = dev(_inv_freq(d)), 17
    u = torch.rand(20, generator=g, device="cuda")
    drawn = []
    for step in range(18):                              # past the first page
        pos = torch.tensor([step], dtype=torch.int32, device="cuda")
        x = emb[token].clone()
        for l, (k, v) in zip(L, cache):
            qkv = gpu.gemv_rmsnorm(l["qkv"], hidden, x, one, 1e-5)
            q = gpu.rope_append(qkv.view(1, -1), k, v, table, pos, inv, interleaved=True)
            o = gpu.paged_attention(q, k, v, table, pos)
            want, bound = S.attention(host(q).reshape(1, heads, d), host(k.float()), host(v.float()), host(table), host(pos), d ** -0.5)
            assert (np.abs(host(o).reshape(1, heads, d) - want).max(-1) <= bound).all()
            y = gpu.gemv_q4_0_f32(l["o"], heads * d, o[0])
            before = host(x)
            gpu.residual_rmsnorm(x, y, out=x)
            assert_bytes_equal(host(x), before + host(y))
            act = gpu.gemv_gate_up_silu(l["gu"], hidden, x, one, 1e-5)
            gpu.residual_rmsnorm(x, gpu.gemv_q4_0_f32(l["down"], ffn, act), out=x)
        logits = gpu.gemv_rmsnorm(lm, hidden, x, one, 1e-5)
        token = int(host(gpu.sample(logits, u[step:step + 1], temperature=0.8, top_k=40, top_p=0.95)).item())
        assert token == S.sample(host(logits), host(u)[step], 0.8, 40, 0.95)
        drawn.append(token)
    assert len(set(drawn)) > 3


# ----------------------------------------------------------- far positions


@pytest.mark.parametrize("first,freqs", [(0, (0.0, 1.0)), (2 ** 29, (0.5, 1.0)), (2 ** 31 - 4000, (0.5, 1.0)),
                                         (2 ** 31 - 4000, (1e-6, 1e-2)), (2 ** 31 - 4000, (1.0, 512.0))])
def test_append_angles(gpu, first, freqs):
    """Sine and cosine themselves, of unit pairs: within 2^-23 of the exact angle's at every position and frequency of
    up to 2^40 radians. The positions lie past the table: nothing is stored."""
    m, d = 2000, 64
    rng = np.random.default_rng(first % 1000 + 1)
    inv = rng.uniform(*freqs, d // 2).astype(np.float32)
    pos = np.sort(rng.integers(first, min(first + 200000, 2 ** 31), m)).astype(np.int32)
    c = Cached([16], 1, d, 16, "float16")
    qkv = np.zeros((m, 3 * d), np.float32)
    qkv[:, : d // 2] = 1.0
    got = host(gpu.rope_append(dev(qkv), c.k, c.v, dev(np.full((1, 1), -1, np.int32)).expand(m, -1), dev(pos), dev(inv)))
    angle = np.stack([S.angles(pos, f) for f in inv], 1)
    err = np.abs(got - np.concatenate([np.cos(angle), np.sin(angle)], 1))
    assert err.max() <= 2.0 ** -23, err.max() * 2.0 ** 23
