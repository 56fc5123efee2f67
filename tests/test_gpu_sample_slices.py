"""The sampler's draw over slices of the rows (include/w4a8_step.h): the three launches that vocabularies take, with a
workspace between them, on the inputs that are hard for them. Tokens against the oracle, exactly."""

from __future__ import annotations

import numpy as np
import pytest

import step_oracle as S
from gpu_helpers import dev, host
from test_gpu_step import check_sample

pytestmark = pytest.mark.gpu

SIZES = [20011, 131073]          # five slices and thirty-three, the last ones short


def _need(gpu, m, n):
    """The workspace of m rows of n logits: nothing but slices takes one."""
    need = gpu.lib().w4a8_sample_workspace_bytes(m, n)
    assert need > 0
    return need


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("settings", [dict(), dict(temperature=0), dict(top_k=20), dict(top_p=0.7), dict(min_p=0.3),
                                      dict(temperature=50.0), dict(temperature=0.7, top_k=200, top_p=0.9, min_p=0.01)], ids=str)
def test_masked_rows(gpu, n, settings):
    """Rows of -inf or NaN alone, between rows that have a token; single tokens in the first, a middle and the last
    slice; slices with nothing to draw; the type's lowest value as a mask; +inf in some slices."""
    _need(gpu, 12, n)
    rng = np.random.default_rng(n)
    logits = rng.standard_normal((12, n)).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2:5] = -np.inf
    logits[2, 3], logits[3, n // 2], logits[4, n - 1] = -1e30, 5.0, np.finfo(np.float32).max
    logits[5, rng.permutation(n)[: n - 50]] = -np.inf
    logits[6, rng.permutation(n)[: n - 50]] = np.nan
    logits[7, 4096:] = -np.finfo(np.float32).max
    logits[8, 5000:9000] = np.inf
    logits[9] = np.finfo(np.float32).max * np.where(np.arange(n) % 2, 1, -1)
    logits[10, 1:] = np.nan
    logits[11] = np.where(np.arange(n) % 5, -np.inf, np.nan)
    for u in (0.0, 0.4, 0.99999):
        want = check_sample(gpu, logits, np.full(12, u), **settings)
        assert want[0] == want[1] == want[11] == -1 and want[2:5] == [3, n // 2, n - 1] and want[7] < 4096 and want[10] == 0
        assert 5000 <= want[8] < 9000 and want[9] % 2 == 1


@pytest.mark.parametrize("n", SIZES)
def test_extreme_temperatures(gpu, n):
    _need(gpu, 4, n)
    rng = np.random.default_rng(15)
    big = np.finfo(np.float32).max
    logits = np.stack([rng.standard_normal(n) * 3, rng.standard_normal(n) * 1e37, rng.choice([-big, big, 0.0, 1.0], n),
                       np.where(rng.random(n) < 0.5, -np.inf, np.clip(rng.standard_normal(n), -3, 3) * 1e38)])
    u = np.full(4, 0.61)
    for t in (np.inf, big, 1e30, 1e-45, 1e-38):
        check_sample(gpu, logits, u, temperature=np.full(4, t))
        check_sample(gpu, logits, u, temperature=np.full(4, t), top_k=n // 2 + 100, top_p=0.7)


@pytest.mark.parametrize("n", SIZES)
def test_random_numbers_out_of_range(gpu, n):
    _need(gpu, 7, n)
    logits = np.random.default_rng(13).standard_normal((7, n))
    u = [-0.5, -0.0, np.nan, 1.0, 2.0, np.inf, 1 - 2.0 ** -24]
    for more in (dict(), dict(top_p=0.6), dict(top_k=300)):
        check_sample(gpu, logits, u, **more)


@pytest.mark.parametrize("n", SIZES)
def test_ties_and_zeros(gpu, n):
    """Few distinct values, -0 equal to +0, ties over the slices' ends."""
    _need(gpu, 6, n)
    rng = np.random.default_rng(11)
    logits = np.round(rng.standard_normal((6, n)) * 2) / 2
    logits[:, ::7] *= -1.0
    u = rng.random(6)
    for more in (dict(), dict(top_k=33), dict(top_k=n // 8, top_p=0.8)):
        check_sample(gpu, logits, u, **more)
    zeros = np.where(np.arange(n) % 2, 0.0, -0.0)[None].repeat(4, 0)
    at = np.array([0.0, 0.25, 0.5, 0.75])
    assert check_sample(gpu, zeros, at) == [int(f * n) for f in at]


@pytest.mark.parametrize("n", SIZES)
def test_strided_rows_and_single_row(gpu, n):
    """Rows of a padded vocabulary, whose padding is above every logit, at an odd offset; each alone as well."""
    import torch
    _need(gpu, 5, n)
    rng = np.random.default_rng(14)
    wide = np.full((5, n + 9), 1e9, np.float32)
    wide[:, 3:n + 3] = rng.standard_normal((5, n))
    u = rng.random(5).astype(np.float32)
    d = dev(wide)
    want = [S.sample(wide[i, 3:n + 3], u[i], top_p=0.9) for i in range(5)]
    assert host(gpu.sample(d[:, 3:n + 3], dev(u), top_p=0.9)).tolist() == want
    for i in range(5):
        assert host(gpu.sample(d[i, 3:n + 3], dev(u[i:i + 1]), top_p=0.9)).tolist() == want[i:i + 1]
    out = torch.full((7,), 9, dtype=torch.int32, device="cuda")
    gpu.sample(d[:, 3:n + 3], dev(u), top_p=0.9, out=out)
    assert host(out).tolist() == want + [9, 9]


def test_workspace_of_any_contents(gpu):
    """Calls of every kind in a row into one workspace, filled with bits of each kind before: the tokens of a fresh one,
    and nothing behind the workspace or the tokens."""
    import torch
    m, n = 6, 33333
    need = _need(gpu, m, n)
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((m, n)).astype(np.float32) * 2
    logits[2] = -np.inf
    u = rng.random(m).astype(np.float32)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    out = torch.full((m + 2,), 77, dtype=torch.int32, device="cuda")
    dl, du = dev(logits), dev(u)
    for poison in (0, 255, 0x7F, 1):
        ws[:need].fill_(poison)
        ws[need:].fill_(0xAA)
        for more in (dict(top_k=50), dict(top_p=0.95), dict(), dict(temperature=0), dict(top_k=20000, top_p=0.9), dict(top_k=50)):
            assert gpu.sample(dl, du, out=out, workspace=ws[:need], **more) is out
            assert host(out).tolist() == [S.sample(logits[i], u[i], **more) for i in range(m)] + [77, 77]
        assert (host(ws[need:]) == 0xAA).all()
    # Fewer rows, then more slices a row, in the same memory.
    for k in (1, 3):
        assert _need(gpu, k, n) <= need
        assert host(gpu.sample(dl[:k], du[:k], workspace=ws[:need])).tolist() == [S.sample(logits[i], u[i]) for i in range(k)]
    for short in (ws[:need - 1], ws[:0]):
        with pytest.raises(ValueError, match="the call needs"):
            gpu.sample(dl, du, workspace=short)
    with pytest.raises(gpu.W4A8Error) as e:                      # not 16-byte aligned
        gpu.sample(dl, du, workspace=ws[8:need + 8])
    assert e.value.status == -3


def test_side_stream(gpu):
    """On a side stream, behind work that is still running there."""
    import torch
    m, n = 3, 40009
    _need(gpu, m, n)
    g = torch.Generator(device="cuda").manual_seed(3)
    logits, u = 2 * torch.randn((m, n), generator=g, device="cuda"), torch.rand(m, generator=g, device="cuda")
    settings = (dict(top_p=0.9), dict(top_k=40), dict())
    want = [host(gpu.sample(2 * logits, u, **s)).tolist() for s in settings]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-2
        lead = big[0, 0] * 0 + 2
        lead = torch.where(torch.isfinite(lead), lead, torch.full_like(lead, 2.0))
        got = [gpu.sample(lead * logits, u, **s) for s in settings]
    assert [host(t).tolist() for t in got] == want


def test_graph_replays(gpu):
    """Two graphs of their own workspaces, replayed on new inputs, rows without a token coming and going, with eager
    calls between: every replay against the eager call and the oracle."""
    import torch
    m, n = 4, 24001
    need = _need(gpu, m, n)
    settings = (dict(temperature=0.8, top_k=40, top_p=0.95), dict(top_p=0.8, min_p=0.001))
    runs = []
    for s in settings:
        t = dict(logits=torch.randn((m, n), device="cuda"), u=torch.rand(m, device="cuda"),
                 ws=torch.full((need,), 255, dtype=torch.uint8, device="cuda"),
                 out=torch.zeros(m, dtype=torch.int32, device="cuda"))

        def call(t=t, s=s):
            return gpu.sample(t["logits"], t["u"], out=t["out"], workspace=t["ws"], **s)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        runs.append((t, s, graph))
    rng = np.random.default_rng(5)
    for i in range(6):
        for t, _, _ in runs:
            logits = rng.standard_normal((m, n)).astype(np.float32) * (1 + i)
            if i % 2:
                logits[i % m] = (-np.inf, np.nan)[i % 3 == 0]
            t["logits"].copy_(dev(logits))
            t["u"].copy_(dev(rng.random(m).astype(np.float32)))
            t["out"].fill_(-9)
        torch.cuda.synchronize()
        for _, _, graph in runs:
            graph.replay()
        torch.cuda.synchronize()
        for t, s, _ in runs:
            got = host(t["out"]).tolist()
            logits, u = host(t["logits"]), host(t["u"])
            assert got == host(gpu.sample(t["logits"], t["u"], **s)).tolist()
            assert got == [S.sample(logits[j], u[j], **s) for j in range(m)]


@pytest.mark.parametrize("m,n", [(1, 262144), (1, 524288), (8, 250007), (64, 128256)])
def test_most_slices(gpu, m, n):
    """A slice for every lane of a wave (64, and longer ones past 2^18 logits), and many rows of eight."""
    _need(gpu, m, n)
    rng = np.random.default_rng(m)
    logits = rng.standard_normal((m, n)).astype(np.float32) * 2
    u = rng.random(m)
    for more in (dict(top_k=40), dict(top_p=0.9)):
        few = min(m, 8)
        got = host(gpu.sample(dev(logits), dev(u.astype(np.float32)), **more))
        assert got[:few].tolist() == [S.sample(logits[i], u[i], **more) for i in range(few)]
