"""Tokens drawn from logits with given uniform numbers (kllm_sample) against
the definition in 64 bits.  The weights are 2^-40 fixed point: a draw can
differ only where u falls within about 2^-35 of a border, so tokens are
compared for equality."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

VOCABS = [1, 2, 3, 31, 33, 600, 2049, 5000, 32000, 40001, 128256]


def _settings(rng, rows):
    T = rng.uniform(0.3, 2.0, rows).astype(np.float32)
    k = rng.integers(0, 60, rows).astype(np.int32)
    p = rng.uniform(0.1, 1.2, rows).astype(np.float32)
    mp = rng.uniform(-0.1, 0.3, rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    T[::5], k[1::4], p[2::4], mp[::3] = 0, 0, 1, 0
    return T, k, p, mp, u


def _want(x, T, k, p, mp, u):
    import servecases as S
    n = len(x)
    f = lambda a, d: np.full(n, d) if a is None else a
    T, k, p, mp = f(T, 1.0), f(k, 0), f(p, 1.0), f(mp, 0.0)
    return [S.sample_plain(x[i], float(T[i]), int(k[i]), float(p[i]), float(mp[i]), float(u[i]))
            for i in range(n)]


def _logits(rng, rows, V, kind):
    x = rng.standard_normal((rows, V)).astype(np.float32) * np.float32(2)
    if kind == "peaked":
        x[np.arange(rows), rng.integers(0, V, rows)] += 12
    elif kind == "ties":      # few distinct values
        x = np.round(x).astype(np.float32)
    elif kind == "equal":
        x[:] = np.float32(-3.25)
    elif kind == "far":       # nearly everything without weight
        x *= 100
    return x


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("kind", ["bulk", "peaked", "ties", "equal", "far"])
def test_against_the_definition(gpu, V, kind):
    import servecases as S
    rng = np.random.default_rng(V + len(kind))
    rows = 24 if V < 20000 else 12
    x = _logits(rng, rows, V, kind)
    T, k, p, mp, u = _settings(rng, rows)
    for sel in ((T, k, p, mp), (T, None, p, None), (None, k, None, None), (T, None, None, mp),
                (None, None, None, None), (T, k, p, None)):
        got = S.run_sample(S.dev(x), *sel, u)
        assert got.tolist() == _want(x, *sel, u), sel


def test_edges_of_the_draw(gpu):
    """u at 0, just below 1 and outside [0, 1), NaN; the borders of equal weights."""
    import servecases as S
    x = np.zeros((9, 64), np.float32)
    u = np.array([0, 1 - 2.0 ** -24, 1, 7, -1, np.nan, 0.5, 0.25, 0.015625], np.float32)
    got = S.run_sample(S.dev(x), u=u)
    # 64 equal weights: the first index whose (i + 1) / 64 exceeds u
    assert got.tolist() == [0, 63, 63, 63, 0, 0, 32, 16, 1]


def test_masked_and_non_finite_logits(gpu):
    """-infinity masks, NaN, +infinity, rows without any finite logit, the type's lowest."""
    import servecases as S
    V = 5000
    rng = np.random.default_rng(1)
    x = rng.standard_normal((10, V)).astype(np.float32)
    x[0, :-1] = -np.inf                    # one token left
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 100], x[3, 4000] = np.inf, np.inf
    x[4, ::2] = np.nan
    x[5, 0] = np.nan
    x[6, 0] = np.nan                       # greedy: the decode's rule keeps 0
    x[7, :] = np.finfo(np.float32).min
    x[8, 1:] = np.finfo(np.float32).min
    x[9, 7] = np.inf
    T = np.ones(10, np.float32)
    T[6] = 0
    for u in (0.0, 0.3, 0.77, 0.999):
        us = np.full(10, u, np.float32)
        for k, p in ((None, None), (np.full(10, 3, np.int32), None), (None, np.full(10, .5, np.float32)),
                     (np.full(10, 40, np.int32), np.full(10, .9, np.float32))):
            got = S.run_sample(S.dev(x), T, k, p, None, us)
            assert got.tolist() == _want(x, T, k, p, None, us), (u, k, p)
    assert got[0] == V - 1 and got[1] == 0 and got[2] == 0 and got[6] == 0


def test_odd_settings(gpu):
    """Settings at and past their ends, NaN ones: off, or the first of the order."""
    import servecases as S
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, 700)).astype(np.float32)
    u = rng.random(8).astype(np.float32)
    nan = float("nan")
    T = np.array([1e-30, 1e30, 1, 1, 1, 1, 1, nan], np.float32)
    k = np.array([0, 0, -5, 700, 10 ** 9, 1, 0, 0], np.int32)
    p = np.array([1, 1, 0, -1, nan, 1, 1, 1], np.float32)
    mp = np.array([0, 0, 0, 0, nan, 0, 5, 0], np.float32)
    want = _want(x, np.where(np.isnan(T), 1, T), k, np.where(np.isnan(p), 1, p),
                 np.where(np.isnan(mp), 0, mp), u)
    assert S.run_sample(S.dev(x), T, k, p, mp, u).tolist() == want


@pytest.mark.parametrize("V", [1 << 20, 500001])
def test_vocabularies_past_the_blocks_memory(gpu, V):
    import servecases as S
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, V)).astype(np.float32)
    T, k, p, mp, u = _settings(rng, 3)
    got = S.run_sample(S.dev(x), T, k, p, None, u)
    assert got.tolist() == _want(x, T, k, p, None, u)


def test_row_stride_and_unaligned_rows(gpu):
    import servecases as S
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 1003)).astype(np.float32)
    T, k, p, mp, u = _settings(rng, 6)
    got = S.run_sample(S.dev(x), T, k, p, mp, u, vocab=999)
    assert got.tolist() == _want(x[:, :999], T, k, p, mp, u)


def test_a_rows_token_does_not_depend_on_the_others(gpu):
    import servecases as S
    rng = np.random.default_rng(6)
    x = rng.standard_normal((128, 3001)).astype(np.float32)
    T, k, p, mp, u = _settings(rng, 128)
    every = S.run_sample(S.dev(x), T, k, p, mp, u)
    for i in (0, 1, 77, 127):
        s = slice(i, i + 1)
        assert S.run_sample(S.dev(x[s]), T[s], k[s], p[s], mp[s], u[s])[0] == every[i]


def test_frequencies(gpu):
    """Evenly spaced u draw each token as often as its probability says: within one draw."""
    import servecases as S
    n = 4096
    x = np.tile(np.log(np.array([1, 2, 3, 4, 6], np.float64)).astype(np.float32), (n, 1))
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = np.bincount(S.run_sample(S.dev(x), u=u), minlength=5)
    assert (np.abs(got - n * np.array([1, 2, 3, 4, 6]) / 16) <= 1).all()


def test_in_a_graph(gpu):
    import torch

    import kmap_b200 as K
    import servecases as S
    rng = np.random.default_rng(7)
    x = rng.standard_normal((16, 32000)).astype(np.float32)
    u1, u2 = (rng.random(16).astype(np.float32) for _ in "ab")
    dx, du = S.dev(x), S.dev(u1)
    p = S.dev(np.full(16, 0.9, np.float32))
    out = torch.zeros(16, dtype=torch.int32, device="cuda")
    a = K.SampleRows(16, 32000, dx.data_ptr(), 32000, None, None, p.data_ptr(), None,
                     du.data_ptr(), out.data_ptr())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.check(K.lib().kllm_sample(C.byref(a), torch.cuda.current_stream().cuda_stream))
    for u in (u2, u1):
        du.copy_(S.dev(u))
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == _want(x, None, None, np.full(16, np.float32(0.9)), None, u)


@pytest.mark.parametrize("V", [7000, 16000, 33000])
@pytest.mark.parametrize("rows", [40, 160])
def test_many_rows_and_their_split(gpu, V, rows):
    """Rows take fewer blocks each where there are many: the tokens are those
    of a row alone, and of the definition."""
    import servecases as S
    rng = np.random.default_rng(V + rows)
    x = _logits(rng, rows, V, "ties" if rows == 40 else "bulk")
    T, k, p, mp, u = _settings(rng, rows)
    k[::2] = 0
    got = S.run_sample(S.dev(x), T, k, p, mp, u).tolist()
    assert got[:12] == _want(x[:12], T[:12], k[:12], p[:12], mp[:12], u[:12])
    for i in range(0, rows, 7):
        s = slice(i, i + 1)
        assert S.run_sample(S.dev(x[s]), T[s], k[s], p[s], mp[s], u[s]).tolist() == got[s], i


def test_two_calls_at_once(gpu):
    import torch

    import servecases as S
    rng = np.random.default_rng(77)
    x = [S.dev(_logits(rng, 16, 128256, "bulk")) for _ in "ab"]
    T, k, p, mp, u = _settings(rng, 16)
    k[:] = 0
    want = [S.run_sample(t, T, k, p, mp, u).tolist() for t in x]
    streams = [torch.cuda.Stream() for _ in "ab"]
    a = [S.sample_args(t, T, k, p, mp, u) for t in x]
    torch.cuda.synchronize()
    import kmap_b200 as K
    for _ in range(5):
        for args, s in zip(a, streams):
            K.check(K.lib().kllm_sample(C.byref(args[0]), s.cuda_stream))
    torch.cuda.synchronize()
    assert [args[1][:-1].cpu().tolist() for args in a] == want
