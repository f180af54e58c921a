"""Ends of kllm_sample's range: rows whose largest logit is a zero, a
subnormal or the lowest number, at the ends of the temperatures.  Tokens are
compared for equality with the definition in 64 bits, temperatures taken into
[1e-30, 1e30] as the header has it; no number lies within 2^-24 of a border."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SUB = np.float32(1e-40)     # a subnormal number


def _tops(V, rng):
    """Rows by their largest logit: zeros of either sign, subnormals, alone and many."""
    below = -np.abs(rng.standard_normal((8, V))).astype(np.float32) - np.float32(0.5)
    x = below.copy()
    at = rng.integers(0, V, 8)
    x[0, at[0]] = 0.0                              # shifted by its maximum
    x[1, at[1]] = -0.0
    x[2, at[2]] = SUB
    x[3] = 0.0                                     # equal ones
    x[4] = -0.0
    x[5] = SUB
    x[6] = np.where(rng.random(V) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[7] = np.where(rng.random(V) < 0.5, SUB, np.float32(0.0))
    return x


def _check(x, T, k, p, mp, u):
    import servecases as S
    n = len(x)
    full = lambda a, d, t: None if a is None else np.full(n, a, t)
    Tc = min(max(float(np.float32(T)), float(np.float32(1e-30))), float(np.float32(1e30)))
    got = S.run_sample(S.dev(x), np.full(n, T, np.float32), full(k, 0, np.int32), full(p, 1, np.float32),
                       full(mp, 0, np.float32), u)
    want = [S.sample_plain(r, Tc, k or 0, 1.0 if p is None else float(np.float32(p)),
                           0.0 if mp is None else float(np.float32(mp)), float(u[i])) for i, r in enumerate(x)]
    assert got.tolist() == want, (T, k, p, mp)


@pytest.mark.parametrize("V", [3, 700, 5000, 40001])
@pytest.mark.parametrize("T", [1e-38, 1e-30, 5e-29, 7.2e-29, 1e-28, 1e-10, 1.0])
@pytest.mark.parametrize("k,p,mp", [(None, None, None), (2, None, None), (600, None, None), (None, 0.7, None),
                                    (650, 0.9, None), (None, None, 0.5), (20, 0.5, 0.1)])
def test_largest_logit_of_zero_or_subnormal(gpu, V, T, k, p, mp):
    rng = np.random.default_rng(V)
    _check(_tops(V, rng), T, k, p, mp, rng.random(8).astype(np.float32))


@pytest.mark.parametrize("V", [600, 5000, 40001])
@pytest.mark.parametrize("T", [1e28, 1e30])
@pytest.mark.parametrize("k,p,mp", [(None, None, None), (3, None, None), (None, 0.6, None), (900, 0.9, None),
                                    (None, None, 0.5)])
def test_masked_tokens_beside_the_lowest_number(gpu, V, T, k, p, mp):
    """-infinity weighs nothing, even where the largest logit is the type's lowest
    number and the temperature so high that the distance to 2^128 is small."""
    rng = np.random.default_rng(V)
    low = np.finfo(np.float32).min
    x = np.full((6, V), -np.inf, np.float32)
    x[0, V // 2] = low
    x[1, 1:] = low
    x[2, 5::2] = low
    x[3] = np.where(rng.random(V) < 0.2, low, -np.inf)
    x[4, V - 3:] = low * np.float32(0.75)
    x[5] = np.where(rng.random(V) < 0.2, low * rng.random(V).astype(np.float32), -np.inf)
    for u in (0.0, 0.5, 0.999):
        _check(x, T, k, p, mp, np.full(6, u, np.float32))


def test_clusters_on_a_busy_gpu(gpu):
    """A row's blocks start whenever the work beside them leaves room: the tokens stay."""
    import ctypes as C

    import kmap_b200 as K
    import torch

    import servecases as S
    rng = np.random.default_rng(21)
    x = S.dev(rng.standard_normal((96, 128256)).astype(np.float32))
    p, u = np.full(96, 0.9, np.float32), rng.random(96).astype(np.float32)
    want = S.run_sample(x, None, None, p, None, u).tolist()
    outs = [S.sample_args(x, None, None, p, None, u) for _ in range(20)]
    work, side = torch.randn(4096, 4096, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for a, _, _ in outs:
        work @ work
        K.check(K.lib().kllm_sample(C.byref(a), side.cuda_stream))
    torch.cuda.synchronize()
    assert [o[:-1].cpu().tolist() for _, o, _ in outs] == [want] * len(outs)
