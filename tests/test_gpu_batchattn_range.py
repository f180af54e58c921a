"""kllm_batch_attention at the ends of fp32's range: scores, queries, keys and
values that are finite but very large."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _caches(fmt, n, nkv, hd, P, m, k, v):
    """A prefix of P positions and m own ones of n sequences, every key row k, every value row v."""
    import servecases as S
    pre = S.Cache(fmt, 1, nkv, P, hd) if P else None
    own = S.Cache(fmt, n, nkv, max(m, 1), hd)
    for c, length, seqs in ((pre, P, 1), (own, m, n)):
        if c is not None and length:
            c.put("k", np.broadcast_to(np.float32(k), (seqs, nkv, length, hd)).copy())
            c.put("v", np.broadcast_to(np.float32(v), (seqs, nkv, length, hd)).copy())
    return pre, own


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("P,m", [(0, 1), (0, 40), (0, 1500), (70, 0), (70, 3), (2700, 3)])
def test_no_score_above_minus_infinity_is_nan(gpu, fmt, P, m):
    """Finite queries and keys whose products are below fp32's range, in every split of the
    positions: NaN, never the zeros of a row without positions."""
    import torch

    import servecases as S
    n, nh, nkv, hd = 50, 8, 2, 64
    k = np.zeros(hd, np.float32)
    k[0] = -2.0 ** 100
    pre, own = _caches(fmt, n, nkv, hd, P, m, k, 1.0)
    q = np.zeros((n, nh, hd), np.float32)
    q[..., 0] = 2.0 ** 100
    lens = S.dev(np.full(n, m, np.int32))
    out = torch.zeros(n, nh * hd, device="cuda")
    S.run_attention(S.dev(q.reshape(n, -1)), out, nh, 1.0, pre, P, own, lens, max(m, 1))
    assert np.isnan(out.cpu().numpy()).all()


def _few(hd, nh, nkv, n, P, seed, qsize, ksize, vsize):
    """Inputs of test_gpu_batchattn_accuracy's sparse() brought to other sizes, with one position of
    30 above the others' scores for each query row's dims: sums of p |v| stay near the largest |v|."""
    import test_gpu_batchattn_accuracy as A
    q, k, v = A.sparse(seed, hd, nh, nkv, n, P)
    q[..., 4] = 1
    k[..., 4] = -30
    k[:, P // 2, 4] = 0
    q, k, v = (np.float32(x * s) for x, s in ((q, qsize), (k, ksize), (v, vsize)))
    return q, k, v


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", [(128, 8, 2, 5, 300), (128, 8, 2, 64, 3001), (64, 8, 8, 33, 4100)])
@pytest.mark.parametrize("qsize,ksize,vsize", [
    (1.0, 1.0, 2.0 ** 112), (1.0, 1.0, 2.0 ** 116), (1.0, 1.0, 2.0 ** -90),
    (2.0 ** 95, 2.0 ** -95, 1.0), (2.0 ** 120, 2.0 ** -120, 1.0), (2.0 ** -90, 2.0 ** 90, 2.0 ** 116)])
def test_large_finite_numbers(gpu, fmt, hd, nh, nkv, n, P, qsize, ksize, vsize):
    """Queries up to 2^121, values up to 2^117: as near as of moderate size.  (Larger values are
    documented to overflow: a part's sum of p |v|, p relative to the part's own largest score, is
    up to its positions times |v|, 128 x 2^126 at the least.)"""
    import test_gpu_batchattn_accuracy as A
    q, k, v = _few(hd, nh, nkv, n, P, hd + n, qsize, ksize, vsize)
    got, k, v = A.run(fmt, q, k, v, 2)
    want, norm = A.exact(q, k, v)
    # (scores reach 33: the 595 units of scores up to 21 there become 935, with the 310 2^-13.7)
    assert np.isfinite(got).all() and (np.abs(got - want) <= 2.0 ** -13.7 * norm[..., None]).all()


@pytest.mark.parametrize("n,P", [(5, 300), (50, 2700)])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_one_number_of_a_value_that_is_not_finite(gpu, n, P, bad):
    """An fp32 value with one such number: NaN in that dim for every row of its kv head; the other dims
    are NaN or what they were, and never something else."""
    import torch

    import servecases as S
    rng = np.random.default_rng(3)
    nh, nkv, hd = 8, 2, 64
    pre = S.Cache("f32", 1, nkv, P, hd)
    for name in "kv":
        pre.put(name, rng.standard_normal((1, nkv, P, hd)).astype(np.float32))
    q = S.dev(rng.standard_normal((n, nh * hd)).astype(np.float32))
    a, b = (torch.zeros(n, nh * hd, device="cuda") for _ in "ab")
    S.run_attention(q, a, nh, 0.125, pre, P)
    pre.v.view(-1)[(P // 2) * hd + 7] = float(bad)
    S.run_attention(q, b, nh, 0.125, pre, P)
    a, b = (t.cpu().numpy().reshape(n, nh, hd) for t in (a, b))
    head = np.arange(nh) < nh // nkv
    assert np.isnan(b[:, head, 7]).all() and np.array_equal(a[:, ~head], b[:, ~head])
    assert (np.isnan(b[:, head]) | (a[:, head] == b[:, head])).all()
