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
