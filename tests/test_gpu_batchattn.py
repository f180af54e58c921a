"""Attention of a batch that shares a prefix (kllm_batch_attention) against
softmax(q k^T) v in 64 bits on the values that the caches hold.

Tolerance, per row: a score is a sum of products whose queries carry 22 bits
(two 11-bit terms) and whose keys are exact (8-bit codes) or carry 22, added in
fp32; a product operation of 16 terms may lose half a unit of 2^-23 of its
largest term for each, so 2^-18 of sum |q k| bounds it: |ds| <= 2^-18 S with
S = scale max_j sum_d |q_d k_jd|.  Weights then carry exp(ds): a relative
2 |ds| at most, numerator and denominator; the sum of p v carries another
2^-18 from its own terms, exp2 and the join of the parts 2^-20 each.
Together (2 S + 4) 2^-18 max |v|."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HEADS = [(4, 2, 32), (32, 4, 64), (3, 3, 64), (32, 8, 128), (2, 2, 128), (10, 1, 128), (12, 4, 64)]


def _check(fmt, nh, nkv, hd, n, P, lens, max_pos, seed, kscale=1.0, vscale=None, qpad=0, max_len=None,
           prefix=True, own=True, stream=None):
    import torch

    import servecases as S
    rng = np.random.default_rng(seed)
    G, scale = nh // nkv, float(np.float32(1 / np.sqrt(hd)))
    q = (2 * rng.standard_normal((n, nh * hd + qpad))).astype(np.float32)
    fill = 0x7f if fmt == "e4m3" else float("nan") if fmt == "f32" else 0x55   # behind the lengths
    pre = S.Cache(fmt, 1, nkv, max(P, 1) + 3, hd, fill=fill) if prefix else None
    mine = S.Cache(fmt, n, nkv, max_pos, hd, pad=16, fill=fill) if own else None

    def rows(m, seqs):
        x = rng.standard_normal((seqs, nkv, m, hd)).astype(np.float32)
        return x * np.float32(kscale)

    pk = pv = np.zeros((1, nkv, 0, hd))
    if prefix and P:
        pk = pre.put("k", rows(P, 1))
        x = rows(P, 1)
        pv = pre.put("v", x * vscale(x.shape[2]) if vscale else x)
    lens = np.asarray(lens, np.int32)
    ok = ov = np.zeros((n, nkv, 0, hd))
    most = 0
    if own:
        most = int(min(max(lens.max(), 0), max_pos))
        ok, ov = mine.put("k", rows(most, n)), None
        x = rows(most, n)
        ov = mine.put("v", x * vscale(x.shape[2]) if vscale and most else x)
        # positions behind a sequence's length hold what must not be read
        for i, m in enumerate(lens):
            m = max(int(m), 0)
            for t in (mine.k, mine.v):
                t[i, :nkv * max_pos * hd].view(nkv, max_pos, hd)[:, m:] = fill
            for t in (mine.ks, mine.vs):
                t[i, :nkv * max_pos].view(nkv, max_pos)[:, m:] = float("nan")
    out = torch.full((n, nh * hd + qpad), -9.0, device="cuda")
    S.run_attention(S.dev(q), out, nh, scale, pre, P, mine, S.dev(lens) if own else None,
                    max_pos if max_len is None else max_len, stream)
    got = out.cpu().numpy().astype(np.float64)
    assert (got[:, nh * hd:] == -9).all()
    cap = max_pos if max_len is None else min(max_pos, max_len)
    for i in range(n):
        if own and lens[i] < 0:
            assert (got[i] == -9).all()
            continue
        m = min(int(lens[i]), cap) if own else 0
        for h in range(nkv):
            k = np.concatenate([pk[0, h], ok[i, h, :m]])
            v = np.concatenate([pv[0, h], ov[i, h, :m]])
            qi = q[i, :nh * hd].astype(np.float64).reshape(nkv, G, hd)[h]
            want, s, vm = S.attend(qi, k, v, scale)
            tol = (2 * s + 4) * 2.0 ** -18 * vm
            err = np.abs(got[i, :nh * hd].reshape(nkv, G, hd)[h] - want)
            assert (err <= tol[:, None]).all(), (i, h, err.max(), tol.min())


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_prefix_and_own(gpu, fmt, nh, nkv, hd):
    """Lengths around the tiles' edges, none at all, padding rows."""
    _check(fmt, nh, nkv, hd, 7, 97, [0, 1, 33, -1, 64, 31, 17], 64, nh + hd)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("P", [0, 1, 31, 32, 128, 129, 1000])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_prefix_lengths(gpu, fmt, P, n):
    rng = np.random.default_rng(P + n)
    _check(fmt, 8, 2, 128, n, P, rng.integers(0, 20, n), 20, P + n)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv", [(64, 32, 4), (128, 32, 8), (32, 4, 4)])
@pytest.mark.parametrize("n,P", [(33, 517), (16, 300), (64, 1100), (5, 2000)])
def test_many_rows_on_a_prefix(gpu, fmt, hd, nh, nkv, n, P):
    _check(fmt, nh, nkv, hd, n, P, np.arange(n) % 9, 8, n + P + hd)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
def test_prefix_alone_and_own_alone(gpu, fmt):
    _check(fmt, 8, 2, 64, 5, 333, [0] * 5, 4, 1, own=False)
    _check(fmt, 8, 2, 64, 5, 0, [1, 2, 700, 0, 129], 800, 2, prefix=False)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
def test_long_ragged(gpu, fmt):
    _check(fmt, 8, 2, 128, 6, 0, [2500, 1, 777, 2499, 0, 1300], 2500, 3, prefix=False)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("kscale", [1e-6, 1e3])
def test_magnitudes(gpu, fmt, kscale):
    """Tiny rows, and rows so large that the softmax picks one position."""
    _check(fmt, 8, 2, 64, 4, 200, [50, 3, 0, 7], 50, 5, kscale=kscale)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
def test_values_of_very_different_scale(gpu, fmt):
    """Value rows whose scales span 2^40: the sums keep the largest's precision."""
    def scales(n):
        return np.float32(2.0) ** (np.arange(n) * 7 % 41 - 20).astype(np.float32)[:, None]
    _check(fmt, 8, 2, 128, 20, 300, [9] * 20, 9, 6, vscale=scales)


def test_lengths_past_the_bounds_are_cut(gpu):
    _check("i8", 4, 2, 64, 3, 10, [90, 64, 5], 64, 7)
    _check("i8", 4, 2, 64, 3, 10, [60, 64, 5], 64, 8, max_len=40)
    _check("i8", 4, 2, 64, 3, 10, [60, 64, 5], 64, 8, max_len=0)


def test_strides(gpu):
    _check("e4m3", 4, 2, 64, 3, 70, [5, 64, 0], 64, 9, qpad=5)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
def test_no_row_matters_to_another(gpu, fmt):
    """A query of NaN or infinities and a key scale of NaN spoil their own rows only."""
    import torch

    import servecases as S
    rng = np.random.default_rng(4)
    nh, nkv, hd, n, P = 8, 2, 64, 24, 300
    pre, own = S.Cache(fmt, 1, nkv, P, hd), S.Cache(fmt, n, nkv, 16, hd)
    for c, m, s in ((pre, P, 1), (own, 16, n)):
        c.put("k", rng.standard_normal((s, nkv, m, hd)).astype(np.float32))
        c.put("v", rng.standard_normal((s, nkv, m, hd)).astype(np.float32))
    q = rng.standard_normal((n, nh * hd)).astype(np.float32)
    lens = S.dev(np.full(n, 16, np.int32))
    a, b = (torch.zeros(n, nh * hd, device="cuda") for _ in "ab")
    S.run_attention(S.dev(q), a, nh, 0.125, pre, P, own, lens, 16)
    q[5], q[9, :hd] = np.nan, np.inf
    if fmt == "f32":
        own.k[11] = float("nan")
    else:
        own.ks[11] = float("nan")
    S.run_attention(S.dev(q), b, nh, 0.125, pre, P, own, lens, 16)
    a, b = a.cpu().numpy().reshape(n, nh, hd), b.cpu().numpy().reshape(n, nh, hd)
    assert np.isnan(b[5]).all() and np.isnan(b[9, 0]).all() and np.isnan(b[11]).all()
    keep = np.ones((n, nh), bool)
    keep[5] = keep[11] = keep[9, 0] = False
    assert np.array_equal(a[keep], b[keep])


def test_same_bits_again_and_in_a_graph(gpu):
    """Two runs, a captured and replayed one with new lengths, another stream."""
    import torch

    import kmap_b200 as K
    import servecases as S
    rng = np.random.default_rng(8)
    nh, nkv, hd, n, P, mp = 32, 8, 128, 32, 700, 200
    pre, own = S.Cache("i8", 1, nkv, P, hd), S.Cache("i8", n, nkv, mp, hd)
    for c, m, s in ((pre, P, 1), (own, mp, n)):
        c.put("k", rng.standard_normal((s, nkv, m, hd)).astype(np.float32))
        c.put("v", rng.standard_normal((s, nkv, m, hd)).astype(np.float32))
    q = S.dev(rng.standard_normal((n, nh * hd)).astype(np.float32))
    l1, l2 = (rng.integers(0, mp + 1, n).astype(np.int32) for _ in "ab")
    want = []
    for l in (l1, l2):
        o = torch.zeros(n, nh * hd, device="cuda")
        S.run_attention(q, o, nh, 0.1, pre, P, own, S.dev(l), mp)
        want.append(o.clone())
    o = torch.zeros(n, nh * hd, device="cuda")
    S.run_attention(q, o, nh, 0.1, pre, P, own, S.dev(l1), mp)
    assert torch.equal(o, want[0])
    lens, o = S.dev(l1), torch.zeros(n, nh * hd, device="cuda")
    a = K.BatchAttn(n, nh, P, mp, 0.1, q.data_ptr(), nh * hd, C.addressof(pre.c),
                    C.addressof(own.c), lens.data_ptr(), o.data_ptr(), nh * hd, None, 0)
    size = K.lib().kllm_batch_attention_workspace(C.byref(a))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        K.check(K.lib().kllm_batch_attention(C.byref(a), torch.cuda.current_stream().cuda_stream))
    for l, w in ((l2, want[1]), (l1, want[0])):
        lens.copy_(S.dev(l))
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, w)


# The prefix's tiles of 128 rows: enough positions x rows x kv heads, rows and
# positions that end inside a tile.
WIDE = [(128, 8, 2, 64, 3001), (128, 4, 4, 129, 3000), (64, 8, 1, 41, 2500), (64, 8, 8, 33, 4100),
        (32, 8, 2, 35, 3700), (128, 8, 1, 37, 5300)]


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", WIDE)
def test_128_row_tiles(gpu, fmt, hd, nh, nkv, n, P):
    lens = np.arange(n) % 9 - (np.arange(n) % 13 == 5)
    _check(fmt, nh, nkv, hd, n, P, lens, 8, n + P)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("kscale", [1e-6, 30.0])
def test_128_row_tiles_magnitudes(gpu, fmt, kscale):
    def scales(n):
        return np.float32(2.0) ** (np.arange(n) * 7 % 41 - 20).astype(np.float32)[:, None]
    _check(fmt, 8, 2, 64, 50, 2700, [3] * 50, 3, 6, kscale=kscale, vscale=scales, qpad=3)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("n,P", [(50, 2700), (5, 300)])
@pytest.mark.parametrize("what,bad", [("v", "nan"), ("k", "nan"), ("v", "inf"), ("k", "-inf")])
def test_rows_spoil_only_what_sees_them(gpu, fmt, n, P, what, bad):
    """Queries of NaN and infinities, one position of a kv head that is not
    finite: the other rows and heads keep their bits."""
    import torch

    import servecases as S
    rng = np.random.default_rng(14)
    nh, nkv, hd = 8, 2, 64
    pre, own = S.Cache(fmt, 1, nkv, P, hd), S.Cache(fmt, n, nkv, 16, hd)
    for c, m, s in ((pre, P, 1), (own, 16, n)):
        c.put("k", rng.standard_normal((s, nkv, m, hd)).astype(np.float32))
        c.put("v", rng.standard_normal((s, nkv, m, hd)).astype(np.float32))
    q = rng.standard_normal((n, nh * hd)).astype(np.float32)
    lens = S.dev(np.full(n, 16, np.int32))
    a, b, d = (torch.zeros(n, nh * hd, device="cuda") for _ in "abd")
    S.run_attention(S.dev(q), a, nh, 0.125, pre, P, own, lens, 16)
    q[1], q[3, :hd], q[4, hd:2 * hd] = np.nan, np.inf, -np.inf
    S.run_attention(S.dev(q), b, nh, 0.125, pre, P, own, lens, 16)
    at = P - 2                                          # of kv head 0
    if fmt == "f32":
        getattr(pre, what).view(-1)[at * hd:(at + 1) * hd] = float(bad)
    else:
        getattr(pre, what + "s").view(-1)[at] = float("nan")
    S.run_attention(S.dev(q), d, nh, 0.125, pre, P, own, lens, 16)
    a, b, d = (t.cpu().numpy().reshape(n, nh, hd) for t in (a, b, d))
    spoilt = np.zeros((n, nh), bool)
    spoilt[1] = spoilt[3, 0] = spoilt[4, 1] = True
    assert np.isnan(b[spoilt]).all() and np.array_equal(a[~spoilt], b[~spoilt])
    spoilt[:, :nh // nkv] = True
    assert np.isnan(d[spoilt]).all() and np.array_equal(a[~spoilt], d[~spoilt])


@pytest.mark.parametrize("fmt", ["i8", "f32"])
def test_two_calls_at_once(gpu, fmt):
    """Two streams, each with its own workspace, over the same prefix."""
    import torch

    import kmap_b200 as K
    import servecases as S
    rng = np.random.default_rng(18)
    nh, nkv, hd, n, P, mp = 8, 2, 128, 64, 3100, 300
    pre = S.Cache(fmt, 1, nkv, P, hd)
    pre.put("k", rng.standard_normal((1, nkv, P, hd)).astype(np.float32))
    pre.put("v", rng.standard_normal((1, nkv, P, hd)).astype(np.float32))
    calls = []
    for _ in range(2):
        own = S.Cache(fmt, n, nkv, mp, hd)
        own.put("k", rng.standard_normal((n, nkv, mp, hd)).astype(np.float32))
        own.put("v", rng.standard_normal((n, nkv, mp, hd)).astype(np.float32))
        q = S.dev(rng.standard_normal((n, nh * hd)).astype(np.float32))
        lens = S.dev(rng.integers(0, mp + 1, n).astype(np.int32))
        o = torch.zeros(n, nh * hd, device="cuda")
        a = K.BatchAttn(n, nh, P, mp, 0.1, q.data_ptr(), nh * hd, C.addressof(pre.c), C.addressof(own.c),
                        lens.data_ptr(), o.data_ptr(), nh * hd, None, 0)
        size = K.lib().kllm_batch_attention_workspace(C.byref(a))
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
        stream = torch.cuda.Stream()
        K.check(K.lib().kllm_batch_attention(C.byref(a), stream.cuda_stream))
        torch.cuda.synchronize()
        calls.append((a, stream, o, o.clone(), (own, q, lens, ws)))
    for a, stream, o, want, _ in calls:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for a, stream, *_ in calls:
            K.check(K.lib().kllm_batch_attention(C.byref(a), stream.cuda_stream))
    torch.cuda.synchronize()
    for a, stream, o, want, _ in calls:
        assert torch.equal(o, want)


@pytest.mark.parametrize("n", [1, 40])
def test_a_prefix_past_32_bits(gpu, n):
    """2^31 codes of keys and of values: every weight is one, the last
    position alone has a value.  Its share is exact but for the tolerance
    above (S = 0)."""
    import torch

    import kmap_b200 as K
    import servecases as S
    nkv, hd, mp = 8, 128, (1 << 21) + 77
    codes = torch.zeros(2, nkv, mp, hd, dtype=torch.uint8, device="cuda")
    codes[1, :, mp - 1] = torch.arange(1, 1 + hd, device="cuda", dtype=torch.uint8).clamp(max=127)
    scales = torch.ones(nkv, mp, device="cuda")
    c = K.KvCache(S.FORMATS["i8"], 1, nkv, hd, mp, codes[0].data_ptr(), codes[1].data_ptr(), scales.data_ptr(),
                  scales.data_ptr(), nkv * mp * hd, nkv * mp)

    class Prefix:
        pass
    pre = Prefix()
    pre.c = c
    q, out = torch.ones(n, nkv * hd, device="cuda"), torch.zeros(n, nkv * hd, device="cuda")
    S.run_attention(q, out, nkv, 1.0, pre, mp)
    want = np.minimum(np.arange(1, 1 + hd), 127) / mp
    got = out.cpu().numpy().astype(np.float64).reshape(n, nkv, hd)
    assert (np.abs(got - want) <= 4 * 2.0 ** -18 * want).all()
