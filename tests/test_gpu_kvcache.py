"""The quantised key/value cache: kllm_kv_append and kllm_kv_read.

The stored codes and scales are defined by fp32 operations that are each
rounded once, so they are compared bit for bit with the plain definition on
the host; so are the turned queries and the values read back (one product)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _case(rng, rows, nh, nkv, hd, gap=0):
    x = rng.standard_normal((rows, (nh + 2 * nkv) * hd + gap)).astype(np.float32)
    ang = np.outer(np.arange(300), 10000.0 ** (-np.arange(0, hd, 2) / hd))
    ang = np.concatenate([ang, ang], -1)
    return x, np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _heads(x, nh, nkv, hd):
    y = x[:, :(nh + 2 * nkv) * hd].reshape(len(x), nh + 2 * nkv, hd)
    return y[:, :nh], y[:, nh:nh + nkv], y[:, nh + nkv:]


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 32), (8, 1, 64), (3, 3, 64), (32, 8, 128), (5, 5, 128)])
@pytest.mark.parametrize("rows,gap,rope", [(1, 0, True), (7, 4, True), (33, 3, True), (130, 0, False)])
def test_rows_of_many_sequences(gpu, fmt, nh, nkv, hd, rows, gap, rope):
    """One row per sequence at its own position; rows outside the cache or the
    angle tables (negative, past the end) leave everything as it was.  A row
    stride that is no multiple of four floats takes the unaligned loads."""
    import torch

    import kmap_b200 as K
    import servecases as S
    rng = np.random.default_rng(rows * hd + nh)
    x, cos, sin = _case(rng, rows, nh, nkv, hd, gap)
    mp, off = 37, 11
    pos = rng.integers(0, mp, rows).astype(np.int32)
    seq = rng.permutation(rows).astype(np.int32)
    if rows > 4:
        pos[1], pos[2], seq[3], seq[4] = -1, mp, -1, rows
    skip = (pos < 0) | (pos >= mp) | (seq < 0) | (seq >= rows)
    cache = S.Cache(fmt, rows, nkv, mp, hd, pad=16, fill=7)
    dx, dc, ds, dp, dq = S.dev(x), S.dev(cos), S.dev(sin), S.dev(pos), S.dev(seq)
    q_out = torch.full((rows, nh * hd), -5.0, device="cuda")
    at, w = dx.data_ptr(), 4 * hd
    r = K.KvRows(rows, nh, 0, 300, off, dq.data_ptr(), dp.data_ptr(), at, at + w * nh,
                 at + w * (nh + nkv), x.shape[1], hd, q_out.data_ptr(),
                 dc.data_ptr() if rope else None, ds.data_ptr() if rope else None)
    before = {n: cache.raw(n) for n in "kv"}
    K.check(K.lib().kllm_kv_append(cache.by(), C.byref(r), None))
    torch.cuda.synchronize()
    q, k, v = _heads(x, nh, nkv, hd)
    ang = np.where(skip, 0, pos + off)
    if rope:
        q, k = (S.rope32(t, cos[ang], sin[ang]) for t in (q, k))
    want_q = np.where(skip[:, None], np.float32(-5), q.reshape(rows, -1))
    assert np.array_equal(q_out.cpu().numpy(), want_q)
    for name, new in (("k", k), ("v", v)):
        codes, scale = S.quantise(new, fmt)
        got, got_s = cache.raw(name)
        want, want_s = before[name]
        want = want.copy()
        for i in range(rows):
            if not skip[i]:
                want[seq[i], :, pos[i]] = codes[i]
        assert np.array_equal(got, want, equal_nan=True)
        if scale is not None:
            want_s = want_s.copy()
            for i in range(rows):
                if not skip[i]:
                    want_s[seq[i], :, pos[i]] = scale[i]
            assert np.array_equal(got_s, want_s, equal_nan=True)
    # and back, into rows with a gap between heads
    back = [torch.full((rows, nkv, hd + gap), -3.0, device="cuda") for _ in "kv"]
    K.check(K.lib().kllm_kv_read(cache.by(), rows, dq.data_ptr(), dp.data_ptr(), 0,
                                 back[0].data_ptr(), back[1].data_ptr(), nkv * (hd + gap), hd + gap,
                                 None))
    torch.cuda.synchronize()
    for new, b in ((k, back[0]), (v, back[1])):
        want = S.values32(*S.quantise(new, fmt))
        want = np.where(skip[:, None, None], np.float32(-3), want)
        b = b.cpu().numpy()
        assert np.array_equal(b[..., :hd], want)
        assert (b[..., hd:] == -3).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("n,pos0", [(1, 0), (96, 4), (101, 0), (250, 50)])
def test_prompt_from_a_cache_layout(gpu, fmt, n, pos0):
    """Consecutive positions of one sequence, k and v in the prompt pass's own
    layout ([head][position][dim]), no q; rows past the cache are dropped."""
    import torch

    import kmap_b200 as K
    import servecases as S
    nkv, hd, mp, src = 4, 64, 200, 260
    rng = np.random.default_rng(n)
    k, v = (rng.standard_normal((nkv, src, hd)).astype(np.float32) for _ in "kv")
    dk, dv = S.dev(k), S.dev(v)
    cache = S.Cache(fmt, 1, nkv, mp, hd)
    r = K.KvRows(n, 0, pos0, 0, 0, None, None, None, dk.data_ptr(), dv.data_ptr(), hd, src * hd)
    K.check(K.lib().kllm_kv_append(cache.by(), C.byref(r), None))
    torch.cuda.synchronize()
    m = min(n, mp - pos0)
    for name, x in (("k", k), ("v", v)):
        codes, scale = S.quantise(x[:, :m], fmt)
        got, got_s = cache.raw(name)
        assert np.array_equal(got[0, :, pos0:pos0 + m], codes)
        if scale is not None:
            assert np.array_equal(got_s[0, :, pos0:pos0 + m], scale)
            assert np.isnan(got_s[0, :, :pos0]).all() and np.isnan(got_s[0, :, pos0 + m:]).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_odd_values(gpu, fmt):
    """Zeros, denormals, the type's largest, an infinity, a NaN."""
    import torch

    import kmap_b200 as K
    import servecases as S
    hd = 64
    x = np.zeros((7, hd), np.float32)
    x[1] = 1e-40
    x[2, 5] = -np.finfo(np.float32).max
    x[3, 9], x[4, 9], x[5, 63] = np.inf, np.nan, -np.inf
    x[6] = np.linspace(-1, 1, hd)
    d = S.dev(x)
    cache = S.Cache(fmt, 1, 1, 7, hd)
    r = K.KvRows(7, 0, 0, 0, 0, None, None, None, d.data_ptr(), d.data_ptr(), hd, hd)
    K.check(K.lib().kllm_kv_append(cache.by(), C.byref(r), None))
    out = torch.zeros(7, hd, device="cuda")
    K.check(K.lib().kllm_kv_read(cache.by(), 7, None, None, 0, out.data_ptr(), out.data_ptr(), hd,
                                 hd, None))
    got = out.cpu().numpy()
    assert np.array_equal(got, S.values32(*S.quantise(x, fmt)), equal_nan=True)
    assert (got[:2] == 0).all() and np.isnan(got[3:6]).all() and np.isfinite(got[2]).all()
    # within half a step of the largest value's code
    step = 1 / 127 if fmt == "i8" else 2.0 ** -3
    assert (np.abs(got[6] - x[6]) <= step / 2 * (1 + 2.0 ** -20)).all()


def test_nothing_to_do(gpu):
    import kmap_b200 as K
    import servecases as S
    cache = S.Cache("i8", 1, 1, 4, 32)
    r = K.KvRows(0, 0, 0, 0, 0, None, None, None, 16, 16, 32, 32)
    n = K.lib().kllm_launch_count()
    K.check(K.lib().kllm_kv_append(cache.by(), C.byref(r), None))
    K.check(K.lib().kllm_kv_read(cache.by(), 0, None, None, 0, 16, 16, 32, 32, None))
    assert K.lib().kllm_launch_count() == n


@pytest.mark.parametrize("fmt", ["i8", "f32"])
def test_in_a_graph(gpu, fmt):
    """A captured append, replayed with new rows and positions, on another stream."""
    import torch

    import kmap_b200 as K
    import servecases as S
    rng = np.random.default_rng(3)
    n, nkv, hd, mp = 5, 2, 64, 40
    x = [rng.standard_normal((n, 2 * nkv, hd)).astype(np.float32) for _ in range(3)]
    at = [rng.permutation(mp)[:n].astype(np.int32) for _ in range(3)]
    a, b = S.Cache(fmt, n, nkv, mp, hd), S.Cache(fmt, n, nkv, mp, hd)
    dx, dp = S.dev(x[0]), S.dev(at[0])

    def call(cache, stream):
        r = K.KvRows(n, 0, 0, 0, 0, None, dp.data_ptr(), None, dx.data_ptr(), dx.data_ptr() + 4 * nkv * hd,
                     2 * nkv * hd, hd)
        K.check(K.lib().kllm_kv_append(cache.by(), C.byref(r), stream))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        call(a, torch.cuda.current_stream().cuda_stream)
    for xi, pi in zip(x, at):
        dx.copy_(S.dev(xi))
        dp.copy_(S.dev(pi))
        graph.replay()
        call(b, None)
        torch.cuda.synchronize()
    for t in ("k", "v", "ks", "vs"):
        assert torch.equal(getattr(a, t).nan_to_num(), getattr(b, t).nan_to_num())
        assert fmt == "f32" and t[1:] or bool((getattr(a, t).nan_to_num() != 0).any())


def test_sequences_more_than_32_bits_apart(gpu):
    """Sequences 2^31 codes apart: written, read and attended as those of a small cache."""
    import torch

    import kmap_b200 as K
    import servecases as S
    rng = np.random.default_rng(9)
    nkv, hd, mp, n = 2, 128, 16, 2
    x = S.dev(rng.standard_normal((n, 2 * nkv, hd)).astype(np.float32))
    q = S.dev(rng.standard_normal((n, 2 * nkv * hd)).astype(np.float32))
    seq, lens = S.dev(np.array([1, 0], np.int32)), S.dev(np.array([3, 3], np.int32))
    pos = S.dev(np.array([2, 2], np.int32))
    got = []
    for pad in (0, 2 ** 31 + 64):
        c = S.Cache("i8", n, nkv, mp, hd)
        c.stride += pad
        c.k, c.v = (torch.zeros(c.stride + nkv * mp * hd, dtype=torch.uint8, device="cuda") for _ in "kv")
        c.ks.zero_(), c.vs.zero_()
        c.c.k, c.c.v, c.c.seq_stride = c.k.data_ptr(), c.v.data_ptr(), c.stride
        r = K.KvRows(n, 0, 0, 0, 0, seq.data_ptr(), pos.data_ptr(), None, x.data_ptr(),
                     x.data_ptr() + 4 * nkv * hd, 2 * nkv * hd, hd)
        K.check(K.lib().kllm_kv_append(c.by(), C.byref(r), None))
        back = torch.zeros(2, n, nkv, hd, device="cuda")
        K.check(K.lib().kllm_kv_read(c.by(), n, seq.data_ptr(), pos.data_ptr(), 0, back[0].data_ptr(),
                                     back[1].data_ptr(), nkv * hd, hd, None))
        out = torch.zeros(n, 2 * nkv * hd, device="cuda")
        S.run_attention(q, out, 2 * nkv, 0.1, own=c, lens=lens, max_len=mp)
        got.append((back, out))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert bool((got[0][0] != 0).any(-1).all()) and bool((got[0][1] != 0).any(-1).all())
