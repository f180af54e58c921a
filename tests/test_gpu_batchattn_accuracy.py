"""How many bits kllm_batch_attention keeps of queries, keys, weights and values,
on inputs that leave its other roundings little to do.

A query row has one element that is not zero, so a score is one product; each
output dim has one position with a value (every position has one in the last dim
besides, so that none is a row of zeros).  |s| <= 1.5.  Then out_d = p_j v_jd / L,
relative to which, in units of 2^-24:
  queries (2^-22 of the element) and keys (2^-21, cut to two terms) change a
  score by 12 |s|, a weight and the sum L by that at most      2 x 18
  three roundings of a score in log2 (|s| log2 e < 2.2), exp2    2 x 15
  weight and value to two terms, their product without the
  smallest (4 + 8 + 4), cut off while it is added (2 a term)         24
  corrections by exp2 where the maximum moves, some 10               40
  L: at most 64 additions a thread, 40 tiles, 74 parts              180
in all 310 < 2^-24 x 2^8.3: the bound is 2^-15.5.  A form that leaves out the
second term of any operand is off by up to 2^-11, which the last test shows on
the host for these inputs."""
import numpy as np
import pytest

TOL = 2.0 ** -15.5
# (hd, nh, nkv, n, P): the few-row kernel, the 128-row tiles
NARROW = [(128, 8, 2, 5, 300), (64, 8, 1, 3, 517), (32, 4, 4, 9, 1000)]
WIDE = [(128, 8, 2, 64, 3001), (128, 4, 4, 129, 3000), (64, 8, 1, 41, 2500), (64, 8, 8, 33, 4100),
        (32, 8, 2, 35, 3700)]


def sparse(seed, hd, nh, nkv, n, P):
    """q [n][nh][hd], k and v [nkv][P][hd] as above; dims 0..3 carry scores."""
    rng = np.random.default_rng(seed)
    q = np.zeros((n, nh, hd), np.float32)
    at = rng.integers(0, 4, (n, nh))
    i, h = np.mgrid[:n, :nh]
    q[i, h, at] = rng.uniform(1, 1.5, (n, nh)) * rng.choice([-1, 1], (n, nh))
    k = np.zeros((nkv, P, hd), np.float32)
    k[..., :4] = rng.uniform(-1, 1, (nkv, P, 4))
    v = np.zeros((nkv, P, hd), np.float32)
    v[..., hd - 1] = rng.uniform(1, 2, (nkv, P))
    for g in range(nkv):
        v[g, rng.permutation(P)[:hd - 1], np.arange(hd - 1)] = rng.uniform(1, 2, hd - 1)
    return q, k, v


def exact(q, k, v):
    """Output [n][nh][hd] and the mean of the rows' largest |v|, weighted as the output is, in 64 bits."""
    n, nh, hd = q.shape
    nkv = k.shape[0]
    x = q.astype(np.float64).reshape(n, nkv, nh // nkv, hd)
    out, norm = np.empty(x.shape), np.empty(x.shape[:3])
    for g in range(nkv):
        s = x[:, g] @ k[g].astype(np.float64).T
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, g], norm[:, g] = p @ v[g].astype(np.float64), p @ np.abs(v[g]).max(-1)
    return out.reshape(n, nh, hd), norm.reshape(n, nh)


def run(fmt, q, k, v, own=0):
    """kllm_batch_attention of q on a prefix k, v but its last `own` positions, which every
    sequence has in a cache of its own.  The output and the keys and values that the caches hold."""
    import torch

    import servecases as S
    n, nh, hd = q.shape
    nkv, P = k.shape[:2]
    pre = S.Cache(fmt, 1, nkv, P - own, hd)
    held = [pre.put(name, x[None, :, :P - own])[0] for name, x in (("k", k), ("v", v))]
    mine = lens = None
    if own:
        mine = S.Cache(fmt, n, nkv, own, hd)
        lens = S.dev(np.full(n, own, np.int32))
        for j, (name, x) in enumerate((("k", k), ("v", v))):
            y = mine.put(name, np.broadcast_to(x[None, :, P - own:], (n, nkv, own, hd)).copy())
            held[j] = np.concatenate([held[j], y[0]], 1)
    out = torch.zeros(n, nh * hd, device="cuda")
    S.run_attention(S.dev(q.reshape(n, -1)), out, nh, 1.0, pre, P - own, mine, lens, own)
    return out.cpu().numpy().astype(np.float64).reshape(q.shape), *held


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", NARROW + WIDE)
@pytest.mark.parametrize("own", [0, 3])
def test_every_operand_keeps_its_second_term(gpu, fmt, hd, nh, nkv, n, P, own):
    q, k, v = sparse(hd + n, hd, nh, nkv, n, P)
    got, k, v = run(fmt, q, k, v, own)
    want, _ = exact(q, k, v)
    assert (np.abs(got - want) <= TOL * np.abs(want)).all()


def _two(x, drop=False):
    """Two terms of 11 bits, or one."""
    hi = np.float16(x).astype(np.float64)
    return hi if drop else hi + np.float16(x - hi).astype(np.float64)


@pytest.mark.parametrize("hd,nh,nkv,n,P", NARROW + WIDE)
def test_one_term_would_show(hd, nh, nkv, n, P):
    """The bound on these inputs, on the host: met with two terms of everything, not with one term
    of the queries, the keys, the weights or the values."""
    q, k, v = sparse(hd + n, hd, nh, nkv, n, P)
    want, _ = exact(q, k, v)
    at = {}
    for drop in (None, "q", "k", "p", "v"):
        qq, kk, vv = (_two(x.astype(np.float64) * 2.0 ** 13, drop == name) * 2.0 ** -13
                      for name, x in (("q", q), ("k", k), ("v", v)))
        x = qq.reshape(n, nkv, nh // nkv, hd)
        out = np.empty(x.shape)
        for g in range(nkv):
            s = x[:, g] @ kk[g].T
            p = np.exp(s - s.max(-1, keepdims=True))
            out[:, g] = _two(p * 2.0 ** 13, drop == "p") * 2.0 ** -13 @ vv[g] / p.sum(-1, keepdims=True)
        err = np.abs(out.reshape(want.shape) - want)
        at[drop] = (err[want != 0] / np.abs(want[want != 0])).max()
    assert at.pop(None) < TOL / 8
    assert min(at.values()) > 4 * TOL, at


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", NARROW + WIDE)
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 30, 2.0 ** 100])
def test_a_key_beside_much_larger_ones(gpu, fmt, hd, nh, nkv, n, P, size):
    """Every 16th key has a very large element where the queries have none: it changes
    no score, and no other key's.

    The 128-row tiles bring an fp32 key's largest element to [2^13, 2^14) and round its second
    terms to multiples of 2^-24 there: the key's smaller elements are off by up to 2^-38 of the
    largest, or are lost (a change by their score).  Such a position's weight is off by
    e^d - 1, d = min(2^-38 size |q|, |s|) at most, and with L, of which it is 1 / 16, every
    output by that times its share."""
    q, k, v = sparse(hd + n, hd, nh, nkv, n, P)
    k[:, 3::16, 5] = size
    got, k, v = run(fmt, q, k, v)
    want, _ = exact(q, k, v)
    tol = np.full(want.shape, TOL)
    if fmt == "f32" and (hd, nh, nkv, n, P) in WIDE:
        x = q.astype(np.float64).reshape(n, nkv, nh // nkv, hd)
        tol = tol.reshape(x.shape)
        for g in range(nkv):
            s = x[:, g] @ k[g].T
            p = np.exp(s)
            d = np.minimum(2.0 ** -38 * size * np.abs(x[:, g]).sum(-1), 1.5)[..., None] * (np.arange(P) % 16 == 3)
            d = np.expm1(np.minimum(d, np.abs(s)))
            share = (p * d).sum(-1, keepdims=True) / p.sum(-1, keepdims=True)
            # the position that dim e's value comes from: its own weight is off too
            own = np.zeros(x[:, g].shape)
            for e in range(hd - 1):
                own[..., e] = d[..., np.nonzero(v[g, :, e])[0][0]]
            own[..., hd - 1] = 2 * share[..., 0]        # (values of 1 to 2 at every position)
            tol[:, g] += own + share + own * share
        tol = tol.reshape(want.shape)
    assert (np.abs(got - want) <= tol * np.abs(want)).all()


def _spread(seed, hd, nh, nkv, n, P):
    """As sparse(), with dim 4 for scores that all query rows share."""
    q, k, v = sparse(seed, hd, nh, nkv, n, P)
    q[..., 4] = 1
    return q, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", NARROW + WIDE)
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 30, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("step", [16, 601])
def test_values_beside_much_larger_ones_without_weight(gpu, fmt, hd, nh, nkv, n, P, size, step):
    """Every 16th (or 601st) position has a very large value and a weight of e^-300: nothing
    of it shows, and nothing of the others is lost."""
    q, k, v = _spread(hd + n, hd, nh, nkv, n, P)
    k[:, 3::step, 4] = -300
    v[:, 3::step] = 0
    v[:, 3::step, hd - 1] = size
    got, k, v = run(fmt, q, k, v, 2)
    want, _ = exact(q, k, v)
    assert (np.abs(got - want) <= TOL * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", NARROW + WIDE)
def test_values_of_every_size(gpu, fmt, hd, nh, nkv, n, P):
    """Value rows of 2^-30 to 2^30 whose weights nearly make up for it: every position counts.
    Scores reach |s| = 21, where a score's roundings come to 2 (12 |s|) + 2 (3 |s| log2 e / 2) of the
    units above, 595: with the 310 there less than 2^10, 2^-14 of the mean largest value."""
    rng = np.random.default_rng(hd)
    q, k, _ = _spread(hd + n, hd, nh, nkv, n, P)
    e = rng.uniform(-30, 30, (nkv, P))
    v = (rng.uniform(-1, 1, (nkv, P, hd)) * 2.0 ** e[..., None]).astype(np.float32)
    k[..., :4] *= np.float32(0.2)
    k[..., 4] = -0.9 * np.log(2) * e + rng.uniform(-1, 1, (nkv, P))
    got, k, v = run(fmt, q, k, v, 3)
    want, norm = exact(q, k, v)
    assert (np.abs(got - want) <= 2.0 ** -14 * norm[..., None]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["i8", "e4m3", "f32"])
@pytest.mark.parametrize("hd,nh,nkv,n,P", [NARROW[0], WIDE[0]])
def test_values_without_any(gpu, fmt, hd, nh, nkv, n, P):
    """Rows of zeros among the values, a tile of them, and all of them."""
    q, k, v = sparse(hd + n, hd, nh, nkv, n, P)
    v[:, 5::7] = 0
    v[:, :140] = 0
    got, kk, vv = run(fmt, q, k, v, 3)
    want, _ = exact(q, kk, vv)
    assert (np.abs(got - want) <= TOL * np.abs(want)).all()
    got, _, _ = run(fmt, q, k, 0 * v, 3)
    assert (got == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,P", [("i8", 1000003), ("e4m3", 1000003), ("f32", 500003)])
def test_sums_over_many_positions(gpu, fmt, P):
    """The mean of a million values of one sign, all weights being one: additions that are cut
    off instead of rounded lean one way and would add up.

    A part's sum takes 32 cut additions (8 bits; fp32: four, its other sums are rounded), each
    of at most 2^-23 of a partial sum that is half the whole in the mean: 2^-19.  Some 2^9 parts
    and turns are added with roundings of either sign: six standard deviations of
    2^-25 sqrt(2^9 / 3) are 2^-18.7.  Together less than 2^-17."""
    import torch

    import kmap_b200 as K
    import servecases as S
    nkv, hd = 32, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    if fmt == "f32":
        x = torch.rand(nkv, P, hd, generator=g, device="cuda") + 1
        mean = torch.stack([x[h].sum(0, dtype=torch.float64) / P for h in range(nkv)])
    else:
        x = torch.randint(40, 120, (nkv, P, hd), generator=g, device="cuda", dtype=torch.uint8)
        if fmt == "e4m3":      # codes of 0x40 to 0x50: 2 to 8
            x = (x & 15) + 0x40
        y = x.view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn)
        mean = torch.stack([y[h].float().sum(0, dtype=torch.float64) / P for h in range(nkv)])
    scales = torch.full((nkv, P), 0.8, device="cuda")
    c = K.KvCache(S.FORMATS[fmt], 1, nkv, hd, P, x.data_ptr(), x.data_ptr(), scales.data_ptr(), scales.data_ptr(),
                  nkv * P * hd, nkv * P)

    class Prefix:
        pass
    pre = Prefix()
    pre.c = c
    if fmt != "f32":
        mean *= float(np.float32(0.8))
    q, out = torch.zeros(1, nkv * hd, device="cuda"), torch.zeros(1, nkv * hd, device="cuda")
    S.run_attention(q, out, nkv, 1.0, pre, P)
    err = ((out.view(nkv, hd).double() - mean) / mean).abs().max().item()
    del x, scales, pre, c
    torch.cuda.empty_cache()
    assert err <= 2.0 ** -17
